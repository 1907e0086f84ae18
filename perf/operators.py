"""Operators around and inside the expert layers, as a user's program calls them, with their plain forms.

Six operators, three pairs that are used together:

  norm / norm_grad      residual addition + root-mean-square norm + 1x128 quantisation to e4m3 (what feeds the 8-bit
                        grouped GEMM), and its gradient
  route / route_grad    top-k routing from softmax or sigmoid scores with bias and groups, and its gradient
  quant4 / product4     quantisation to 4-bit blocks (nvfp4: 16 values under an e4m3 scale and one fp32 factor;
                        mxfp4: 32 values under a power of two) and the grouped product of such operands

``run`` computes them from elementary torch operations, or, where ``own`` is true, through tirx_harness_b200.
"""
import math

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
#: e2m1 magnitudes by code; the sign is bit 3
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BLOCK = {"nvfp4": 16, "mxfp4": 32}          # values under one scale
WORDS = {"nvfp4": 4, "mxfp4": 2}            # 512-byte scale tiles per 256 values of K


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a decode step of a few sequences at the model width of the MoE layer: latency
        dict(name="norm, 8 tokens", op="norm", T=8, H=7168, dtype="bf16", residual=True, pow2=True, mn=False, y=True),
        # the MoE layer's own prefill batch: 16384 tokens of hidden 7168
        dict(name="norm, 16384 tokens", op="norm", T=16384, H=7168, dtype="bf16", residual=True, pow2=False, mn=True, y=False),
        # training micro-batches: an odd one in fp32 without a residual stream, and a full one
        dict(name="norm gradient, 517 x 2048 fp32", op="norm_grad", T=517, H=2048, dtype="fp32", dh=False),
        dict(name="norm gradient, 8192 x 7168", op="norm_grad", T=8192, H=7168, dtype="bf16", dh=True),
        # one token among the decode layer's 512 experts, softmax
        dict(name="route, 1 token of 512", op="route", T=1, E=512, k=10, dtype="bf16", score="softmax", bias=False, n_group=1,
             topk_group=1, group_score="max", renorm=True, masked=False),
        # the registered layer's router (256 experts in 8 groups, sigmoid with a balancing bias) over a prefill batch
        dict(name="route, 16384 tokens in groups", op="route", T=16384, E=256, k=8, dtype="fp32", score="sigmoid", bias=True, n_group=8,
             topk_group=4, group_score="top2", renorm=True, masked=False),
        # gradients: an odd batch of masked 16-bit sigmoid logits, and the MoE layer's 16384 tokens of softmax
        dict(name="route gradient, 777 sigmoid", op="route_grad", T=777, E=160, k=6, dtype="bf16", score="sigmoid", renorm=True, masked=True),
        dict(name="route gradient, 16384 softmax", op="route_grad", T=16384, E=256, k=8, dtype="fp32", score="softmax", renorm=True, masked=False),
        # the activations between the two expert products of a small ragged batch: SiLU(gate) * up, then 4 bits
        dict(name="quantise SiLU*mul, 333 mxfp4", op="quant4", T=333, K=2048, dtype="bf16", fmt="mxfp4", kind="silu", top_k=1),
        # the prefill batch's tokens gathered into the experts' rows (top 2 of them kept on this GPU)
        dict(name="quantise gathered, 32768 nvfp4", op="quant4", T=16384, K=7168, dtype="bf16", fmt="nvfp4", kind="gather", top_k=2),
        # one token's eight experts: a masked layout with one row at most, bound by the weights
        dict(name="product, 1 token in 8 experts", op="product4", layout="masked", G=8, M=1, N=4096, K=7168, fmt="mxfp4", align=1, out="bf16"),
        # prefill: 32 experts, ragged groups, the gate_up shape
        dict(name="product, 32 experts prefill", op="product4", layout="contiguous", G=32, M=28672, N=4096, K=7168, fmt="nvfp4", align=128, out="bf16"),
    ]


def _spread(rng, low, high, step=1):
    """Log-uniform whole number of [low, high], a multiple of `step`."""
    v = math.exp(rng.uniform(math.log(low), math.log(high + 0.999)))
    return max(low, min(high, int(v / step) * step))


def draw(rng):
    op = rng.choice(("norm", "norm_grad", "route", "route_grad", "quant4", "product4"))
    if op in ("norm", "norm_grad"):
        H = _spread(rng, 128, 8192, 8)
        d = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        top = (16384 if op == "norm" else 8192) * 7168 * 2 // (H * SIZE[d])
        T = _spread(rng, 1, min(top, 16384))
        if op == "norm_grad":
            return dict(op=op, T=T, H=H, dtype=d, dh=rng.random() < 0.5)
        return dict(op=op, T=T, H=H, dtype=d, residual=rng.random() < 0.6, pow2=T * H < 1 << 20 and rng.random() < 0.5,
                    mn=rng.random() < 0.5, y=rng.random() < 0.4)
    if op in ("route", "route_grad"):
        c = dict(op=op, T=_spread(rng, 1, 16384), dtype=rng.choice(("fp32", "bf16", "fp16")), score=rng.choice(("softmax", "sigmoid")),
                 renorm=rng.random() < 0.7, masked=rng.random() < 0.3)
        groups = rng.choice((1, 1, 4, 8)) if op == "route" else 1
        E = _spread(rng, 8, 256 // groups) * groups
        c.update(E=E, k=rng.randint(1, 8))
        c["renorm"] = c["renorm"] and c["k"] > 1           # one renormalised weight is the constant 1: no gradient to compare
        if op == "route":
            c.update(bias=rng.random() < 0.5, n_group=groups, topk_group=1 if groups == 1 else rng.randint(2, groups),
                     group_score=rng.choice(("max", "top2")))
        return c
    if op == "quant4":
        kind = rng.choice(("rows", "gather", "silu"))
        K = _spread(rng, 128, 7168, 128)
        top_k = rng.randint(1, 4) if kind == "gather" else 1
        T = _spread(rng, 1, min(16384, 16384 * 7168 // (K * top_k)))
        return dict(op=op, T=T, K=K, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), fmt=rng.choice(("nvfp4", "mxfp4")), kind=kind, top_k=top_k)
    layout = rng.choice(("masked", "contiguous"))
    G, N, K = _spread(rng, 1, 32), _spread(rng, 64, 7168, 8), _spread(rng, 128, 7168, 128)
    G = min(G, max(1, 32 * 4096 * 7168 // (N * K)))
    M = _spread(rng, 1, 256) if layout == "masked" else _spread(rng, 1, min(16384, 28672 * 4096 * 7168 // (N * K)))
    return dict(op=op, layout=layout, G=G, M=M, N=N, K=K, fmt=rng.choice(("nvfp4", "mxfp4")), align=rng.choice((1, 16, 128)),
                out=rng.choice(("bf16", "bf16", "fp32")))


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _counts(case, seed):
    """Rows of each group: between half and one and a half of the mean (masked layout: between none and all)."""
    cpu = torch.Generator()
    cpu.manual_seed(seed + 77)
    G, M = case["G"], case["M"]
    if case["layout"] == "masked":
        counts = torch.randint(0, M + 1, (G,), generator=cpu) if M > 1 else torch.ones(G, dtype=torch.int64)
        counts[seed % G] = M
        return counts
    share = 0.5 + torch.rand(G, generator=cpu)
    counts = (share * (M / share.sum())).long()
    counts[seed % G] += M - counts.sum()
    return counts


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op in ("norm", "norm_grad"):
        T, H, dt = case["T"], case["H"], DT[case["dtype"]]
        loud = 1 + 7 * (torch.rand(H, generator=g, device=DEV) < 0.01).float()       # a few outlier channels
        s = dict(case=case, weight=(1 + 0.1 * _randn(g, H)).to(dt))
        x = (_randn(g, T, H) * loud).to(dt)
        if op == "norm":
            s.update(x=x, residual=(3 * _randn(g, T, H)).to(dt) if case["residual"] else None)
        else:
            # what the forward pass kept: its sum and the reciprocal root mean square
            s.update(h=x, rstd=(x.double().square().mean(1) + 1e-6).rsqrt().float(), dy=_randn(g, T, H).to(dt),
                     dh=_randn(g, T, H).to(dt) if case["dh"] else None)
        return s
    if op in ("route", "route_grad"):
        T, E, k = case["T"], case["E"], case["k"]
        logits = (1.5 * _randn(g, T, E)).to(DT[case["dtype"]])
        if case["masked"]:               # experts that are switched off, and one padding token with all of them off
            logits[:, torch.rand(E, generator=g, device=DEV) < 0.1] = -math.inf
            if T > 2:
                logits[T // 2] = -math.inf
        s = dict(case=case, logits=logits)
        if op == "route":
            s["bias"] = 0.05 * _randn(g, E) if case["bias"] else None
        else:
            key = torch.where(logits == -math.inf, torch.tensor(-math.inf, device=DEV), logits.float())
            top = key.sort(dim=1, descending=True, stable=True)
            s["ids"] = torch.where(top.values[:, :k] == -math.inf, -1, top.indices[:, :k]).int().contiguous()
            s["grad"] = _randn(g, T, k)
        return s
    if op == "quant4":
        T, K, kind, fmt = case["T"], case["K"], case["kind"], case["fmt"]
        x = _randn(g, T, 2 * K if kind == "silu" else K) * torch.exp2(2 * _randn(g, T, 1))
        s = dict(case=case, x=x.to(DT[case["dtype"]]), src=None)
        rows = T
        if kind == "gather":             # every expert's rows padded to 128: negative entries are padding
            pairs = T * case["top_k"]
            rows = (pairs + 127) // 128 * 128
            src = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
            src[:pairs] = torch.randperm(pairs, generator=g, device=DEV).int()
            s["src"] = src
        # the factor a calibration run gives
        s["factor"] = (x.abs().amax() / (448 * 6)).float().reshape(1) if fmt == "nvfp4" else None
        s["q"] = torch.zeros((rows, K // 2), dtype=torch.uint8, device=DEV)
        s["sf"] = torch.zeros(((rows + 127) // 128, (K + 255) // 256 * WORDS[fmt], 512), dtype=torch.uint8, device=DEV)
        return s
    G, M, N, K, fmt = (case[k] for k in ("G", "M", "N", "K", "fmt"))
    wq = torch.empty((G, N, K // 2), dtype=torch.uint8, device=DEV)
    wsf = torch.empty((G, (N + 127) // 128, (K + 255) // 256 * WORDS[fmt], 512), dtype=torch.uint8, device=DEV)
    wf = (5 / (448 * 6 * math.sqrt(K))) * (1 + torch.rand(G, generator=g, device=DEV))
    for e in range(G):
        c, b = _codes(_randn(g, N, K) / math.sqrt(K), fmt, wf[e])
        wq[e], wsf[e] = _pack(c), _tile(b, fmt)
    af = torch.full((1,), 5 / (448 * 6), device=DEV)
    counts = _counts(case, seed)
    s = dict(case=case, b=wq, sfb=wsf, alpha=(af * wf).contiguous() if fmt == "nvfp4" else None)
    if case["layout"] == "masked":
        rows, shape = G * M, (G, M)
        s["masked_m"] = counts.int().to(DEV)
        valid = (torch.arange(M)[None] < counts[:, None]).reshape(-1)
        s["group"] = torch.where(valid, torch.arange(G).repeat_interleave(M), -1).int().to(DEV)
        slot = torch.arange(M).repeat(G)
        s["cap"] = M
    else:
        al = case["align"]
        padded = (counts + al - 1) // al * al
        start = torch.cumsum(padded, 0) - padded
        rows = M + G * (al - 1)            # the fixed capacity a plan reserves; what no group fills is padding
        shape = (rows,)
        group = torch.full((rows,), -1, dtype=torch.int32)
        slot = torch.zeros(rows, dtype=torch.int64)
        for e in range(G):
            group[start[e]:start[e] + counts[e]] = e
            slot[start[e]:start[e] + counts[e]] = torch.arange(int(counts[e]))
        s["group"] = group.to(DEV)
        s["cap"] = max(1, int(counts.max()))
    s["slot"] = slot.to(DEV)
    c, b = _codes(_randn(g, rows, K), fmt, af)
    s["a"] = _pack(c).byte().reshape(*shape, K // 2)
    s["sfa"] = torch.stack([_tile(x, fmt) for x in b.reshape(G, M, -1)]) if case["layout"] == "masked" else _tile(b, fmt)
    s["d"] = torch.zeros((*shape, N), dtype=DT[case["out"]], device=DEV)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _codes(x, fmt, factor):
    """x [rows, K] in 32 bits -> (e2m1 codes, scale bytes [rows, K / block]), each of them rounded to nearest, ties to even."""
    v = x.reshape(x.shape[0], -1, BLOCK[fmt])
    amax = v.abs().amax(2)
    if fmt == "nvfp4":
        scale = (amax / (6 * factor)).clamp(max=448).to(torch.float8_e4m3fn)
        byte, unit = scale.view(torch.uint8), scale.to(x.dtype) * factor
    else:
        e = torch.where(amax > 0, torch.frexp(amax).exponent + (127 - 3), 0).clamp(0, 254)       # floor(log2) - 2, biased
        byte, unit = e.to(torch.uint8), _power(e)
    a = (v.abs() / torch.where(unit > 0, unit, math.inf)[..., None])
    code = (a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    return (code + 8 * torch.signbit(v)).reshape(x.shape), byte


def _power(biased):
    """2 ** (biased - 127), put together from its bits (0 stands for 2 ** -127)"""
    b = biased.int()
    return torch.where(b == 0, 1 << 22, b << 23).view(torch.float32)


def _pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _unpack(q):
    """The values of packed codes, low half first, as e4m3 (which holds all of them)."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=q.device).to(torch.float8_e4m3fn).view(torch.uint8)
    both = torch.stack((q & 15, q >> 4), dim=-1).int()
    return table[both].reshape(*q.shape[:-1], -1).view(torch.float8_e4m3fn)


def _tile(byte, fmt):
    """Scale bytes [rows, blocks] -> tiles [ceil(rows/128), ceil(K/256) * words, 512]: a tile holds 4 blocks of 128 rows,
    row r's four bytes at (r % 32) * 16 + (r // 32) * 4; what lies behind the last row and block is zero."""
    rows, blocks = byte.shape
    kt = (blocks * BLOCK[fmt] + 255) // 256 * WORDS[fmt]
    full = torch.zeros(((rows + 127) // 128 * 128, kt * 4), dtype=torch.uint8, device=byte.device)
    full[:rows, :blocks] = byte
    return full.reshape(-1, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).reshape(-1, kt, 512)


def _untile(tiles, rows, blocks):
    """[..., row blocks, kt, 512] -> [..., rows, blocks]"""
    lead, (rb, kt, _) = tiles.shape[:-3], tiles.shape[-3:]
    v = tiles.reshape(*lead, rb, kt, 32, 4, 4).movedim(-4, -2).transpose(-4, -3)      # rb, 4, 32, kt, 4
    return v.reshape(*lead, rb * 128, kt * 4)[..., :rows, :blocks]


def _value(q, sf, rows, fmt, dtype):
    """Packed codes and scale tiles -> their values."""
    K = q.shape[-1] * 2
    b = _untile(sf, rows, K // BLOCK[fmt])
    s = b.view(torch.float8_e4m3fn).to(dtype) if fmt == "nvfp4" else _power(b).to(dtype)
    return (_unpack(q).to(dtype).reshape(*q.shape[:-1], -1, BLOCK[fmt]) * s[..., None]).reshape(*q.shape[:-1], K)


def _blocks128(y):
    """[T, H] -> [T, ceil(H/128), 128], the last block filled up with zeros"""
    T, H = y.shape
    return torch.nn.functional.pad(y, (0, -H % 128)).reshape(T, -1, 128)


def _norm(s):
    c, x = s["case"], s["x"]
    h = x if s["residual"] is None else (x.float() + s["residual"].float()).to(x.dtype)
    rstd = (h.float().square().mean(1) + 1e-6).rsqrt()
    y = h.float() * rstd[:, None] * s["weight"].float()
    v = _blocks128(y)
    scale = v.abs().amax(2).clamp(min=1e-8) / 448
    if c["pow2"]:
        m, e = torch.frexp(scale)
        scale = _power(e - (m == 0.5).int() + 127)
    q = (v / scale[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).reshape(len(x), -1)[:, : c["H"]]
    return dict(q=q, scales=scale, h=h if s["residual"] is not None else None, y=y.to(x.dtype) if c["y"] else None, rstd=rstd)


def _norm_grad(s):
    h, rstd, dy = s["h"].float(), s["rstd"][:, None], s["dy"].float()
    n = h * rstd
    g = dy * s["weight"].float()
    dx = rstd * (g - n * (g * n).mean(1, keepdim=True))
    if s["dh"] is not None:
        dx = dx + s["dh"].float()
    return dict(dx=dx.to(s["h"].dtype), dw=(dy * n).sum(0))


def _scores(logits, score):
    """In 32 or 64 bits, as the logits are; 0 where the mask leaves nothing."""
    if score == "sigmoid":
        return 1 / (1 + torch.exp(-logits))
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - torch.where(top == -math.inf, 0, top))
    total = e.sum(1, keepdim=True)
    return e / torch.where(total == 0, 1, total)


def _choose(s):
    """The experts, decided in 64 bits (the scores of two of them may be closer than 32 bits tell)."""
    c = s["case"]
    logits = s["logits"].double()
    key = _scores(logits, c["score"])
    if s["bias"] is not None:
        key = key + s["bias"].double()
    key = torch.where(logits == -math.inf, -math.inf, key)
    if c["n_group"] > 1:
        per = key.reshape(len(key), c["n_group"], -1)
        best = per.sort(dim=2, descending=True).values
        g = best[..., 0]
        if c["group_score"] == "top2" and best.shape[2] > 1:
            g = g + torch.where(best[..., 1] == -math.inf, 0, best[..., 1])
        keep = g.sort(dim=1, descending=True, stable=True).indices[:, : c["topk_group"]]
        kept = torch.zeros_like(g, dtype=torch.bool).scatter_(1, keep, True)
        key = torch.where(kept[..., None], per, -math.inf).reshape(key.shape)
    top = key.sort(dim=1, descending=True, stable=True)
    return torch.where(top.values == -math.inf, -1, top.indices)[:, : c["k"]].int()


def _route(s):
    c = s["case"]
    ids = _choose(s)
    return dict(ids=ids, weights=_weights(_scores(s["logits"].float(), c["score"]), ids, c["renorm"]))


def _weights(score, ids, renorm):
    w = torch.where(ids < 0, 0, score.gather(1, ids.clamp(min=0).long()))
    return w / (w.sum(1, keepdim=True) + 1e-20) if renorm else w


def _route_grad(logits, ids, grad, c):
    p = _scores(logits, c["score"])
    at = ids.clamp(min=0).long()
    sel = torch.where(ids < 0, 0, p.gather(1, at))
    g = torch.where(ids < 0, 0, grad)
    if c["renorm"]:
        total = sel.sum(1, keepdim=True) + 1e-20
        g = torch.where(ids < 0, 0, (g - (g * sel).sum(1, keepdim=True) / total) / total)
    ds = torch.zeros_like(p).scatter_add_(1, at, g)
    if c["score"] == "sigmoid":
        return ds * p * (1 - p)
    return p * (ds - (g * sel).sum(1, keepdim=True))


def _source(s, dtype):
    """The rows that are quantised: the tokens', the gathered ones, or SiLU(gate) * up."""
    c, x = s["case"], s["x"].to(dtype)
    if c["kind"] == "gather":
        return x[(s["src"] // c["top_k"]).clamp(min=0).long()]
    if c["kind"] == "silu":
        gate, up = x[:, : c["K"]], x[:, c["K"]:]
        return gate / (1 + torch.exp(-gate)) * up
    return x


def _quant4(s):
    c = s["case"]
    code, byte = _codes(_source(s, torch.float32), c["fmt"], s["factor"])
    q = _pack(code)
    sf = _tile(byte, c["fmt"])
    if c["kind"] == "gather":            # padding rows keep what the buffers held
        live = s["src"] >= 0
        q = torch.where(live[:, None], q, s["q"])
        sf = torch.where(_tile(live[:, None].expand(byte.shape).byte(), c["fmt"]) > 0, sf, s["sf"])
    return _as_values(_unpack(q), sf, c["fmt"])


def _as_values(values, sf, fmt):
    return dict(values=values, scales=sf.view(torch.float8_e4m3fn if fmt == "nvfp4" else torch.float8_e8m0fnu))


def _product4(s):
    c = s["case"]
    G, N, K, fmt = c["G"], c["N"], c["K"], c["fmt"]
    w = _value(s["b"], s["sfb"], N, fmt, torch.float32)
    rows = c["M"] if c["layout"] == "masked" else s["a"].shape[0]
    a = _value(s["a"], s["sfa"], rows, fmt, torch.float32).reshape(-1, K)
    live, group = s["group"] >= 0, s["group"].clamp(min=0).long()
    x = torch.zeros((G * s["cap"], K), device=DEV)
    at = group * s["cap"] + s["slot"]
    x.index_add_(0, at, torch.where(live[:, None], a, 0))
    y = torch.bmm(x.reshape(G, s["cap"], K), w.transpose(1, 2)).reshape(-1, N)[at]
    if s["alpha"] is not None:
        y = y * s["alpha"][group][:, None]
    return torch.where(live[:, None], y.to(s["d"].dtype), s["d"].reshape(-1, N)).reshape(s["d"].shape)


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if not own:
        if op == "route_grad":
            return _route_grad(s["logits"].float(), s["ids"], s["grad"], c).to(s["logits"].dtype)
        return {"norm": _norm, "norm_grad": _norm_grad, "route": _route, "quant4": _quant4, "product4": _product4}[op](s)
    from tirx_harness_b200 import grouped_gemm, moe_ops
    if op == "norm":
        r = moe_ops.rms_norm_quant(s["x"], s["weight"], residual=s["residual"], eps=1e-6, pow2=c["pow2"], mn_major=c["mn"], want_y=c["y"])
        return dict(q=r["q"], scales=r["scales"], h=r["h"] if s["residual"] is not None else None, y=r["y"], rstd=r["rstd"])
    if op == "norm_grad":
        dx, dw = moe_ops.rms_norm_backward(s["dy"], s["h"], s["weight"], s["rstd"], dh=s["dh"])
        return dict(dx=dx, dw=dw)
    if op == "route":
        ids, w = moe_ops.route(s["logits"], c["k"], score=c["score"], bias=s["bias"], n_group=c["n_group"], topk_group=c["topk_group"],
                               group_score=c["group_score"], renormalize=c["renorm"])
        return dict(ids=ids, weights=w)
    if op == "route_grad":
        return moe_ops.route_backward(s["grad"], s["logits"], s["ids"], score=c["score"], renormalize=c["renorm"])
    if op == "quant4":
        q, sf = moe_ops.quant_fp4(s["x"], fmt=c["fmt"], global_scale=s["factor"], act="silu_mul" if c["kind"] == "silu" else None,
                                  src_pair=s["src"], top_k=c["top_k"], out=(s["q"], s["sf"]))
        return _as_values(moe_ops.unpack_fp4(q), sf, c["fmt"])
    if c["layout"] == "masked":
        return grouped_gemm.bind_masked_fp4(s["a"], s["sfa"], s["b"], s["sfb"], s["d"], s["masked_m"], alpha=s["alpha"], fmt=c["fmt"])()
    return grouped_gemm.bind_contiguous_fp4(s["a"], s["sfa"], s["b"], s["sfb"], s["d"], s["group"], alpha=s["alpha"], fmt=c["fmt"])()


def work(case):
    op = case["op"]
    if op in ("norm", "norm_grad"):
        n, e = case["T"] * case["H"], SIZE[case["dtype"]]
        if op == "norm":
            return dict(bytes=n * (e * (1 + 2 * case["residual"] + case["y"]) + 1) + n // 128 * 4 + 4 * case["T"] + e * case["H"], flops=8 * n)
        return dict(bytes=n * e * (3 + case["dh"]) + 4 * case["T"] + (e + 4) * case["H"], flops=10 * n)
    if op in ("route", "route_grad"):
        n = case["T"] * case["E"] * SIZE[case["dtype"]]
        return dict(bytes=n * (1 if op == "route" else 2) + case["T"] * case["k"] * 8, flops=8 * case["T"] * case["E"])
    if op == "quant4":
        rows, K, e = case["T"] * case["top_k"], case["K"], SIZE[case["dtype"]]
        # codes, the scales, and the codes' values
        return dict(bytes=case["T"] * K * e * (2 if case["kind"] == "silu" else 1) + rows * K * 3 // 2 + rows * K // BLOCK[case["fmt"]], flops=8 * rows * K)
    G, M, N, K = (case[k] for k in ("G", "M", "N", "K"))
    rows = (G * (M + 1) // 2 if M > 1 else G) if case["layout"] == "masked" else M
    per = 0.5 + 1 / BLOCK[case["fmt"]]
    return dict(bytes=per * K * (min(G, rows) * N + rows) + rows * N * SIZE[case["out"]], flops=2 * rows * N * K)


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op, f = case["op"], torch.float64
    if op == "norm":
        x = s["x"].to(f)
        h = x if s["residual"] is None else x + s["residual"].to(f)
        used = h.to(s["x"].dtype).to(f)                    # the residual stream is kept in the inputs' type
        rstd = 1 / torch.sqrt((used * used).sum(1) / case["H"] + 1e-6)
        y = used * rstd[:, None] * s["weight"].to(f)[None]
        pad = torch.zeros((case["T"], -case["H"] % 128), dtype=f, device=DEV)
        v = torch.cat((y, pad), 1).reshape(case["T"], -1, 128)
        scale = torch.maximum(v.abs().amax(2), torch.tensor(1e-8, dtype=f, device=DEV)) / 448
        if case["pow2"]:
            scale = torch.exp2(torch.ceil(torch.log2(scale)))
        q = (v / scale[:, :, None]).flatten(1)[:, : case["H"]]
        return dict(q=q, scales=scale, h=h if s["residual"] is not None else None, y=y if case["y"] else None, rstd=rstd)
    if op == "norm_grad":
        h, dy, w, r = s["h"].to(f), s["dy"].to(f), s["weight"].to(f), s["rstd"].to(f)
        dot = (dy * w * h).sum(1)
        dx = r[:, None] * dy * w - h * (r ** 3 * dot / case["H"])[:, None]
        return dict(dx=dx if s["dh"] is None else dx + s["dh"].to(f), dw=torch.einsum("th,th,t->h", dy, h, r))
    if op == "route":
        ids = _choose(s)
        z = s["logits"].to(f)
        score = torch.sigmoid(z) if case["score"] == "sigmoid" else torch.nan_to_num(torch.softmax(z, 1))
        w = torch.gather(torch.cat((score, torch.zeros_like(score[:, :1])), 1), 1, torch.where(ids < 0, case["E"], ids).long())
        return dict(ids=None, weights=w / (w.sum(1, keepdim=True) + 1e-20) if case["renorm"] else w)
    if op == "route_grad":
        z = torch.where(s["logits"] == -math.inf, -1e4, s["logits"].to(f)).requires_grad_()
        score = torch.sigmoid(z) if case["score"] == "sigmoid" else torch.softmax(z, 1)
        on = s["ids"] >= 0
        w = score.gather(1, s["ids"].clamp(min=0).long()) * on
        if case["renorm"]:
            w = w / (w.sum(1, keepdim=True) + 1e-20)
        (w * s["grad"].to(f) * on).sum().backward()
        return torch.where(s["logits"] == -math.inf, 0, z.grad)
    if op == "quant4":
        # the codes of SiLU(gate) * up have no value of their own in 64 bits: those next to a border go by the last bit of 32
        v = _source(s, f).reshape(-1, case["K"] // BLOCK[case["fmt"]], BLOCK[case["fmt"]])
        amax = v.abs().amax(2)
        if case["fmt"] == "nvfp4":
            byte = torch.clamp(amax / (6 * s["factor"].to(f)), max=448).to(torch.float8_e4m3fn)
            unit, byte = byte.to(f) * s["factor"].to(f), byte.view(torch.uint8)
        else:
            e = torch.where(amax > 0, torch.clamp(torch.floor(torch.log2(amax)) - 2, min=-127), -127)
            unit, byte = torch.exp2(e), (e + 127).to(torch.uint8)
        t = torch.nan_to_num(v / unit[:, :, None], nan=0.0)
        # e2m1: steps of 1/2 below 2, of 1 below 4, of 2 up to 6; round() takes ties to even
        step = torch.where(t.abs() < 2, 0.5, torch.where(t.abs() < 4, 1.0, 2.0))
        val = torch.clamp(torch.round(t / step) * step, -6, 6).reshape(-1, case["K"])
        tiles = _tile(byte, case["fmt"])
        if case["kind"] == "gather":
            val[s["src"] < 0] = 0
            on = (s["src"] >= 0)[:, None].expand(byte.shape).byte()
            tiles = torch.where(_tile(on, case["fmt"]) > 0, tiles, 0)
        scales = tiles.view(torch.float8_e4m3fn).to(f) if case["fmt"] == "nvfp4" else _power(tiles).to(f)
        return dict(values=None if case["kind"] == "silu" else val, scales=scales)
    d = s["d"].to(f).reshape(-1, case["N"])
    rows = case["M"] if case["layout"] == "masked" else s["a"].shape[0]
    a = _value(s["a"], s["sfa"], rows, case["fmt"], f).reshape(-1, case["K"])
    for e in range(case["G"]):
        at = torch.nonzero(s["group"] == e).flatten()
        if len(at):
            w = _value(s["b"][e], s["sfb"][e], case["N"], case["fmt"], f)
            d[at] = a[at] @ w.T * (1.0 if s["alpha"] is None else s["alpha"][e].to(f))
    return d.reshape(s["d"].shape)
