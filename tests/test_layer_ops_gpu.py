"""Norm, routing and 4-bit operators against plain implementations in 64 bits.

Tolerances count roundings: a rounding to type t is off by at most eps(t) / 2 relative to the value (bf16 2^-8, fp16 2^-11,
fp32 2^-24, e4m3 2^-4), a sum of n terms in fp32 by n 2^-24 of the sum of their magnitudes.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0**-24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from tirx_harness_b200 import moe_ops
    return moe_ops


@pytest.fixture(scope="module")
def gg():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from tirx_harness_b200 import grouped_gemm
    return grouped_gemm


def gen(seed):
    return torch.Generator().manual_seed(seed)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def within(got, ref, allowed, what=""):
    got, ref = got.detach().cpu().double(), ref.double()
    assert got.shape == ref.shape, what
    assert torch.isfinite(got).all(), what
    over = (got - ref).abs() - allowed
    assert (over <= 0).all(), f"{what}: off by {float((got - ref).abs().max())}, {float(over.max())} more than allowed"


# ------------------------------------------------------------------ norm
NORM_CASES = [
    # T, H, dtype, weight in fp32, residual, pow2, mn_major, columns between rows beyond H
    (1, 7168, "bf16", False, True, False, False, 0),
    (3, 8, "bf16", False, False, False, False, 8),
    (5, 136, "fp16", True, True, True, True, 24),
    (37, 1000, "bf16", True, True, False, True, 0),
    (130, 2048, "fp32", True, False, True, False, 0),
    (9, 4104, "fp32", False, True, False, True, 8),
    (4, 16384, "bf16", False, True, True, False, 0),
    (2, 12296, "fp32", True, True, False, False, 0),
]


def _norm_inputs(T, H, dtype, w32, pad, seed):
    g = gen(seed)
    x = torch.zeros((T, H + pad)).normal_(generator=g)
    x[:, ::17] *= 30
    r = torch.zeros((T, H + pad)).normal_(generator=g) * 2
    w = (1 + 0.2 * torch.zeros(H).normal_(generator=g)).to(torch.float32 if w32 else DT[dtype])
    return x.to(DT[dtype])[:, :H], r.to(DT[dtype])[:, :H], w


def _cuda_strided(t):
    """A copy on the GPU with the same distance between rows."""
    base = torch.zeros((t.shape[0], t.stride(0)), dtype=t.dtype, device="cuda")
    out = base[:, : t.shape[1]]
    out.copy_(t)
    return out


@pytest.mark.parametrize("T,H,dtype,w32,residual,pow2,mn,pad", NORM_CASES)
def test_norm(ops, T, H, dtype, w32, residual, pow2, mn, pad):
    x, r, w = _norm_inputs(T, H, dtype, w32, pad, 1)
    got = ops.rms_norm_quant(_cuda_strided(x), w.cuda(), residual=_cuda_strided(r) if residual else None, eps=1e-5, pow2=pow2,
                             mn_major=mn, want_y=True)
    u = half_step(x.dtype)
    h = x.double()
    if residual:
        exact = x.double() + r.double()
        within(got["h"], exact, (u + 2 * U32) * exact.abs(), "h")
        h = got["h"].cpu().double()
    rstd = (h.square().mean(1) + 1e-5).rsqrt()
    # a thread adds up to 32 squares, then ten levels of pairs; the mean, eps and the root add four roundings
    e = 50 * U32
    within(got["rstd"], rstd, e * rstd, "rstd")
    y = h * rstd[:, None] * w.double()
    within(got["y"], y, (u + e + 2 * U32) * y.abs() + torch.finfo(x.dtype).tiny, "y")
    nb = (H + 127) // 128
    yb = torch.zeros((T, nb * 128), dtype=torch.float64)
    yb[:, :H] = y
    s = yb.reshape(T, nb, 128).abs().amax(2).clamp(min=1e-8) / 448
    sc = got["scales"].cpu().double()
    assert tuple(got["scales"].shape) == (T, nb) and (got["scales"].stride(0) == 1 or not mn or T == 1)
    if pow2:
        up = torch.exp2(torch.ceil(torch.log2(s)))
        near = (torch.log2(s) - torch.log2(s).round()).abs() < 2 * e
        assert ((sc == up) | near).all()
        m, _ = torch.frexp(sc)
        assert (m == 0.5).all()
    else:
        within(sc, s, (e + 4 * U32) * s, "scales")
    t = y / sc.repeat_interleave(128, 1)[:, :H]
    step = torch.maximum(t.abs() * 2.0**-4, torch.tensor(2.0**-10, dtype=torch.float64))       # subnormals: steps of 2^-9
    within(got["q"].float(), t, step + 2 * e * t.abs(), "q")


def test_norm_q_is_the_quantisation_of_y(ops):
    """fp32: y is not rounded, so codes and scales are those of the two-step path on it, exactly."""
    x, r, w = _norm_inputs(33, 1024, "fp32", True, 0, 2)
    got = ops.rms_norm_quant(x.cuda(), w.cuda(), residual=r.cuda(), want_y=True)
    y = got["y"].cpu().numpy().reshape(33, 8, 128)
    s = np.maximum(np.abs(y).max(2), np.float32(1e-8)) / np.float32(448)
    np.testing.assert_array_equal(got["scales"].cpu().numpy(), s)
    q = torch.from_numpy(y / s[:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn).reshape(33, 1024)
    assert torch.equal(got["q"].cpu().float(), q.float())


def test_norm_zero_rows_nan_and_infinity(ops):
    x = torch.ones((5, 256))
    x[0] = 0
    x[1, 3] = math.nan
    x[2, 200] = math.inf
    x[4] = 1e-30
    got = ops.rms_norm_quant(x.bfloat16().cuda(), torch.ones(256, device="cuda"))
    q, s = got["q"].float().cpu(), got["scales"].cpu()
    assert (q[0] == 0).all() and (s[0] == np.float32(1e-8) / np.float32(448)).all()
    assert torch.isnan(s[1]).all() and torch.isnan(q[1]).all()
    assert torch.isnan(s[2, 1]) and (q[2, :128] == 0).all()
    assert (q[3] == 448).all() and torch.isfinite(s[3]).all()
    assert torch.isfinite(s[4]).all() and torch.isfinite(q[4]).all()
    empty = ops.rms_norm_quant(torch.empty((0, 256), device="cuda"), torch.ones(256, device="cuda"), residual=torch.empty((0, 256), device="cuda"))
    assert empty["q"].shape == (0, 256) and empty["scales"].shape == (0, 2)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("H", [256, 1000, 7168, 16384])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_rows_whose_squares_pass_the_range(ops, dtype, H, residual):
    """Finite rows of any size are normalised; one with an infinity shows it in its own block and is zero elsewhere."""
    size = [1e18, 2e19, 1.0, 1e25, 5e30, 8e36, 3e38, 1e22]
    x = torch.zeros((8, H)).normal_(generator=gen(6)).clamp(-1, 1) * torch.tensor(size)[:, None]
    x[6] = 3.3e38 * torch.sign(x[6])
    x[7, H // 2] = math.inf
    x = x.to(DT[dtype])
    r = torch.zeros_like(x) if residual else None
    w = 1 + 0.2 * torch.zeros(H).normal_(generator=gen(7))
    got = ops.rms_norm_quant(x.cuda(), w.cuda(), residual=r.cuda() if residual else None, want_y=True)
    h = x.double()[:7]
    rstd = (h.square().mean(1) + 1e-6).rsqrt()
    e = 50 * U32                               # as above
    within(got["rstd"][:7], rstd, e * rstd + 2.0**-149, "rstd")
    y = h * rstd[:, None] * w.double()
    within(got["y"][:7], y, (half_step(x.dtype) + e + 2 * U32) * y.abs() + torch.finfo(x.dtype).tiny, "y")
    nb = (H + 127) // 128
    s = torch.nn.functional.pad(y, (0, nb * 128 - H)).reshape(7, nb, 128).abs().amax(2).clamp(min=1e-8) / 448
    within(got["scales"][:7], s, (e + 4 * U32) * s, "scales")
    t = y / got["scales"][:7].cpu().double().repeat_interleave(128, 1)[:, :H]
    step = torch.maximum(t.abs() * 2.0**-4, torch.tensor(2.0**-10, dtype=torch.float64))
    within(got["q"][:7].float(), t, step + 2 * e * t.abs(), "q")
    own = H // 2 // 128
    scales, codes = got["scales"][7].cpu(), got["q"][7].float().cpu()
    assert torch.isnan(scales[own]) and torch.isnan(codes[own * 128 : (own + 1) * 128]).all()
    rest = torch.arange(nb) != own
    assert (scales[rest] == np.float32(1e-8) / np.float32(448)).all() and (codes[rest.repeat_interleave(128)[:H]] == 0).all()


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("mn", [False, True])
@pytest.mark.parametrize("T,H,N", [(1, 256, 128), (300, 1024, 384)])
def test_norm_feeds_the_grouped_product(ops, gg, T, H, N, pow2, mn):
    """q and scales are the left operand of the 8-bit grouped product, in each of their layouts."""
    from tirx_harness_b200.workloads import make_operand_b
    x, r, w = _norm_inputs(T, H, "bf16", True, 0, 8)
    n = ops.rms_norm_quant(x.cuda(), w.cuda(), residual=r.cuda(), pow2=pow2, mn_major=mn, want_y=True)
    b, sb = make_operand_b(2, N, H, gen(9))
    layout = (torch.arange(T, dtype=torch.int32) * 2) // T
    d = torch.zeros((T, N), device="cuda")
    gg.bind_contiguous(n["q"], n["scales"], b.cuda(), sb.cuda(), d, layout.cuda())()
    assert gg.device_status() == 0
    a = n["q"].float().cpu().double() * n["scales"].cpu().double().repeat_interleave(128, 1)
    wide = b.float().double() * sb.double().repeat_interleave(128, 1)[:, :N].repeat_interleave(128, 2)
    ref = torch.stack([a[t] @ wide[layout[t]].T for t in range(T)])
    # that product's own tolerance: 1e-3 of the value, or of 2^-7 of the outputs' root mean square
    within(d, ref, 1e-3 * torch.maximum(ref.abs(), 2.0**-7 * ref.square().mean().sqrt()), "product")
    # and the operand stands for y: half a step of e4m3, or of its subnormals, and y's own rounding
    y = n["y"].cpu().double()
    s = n["scales"].cpu().double().repeat_interleave(128, 1)
    assert ((a - y).abs() <= torch.maximum(2.0**-4 * y.abs(), 2.0**-10 * s) * (1 + 2.0**-6) + 2.0**-8 * y.abs()).all()


@pytest.mark.parametrize("T,H,dtype,w32,dh", [(1, 7168, "bf16", False, True), (3, 8, "fp32", True, False), (517, 1000, "fp16", True, True),
                                              (700, 2048, "fp32", False, False), (300, 7168, "bf16", True, True), (5, 12296, "fp32", False, True),
                                              (6, 16384, "bf16", False, False)])
def test_norm_gradient(ops, T, H, dtype, w32, dh):
    h, dy, w = _norm_inputs(T, H, dtype, w32, 8, 3)
    past = (_norm_inputs(T, H, dtype, w32, 16, 4)[0]) if dh else None
    rstd = (h.double().square().mean(1) + 1e-6).rsqrt().float()
    dx, dw = ops.rms_norm_backward(_cuda_strided(dy), _cuda_strided(h), w.cuda(), rstd.cuda(), dh=_cuda_strided(past) if dh else None)
    n, g, r = h.double() * rstd.double()[:, None], dy.double() * w.double(), rstd.double()[:, None]
    dot, mag = (g * n).mean(1, keepdim=True), (g * n).abs().mean(1, keepdim=True)
    ref = r * (g - n * dot) + (past.double() if dh else 0)
    # each term of the mean has three roundings, its sum at most 32 in a thread and ten levels; then six more
    allowed = half_step(h.dtype) * ref.abs() + U32 * (8 * r * g.abs() + 8 * (r * n * dot).abs() + r * n.abs() * 50 * mag + 4 * ref.abs())
    within(dx, ref, allowed + torch.finfo(h.dtype).tiny, "dx")
    terms = dy.double() * n
    within(dw, terms.sum(0), (T + 50) * U32 * terms.abs().sum(0), "dw")
    again = ops.rms_norm_backward(_cuda_strided(dy), _cuda_strided(h), w.cuda(), rstd.cuda(), dh=_cuda_strided(past) if dh else None)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


def test_norm_gradient_against_differences(ops):
    T, H, eps = 4, 128, 1e-6
    h, c, w = (t.double() for t in _norm_inputs(T, H, "fp32", True, 0, 5))

    def f(h, w):
        return (c * h * (h.square().mean(1, keepdim=True) + eps).rsqrt() * w).sum()
    rstd = (h.square().mean(1) + eps).rsqrt()
    dx, dw = ops.rms_norm_backward(c.float().cuda(), h.float().cuda(), w.float().cuda(), rstd.float().cuda())
    step = 1e-5
    for i, j in ((0, 0), (1, 17), (3, 127), (2, 64)):
        d = torch.zeros_like(h)
        d[i, j] = step
        diff = (f(h + d, w) - f(h - d, w)) / (2 * step)
        # differences are off by step^2 times a third derivative of order one; fp32 sums by 100 roundings of terms of size 30
        assert abs(float(diff) - float(dx[i, j])) < 2e-4
        d = torch.zeros_like(w)
        d[j] = step
        assert abs(float((f(h, w + d) - f(h, w - d)) / (2 * step)) - float(dw[j])) < 2e-3
    dx0, dw0 = ops.rms_norm_backward(torch.empty((0, H), device="cuda"), torch.empty((0, H), device="cuda"), torch.ones(H, device="cuda"),
                                     torch.empty(0, device="cuda"))
    assert dx0.shape == (0, H) and (dw0 == 0).all()


# ------------------------------------------------------------------ routing
def _scores64(logits, score):
    z = logits.double()
    off = ~(z > -math.inf)
    z = torch.where(off, torch.full_like(z, -math.inf), z)
    if score == "sigmoid":
        p = torch.sigmoid(z)
    else:
        m = z.clamp(max=3.4028234663852886e38).amax(1, keepdim=True)
        e = torch.where(off, torch.zeros_like(z), torch.exp(z.clamp(max=3.4028234663852886e38) - torch.where(m > -math.inf, m, torch.zeros_like(m))))
        total = e.sum(1, keepdim=True)
        p = e / torch.where(total > 0, total, torch.ones_like(total))
    return p, off


def _route64(logits, k, score, bias, n_group, topk_group, group_score, renorm, scale):
    p, off = _scores64(logits, score)
    T, E = p.shape
    key = p + (bias.double() if bias is not None else 0)
    key[off] = -math.inf
    if n_group > 1:
        gs = E // n_group
        best = key.reshape(T, n_group, gs).sort(dim=2, descending=True).values
        g = best[..., 0].clone()
        if group_score == "top2" and gs > 1:
            g += torch.where(best[..., 1] > -math.inf, best[..., 1], torch.zeros_like(g))
        keep = g.sort(dim=1, descending=True, stable=True).indices[:, :topk_group]
        kept = torch.zeros((T, n_group), dtype=torch.bool).scatter_(1, keep, True).repeat_interleave(gs, 1)
        key[~kept] = -math.inf
    v, i = key.sort(dim=1, descending=True, stable=True)
    ids = torch.where(v[:, :k] > -math.inf, i[:, :k], torch.full_like(i[:, :k], -1))
    w = torch.where(ids >= 0, p.gather(1, ids.clamp(min=0)), torch.zeros((), dtype=torch.float64))
    if renorm:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return ids.int(), w * scale


ROUTE_CASES = [
    # T, E, top_k, dtype, score, bias, n_group, topk_group, group_score, renorm, scale, off
    (1, 512, 10, "bf16", "softmax", None, 1, 1, "top2", True, 1.0, 0.0),
    (65, 256, 8, "fp32", "sigmoid", "bf16", 8, 4, "top2", True, 2.5, 0.0),
    (33, 160, 6, "bf16", "softmax", None, 8, 3, "max", False, 16.0, 0.2),
    (7, 7, 7, "fp16", "softmax", None, 1, 1, "top2", False, 1.0, 0.4),
    (130, 60, 4, "fp16", "sigmoid", "fp32", 1, 1, "top2", False, 1.0, 0.3),
    (40, 1024, 32, "fp32", "softmax", "fp32", 32, 7, "top2", True, 1.0, 0.0),
    (300, 33, 5, "fp32", "softmax", "bf16", 3, 2, "max", True, 1.0, 0.5),
    (64, 1, 1, "fp32", "sigmoid", None, 1, 1, "max", True, 1.0, 0.0),
    (50, 96, 8, "bf16", "sigmoid", None, 12, 5, "top2", True, 1.0, 0.7),
    (20, 32, 2, "fp32", "softmax", "fp32", 32, 4, "top2", True, 1.0, 0.0),
]


def _route_inputs(T, E, dtype, off, seed, pad=0):
    g = gen(seed)
    logits = torch.zeros((T, E + pad)).normal_(generator=g) * 2
    logits[torch.rand((T, E + pad), generator=g) < off] = -math.inf
    if off:
        logits[T // 2] = -math.inf
        logits[0, 0] = math.nan
    return logits.to(DT[dtype])[:, :E]


@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("T,E,k,dtype,score,bias,n_group,topk_group,group_score,renorm,scale,off", ROUTE_CASES)
def test_route(ops, T, E, k, dtype, score, bias, n_group, topk_group, group_score, renorm, scale, off, pad):
    logits = _route_inputs(T, E, dtype, off, 7, pad)
    b = None if bias is None else (0.1 * torch.zeros(E).normal_(generator=gen(8))).to(DT[bias])
    ids, w = ops.route(_cuda_strided(logits), k, score=score, bias=b.cuda() if b is not None else None, n_group=n_group, topk_group=topk_group,
                       group_score=group_score, renormalize=renorm, scale=scale)
    rid, rw = _route64(logits, k, score, b, n_group, topk_group, group_score, renorm, scale)
    assert torch.equal(ids.cpu(), rid)
    # exp is off by 2 steps and the rounding of its argument (at most 32 here); the sums by their 40 roundings
    within(w, rw, (2 * 32 + 2 * 4 + 2 * 40) * U32 * rw.abs() + 1e-37, "weights")


def test_route_equal_logits_go_to_the_lowest_index(ops):
    logits = torch.zeros((2, 100))
    logits[1, 50:] = 1
    ids, w = ops.route(logits.cuda(), 4)
    assert ids.cpu().tolist() == [[0, 1, 2, 3], [50, 51, 52, 53]] and (w == 0.25).all()
    ids, _ = ops.route(logits.cuda(), 4, score="sigmoid", bias=torch.zeros(100, device="cuda"), n_group=10, topk_group=2)
    assert ids.cpu().tolist() == [[0, 1, 2, 3], [50, 51, 52, 53]]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("E,n_group,topk_group", [(2, 1, 1), (8, 4, 2), (96, 1, 1), (96, 8, 3), (96, 3, 2)])
def test_route_zeros_of_either_sign_are_equal(ops, dtype, E, n_group, topk_group):
    """-0 and +0 have the same score: the lowest index comes first, among few keys and among more than a warp holds."""
    logits = torch.full((4, E), -1.0)
    logits[0, 0::2], logits[0, 1::2] = -0.0, 0.0
    logits[1, : E // 2], logits[1, E // 2:] = -0.0, 0.0
    logits[2, 1::4], logits[2, 3::4] = -0.0, 0.0
    logits[3] = -0.0
    logits = logits.to(DT[dtype])
    k = 1 if E == 2 else 4
    for score in ("sigmoid", "softmax"):
        for bias in (None, torch.zeros(E), torch.full((E,), -0.0)):
            ids, _ = ops.route(logits.cuda(), k, score=score, bias=None if bias is None else bias.cuda(), n_group=n_group, topk_group=topk_group)
            rid, _ = _route64(logits, k, score, bias, n_group, topk_group, "top2", True, 1.0)
            assert torch.equal(ids.cpu(), rid)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_route_keys_closer_than_fp32(ops, score):
    """Keys that all lie within an fp32 step of one another keep the order that 64 bits give them."""
    T, E = 16, 256
    logits = torch.zeros((1, E)).normal_(generator=gen(9)).repeat(T, 1)
    p, _ = _scores64(logits, score)
    bias = (0.5 - p[0]).float()
    for n_group, topk_group in ((1, 1), (8, 3)):
        ids, _ = ops.route(logits.cuda(), 8, score=score, bias=bias.cuda(), n_group=n_group, topk_group=topk_group)
        rid, _ = _route64(logits, 8, score, bias, n_group, topk_group, "top2", True, 1.0)
        assert torch.equal(ids.cpu(), rid)


@pytest.mark.parametrize("E", [128, 256, 512, 1024])
def test_route_one_dominating_expert(ops, E):
    """Scores whose fp32 sum is off by a rounding per term: a bias puts another expert's key next to the dominating one's."""
    for other in (math.log(0.51 * 2.0**-23), math.log(0.97 * 2.0**-24), -16.7, -15.544, -7.0):
        logits = torch.full((1, E), other)
        logits[0, 0] = 0
        p, _ = _scores64(logits, "softmax")
        for second in (1, E // 4, E - 1):
            for apart in (-3e-6, -1.6e-6, -9e-7, -3e-7, 9e-8, 3e-7, 6e-7, 1.2e-6, 1.6e-6, 3e-6):
                bias = torch.full((E,), -10.0)
                bias[0] = 0
                bias[second] = float(p[0, 0] - p[0, second]) - apart
                for n_group in (1, 4):
                    ids, _ = ops.route(logits.cuda(), 2, bias=bias.cuda(), n_group=n_group, topk_group=1, group_score="max")
                    rid, _ = _route64(logits, 2, "softmax", bias, n_group, 1, "max", True, 1.0)
                    assert torch.equal(ids.cpu(), rid), (other, second, apart, n_group)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,n_group", [(64, 32), (96, 8), (1024, 32)])
def test_route_groups_whose_two_best_cancel(ops, score, E, n_group):
    """The sum of a large and a largely negative key has their rounding errors, not those of its own size."""
    logits = _route_inputs(32, E, "fp32", 0.0, 14)
    bias = torch.full((E,), -5000.0)
    gs = E // n_group
    bias[0::gs], bias[1::gs] = 1000.0, -1000.0
    bias[: 4 * gs : gs], bias[1 : 4 * gs : gs] = 0.0, 0.0
    ids, _ = ops.route(logits.cuda(), 4, score=score, bias=bias.cuda(), n_group=n_group, topk_group=n_group // 4)
    rid, _ = _route64(logits, 4, score, bias, n_group, n_group // 4, "top2", True, 1.0)
    assert torch.equal(ids.cpu(), rid)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_route_extreme_biases(ops, score):
    """+infinity counts as the largest number; sums of two biases may pass the range of fp32; -infinity and NaN switch off."""
    big, inf, off = torch.finfo(torch.float32).max, math.inf, -math.inf
    for bias, n_group, topk_group, k in [
            ([big, inf, 0, 0], 1, 1, 2), ([inf, big, inf, 0], 1, 1, 3), ([-big, -big, -inf, math.nan], 1, 1, 4),
            ([inf, 1.7e38, inf, inf], 2, 1, 1), ([1.8e38, 1.7e38, 1.9e38, 1.7e38, 0, 0], 3, 1, 2), ([off, off, -big, -big], 2, 1, 2),
            ([off, math.nan, -3e38, -2e38, -2e38, -2e38], 3, 1, 2), ([off, off, -big, off, -big, -big], 3, 2, 2), ([inf] * 96, 8, 2, 4)]:
        b = torch.tensor(bias)
        logits = torch.zeros((3, len(bias))).normal_(generator=gen(15))
        logits[1] = 0
        logits[2, :2] = off
        ids, w = ops.route(logits.cuda(), k, score=score, bias=b.cuda(), n_group=n_group, topk_group=topk_group)
        held = b.double().clamp(max=big)
        gone = ~(logits > off)
        z = torch.where(gone | ~(held > off), torch.tensor(off, dtype=torch.float64), logits.double())       # not chosen, but part of the softmax
        rid, _ = _route64(z, k, score, torch.where(held > off, held, torch.zeros_like(held)), n_group, topk_group, "top2", True, 1.0)
        assert torch.equal(ids.cpu(), rid), (bias, n_group)
        assert torch.isfinite(w).all()


def test_route_extreme_logits(ops):
    big = torch.finfo(torch.float32).max
    rows = torch.tensor([[-big, -big, -big, -big], [big, 0, -big, big], [math.inf, 0, 1, 2], [-math.inf, math.nan, 5, -math.inf],
                         [-math.inf, -math.inf, math.nan, math.nan], [-200, -300, -250, -400]])
    ids, w = ops.route(rows.cuda(), 2)
    assert ids.cpu().tolist() == [[0, 1], [0, 3], [0, 3], [2, -1], [-1, -1], [0, 2]]
    torch.testing.assert_close(w.cpu(), torch.tensor([[.5, .5], [.5, .5], [1., 0.], [1., 0.], [0., 0.], [1., math.exp(-50)]]), rtol=1e-4, atol=1e-30)
    ids, w = ops.route(rows.cuda(), 2, score="sigmoid", renormalize=False)
    assert ids.cpu().tolist() == [[0, 1], [0, 3], [0, 3], [2, -1], [-1, -1], [0, 2]]
    assert torch.isfinite(w).all()
    ids, w = ops.route(torch.empty((0, 16), device="cuda"), 2)
    assert ids.shape == (0, 2) and w.shape == (0, 2)


def _route_grad64(grad, logits, ids, score, renorm, scale):
    z = logits.double()
    off = ~(z > -math.inf)
    z = torch.where(off, torch.full_like(z, -1e30), z).requires_grad_()
    p = torch.sigmoid(z) if score == "sigmoid" else torch.softmax(z, 1)
    on = (ids >= 0) & ~off.gather(1, ids.clamp(min=0).long())
    w = torch.where(on, p.gather(1, ids.clamp(min=0).long()), torch.zeros((), dtype=torch.float64))
    total = w.sum(1, keepdim=True) + 1e-20
    if renorm:
        w = w / total
    (w * scale * torch.where(on, grad.double(), torch.zeros((), dtype=torch.float64))).sum().backward()
    return torch.where(off, torch.zeros_like(z), z.grad)


@pytest.mark.parametrize("T,E,k,dtype,score,renorm,off,pad", [
    (1, 256, 8, "fp32", "softmax", True, 0.0, 0), (65, 160, 6, "bf16", "sigmoid", True, 0.3, 0), (33, 7, 3, "fp16", "softmax", False, 0.4, 3),
    (130, 512, 10, "fp32", "sigmoid", False, 0.0, 4), (20, 1000, 32, "bf16", "softmax", True, 0.1, 8), (9, 33, 2, "fp32", "softmax", True, 0.0, 0)])
def test_route_gradient(ops, T, E, k, dtype, score, renorm, off, pad):
    logits = _route_inputs(T, E, dtype, off, 10, pad)
    ids, _ = _route64(logits, k, score, None, 1, 1, "max", renorm, 1.0)
    if k > 2:
        ids[0, 1] = ids[0, 0]                    # the same index twice, and one that is out of range
        ids[T - 1, 2] = -5
    grad = torch.zeros((T, k)).normal_(generator=gen(11))
    got = ops.route_backward(grad.cuda(), _cuda_strided(logits), ids.cuda(), score=score, renormalize=renorm, scale=1.5)
    ref = _route_grad64(grad, logits, ids, score, renorm, 1.5)
    # shares of the gradient before they cancel: |G| and the sum of |G p|, over the chosen scores' sum where that is divided by
    p, _ = _scores64(logits, score)
    on = ids >= 0
    sel = torch.where(on, p.gather(1, ids.clamp(min=0).long()), torch.zeros((), dtype=torch.float64))
    G = 1.5 * grad.double().abs().amax(1, keepdim=True)
    if renorm:
        G = 2 * G / (sel.sum(1, keepdim=True) + 1e-20).clamp(min=1e-18)
    allowed = half_step(logits.dtype) * ref.abs() + 256 * U32 * p * k * G + torch.finfo(logits.dtype).tiny
    within(got, ref, allowed, "dlogits")


def _route_grad64_of_differences(grad, logits, ids, score, renorm):
    """The same without differences of nearly equal scores, and the sum of the magnitudes of its terms."""
    p, _ = _scores64(logits, score)
    T, E = p.shape
    out, mag = torch.zeros_like(p), torch.zeros_like(p)
    for t in range(T):
        at = [int(i) for i in ids[t] if i >= 0]
        G = torch.tensor([float(grad[t, j]) for j in range(ids.shape[1]) if ids[t, j] >= 0], dtype=torch.float64)
        s = p[t, at]
        rest = 1.0 if score == "sigmoid" else float(p[t, [e for e in range(E) if e not in at]].sum())
        total = float(s.sum()) + 1e-20
        d = (G[:, None] - G[None]) * s[None]
        if renorm:
            h, hm = (d.sum(1) + 1e-20 * G) / total**2, (d.abs().sum(1) + 1e-20 * G.abs()) / total**2
            others = float((G * s).sum()) * 1e-20 / total**2
        elif score == "softmax":
            h, hm, others = d.sum(1) + G * rest, d.abs().sum(1) + G.abs() * rest, float((G * s).sum())
        else:
            h, hm = G, G.abs()
        if score == "sigmoid":
            f = torch.sigmoid(-logits[t, at].double())
            once, oncem = s * f * h, s * f * hm
        else:
            once = s * (h - (others if renorm else 0))
            oncem = s * (hm + (abs(others) if renorm else 0))
            out[t], mag[t] = -p[t] * others, p[t] * float((G * s).abs().sum()) * (1e-20 / total**2 if renorm else 1)
            out[t, at], mag[t, at] = 0, 0
        for j, e in enumerate(at):
            out[t, e] += once[j]
            mag[t, e] += oncem[j]
    return out, mag


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dtype,E,k", [("fp32", 64, 8), ("bf16", 256, 3), ("fp32", 1000, 32), ("fp32", 6, 1)])
def test_route_gradient_where_one_score_dominates(ops, score, renorm, dtype, E, k):
    """Relative to the terms that are left once p next to 1 is not subtracted from 1."""
    logits = _route_inputs(12, E, "fp32", 0.0, 17) * 0.5
    for t in range(12):
        logits[t, (5 * t) % E] = 2.5 * t
    logits = logits.to(DT[dtype])
    grad = torch.zeros((12, k)).normal_(generator=gen(18))
    grad[1] = 0.75                                     # equal gradients: nothing left where they are renormalised
    ids, _ = _route64(logits, k, score, None, 1, 1, "max", renorm, 1.0)
    if k > 2:
        ids[2, 1], ids[3, 0] = -1, ids[3, 2]           # the same index twice counts twice
        twice = ids[3].clone()
    got = ops.route_backward(grad.cuda(), logits.cuda(), ids.cuda(), score=score, renormalize=renorm)
    rows = [t for t in range(12) if t != 3]            # a row with an index twice: against the plain form below
    ref, mag = _route_grad64_of_differences(grad[rows], logits[rows], ids[rows], score, renorm)
    plain = _route_grad64(grad[rows], logits[rows], ids[rows], score, renorm, 1.0)
    assert ((ref - plain).abs() <= 1e-12 * (1 + plain.abs())).all()
    # a score: 4 roundings of its exponential and as many as its argument's size (at most 30, from three roundings each), the sum
    # of up to 32 in a lane and five levels, and a division; four scores, k products and a few more steps
    allowed = 4 * (4 + 3 * 30 + 40) + k + 10
    within(got[rows], ref, half_step(logits.dtype) * ref.abs() + allowed * U32 * mag + torch.finfo(logits.dtype).tiny, "dlogits")
    if k > 2:
        plain = _route_grad64(grad[3:4], logits[3:4], twice[None], score, renorm, 1.0)
        p, _ = _scores64(logits[3:4], score)
        total = p.gather(1, twice[None].long()).sum() if renorm else 1
        within(got[3:4], plain, half_step(logits.dtype) * plain.abs() + 256 * U32 * p * k * grad[3].abs().max() * (2 / total if renorm else 1), "twice")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_route_gradient_of_confident_sigmoids(ops, dtype):
    """p (1 - p) keeps its relative precision where p is next to 1, and next to 0."""
    logits = torch.cat((torch.linspace(-80, 80, 97), torch.linspace(8, 30, 63)))[None].to(DT[dtype]).repeat(5, 1)
    ids = torch.arange(160, dtype=torch.int32).reshape(5, 32)
    grad = torch.zeros((5, 32)).normal_(generator=gen(16))
    got = ops.route_backward(grad.cuda(), logits.cuda(), ids.cuda(), score="sigmoid", renormalize=False)
    z = logits.double()
    ref = torch.zeros_like(z).scatter(1, ids.long(), grad.double() * (torch.sigmoid(z) * torch.sigmoid(-z)).gather(1, ids.long()))
    # p and 1 - p: an exponential of 2 steps (4 roundings), a sum and a division each; then three products
    within(got, ref, (half_step(DT[dtype]) + 16 * U32) * ref.abs() + torch.finfo(DT[dtype]).tiny, "dlogits")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_gradient_against_differences(ops, score, renorm):
    logits = _route_inputs(3, 24, "fp32", 0.0, 12)
    ids, w = ops.route(logits.cuda(), 4, score=score, renormalize=renorm)
    grad = torch.zeros((3, 4)).normal_(generator=gen(13))
    got = ops.route_backward(grad.cuda(), logits.cuda(), ids, score=score, renormalize=renorm).cpu()
    at = ids.cpu().long()

    def f(z):
        p, _ = _scores64(z, score)
        s = p.gather(1, at)
        return (grad.double() * (s / (s.sum(1, keepdim=True) + 1e-20) if renorm else s)).sum()
    z = logits.double()
    for i, e in ((0, int(at[0, 0])), (1, int(at[1, 3])), (2, 5), (2, int(at[2, 1]))):
        d = torch.zeros_like(z)
        d[i, e] = 1e-5
        assert abs(float((f(z + d) - f(z - d)) / 2e-5) - float(got[i, e])) < 1e-5


# ------------------------------------------------------------------ 4-bit blocks
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=np.float64)
BLOCK = {"nvfp4": 16, "mxfp4": 32}


def codes_of(q):
    """uint8 [.., K/2] -> codes [.., K]"""
    q = q.cpu().numpy()
    return np.stack((q & 15, q >> 4), -1).reshape(*q.shape[:-1], -1)


def scale_bytes(tiles, rows, K, fmt):
    """One group's scale tiles -> bytes [rows, K / block], entry by entry."""
    t = tiles.cpu().numpy()
    r = np.arange(rows)[:, None]
    b = np.arange(K // BLOCK[fmt])[None]
    return t[r // 128, b // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4]


def scale_values(byte, fmt):
    if fmt == "nvfp4":
        return torch.from_numpy(byte.copy()).view(torch.float8_e4m3fn).double().numpy()
    return np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))


def quant32(x, fmt, g):
    """The definition in single roundings: x float32 [rows, K] -> (codes, scale bytes)."""
    v = x.reshape(x.shape[0], -1, BLOCK[fmt])
    amax = np.abs(v).max(2)
    with np.errstate(all="ignore"):
        if fmt == "nvfp4":
            t = np.minimum(amax / (np.float32(6) * np.float32(g)), np.float32(448))
            sf = torch.from_numpy(t).to(torch.float8_e4m3fn)
            byte, unit = sf.view(torch.uint8).numpy(), sf.float().numpy() * np.float32(g)
        else:
            e = np.where(amax > 0, np.frexp(amax)[1] - 1 - 2 + 127, 0).clip(0, 254)
            byte, unit = e.astype(np.uint8), np.exp2(e - 127.0).astype(np.float32)
        a = np.abs(v) / np.where(unit > 0, unit, np.float32(np.inf))[..., None]
    mid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=np.float32)
    code = np.zeros(a.shape, dtype=np.uint8)
    for i, m in enumerate(mid):
        code += (a > m) if i % 2 == 0 else (a >= m)           # ties to the even code
    return (code + 8 * np.signbit(v)).reshape(x.shape).astype(np.uint8), byte


def same_codes(got, ref):
    return np.array_equal(E2M1[got], E2M1[ref])


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("rows,K,dtype,pad", [(1, 128, "bf16", 0), (37, 384, "fp16", 8), (128, 256, "fp32", 0), (333, 1152, "bf16", 40), (300, 640, "fp32", 16)])
def test_quant_fp4(ops, fmt, rows, K, dtype, pad):
    g = gen(20)
    x = (torch.zeros((rows, K + pad)).normal_(generator=g) * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g).float())).to(DT[dtype])[:, :K]
    x[0, :64] = 0
    x[rows // 2, 32:64] = 1e-7 if dtype != "fp16" else 6e-8
    x[rows - 1, :8] = torch.tensor([6, 5, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25])          # exact ties under a scale of 1
    x[rows - 1, 8:32] = 0
    for factor in ((None, 0.25, 1.7e-3) if fmt == "nvfp4" else (None,)):
        f = None if factor is None else torch.tensor([factor], device="cuda")
        q, sf = ops.quant_fp4(_cuda_strided(x), fmt=fmt, global_scale=f)
        rc, rb = quant32(x.float().numpy(), fmt, 1.0 if factor is None else np.float32(factor))
        np.testing.assert_array_equal(scale_bytes(sf, rows, K, fmt), rb)
        assert same_codes(codes_of(q), rc)
        # nothing but zero behind the last row and block
        full = scale_bytes(sf, (rows + 127) // 128 * 128, (K + 255) // 256 * 256, fmt)
        assert not full[rows:].any() and not full[:, K // BLOCK[fmt]:].any()
        assert torch.equal(ops.unpack_fp4(q).double().cpu(), torch.from_numpy(E2M1[codes_of(q)]))


def test_quant_fp4_not_finite_and_extreme(ops):
    x = torch.ones((4, 128))
    x[0, 5] = math.nan
    x[1, 40] = -math.inf
    x[2] = torch.finfo(torch.float32).max
    x[3] = 1e-42
    for fmt, nan in (("nvfp4", 0x7F), ("mxfp4", 0xFF)):
        q, sf = ops.quant_fp4(x.cuda(), fmt=fmt)
        b, c = scale_bytes(sf, 4, 128, fmt), codes_of(q)
        blk = BLOCK[fmt]
        bad = np.zeros((4, 128 // blk), dtype=bool)
        bad[0, 5 // blk] = bad[1, 40 // blk] = True
        np.testing.assert_array_equal(b == nan, bad)
        assert not c[0, : blk].any() and (c[0, blk:] > 0).all()
        ref, rb = quant32(x.numpy()[2:], fmt, 1.0)
        np.testing.assert_array_equal(b[2:], rb)
        assert same_codes(c[2:], ref)


@pytest.mark.parametrize("factor", [1e-10, 1e-36, 1e36, 2.0**-126, 1.5])
def test_quant_fp4_far_away_factors(ops, factor):
    """Values that overflow against the largest scale keep their sign and become 6; scales that come out as zero leave zeros;
    factors at the ends of the range are divided by like any other."""
    g = gen(27)
    x = torch.zeros((8, 256)).normal_(generator=g) * 10.0 ** torch.arange(-32, 48, 10).float().clamp(max=37)[:, None]
    q, sf = ops.quant_fp4(x.cuda(), global_scale=torch.tensor([factor], device="cuda"))
    rc, rb = quant32(x.numpy(), "nvfp4", np.float32(factor))
    np.testing.assert_array_equal(scale_bytes(sf, 8, 256, "nvfp4"), rb)
    live = np.repeat(rb, 16, 1) != 0
    assert same_codes(codes_of(q)[live], rc[live])
    assert not E2M1[codes_of(q)][~live].any()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_quant_fp4_gather_leaves_padding_alone(ops, fmt):
    T, K, top_k = 50, 256, 3
    x = torch.zeros((T, K)).normal_(generator=gen(21)).bfloat16()
    src = torch.full((256,), -1, dtype=torch.int32)
    src[:150] = torch.randperm(150, generator=gen(22)).int()
    src[200:210] = 7
    q = torch.full((256, K // 2), 0xA5, dtype=torch.uint8, device="cuda")
    sf = torch.full(ops.fp4_scale_shape(256, K, fmt), 0x5A, dtype=torch.uint8, device="cuda")
    r = ops.quant_fp4(x.cuda(), fmt=fmt, src_pair=src.cuda(), top_k=top_k, out=(q, sf))
    assert r[0] is q and r[1] is sf
    live = (src >= 0).numpy()
    rc, rb = quant32(x[(src // top_k).clamp(min=0).long()].float().numpy(), fmt, 1.0)
    b = scale_bytes(sf, 256, K, fmt)
    np.testing.assert_array_equal(b[live], rb[live])
    assert same_codes(codes_of(q)[live], rc[live])
    assert (b[~live] == 0x5A).all() and (q.cpu().numpy()[~live] == 0xA5).all()


@pytest.mark.parametrize("fmt,dtype", [("nvfp4", "bf16"), ("mxfp4", "fp32"), ("nvfp4", "fp16")])
def test_quant_fp4_gather_many_rows_of_each(ops, fmt, dtype):
    """So many rows that x is quantised once and its rows are copied: ragged lengths, pairs that two rows have, skipped rows,
    a stream of its own and a replayed graph that gets other pairs."""
    from tirx_harness_b200 import _lib
    T, K, top_k, rows = 900, 1152, 9, 7300
    need = _lib.lib().moe_quant_fp4_workspace_bytes(rows, T, K, 0 if fmt == "nvfp4" else 1)
    assert need > 0
    x = torch.zeros((T, K + 16)).normal_(generator=gen(25)).to(DT[dtype])[:, :K]
    x[3, 40] = math.nan
    src = torch.randperm(T * top_k, generator=gen(26))[:rows].int()
    src[100:140], src[200], src[rows - 1], src[300:500] = -1, 27, 27, 5
    f = torch.tensor([7e-4], device="cuda") if fmt == "nvfp4" else None
    xd, srcd = _cuda_strided(x), src.cuda()
    shape = ops.fp4_scale_shape(rows, K, fmt)
    q, sf = torch.full((rows, K // 2), 0xA5, dtype=torch.uint8, device="cuda"), torch.full(shape, 0x5A, dtype=torch.uint8, device="cuda")
    rc, rb = quant32(x.float().numpy(), fmt, np.float32(7e-4) if fmt == "nvfp4" else 1.0)
    block = 40 // BLOCK[fmt]                                       # the NaN's, which quant32 does not know
    rb[3, block] = 0x7F if fmt == "nvfp4" else 0xFF
    rc[3, block * BLOCK[fmt]:(block + 1) * BLOCK[fmt]] = 0

    def check(src):
        live, t = (src >= 0).numpy(), (src // top_k).clamp(min=0).long().numpy()
        b = scale_bytes(sf, rows, K, fmt)
        np.testing.assert_array_equal(b[live], rb[t][live])
        assert same_codes(codes_of(q)[live], rc[t][live])
        assert (b[~live] == 0x5A).all() and (q.cpu().numpy()[~live] == 0xA5).all()
        full = scale_bytes(sf, shape[0] * 128, (K + 255) // 256 * 256, fmt)
        assert not full[rows:].any() and not full[:rows][live][:, K // BLOCK[fmt]:].any()

    def call():
        ops.quant_fp4(xd, fmt=fmt, global_scale=f, src_pair=srcd, top_k=top_k, out=(q, sf))

    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    check(src)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call()
    other = src.clone()
    other[src >= 0] = other[src >= 0].flip(0)
    srcd.copy_(other)
    graph.replay()
    check(other)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("gate_first", [True, False])
def test_quant_fp4_silu_mul(ops, fmt, gate_first):
    rows, K = 45, 384
    x = (torch.zeros((rows, 2 * K)).normal_(generator=gen(23)) * 3).bfloat16()
    f = torch.tensor([3e-3], device="cuda") if fmt == "nvfp4" else None
    q, sf = ops.quant_fp4(x.cuda(), fmt=fmt, global_scale=f, act="silu_mul", gate_first=gate_first)
    a, b = x[:, :K].double(), x[:, K:].double()
    gate, up = (a, b) if gate_first else (b, a)
    v = (gate * torch.sigmoid(gate) * up).numpy().reshape(rows, -1, BLOCK[fmt])
    s = scale_values(scale_bytes(sf, rows, K, fmt), fmt)
    amax = np.abs(v).max(2)
    # SiLU in fp32 is off by a few roundings: exp2's argument (at most 20 here), exp2, the sum, the quotient, the product
    tol = (20 + 8) * U32
    if fmt == "nvfp4":
        t = np.minimum(amax / (6 * float(np.float32(3e-3))), 448)
        assert (np.abs(s - t) <= np.maximum(t * 2.0**-4, 2.0**-10) * (1 + 1e-5)).all()
        unit = s * float(np.float32(3e-3))
    else:
        up2 = np.exp2(np.floor(np.log2(amax * (1 + tol))) - 2)
        down2 = np.exp2(np.floor(np.log2(amax * (1 - tol))) - 2)
        assert ((s == up2) | (s == down2)).all()
        unit = s
    t = np.minimum(np.abs(v) / unit[..., None], 6)
    c = np.abs(E2M1[codes_of(q)]).reshape(v.shape)
    half = np.where(t < 2, 0.25, np.where(t < 4, 0.5, 1.0))        # half a step of e2m1
    assert (np.abs(c - t) <= half + 8 * tol).all()
    signs = E2M1[codes_of(q)].reshape(v.shape) * v
    assert (signs >= 0).all()


def test_quant_fp4_groups(ops):
    """Three dimensions: every group has scale tiles and a factor of its own."""
    w = torch.zeros((3, 200, 256)).normal_(generator=gen(24)).bfloat16()
    f = torch.tensor([1e-3, 2e-3, 0.5])
    q, sf = ops.quant_fp4(w.cuda(), global_scale=f.cuda())
    assert q.shape == (3, 200, 128) and sf.shape == (3, 2, 4, 512)
    for g in range(3):
        rc, rb = quant32(w[g].float().numpy(), "nvfp4", f[g].numpy())
        np.testing.assert_array_equal(scale_bytes(sf[g], 200, 256, "nvfp4"), rb)
        assert same_codes(codes_of(q[g]), rc)


# ------------------------------------------------------------------ 4-bit product
def make_operand(lead, rows, K, fmt, seed):
    """Random codes and scales -> (codes, tiles, values in float64 on the CPU)."""
    rng = np.random.default_rng(seed)
    n = int(np.prod(lead, dtype=np.int64)) if lead else 1
    q = rng.integers(0, 256, size=(n, rows, K // 2), dtype=np.uint8)
    nb = K // BLOCK[fmt]
    byte = rng.integers(0x20, 0x50, size=(n, rows, nb), dtype=np.uint8) if fmt == "nvfp4" else rng.integers(120, 131, size=(n, rows, nb), dtype=np.uint8)
    kt = (K + 255) // 256 * (64 // BLOCK[fmt])
    tiles = rng.integers(0, 0x70, size=(n, (rows + 127) // 128, kt, 512), dtype=np.uint8)       # finite everywhere
    r, b = np.arange(rows)[:, None], np.arange(nb)[None]
    for g in range(n):
        tiles[g][r // 128, b // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4] = byte[g]
    val = E2M1[np.stack((q & 15, q >> 4), -1).reshape(n, rows, K)] * np.repeat(scale_values(byte, fmt), BLOCK[fmt], -1)
    shape = (*lead, rows) if lead else (rows,)
    return (torch.from_numpy(q).reshape(*shape, K // 2).cuda(), torch.from_numpy(tiles).reshape(*lead, *tiles.shape[1:]).cuda(),
            torch.from_numpy(val).reshape(*shape, K))


def check_product(d, before, a, b, group, alpha, dtype):
    """d [rows, N] against the 64-bit product of each row with its group's b; rows without a group as they were."""
    d, group = d.cpu(), group.cpu()
    assert torch.equal(d[group < 0], before.cpu()[group < 0])
    for g in range(b.shape[0]):
        at = torch.nonzero(group == g).flatten()
        if not len(at):
            continue
        al = 1.0 if alpha is None else float(alpha.reshape(-1)[min(g, alpha.numel() - 1)])
        ref, mag = a[at] @ b[g].T * al, a[at].abs() @ b[g].abs().T * abs(al)
        # exact products, K of them added up in fp32; the factor and the output's rounding
        u = half_step(dtype) if dtype != torch.float32 else U32
        within(d[at], ref, u * ref.abs() + (a.shape[1] + 2) * U32 * mag, f"group {g}")


CONTIGUOUS = [
    # rows per group, rows of padding after each, N, K, fmt, dtype
    ((1,), (0,), 8, 128, "nvfp4", "fp32"),
    ((5, 0, 3), (0, 0, 0), 72, 384, "mxfp4", "bf16"),
    ((100, 1, 28, 127), (28, 0, 100, 1), 200, 640, "nvfp4", "bf16"),
    ((200, 70), (56, 58), 512, 256, "mxfp4", "fp32"),
    ((300, 0, 260, 40), (84, 0, 124, 88), 456, 1152, "nvfp4", "fp32"),
    ((17, 19, 23, 29, 31), (0, 0, 0, 0, 5), 264, 2048, "mxfp4", "bf16"),
    ((1, 1, 1, 1, 1, 1, 1, 1), (0,) * 8, 640, 1024, "nvfp4", "bf16"),
    # at most 32 and 128 rows: several tiles per block, blocks that share K, K shorter than the blocks that share it
    ((3, 4) * 4, (0,) * 8, 2560, 512, "mxfp4", "fp32"),
    ((40, 30, 0, 50), (2, 0, 0, 6), 4096, 768, "nvfp4", "bf16"),
    ((33,), (0,), 1024, 256, "mxfp4", "fp32"),
    ((20, 2), (0, 0), 1032, 1280, "nvfp4", "fp32"),
]


def _contiguous(rows, pads, N, K, fmt, seed=30):
    layout = torch.cat([torch.cat((torch.full((r,), g), torch.full((p,), -1))) for g, (r, p) in enumerate(zip(rows, pads))]).int()
    a, sfa, av = make_operand((), len(layout), K, fmt, seed)
    b, sfb, bv = make_operand((len(rows),), N, K, fmt, seed + 1)
    return layout, (a, sfa, av), (b, sfb, bv)


@pytest.mark.parametrize("rows,pads,N,K,fmt,dtype", CONTIGUOUS)
def test_product_contiguous(gg, rows, pads, N, K, fmt, dtype):
    layout, (a, sfa, av), (b, sfb, bv) = _contiguous(rows, pads, N, K, fmt)
    base = torch.full((len(layout), N + 24), 7.0, dtype=DT[dtype], device="cuda")
    d = base[:, :N]
    before = d.clone()
    alpha = torch.rand(len(rows), generator=gen(31)) + 0.5
    out = gg.bind_contiguous_fp4(a, sfa, b, sfb, d, layout.cuda(), alpha=alpha.cuda(), fmt=fmt)()
    assert out is d and gg.device_status() == 0
    check_product(d, before, av, bv, layout, alpha, DT[dtype])
    assert (base[:, N:] == 7).all()
    # one factor for all groups; only the leading rows
    used = torch.tensor([max(1, len(layout) // 2)], dtype=torch.int32, device="cuda")
    d2 = torch.full((len(layout), N), 3.0, dtype=DT[dtype], device="cuda")
    gg.bind_contiguous_fp4(a, sfa, b, sfb, d2, layout.cuda(), alpha=alpha[:1].cuda(), fmt=fmt, rows_used=used)()
    half = layout.clone()
    half[int(used):] = -1
    check_product(d2, torch.full_like(d2, 3.0), av, bv, half, alpha[:1], DT[dtype])


@pytest.mark.parametrize("M,G,low", [(300, 3, -1), (1500, 150, 0), (90, 5, -1), (700, 4, -300)])
def test_product_rows_in_any_order(gg, M, G, low):
    """Several groups in every block of rows, in no order; 1500 rows of 150 groups are more than the list of blocks holds."""
    layout = torch.randint(low, G, (M,), generator=gen(32)).int()
    layout[M // 3] = G + 5                                # no such group: a padding row
    a, sfa, av = make_operand((), M, 256, "nvfp4", 33)
    b, sfb, bv = make_operand((G,), 136, 256, "nvfp4", 34)
    d = torch.zeros((M, 136), dtype=torch.bfloat16, device="cuda")
    gg.bind_contiguous_fp4(a, sfa, b, sfb, d, layout.cuda())()
    assert gg.device_status() == 0
    layout[M // 3] = -1
    check_product(d, torch.zeros_like(d), av, bv, layout, None, torch.bfloat16)


def test_product_more_row_blocks_than_the_list_holds(gg):
    """131073 rows and more: 1025 blocks of 128."""
    M, N, K = 131072 + 300, 64, 128
    layout = torch.arange(M, dtype=torch.int32) // 70000
    a, sfa, av = make_operand((), M, K, "mxfp4", 35)
    b, sfb, bv = make_operand((2,), N, K, "mxfp4", 36)
    d = torch.zeros((M, N), dtype=torch.bfloat16, device="cuda")
    gg.bind_contiguous_fp4(a, sfa, b, sfb, d, layout.cuda(), fmt="mxfp4")()
    check_product(d, torch.zeros_like(d), av, bv, layout, None, torch.bfloat16)


MASKED = [
    # masked_m, max_m, N, K, fmt, dtype
    ((1,), 1, 8, 128, "mxfp4", "bf16"),
    ((0, 3, 1, 8), 8, 136, 640, "nvfp4", "bf16"),
    ((33, 0, 40, 17, 5), 40, 256, 384, "mxfp4", "fp32"),
    ((200, 129, 0, 64), 200, 328, 512, "nvfp4", "bf16"),
    ((9, -3, 1000), 16, 400, 7168, "nvfp4", "fp32"),
    ((1, 1, 1, 1, 1, 1, 1, 1), 1, 1024, 2048, "nvfp4", "bf16"),
    ((0, 0), 4, 64, 128, "mxfp4", "bf16"),
    ((300, 256, 257), 300, 512, 1024, "mxfp4", "bf16"),
    # at most 32 and 128 rows: several tiles per block, no tile at all for most groups, blocks that share K
    (tuple(i % 9 for i in range(48)), 8, 1096, 512, "nvfp4", "bf16"),
    (tuple(128 - i for i in range(12)), 128, 2048, 384, "mxfp4", "fp32"),
    (tuple(5 * (i % 200 == 7) for i in range(1024)), 5, 256, 512, "mxfp4", "bf16"),
    ((100,), 100, 512, 2048, "nvfp4", "fp32"),
    ((12, 0, 0, 31), 32, 1000, 128, "mxfp4", "fp32"),
]


@pytest.mark.parametrize("counts,max_m,N,K,fmt,dtype", MASKED)
def test_product_masked(gg, counts, max_m, N, K, fmt, dtype):
    G = len(counts)
    a, sfa, av = make_operand((G,), max_m, K, fmt, 40)
    b, sfb, bv = make_operand((G,), N, K, fmt, 41)
    d = torch.full((G, max_m, N), 5.0, dtype=DT[dtype], device="cuda")
    alpha = torch.rand(G, generator=gen(42)) + 0.5
    gg.bind_masked_fp4(a, sfa, b, sfb, d, torch.tensor(counts, dtype=torch.int32, device="cuda"), alpha=alpha.cuda(), fmt=fmt)()
    assert gg.device_status() == 0
    group = torch.cat([torch.where(torch.arange(max_m) < c, g, -1) for g, c in enumerate(counts)])
    check_product(d.reshape(-1, N), torch.full((G * max_m, N), 5.0, dtype=DT[dtype]), av.reshape(-1, K), bv, group, alpha, DT[dtype])


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("M", [3, 150])
def test_product_shows_a_scale_that_is_nan(ops, gg, fmt, M):
    """Only the rows and columns whose blocks hold an infinity or a NaN become NaN."""
    x = torch.zeros((M, 256)).normal_(generator=gen(50))
    w = torch.zeros((1, 64, 256)).normal_(generator=gen(51))
    x[1, 100] = math.nan
    w[0, 9, 200] = math.inf
    a, sfa = ops.quant_fp4(x.cuda(), fmt=fmt)
    b, sfb = ops.quant_fp4(w.cuda(), fmt=fmt)
    d = torch.zeros((M, 64), device="cuda")
    gg.bind_contiguous_fp4(a, sfa, b, sfb, d, torch.zeros(M, dtype=torch.int32, device="cuda"), fmt=fmt)()
    bad = torch.zeros((M, 64), dtype=torch.bool)
    bad[1] = True
    bad[:, 9] = True
    assert torch.equal(torch.isnan(d).cpu(), bad)


def test_product_empty(gg):
    b, sfb, _ = make_operand((2,), 64, 128, "nvfp4", 60)
    d = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda")
    gg.bind_contiguous_fp4(torch.empty((0, 64), dtype=torch.uint8, device="cuda"), torch.empty((0, 4, 512), dtype=torch.uint8, device="cuda"),
                           b, sfb, d, torch.empty(0, dtype=torch.int32, device="cuda"))()
    a, sfa, _ = make_operand((), 130, 128, "nvfp4", 61)
    d = torch.full((130, 64), 2.0, device="cuda")
    gg.bind_contiguous_fp4(a, sfa, b, sfb, d, torch.full((130,), -1, dtype=torch.int32, device="cuda"))()
    assert (d == 2).all() and gg.device_status() == 0


# ------------------------------------------------------------------ together
def _layer(ops, gg, x, res, wn, wr, bias, w13, w2, top_k, work):
    """A MoE block with 4-bit experts: norm -> routing -> plan -> 4-bit rows -> product -> SiLU*mul -> product -> sum."""
    E = w13[0].shape[0]
    n = ops.rms_norm_quant(x, wn, residual=res, want_y=True)
    ids, w = ops.route(n["y"].float() @ wr, top_k, score="sigmoid", bias=bias, n_group=2, topk_group=1)
    plan = ops.permute_plan(ids, 0, E, 128)
    a1 = ops.quant_fp4(n["y"], src_pair=plan["src_pair"], top_k=top_k, out=work["a1"])
    gg.bind_contiguous_fp4(*a1, *w13, work["g1"], plan["grouped_layout"])()
    a2 = ops.quant_fp4(work["g1"], act="silu_mul")
    gg.bind_contiguous_fp4(*a2, *w2, work["y"], plan["grouped_layout"])()
    return dict(n=n, ids=ids, w=w, plan=plan, a1=a1, a2=a2, out=ops.combine(work["y"], plan["pos"], w))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("local", [256, 32, 4])
def test_quant_fp4_of_a_plan_with_few_local_experts(ops, fmt, local):
    """Gathered by a plan whose rows are mostly padding, as where few of the experts are on this GPU: x quantised once and copied,
    or row by row, gives the same, and rows without a pair are zero."""
    from tirx_harness_b200 import _lib
    T, K, E, top_k = 1500, 1024, 256, 8
    ids = torch.stack([torch.randperm(E, generator=gen(60 + t))[:top_k] for t in range(T)]).int()
    plan = ops.permute_plan(ids.cuda(), 0, local)
    x = torch.zeros((T, K)).normal_(generator=gen(27)).bfloat16()
    rows = plan["cap_rows"]
    assert _lib.lib().moe_quant_fp4_workspace_bytes(rows, T, K, 0) > 0
    src = plan["src_pair"].cpu()
    assert int((src >= 0).sum()) == int((ids < local).sum())
    f = torch.tensor([1e-3], device="cuda") if fmt == "nvfp4" else None
    q, sf = ops.quant_fp4(x.cuda(), fmt=fmt, global_scale=f, src_pair=plan["src_pair"], top_k=top_k)
    rc, rb = quant32(x.float().numpy(), fmt, np.float32(1e-3) if fmt == "nvfp4" else 1.0)
    live, t = (src >= 0).numpy(), (src // top_k).clamp(min=0).long().numpy()
    b = scale_bytes(sf, rows, K, fmt)
    np.testing.assert_array_equal(b[live], rb[t][live])
    assert same_codes(codes_of(q)[live], rc[t][live])
    assert not b[~live].any() and not q.cpu().numpy()[~live].any()
    by_row, xd = (torch.zeros_like(q), torch.zeros_like(sf)), x.cuda()
    _lib.FP4_QUANT(_lib.FP4_QUANT.pack(xd.data_ptr(), K, 0 if f is None else f.data_ptr(), 0, plan["src_pair"].data_ptr(), by_row[0].data_ptr(),
                                       by_row[1].data_ptr(), 1, rows, T, K, top_k, 0, 0 if fmt == "nvfp4" else 1, 0, 1, 0, 0),
                   torch.cuda.current_stream().cuda_stream)
    assert torch.equal(by_row[0], q) and torch.equal(by_row[1], sf)


def test_product_of_quantised_weights_is_near_the_product_of_the_weights(ops, gg):
    """With g = largest magnitude / (6 * 448) no block of ordinary weights vanishes, and the product keeps to the format's steps."""
    E, N, K, rows = 3, 264, 1408, 150
    w = torch.zeros((E, N, K)).normal_(generator=gen(71)) / K**0.5 * torch.tensor([1.0, 0.05, 20.0])[:, None, None]
    x = torch.zeros((rows, K)).normal_(generator=gen(72))
    layout = torch.arange(rows, dtype=torch.int32) * E // rows
    gw, gx = w.abs().amax((1, 2)) / (6 * 448), x.abs().amax().reshape(1) / (6 * 448)
    qw, qx = ops.quant_fp4(w.cuda(), global_scale=gw.cuda()), ops.quant_fp4(x.cuda(), global_scale=gx.cuda())
    d = torch.zeros((rows, N), device="cuda")
    gg.bind_contiguous_fp4(*qx, *qw, d, layout.cuda(), alpha=(gx * gw).cuda())()

    def step(v):                               # of each value: the largest error of its block
        amax = v.double().reshape(*v.shape[:-1], -1, 16).abs().amax(-1)
        # scales of normal e4m3 numbers (half a step: 2^-4); then the codes' largest half step is 1 in units of the scale, amax / 6
        assert (amax > v.double().abs().amax((-2, -1), keepdim=True) * 2.0**-6 / 448).all()
        return ((1 + 2.0**-4 + 1e-6) / 6 * amax).repeat_interleave(16, -1)
    sw, sx = step(w), step(x)
    back = torch.stack([torch.from_numpy(E2M1[codes_of(qw[0][e])] * np.repeat(scale_values(scale_bytes(qw[1][e], N, K, "nvfp4"), "nvfp4"), 16, -1)) * float(gw[e])
                        for e in range(E)])
    assert ((back - w.double()).abs() <= sw).all()
    for e in range(E):
        at = (layout == e).nonzero().flatten()
        ref = x[at].double() @ w[e].double().T
        off = sx[at] @ w[e].double().abs().T + x[at].double().abs() @ sw[e].T + sx[at] @ sw[e].T
        # (fp32 sums: K 2^-24 of the sum of magnitudes, of which `off` is a third and more)
        within(d[at.cuda()], ref, off * (1 + 1e-3), "product")
        # errors of random signs grow with the root of K: a sixth of the sum of the bounds is far above them
        assert (d[at.cuda()].cpu().double() - ref).norm() < off.norm() / 6


def test_run_together_captured_and_on_another_stream(ops, gg):
    T, H, I, E, top_k = 70, 512, 256, 8, 2
    g = gen(70)
    x, res = (torch.zeros((T, H)).normal_(generator=g).bfloat16().cuda() for _ in range(2))
    wn = (1 + 0.1 * torch.zeros(H).normal_(generator=g)).cuda()
    wr = (torch.zeros((H, E)).normal_(generator=g) / H**0.5).cuda()
    bias = (0.05 * torch.zeros(E).normal_(generator=g)).cuda()
    w13 = ops.quant_fp4((torch.zeros((E, 2 * I, H)).normal_(generator=g) / H**0.5).cuda())
    w2 = ops.quant_fp4((torch.zeros((E, H, I)).normal_(generator=g) / I**0.5).cuda())
    cap = ops.plan_cap_rows(T * top_k, E, 128)

    def work():
        return dict(a1=(torch.zeros((cap, H // 2), dtype=torch.uint8, device="cuda"), torch.zeros(ops.fp4_scale_shape(cap, H), dtype=torch.uint8, device="cuda")),
                    g1=torch.zeros((cap, 2 * I), dtype=torch.bfloat16, device="cuda"), y=torch.zeros((cap, H), dtype=torch.bfloat16, device="cuda"))
    w = work()
    r = _layer(ops, gg, x, res, wn, wr, bias, w13, w2, top_k, w)
    assert gg.device_status() == 0

    # each product against 64 bits, on the operands that the step before it made
    def value(op, rows, K):
        b = scale_values(scale_bytes(op[1], rows, K, "nvfp4"), "nvfp4")
        return torch.from_numpy(E2M1[codes_of(op[0])] * np.repeat(b, 16, -1))
    layout = r["plan"]["grouped_layout"]
    for a, b, d, N, K in ((r["a1"], w13, w["g1"], 2 * I, H), (r["a2"], w2, w["y"], H, I)):
        bv = torch.stack([value((b[0][e], b[1][e]), N, K) for e in range(E)])
        check_product(d, torch.zeros_like(d), value(a, cap, K), bv, layout, None, torch.bfloat16)
    pos, y = r["plan"]["pos"].cpu().long(), w["y"].cpu().double()
    terms = r["w"].cpu().double()[..., None] * y[pos]
    ref = terms.sum(1)
    within(r["out"], ref, 2.0**-8 * ref.abs() + 4 * U32 * terms.abs().sum(1), "combine")

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _layer(ops, gg, x, res, wn, wr, bias, w13, w2, top_k, work())
    side.synchronize()
    assert torch.equal(again["out"], r["out"])

    graph, wg = torch.cuda.CUDAGraph(), work()
    with torch.cuda.graph(graph):
        captured = _layer(ops, gg, x, res, wn, wr, bias, w13, w2, top_k, wg)
    for _ in range(2):
        captured["out"].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured["out"], r["out"])
    x.copy_(res)                                      # other inputs, the same graph
    graph.replay()
    fresh = _layer(ops, gg, x, res, wn, wr, bias, w13, w2, top_k, work())
    torch.cuda.synchronize()
    assert torch.equal(captured["out"], fresh["out"])


def test_gradients_captured_beside_one_another(ops):
    """Two captured backward passes, replayed on two streams, keep their own scratch memory."""
    h, dy, w = (t.cuda() for t in _norm_inputs(600, 1024, "bf16", True, 0, 80))
    rstd = (h.float().square().mean(1) + 1e-6).rsqrt()
    ref = [ops.rms_norm_backward(d, h, w, rstd) for d in (dy, -2 * dy)]
    graphs = []
    for d in (dy, -2 * dy):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = ops.rms_norm_backward(d, h, w, rstd)
        graphs.append((gr, out, torch.cuda.Stream(), d))
    torch.cuda.synchronize()
    for _ in range(5):
        for gr, _, st, _ in graphs:
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for (_, out, _, _), r in zip(graphs, ref):
        assert torch.equal(out[0], r[0]) and torch.equal(out[1], r[1])


# ------------------------------------------------------------------ refusals of the Python entry points
def test_refusals(ops, gg):
    x, w = torch.zeros((4, 256), device="cuda"), torch.ones(256, device="cuda")
    r = torch.ones(4, device="cuda")
    ids = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    bad = [
        (ValueError, lambda: ops.rms_norm_quant(x[0], w)),
        (ValueError, lambda: ops.rms_norm_quant(x.t(), w)),
        (ValueError, lambda: ops.rms_norm_quant(x, w[:8])),
        (TypeError, lambda: ops.rms_norm_quant(x, w.half())),
        (TypeError, lambda: ops.rms_norm_quant(x, w, residual=x.half())),
        (ValueError, lambda: ops.rms_norm_quant(x, w, residual=x[:3])),
        (ValueError, lambda: ops.rms_norm_quant(x, w.cpu())),
        (RuntimeError, lambda: ops.rms_norm_quant(x[:, :20], w[:20])),
        (RuntimeError, lambda: ops.rms_norm_quant(x[:, 1:9], w[:8])),
        (ValueError, lambda: ops.rms_norm_backward(x, x, w, r[:3])),
        (TypeError, lambda: ops.rms_norm_backward(x, x.half(), w, r)),
        (ValueError, lambda: ops.rms_norm_backward(x, x, w, r, dh=x[:, :128])),
        (ValueError, lambda: ops.route(x, 0)),
        (ValueError, lambda: ops.route(x, 33)),
        (ValueError, lambda: ops.route(x, 2, score="tanh")),
        (ValueError, lambda: ops.route(x, 2, group_score="mean")),
        (ValueError, lambda: ops.route(x, 2, bias=w[:8])),
        (TypeError, lambda: ops.route(x, 2, bias=w.half())),
        (RuntimeError, lambda: ops.route(x, 2, n_group=7)),
        (RuntimeError, lambda: ops.route(x, 9, n_group=32, topk_group=1)),
        (ValueError, lambda: ops.route(x.t(), 2)),
        (TypeError, lambda: ops.route_backward(x[:, :2].contiguous(), x, ids.long())),
        (ValueError, lambda: ops.route_backward(x[:, :3].contiguous(), x, ids)),
        (ValueError, lambda: ops.quant_fp4(x[:, :64])),
        (ValueError, lambda: ops.quant_fp4(x, fmt="fp4")),
        (ValueError, lambda: ops.quant_fp4(x, fmt="mxfp4", global_scale=r[:1])),
        (ValueError, lambda: ops.quant_fp4(x, global_scale=r)),
        (ValueError, lambda: ops.quant_fp4(x, act="relu")),
        (ValueError, lambda: ops.quant_fp4(x.expand(2, 4, 256))),
        (TypeError, lambda: ops.quant_fp4(x, src_pair=ids[0].long())),
        (ValueError, lambda: ops.quant_fp4(x, src_pair=ids[0], top_k=0)),
        (ValueError, lambda: ops.quant_fp4(x, out=(torch.zeros((4, 64), dtype=torch.uint8, device="cuda"), torch.zeros((1, 4, 512), dtype=torch.uint8, device="cuda")))),
        (ValueError, lambda: ops.unpack_fp4(torch.zeros(12, dtype=torch.uint8, device="cuda"))),
    ]
    a, sfa = ops.quant_fp4(x)
    b, sfb = ops.quant_fp4(torch.zeros((2, 64, 256), device="cuda"))
    d, lay = torch.zeros((4, 64), device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    bad += [
        (ValueError, lambda: gg.bind_contiguous_fp4(a, sfa, b, sfb, d[:, :56], lay)),
        (ValueError, lambda: gg.bind_contiguous_fp4(a, sfa, b, sfb, d, lay[:3])),
        (ValueError, lambda: gg.bind_contiguous_fp4(a, sfa, b, sfb, d, lay.cpu())),
        (ValueError, lambda: gg.bind_contiguous_fp4(a, sfa, b, sfb, d, lay, fmt="mxfp4")),
        (ValueError, lambda: gg.bind_contiguous_fp4(a, sfa, b, sfb, d, lay, alpha=torch.ones(3, device="cuda"))),
        (ValueError, lambda: gg.bind_contiguous_fp4(a[:, :64], sfa, b, sfb, d, lay)),
        (ValueError, lambda: gg.bind_contiguous_fp4(a, sfa, b, sfb, d.half(), lay)),
        (ValueError, lambda: gg.bind_masked_fp4(a, sfa, b, sfb, d, lay)),
        (ValueError, lambda: gg.bind_masked_fp4(a[None], sfa[None], b, sfb, d[None], lay[:1])),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            pytest.fail(f"call {i} is not refused")


def test_product_refuses_an_empty_rows_used(ops, gg):
    """Its address is NULL, which means that all rows are in use."""
    a, sfa = ops.quant_fp4(torch.zeros((4, 256), device="cuda"))
    b, sfb = ops.quant_fp4(torch.zeros((2, 64, 256), device="cuda"))
    d, lay = torch.zeros((4, 64), device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    gg.bind_contiguous_fp4(a, sfa, b, sfb, d, lay, rows_used=lay[:1])
    with pytest.raises(ValueError):
        gg.bind_contiguous_fp4(a, sfa, b, sfb, d, lay, rows_used=lay[:0])


def test_arguments_of_another_kind_are_refused(ops):
    logits = torch.zeros((2, 16), device="cuda")
    for kw in (dict(n_group=2.0), dict(topk_group="1"), dict(scale=None)):
        with pytest.raises(TypeError):
            ops.route(logits, 2, **kw)
    for kw in (dict(n_group=1 << 40), dict(scale=10**400)):
        with pytest.raises(ValueError):
            ops.route(logits, 2, **kw)
    with pytest.raises(TypeError):
        ops.rms_norm_quant(torch.zeros((2, 128), device="cuda"), torch.ones(128, device="cuda"), eps="1e-6")
    with pytest.raises(TypeError):
        ops.quant_fp4(torch.zeros((2, 128), device="cuda"), src_pair=torch.zeros(2, dtype=torch.int32, device="cuda"), top_k=1.5)



# ------------------------------------------------------------------ offsets past 32 bits
def test_offsets_past_32_bits(ops, gg):
    """More than 2^32 bytes (and 2^31 elements) in front of the last rows, which are compared with the same rows alone."""
    T, H, tail = 540000, 4096, 130
    g = gen(90)
    last = torch.zeros((tail, H)).normal_(generator=g).bfloat16().cuda()
    w = torch.ones(H, device="cuda", dtype=torch.bfloat16)
    x = torch.zeros((T, H), dtype=torch.bfloat16, device="cuda")
    x[-tail:] = last
    big, small = ops.rms_norm_quant(x, w), ops.rms_norm_quant(last, w)
    assert torch.equal(big["q"][-tail:].view(torch.uint8), small["q"].view(torch.uint8)) and torch.equal(big["scales"][-tail:], small["scales"])
    del big
    dx, dw = ops.rms_norm_backward(x, x, w, torch.ones(T, device="cuda"))
    dx0, _ = ops.rms_norm_backward(last, last, w, torch.ones(tail, device="cuda"))
    assert torch.equal(dx[-tail:], dx0) and torch.isfinite(dw).all()
    del dx
    q, sf = ops.quant_fp4(x)
    first = (T - tail) // 128 * 128                                       # whole tiles
    q0, sf0 = ops.quant_fp4(x[first:])
    assert torch.equal(q[first:], q0) and torch.equal(sf[first // 128:], sf0)
    assert torch.equal(ops.unpack_fp4(q)[-tail:].view(torch.uint8), ops.unpack_fp4(q[-tail:].contiguous()).view(torch.uint8))
    del q, sf
    ids, wt = ops.route(x[:, :1024], 3)
    ids0, wt0 = ops.route(last[:, :1024], 3)
    assert torch.equal(ids[-tail:], ids0) and torch.equal(wt[-tail:], wt0)
    z = x.view(-1, 1024)                                                  # dense rows for the gradient
    gr = torch.ones((z.shape[0], 2), device="cuda")
    at = torch.tensor([3, 700], dtype=torch.int32, device="cuda").expand(z.shape[0], 2).contiguous()
    assert torch.equal(ops.route_backward(gr, z, at)[-tail:], ops.route_backward(gr[-tail:], z[-tail:], at[-tail:]))
    del x, z, gr, at
    # a product whose output passes 2^32 bytes
    a, sfa, av = make_operand((), 256, 128, "mxfp4", 91)
    b, sfb, bv = make_operand((2,), H, 128, "mxfp4", 92)
    M = T // 128 * 128
    rows = torch.zeros((M, 64), dtype=torch.uint8, device="cuda")
    tiles = torch.zeros(ops.fp4_scale_shape(M, 128, "mxfp4"), dtype=torch.uint8, device="cuda")
    rows[-256:], tiles[-2:] = a, sfa
    layout = torch.zeros(M, dtype=torch.int32, device="cuda")
    layout[-200:] = 1
    d = torch.empty((M, H), dtype=torch.bfloat16, device="cuda")
    gg.bind_contiguous_fp4(rows, tiles, b, sfb, d, layout, fmt="mxfp4")()
    check_product(d[-256:], torch.zeros((256, H), dtype=torch.bfloat16), av, bv, layout[-256:].cpu(), None, torch.bfloat16)
