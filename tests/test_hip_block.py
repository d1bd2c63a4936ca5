"""The feed-forward half of a trainable block (iffnerf_amd/hip_block.py) against the formulas in 64 bits.

Bounds: a result is rounded to its type once (at most u |result|, u = 2^-24 / 2^-8 / 2^-11 for fp32 / bf16 / fp16); what fp32 arithmetic loses
before that is a number of roundings (the depth of the longest chain of additions, written at each bound) times 2^-24 times the sum of
the magnitudes that are added, propagated through the formulas by their derivatives.
"""
import math

import pytest
import torch

from iffnerf_amd import hip_block

gpu = pytest.mark.gpu
E = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}      # the spacing of subnormals
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def normal(shape, seed, dtype=torch.float32, scale=1.0, shift=0.0, device="cuda:0"):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale + shift).to(dtype).to(device)


def within(got, want, before, name):
    """|got - want| <= u (|want| + before) + before + the type's smallest step, per element."""
    u = U[got.dtype]
    lim = u * want.abs() + (1 + u) * before + TINY[got.dtype]
    d = (got.double() - want).abs()
    assert got.shape == want.shape
    bad = ~(d <= lim)
    assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst {float((d / lim).max()):.3g} x the bound"


# ------------------------------------------------------------------------------------------------------------ layer norm
def norm_reference(x, w, b, eps, dy):
    """(y, dx, dw, db) in 64 bits with what fp32 may lose before the last rounding: depth <= 32 additions per lane + 10 across lanes."""
    X, G = x.double().reshape(-1, x.shape[-1]), dy.double().reshape(-1, x.shape[-1])
    W = torch.ones_like(X[0]) if w is None else w.double()
    Bv = torch.zeros_like(X[0]) if b is None else b.double()
    D, rows = X.shape[1], X.shape[0]
    k = 48.0 * E
    if D > 4096:
        k = (48.0 + D / 256.0) * E                                       # the any-width form adds D / 256 values per lane
    mean = X.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt(((X - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (X - mean) * r
    big = X.abs().amax(1, keepdim=True) * r                                # the mean's error, in units of the norm
    exh = k * (big + xh.abs())
    y = xh * W + Bv
    ey = exh * W.abs() + 4 * E * (y.abs() + Bv.abs())
    e = G * W
    m1, m2 = e.mean(1, keepdim=True), (e * xh).mean(1, keepdim=True)
    a1, a2 = e.abs().mean(1, keepdim=True), (e * xh).abs().mean(1, keepdim=True)
    dx = r * (e - m1 - xh * m2)
    em2 = k * a2 + (e.abs() * exh).mean(1, keepdim=True)
    edx = r * (4 * E * e.abs() + k * a1 + xh.abs() * em2 + exh * m2.abs()) + k * (1 + big) * dx.abs() + 4 * E * r * (xh * m2).abs()
    n = (64.0 + rows / 512.0) * E                                           # rows of a workgroup, its waves, the workgroups' shares
    dw, edw = (G * xh).sum(0), (G.abs() * exh).sum(0) + n * (G * xh).abs().sum(0)
    db, edb = G.sum(0), n * G.abs().sum(0)
    return (y, dx.reshape(x.shape), dw, db), (ey, edx.reshape(x.shape), edw, edb)


def check_norm(x, w, b, eps, dy):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = hip_block.layer_norm(leaves[0], leaves[1], leaves[2], eps)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    live = [t for t in leaves if t is not None]
    grads = dict(zip([i for i, t in enumerate(leaves) if t is not None], torch.autograd.grad(y, live, dy)))
    want, lim = norm_reference(x, w, b, eps, dy)
    within(y.detach().reshape(-1, x.shape[-1]), want[0], lim[0], "y")
    for i, name in enumerate(("dx", "dw", "db")):
        if i in grads:
            within(grads[i], want[1 + i], lim[1 + i], name)
    with torch.no_grad():
        assert torch.equal(hip_block.layer_norm(x, w, b, eps), y)            # the form without statistics: the same bits


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 2), (1, 384), (5, 8), (7, 65), (257, 384), (33, 387), (130, 512), (9, 1001), (64, 1024), (6, 1536),
                                    (5, 2049), (4, 4096), (3, 5000), (3, 8192), (2, 8200), (2, 20011)])
def test_layer_norm(dev, rows, D, dtype):
    x = normal((rows, D), 10 * rows + D, dtype, 1.5, 0.7)
    w, b = normal((D,), 1, dtype, 0.2, 1.0), normal((D,), 2, dtype, 0.3)
    check_norm(x, w, b, 1e-6, normal((rows, D), 3, dtype))


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("which", ["no_affine", "no_bias", "bias_only", "fp32_parameters"])
def test_layer_norm_parameters(dev, which, dtype):
    x, dy = normal((70, 136), 4, dtype), normal((70, 136), 5, dtype)
    par = torch.float32 if which == "fp32_parameters" else dtype
    w = None if which in ("no_affine", "bias_only") else normal((136,), 6, par, 0.2, 1.0)
    b = None if which in ("no_affine", "no_bias") else normal((136,), 7, par)
    check_norm(x, w, b, 1e-5, dy)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_layer_norm_layouts(dev, dtype):
    w, b = normal((40,), 8, dtype, 0.2, 1.0), normal((40,), 9, dtype)
    base = normal((3, 11, 48), 10, dtype)
    views = [base[:, 1:, :40], base[:, :, 8:], base[:, :, 3:43], base[:, ::2, :40], base[:, :, :40].transpose(0, 1), base[1, :, :40],
             base[:, 2, :40], base[0, 0, :40], base[:1, :, :40].expand(4, 11, 40), base[:, :, 0::1][..., :40].unsqueeze(1),
             base.permute(2, 0, 1)[:40].permute(1, 2, 0), base.permute(1, 2, 0)[:, :40, :].transpose(1, 2), base[:0, :, :40]]
    for x in views:
        dy = normal(tuple(x.shape), 11, dtype)
        check_norm(x, w, b, 1e-6, dy)
        check_norm(x, w, b, 1e-6, dy[..., :1].expand(x.shape))             # a broadcast gradient
    flat = normal((5 * 40 + 1,), 12, dtype)[1:].view(5, 40)               # a start that no vector access is aligned to
    check_norm(flat, w, b, 1e-6, normal((5, 40), 13, dtype))


@gpu
def test_layer_norm_many_rows(dev):
    """More rows than the backward pass has workgroups; the same bits again; parameters alone, input alone."""
    x, dy = normal((70001, 40), 14), normal((70001, 40), 15)
    w, b = normal((40,), 16, scale=0.2, shift=1.0), normal((40,), 17)
    check_norm(x, w, b, 1e-6, dy)
    X, W, B = x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    full = torch.autograd.grad(hip_block.layer_norm(X, W, B), (X, W, B), dy)
    again = torch.autograd.grad(hip_block.layer_norm(X, W, B), (X, W, B), dy)
    assert all(torch.equal(a, c) for a, c in zip(full, again))
    assert torch.equal(torch.autograd.grad(hip_block.layer_norm(X, W.detach(), B.detach()), (X,), dy)[0], full[0])
    assert torch.equal(torch.autograd.grad(hip_block.layer_norm(X.detach(), W, B.detach()), (W,), dy)[0], full[1])
    assert torch.equal(torch.autograd.grad(hip_block.layer_norm(X.detach(), W.detach(), B), (B,), dy)[0], full[2])


@gpu
def test_layer_norm_values_at_the_edge(dev):
    """Constant rows (variance 0), a level far above the spread, NaN and infinite rows that must not reach their neighbours."""
    x = normal((8, 384), 18)
    x[1] = 5.0
    x[2] += 4096.0
    x[4, 7] = float("nan")
    x[6, 3] = float("inf")
    y = hip_block.layer_norm(x, None, None, 1e-6)
    assert torch.equal(y[1], torch.zeros_like(y[1]))
    assert bool(y[4].isnan().all()) and bool(y[6].isnan().all())
    fine = [0, 2, 3, 5, 7]
    want, lim = norm_reference(x[fine], None, None, 1e-6, x[fine])
    within(y[fine], want[0], lim[0], "y")


@gpu
def test_layer_norm_gradient_against_differences(dev):
    x, dy = normal((6, 48), 19), normal((6, 48), 20)
    w, b = normal((48,), 21, scale=0.2, shift=1.0), normal((48,), 22)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(hip_block.layer_norm(*leaves, 1e-5), leaves, dy)

    def f(X, W, B):
        m = X.mean(1, keepdim=True)
        return (((X - m) / torch.sqrt(((X - m) ** 2).mean(1, keepdim=True) + 1e-5) * W + B) * dy.double()).sum()

    at = [t.detach().double() for t in leaves]
    for i, g in enumerate(grads):
        step = normal(tuple(g.shape), 23 + i).double()
        lo, hi = ([a + s * 1e-5 * step if j == i else a for j, a in enumerate(at)] for s in (-1.0, 1.0))
        num = (f(*hi) - f(*lo)) / 2e-5
        # differences: third derivative times step^2 (1e-10 times O(100)); gradient: 2^-17 of its summed magnitudes
        assert abs(float((g.double() * step).sum() - num)) <= 2.0 ** -17 * float((g.double() * step).abs().sum()) + 1e-6


# ------------------------------------------------------------------------------------------------------------ gated feed-forward
def act64(g, name):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    c = 0.5 * torch.erfc(-g / math.sqrt(2.0))
    return g * c, c + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def mlp_reference(x, w12, b12, w3, b3, act, dy, pairs=False):
    """(y, dx, dw12, db12, dw3, db3) in 64 bits with a bound on what the operator loses before the last rounding.  A product over K runs
    as a chain of K / 16 matrix instructions (six times as many in fp32), 16 + 8 more for the adds inside one, the bias and the join of a
    split; an instruction may truncate: twice.  h and [dg | du] are rounded to the type (u) on the way; |act'| < 1.13, |act''| < 0.8; the
    activation's own evaluation is good to (4 + |g|) 2^-23.  ``pairs``: what the rounding of h and [dg | du] leaves is kept, rounded (u u),
    in products of twice as many terms."""
    u = U[x.dtype] ** 2 if pairs else U[x.dtype]
    six = 6 if x.dtype == torch.float32 else 1
    u_way = 0.0 if x.dtype == torch.float32 else u                         # (fp32 h and [dg | du] are split exactly, but are fp32: E below)

    def depth(k):
        return 2.0 * (six * (2 if pairs else 1) * k / 16.0 + 24.0) * E

    X, W, V, G = x.double(), w12.double(), w3.double(), dy.double()
    H = V.shape[1]
    gu = X @ W.t() + (0 if b12 is None else b12.double())
    egu = depth(X.shape[1]) * (X.abs() @ W.abs().t() + (0 if b12 is None else b12.double().abs()))
    g, uu, eg, eu = gu[:, :H], gu[:, H:], egu[:, :H], egu[:, H:]
    f, df = act64(g, act)
    c = (4.0 + g.abs()) * 2 * E
    ef, edf = 1.13 * eg + c * (f.abs() + c), 0.8 * eg + c * (df.abs() + 1.0)
    h = f * uu
    eh = f.abs() * eu + (uu.abs() + eu) * ef + (u_way + 2 * E) * h.abs() + TINY[x.dtype]
    y = h @ V.t() + (0 if b3 is None else b3.double())
    ey = eh @ V.abs().t() + depth(H) * (h.abs() @ V.abs().t() + (0 if b3 is None else b3.double().abs()))
    dh = G @ V
    edh = depth(G.shape[1]) * (G.abs() @ V.abs())
    p, ep = uu * df, df.abs() * eu + (uu.abs() + eu) * edf + 2 * E * (uu * df).abs()
    dg, du = dh * p, dh * f
    edg = (dh.abs() + edh) * ep + edh * p.abs() + (u_way + 2 * E) * dg.abs() + TINY[x.dtype]
    edu = (dh.abs() + edh) * ef + edh * f.abs() + (u_way + 2 * E) * du.abs() + TINY[x.dtype]
    d, ed = torch.cat((dg, du), 1), torch.cat((edg, edu), 1)
    M = X.shape[0]
    out = (y, d @ W, d.t() @ X, d.sum(0), G.t() @ h, G.sum(0))
    lim = (ey, ed @ W.abs() + depth(2 * H) * (d.abs() @ W.abs()), ed.t() @ X.abs() + depth(M) * (d.abs().t() @ X.abs()),
           ed.sum(0) + depth(M) * d.abs().sum(0), G.abs().t() @ eh + depth(M) * (G.abs().t() @ h.abs()), depth(M) * G.abs().sum(0))
    return out, lim


def make_mlp(M, D, H, O, dtype, bias, seed=0):
    x, dy = normal((M, D), seed + 1, dtype), normal((M, O), seed + 2, dtype, 0.1)
    w12, w3 = normal((2 * H, D), seed + 3, dtype, D ** -0.5), normal((O, H), seed + 4, dtype, H ** -0.5)
    b12, b3 = (normal((2 * H,), seed + 5, dtype, 0.3), normal((O,), seed + 6, dtype, 0.3)) if bias else (None, None)
    return x, w12, b12, w3, b3, dy


NAMES = ("dx", "dw12", "db12", "dw3", "db3")


def check_mlp(x, w12, b12, w3, b3, dy, act):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w12, b12, w3, b3)]
    y = hip_block.gated_mlp(*leaves, activation=act)
    live = [i for i, t in enumerate(leaves) if t is not None]
    grads = torch.autograd.grad(y, [leaves[i] for i in live], dy)
    want, lim = mlp_reference(x, w12, b12, w3, b3, act, dy)
    within(y.detach(), want[0], lim[0], "y")
    for i, g in zip(live, grads):
        within(g, want[1 + i], lim[1 + i], NAMES[i])
    with torch.no_grad():
        within(hip_block.gated_mlp(x, w12, b12, w3, b3, activation=act), want[0], lim[0], "y without gradients")
    return grads


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,D,H,O,act,bias", [
    (1, 1, 1, 1, "silu", True), (1, 384, 1024, 384, "silu", True), (2, 8, 16, 8, "gelu", True), (3, 387, 131, 65, "silu", False),
    (5, 64, 264, 72, "gelu", True), (16, 384, 1024, 384, "silu", True), (17, 72, 200, 136, "gelu", False), (64, 65, 67, 66, "silu", True),
    (100, 384, 1024, 384, "gelu", True), (129, 129, 129, 129, "silu", True), (257, 384, 1024, 384, "silu", True),
    (300, 40, 520, 24, "gelu", True), (515, 256, 256, 256, "silu", False), (1100, 96, 328, 104, "gelu", True), (1031, 97, 259, 101, "silu", True)])
def test_gated_mlp(dev, M, D, H, O, act, bias, dtype):
    check_mlp(*make_mlp(M, D, H, O, dtype, bias, seed=M + D), act)


@gpu
@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("M,D,H,O,act,bias", [
    (1, 1, 1, 1, "silu", True), (1, 384, 1024, 384, "gelu", True), (2, 568, 2392, 568, "gelu", False), (3, 387, 1029, 395, "silu", True),
    (8, 1536, 4096, 1536, "silu", True), (8, 65, 67, 66, "gelu", True)])
def test_gated_mlp_few_rows_are_exact_to_one_rounding(dev, M, D, H, O, act, bias, dtype):
    """Up to 8 rows the hidden activation and its gradient keep what their rounding leaves: every result is its own rounding off, and no more."""
    x, w12, b12, w3, b3, dy = make_mlp(M, D, H, O, dtype, bias, seed=7 * M + D)
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w12, b12, w3, b3)]
    y = hip_block.gated_mlp(*leaves, activation=act)
    live = [i for i, t in enumerate(leaves) if t is not None]
    grads = torch.autograd.grad(y, [leaves[i] for i in live], dy)
    want, lim = mlp_reference(x, w12, b12, w3, b3, act, dy, pairs=True)
    within(y.detach(), want[0], lim[0], "y")
    for i, g in zip(live, grads):
        within(g, want[1 + i], lim[1 + i], NAMES[i])


# large sizes: whole 256 x 256 tiles, 256 x 192 ones of a weight gradient, a gate product in two launches, shares of a weight gradient, one round
# and several; one row more, one less (tests/test_hip_block_plans.py holds sizes that take every form)
@gpu
@pytest.mark.parametrize("M,D,H,O,dtype", [
    (16384 + 64, 1536, 256, 192, torch.bfloat16), (8192 + 40, 192, 1024, 1536, torch.bfloat16), (16384, 192, 2048, 384, torch.float16),
    (4096 + 1, 768, 520, 768, torch.float16), (2048 + 255, 1536, 4096, 1536, torch.bfloat16), (4111, 384, 1023, 385, torch.float32),
    (2049, 1536, 512, 1536, torch.float32), (8192 + 64, 128, 4096, 64, torch.bfloat16)])
def test_gated_mlp_tile_shapes(dev, M, D, H, O, dtype):
    check_mlp(*make_mlp(M, D, H, O, dtype, True, seed=M), "silu")


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_gated_mlp_layouts_and_partial_gradients(dev, dtype):
    """Leading axes, strided inputs and weights, starts no 16-byte access is aligned to; every subset of gradients the same bits."""
    x, w12, b12, w3, b3, dy = make_mlp(60, 48, 80, 40, dtype, True, seed=50)
    full = check_mlp(x, w12, b12, w3, b3, dy, "silu")
    y = hip_block.gated_mlp(x, w12, b12, w3, b3)
    assert torch.equal(hip_block.gated_mlp(x.reshape(3, 4, 5, 48), w12, b12, w3, b3), y.reshape(3, 4, 5, 40))
    wide = torch.zeros(60, 64, dtype=dtype, device=dev)
    wide[:, 8:56] = x
    assert torch.equal(hip_block.gated_mlp(wide[:, 8:56], w12.t().contiguous().t(), b12, w3.t().contiguous().t(), b3), y)
    off = lambda t: torch.cat((t.new_zeros(1), t.reshape(-1)))[1:].view(t.shape)  # noqa: E731
    assert torch.equal(hip_block.gated_mlp(x[0], w12, b12, w3, b3), hip_block.gated_mlp(x[:1], w12, b12, w3, b3)[0])
    check_mlp(off(x), off(w12), off(b12), off(w3), off(b3), off(dy), "silu")
    args = [x, w12, b12, w3, b3]
    for i in range(5):
        one = [t.detach().requires_grad_(j == i) for j, t in enumerate(args)]
        assert torch.equal(torch.autograd.grad(hip_block.gated_mlp(*one), (one[i],), dy)[0], full[i]), NAMES[i]
    # a broadcast gradient, no rows
    leaves = [t.detach().requires_grad_(True) for t in args]
    g1 = torch.autograd.grad(hip_block.gated_mlp(*leaves).sum(), leaves)
    g2 = torch.autograd.grad(hip_block.gated_mlp(*leaves), leaves, torch.ones(60, 40, dtype=dtype, device=dev))
    assert all(torch.equal(a, c) for a, c in zip(g1, g2))
    none = torch.autograd.grad(hip_block.gated_mlp(x[:0], *leaves[1:]), leaves[1:], dy[:0])
    assert all(bool((t == 0).all()) for t in none)


@gpu
def test_gated_mlp_values_at_the_edge(dev):
    """Gates far out on both sides (the exponential overflows), zeros, the type's range in the hidden activation; a NaN row stays a row."""
    for act in ("silu", "gelu"):
        x, w12, b12, w3, b3, dy = make_mlp(6, 16, 32, 16, torch.float32, True, seed=70)
        b12[:32] = torch.linspace(-300.0, 300.0, 32)
        check_mlp(x, w12, b12, w3, b3, dy, act)
        x[2] = 0.0
        check_mlp(x, w12, b12, w3, b3, dy, act)
        x[4, 3] = float("nan")
        y = hip_block.gated_mlp(x, w12, b12, w3, b3, activation=act)
        assert bool(y[4].isnan().all()) and not bool(y[[0, 1, 2, 3, 5]].isnan().any())
    x, w12, b12, w3, b3, dy = make_mlp(6, 16, 32, 16, torch.bfloat16, True, seed=71)
    check_mlp(x * 1e3, w12, b12, w3, b3, dy, "silu")                         # g and u beyond fp16's range, inside bf16's
    x, w12, b12, w3, b3, dy = make_mlp(6, 16, 32, 16, torch.float32, True, seed=72)
    check_mlp(x * 1e18, w12 * 1e-18, b12, w3 * 1e12, b3, dy * 1e-12, "silu")   # pieces of very large and very small values


@gpu
def test_gated_mlp_gradient_against_differences(dev):
    x, w12, b12, w3, b3, dy = make_mlp(7, 24, 40, 16, torch.float32, True, seed=80)
    leaves = [t.requires_grad_(True) for t in (x, w12, b12, w3, b3)]
    grads = torch.autograd.grad(hip_block.gated_mlp(*leaves, activation="gelu"), leaves, dy)

    def f(X, W, B, V, C):
        gu = X @ W.t() + B
        return ((act64(gu[:, :40], "gelu")[0] * gu[:, 40:] @ V.t() + C) * dy.double()).sum()

    at = [t.detach().double() for t in leaves]
    for i, g in enumerate(grads):
        step = normal(tuple(g.shape), 90 + i).double()
        lo, hi = ([a + s * 1e-5 * step if j == i else a for j, a in enumerate(at)] for s in (-1.0, 1.0))
        num = (f(*hi) - f(*lo)) / 2e-5
        assert abs(float((g.double() * step).sum() - num)) <= 2.0 ** -17 * float((g.double() * step).abs().sum()) + 1e-6


# ------------------------------------------------------------------------------------------------------------ dropout
def philox_bits(n, seed, offset):
    """16 bits per value with Python integers: Philox 4x32-10 of (block, offset) under ``seed``."""
    out = []
    for block in range((n + 7) // 8):
        c = [block & 0xFFFFFFFF, block >> 32, offset & 0xFFFFFFFF, offset >> 32]
        k = [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(10):
            p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        for w in c:
            out += [w & 0xFFFF, w >> 16]
    return torch.tensor(out[:n])


def test_the_generator_of_this_file_is_philox():
    """The published known answers of Philox 4x32-10 (counter and key all zeros; all ones), as the words the bits above are halves of."""
    z = philox_bits(8, 0, 0).tolist()
    assert [z[2 * i] | z[2 * i + 1] << 16 for i in range(4)] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("n,p,seed,offset,res", [(1, 0.5, 0, 0, False), (7, 0.3, 1, 2, True), (8, 0.1, 2 ** 63 + 5, 2 ** 40 + 1, True),
                                                 (4099, 0.1, 12345, 0, True), (4099, 0.5, 2 ** 64 - 1, 2 ** 64 - 1, False),
                                                 (1000, 0.0, 3, 3, True), (1000, 1.0, 3, 3, True), (1000, 1.0, 3, 3, False), (2051, 1e-6, 9, 9, False)])
def test_dropout(dev, n, p, seed, offset, res, dtype):
    x, dy = normal((n,), n, dtype).requires_grad_(True), normal((n,), n + 1, dtype)
    r = normal((n,), n + 2, dtype).requires_grad_(True) if res else None
    y = hip_block.dropout(x, p, seed, offset, residual=r)
    t = int(math.floor(p * 65536 + 0.5))
    keep = (philox_bits(n, seed, offset) >= t).to(dev)
    scale = 65536.0 / (65536 - t) if t < 65536 else 0.0
    want = torch.where(keep, x.detach().double() * scale, 0.0)
    lost = 2 * E * want.abs()                                                # the factor is fp32, the product (or the fused add) one rounding
    within(y.detach(), want + (r.detach().double() if res else 0.0), lost, "y")
    grads = torch.autograd.grad(y, (x, r) if res else (x,), dy)
    gwant = torch.where(keep, dy.double() * scale, 0.0)
    within(grads[0], gwant, 2 * E * gwant.abs(), "dx")
    if res:
        assert torch.equal(grads[1], dy)
    tensor = torch.tensor([seed - 2 ** 64 if seed >= 2 ** 63 else seed], dtype=torch.int64, device=dev)
    y2 = hip_block.dropout(x, p, tensor, offset, residual=r)
    assert torch.equal(y2, y)
    assert torch.equal(torch.autograd.grad(y2, (x,), dy)[0], grads[0])


@gpu
def test_dropout_layouts_and_values(dev):
    x = normal((37, 11, 6), 30, torch.bfloat16)
    y = hip_block.dropout(x, 0.4, 77)
    assert torch.equal(hip_block.dropout(x.transpose(0, 1).contiguous().transpose(0, 1), 0.4, 77), y)       # positions go by index, not by address
    off = torch.cat((x.new_zeros(1), x.reshape(-1)))[1:].view(x.shape)                                     # no 16-byte alignment
    assert torch.equal(hip_block.dropout(off, 0.4, 77), y)
    assert torch.equal(hip_block.dropout(x.float(), 0.4, 77) == 0, y == 0)                                 # ... nor by type
    assert not torch.equal(hip_block.dropout(x, 0.4, 78) == 0, y == 0) and not torch.equal(hip_block.dropout(x, 0.4, 77, 1) == 0, y == 0)
    bad = torch.where(y == 0, torch.tensor(float("nan"), device=dev, dtype=x.dtype), x)
    assert torch.equal(hip_block.dropout(bad, 0.4, 77), y)                                                 # what is dropped never arrives
    assert hip_block.dropout(x[:0], 0.4, 77).shape == (0, 11, 6)
    # the share that is kept: 5 standard deviations of a binomial count
    n = 1 << 20
    kept = int((hip_block.dropout(torch.ones(n, device=dev), 0.25, 5) != 0).sum())
    assert abs(kept - 0.75 * n) <= 5 * math.sqrt(n * 0.25 * 0.75)


@gpu
def test_offsets_past_32_bits(dev):
    """Tensors of more than 2^31 elements (2^32 bytes and more): the last values against small calls on the same values."""
    n = 2 ** 31 + 13
    y = hip_block.dropout(torch.ones(n, dtype=torch.bfloat16, device=dev), 0.5, 11)
    last = (n - 1) // 8
    bits = []
    c, k = [last, 0, 0, 0], [11, 0]
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    for w in c:
        bits += [w & 0xFFFF, w >> 16]
    assert y[last * 8:].tolist() == [2.0 if b >= 32768 else 0.0 for b in bits[:n - last * 8]]
    del y
    base = torch.zeros(2 ** 32 + 128, dtype=torch.float16, device=dev)
    x = base.as_strided((2, 64), (2 ** 32 + 64, 1))
    x.copy_(normal((2, 64), 60, torch.float16))
    assert torch.equal(hip_block.layer_norm(x), hip_block.layer_norm(x.contiguous()))
    del base, x
    rows = normal((2 ** 24 + 7, 1), 64, torch.float16).expand(-1, 8) * torch.arange(8, device=dev, dtype=torch.float16)
    assert torch.equal(hip_block.layer_norm(rows)[-9:], hip_block.layer_norm(rows[-9:]))       # more rows than one launch has workgroups for
    del rows
    M, D, H = 2 ** 20 + 300, 2048, 8
    x = torch.zeros(M, D, dtype=torch.bfloat16, device=dev)
    tail = normal((300, D), 61, torch.bfloat16)
    x[-300:] = tail
    _, w12, b12, w3, b3, _ = make_mlp(1, D, H, 8, torch.bfloat16, True, seed=62)
    small, large = tail.requires_grad_(True), x.requires_grad_(True)
    dy = normal((300, 8), 63, torch.bfloat16)
    ys, yl = hip_block.gated_mlp(small, w12, b12, w3, b3), hip_block.gated_mlp(large, w12, b12, w3, b3)
    gs = torch.autograd.grad(ys, small, dy)[0]
    gl = torch.autograd.grad(yl, large, torch.cat((torch.zeros(M - 300, 8, dtype=torch.bfloat16, device=dev), dy)))[0]
    want, lim = mlp_reference(tail.detach(), w12, b12, w3, b3, "silu", dy)
    for got, i in ((ys, 0), (yl[-300:], 0), (gs, 1), (gl[-300:], 1)):
        within(got.detach(), want[i], lim[i], "the last rows")
    assert not bool(gl[:-300].any())


@gpu
def test_dropout_seed_tensor_that_changes_is_noticed(dev):
    x, seed = normal((64,), 31).requires_grad_(True), torch.tensor([4], device=dev)
    y = hip_block.dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), (x,))


# ------------------------------------------------------------------------------------------------------------ together
def half_block(x, nw, nb, w12, b12, w3, b3, seed):
    return hip_block.dropout(hip_block.gated_mlp(hip_block.layer_norm(x, nw, nb), w12, b12, w3, b3), 0.1, seed, residual=x)


def half_block_64(x, nw, nb, w12, b12, w3, b3, keep):
    m = x.mean(-1, keepdim=True)
    n = (x - m) / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + 1e-6) * nw + nb
    gu = n @ w12.t() + b12
    H = w3.shape[1]
    t = 6554
    return x + (torch.nn.functional.silu(gu[..., :H]) * gu[..., H:] @ w3.t() + b3) * keep * (65536.0 / (65536 - t))


def block_inputs(dtype, B=3, T=33, D=96, H=256):
    x = normal((B, T, D), 100, dtype)
    nw, nb = normal((D,), 101, dtype, 0.2, 1.0), normal((D,), 102, dtype, 0.2)
    _, w12, b12, w3, b3, _ = make_mlp(1, D, H, D, dtype, True, seed=103)
    return [x, nw, nb, w12, b12, w3, b3], normal((B, T, D), 110, dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_the_half_block(dev, dtype):
    """All three together, forward and backward.  Normwise: every tensor on the way is rounded once (6 roundings forward, 7 more back),
    each at most u of the 2-norm, and the linear maps between them have condition O(1) here: 16 u of the gradient's norm.  In fp32 the
    sums themselves round in u too, over chains of up to 256 / 16 x 6 = 96 matrix instructions, whose random roundings add to
    sqrt(96) < 10 half-u each: 3 products deep, 16 u + 3 x 10 u < 64 u."""
    args, dy = block_inputs(dtype)
    leaves = [t.requires_grad_(True) for t in args]
    y = half_block(*leaves, 99)
    grads = torch.autograd.grad(y, leaves, dy)
    keep = (philox_bits(dy.numel(), 99, 0) >= 6554).double().to(dev).reshape(dy.shape)
    l64 = [t.detach().double().requires_grad_(True) for t in args]
    y64 = half_block_64(*l64, keep)
    g64 = torch.autograd.grad(y64, l64, dy.double())
    for name, a, b in zip(("y", "dx", "dnw", "dnb", "dw12", "db12", "dw3", "db3"), (y, *grads), (y64, *g64)):
        assert float((a.detach().double() - b.detach()).norm() / b.detach().norm()) <= 16 * U[dtype] * (4 if dtype == torch.float32 else 1), name


@gpu
def test_the_half_block_in_a_graph_and_on_other_streams(dev):
    """A captured step (forward and gradients) replayed on refilled inputs and seeds against the eager result, two graphs in turn with
    eager work between; the eager step on a side stream."""
    args, dy = block_inputs(torch.bfloat16)
    seed = torch.tensor([7], device=dev)

    def step(leaves, seed):
        y = half_block(*leaves, seed)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    def make():
        leaves = [t.clone().requires_grad_(True) for t in args]
        s = seed.clone()
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            step(leaves, s)
        torch.cuda.current_stream(dev).wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(leaves, s)
        return g, leaves, s, out

    graphs = [make(), make()]
    for k in range(4):
        for j, (g, leaves, s, out) in enumerate(graphs):
            fresh = normal((3, 33, 96), 200 + 2 * k + j, torch.bfloat16)
            with torch.no_grad():
                leaves[0].copy_(fresh)
                s.fill_(1000 + 2 * k + j)
        for g, *_ in graphs:
            g.replay()
        want = [step([t.detach().clone().requires_grad_(True) for t in leaves], s.clone()) for _, leaves, s, _ in graphs]
        torch.cuda.synchronize()
        for (_, _, _, out), w in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w))
    side = torch.cuda.Stream(dev)
    leaves = [t.detach().clone().requires_grad_(True) for t in args]
    base = step(leaves, seed)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = step(leaves, seed)
    torch.cuda.current_stream(dev).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(base, other))


@gpu
def test_the_half_block_twice_from_one_graph_and_from_two_threads(dev):
    """Gradients taken twice from a graph that is kept, and two threads that run the block at once on streams of their own: the same bits."""
    import threading
    args, dy = block_inputs(torch.bfloat16)

    def leaves():
        return [t.detach().clone().requires_grad_(True) for t in args]

    mine = leaves()
    y = half_block(*mine, 11)
    first = torch.autograd.grad(y, mine, dy, retain_graph=True)
    second = torch.autograd.grad(y, mine, dy)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    torch.cuda.synchronize()
    got = {}

    def run(k):
        stream = torch.cuda.Stream(dev)
        with torch.cuda.stream(stream):
            for _ in range(5):
                own = leaves()
                out = half_block(*own, 11)
                got[k] = (out.detach(), *torch.autograd.grad(out, own, dy))
        stream.synchronize()

    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(2):
        assert all(torch.equal(a, b) for a, b in zip((y.detach(), *first), got[k]))


@gpu
def test_first_derivatives_only(dev):
    x = normal((4, 16), 40).requires_grad_(True)
    g, = torch.autograd.grad(hip_block.layer_norm(x).sum(), (x,), create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ------------------------------------------------------------------------------------------------------------ the backbone in training
def backbone(ffn, drop, **kw):
    from iffnerf_amd.pose_estimation.backbone import SeededViTS14
    return SeededViTS14(seed=3, dim=96, depth=2, heads=3, pretrain_grid=4, ffn=ffn, drop=drop, **kw)


def test_train_natively_keeps_the_module():
    """Same object, keys and classes; undone without a trace; a copy serves its own parameters.  The default stand-in is untouched by the
    gated form: the keys and values it always had."""
    import copy
    from iffnerf_amd import hip_vit
    m = backbone("swiglu", 0.1)
    keys, kinds = list(m.state_dict()), [type(k) for k in m.modules()]
    assert "blocks.0.mlp.w12.weight" in keys and m.state_dict()["blocks.0.mlp.w12.weight"].shape == (512, 96)
    assert hip_vit.train_natively(m) is m and list(m.state_dict()) == keys and [type(k) for k in m.modules()] == kinds
    assert "forward" in m.norm.__dict__ and "forward" in m.blocks[1].mlp.__dict__ and "forward" not in m.blocks[1].attn.__dict__
    c = copy.deepcopy(m)
    assert c.norm.__dict__["forward"].module is c.norm
    with pytest.raises(RuntimeError, match="no CPU path"):
        m.norm(torch.zeros(2, 96))
    hip_vit.train_stock(m)
    assert not any("forward" in k.__dict__ for k in m.modules())
    m.norm(torch.zeros(2, 96))
    plain = backbone("mlp", 0.0)
    assert "blocks.0.mlp.fc1.weight" in plain.state_dict() and not any("add" in k for k in plain.state_dict())
    for bad in (dict(ffn="relu", drop=0.0), dict(ffn="mlp", drop=1.0)):
        with pytest.raises(RuntimeError, match="ffn must be"):
            backbone(**bad)


def test_train_natively_leaves_what_computes_something_else():
    """Subclasses and instances with a forward of their own, gated feed-forwards with another activation or more inside, projections that a
    hook watches or changes (weight norm): each keeps its own forward and its own result, on the CPU here."""
    from iffnerf_amd import hip_vit
    nn = torch.nn

    class ChannelNorm(nn.LayerNorm):
        def forward(self, x):
            return super().forward(x.movedim(1, -1)).movedim(-1, 1)

    class Scaled(nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    class Gated(nn.Module):
        def __init__(self, linear=nn.Linear, **more):
            super().__init__()
            self.w12, self.w3 = linear(8, 12), nn.Linear(6, 8)
            for name, value in more.items():
                setattr(self, name, value)

        def forward(self, x):
            g, u = self.w12(x).chunk(2, dim=-1)
            return self.w3(getattr(self, "act", nn.functional.silu)(g) * u)

    patched = nn.LayerNorm(8)
    patched.forward = lambda x: x + 1
    others = [ChannelNorm(8), patched, Gated(Scaled), Gated(act=nn.GELU()), Gated(act=nn.functional.gelu), Gated(inner=nn.LayerNorm(6)),
              Gated(drop=nn.Dropout(0.1))]
    watched = Gated()
    seen = []
    watched.w12.register_forward_hook(lambda *a: seen.append(1))
    whole = nn.ModuleList([*others, watched]).eval()
    x = torch.randn(2, 8, generator=torch.Generator().manual_seed(1))
    want = [m(x) for m in whole if not hasattr(m, "inner")]
    hip_vit.train_natively(whole)
    assert not any("forward" in m.__dict__ for m in whole if m is not patched)
    assert all(torch.equal(m(x), w) for m, w in zip((m for m in whole if not hasattr(m, "inner")), want)) and len(seen) == 2
    for m in (Gated(), Gated(act=nn.SiLU()), Gated(drop=nn.Dropout(0.0))):
        hip_vit.train_natively(m)
        assert "forward" in m.__dict__
        with pytest.raises(RuntimeError, match="no CPU path"):
            m(x)
        m.w3.register_forward_pre_hook(lambda *a: None)              # (installed later: from then on the module's own forward)
        assert torch.equal(m(x), type(m).forward(m, x))
    hip_vit.train_stock(patched)
    assert torch.equal(patched(x), x + 1)


@gpu
@pytest.mark.parametrize("ffn", ["mlp", "swiglu"])
def test_a_backbone_trains_on_them(dev, ffn, monkeypatch):
    """Gradients of every parameter against the same backbone in 64 bits, dropout off; with dropout on: the same seed gives the same step,
    another seed another one, evaluation none.  Normwise 2^-15 relative: fp32 throughout, O(30) roundings of tensors and stock products
    over up to 256 terms on the way, each well under 2^-21 of its norm."""
    from iffnerf_amd import hip_vit
    m = backbone(ffn, 0.0).to(dev)
    img = normal((2, 3, 56, 56), 300)
    want = backbone(ffn, 0.0).to(dev)
    want.load_state_dict(m.state_dict())                                    # (the stand-in's biases are torch's own default)
    want.double()
    monkeypatch.setattr(hip_vit, "interpolate_pos_embed", lambda pos, *a, **k: pos[0])      # (the grid is the table's, and fp64 stays fp64)

    def loss(net, x):
        out = net.forward_features(x)["x_norm_patchtokens"]
        return (out * torch.linspace(-1, 1, out.numel(), device=dev, dtype=out.dtype).view_as(out)).sum()

    hip_vit.train_natively(m).train()
    names = [n for n, p in m.named_parameters() if n not in ("mask_token",)]
    got = torch.autograd.grad(loss(m, img), [dict(m.named_parameters())[n] for n in names])
    ref = torch.autograd.grad(loss(want, img.double()), [dict(want.named_parameters())[n] for n in names])
    for n, a, b in zip(names, got, ref):
        assert float((a.double() - b).norm()) <= 2.0 ** -15 * float(b.norm()) + 1e-9, n
    d = hip_vit.train_natively(backbone(ffn, 0.2).to(dev)).train()
    d.load_state_dict(m.state_dict())

    def step(seed):
        torch.manual_seed(seed)
        return torch.autograd.grad(loss(d, img), [d.blocks[0].norm1.weight])[0]

    a, b, c = step(1), step(1), step(2)
    assert torch.equal(a, b) and not torch.equal(a, c)
    with torch.no_grad():
        assert torch.equal(d.eval().forward_features(img)["x_prenorm"], m.eval().forward_features(img)["x_prenorm"])


@gpu
def test_a_backbone_step_under_autocast_and_checkpointing(dev):
    from torch.utils.checkpoint import checkpoint
    from iffnerf_amd import hip_vit
    m = hip_vit.train_natively(backbone("swiglu", 0.2).to(dev)).train()
    x = normal((2, 17, 96), 301).requires_grad_(True)
    torch.manual_seed(5)
    plain = torch.autograd.grad(m.blocks[0](x).square().sum(), (x, m.blocks[0].mlp.w12.weight))
    torch.manual_seed(5)
    again = torch.autograd.grad(checkpoint(m.blocks[0], x, use_reentrant=False).square().sum(), (x, m.blocks[0].mlp.w12.weight))
    assert all(torch.equal(a, b) for a, b in zip(plain, again))             # the recomputation drops what the forward pass dropped
    torch.manual_seed(5)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m.blocks[0](x)
    assert y.dtype == torch.float32
    g = torch.autograd.grad(y.square().sum(), (x, m.blocks[0].mlp.w12.weight))
    for a, b in zip(g, plain):                                              # bf16 products: a dozen roundings of 2^-8
        assert a.dtype == torch.float32 and float((a - b).norm() / b.norm()) <= 12 * 2.0 ** -8


# ------------------------------------------------------------------------------------------------------------ refusals
def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 4), torch.zeros(4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        hip_block.layer_norm(x, w, w)
    with pytest.raises(RuntimeError, match="no CPU path"):
        hip_block.gated_mlp(x, torch.zeros(6, 4), None, torch.zeros(4, 3), None)
    with pytest.raises(RuntimeError, match="no CPU path"):
        hip_block.dropout(x, 0.5, 1)


def test_c_entries_refuse_bad_arguments_without_a_gpu():
    from iffnerf_amd import _lib
    L = _lib.lib()

    def refused(rc, text):
        assert rc != 0 and text in L.iff_last_error(), L.iff_last_error()

    refused(L.iff_layer_norm_forward(None, 3, 1, 1, 0, 4, 4, None, None, 0, 1e-6, None, None, None), b"type 3")
    refused(L.iff_layer_norm_forward(None, 1, 1, 1, 0, 4, 4, None, None, 2, 1e-6, None, None, None), b"parameters of type 2")
    refused(L.iff_layer_norm_forward(None, 0, 1, 1, 0, 4, 0, None, None, 0, 1e-6, None, None, None), b"bad width")
    refused(L.iff_layer_norm_forward(16, 0, 1, 1, 0, 4, 4, None, None, 0, 1e-6, 16, 20, None), b"8-byte aligned")
    refused(L.iff_layer_norm_forward(None, 0, 1, 1, 0, 4, (1 << 24) + 1, None, None, 0, 1e-6, None, None, None), b"bad width")
    refused(L.iff_layer_norm_forward(None, 0, 1 << 20, 1 << 20, 0, 4, 4, None, None, 0, 1e-6, None, None, None), b"bad row counts")
    refused(L.iff_layer_norm_forward(None, 0, -1, 2, 0, 4, 4, None, None, 0, 1e-6, None, None, None), b"bad row counts")
    refused(L.iff_layer_norm_forward(None, 0, 1, 1, 0, 4, 4, None, None, 0, -1.0, None, None, None), b"eps")
    refused(L.iff_layer_norm_forward(None, 0, 1, 1, 0, 4, 4, None, None, 0, float("nan"), None, None, None), b"eps")
    refused(L.iff_layer_norm_forward(None, 0, 1, 1, 0, 4, 4, None, None, 0, 1e-6, None, None, None), b"null")
    assert L.iff_layer_norm_forward(None, 0, 0, 5, 0, 4, 4, None, None, 0, 1e-6, None, None, None) == 0
    assert L.iff_layer_norm_backward_workspace(257, 384) > 0 and L.iff_layer_norm_backward_workspace(0, 384) == 0
    one = 16
    refused(L.iff_layer_norm_backward(one, 0, 1, 4, 0, 4, 4, None, 0, one, one, one, one, None, None, 0, None), b"workspace")
    refused(L.iff_layer_norm_backward(None, 0, 1, 4, 0, 4, 4, None, 0, None, None, one, None, None, None, 0, None), b"null")
    assert L.iff_layer_norm_backward(None, 0, 1, 4, 0, 4, 4, None, 0, None, None, None, None, None, None, 0, None) == 0
    G, B = L.iff_gated_mlp_forward, L.iff_gated_mlp_backward
    refused(G(None, 5, 1, 4, 4, 4, None, None, None, None, 0, None, None, 0, None, 0, None), b"type 5")
    refused(G(None, 0, -1, 4, 4, 4, None, None, None, None, 0, None, None, 0, None, 0, None), b"bad row count")
    refused(G(None, 0, 1, 4, 0, 4, None, None, None, None, 0, None, None, 0, None, 0, None), b"bad widths")
    refused(G(None, 0, 1, 4, (1 << 20) + 1, 4, None, None, None, None, 0, None, None, 0, None, 0, None), b"bad widths")
    refused(G(None, 0, 1, 4, 4, 4, None, None, None, None, 7, None, None, 0, None, 0, None), b"activation 7")
    refused(G(None, 0, 1, 4, 4, 4, None, None, None, None, 0, None, None, 0, None, 0, None), b"null")
    refused(G(one, 0, 1, 4, 4, 4, one, None, one, None, 0, one, one, 8, one, 1 << 20, None), b"kept 8")
    refused(G(one, 0, 1, 4, 4, 4, one, None, one, None, 0, one, None, 0, None, 0, None), b"workspace 0")
    refused(G(one, 0, 1, 4, 4, 4, one, None, one, None, 0, one, None, 0, 24, 1 << 20, None), b"aligned")
    assert G(None, 0, 0, 4, 4, 4, None, None, None, None, 0, None, None, 0, None, 0, None) == 0
    refused(B(one, 0, 8, 4, 4, 4, one, one, one, one, one, None, None, None, None, None, 0, None), b"workspace 0")
    refused(B(None, 0, 8, 4, 4, 4, None, None, None, None, one, None, None, None, None, None, 0, None), b"null")
    refused(B(one, 0, 8, 4, 4, 4, one, one, 24, one, one, None, None, None, None, one, 1 << 30, None), b"aligned")
    assert L.iff_gated_mlp_kept_bytes(1, 8, 4, 4, 4) > 0 and L.iff_gated_mlp_kept_bytes(9, 8, 4, 4, 4) == 0
    refused(L.iff_dropout(None, 9, 4, None, 0, 0, None, 0, None, None), b"type 9")
    refused(L.iff_dropout(None, 0, -4, None, 0, 0, None, 0, None, None), b"bad size")
    refused(L.iff_dropout(None, 0, 4, None, 65537, 0, None, 0, None, None), b"threshold")
    refused(L.iff_dropout(None, 0, 4, None, 0, 0, None, 0, None, None), b"null")
    assert L.iff_dropout(None, 0, 0, None, 0, 0, None, 0, None, None) == 0


@gpu
def test_refusals(dev):
    x, w = torch.zeros(2, 4, device=dev), torch.zeros(4, device=dev)
    L, G, Dr = hip_block.layer_norm, hip_block.gated_mlp, hip_block.dropout
    w12, w3 = torch.zeros(6, 4, device=dev), torch.zeros(5, 3, device=dev)
    for call, text in [
            (lambda: L(x.double()), "fp32, bf16 or fp16"), (lambda: L(torch.zeros(3, 0, device=dev)), "at least one value"),
            (lambda: L(torch.tensor(1.0, device=dev)), "at least one value"), (lambda: L(x, w[:3]), "shape"), (lambda: L(x, w.half()), "float16"),
            (lambda: L(x.bfloat16(), w.half()), "float16"), (lambda: L(x.bfloat16(), w, w.bfloat16()), "bfloat16"), (lambda: L(x, w, eps=-1.0), "eps"),
            (lambda: L(x, w.cpu()), "is on cpu"), (lambda: L(x, eps=float("nan")), "eps"),
            (lambda: G(x, w12, None, w3, None, activation="tanh"), "activation"), (lambda: G(x, w12[:5], None, w3, None), "shape"),
            (lambda: G(x, w12.half(), None, w3, None), "float16"), (lambda: G(x, w12, w, w3, None), "shape"), (lambda: G(x, w12, None, w3, w), "shape"),
            (lambda: G(x, w12, None, w3[0], None), "w3"), (lambda: G(x, w12, None, w3[:, :0], None), "empty width"),
            (lambda: G(x, w12.cpu(), None, w3, None), "is on cpu"),
            (lambda: Dr(x, -0.1, 0), "between 0 and 1"), (lambda: Dr(x, 1.5, 0), "between 0 and 1"), (lambda: Dr(x, float("nan"), 0), "between 0 and 1"),
            (lambda: Dr(x, 0.1, -1), "seed"), (lambda: Dr(x, 0.1, 2 ** 64), "seed"), (lambda: Dr(x, 0.1, 1.5), "seed"), (lambda: Dr(x, 0.1, 0, -2), "offset"),
            (lambda: Dr(x, 0.1, torch.tensor([1])), "seed tensor"), (lambda: Dr(x, 0.1, torch.tensor([1, 2], device=dev)), "seed tensor"),
            (lambda: Dr(x, 0.1, 0, residual=w), "shape"), (lambda: Dr(x, 0.1, 0, residual=x.half()), "float16")]:
        with pytest.raises(RuntimeError, match=text):
            call()
