"""The dense operators of the graph layers (linear, group norm, dropout) against plain implementations in
64 bits.  Every tolerance is an elementwise bound worked out from the arithmetic: ``u`` is half the spacing
of the value type (each rounding of a result is off by at most u relative to it), ``ua`` the same of the
accumulation type (float32 for the narrow types), a sum of n terms in it is off by at most 2 n ua times the
sum of their magnitudes (the factor 2 covers accumulators that truncate), and an activation passes an error
of its argument on with a factor of at most 1.13 (the largest slope, gelu's) and its slope with at most 0.8
(the largest curvature, gelu's)."""
import itertools
import math

import pytest
import torch

import numml_b200.functional as F
import numml_b200.nn as nn
import numml_b200.sparse as sp
from numml_b200 import numml_torch_cpp


@pytest.fixture(autouse=True, params=["compiled", "python"])
def shim(request, monkeypatch):
    """Every test runs through the compiled per-call path and through the Python one."""
    monkeypatch.setattr(numml_torch_cpp, "use_compiled_shim", request.param == "compiled")
    return request.param


TYPES = [torch.float32, torch.float64, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu
SLOPE, CURVE = 1.13, 0.8


def units(dtype):
    u = torch.finfo(dtype).eps / 2
    return u, torch.finfo(torch.float64 if dtype == torch.float64 else torch.float32).eps / 2


def tiny(dtype):
    """Half the spacing of the subnormals of the type: a rounding near zero is off by that much."""
    f = torch.finfo(dtype)
    return f.tiny * f.eps / 2


def normal(shape, seed, dtype, scale=1.0, shift=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * scale + shift).to(dtype)


def act64(z, act):
    """Value and slope in 64 bits."""
    if act == "relu":
        on = (z > 0).double()
        return z * on, on
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "tanh":
        return torch.tanh(z), 1 - torch.tanh(z) ** 2
    return z, torch.ones_like(z)


def check(got, ref, bound, what):
    got, ref, bound = got.detach().cpu().double(), ref.cpu(), bound.cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bad = (got - ref).abs() > bound
    worst = ((got - ref).abs() / bound.clamp(min=1e-300)).max().item() if got.numel() else 0.0
    assert not bad.any(), f"{what}: {int(bad.sum())} of {got.numel()} entries off, worst {worst:.2f} of the bound"


# ---------------------------------------------------------------------------------------------------------
# linear
# ---------------------------------------------------------------------------------------------------------
def linear_oracle(X, W, b, R, dY, act, dtype):
    """(values, elementwise bounds) of y, dX, dW, db from the definitions in 64 bits."""
    u, ua = units(dtype)
    least = tiny(dtype)
    x, w, g = X.double().flatten(0, -2), W.double(), dY.double().flatten(0, -2)
    m, k, n = x.shape[0], w.shape[0], w.shape[1]
    z = x @ w
    ez = 2 * (k + 2) * ua * (x.abs() @ w.abs())
    if b is not None:
        z = z + b.double()
        ez = ez + 2 * ua * (z.abs() + b.double().abs())
    a, slope = act64(z, act)
    y = a + R.double().flatten(0, -2) if R is not None else a
    ey = SLOPE * ez + 8 * ua * (z.abs() + a.abs()) + u * y.abs() + ua * y.abs() + least
    dz = g * slope
    # the slope is taken at z as the forward pass rounded it; dz is rounded once more where it feeds products
    if act in (None, "none"):
        edz = torch.zeros_like(dz)
    elif act == "relu":
        edz = torch.zeros_like(dz)          # exact: tests with relu keep z away from rounding
    else:
        edz = g.abs() * (CURVE * (ez + u * z.abs() + least) + 8 * ua * (1 + z.abs())) + u * dz.abs() + least
    edz = edz + 4 * ua * dz.abs()
    dx, dw, db = dz @ w.T, x.T @ dz, dz.sum(0)
    edx = edz @ w.abs().T + 2 * (n + 2) * ua * (dz.abs() @ w.abs().T) + u * dx.abs() + least
    edw = x.abs().T @ edz + 2 * (m + 2) * ua * (x.abs().T @ dz.abs()) + u * dw.abs() + least
    edb = edz.sum(0) + 2 * (m + 2) * ua * dz.abs().sum(0) + u * db.abs() + least
    shape = X.shape[:-1]
    return {"y": (y.view(*shape, n), ey.view(*shape, n)), "dX": (dx.view(X.shape), edx.view(X.shape)), "dW": (dw, edw), "db": (db, edb)}


def run_linear(m, k, n, dtype, act, bias, residual, seed=0, integers=False):
    if integers:        # z is exact in every type and away from zero: half-integers
        gen = torch.Generator().manual_seed(seed)
        X, W = (torch.randint(-2, 3, s, generator=gen).to(dtype) for s in ((m, k), (k, n)))
        b = torch.full((n,), 0.5, dtype=dtype)
    else:
        X, W = normal((m, k), seed, dtype), normal((k, n), seed + 1, dtype, max(k, 1) ** -0.5)
        b = normal((n,), seed + 2, dtype) if bias else None
    R = normal((m, n), seed + 3, dtype) if residual else None
    dY = normal((m, n), seed + 4, dtype)
    ref = linear_oracle(X, W, b, R, dY, act, dtype)
    leaves = [t.cuda().requires_grad_(True) if t is not None else None for t in (X, W, b, R)]
    y = F.linear(leaves[0], leaves[1], leaves[2], act, leaves[3])
    with torch.no_grad():
        quiet = F.linear(leaves[0], leaves[1], leaves[2], act, leaves[3])
    assert torch.equal(quiet, y), "with and without a gradient to follow"
    grads = dict(zip([q for q, t in zip(("dX", "dW", "db", "dR"), leaves) if t is not None],
                     torch.autograd.grad(y, [t for t in leaves if t is not None], dY.cuda())))
    check(y, *ref["y"], "y")
    for q, v in grads.items():
        if q == "dR":
            assert torch.equal(v.cpu(), dY)
        else:
            check(v, *ref[q], q)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 64, 40), (3, 129, 7), (17, 5, 300), (64, 64, 64), (127, 65, 129), (128, 128, 128),
                                   (130, 256, 16), (257, 33, 65), (1000, 16, 200), (2049, 96, 130), (5, 1024, 1024), (16, 700, 24),
                                   (33, 512, 513), (513, 64, 64), (700, 200, 36), (640, 33, 140), (1025, 520, 260), (900, 1, 1)])
def test_linear_sizes(m, k, n, dtype):
    run_linear(m, k, n, dtype, "gelu", True, True, seed=m + k + n)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("act", [None, "silu", "gelu", "tanh"])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_linear_parts(act, bias, residual, dtype):
    run_linear(200, 72, 56, dtype, act, bias, residual, seed=7)
    run_linear(2, 72, 56, dtype, act, bias, residual, seed=8)
    run_linear(600, 136, 72, dtype, act, bias, residual, seed=9)          # tiles of more than 512 rows, three chunks


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m", [2, 300, 700])
def test_linear_relu(m, dtype):
    run_linear(m, 24, 40, dtype, "relu", True, True, seed=3, integers=True)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_linear_many_rows(dtype):
    """A long sum for dW, cut into parts and joined; twice the same bits."""
    run_linear(20011, 40, 24, dtype, "silu", True, False, seed=5)
    X, W = normal((20011, 40), 1, dtype).cuda().requires_grad_(True), normal((40, 24), 2, dtype).cuda().requires_grad_(True)
    dY = normal((20011, 24), 3, dtype).cuda()
    runs = [torch.autograd.grad(F.linear(X, W, activation="silu"), (X, W), dY) for _ in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows", [150, 1200])
def test_linear_views(rows, dtype):
    """Row-strided, odd-offset, transposed and 3-D operands give what their contiguous copies give, bit for bit."""
    big = normal((rows, 201), 0, dtype).cuda()
    W = normal((101, 90), 1, dtype, 0.1).cuda()
    R = normal((rows, 100), 2, dtype).cuda()
    b = normal((90,), 3, dtype).cuda()
    for X, w, r in ((big[:, :101], W, R[:, 3:93]), (big[:, 97:198], W[:, :], R[:, :90]), (big[::2, 1:102], W, R[:rows // 2, 10:]),
                    (big[:, 5:55], normal((70, 50), 4, dtype, 0.1).cuda().T[:, :70], R[:, :70]),
                    (big[:, 0:1].expand(rows, 101), W, R[:, :90]), (big[:, 100:].view(rows, 101)[:, :101], W, None)):
        bias = b[:w.shape[1]]
        got = F.linear(X, w, bias, "silu", r)
        want = F.linear(X.contiguous(), w.contiguous(), bias.clone(), "silu", r.contiguous() if r is not None else None)
        assert torch.equal(got, want)
    X4 = normal((3, 5, 7, 33), 5, dtype).cuda()
    W4 = normal((33, 9), 6, dtype).cuda()
    assert torch.equal(F.linear(X4, W4).view(-1, 9), F.linear(X4.view(-1, 33), W4))
    xl, wl = big[:, :101].detach().requires_grad_(True), W.detach().requires_grad_(True)
    y = F.linear(xl, wl, activation="tanh")
    gx, gw = torch.autograd.grad(y.sum(), (xl, wl))                       # an expanded upstream gradient
    y2 = F.linear(xl, wl, activation="tanh")
    gx2, gw2 = torch.autograd.grad(y2, (xl, wl), torch.ones_like(y2))
    assert torch.equal(gx, gx2) and torch.equal(gw, gw2)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", [(0, 4, 5), (4, 0, 5), (4, 5, 0), (0, 0, 0)])
def test_linear_empty(m, k, n, dtype):
    X, W = torch.ones(m, k, dtype=dtype, device="cuda", requires_grad=True), torch.ones(k, n, dtype=dtype, device="cuda", requires_grad=True)
    b = torch.full((n,), 0.5, dtype=dtype, device="cuda", requires_grad=True)
    y = F.linear(X, W, b, "tanh")
    assert y.shape == (m, n)
    assert torch.allclose(y.double(), torch.tanh(torch.full_like(y, 0.5 + k, dtype=torch.float64)), atol=8 * units(dtype)[0])
    gx, gw, gb = torch.autograd.grad(y, (X, W, b), torch.ones_like(y))
    assert gx.shape == X.shape and gw.shape == W.shape and gb.shape == b.shape
    if m == 0:
        assert not gw.any() and not gb.any()
    if n == 0:
        assert not gx.any()


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m", [1, 5, 200, 600])
def test_linear_infinities_and_nan_stay_in_their_rows_and_columns(m, dtype):
    """An infinity times a positive weight is an infinity, a NaN a NaN, and other rows do not notice."""
    X = normal((m, 130), 1, dtype).cuda()
    W = normal((130, 70), 2, dtype).abs().cuda() + 0.25
    clean = F.linear(X, W)
    Xi = X.clone()
    Xi[m - 1, 77] = float("inf")
    y = F.linear(Xi, W)
    assert (y[m - 1] == float("inf")).all() and torch.equal(y[:m - 1], clean[:m - 1])
    Xi[m - 1, 77] = float("nan")
    y = F.linear(Xi, W)
    assert y[m - 1].isnan().all() and torch.equal(y[:m - 1], clean[:m - 1])
    Wi = W.clone()
    Wi[3, 11] = -float("inf")
    Xp = X.abs() + 0.25
    y, c = F.linear(Xp, Wi), F.linear(Xp, W)
    keep = torch.arange(70) != 11
    assert (y[:, 11] == -float("inf")).all() and torch.equal(y[:, keep], c[:, keep])


@gpu
@pytest.mark.parametrize("m", [100, 600])
@pytest.mark.parametrize("power", [-36, -38, 37])
def test_linear_float32_ends_of_the_range(power, m):
    """Values whose low-order pieces are subnormal in 16 bits, and values near the largest.  A piece below 2^-126 counts
    as zero, so of a value at most 2^-126 is lost per piece: two pieces of x times |w|, and two of w times |x|."""
    X = (normal((m, 40), 1, torch.float64) * 10.0 ** power).float()
    W = normal((40, 70), 2, torch.float32, 0.5)
    ref, mag = X.double() @ W.double(), X.double().abs() @ W.double().abs()
    keep = mag < 3e38
    y = F.linear(X.cuda(), W.cuda()).cpu().double()
    lost = 2.0 ** -125 * (W.double().abs().sum(0)[None, :] + X.double().abs().sum(1)[:, None] + 40)
    bound = 2 * 42 * units(torch.float32)[1] * mag + lost
    assert ((y - ref).abs() <= bound)[keep].all(), ((y - ref).abs() / bound)[keep].max()


@gpu
def test_linear_float32_keeps_small_and_large_values():
    """float32 inputs use their whole range: products of very large and very small factors, and values with all
    24 bits, whose sums with few terms are off by a few units in the last place only."""
    ua = units(torch.float32)[1]
    for m, k in ((150, 3), (150, 64), (600, 3), (600, 64), (600, 200)):
        X = normal((m, k), k, torch.float64).mul(10.0 ** torch.linspace(-30, 30, k, dtype=torch.float64)).float()
        W = normal((k, 90), k + 1, torch.float64).mul(10.0 ** torch.linspace(30, -30, k, dtype=torch.float64)[:, None] * 1e-3).float()
        y = F.linear(X.cuda(), W.cuda())
        ref, mag = X.double() @ W.double(), X.double().abs() @ W.double().abs()
        check(y, ref, 2 * (k + 2) * ua * mag, f"k {k}")


@gpu
@pytest.mark.parametrize("m", [3, 140])
def test_linear_gradient_against_differences(m):
    torch.manual_seed(0)
    X, W, b, R = (torch.randn(*s, dtype=torch.float64, device="cuda", requires_grad=True) for s in ((m, 6), (6, 4), (4,), (m, 4)))
    for act in (None, "silu", "gelu", "tanh"):
        assert torch.autograd.gradcheck(lambda *a: F.linear(a[0], a[1], a[2], act, a[3]), (X, W, b, R), fast_mode=True)


def test_linear_refusals():
    X, W = torch.ones(3, 4), torch.ones(4, 5)
    with pytest.raises(RuntimeError, match="CUDA"):
        F.linear(X, W)
    with pytest.raises(RuntimeError, match="unknown activation"):
        F.linear(X, W, activation="swish")
    with pytest.raises(RuntimeError, match="torch.Tensor"):
        F.linear([1.0], W)


@gpu
def test_linear_refusals_on_the_device():
    X, W = torch.ones(3, 4, device="cuda"), torch.ones(4, 5, device="cuda")
    for call, match in ((lambda: F.linear(X, W.double()), "floating type"), (lambda: F.linear(X.long(), W.long()), "support"),
                        (lambda: F.linear(X, W.T), "weights must be"), (lambda: F.linear(X[0], W), "at least 2"),
                        (lambda: F.linear(X, W, torch.ones(4, device="cuda")), "bias must be"),
                        (lambda: F.linear(X, W, torch.ones(5)), "CUDA"), (lambda: F.linear(X, W, residual=X), "residual must"),
                        (lambda: F.linear(X, W, residual=torch.ones(1, 5, device="cuda")), "residual must")):
        with pytest.raises(RuntimeError, match=match):
            call()
    x = X.requires_grad_(True)
    (g,) = torch.autograd.grad(F.linear(x, W, activation="tanh").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        g.sum().backward()


# ---------------------------------------------------------------------------------------------------------
# group norm
# ---------------------------------------------------------------------------------------------------------
def group_norm_oracle(X, groups, w, b, eps, act, bounds, dY, dtype):
    u, ua = units(dtype)
    least = tiny(dtype)
    C = X.shape[-1]
    x, g = X.double().reshape(-1, C), dY.double().reshape(-1, C)
    wd = w.double() if w is not None else torch.ones(C, dtype=torch.float64)
    bd = b.double() if b is not None else torch.zeros(C, dtype=torch.float64)
    out = {q: (torch.zeros_like(x), torch.full_like(x, least)) for q in ("y", "dX")}
    sums = {q: (torch.zeros(C, dtype=torch.float64), torch.full((C,), least, dtype=torch.float64)) for q in ("dw", "db")}
    for lo, hi in zip(bounds[:-1], bounds[1:]):
        if hi <= lo:
            continue
        rows = hi - lo
        v = x[lo:hi].view(rows, groups, C // groups)
        # from differences to one entry: the oracle's own sums must not carry the level, or for float64 they would be
        # off by as much as the kernel may be
        v = v - v[:1, :, :1]
        level = (x[lo:hi].view(rows, groups, C // groups)[:1, :, :1]).abs()
        mean, var = v.mean((0, 2), keepdim=True), v.var((0, 2), correction=0, keepdim=True)
        rstd = (var + eps) ** -0.5
        xh = (v - mean) * rstd
        # a thread adds at most `terms` differences from its first value, all within `spread`; partial results
        # are joined in 64 bits, or over at most 256 row lanes in 8 steps in the accumulation type.  The square
        # sum of a thread relative to its own mean loses at most 2 terms ua spread^2.
        spread = (v.amax((0, 2), keepdim=True) - v.amin((0, 2), keepdim=True))
        terms = min(rows, 64) + 16
        em = 2 * terms * ua * spread + ua * (level + mean.abs())
        ev = 4 * terms * ua * spread ** 2
        ers = 0.5 * ev / (var + eps) + 2 * ua                                   # relative
        exh = rstd * (em + ua * (v - mean).abs()) + xh.abs() * (ers + 2 * ua)
        W3, flat = wd.view(groups, -1), lambda t: t.reshape(rows, C)
        z = flat(xh * W3) + bd
        ez = flat(exh * W3.abs()) + 2 * ua * (z.abs() + bd.abs())
        a, slope = act64(z, act)
        out["y"][0][lo:hi] = a
        out["y"][1][lo:hi] += SLOPE * ez + 8 * ua * (z.abs() + a.abs()) + u * a.abs()
        dz = g[lo:hi] * slope
        edz = g[lo:hi].abs() * ((CURVE * ez if act not in (None, "none") else 0) + 8 * ua * (1 + z.abs())) + 2 * ua * dz.abs()
        fx, efx = flat(xh.expand_as(v)), flat(exh.expand_as(v))
        sums["db"][0].add_(dz.sum(0))
        sums["db"][1].add_(edz.sum(0) + 2 * terms * ua * dz.abs().sum(0))
        sums["dw"][0].add_((dz * fx).sum(0))
        sums["dw"][1].add_((edz * fx.abs() + dz.abs() * efx).sum(0) + 2 * terms * ua * (dz * fx).abs().sum(0))
        h, eh = (dz * wd).view(v.shape), (edz * wd.abs()).view(v.shape)
        c1, c2 = h.mean((0, 2), keepdim=True), (h * xh).mean((0, 2), keepdim=True)
        e1 = eh.mean((0, 2), keepdim=True) + 2 * terms * ua * h.abs().mean((0, 2), keepdim=True)
        e2 = (eh * xh.abs() + h.abs() * exh).mean((0, 2), keepdim=True) + 2 * terms * ua * (h * xh).abs().mean((0, 2), keepdim=True)
        dx = rstd * (h - c1 - xh * c2)
        mag = h.abs() + c1.abs() + (xh * c2).abs()
        edx = rstd * (eh + e1 + exh * c2.abs() + xh.abs() * e2 + mag * (ers + 6 * ua))
        out["dX"][0][lo:hi] = flat(dx)
        out["dX"][1][lo:hi] += flat(edx) + u * flat(dx).abs()
    for q in sums:
        sums[q] = (sums[q][0], sums[q][1] + (u + 4 * ua) * sums[q][0].abs())
    return {**{q: (r.view(X.shape), e.view(X.shape)) for q, (r, e) in out.items()}, **sums}


def run_group_norm(X, groups, dtype, act=None, affine=True, ptr=None, eps=1e-5, seed=0):
    C = X.shape[-1]
    rows = X.numel() // C
    w = normal((C,), seed + 1, dtype, 0.3, 1.0) if affine else None
    b = normal((C,), seed + 2, dtype, 0.3) if affine else None
    dY = normal(X.shape, seed + 3, dtype)
    if ptr is not None:
        bounds = list(ptr)
    else:
        segments = 1 if X.ndim == 2 else X.shape[0]
        bounds = [rows // segments * s for s in range(segments + 1)]
    ref = group_norm_oracle(X, groups, w, b, eps, act, bounds, dY, dtype)
    x = X.cuda().requires_grad_(True)
    wc, bc = (t.cuda().requires_grad_(True) if t is not None else None for t in (w, b))
    pc = torch.tensor(ptr, device="cuda") if ptr is not None else None
    y = F.group_norm(x, groups, wc, bc, eps, act, pc)
    grads = torch.autograd.grad(y, [t for t in (x, wc, bc) if t is not None], dY.cuda())
    check(y, *ref["y"], "y")
    for q, v in zip(("dX", "dw", "db"), grads):
        check(v, *ref[q], q)
    with torch.no_grad():
        assert torch.equal(F.group_norm(x, groups, wc, bc, eps, act, pc), y)
    assert all(torch.equal(p, q) for p, q in zip(grads, torch.autograd.grad(F.group_norm(x, groups, wc, bc, eps, act, pc),
                                                                            [t for t in (x, wc, bc) if t is not None], dY.cuda())))


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,C,groups", [(40, 1, 1), (33, 8, 1), (50, 24, 3), (1000, 64, 8), (300, 33, 3), (257, 130, 13),
                                           (129, 512, 32), (64, 2050, 2), (5000, 16, 16), (17, 36, 2), (3001, 4, 4)])
def test_group_norm_sizes(rows, C, groups, dtype):
    run_group_norm(normal((rows, C), rows, dtype, 1.5, 0.5), groups, dtype, "silu", seed=rows)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("act", [None, "gelu", "tanh"])
@pytest.mark.parametrize("affine", [True, False])
def test_group_norm_parts(act, affine, dtype):
    run_group_norm(normal((200, 48), 1, dtype), 6, dtype, act, affine, seed=2)
    run_group_norm(normal((5, 7, 9, 24), 1, dtype), 2, dtype, act, affine, seed=3)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_group_norm_batch(dtype):
    """Graphs of 0, 1, a few and many rows, pieces that end anywhere, rows before the first and behind the last graph."""
    sizes = [0, 40, 1, 0, 0, 63, 700, 64, 2, 33, 0, 5000, 31, 0]
    ptr = [3]
    for s in sizes:
        ptr.append(ptr[-1] + s)
    X = normal((ptr[-1] + 77, 32), 9, dtype, 1.0, -2.0)
    run_group_norm(X, 4, dtype, "silu", ptr=ptr, seed=5)
    run_group_norm(X[:, :30].contiguous(), 5, dtype, None, ptr=ptr, seed=6)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("C,groups", [(600, 2), (303, 1)])
def test_group_norm_batch_in_row_chunks(C, groups, dtype):
    """Groups too wide for the one-block-per-graph kernels: pieces of graphs in chunks of rows."""
    sizes = [0, 40, 1, 0, 0, 63, 700, 64, 2, 33, 0, 1500, 31, 0]
    ptr = [3]
    for s in sizes:
        ptr.append(ptr[-1] + s)
    X = normal((ptr[-1] + 77, C), 9, dtype, 1.0, -2.0)
    run_group_norm(X, groups, dtype, "silu", ptr=ptr, seed=5)
    run_group_norm(X[:1000], groups, dtype, "gelu", affine=False, seed=6)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_group_norm_long_graphs(dtype):
    """Graphs of tens of thousands of rows beside short ones."""
    ptr = [0, 70000, 70000, 70003, 140000, 140100, 150000]
    run_group_norm(normal((150010, 64), 9, dtype, 1.0, 3.0), 1, dtype, "tanh", ptr=ptr, seed=5)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_group_norm_many_small_graphs(dtype):
    gen = torch.Generator().manual_seed(3)
    ptr = [0] + torch.cumsum(torch.randint(0, 12, (700,), generator=gen), 0).tolist()
    run_group_norm(normal((ptr[-1] + 5, 64), 4, dtype), 2, dtype, "gelu", ptr=ptr, seed=1)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64], ids=str)
def test_group_norm_level_far_above_spread(dtype):
    """A level of a thousand spreads costs the bits of the inputs, not those of the statistics."""
    run_group_norm(normal((4000, 16), 2, dtype, 1.0, 1000.0), 4, dtype, "tanh")


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_group_norm_constant_and_single_entries(dtype):
    """No variance: xhat is 0, y is act(bias), and the gradient of x vanishes."""
    C = 8
    w, b = normal((C,), 1, dtype).cuda(), normal((C,), 2, dtype).cuda()
    for X in (torch.full((50, C), 3.25, dtype=dtype), normal((1, C), 4, dtype)):
        x = X.cuda().requires_grad_(True)
        y = F.group_norm(x, C, w, b, activation="tanh")
        assert torch.allclose(y.double(), torch.tanh(b.double()).expand_as(y), atol=4 * units(dtype)[0])
        dY = torch.ones_like(y)
        (gx,) = torch.autograd.grad(y, x, dY)
        # h = slope * w is one value per channel, so dX = rstd (h - mean h) with rstd = eps^(-1/2); mean h is a sum of 50
        # equal terms in any order, off by at most 50 ua |h|, divided and multiplied by rounded numbers (4 ua more)
        assert gx.abs().max().item() <= 1e-5 ** -0.5 * (50 + 4) * units(dtype)[1] * w.abs().max().item()


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_group_norm_nan_stays_in_its_graph_and_group(dtype):
    X = normal((90, 16), 1, dtype).cuda()
    ptr = torch.tensor([0, 30, 60, 90], device="cuda")
    clean = F.group_norm(X, 2, ptr=ptr)
    X[40, 3] = float("nan")
    y = F.group_norm(X, 2, ptr=ptr)
    assert y[30:60, :8].isnan().all()
    same = torch.ones(90, 16, dtype=torch.bool)
    same[30:60, :8] = False
    assert torch.equal(y[same], clean[same])


@gpu
def test_group_norm_broken_row_pointers_touch_nothing_else():
    """Row numbers out of order or out of range: values are unspecified, the rest of memory is not touched."""
    for C, ptr in itertools.product((16, 1600), ([5, 2, 40, 10], [-7, 20, 1 << 40, 30], [0, 100, 100, 100000], [60, 50, 40, 30],
                                                 [90, 90, 90, 90])):
        arena = torch.full((3, 60, C), 7.0, device="cuda")
        x = arena[1].requires_grad_(True)
        y = F.group_norm(x, 4, ptr=torch.tensor(ptr, device="cuda"))
        torch.autograd.grad(y.sum(), x)
        torch.cuda.synchronize()
        assert (arena == 7.0).all()


@gpu
def test_group_norm_views_and_empty():
    X = normal((40, 70), 1, torch.float32).cuda()
    assert torch.equal(F.group_norm(X[:, 3:67], 4), F.group_norm(X[:, 3:67].contiguous(), 4))
    assert torch.equal(F.group_norm(X.T, 4), F.group_norm(X.T.contiguous(), 4))
    odd = normal((1 + 40 * 64,), 2, torch.float32).cuda()[1:].view(40, 64)                  # not on a 16-byte boundary
    assert torch.equal(F.group_norm(odd, 4), F.group_norm(odd.clone(), 4))
    for shape, ptr in (((0, 8), None), ((0, 5, 8), None), ((4, 0, 8), None), ((0, 8), [0, 0, 0]), ((6, 8), [2])):
        x = torch.ones(shape, device="cuda", requires_grad=True)
        w = torch.ones(8, device="cuda", requires_grad=True)
        y = F.group_norm(x, 2, w, ptr=torch.tensor(ptr, device="cuda") if ptr else None)
        assert y.shape == shape and not y.any()
        gx, gw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert not gx.any() and not gw.any()


@gpu
def test_group_norm_gradient_against_differences():
    torch.manual_seed(0)
    X, w, b = (torch.randn(*s, dtype=torch.float64, device="cuda", requires_grad=True) for s in ((23, 6), (6,), (6,)))
    ptr = torch.tensor([1, 9, 9, 20], device="cuda")
    for act in (None, "silu", "gelu", "tanh"):
        assert torch.autograd.gradcheck(lambda *a: F.group_norm(a[0], 2, a[1], a[2], 1e-3, act, ptr), (X, w, b), fast_mode=True)


def test_group_norm_refusals():
    X = torch.ones(3, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        F.group_norm(X, 2)
    with pytest.raises(RuntimeError, match="unknown activation"):
        F.group_norm(X, 2, activation=3)
    with pytest.raises(RuntimeError, match="groups"):
        nn.GroupNorm(3, 4)


@gpu
def test_group_norm_refusals_on_the_device():
    X, w = torch.ones(3, 4, device="cuda"), torch.ones(4, device="cuda")
    p = torch.tensor([0, 3], device="cuda")
    for call, match in ((lambda: F.group_norm(X, 3), "groups"), (lambda: F.group_norm(X, 0), "groups"), (lambda: F.group_norm(X[0], 1), "2 dim"),
                        (lambda: F.group_norm(X, 2, w.double()), "floating type"), (lambda: F.group_norm(X, 2, w[:2]), "weight must"),
                        (lambda: F.group_norm(X, 2, w, w[:3]), "bias must"), (lambda: F.group_norm(X, 2, eps=-1), "eps"),
                        (lambda: F.group_norm(X, 2, eps=float("nan")), "eps"), (lambda: F.group_norm(X, 2, ptr=p.int()), "ptr must"),
                        (lambda: F.group_norm(X, 2, ptr=p[:0]), "ptr must"), (lambda: F.group_norm(X, 2, ptr=p.cpu()), "CUDA"),
                        (lambda: F.group_norm(X[None], 2, ptr=p), "with ptr"), (lambda: F.group_norm(X.int(), 2), "support")):
        with pytest.raises(RuntimeError, match=match):
            call()


# ---------------------------------------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------------------------------------
def philox(counter, key):
    """Philox4x32-10 on Python integers."""
    c, (k0, k1) = list(counter), key
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [p1 >> 32 ^ c[1] ^ k0, p1 & 0xFFFFFFFF, p0 >> 32 ^ c[3] ^ k1, p0 & 0xFFFFFFFF]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def uniform32(i, seed, offset):
    block, q = divmod(i, 8)
    half = []
    for stream in (0, 1):
        ctr = (block & 0xFFFFFFFF, block >> 32, offset & 0xFFFFFFFF, offset >> 32 | stream << 31)
        half.append(philox(ctr, (seed & 0xFFFFFFFF, seed >> 32))[q // 2] >> 16 * (q % 2) & 0xFFFF)
    return half[0] << 16 | half[1]


def test_philox_known_answers():
    """Published vectors of the generator (all-zero, all-one and pi-digit inputs)."""
    assert philox([0] * 4, (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox([0xFFFFFFFF] * 4, (0xFFFFFFFF, 0xFFFFFFFF)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], (0xA4093822, 0x299F31D0)) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2051])
@pytest.mark.parametrize("p,seed,offset", [(0.1, 0, 0), (0.5, 2 ** 64 - 1, 2 ** 63 - 1), (0.75, 12345678901234567, 1 << 33)])
def test_dropout_mask_and_values(n, p, seed, offset, dtype):
    u, ua = units(dtype)
    X, R, dY = (normal((n,), s, dtype) for s in (1, 2, 3))
    keep = torch.tensor([uniform32(i, seed, offset) >= round(p * 2 ** 32) for i in range(n)])
    x, r = X.cuda().requires_grad_(True), R.cuda().requires_grad_(True)
    y = F.dropout(x, p, seed, offset)
    ref = torch.where(keep, X.double() / (1 - p), torch.zeros(n, dtype=torch.float64))
    check(y, ref, (u + 3 * ua) * ref.abs() + tiny(dtype), "y")
    assert (y.cpu()[~keep] == 0).all()
    (gx,) = torch.autograd.grad(y, x, dY.cuda())
    ref = torch.where(keep, dY.double() / (1 - p), torch.zeros(n, dtype=torch.float64))
    check(gx, ref, (u + 3 * ua) * ref.abs() + tiny(dtype), "dx")
    y = F.dropout(x, p, seed, offset, residual=r)
    drop = torch.where(keep, X.double() / (1 - p), torch.zeros(n, dtype=torch.float64))
    ref = drop + R.double()
    check(y, ref, (u + ua) * ref.abs() + 3 * ua * (drop.abs() + ref.abs()) + tiny(dtype), "y with residual")
    gx2, gr = torch.autograd.grad(y, (x, r), dY.cuda())
    assert torch.equal(gx2, gx) and torch.equal(gr.cpu(), dY)


@gpu
def test_dropout_low_halves_decide_ties():
    """A threshold placed on the numbers themselves: element i is kept exactly from p = u[i] / 2^32 downwards."""
    seed, offset = 99, 5
    x = torch.ones(64, dtype=torch.float64, device="cuda")
    for i in (0, 13, 42, 63):
        u = uniform32(i, seed, offset)
        assert F.dropout(x, u / 2 ** 32, seed, offset)[i] != 0
        assert F.dropout(x, (u + 1) / 2 ** 32, seed, offset)[i] == 0


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_dropout_ends_of_the_range(dtype):
    X = normal((100, 3), 1, dtype).cuda()
    assert torch.equal(F.dropout(X, 0.0, 1), X)
    X[3, 1], X[4, 2] = float("inf"), float("nan")
    assert torch.equal(F.dropout(X, 1.0, 1), torch.zeros_like(X))
    y = F.dropout(X, 0.5, 1)
    assert ((y == 0) | (y == 2 * X) | y.isnan()).all() and not y[torch.isfinite(X)].isnan().any()
    assert F.dropout(X[:0], 0.5, 1).shape == (0, 3)


@gpu
def test_dropout_share_and_independence():
    """Share of kept elements and of agreements between neighbouring offsets, seeds and elements: each of n
    independent draws, so within 5 standard deviations of its mean (missed once in 1.7 million runs; the
    inputs are fixed)."""
    n, p = 1 << 20, 0.3
    one = torch.ones(n, device="cuda")
    masks = [F.dropout(one, p, s, o) != 0 for s, o in ((1, 0), (1, 1), (2, 0), (1 << 40, 0), (1, 1 << 40))]
    for m in masks:
        assert abs(m.double().mean().item() - (1 - p)) <= 5 * math.sqrt(p * (1 - p) / n)
    agree = p * p + (1 - p) * (1 - p)
    for a, b in [(masks[0], m) for m in masks[1:]] + [(masks[0][1:], masks[0][:-1]), (masks[0][8:], masks[0][:-8])]:
        # neighbouring pairs of one mask share elements: twice the variance of independent pairs covers them
        assert abs((a == b).double().mean().item() - agree) <= 5 * math.sqrt(2 * agree * (1 - agree) / n)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_dropout_views_and_device_state(dtype):
    X = normal((60, 41), 1, dtype).cuda()
    for v in (X.T, X[:, 3:20], X[::3], X.flatten()[1:]):
        assert torch.equal(F.dropout(v, 0.4, 11, 2), F.dropout(v.clone(memory_format=torch.contiguous_format), 0.4, 11, 2))
    state = torch.tensor([11, 2], device="cuda")
    assert torch.equal(F.dropout(X, 0.4, state), F.dropout(X, 0.4, 11, 2))
    x = X.requires_grad_(True)
    y = F.dropout(x, 0.4, state)
    state[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


@gpu
def test_dropout_of_a_sparse_matrix():
    A = sp.eye(50).to("cuda") * 2 - sp.eye(50, k=1).to("cuda")
    A.requires_grad = True
    B = F.dropout(A, 0.3, 4)
    assert B.shape == A.shape and torch.equal(B.indices, A.indices) and torch.equal(B.indptr, A.indptr)
    assert torch.equal(B.data, F.dropout(A.data, 0.3, 4))
    (B @ torch.ones(50, 2, device="cuda")).sum().backward()
    assert torch.equal(A.data.grad, F.dropout(torch.full_like(A.data, 2.0), 0.3, 4).detach())
    with pytest.raises(RuntimeError, match="residual"):
        F.dropout(A, 0.3, 4, residual=A.data)


def test_dropout_refusals():
    X = torch.ones(3, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        F.dropout(X, 0.5, 0)
    with pytest.raises(RuntimeError, match="probability"):
        nn.Dropout(1.5)


@gpu
def test_dropout_refusals_on_the_device():
    X = torch.ones(3, 4, device="cuda")
    s = torch.tensor([1, 2], device="cuda")
    for call, match in ((lambda: F.dropout(X, -0.1, 0), "probability"), (lambda: F.dropout(X, float("nan"), 0), "probability"),
                        (lambda: F.dropout(X, 0.5, -1), "seed"), (lambda: F.dropout(X, 0.5, 1 << 64), "seed"),
                        (lambda: F.dropout(X, 0.5, 0, 1 << 63), "offset"), (lambda: F.dropout(X, 0.5, s.int()), "int64"),
                        (lambda: F.dropout(X, 0.5, s[:1]), "int64"), (lambda: F.dropout(X, 0.5, s.cpu()), "CUDA"),
                        (lambda: F.dropout(X, 0.5, s, 3), "second word"), (lambda: F.dropout(X.int(), 0.5, 0), "support"),
                        (lambda: F.dropout(X, 0.5, 0, residual=X[0]), "residual")):
        with pytest.raises(RuntimeError, match=match):
            call()


# ---------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------
def _batch_graph(sizes, seed):
    """Rings of the given sizes as one block-diagonal matrix, and the row pointers of the blocks."""
    rows, cols, start, ptr = [], [], 0, [0]
    for s in sizes:
        for i in range(s):
            for j in sorted({(i - 1) % s, (i + 1) % s}):
                rows.append(start + i)
                cols.append(start + j)
        start += s
        ptr.append(start)
    vals = normal((len(rows),), seed, torch.float64, 0.2, 1.0)
    return vals, torch.tensor(rows), torch.tensor(cols), start, ptr


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64], ids=str)
def test_a_network_of_the_operators(dtype):
    """Edge dropout, convolution, group norm with an activation, feature dropout in front of a residual product, as
    a training step uses them, against the same network in 64 bits on the CPU with dense matrices."""
    vals, r, c, nodes, ptr = _batch_graph([3, 40, 7, 120, 5], 1)
    ptr_d = torch.tensor(ptr, device="cuda")
    X0, w1, b1, w2, b2, gw, gb, dY = (normal(s, 10 + q, dtype, 0.5) for q, s in enumerate(
        [(nodes, 12), (12, 16), (16,), (16, 16), (16,), (16,), (16,), (nodes, 16)]))

    A = sp.SparseCSRTensor((vals.to(dtype), (r, c)), shape=(nodes, nodes)).to("cuda")
    A.requires_grad = True
    conv = nn.GCNConv(12, 16, normalize=False, fused=True)
    norm = nn.GroupNorm(4, 16, activation="silu")
    drop = nn.Dropout(0.25, seed=7)
    lin = nn.Linear(16, 16, activation="gelu")
    for layer, params in ((conv, (w1, b1)), (norm, (gw, gb)), (lin, (w2, b2))):
        layer.to(device="cuda", dtype=dtype)
        with torch.no_grad():
            for p, v in zip(layer.parameters(), params):
                p.copy_(v)
    x = X0.cuda().requires_grad_(True)
    H = norm(A, conv(F.dropout(A, 0.2, 3), x), ptr_d)
    Y = lin(A, drop(A, H), residual=H)
    Y.backward(dY.cuda())

    def keep(n, p, seed, offset):
        return torch.tensor([uniform32(i, seed, offset) >= round(p * 2 ** 32) for i in range(n)]).double() / (1 - p)

    order = torch.argsort(r * nodes + c)
    v64 = vals.to(dtype).double()[order].requires_grad_(True)
    x64, *p64 = (t.double().requires_grad_(True) for t in (X0, w1, b1, w2, b2, gw, gb))
    Ad = torch.zeros(nodes, nodes, dtype=torch.float64).index_put((r[order], c[order]), v64 * keep(v64.numel(), 0.2, 3, 0))
    C = Ad @ (x64 @ p64[0]) + p64[1]
    parts = []
    for lo, hi in zip(ptr[:-1], ptr[1:]):
        g = C[lo:hi].view(hi - lo, 4, 4)
        g = (g - g.mean((0, 2), keepdim=True)) / (g.var((0, 2), correction=0, keepdim=True) + 1e-5).sqrt()
        parts.append(torch.nn.functional.silu(g.reshape(hi - lo, 16) * p64[4] + p64[5]))
    H64 = torch.cat(parts)
    D64 = H64 * keep(H64.numel(), 0.25, 7, 0).view(nodes, 16)
    Y64 = torch.nn.functional.gelu(D64 @ p64[2] + p64[3]) + H64
    Y64.backward(dY.double())
    # a chain of a dozen roundings of sums of up to 16 (rows: 1920) terms, conditioned by the norm: 1000 units norm-wise
    tol = 1000 * units(dtype)[1]
    pairs = [(Y, Y64), (x.grad, x64.grad), (A.data.grad, v64.grad)]
    pairs += list(zip((p.grad for p in (conv.weights, conv.bias, lin.weights, lin.bias, norm.weight, norm.bias)), (p.grad for p in p64)))
    for q, (got, ref) in enumerate(pairs):
        err = (torch.linalg.norm(got.detach().cpu().double() - ref.detach()) / torch.linalg.norm(ref.detach())).item()
        assert err <= tol, f"output {q}: {err:.2e} > {tol:.2e}"


@gpu
@pytest.mark.parametrize("normalize", [True, False])
def test_fused_layers_agree_with_the_plain_ones(normalize):
    """The same layer with its dense products by torch and by this package: both within float32 rounding of sums of
    at most 24 products, taken over at most 3 hops and 3 entries of a row."""
    vals, r, c, nodes, _ = _batch_graph([50, 30], 2)
    A = sp.SparseCSRTensor((vals.float().abs(), (r, c)), shape=(nodes, nodes)).to("cuda")
    X = normal((nodes, 8), 1, torch.float32).cuda()
    for make in (lambda f: nn.GCNConv(8, 6, normalize, fused=f), lambda f: nn.TAGConv(8, 6, 3, normalize, fused=f)):
        torch.manual_seed(0)
        plain = make(False).cuda()
        torch.manual_seed(0)
        fused = make(True).cuda()
        ref, got = plain(A, X), fused(A, X)
        assert torch.linalg.norm(ref - got) <= 200 * units(torch.float32)[1] * torch.linalg.norm(ref)
        ref.sum().backward()
        got.sum().backward()
        assert torch.allclose(plain.weights.grad, fused.weights.grad, rtol=1e-4, atol=1e-4)
        assert torch.equal(plain.bias.grad, fused.bias.grad) or torch.allclose(plain.bias.grad, fused.bias.grad, rtol=1e-5)


@gpu
def test_sequential_and_evaluation_mode():
    vals, r, c, nodes, _ = _batch_graph([20], 3)
    A = sp.SparseCSRTensor((vals.float(), (r, c)), shape=(nodes, nodes)).to("cuda")
    model = nn.Sequential(nn.Linear(5, 16, activation="relu"), nn.GCNConv(16, 16, normalize=False, fused=True),
                          nn.GroupNorm(2, 16, activation="silu"), nn.Dropout(0.5, seed=1), nn.Linear(16, 1)).cuda()
    X = normal((nodes, 5), 1, torch.float32).cuda()
    a, b = model(A, X), model(A, X)
    assert a.shape == (nodes,) and not torch.equal(a, b)                 # another mask at every call
    model.eval()
    assert torch.equal(model(A, X), model(A, X))
    model.train()
    model(A, X).square().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())


@gpu
def test_captured_and_replayed():
    """A captured training step replays to the eager step's bits; a capturable dropout takes new masks at each
    replay, a dropout with host counters refuses to be captured."""
    nodes, C = 300, 32
    X, dY = normal((nodes, C), 1, torch.float32).cuda(), normal((nodes, C), 2, torch.float32).cuda()
    W, b = normal((C, C), 3, torch.float32, 0.2).cuda(), normal((C,), 4, torch.float32).cuda()
    ptr = torch.tensor([0, 100, 100, 280], device="cuda")
    drop = nn.Dropout(0.5, seed=2 ** 63 + 5, capturable=True).cuda()

    def step():
        x, w = X.detach().requires_grad_(True), W.detach().requires_grad_(True)
        y = F.linear(drop(None, F.group_norm(x, 4, activation="silu", ptr=ptr)), w, b, "gelu", residual=x)
        return [y.detach(), *torch.autograd.grad(y, (x, w), dY)]

    eager = [[t.clone() for t in step()] for _ in range(3)]
    drop.state[1] = 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                       # two graphs, whose workspaces must not be one another's
        drop.state[1] = 0
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    drop.state[1] = 0
    for q in range(3):
        g, out = graphs[q % 2]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager[q])), q
    assert not torch.equal(eager[0][0], eager[1][0])
    plain = nn.Dropout(0.5, seed=3).cuda()
    refused = []
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        try:
            plain(None, X)
        except RuntimeError as e:
            refused.append(str(e))
        _ = X + 1
    assert refused and "capturable" in refused[0]


@gpu
def test_capture_beside_a_live_eager_graph(shim):
    """A captured backward pass into leaves that a live eager graph holds on another stream raises and leaves the capture
    intact (the compiled path alone can ask the engine what it is about to run)."""
    if shim == "python":
        return
    x = normal((700, 32), 1, torch.float32).cuda().requires_grad_(True)
    w = normal((32, 48), 2, torch.float32).cuda().requires_grad_(True)
    alive = F.linear(x, w, activation="gelu")
    torch.cuda.synchronize()
    for make in (lambda: F.linear(x, w), lambda: F.dropout(x, 0.5, 1), lambda: F.group_norm(x, 4)):
        for backward in (lambda y: y.backward(torch.ones_like(y)), lambda y: torch.autograd.grad(y, x, torch.ones_like(y))):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = make()
                with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
                    backward(y)
                y = y.detach() + 1
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, make().detach() + 1)
    assert x.grad is None and w.grad is None
    del alive, y
    x2 = x.detach().requires_grad_(True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):                                     # with no eager graph of the leaf the same capture works
        (dx,) = torch.autograd.grad(F.linear(x2, w.detach()), x2, torch.ones(700, 48, device="cuda"))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(dx, torch.autograd.grad(F.linear(x2, w.detach()), x2, torch.ones(700, 48, device="cuda"))[0])


@gpu
def test_on_another_stream():
    X = normal((500, 64), 1, torch.float32).cuda()
    W = normal((64, 48), 2, torch.float32).cuda()
    want = F.linear(F.dropout(F.group_norm(X, 4, activation="gelu"), 0.3, 1), W)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = F.linear(F.dropout(F.group_norm(X, 4, activation="gelu"), 0.3, 1), W)
    s.synchronize()
    assert torch.equal(got, want)


@gpu
def test_two_streams_at_once():
    """Calls of the same operators that overlap on two streams do not see one another."""
    data = [(normal((4000, 96), q, torch.float32).cuda(), normal((96, 120), q + 9, torch.float32).cuda()) for q in range(2)]
    dY = normal((4000, 120), 5, torch.float32).cuda()

    def step(X, W):
        x, w = X.detach().requires_grad_(True), W.detach().requires_grad_(True)
        y = F.group_norm(F.linear(F.dropout(x, 0.2, 4), w, activation="gelu"), 8)
        return [y.detach(), *torch.autograd.grad(y, (x, w), dY)]

    want = [step(*d) for d in data]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(5):
        for q in range(2):
            with torch.cuda.stream(streams[q]):
                got[q] = step(*data[q])
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(a, b) for a, b in zip(w, g))
