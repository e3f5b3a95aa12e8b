"""The dense operators of the graph layers at their edges: values beyond the range of 16 bits, forward passes that are
recomputed or differentiated in other ways, waits that run out, infinities in long sums, very long sums, skewed batches.
Tolerances as in test_dense_ops.py: ``u`` and ``ua`` are half the spacing of the value and the accumulation type."""
import math

import pytest
import torch

import numml_b200.functional as F
import numml_b200.nn as nn
from numml_b200 import numml_torch_cpp
from test_dense_ops import CURVE, TYPES, act64, check, normal, run_group_norm, run_linear, tiny, units

gpu = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["compiled", "python"])
def shim(request, monkeypatch):
    """Every test runs through the compiled per-call path and through the Python one."""
    monkeypatch.setattr(numml_torch_cpp, "use_compiled_shim", request.param == "compiled")
    return request.param


# ---------------------------------------------------------------------------------------------------------
# pre-activations that 16 bits cannot hold
# ---------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype,big", [(torch.float16, (100.0, 700.0, 0.0)), (torch.bfloat16, (255 / 128 * 2.0 ** 63, 255 / 128 * 2.0 ** 63, 1.0))],
                         ids=["float16", "bfloat16"])
@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "tanh"])
@pytest.mark.parametrize("m,n", [(4, 40), (4, 41), (700, 48), (700, 41)])
def test_linear_backward_beyond_the_range_of_16_bits(m, n, act, dtype, big):
    """z = -70000 and +70000 in float16, beyond the largest bfloat16 (and within float32) in bfloat16: the slopes there
    are those of the 32-bit value that the forward pass activated, 0 and 1, and nothing becomes a NaN."""
    u, ua = units(dtype)
    X, W, b, dY = normal((m, 3), 1, dtype), normal((3, n), 2, dtype, 0.5), normal((n,), 3, dtype), normal((m, n), 4, dtype)
    W[0] = 0
    X[:, 0] = 0
    X[1, 0], X[2, 0], W[0, 5], W[1:, 5] = -big[0], big[0], big[1], 0
    X[0, 1:] = 0.25                                              # row 0 keeps clear of relu's corner
    b[5] = 0
    if big[2]:                                                   # the last step beyond the largest bfloat16 through the second column
        W[1, 5], X[1, 1], X[2, 1] = 2.0 ** 60, -1.9375 * 2.0 ** 60, 1.9375 * 2.0 ** 60
        X[0, 1] = X[3:, 1] = 0
    x, w, g = X.double(), W.double(), dY.double()
    z = x @ w + b.double()
    assert (z[1, 5] < -torch.finfo(dtype).max) and (z[2, 5] > torch.finfo(dtype).max) and (z.abs() < 3.4028e38).all()
    if act == "relu":
        keep = z.abs() > 1e-2                                    # away from the corner; elsewhere no gradient arrives
        dY, g = torch.where(keep, dY, 0), torch.where(keep, g, 0)
    ez = 2 * 6 * ua * (x.abs() @ w.abs() + b.double().abs())
    a, slope = act64(z, act)
    far = z.abs() > 30                                           # the slope is constant there, to less than 1e-12
    dz = g * slope
    edz = (g.abs() * (CURVE * (ez + u * z.abs()) + 8 * ua * (1 + z.abs()))).masked_fill(far, 0.0) if act != "relu" else torch.zeros_like(dz)
    edz = edz + (u + 4 * ua) * dz.abs() + tiny(dtype) + 1e-12 * g.abs()
    leaves = [t.cuda().requires_grad_(True) for t in (X, W, b)]
    y = F.linear(*leaves, act)
    grads = torch.autograd.grad(y, leaves, dY.cuda())
    refs = [dz @ w.T, x.T @ dz, dz.sum(0)]
    bounds = [edz @ w.abs().T + 2 * (n + 2) * ua * (dz.abs() @ w.abs().T), x.abs().T @ edz + 2 * (m + 2) * ua * (x.abs().T @ dz.abs()),
              edz.sum(0) + 2 * (m + 2) * ua * dz.abs().sum(0)]
    for what, got, ref, bound in zip(("dX", "dW", "db"), grads, refs, bounds):
        check(got, ref, bound + u * ref.abs() + tiny(dtype), what)
    y = y.detach().cpu().double()
    if act == "tanh":
        assert y[1, 5] == -1 and y[2, 5] == 1
    else:
        assert y[1, 5] == 0 and y[2, 5] == math.inf


# ---------------------------------------------------------------------------------------------------------
# forward passes that are run again in order to be differentiated
# ---------------------------------------------------------------------------------------------------------
def _dropout_on_the_host(X, p, seed, offset=0, residual=None):
    """A stand-in for the kernel: another mask for another (seed, offset)."""
    if isinstance(seed, torch.Tensor):
        seed, offset = seed.tolist()
    gen = torch.Generator().manual_seed(seed * 1000 + offset)
    return X * (torch.rand(X.shape, generator=gen, dtype=X.dtype) >= p)


def _checkpointed_mask(drop, X, use_reentrant, named):
    """Masks of the output and of the gradient of x -> dropout(x) in a checkpointed region, for two regions in turn."""
    from torch.utils.checkpoint import checkpoint
    masks = []
    for _ in range(2):
        x = X.detach().requires_grad_(True)
        call = drop.next_call() if named else None
        y = checkpoint(lambda t: drop(None, t, call) * t.detach(), x, use_reentrant=use_reentrant)
        y.sum().backward()
        masks.append((y.detach() != 0, x.grad != 0))
    return masks


@pytest.mark.parametrize("use_reentrant", [False, True])
@pytest.mark.parametrize("capturable", [False, True])
def test_dropout_recomputed_on_the_host(use_reentrant, capturable, monkeypatch):
    monkeypatch.setattr(nn.F, "dropout", _dropout_on_the_host)
    drop = nn.Dropout(0.5, seed=11, capturable=capturable)
    X = torch.ones(40, 5)
    (y0, g0), (y1, g1) = _checkpointed_mask(drop, X, use_reentrant, True)
    assert torch.equal(y0, g0) and torch.equal(y1, g1) and not torch.equal(y0, y1)
    with pytest.raises(RuntimeError, match="next_call"):
        _checkpointed_mask(drop, X, use_reentrant, False)
    want = _dropout_on_the_host(X, 0.5, 11, 3) != 0            # the refused call has advanced the counter once, in its forward pass
    assert torch.equal(drop(None, X) != 0, want)
    (y0, g0), _ = _checkpointed_mask(nn.Dropout(0.0, seed=5, capturable=capturable), X, use_reentrant, False)
    assert y0.all() and g0.all()                               # p = 0: there is but one mask


@pytest.mark.parametrize("seed", [11, 2 ** 64 - 3, None])
@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("second", [False, True])
def test_dropout_resumed_from_a_state_dict(first, second, seed, monkeypatch, tmp_path):
    """A layer that is loaded goes on with the masks that the saved one would have taken next, whichever form either has."""
    offsets = []
    monkeypatch.setattr(nn.F, "dropout", lambda X, p, seed, offset=0, residual=None: offsets.append(
        [int(seed[0]) % 2 ** 64, int(seed[1])] if isinstance(seed, torch.Tensor) else [seed, offset]) or X)
    net = nn.Sequential(nn.Dropout(0.5, seed=seed, capturable=first), nn.SeqWrapper(torch.nn.Linear(2, 2)))
    X = torch.ones(3, 2)
    for _ in range(3):
        net.modlist[0](None, X)
    torch.save(net.state_dict(), tmp_path / "net.pt")
    other = nn.Sequential(nn.Dropout(0.5, seed=5, capturable=second), nn.SeqWrapper(torch.nn.Linear(2, 2)))
    place = other.modlist[0].state.data_ptr() if second else None
    other.load_state_dict(torch.load(tmp_path / "net.pt", weights_only=True))
    net.modlist[0](None, X), other.modlist[0](None, X), other.modlist[0](None, X)
    assert offsets[3] == offsets[4] == [net.modlist[0].seed, 3] and offsets[5] == [net.modlist[0].seed, 4]
    assert not second or other.modlist[0].state.data_ptr() == place
    old = {k: v for k, v in net.state_dict().items() if "_extra_state" not in k}
    other.load_state_dict(old)                                   # strict: saved before there was such a state
    other.modlist[0](None, X)
    assert offsets[-1] == [net.modlist[0].seed, 5]


def test_dropout_seed_out_of_range():
    for seed in (-1, 2 ** 64):
        with pytest.raises(RuntimeError, match="seed"):
            nn.Dropout(0.5, seed=seed)


@gpu
@pytest.mark.parametrize("use_reentrant", [False, True])
@pytest.mark.parametrize("capturable", [False, True])
def test_dropout_recomputed(use_reentrant, capturable):
    drop = nn.Dropout(0.5, seed=11, capturable=capturable).cuda()
    X = normal((300, 17), 1, torch.float32).cuda().abs() + 1
    (y0, g0), (y1, g1) = _checkpointed_mask(drop, X, use_reentrant, True)
    assert torch.equal(y0, g0) and torch.equal(y1, g1) and not torch.equal(y0, y1)
    assert torch.equal(y1, F.dropout(X, 0.5, 11, 1) != 0)
    with pytest.raises(RuntimeError, match="next_call"):
        _checkpointed_mask(drop, X, use_reentrant, False)


@gpu
@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode_tangents_are_refused(leaf):
    import torch.autograd.forward_ad as fw
    X, W, v, R = (normal(s, q, torch.float32).cuda() for q, s in enumerate(((20, 8), (8, 8), (8,), (20, 8))))
    calls = [(X, lambda t: F.linear(t, W)), (W, lambda t: F.linear(X, t)), (v, lambda t: F.linear(X, W, t)),
             (R, lambda t: F.linear(X, W, residual=t)), (X, lambda t: F.group_norm(t, 2)), (v, lambda t: F.group_norm(X, 2, t)),
             (v, lambda t: F.group_norm(X, 2, None, t)), (X, lambda t: F.dropout(t, 0.5, 1)), (R, lambda t: F.dropout(X, 0.5, 1, residual=t))]
    for operand, call in calls:
        operand = operand.clone().requires_grad_(leaf)
        with fw.dual_level():
            dual = fw.make_dual(operand, torch.ones_like(operand))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)
            with torch.inference_mode():                         # no derivative of any kind is formed there
                quiet = call(dual)
            assert torch.equal(quiet, call(operand))             # without a tangent all is as before


# ---------------------------------------------------------------------------------------------------------
# waits that run out
# ---------------------------------------------------------------------------------------------------------
@gpu
def test_a_wait_that_ran_out_is_seen_by_check_status(shim):
    """The kernels of the compiled path report into the word that check_status reads (written here by the host)."""
    X, W = normal((700, 40), 1, torch.float32).cuda(), normal((40, 24), 2, torch.float32).cuda()
    want = F.linear(X, W)
    numml_torch_cpp.check_status()
    if shim == "compiled":
        word = numml_torch_cpp.compiled_shim().known_status_word(X.device.index)
        assert word.data_ptr() == numml_torch_cpp._status_word(X.device).data_ptr()
    else:
        word = numml_torch_cpp._status_word(X.device)
    word.fill_(5)
    with pytest.raises(RuntimeError, match="status 5"):
        numml_torch_cpp.check_status()
    numml_torch_cpp.check_status()                               # read and cleared
    assert torch.equal(F.linear(X, W), want)
    numml_torch_cpp.check_status()


# ---------------------------------------------------------------------------------------------------------
# infinities and NaN in the sums of the backward pass
# ---------------------------------------------------------------------------------------------------------
def _products(X, W, dY):
    x, w = X.detach().requires_grad_(True), W.detach().requires_grad_(True)
    b = torch.zeros(W.shape[1], dtype=X.dtype, device=X.device, requires_grad=True)
    return torch.autograd.grad(F.linear(x, w, b), (x, w, b), dY)


def _same_but(got, clean, row=None, column=None, value=None, what=""):
    """`got` is `clean`, bit for bit, but for one row or column, which is `value`."""
    want = clean.clone()
    if row is not None:
        want[row] = value
    else:
        want[:, column] = value
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(1.5), want.nan_to_num(1.5)), what


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("m,k,n", [(700, 40, 24), (20011, 40, 130), (3000, 1700, 1601)])
def test_linear_infinities_in_the_backward_pass(m, k, n, dtype):
    """One infinity in x: a row of dW infinite with the signs of dY's row (an infinity times a number), all else as it was;
    one in dY: a row of dX and a column of dW; NaN and infinities of both signs: NaN.  The last size has more tiles of dW
    than the GPU has multiprocessors, so its sum over the rows is one piece, behind which other tiles wait."""
    X, W, dY = normal((m, k), 1, dtype).cuda(), normal((k, n), 2, dtype, 0.1).cuda(), normal((m, n), 3, dtype).cuda()
    X[X == 0], W[W == 0], dY[dY == 0] = 1, 1, 1
    clean = _products(X, W, dY)
    inf = float("inf")
    i, r, c = m - 2, k // 2, n - 1
    Xi = X.clone()
    Xi[i, r] = inf
    dx, dw, db = _products(Xi, W, dY)
    assert torch.equal(dx, clean[0]) and torch.equal(db, clean[2])
    _same_but(dw, clean[1], row=r, value=dY[i].sign() * inf, what="infinity in x")
    Xi[3, r] = -inf                                              # NaN where the two meet with opposite signs
    meet = dY[i].sign() * inf - dY[3].sign() * inf
    _same_but(_products(Xi, W, dY)[1], clean[1], row=r, value=meet, what="two infinities in x")
    Xi = X.clone()
    Xi[i, r] = float("nan")
    _same_but(_products(Xi, W, dY)[1], clean[1], row=r, value=float("nan"), what="NaN in x")
    Gi = dY.clone()
    Gi[i, c] = -inf
    dx, dw, db = _products(X, W, Gi)
    _same_but(dx, clean[0], row=i, value=-W[:, c].sign() * inf, what="infinity in dY, dX")
    _same_but(dw, clean[1], column=c, value=-X[i].sign() * inf, what="infinity in dY, dW")
    assert db[c] == -inf and torch.equal(db[:c], clean[2][:c])
    Xi = X.clone()
    Xi[:, r] = inf                                               # every term of a row of dW
    both = (dY.sign().amax(0) > 0) & (dY.sign().amin(0) < 0)
    _same_but(_products(Xi, W, dY)[1], clean[1], row=r, value=torch.where(both, float("nan"), dY[0].sign() * inf).to(dtype), what="a column of infinities")
    numml_torch_cpp.check_status()


# ---------------------------------------------------------------------------------------------------------
# very long sums of 16-bit values
# ---------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("which", ["y", "dX", "dW"])
def test_linear_long_sums_do_not_drift(which, dtype):
    """Sums of 2^18 terms of one sign.  The tensor cores cut off where they add, always in one direction, up to 2^-23 of the
    sum so far with every eight terms; the 4096 terms that share an accumulator come to 512 / 2 * 2^-23 = 2^-15 (the sum
    grows evenly), and what is added to nearest after that has no direction.  The mean relative error over N results whose
    logarithms are spread evenly is then below 2^-15 + 6 sigma / sqrt(N), sigma = half a step."""
    u, _ = units(dtype)
    long, (rows, cols) = 1 << 18, ((1152, 1152) if which == "dW" else (640, 128))
    gen = torch.Generator(device="cuda").manual_seed(3)

    def operand(lines):                                          # [lines, long]: positive, each line at a level of its own
        level = 2.0 ** torch.rand(lines, 1, generator=gen, device="cuda")
        return ((torch.rand(lines, long, generator=gen, device="cuda") + 0.5) * level * 2.0 ** -5).to(dtype)

    a, b = operand(rows), operand(cols)
    if which == "y":
        got = F.linear(a, b.T.contiguous())
    elif which == "dX":                                          # dX = dY W^T, sum over the output channels
        x, w = torch.zeros(rows, cols, dtype=dtype, device="cuda", requires_grad=True), b
        (got,) = torch.autograd.grad(F.linear(x, w), x, a)
    else:                                                        # dW = X^T dY, sum over the rows
        x, w = a.T.contiguous(), torch.zeros(rows, cols, dtype=dtype, device="cuda", requires_grad=True)
        (got,) = torch.autograd.grad(F.linear(x, w), w, b.T.contiguous())
    ref = a.double() @ b.double().T
    error = (got.double() - ref) / ref
    assert error.abs().max() <= u * 1.01 + 2.0 ** -15
    assert error.mean().abs() <= 2.0 ** -15 + 6 * u / math.sqrt(got.numel()), error.mean().item()
    numml_torch_cpp.check_status()


# ---------------------------------------------------------------------------------------------------------
# long graphs among short ones
# ---------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("C,groups,act", [(64, 8, "gelu"), (33, 3, None), (36, 2, "silu")])
def test_group_norm_long_graphs_among_short_ones(C, groups, act, dtype):
    """Long graphs at the start, in the middle, side by side and at the end of a batch of short and empty ones, with rows
    before the first and behind the last."""
    gen = torch.Generator().manual_seed(1)
    short = lambda n: torch.randint(0, 9, (n,), generator=gen).tolist()
    sizes = [9001] + short(150) + [0, 12007, 4999, 8000, 0] + short(200) + [7003, 1, 0]
    ptr = [5]
    for s in sizes:
        ptr.append(ptr[-1] + s)
    run_group_norm(normal((ptr[-1] + 70, C), 9, dtype, 1.0, 2.0), groups, dtype, act, ptr=ptr, seed=5)
    run_group_norm(normal((ptr[-1], C), 8, dtype, 1.0, 2.0), groups, dtype, act, affine=False, ptr=ptr, seed=6)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_group_norm_long_graphs_of_many_channels(dtype):
    """Rows that several blocks side by side cover; a NaN stays in its long graph and group."""
    ptr = [0, 3, 2700, 2700, 2710, 4801, 4850]
    X = normal((4860, 2048), 3, dtype)
    run_group_norm(X, 32, dtype, "silu", ptr=ptr, seed=5)
    clean = F.group_norm(X.cuda(), 32, ptr=torch.tensor(ptr, device="cuda"))
    X[1000, 100] = float("nan")
    got = F.group_norm(X.cuda(), 32, ptr=torch.tensor(ptr, device="cuda"))
    assert got[3:2700, 64:128].isnan().all()
    got[3:2700, 64:128] = clean[3:2700, 64:128]
    assert torch.equal(got, clean)


@gpu
def test_group_norm_long_graphs_among_very_many():
    """More graphs than rows, most of them empty, and as many long ones as there can be."""
    ptr = [0]
    for q in range(13):
        ptr += [ptr[-1]] * 3000 + [ptr[-1] + 4200 + q] + [ptr[-1] + 4200 + q + 1]
    run_group_norm(normal((ptr[-1], 32), 9, torch.float32, 1.0, 2.0), 4, torch.float32, "gelu", ptr=ptr, seed=5)


@gpu
def test_group_norm_broken_row_pointers_of_a_long_batch_touch_nothing_else():
    rows, C = 50000, 64
    ptr = torch.randint(-60000, 120000, (300,), generator=torch.Generator().manual_seed(2)).cuda()
    store = torch.full((rows + 200, C), 7.0, device="cuda")
    x = store[100:rows + 100].normal_().requires_grad_(True)
    y = F.group_norm(x, 8, ptr=ptr)
    torch.autograd.grad(y, x, torch.ones_like(y))
    torch.cuda.synchronize()
    assert (store[:100] == 7).all() and (store[rows + 100:] == 7).all()
    good = torch.tensor([0, 30000, 30010, rows], device="cuda")
    assert torch.isfinite(F.group_norm(x, 8, ptr=good)).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_group_norm_one_long_graph_is_not_left_to_one_block(dtype):
    """One graph of most of a batch's rows beside 511 of one row: a training step of it takes no more than a few times
    that of equal graphs (a block that had the long one to itself took 20 to 30 times as long)."""
    rows, graphs = 61440, 512
    X, dY = normal((rows, 128), 1, dtype).cuda().requires_grad_(True), normal((rows, 128), 2, dtype).cuda()
    equal = torch.arange(graphs + 1, device="cuda") * (rows // graphs)
    skewed = torch.arange(graphs + 1, device="cuda")
    skewed[-1] = rows

    def time(ptr):
        best = math.inf
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            a.record()
            for _ in range(5):
                torch.autograd.grad(F.group_norm(X, 16, activation="gelu", ptr=ptr), X, dY)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    assert time(skewed) < 8 * time(equal)


@gpu
def test_group_norm_long_batch_captured_and_on_two_streams():
    """The pass over long graphs under capture (two graphs, replayed in turn with other row pointers) and on two streams."""
    rows, C = 30000, 64
    X, dY = normal((rows, C), 1, torch.float32).cuda(), normal((rows, C), 2, torch.float32).cuda()
    w = normal((C,), 3, torch.float32, 0.3, 1.0).cuda()
    ptrs = [torch.tensor(p, device="cuda") for p in ([0, 20000, 20001, 29000, 30000], [0, 10, 20, 30, 30000], [0, 7500, 15000, 22500, 30000])]
    ptrs.append(torch.arange(5, device="cuda") * 600)                     # none that is long

    def step(ptr):
        x, wl = X.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = F.group_norm(x, 8, wl, activation="silu", ptr=ptr)
        return [y.detach(), *torch.autograd.grad(y, (x, wl), dY)]

    want = [[t.clone() for t in step(p)] for p in ptrs]
    graphs = []
    for _ in range(2):
        ptr = ptrs[0].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(ptr)
        graphs.append((g, ptr, out))
    for q in (1, 0, 3, 2, 1):
        g, ptr, out = graphs[q % 2]
        ptr.copy_(ptrs[q])
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[q])), q
    streams, got = [torch.cuda.Stream() for _ in range(2)], {}
    torch.cuda.synchronize()
    for q in (0, 1, 2, 3, 0, 1):
        with torch.cuda.stream(streams[q % 2]):
            got[q] = step(ptrs[q])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for q in got for a, b in zip(got[q], want[q]))


# ---------------------------------------------------------------------------------------------------------
# the slope of tanh
# ---------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("m", [40, 3000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64], ids=str)
def test_slope_of_tanh_to_the_last_places(dtype, m):
    """The slope relative to itself, for z of both signs: 4 e / (1 + e)^2, e = exp(-2 |z|).  The exponential is good to
    2 + 1.173 * 2 |z| units in the last place (the short one of 32 bits; the other to one), twice ua each; two
    divisions and four products come to 16 ua more."""
    _, ua = units(dtype)
    z = torch.linspace(-40, 40, m, dtype=torch.float64).to(dtype)
    one = torch.ones(1, 1, dtype=dtype)
    x = z[:, None].cuda().requires_grad_(True)
    (got,) = torch.autograd.grad(F.linear(x, one.cuda(), None, "tanh"), x, torch.ones(m, 1, dtype=dtype, device="cuda"))
    e = torch.exp(-2 * z.double().abs())
    ref = 4 * e / (1 + e) ** 2
    bound = ref * ua * (16 + 2 * (2 + 2.35 * z.double().abs())) + (ref * 2.0 ** -50 if dtype == torch.float64 else 0)
    check(got[:, 0], ref, bound + 2.0 ** -125, "slope")
    y = F.group_norm(torch.stack([z, -z], 1).cuda().requires_grad_(True), 2, activation="tanh")     # the same slope there
    assert torch.isfinite(torch.autograd.grad(y.sum(), y.grad_fn.next_functions[0][0].variable)[0]).all()


# ---------------------------------------------------------------------------------------------------------
# captures
# ---------------------------------------------------------------------------------------------------------
@gpu
def test_capture_after_a_warm_up_whose_results_live():
    """The usual way to capture a training step: warm-up on a side stream, whose last results are still there when the
    step is captured."""
    net = nn.Sequential(nn.Linear(32, 48, activation="gelu"), nn.GroupNorm(4, 48, activation="silu"),
                        nn.Dropout(0.5, seed=3, capturable=True), nn.Linear(48, 24)).cuda()
    X = normal((700, 32), 1, torch.float32).cuda().requires_grad_(True)
    leaves = [X, *net.parameters()]

    def step():
        for t in leaves:
            t.grad = None
        net.modlist[2].state[1].zero_()
        y = net(None, X).square().sum()
        y.backward()
        return y

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            alive = step()
    torch.cuda.current_stream().wait_stream(side)
    want = [t.grad.clone() for t in leaves]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, alive) and all(torch.equal(t.grad, w) for t, w in zip(leaves, want))


# ---------------------------------------------------------------------------------------------------------
# lazily negated operands
# ---------------------------------------------------------------------------------------------------------
@gpu
def test_lazily_negated_operands():
    """Operands whose memory holds the negated values (torch keeps the imaginary part of a conjugate so)."""
    lazy = lambda t: torch._neg_view(-t)
    X, W, v, R, dY = (normal(s, q, torch.float32).cuda() for q, s in enumerate(((300, 16), (16, 16), (16,), (300, 16), (300, 16))))
    column = torch.view_as_complex(torch.stack((R[:, :1], X[:, :1]), -1)).conj().imag                 # one channel: any stride will do
    assert lazy(X).is_neg() and column.is_neg()

    def run(X, W, v, R, dY, column):
        leaves = [t.detach().requires_grad_(True) for t in (X, W, v, R)]
        x, w, b, r = leaves
        out = []
        for y in (F.linear(x, w, b, "silu", r), F.group_norm(x, 4, b, v, activation="gelu"), F.dropout(x, 0.3, 5, residual=r)):
            out += [y, *torch.autograd.grad(y, leaves, dY, allow_unused=True)]
        with torch.no_grad():
            out += [F.linear(column, w[:1]), F.linear(x[:3], w), F.group_norm(column, 1), F.dropout(column, 0.3, 5)]
        return [t for t in out if t is not None]

    plain = run(X, W, v, R, dY, -X[:, :1])
    for got, want in zip(run(*(lazy(t) for t in (X, W, v, R, dY)), column), plain):
        assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("m,k,n", [(640, 4097, 72), (1300, 5000, 136), (700, 9001, 41)])
def test_linear_long_sums_with_everything(m, k, n, dtype):
    """Sums in several runs, with bias, activation, residual and the backward pass, tiled and gathered; dX's over few."""
    run_linear(m, k, n, dtype, "gelu", True, True, seed=m)
    run_linear(k, 48, n, dtype, "silu", True, False, seed=n)


@gpu
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "tanh"])
@pytest.mark.parametrize("m,k,n", [(600, 130, 72), (900, 70, 41), (3, 130, 72)])
def test_linear_infinities_through_the_epilogue(m, k, n, act):
    """Float sums that are not finite get bias, activation and residual like the others, with and without z kept, and
    the values around them do not notice."""
    X, W = normal((m, k), 1, torch.float32), normal((k, n), 2, torch.float32, 0.2)
    b, R, dY = normal((n,), 3, torch.float32), normal((m, n), 4, torch.float32), normal((m, n), 5, torch.float32)
    clean = F.linear(X.cuda(), W.cuda(), b.cuda(), act, R.cuda()).cpu()
    X[m - 2, 7], X[0, 3], X[m - 1, 5] = float("inf"), float("nan"), -float("inf")
    W[9, n - 1] = float("inf")                                   # a column, of either sign
    z = X.double() @ W.double() + b.double()
    odd = ~torch.isfinite(z)
    a, _ = act64(z, act)
    if act == "relu":                                            # there the formula is -infinity * 0
        a = torch.relu(z)
    want = (a + R.double()).float()
    with torch.no_grad():
        quiet = F.linear(X.cuda(), W.cuda(), b.cuda(), act, R.cuda()).cpu()
    x, w, r = X.cuda().requires_grad_(True), W.cuda().requires_grad_(True), R.cuda().requires_grad_(True)
    y = F.linear(x, w, b.cuda(), act, r)
    grads = torch.autograd.grad(y, (x, w, r), dY.cuda())
    assert torch.equal(quiet.nan_to_num(1.5), y.detach().cpu().nan_to_num(1.5)) and torch.equal(quiet.isnan(), y.detach().cpu().isnan())
    assert torch.equal(quiet[~odd], clean[~odd])                 # what is finite is what it was without them
    got = quiet[odd]
    assert torch.equal(got.isnan(), want[odd].isnan())
    assert torch.equal(got.isinf(), want[odd].isinf()) and torch.equal(got[got.isinf()], want[odd][got.isinf()])
    fine = torch.isfinite(got)
    assert ((got[fine] - want[odd][fine]).abs() <= 4 * 2.0 ** -24 * (1 + want[odd][fine].abs())).all()
    assert torch.equal(grads[2].cpu(), dY)
    rows = torch.ones(m, dtype=torch.bool)
    rows[[m - 2, 0, m - 1]] = False
    if act in ("relu", "tanh"):                                  # slopes of 0 and 1 there: dX of the other rows stays finite
        assert torch.isfinite(grads[0].cpu()[rows][:, :9]).all()
    numml_torch_cpp.check_status()
