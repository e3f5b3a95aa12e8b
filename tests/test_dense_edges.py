"""The dense operators of the graph layers at their edges: values beyond the range of 16 bits, forward passes that are
recomputed or differentiated in other ways, waits that run out, infinities in long sums, very long sums, skewed batches.
Tolerances as in test_dense_ops.py: ``u`` and ``ua`` are half the spacing of the value and the accumulation type."""
import math

import pytest
import torch

import numml_b200.functional as F
from numml_b200 import numml_torch_cpp
from test_dense_ops import CURVE, act64, check, normal, tiny, units

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
