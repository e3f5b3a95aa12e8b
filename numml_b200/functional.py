"""Dense operators of the graph layers, differentiable, on this package's CUDA kernels.

    linear(X, weights, bias, activation, residual)     act(X W + b) + R in one kernel
    group_norm(X, groups, weight, bias, activation, ptr)   group norm over the nodes of each graph, then act
    dropout(X, p, seed, offset, residual)              dropout whose mask is recomputed, never stored

They complete what a layer of :mod:`numml_b200.nn` does around its sparse product.  Node features are
channels-last, ``[nodes, channels]``; a batch of graphs is a concatenation of their rows with a pointer
array.  Values are float32, float64, bfloat16 or float16 (one type per call); sums, statistics and
activations are held in 32 bits (64 for float64) and results are rounded at the end.  One more rounding is
made on purpose: :func:`linear` in a 16-bit type keeps its pre-activation, and takes the gradient behind the
activation's slope to its products, in that type, as a layer of 16-bit operators does (32-bit ones would be twice
the bytes, and twice the products).  All tensors are on
one CUDA device (there is no CPU path); calls run on that device's current stream.  Results do not
depend on the run: no operator adds with atomics.  Gradients of gradients and forward-mode tangents are refused.

Calls go through the compiled extension (``csrc_ext/dense_ops.cpp``) when it has been built; the Python
functions below do the same work otherwise, with identical results (see
``numml_torch_cpp.use_compiled_shim``).
"""
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _cabi, numml_torch_cpp
from .numml_torch_cpp import _on, _ptr, _require_cuda, _status_word, _stream

_DTYPES = {torch.float32: _cabi.F32, torch.float64: _cabi.F64, torch.bfloat16: _cabi.BF16, torch.float16: _cabi.F16}
_ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu": 3, "tanh": 4}


def _dtype_code(t):
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise RuntimeError(f"the dense operators support float32, float64, bfloat16 and float16, got {t.dtype}")
    return code


def _activation_code(activation):
    code = _ACTIVATIONS.get(activation)
    if code is None:
        raise RuntimeError(f"unknown activation {activation!r}: expected one of {sorted(a for a in _ACTIVATIONS if a)}")
    return code


def _check_operands(X, **others):
    """All given operands on one CUDA device and of X's floating type."""
    given = [t for t in others.values() if t is not None]
    dev = _require_cuda(X, *given)
    code = _dtype_code(X)
    for name, t in others.items():
        if t is not None and t.dtype != X.dtype:
            raise RuntimeError(f"operands must share one floating type, got {X.dtype} and {t.dtype} ({name})")
    return dev, code


def _rows(t, cols):
    """A [rows, cols] matrix over t's memory (a copy only where rows are not evenly strided runs) and its row stride.
    Lazily negated values (the imaginary part of a conjugate) are negated first, here and below."""
    t = t.resolve_neg()
    if t.ndim == 2 and (cols <= 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= cols):
        return t, (t.stride(0) if t.shape[0] > 1 else cols)
    return t.contiguous().view(-1, cols) if cols > 0 else t.reshape(math.prod(t.shape[:-1]), 0), cols


def _aligned(t):
    """Contiguous and on a 16-byte boundary, as the vector loads need it."""
    t = t.resolve_neg().contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _vector(t):
    """Contiguous, or None."""
    return t.resolve_neg().contiguous() if t is not None else None


def _shim(*operands):
    """The compiled per-call path, or None when it has not been built; operands of it are tensors."""
    for t in operands:
        if t is not None and not isinstance(t, torch.Tensor):
            raise RuntimeError(f"expected a torch.Tensor, got {type(t)}")
    return numml_torch_cpp.compiled_shim()


def _status_pointer(dev):
    """The device's status word; none while a graph is being captured that would otherwise come to own it."""
    key = dev.index if dev.index is not None else torch.cuda.current_device()
    if key not in numml_torch_cpp._status_words and torch.cuda.is_current_stream_capturing():
        return None
    return _ptr(_status_word(dev))


def _refuse_tangents(*tensors):
    """Tangents of forward-mode differentiation: no operator passes them on, and a result without one reads as zero."""
    if not torch._C._is_fwd_grad_enabled() or forward_ad._current_level < 0:
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("the dense operators have no forward-mode derivative; an operand carries a tangent")


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# -------------------------------------------------------------------------------------------------
# linear
# -------------------------------------------------------------------------------------------------
def _linear_forward(X, weights, bias, residual, act, keep_z):
    """(y, z): z is None unless a backward pass will need it."""
    K, N = weights.shape
    x, ldx = _rows(X, K)
    w, ldw = _rows(weights, N)
    r, ldr = _rows(residual, N) if residual is not None else (None, 0)
    b = _vector(bias)
    M = x.shape[0]
    with _on(X.device):
        y = torch.empty(X.shape[:-1] + (N,), dtype=X.dtype, device=X.device)
        z = torch.empty((M, N), dtype=X.dtype, device=X.device) if keep_z and act else None
        _cabi.call("nb200_linear_forward", M, K, N, _ptr(x), ldx, _ptr(w), ldw, _ptr(b), _ptr(r), ldr, act, _ptr(z), _ptr(y),
                   _status_pointer(X.device), _DTYPES[X.dtype], _stream())
    return y, z


def _linear_backward(dY, X, weights, z, act, want_x, want_w, want_b):
    K, N = weights.shape
    x, ldx = _rows(X, K)
    w, ldw = _rows(weights, N)
    g, ldg = _rows(dY, N)
    M = x.shape[0]
    code = _DTYPES[X.dtype]
    with _on(X.device):
        dx = torch.empty(X.shape, dtype=X.dtype, device=X.device) if want_x else None
        dw = torch.empty((K, N), dtype=X.dtype, device=X.device) if want_w else None
        db = torch.empty((N,), dtype=X.dtype, device=X.device) if want_b else None
        work = torch.empty(_cabi.lib().nb200_linear_backward_workspace_bytes(M, K, N, act, code), dtype=torch.uint8, device=X.device)
        _cabi.call("nb200_linear_backward", M, K, N, _ptr(g), ldg, _ptr(x), ldx, _ptr(w), ldw, _ptr(z), act, _ptr(dx), _ptr(dw),
                   _ptr(db), _ptr(work), work.numel(), _status_pointer(X.device), code, _stream())
    return dx, dw, db


class linear_fn(torch.autograd.Function):
    """Autograd node of :func:`linear`."""

    @staticmethod
    def forward(ctx, X, weights, bias, residual, act):
        y, z = _linear_forward(X, weights, bias, residual, act, True)
        ctx.save_for_backward(X, weights, z)
        ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dY):
        X, weights, z = ctx.saved_tensors
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if want_x or want_w or want_b:
            dx, dw, db = _linear_backward(dY, X, weights, z, ctx.act, want_x, want_w, want_b)
        return dx, dw, db, dY if want_r else None, None


def linear(X, weights, bias=None, activation=None, residual=None):
    """``act(X @ weights + bias) + residual`` in one pass.

    X: [..., K]; weights: [K, N]; bias: [N] or None; residual: [..., N] or None (no broadcasting);
    activation: None / 'none', 'relu', 'silu', 'gelu' (the erf form; in 32 bits with an erf that is good to 1.5e-7
    absolute, so relative to itself gelu(-3) is off by up to 5e-5) or 'tanh'.  X, weights and residual
    may be 2-D views with any row stride.  float32 products are as exact as float32 multiply-adds, for factors
    from 2^-102 (2e-31) upwards; of smaller ones up to 2^-125 may be lost."""
    act = _activation_code(activation)
    ext = _shim(X, weights, bias, residual)
    if ext is not None:
        return ext.linear(X, weights, bias, residual, act)
    _check_operands(X, weights=weights, bias=bias, residual=residual)
    if X.ndim < 2:
        raise RuntimeError(f"expected node features [..., channels] with at least 2 dimensions, got {X.ndim}")
    if weights.ndim != 2 or weights.shape[0] != X.shape[-1]:
        raise RuntimeError(f"weights must be [{X.shape[-1]}, out_channels], got {tuple(weights.shape)}")
    if bias is not None and tuple(bias.shape) != (weights.shape[1],):
        raise RuntimeError(f"bias must be [{weights.shape[1]}], got {tuple(bias.shape)}")
    out_shape = tuple(X.shape[:-1]) + (weights.shape[1],)
    if residual is not None and tuple(residual.shape) != out_shape:
        raise RuntimeError(f"residual must have the output's shape {out_shape}, got {tuple(residual.shape)}")
    _refuse_tangents(X, weights, bias, residual)
    if _wants_grad(X, weights, bias, residual):
        return linear_fn.apply(X, weights, bias, residual, act)
    return _linear_forward(X, weights, bias, residual, act, False)[0]


# -------------------------------------------------------------------------------------------------
# group norm
# -------------------------------------------------------------------------------------------------
def _segments(X, ptr):
    """(rows, number of segments) of the features X."""
    rows = X.numel() // X.shape[-1]
    if ptr is not None:
        return rows, ptr.numel() - 1
    return rows, (1 if X.ndim == 2 else X.shape[0])


def _group_norm_forward(X, groups, weight, bias, eps, act, ptr):
    x = _aligned(X)
    w = _vector(weight)
    b = _vector(bias)
    p = ptr.contiguous() if ptr is not None else None
    C = X.shape[-1]
    rows, segments = _segments(X, ptr)
    code = _DTYPES[X.dtype]
    wide = torch.float64 if X.dtype == torch.float64 else torch.float32
    with _on(X.device):
        y = torch.empty(X.shape, dtype=X.dtype, device=X.device)
        stats = torch.empty((2, segments, groups), dtype=wide, device=X.device)
        work = torch.empty(_cabi.lib().nb200_group_norm_workspace_bytes(rows, C, groups, segments, code), dtype=torch.uint8, device=X.device)
        _cabi.call("nb200_group_norm_forward", rows, C, groups, segments, _ptr(p), _ptr(x), _ptr(w), _ptr(b), eps, act, _ptr(y),
                   _ptr(stats[0]), _ptr(stats[1]), _ptr(work), work.numel(), code, _stream())
    return y, stats


def _group_norm_backward(dY, X, groups, weight, bias, act, ptr, stats, want_x, want_w, want_b):
    x, g = _aligned(X), _aligned(dY)
    w = _vector(weight)
    b = _vector(bias)
    p = ptr.contiguous() if ptr is not None else None
    C = X.shape[-1]
    rows, segments = _segments(X, ptr)
    code = _DTYPES[X.dtype]
    with _on(X.device):
        dx = torch.empty(X.shape, dtype=X.dtype, device=X.device) if want_x else None
        dw = torch.empty((C,), dtype=X.dtype, device=X.device) if want_w else None
        db = torch.empty((C,), dtype=X.dtype, device=X.device) if want_b else None
        work = torch.empty(_cabi.lib().nb200_group_norm_workspace_bytes(rows, C, groups, segments, code), dtype=torch.uint8, device=X.device)
        _cabi.call("nb200_group_norm_backward", rows, C, groups, segments, _ptr(p), _ptr(g), _ptr(x), _ptr(w), _ptr(b), _ptr(stats[0]),
                   _ptr(stats[1]), act, _ptr(dx), _ptr(dw), _ptr(db), _ptr(work), work.numel(), code, _stream())
    return dx, dw, db


class group_norm_fn(torch.autograd.Function):
    """Autograd node of :func:`group_norm`."""

    @staticmethod
    def forward(ctx, X, weight, bias, ptr, groups, eps, act):
        y, stats = _group_norm_forward(X, groups, weight, bias, eps, act, ptr)
        ctx.save_for_backward(X, weight, bias, ptr, stats)
        ctx.groups, ctx.act = groups, act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dY):
        X, weight, bias, ptr, stats = ctx.saved_tensors
        dx, dw, db = _group_norm_backward(dY, X, ctx.groups, weight, bias, ctx.act, ptr, stats, *ctx.needs_input_grad[:3])
        return dx, dw, db, None, None, None, None


def group_norm(X, groups, weight=None, bias=None, eps=1e-5, activation=None, ptr=None):
    """``act((X - mean) / sqrt(var + eps) * weight + bias)`` with mean and biased variance over the nodes
    of one graph and the channels of one group (``channels / groups`` neighbouring ones).

    X [nodes, channels] is one graph; X [graphs, ..., channels] normalises every ``X[g]`` by itself; with
    ``ptr`` (int64 on the device, ``graphs + 1`` ascending row numbers) X [nodes, channels] is a batch in
    which graph g has rows ``ptr[g]:ptr[g+1]``; graphs may be empty, and rows outside every graph give zeros
    and receive no gradient.  weight and bias: [channels] or None."""
    act = _activation_code(activation)
    ext = _shim(X, weight, bias, ptr)
    if ext is not None:
        return ext.group_norm(X, int(groups), weight, bias, float(eps), act, ptr)
    _check_operands(X, weight=weight, bias=bias)
    if X.ndim < 2 or X.shape[-1] < 1:
        raise RuntimeError(f"expected features [..., channels] with at least 2 dimensions and one channel, got {tuple(X.shape)}")
    C = X.shape[-1]
    groups = int(groups)
    if groups < 1 or C % groups != 0:
        raise RuntimeError(f"{C} channels cannot be split into {groups} groups")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (C,):
            raise RuntimeError(f"{name} must be [{C}], got {tuple(t.shape)}")
    eps = float(eps)
    if not eps >= 0.0:
        raise RuntimeError(f"eps must not be negative, got {eps}")
    if ptr is not None:
        _require_cuda(X, ptr)
        if ptr.dtype != torch.int64 or ptr.ndim != 1 or ptr.numel() < 1:
            raise RuntimeError(f"ptr must be a 1-D int64 tensor of graphs + 1 row numbers, got {ptr.dtype} {tuple(ptr.shape)}")
        if X.ndim != 2:
            raise RuntimeError(f"with ptr the features must be [nodes, channels], got {tuple(X.shape)}")
    _refuse_tangents(X, weight, bias)
    if _wants_grad(X, weight, bias):
        return group_norm_fn.apply(X, weight, bias, ptr, groups, eps, act)
    return _group_norm_forward(X, groups, weight, bias, eps, act, ptr)[0]


# -------------------------------------------------------------------------------------------------
# dropout
# -------------------------------------------------------------------------------------------------
def _dropout_run(X, p, seed, offset, state, residual):
    x = _aligned(X)
    r = _aligned(residual) if residual is not None else None
    with _on(X.device):
        y = torch.empty(X.shape, dtype=X.dtype, device=X.device)
        _cabi.call("nb200_dropout", x.numel(), _ptr(x), _ptr(r), _ptr(y), p, seed, offset, _ptr(state), _DTYPES[X.dtype], _stream())
    return y


class dropout_fn(torch.autograd.Function):
    """Autograd node of :func:`dropout`: keeps the seed, not the mask."""

    @staticmethod
    def forward(ctx, X, residual, p, seed, offset, state):
        ctx.save_for_backward(state)
        ctx.args = (p, seed, offset)
        return _dropout_run(X, p, seed, offset, state, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dY):
        (state,) = ctx.saved_tensors
        dx = _dropout_run(dY, *ctx.args, state, None) if ctx.needs_input_grad[0] else None
        return dx, dY if ctx.needs_input_grad[1] else None, None, None, None, None


def dropout(X, p, seed, offset=0, residual=None):
    """Zero every element of X with probability p, scale the others by 1 / (1 - p), add the residual.

    Element i (in row-major order) is kept where a 32-bit number that depends on (seed, offset, i) alone is
    at least ``round(p * 2**32)``: Philox4x32-10, see ``nb200_dropout`` in the C header for the counter's layout.
    The backward pass recomputes it.  seed: 0 <= seed < 2**64 and offset: 0 <= offset < 2**63, or a device tensor
    of two int64 words [seed, offset] (offset argument left at 0), which a captured CUDA graph re-reads at every
    replay and which must not change between a forward pass and its backward pass.  Take another offset for every
    use.  X may be a ``SparseCSRTensor``: its stored values are dropped (edge dropout), the pattern stays."""
    if hasattr(X, "indptr") and hasattr(X, "indices"):
        if residual is not None:
            raise RuntimeError("the dropout of a sparse tensor takes no residual")
        from .sparse import SparseCSRTensor
        return SparseCSRTensor((dropout(X.data, p, seed, offset), X.indices, X.indptr), X.shape, clone=False)
    p, state = float(p), None
    if isinstance(seed, torch.Tensor):
        if offset != 0:
            raise RuntimeError("with a seed tensor the offset is its second word; leave the offset argument at 0")
        state, seed = seed, 0
    seed, offset = int(seed), int(offset)
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 63):
        raise RuntimeError(f"seed must be in [0, 2**64) and offset in [0, 2**63), got {seed} and {offset}")
    ext = _shim(X, residual, state)
    if ext is not None:
        return ext.dropout(X, p, seed, offset, state, residual)
    _check_operands(X, residual=residual)
    if not 0.0 <= p <= 1.0:
        raise RuntimeError(f"dropout probability must be in [0, 1], got {p}")
    if residual is not None and residual.shape != X.shape:
        raise RuntimeError(f"residual must have the shape {tuple(X.shape)}, got {tuple(residual.shape)}")
    if state is not None:
        _require_cuda(X, state)
        if state.dtype != torch.int64 or tuple(state.shape) != (2,) or not state.is_contiguous():
            raise RuntimeError(f"a seed tensor must hold two int64 words [seed, offset], got {state.dtype} {tuple(state.shape)}")
    _refuse_tangents(X, residual)
    if _wants_grad(X, residual):
        return dropout_fn.apply(X, residual, p, seed, offset, state)
    return _dropout_run(X, p, seed, offset, state, residual)
