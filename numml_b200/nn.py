"""Graph-convolution layers whose graph argument is a sparse matrix.

Mirror of the reference's ``numml/nn.py`` (layers ``:6-168``, containers and the parameter-vector
helpers ``:171-234``): same class names, constructor arguments, parameter names (``weights``,
``bias``) and arithmetic, so that a ``state_dict`` moves between the two.  The sparse work of a layer
is the SpMM ``A @ X`` (``SparseCSRTensor.__matmul__`` -> ``spdmm``) and, when the layer normalises,
the row sums of A (``SparseCSRTensor.row_sum`` -> ``sprowsum``); both run on this package's CUDA
kernels and are differentiable with respect to the stored values of A as well as X.

Beside them, for the dense half of a network and with the same calling convention ``layer(A, X)``:
``Linear`` (product, bias, activation and residual in one kernel), ``GroupNorm`` (with an activation, per
graph of a batch) and ``Dropout`` (mask recomputed from a counter), on :mod:`numml_b200.functional`.
"""
import torch

from . import functional as F


def _as_feature_matrix(X):
    """Node features as [nodes, channels]; a vector is one channel."""
    return X.unsqueeze(1) if X.ndim == 1 else X


def _inv_sqrt_degree(row_sums):
    """Diagonal of D~^(-1/2) for A~ = A + I, as a column that broadcasts over the channels."""
    return ((row_sums + 1.) ** -0.5)[:, None]


class _GraphConv(torch.nn.Module):
    """What the two layers share: channel counts, the normalisation switch, the bias, and how the dense
    products X W run: by ``torch.matmul``, or with ``fused=True`` by ``functional.linear`` (which needs CUDA
    tensors, adds a bias or the sum so far in its epilogue and takes float32 products to the tensor cores)."""

    def __init__(self, in_channels, out_channels, normalize, weight_shape, fused=False):
        super().__init__()
        self.fused = fused
        # registration order (weights, then bias) fixes the layout of model_to_vector
        self.weights = torch.nn.Parameter(torch.randn(*weight_shape))
        self.bias = torch.nn.Parameter(torch.randn(out_channels))
        self.in_channels = in_channels
        self.out_channels = out_channels
        self.normalize = normalize


class GCNConv(_GraphConv):
    """Kipf & Welling graph convolution on a matrix:
    ``Y = D~^(-1/2) (A + I) D~^(-1/2) X W + b`` (``normalize=True``) or ``Y = A X W + b``.
    Reference ``numml/nn.py:6-101``."""

    def __init__(self, in_channels, out_channels, normalize=True, fused=False):
        super().__init__(in_channels, out_channels, normalize, (in_channels, out_channels), fused)

    def _convolve(self, matmul, row_sums, X, fused=False):
        X = _as_feature_matrix(X)
        Z = F.linear(X, self.weights) if fused else X @ self.weights
        if self.normalize:
            d = _inv_sqrt_degree(row_sums())
            Z = d * Z
            out = d * (matmul(Z) + Z)            # (A + I) Z without forming A + I
        else:
            out = matmul(Z)
        return out + self.bias

    def forward(self, A, X):
        """A: ``SparseCSRTensor`` or ``LinearOperator``; X: [nodes, in_channels] or [nodes]."""
        return self._convolve(lambda Z: A @ Z, A.row_sum, X, self.fused)

    def forward_dense(self, A, X):
        """The same layer evaluated on ``A.to_dense()`` (a check, and the only form that runs on CPU)."""
        Ad = A.to_dense()
        return self._convolve(lambda Z: Ad @ Z, lambda: Ad.sum(dim=1), X)


class TAGConv(_GraphConv):
    """Topology-adaptive graph convolution: ``Y = sum_{j=1..k} P^j(X) W_j + b`` where one hop is
    ``P(X) = A X`` or, normalised, ``P(X) = d * (A (d * X + X))`` with ``d = (rowsum(A) + 1)^(-1/2)``
    (the reference's update, ``numml/nn.py:104-168``, kept as it is written there)."""

    def __init__(self, in_channels, out_channels, k=2, normalize=True, fused=False):
        super().__init__(in_channels, out_channels, normalize, (k, in_channels, out_channels), fused)
        self.k = k

    def forward(self, A, X):
        Xc = _as_feature_matrix(X)
        d = _inv_sqrt_degree(A.row_sum()) if self.normalize else None
        H = None
        for j in range(self.k):
            Xc = d * (A @ (d * Xc + Xc)) if self.normalize else A @ Xc
            if self.fused:                             # bias with the first hop, each further hop on top of the sum
                H = F.linear(Xc, self.weights[j], bias=self.bias if H is None else None, residual=H)
                continue
            term = Xc @ self.weights[j]
            H = term if H is None else H + term
        if H is None:                                  # k = 0: only the bias
            H = torch.zeros(Xc.shape[0], self.out_channels, dtype=Xc.dtype, device=Xc.device)
        elif self.fused:
            return H
        return H + self.bias


class Linear(torch.nn.Module):
    """``act(X W + b) + residual`` on the node features (the graph argument is not used)."""

    def __init__(self, in_channels, out_channels, bias=True, activation=None):
        super().__init__()
        F._activation_code(activation)
        self.weights = torch.nn.Parameter(torch.randn(in_channels, out_channels) * in_channels ** -0.5 if in_channels else
                                          torch.zeros(in_channels, out_channels))
        self.bias = torch.nn.Parameter(torch.zeros(out_channels)) if bias else None
        self.in_channels, self.out_channels, self.activation = in_channels, out_channels, activation

    def forward(self, A, X, residual=None):
        """X: [nodes, in_channels] or [nodes]; residual: [nodes, out_channels] or None."""
        return F.linear(_as_feature_matrix(X), self.weights, self.bias, self.activation, residual)


class GroupNorm(torch.nn.Module):
    """Group norm over the nodes of each graph with an activation (the matrix argument is not used).
    Call with ``ptr`` for a batch of graphs, see :func:`numml_b200.functional.group_norm`."""

    def __init__(self, groups, channels, eps=1e-5, affine=True, activation=None):
        super().__init__()
        F._activation_code(activation)
        if groups < 1 or channels % groups != 0:
            raise RuntimeError(f"{channels} channels cannot be split into {groups} groups")
        self.groups, self.channels, self.eps, self.activation = groups, channels, eps, activation
        self.weight = torch.nn.Parameter(torch.ones(channels)) if affine else None
        self.bias = torch.nn.Parameter(torch.zeros(channels)) if affine else None

    def forward(self, A, X, ptr=None):
        return F.group_norm(_as_feature_matrix(X), self.groups, self.weight, self.bias, self.eps, self.activation, ptr)


class Dropout(torch.nn.Module):
    """Dropout of the node features in training mode, the identity in evaluation mode.

    ``seed`` (drawn from torch's generator when None) and a counter of the calls made so far name the mask.
    They live on the host, where a captured CUDA graph would freeze them, so a call under capture raises
    unless the layer was made with ``capturable=True``: then they are a buffer on the device that every
    call advances, and a replayed graph takes new masks.  ``state_dict`` holds both, in either form.

    A forward pass that is run again inside the backward pass (``torch.utils.checkpoint``) has to see the mask of
    the first run, and the layer cannot tell which call that was.  Take ``call = layer.next_call()`` in front of the
    recomputed region and call ``layer(A, X, call)`` inside it; a call of the layer that names no mask raises there."""

    def __init__(self, p=0.5, seed=None, capturable=False):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise RuntimeError(f"dropout probability must be in [0, 1], got {p}")
        self.p = p
        self.seed = int(torch.randint(0, 1 << 62, (1,))) if seed is None else int(seed)
        if not 0 <= self.seed < 1 << 64:
            raise RuntimeError(f"seed must be in [0, 2**64), got {self.seed}")
        self.calls = 0
        if capturable:
            self.register_buffer("state", self._words(), persistent=False)
        else:
            self.state = None

    def _words(self):
        """[seed, calls] as int64: a seed of 2**63 and above is the negative number of the same bits."""
        return torch.tensor([self.seed - (1 << 64) if self.seed >= 1 << 63 else self.seed, self.calls], dtype=torch.int64)

    # seed and counter go into state_dict, so that a run that is resumed takes the masks that would have come next
    def get_extra_state(self):
        return self._words() if self.state is None else self.state.detach().cpu().clone()

    def set_extra_state(self, words):
        seed, calls = (int(v) for v in words)
        self.seed = seed % (1 << 64)
        if self.state is None:
            self.calls = calls
        else:
            self.state.copy_(words)                    # in place: a captured graph reads it there

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        key = prefix + "_extra_state"
        if key in missing_keys:                        # saved before there was one: seed and counter stay
            missing_keys.remove(key)

    def _refuse_capture(self):
        if self.state is None and torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("Dropout under CUDA graph capture needs capturable=True: "
                               "the captured graph would repeat one mask for ever")

    def next_call(self):
        """The name of the next call's mask (a number, or the words [seed, number] on the device); counts the call."""
        self._refuse_capture()
        if self.state is None:
            self.calls += 1
            return self.calls - 1
        now = self.state.clone()
        self.state[1] += 1
        return now

    def forward(self, A, X, call=None):
        """call: what ``next_call`` gave, or None for a mask of its own."""
        if not self.training:
            return X
        if call is None:
            if 0.0 < self.p < 1.0 and torch._C._current_graph_task_id() != -1:       # else every mask is the same
                raise RuntimeError("Dropout is being run inside a backward pass, as a recomputed forward pass is, where another mask "
                                   "would belong to the gradients than to the output; take call = layer.next_call() in front of "
                                   "the recomputed region and give it to the layer: layer(A, X, call)")
            call = self.next_call()
        self._refuse_capture()
        return F.dropout(X, self.p, call) if isinstance(call, torch.Tensor) else F.dropout(X, self.p, self.seed, call)


class SeqWrapper(torch.nn.Module):
    """Lets a layer that ignores the graph (an activation, a ``Linear``) sit in a ``Sequential``."""

    def __init__(self, module):
        super().__init__()
        self.module = module

    def forward(self, A, x):
        return self.module(x)


class Sequential(torch.nn.Module):
    """Chain of layers called as ``layer(A, X)``; the result is squeezed (reference ``:180-188``)."""

    def __init__(self, *args):
        super().__init__()
        self.modlist = torch.nn.ModuleList(list(args))

    def forward(self, A, X):
        for layer in self.modlist:
            X = layer(A, X)
        return torch.squeeze(X)


def model_to_vector(model):
    """Every tensor of ``model.state_dict()`` flattened into one float32 vector on the host, in
    state-dict order (reference ``numml/nn.py:193-211``)."""
    parts = [t.detach().flatten().to(device='cpu', dtype=torch.float32) for t in model.state_dict().values()]
    return torch.cat(parts) if parts else torch.zeros(0)


def vector_to_model(model, weights_vector):
    """Replace each parameter of ``model`` by a view of its slice of ``weights_vector`` (in
    ``named_parameters`` order), so that a loss computed with the model differentiates with respect
    to the vector (reference ``numml/nn.py:221-234``).  The parameters stop being ``Parameter``s."""
    offset = 0
    for name, p in list(model.named_parameters()):
        owner_path, _, attr = name.rpartition('.')
        owner = model.get_submodule(owner_path) if owner_path else model
        count = p.numel()
        delattr(owner, attr)
        setattr(owner, attr, weights_vector[offset:offset + count].view_as(p))
        offset += count
