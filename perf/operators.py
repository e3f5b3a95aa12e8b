"""Cases of the dense operators of the graph layers: the matrix product with its epilogue
(``linear``), the group norm with an activation over graphs (``group_norm``) and the dropout whose
mask is recomputed from a counter (``dropout``).

A case is a dict of plain values.  ``prepare`` makes what a program has in hand before the call,
``run`` makes one pass through the operator, either in its plain form (``own`` false: elementary torch
operations in 32 bits, 64 where sums are long) or through ``numml_b200.functional`` (``own`` true), and
``exact`` gives the same outputs from the definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "f64": 8, "bf16": 2, "f16": 2}
ACTIVATIONS = ("none", "relu", "silu", "gelu", "tanh")


def _linear(name, m, k, n, dtype, act, bias, residual, train):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual, "train": train}


def _norm(name, graphs, rows, channels, groups, dtype, act, ragged, train):
    return {"name": name, "op": "group_norm", "graphs": graphs, "rows": rows, "channels": channels, "groups": groups,
            "dtype": dtype, "act": act, "ragged": ragged, "train": train}


def _dropout(name, rows, cols, dtype, p, residual, train):
    return {"name": name, "op": "dropout", "rows": rows, "cols": cols, "dtype": dtype, "p": p, "residual": residual,
            "train": train}


def listed():
    return [
        # one node's features through a layer of a trained network, as a serving loop asks for it
        _linear("linear_one_row_bf16", 1, 1024, 1024, "bf16", "silu", True, True, False),
        # the input layer of a small graph, inference: a call that is all latency
        _linear("linear_small_graph_f32", 257, 64, 40, "f32", "relu", True, False, False),
        # a hidden layer with a skip connection on the nodes of a 256 x 256 grid, one training step
        _linear("linear_grid_f32", 65536, 128, 128, "f32", "gelu", True, True, True),
        # a hidden layer of 128 channels on a graph of a million nodes, one training step
        _linear("linear_graph_f32", 1048576, 128, 128, "f32", "silu", True, False, True),
        # wide hidden layer in mixed-precision training
        _linear("linear_wide_bf16", 131072, 512, 512, "bf16", "silu", True, True, True),
        # a layer in double precision as gradient checks and solvers use it, with sizes that nothing divides
        _linear("linear_odd_f64", 4097, 33, 65, "f64", "tanh", True, False, True),
        # the normalisation after the first layer of one small graph, inference
        _norm("norm_small_graph_f32", 1, 1000, 64, 8, "f32", "silu", False, False),
        # a batch of molecules-sized graphs of unequal length, with unused rows behind the last, one training step
        _norm("norm_batch_bf16", 512, 61441, 128, 16, "bf16", "gelu", True, True),
        # one graph of a million nodes, one training step
        _norm("norm_graph_f32", 1, 1048576, 128, 32, "f32", "silu", False, True),
        # dropout of the features of a small graph, forward
        _dropout("dropout_small_graph_f32", 1000, 64, "f32", 0.5, False, False),
        # dropout of the stored values of the 7-point matrix on a 128^3 grid (edge dropout), one training step
        _dropout("dropout_edges_f64", 14581760, 1, "f64", 0.1, False, True),
        # dropout in front of a skip connection, one training step
        _dropout("dropout_residual_bf16", 262144, 256, "bf16", 0.2, True, True),
    ]


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(("linear", "linear", "group_norm", "dropout"))
    dtype = rng.choice(("f32", "f32", "bf16", "f16", "f64"))
    train = rng.random() < 0.6
    # relu's slope jumps at zero, where two right answers may differ: in training the smooth ones are drawn
    act = rng.choice([a for a in ACTIVATIONS if not (train and a == "relu")])
    if op == "linear":
        k, n = _log_int(rng, 1, 1024), _log_int(rng, 1, 1024)
        m = _log_int(rng, 1, 1048576)
        # no dearer than the largest listed cases, in elements and in products
        m = max(1, min(m, (1 << 28) // (k + n), (1 << (31 if dtype == "f64" else 34)) // (k * n)))
        return {"op": op, "m": m, "k": k, "n": n, "dtype": dtype, "act": act,
                "bias": rng.random() < 0.7, "residual": rng.random() < 0.5, "train": train}
    if op == "group_norm":
        groups = rng.choice((1, 2, 3, 4, 8, 16, 32))
        channels = groups * _log_int(rng, 1, 512 // groups)
        # 32 entries or more to a group of an average graph: of two or three entries the norm leaves only rounding
        least = -(-32 * groups // channels)
        rows = min(_log_int(rng, least, 1048576), (1 << (25 if dtype == "f64" else 26)) // channels)
        ragged = rng.random() < 0.6
        graphs = _log_int(rng, 1, max(1, min(rows // least, 1024)))
        if not ragged:
            rows = graphs * max(1, rows // graphs)
        return {"op": op, "graphs": graphs, "rows": rows, "channels": channels, "groups": groups, "dtype": dtype,
                "act": act, "ragged": ragged, "train": train}
    cols = _log_int(rng, 1, 512)
    rows = max(1, _log_int(rng, 1, 1 << (24 if dtype == "f64" else 26)) // cols)
    return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "p": rng.choice((0.0, 0.05, 0.1, 0.2, 0.5, 0.75)),
            "residual": rng.random() < 0.4, "train": train}


# -----------------------------------------------------------------------------------------------
# Inputs
# -----------------------------------------------------------------------------------------------
def _cut_points(case, gen):
    """Row pointers of a ragged batch: random cuts (empty graphs happen), and some rows behind the last graph."""
    rows, graphs = case["rows"], case["graphs"]
    used = rows - rows // 50
    cuts = torch.randint(0, used + 1, (graphs + 1,), generator=gen, device="cuda").sort().values
    cuts[0] = 0
    cuts[-1] = used
    return cuts


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    wide = torch.float64 if case["dtype"] == "f64" else torch.float32
    train = case["train"]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=gen, device="cuda", dtype=wide) * scale + shift).to(dt)

    state = {"case": case}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        state["x"] = normal(m, k)
        state["w"] = normal(k, n, scale=k ** -0.5)
        state["b"] = normal(n, scale=0.1) if case["bias"] else None
        state["r"] = normal(m, n) if case["residual"] else None
        leaves = ("x", "w", "b", "r")
        if train:
            state["dy"] = normal(m, n)
    elif case["op"] == "group_norm":
        rows, c = case["rows"], case["channels"]
        # features as a layer leaves them: every channel with its own level and spread
        x = torch.randn(rows, c, generator=gen, device="cuda", dtype=wide)
        level = torch.randn(c, generator=gen, device="cuda", dtype=wide)
        spread = torch.rand(c, generator=gen, device="cuda", dtype=wide) + 0.5
        x = (x * spread + level).to(dt)
        state["ptr"] = _cut_points(case, gen) if case["ragged"] else None
        if not case["ragged"] and case["graphs"] > 1:
            x = x.view(case["graphs"], rows // case["graphs"], c)
        state["x"] = x
        state["w"] = normal(c, scale=0.1, shift=1.0)
        state["b"] = normal(c, scale=0.1)
        leaves = ("x", "w", "b")
        if train:
            state["dy"] = normal(*x.shape)
    else:
        shape = (case["rows"], case["cols"]) if case["cols"] > 1 else (case["rows"],)
        state["x"] = normal(*shape)
        state["r"] = normal(*shape) if case["residual"] else None
        state["seed"] = seed * 7919 + 12345
        state["offset"] = seed % 1000
        leaves = ("x", "r")
        if train:
            state["dy"] = normal(*shape)
    state["leaves"] = [state[q].requires_grad_(True) for q in leaves if state[q] is not None] if train else []
    return state


# -----------------------------------------------------------------------------------------------
# One pass
# -----------------------------------------------------------------------------------------------
def run(state):
    forward = _own_forward if own else _plain_forward
    if not state["case"]["train"]:
        with torch.no_grad():
            return [forward(state)]
    y = forward(state)
    grads = torch.autograd.grad(y, state["leaves"], state["dy"])
    return [y.detach(), *grads]


def _own_forward(state):
    from numml_b200 import functional as F
    case = state["case"]
    if case["op"] == "linear":
        return F.linear(state["x"], state["w"], state["b"], activation=case["act"], residual=state["r"])
    if case["op"] == "group_norm":
        return F.group_norm(state["x"], case["groups"], state["w"], state["b"], activation=case["act"], ptr=state["ptr"])
    return F.dropout(state["x"], case["p"], state["seed"], state["offset"], residual=state["r"])


def _plain_activation(z, act):
    if act == "relu":
        return torch.relu(z)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "tanh":
        return torch.tanh(z)
    return z


def _wide(t):
    return t if t is None or t.dtype == torch.float64 else t.float()


def _plain_forward(state):
    case = state["case"]
    x = _wide(state["x"])
    dt = state["x"].dtype
    if case["op"] == "linear":
        z = x @ _wide(state["w"])
        if state["b"] is not None:
            z = z + _wide(state["b"])
        y = _plain_activation(z, case["act"])
        if state["r"] is not None:
            y = y + _wide(state["r"])
        return y.to(dt)
    if case["op"] == "group_norm":
        c, groups = case["channels"], case["groups"]
        if state["ptr"] is None:
            samples = case["graphs"]
            v = x.reshape(samples, -1, groups, c // groups)
            # sums over up to millions of entries: held in 64 bits
            mean = v.mean(dim=(1, 3), keepdim=True, dtype=torch.float64).to(x.dtype)
            d = v - mean
            var = (d * d).mean(dim=(1, 3), keepdim=True, dtype=torch.float64).to(x.dtype)
            h = (d * torch.rsqrt(var + 1e-5)).reshape(x.shape)
            return _plain_activation(h * _wide(state["w"]) + _wide(state["b"]), case["act"]).to(dt)
        ptr, graphs = state["ptr"], case["graphs"]
        row = torch.arange(case["rows"], device=x.device)
        seg = torch.searchsorted(ptr, row, right=True) - 1
        inside = (seg >= 0) & (seg < graphs)
        seg = torch.where(inside, seg, graphs)                     # one more segment for the unused rows
        count = torch.zeros(graphs + 1, device=x.device, dtype=torch.float64)
        count = count.index_add(0, seg, torch.ones_like(row, dtype=torch.float64)).clamp(min=1.0) * (c // groups)
        v = x.reshape(-1, groups, c // groups)
        zero = torch.zeros(graphs + 1, groups, device=x.device, dtype=torch.float64)
        mean = (zero.index_add(0, seg, v.sum(2, dtype=torch.float64)) / count[:, None]).to(x.dtype)
        d = v - mean[seg][:, :, None]
        var = (zero.index_add(0, seg, (d * d).sum(2, dtype=torch.float64)) / count[:, None]).to(x.dtype)
        h = (d * torch.rsqrt(var + 1e-5)[seg][:, :, None]).reshape(x.shape)
        y = _plain_activation(h * _wide(state["w"]) + _wide(state["b"]), case["act"])
        return torch.where(inside[:, None], y, torch.zeros_like(y)).to(dt)
    keep = _plain_keep(x.numel(), case["p"], state["seed"], state["offset"], x.device).view(x.shape)
    y = torch.where(keep, x * (1.0 / (1.0 - case["p"])), torch.zeros_like(x))
    if state["r"] is not None:
        y = y + _wide(state["r"])
    return y.to(dt)


# Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011)
_M0, _M1, _W0, _W1, _LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def _plain_philox(block, seed, offset, stream):
    """The four output words, as int64 tensors, of the counters (block, offset, stream) under the key `seed`."""
    c0, c1 = block & _LOW, block >> 32
    c2 = torch.full_like(block, offset & _LOW)
    c3 = torch.full_like(block, (offset >> 32) & 0x7FFFFFFF | stream << 31)
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        p0, p1 = c0 * _M0, c2 * _M1                    # 64-bit products, modulo 2^64
        c0, c1, c2, c3 = (p1 >> 32) & _LOW ^ c1 ^ k0, p1 & _LOW, (p0 >> 32) & _LOW ^ c3 ^ k1, p0 & _LOW
        k0, k1 = (k0 + _W0) & _LOW, (k1 + _W1) & _LOW
    return c0, c1, c2, c3


def _plain_keep(n, p, seed, offset, device):
    block = torch.arange((n + 7) // 8, device=device)
    halves = []
    for stream in (0, 1):
        words = torch.stack(_plain_philox(block, seed, offset, stream), dim=1)
        halves.append(torch.stack((words & 0xFFFF, words >> 16), dim=2).reshape(-1)[:n])
    u = halves[0] * 65536 + halves[1]
    return u >= round(p * 4294967296.0)


# -----------------------------------------------------------------------------------------------
# What a pass cannot do without
# -----------------------------------------------------------------------------------------------
def work(case):
    s = SIZE[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        elements = m * k + k * n + m * n + (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
        flops = 2 * m * k * n
        if case["train"]:
            # dy read; dx, dw, db written (the residual's gradient is dy itself)
            elements += m * n + m * k + k * n + (n if case["bias"] else 0)
            flops *= 3
        return {"bytes": s * elements, "flops": flops}
    if case["op"] == "group_norm":
        size = case["rows"] * case["channels"]
        elements = 2 * size + 2 * case["channels"]
        if case["train"]:
            elements += 2 * size + 2 * case["channels"]
        return {"bytes": s * elements, "flops": (20 if case["train"] else 8) * size}
    n = case["rows"] * case["cols"]
    passes = 2 + (1 if case["residual"] else 0) + (2 if case["train"] else 0)
    return {"bytes": s * n * passes, "flops": 2 * n}


# -----------------------------------------------------------------------------------------------
# The definitions in 64 bits
# -----------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        t = {q: v.detach().double() for q, v in state.items()
             if isinstance(v, torch.Tensor) and v.is_floating_point()}
        if case["op"] == "linear":
            return _exact_linear(case, t)
        if case["op"] == "group_norm":
            return _exact_group_norm(case, t, state["ptr"])
        return _exact_dropout(case, t, state["seed"], state["offset"])


def _exact_activation(z, act):
    """Value and derivative."""
    if act == "relu":
        on = (z > 0).double()
        return z * on, on
    if act == "silu":
        e = torch.exp(-z.abs())
        s = torch.where(z >= 0, 1 / (1 + e), e / (1 + e))
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "tanh":
        v = torch.tanh(z)
        return v, 1 - v * v
    return z, torch.ones_like(z)


def _exact_linear(case, t):
    z = torch.mm(t["x"], t["w"])
    if "b" in t:
        z += t["b"]
    a, slope = _exact_activation(z, case["act"])
    out = [a + t["r"] if "r" in t else a]
    if case["train"]:
        dz = t["dy"] * slope
        out += [torch.mm(dz, t["w"].T), torch.mm(t["x"].T, dz)]
        if "b" in t:
            out.append(dz.sum(0))
        if "r" in t:
            out.append(t["dy"])
    return out


def _exact_group_norm(case, t, ptr):
    c, groups, graphs = case["channels"], case["groups"], case["graphs"]
    x = t["x"].reshape(-1, c)
    if ptr is None:
        per = case["rows"] // graphs
        bounds = [per * q for q in range(graphs + 1)]
    else:
        bounds = ptr.tolist()
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    dw, db = torch.zeros_like(t["w"]), torch.zeros_like(t["b"])
    for lo, hi in zip(bounds[:-1], bounds[1:]):
        if hi <= lo:
            continue
        v = x[lo:hi].reshape(hi - lo, groups, c // groups)
        var, mean = torch.var_mean(v, dim=(0, 2), correction=0, keepdim=True)
        rstd = 1.0 / torch.sqrt(var + 1e-5)
        xhat = (v - mean) * rstd
        flat = xhat.reshape(hi - lo, c)
        y[lo:hi], slope = _exact_activation(flat * t["w"] + t["b"], case["act"])
        if case["train"]:
            dz = t["dy"].reshape(-1, c)[lo:hi] * slope
            db += dz.sum(0)
            dw += (dz * flat).sum(0)
            h = (dz * t["w"]).reshape(v.shape)
            along = h.mean(dim=(0, 2), keepdim=True)
            radial = (h * xhat).mean(dim=(0, 2), keepdim=True)
            dx[lo:hi] = (rstd * (h - along - xhat * radial)).reshape(hi - lo, c)
    out = [y.reshape(t["x"].shape)]
    return out + [dx.reshape(t["x"].shape), dw, db] if case["train"] else out


def _exact_halfwords(n, seed, offset, stream):
    """The 16-bit halves of the generator's outputs for elements 0..n-1, with products formed from 16-bit limbs."""
    blocks = torch.arange(-(-n // 8), device="cuda")
    tail = torch.zeros_like(blocks)
    ctr = [blocks % 2 ** 32, blocks // 2 ** 32, tail + offset % 2 ** 32, tail + (offset // 2 ** 32 + stream * 2 ** 31)]
    key = [seed % 2 ** 32, seed // 2 ** 32 % 2 ** 32]

    def high_low(a, b):
        a1, a0, b1, b0 = a // 65536, a % 65536, b // 65536, b % 65536
        low = a0 * b0
        mid = a1 * b0 + low // 65536
        cross = a0 * b1 + mid % 65536
        return a1 * b1 + mid // 65536 + cross // 65536, cross % 65536 * 65536 + low % 65536

    for _ in range(10):
        h0, l0 = high_low(ctr[0], _M0)
        h1, l1 = high_low(ctr[2], _M1)
        ctr = [torch.bitwise_xor(torch.bitwise_xor(h1, ctr[1]), key[0]), l1,
               torch.bitwise_xor(torch.bitwise_xor(h0, ctr[3]), key[1]), l0]
        key = [(key[0] + _W0) % 2 ** 32, (key[1] + _W1) % 2 ** 32]
    out = torch.empty(blocks.numel(), 8, dtype=torch.int64, device="cuda")
    for q in range(4):
        out[:, 2 * q] = ctr[q] % 65536
        out[:, 2 * q + 1] = ctr[q] // 65536
    return out.flatten()[:n]


def _exact_dropout(case, t, seed, offset):
    x, p = t["x"], case["p"]
    bar = round(p * 2 ** 32)
    upper, lower = _exact_halfwords(x.numel(), seed, offset, 0), _exact_halfwords(x.numel(), seed, offset, 1)
    mask = ((upper > bar // 65536) | ((upper == bar // 65536) & (lower >= bar % 65536))).double().view(x.shape)
    y = x * mask / (1.0 - p)
    if "r" in t:
        y = y + t["r"]
    out = [y]
    if case["train"]:
        out.append(t["dy"] * mask / (1.0 - p))
        if "r" in t:
            out.append(t["dy"])
    return out
