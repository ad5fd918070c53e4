"""The measured cases of the 8-bit integer operators: the product with scales for each token
and channel, the linear layer made of it (forward and backward), the quantiser that feeds it
and dropout from the counter-based generator.

``run`` computes each case in plain torch operations, or through the package's entry points
where ``own`` is true.  Sizes follow the repository's benchmark shapes (8192 x 28672 x 8192 and
its tokens x weights family) or are generic; odd ones stand for ragged batches and heads.
"""
from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_GOLDEN = 0x9E3779B97F4A7C15
_MUL1, _MUL2 = 0xBF58476D1CE4E5B9, 0x94D049BB133111EB
_TINY = 2.0 ** -126
_ELEM = {"bfloat16": 2, "float16": 2, "float32": 4}


def _pkg():
    name = "microbench_blackwell_b200"
    if name not in sys.modules:
        folder = Path.cwd() / "microbench-blackwell_b200"
        spec = importlib.util.spec_from_file_location(name, folder / "__init__.py",
                                                      submodule_search_locations=[str(folder)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One token through a square projection: the latency of a decoding step.
        dict(name="one_token", op="linear", m=1, n=8192, k=8192, dtype="bfloat16", bias=False, p=0.0, residual=False),
        # A handful of drafted tokens, already quantised, ragged sizes.
        dict(name="few_tokens_odd", op="product", m=5, n=4099, k=1000, dtype="float16", bias=True, p=0.0, residual=False),
        # A decoding batch through the up projection of the benchmark's MLP.
        dict(name="decode_batch", op="linear", m=48, n=28672, k=8192, dtype="bfloat16", bias=False, p=0.0, residual=False),
        # A ragged chunk of a prompt, quantised by an earlier step, fp32 output.
        dict(name="chunk_odd", op="product", m=777, n=5000, k=2056, dtype="float32", bias=True, p=0.0, residual=False),
        # A long prompt through the up projection: the benchmark's 8192 x 28672 x 8192.
        dict(name="prompt", op="linear", m=8192, n=28672, k=8192, dtype="bfloat16", bias=False, p=0.0, residual=False),
        # The output projection of a training step: bias, dropout and the residual stream.
        dict(name="train_forward", op="linear", m=4096, n=8192, k=8192, dtype="bfloat16", bias=True, p=0.1, residual=True),
        # Its gradients for tokens, weights and bias.
        dict(name="train_backward", op="backward", m=4096, n=8192, k=8192, dtype="bfloat16", p=0.1),
        # Gradients of a small ragged layer in fp32.
        dict(name="backward_odd", op="backward", m=333, n=1000, k=2500, dtype="float32", p=0.25),
        # Activations of a prompt, one scale for each token.
        dict(name="quantize_tokens", op="quantize", rows=16384, cols=8192, dtype="bfloat16", transpose=False),
        # Weights for the backward products: one scale for each input channel, transposed.
        dict(name="quantize_transposed", op="quantize", rows=8192, cols=28672, dtype="bfloat16", transpose=True),
        # The residual stream of a long training batch.
        dict(name="dropout_residual", op="dropout", rows=16384, cols=8192, dtype="bfloat16", p=0.1, residual=True,
             col0=0, row_elems=8192),
        # A rank's odd slice of columns of a wider matrix, gradient direction (no residual).
        dict(name="dropout_slice", op="dropout", rows=33, cols=1001, dtype="float32", p=0.5, residual=False,
             col0=1001, row_elems=4004),
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    top = work(listed()[4])
    while True:
        op = rng.choice(["product", "linear", "linear", "backward", "quantize", "dropout"])
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        p = rng.choice([0.0, 0.0, 0.1, 0.25, 0.5])
        if op in ("product", "linear"):
            case = dict(op=op, m=_spread(rng, 1, 8192), n=_spread(rng, 16, 28672), k=_spread(rng, 16, 28672),
                        dtype=dtype, bias=rng.random() < 0.5, p=p, residual=rng.random() < 0.3)
        elif op == "backward":
            case = dict(op=op, m=_spread(rng, 1, 8192), n=_spread(rng, 16, 16384), k=_spread(rng, 16, 16384),
                        dtype=dtype, p=p)
        elif op == "quantize":
            case = dict(op=op, rows=_spread(rng, 1, 16384), cols=_spread(rng, 16, 28672), dtype=dtype,
                        transpose=rng.random() < 0.5)
        else:
            cols = _spread(rng, 16, 28672)
            col0 = rng.choice([0, cols, 3 * cols])
            case = dict(op=op, rows=_spread(rng, 1, 16384), cols=cols, dtype=dtype, p=rng.choice([0.1, 0.25, 0.5]),
                        residual=rng.random() < 0.5, col0=col0, row_elems=4 * cols)
        w = work(case)
        if w["flops"] <= top["flops"] and w["bytes"] <= top["bytes"]:
            return case


def work(case):
    e = _ELEM[case["dtype"]]
    if case["op"] in ("quantize", "dropout"):
        n = case["rows"] * case["cols"]
        if case["op"] == "quantize":
            return {"bytes": n * (e + 1) + 4 * (case["cols"] if case["transpose"] else case["rows"]), "flops": 2 * n}
        return {"bytes": n * e * (3 if case["residual"] else 2), "flops": 2 * n}
    m, n, k = case["m"], case["n"], case["k"]
    if case["op"] == "backward":
        return {"bytes": m * n * e + m * k * e + n * k + 4 * k + m * k * e + 4 * n * k + 4 * n, "flops": 4 * m * n * k}
    read = m * k * (1 if case["op"] == "product" else e) + n * k + 4 * n + (4 * m if case["op"] == "product" else 0)
    read += (e * n if case["bias"] else 0) + (e * m * n if case["residual"] else 0)
    return {"bytes": read + m * n * e, "flops": 2 * m * n * k}


# ------------------------------------------------------------------ inputs
def _activations(g, rows, cols, dtype):
    """Normal values, with a few channels far above the others, as activations have them."""
    x = torch.randn((rows, cols), generator=g, device="cuda", dtype=torch.float32)
    boost = torch.rand((cols,), generator=g, device="cuda")
    return x.mul_(torch.where(boost > 0.995, 8.0, 1.0)).to(dtype)


def _packed(q):
    """int8 rows whose stride is a multiple of 16 bytes."""
    rows, cols = q.shape
    store = torch.zeros((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=q.device)
    store[:, :cols] = q
    return store[:, :cols]


def _quantized(x):
    q, s = _rows(x.float())
    return _packed(q.to(torch.int8)), s.reshape(-1).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    dtype = getattr(torch, case["dtype"])
    s = dict(case=case, seed=int(seed) * 31 + 5)
    if case["op"] in ("quantize", "dropout"):
        s["x"] = _activations(g, case["rows"], case["cols"], dtype)
        s["residual"] = (torch.randn((case["rows"], case["cols"]), generator=g, device="cuda").to(dtype)
                         if case.get("residual") else None)
        return s
    m, n, k = case["m"], case["n"], case["k"]
    x = _activations(g, m, k, dtype)
    w = torch.randn((n, k), generator=g, device="cuda").mul_(0.02)
    if case["op"] == "backward":
        s["x"] = x
        s["dy"] = torch.randn((m, n), generator=g, device="cuda").to(dtype)
        s["wt"], s["wt_scale"] = _quantized(w.t())
        return s
    s["w"], s["w_scale"] = _quantized(w)
    s["bias"] = torch.randn((n,), generator=g, device="cuda").to(dtype) if case["bias"] else None
    s["residual"] = torch.randn((m, n), generator=g, device="cuda").to(dtype) if case["residual"] else None
    if case["op"] == "product":
        s["x"], s["x_scale"] = _quantized(x)
    else:
        s["x"] = x
    return s


# ------------------------------------------------------------------ the plain form
def _rows(x):
    """Whole numbers (as fp32) and scales of the rows of `x`: rint(127 x / max |x|), ties to even.
    The quotient is formed in 64 bits: bf16 rows hold many values that lie exactly between two steps."""
    largest = torch.clamp(x.abs().amax(dim=1, keepdim=True).double(), min=127.0 * _TINY)
    return torch.round(x.double() * 127.0 / largest).float(), (largest / 127.0).float()


def _signed(v):
    v &= 0xFFFFFFFFFFFFFFFF
    return v - (1 << 64) if v >> 63 else v


def _shift(z, bits):
    return (z >> bits) & ((1 << (64 - bits)) - 1)


def _mix(z):
    z = (z ^ _shift(z, 30)) * _signed(_MUL1)
    z = (z ^ _shift(z, 27)) * _signed(_MUL2)
    return z ^ _shift(z, 31)


def _mix_int(z):
    z &= 0xFFFFFFFFFFFFFFFF
    z = ((z ^ (z >> 30)) * _MUL1) & 0xFFFFFFFFFFFFFFFF
    z = ((z ^ (z >> 27)) * _MUL2) & 0xFFFFFFFFFFFFFFFF
    return z ^ (z >> 31)


def _key(seed, stream):
    return _mix_int(seed + _mix_int(stream + _GOLDEN))


def _kept(like, p, seed, col0=0, row_elems=None):
    """Which elements of a matrix of `like`'s shape dropout keeps."""
    rows, cols = like.shape
    row_elems = cols if row_elems is None else row_elems
    index = (torch.arange(rows, device=like.device)[:, None] * row_elems
             + (col0 + torch.arange(cols, device=like.device))[None, :])
    z = _mix(((index >> 1) + 1) * _signed(_GOLDEN) + _signed(_key(seed, 0)))
    word = torch.where((index & 1) == 1, _shift(z, 32), z & 0xFFFFFFFF)
    return word >= round(p * 2 ** 32)


def _drop(x, p, seed, col0=0, row_elems=None):
    """fp32 `x` with its dropped elements zeroed and the others divided by 1 - p."""
    return torch.where(_kept(x, p, seed, col0, row_elems), x * (1.0 / (1.0 - p)), 0.0) if p else x


def _plain_linear(s, q, q_scale):
    case = s["case"]
    y = torch.matmul(q, s["w"].float().t()) * q_scale * s["w_scale"][None, :]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _drop(y, case["p"], s["seed"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(getattr(torch, case["dtype"]))


def _plain(s):
    case = s["case"]
    if case["op"] == "quantize":
        x = s["x"].float()
        q, scale = _rows(x.t() if case["transpose"] else x)
        return {"q": q.to(torch.int8), "scale": scale.reshape(-1)}
    if case["op"] == "dropout":
        y = _drop(s["x"].float(), case["p"], s["seed"], case["col0"], case["row_elems"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return y.to(s["x"].dtype)
    if case["op"] == "product":
        return _plain_linear(s, s["x"].float(), s["x_scale"][:, None])
    if case["op"] == "linear":
        return _plain_linear(s, *_rows(s["x"].float()))
    # Dropout's factor 1 / (1 - p) is common to all kept gradients, so it goes into the scales.
    p = case["p"]
    dz = s["dy"].float()
    if p:
        dz = torch.where(_kept(dz, p, s["seed"]), dz, 0.0)
    grow = 1.0 / (1.0 - p)
    qr, sr = _rows(dz)
    dx = torch.matmul(qr, s["wt"].float().t()) * (sr * grow) * s["wt_scale"][None, :]
    qd, sd = _rows(dz.t())
    qx, sx = _rows(s["x"].float().t())
    dw = torch.matmul(qd, qx.t()) * (sd * grow) * sx.reshape(1, -1)
    return {"dx": dx.to(s["x"].dtype), "dw": dw, "dbias": (dz.double().sum(dim=0) * grow).float()}


def run(state):
    if not own:
        return _plain(state)
    s, case, pkg = state, state["case"], _pkg()
    p = case.get("p", 0.0)
    if case["op"] == "quantize":
        q, scale = pkg.quantize_int8(s["x"], transpose=case["transpose"])
        return {"q": q, "scale": scale}
    if case["op"] == "dropout":
        drop = pkg.Dropout(p, s["seed"], col0=case["col0"], row_elems=case["row_elems"])
        return pkg.dropout(s["x"], drop, residual=s["residual"])
    drop = pkg.Dropout(p, s["seed"]) if p else None
    if case["op"] == "product":
        return pkg.gemm_int8(s["x"], s["x_scale"], s["w"], s["w_scale"], bias=s["bias"], dropout=drop,
                             residual=s["residual"], out_dtype=getattr(torch, case["dtype"]))
    if case["op"] == "linear":
        return pkg.linear_int8(s["x"], s["w"], s["w_scale"], bias=s["bias"], dropout=drop, residual=s["residual"])
    dx, dw, dbias = pkg.linear_int8_backward(s["dy"], s["x"], s["wt"], s["wt_scale"], dropout=drop)
    return {"dx": dx, "dw": dw, "dbias": dbias}


# ------------------------------------------------------------------ the definition, in 64 bits
def _exact_quantized(x):
    """Whole numbers and scales of the rows of an fp64 matrix whose values fit in fp32."""
    largest = x.abs().max(dim=1).values
    largest = torch.where(largest < 127.0 * _TINY, torch.full_like(largest, 127.0 * _TINY), largest)
    return torch.round((127.0 * x) / largest[:, None]), largest / 127.0


def _exact_mask(like, p, seed, col0=0, row_elems=None):
    """1.0 where an element is kept, word by word with unsigned numpy integers, a block of rows at a time."""
    rows, cols = like.shape
    row_elems = cols if row_elems is None else row_elems
    with np.errstate(over="ignore"):
        def finish(v):
            v ^= v >> np.uint64(30)
            v *= np.uint64(_MUL1)
            v ^= v >> np.uint64(27)
            v *= np.uint64(_MUL2)
            v ^= v >> np.uint64(31)
            return v

        key = finish(np.array([seed], np.uint64) + finish(np.array([_GOLDEN], np.uint64)))
        mask = torch.empty_like(like)
        block = max(1, (1 << 22) // cols)
        for r in range(0, rows, block):
            here = np.arange(r, min(rows, r + block), dtype=np.uint64)[:, None] * np.uint64(row_elems)
            at = here + np.arange(col0, col0 + cols, dtype=np.uint64)[None, :]
            v = finish((at // np.uint64(2) + np.uint64(1)) * np.uint64(_GOLDEN) + key)
            odd = (at % np.uint64(2)).astype(bool)
            word = np.where(odd, v >> np.uint64(32), v % np.uint64(1 << 32))
            mask[r:r + block] = torch.from_numpy(word >= np.uint64(round(p * 2 ** 32))).to(like.device)
    return mask


def _exact_drop(x, p, seed, col0=0, row_elems=None):
    return x / (1.0 - p) * _exact_mask(x, p, seed, col0, row_elems) if p else x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        x = s["x"].double()
        q, scale = _exact_quantized(x.t().contiguous() if case["transpose"] else x)
        return {"q": None, "scale": scale}
    if case["op"] == "dropout":
        y = _exact_drop(s["x"].double(), case["p"], s["seed"], case["col0"], case["row_elems"])
        return y if s["residual"] is None else y + s["residual"].double()
    if case["op"] == "backward":
        dz = s["dy"].double()
        if case["p"]:
            dz = dz * _exact_mask(dz, case["p"], s["seed"])
        q, scale = _exact_quantized(dz)
        dx = (q @ s["wt"].double().t()) * torch.outer(scale / (1.0 - case["p"]), s["wt_scale"].double())
        q, scale = _exact_quantized(dz.t().contiguous())
        t, t_scale = _exact_quantized(s["x"].double().t().contiguous())
        dw = (q @ t.t()) * torch.outer(scale / (1.0 - case["p"]), t_scale)
        return {"dx": dx, "dw": dw, "dbias": dz.sum(dim=0) / (1.0 - case["p"])}
    q, scale = (s["x"].double(), s["x_scale"].double()) if case["op"] == "product" else _exact_quantized(s["x"].double())
    y = (q @ s["w"].double().t()) * torch.outer(scale, s["w_scale"].double())
    if s["bias"] is not None:
        y += s["bias"].double()
    y = _exact_drop(y, case["p"], s["seed"])
    return y if s["residual"] is None else y + s["residual"].double()
