"""The measured cases of the 4-bit floating operators and of the norms around a block: the quantiser to
microscaled e2m1 (blocks of 16 with e4m3 scales, or of 32 with powers of two), the product of such
operands, the linear layer made of both, and the residual stream's update with the norms before and after
it (forward, backward, and straight into a 4-bit operand).

``run`` computes each case in plain torch operations, or through the package's entry points
where ``own`` is true.  Sizes follow the repository's benchmark shapes (8192 x 28672 x 8192 and
its tokens x weights family) or are generic; odd ones stand for ragged batches and heads.
"""
from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

_ELEM = {"bfloat16": 2, "float16": 2, "float32": 4}
_EPS = 1e-6
_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


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
        dict(name="one_token", op="linear", m=1, n=8192, k=8192, block=16, dtype="bfloat16", bias=False, residual=False),
        # A handful of drafted tokens, already quantised, ragged sizes, scales that are powers of two.
        dict(name="few_tokens_odd", op="product", m=5, n=4099, k=1000, block=32, dtype="float16", bias=True, residual=False),
        # A decoding batch through the up projection of the benchmark's MLP.
        dict(name="decode_batch", op="linear", m=48, n=28672, k=8192, block=16, dtype="bfloat16", bias=False, residual=False),
        # A ragged chunk of a prompt, quantised by an earlier step, added to the residual stream.
        dict(name="chunk_odd", op="product", m=777, n=5000, k=2056, block=16, dtype="bfloat16", bias=True, residual=True),
        # A long prompt through the up projection: the benchmark's 8192 x 28672 x 8192.
        dict(name="prompt", op="linear", m=8192, n=28672, k=8192, block=16, dtype="bfloat16", bias=False, residual=False),
        # Activations of a prompt to 4 bits and back.
        dict(name="quantize_tokens", op="quantize", rows=16384, cols=8192, block=16, dtype="bfloat16"),
        # A ragged fp32 matrix, blocks of 32.
        dict(name="quantize_odd", op="quantize", rows=777, cols=5001, block=32, dtype="float32"),
        # The entry of a block for one decoded token: residual stream, both norms, 4-bit operand, projection.
        dict(name="block_entry_token", op="norm_product", m=1, n=8192, k=8192, block=16, dtype="bfloat16",
             post=True, gate="vector", params="bfloat16"),
        # The same for a long prompt.
        dict(name="block_entry_prompt", op="norm_product", m=4096, n=8192, k=8192, block=16, dtype="bfloat16",
             post=True, gate="none", params="bfloat16"),
        # A long training batch: residual stream, gate, both norms.
        dict(name="norm_train", op="norm", rows=16384, cols=8192, dtype="bfloat16", post=True, gate="vector", params="float32"),
        # Its gradients.
        dict(name="norm_train_backward", op="norm_backward", rows=16384, cols=8192, dtype="bfloat16", post=True,
             gate="vector", params="float32"),
        # Gradients of a small ragged block in fp32, one gate for each token.
        dict(name="norm_backward_odd", op="norm_backward", rows=333, cols=1001, dtype="float32", post=True,
             gate="matrix", params="float32"),
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    every = listed()
    top = work(every[4])
    most = work(every[10])["bytes"]
    while True:
        op = rng.choice(["product", "linear", "linear", "quantize", "norm_product", "norm", "norm_backward"])
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        half = rng.choice(["bfloat16", "bfloat16", "float16"])
        block = rng.choice([16, 16, 32])
        around = dict(post=rng.random() < 0.6, gate=rng.choice(["none", "vector", "matrix"]))
        if op in ("product", "linear"):
            case = dict(op=op, m=_spread(rng, 1, 8192), n=_spread(rng, 16, 28672), k=_spread(rng, 16, 28672),
                        block=block, dtype=half, bias=rng.random() < 0.5, residual=rng.random() < 0.3)
        elif op == "norm_product":
            case = dict(op=op, m=_spread(rng, 1, 8192), n=_spread(rng, 16, 28672), k=_spread(rng, 16, 16384),
                        block=block, dtype=half, params=rng.choice([half, "float32"]), **around)
        elif op == "quantize":
            case = dict(op=op, rows=_spread(rng, 1, 16384), cols=_spread(rng, 16, 28672), block=block, dtype=dtype)
        else:
            case = dict(op=op, rows=_spread(rng, 1, 16384), cols=_spread(rng, 16, 16384), dtype=dtype,
                        params=rng.choice([dtype, "float32"]), **around)
        w = work(case)
        if w["flops"] <= top["flops"] and w["bytes"] <= most:
            return case


def _four_bits(rows, cols, block):
    """Bytes of a 4-bit operand: values, block scales and row scales."""
    return rows * ((cols + 1) // 2 + (cols + block - 1) // block + 4)


def work(case):
    e = _ELEM[case["dtype"]]
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * e + _four_bits(case["rows"], case["cols"], case["block"]), "flops": 4 * n}
    if op in ("product", "linear"):
        m, n, k = case["m"], case["n"], case["k"]
        read = _four_bits(m, k, case["block"]) if op == "product" else m * k * e
        read += _four_bits(n, k, case["block"]) + (e * n if case["bias"] else 0) + (e * m * n if case["residual"] else 0)
        return {"bytes": read + m * n * e, "flops": 2 * m * n * k}
    rows, cols = (case["m"], case["k"]) if op == "norm_product" else (case["rows"], case["cols"])
    params = _ELEM[case["params"]] * cols * (1 + case["post"] + (case["gate"] == "vector"))
    gate = rows * cols * e if case["gate"] == "matrix" else 0
    n = rows * cols
    if op == "norm":
        return {"bytes": 4 * n * e + params + gate, "flops": 12 * n}
    if op == "norm_product":
        return {"bytes": 3 * n * e + params + gate + _four_bits(case["n"], cols, case["block"]) + rows * case["n"] * e,
                "flops": 2 * rows * cols * case["n"]}
    grads = 4 * cols * (1 + case["post"] + (case["gate"] == "vector"))
    return {"bytes": 6 * n * e + params + 2 * gate + grads, "flops": 30 * n}


# ------------------------------------------------------------------ inputs
def _activations(g, rows, cols, dtype):
    """Normal values, with a few channels far above the others, as activations have them."""
    x = torch.randn((rows, cols), generator=g, device="cuda", dtype=torch.float32)
    boost = torch.rand((cols,), generator=g, device="cuda")
    return x.mul_(torch.where(boost > 0.995, 8.0, 1.0)).to(dtype)


def _scale_columns(cols, block):
    """Scales of a row as stored: those of whole 256-element steps."""
    return (cols + 255) // 256 * (256 // block)


def _scale_place(rows, cols, block):
    """Where the scale of (row, block column) lies: tiles of 128 rows x 4 scales, 512 bytes each."""
    r = torch.arange(rows, device="cuda")[:, None]
    c = torch.arange(_scale_columns(cols, block), device="cuda")[None, :]
    return (r // 128 * (_scale_columns(cols, block) // 4) + c // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + c % 4


def _packed(x, block):
    """A 4-bit operand as a program keeps it: codes two to a byte, scales in their tiles, row scales."""
    rows, cols = x.shape
    q, s, g = _quantized(x, block)
    code = torch.bucketize(q.abs(), torch.tensor(_E2M1, device="cuda")).to(torch.uint8) + (q < 0).to(torch.uint8) * 8
    if cols % 2:
        code = torch.nn.functional.pad(code, (0, 1))
    store = torch.zeros((rows, (cols + 255) // 256 * 128), dtype=torch.uint8, device="cuda")
    values = store[:, : (cols + 1) // 2]
    values.copy_(code[:, 0::2] | code[:, 1::2] << 4)
    if block == 16:
        byte = s.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        byte = (torch.frexp(s)[1] + 126).to(torch.uint8)
    wide = torch.zeros((rows, _scale_columns(cols, block)), dtype=torch.uint8, device="cuda")
    wide[:, : byte.shape[1]] = byte
    scales = torch.zeros(((rows + 127) // 128 * _scale_columns(cols, block) * 128,), dtype=torch.uint8, device="cuda")
    scales[_scale_place(rows, cols, block).reshape(-1)] = wide.reshape(-1)
    return dict(values=values, scales=scales, row_scale=g.reshape(-1).contiguous(), cols=cols, block=block)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 29)
    dtype = getattr(torch, case["dtype"])
    op = case["op"]
    s = dict(case=case)

    def normal(*shape, scale=1.0, around=0.0, to=dtype):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale).add_(around).to(to)

    if op == "quantize":
        s["x"] = _activations(g, case["rows"], case["cols"], dtype)
        return s
    if op.startswith("norm"):
        rows, cols = (case["m"], case["k"]) if op == "norm_product" else (case["rows"], case["cols"])
        params = getattr(torch, case["params"])
        s["x"] = _activations(g, rows, cols, dtype)
        s["y"] = normal(rows, cols, scale=0.3)
        s["weight"] = normal(cols, scale=0.2, around=1.0, to=params)
        s["post"] = normal(cols, scale=0.2, around=0.5, to=params) if case["post"] else None
        s["gate"] = {"none": None, "vector": normal(cols, scale=0.3, around=0.7, to=params),
                     "matrix": torch.sigmoid(normal(rows, cols)) if case["gate"] == "matrix" else None}[case["gate"]]
        s["scale"] = 0.5 if case["gate"] != "none" else 1.0
        if op == "norm_backward":
            s["dh"] = normal(rows, cols)
            s["dx"] = normal(rows, cols)
        if op == "norm_product":
            s["w"] = _packed(normal(case["n"], cols, scale=0.02), case["block"])
        return s
    m, n, k = case["m"], case["n"], case["k"]
    x = _activations(g, m, k, dtype)
    s["w"] = _packed(normal(n, k, scale=0.02), case["block"])
    s["bias"] = normal(n) if case["bias"] else None
    s["residual"] = normal(m, n) if case["residual"] else None
    s["x"] = _packed(x, case["block"]) if op == "product" else x
    return s


# ------------------------------------------------------------------ the plain form
def _power(e):
    """2^e of whole numbers as fp64, put together from its bits (a power function may be off by a step)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _quantized(x, block):
    """e2m1 values, block scales and row scales (fp32) of the rows of `x`: x ~ value * block scale * row scale.
    The row scale is a power of two that brings the largest element to [1024, 2048), the block scale
    the least e4m3 number (or power of two) that lets no element pass 6; quotients next to a border are formed in 64 bits."""
    rows, cols = x.shape
    x = x.float()
    top = torch.frexp(torch.clamp(x.abs().amax(dim=1, keepdim=True), min=2.0 ** -116))[1] - 1   # floor(log2)
    y = (x.double() * _power(10 - top)).float()
    pad = -cols % block
    y = torch.nn.functional.pad(y, (0, pad)) if pad else y
    y = y.view(rows, -1, block)
    need = y.abs().amax(dim=2, keepdim=True).double() / 6.0
    if block == 16:
        step = _power(torch.clamp(torch.frexp(need)[1] - 1, min=-6) - 3)
        s = torch.ceil(need / step) * step
    else:
        part, e = torch.frexp(need)                     # need = part * 2^e, part in [1/2, 1) or 0
        s = _power(torch.where(need > 0, torch.clamp(torch.where(part > 0.5, e, e - 1), min=-126), -126))
    t = torch.where(s > 0, y.double() / torch.where(s > 0, s, 1.0), 0.0).float()
    a = t.abs()
    q = torch.where(a <= 2, torch.round(a * 2) / 2, torch.where(a <= 4, torch.round(a), torch.round(a / 2) * 2))
    q = torch.copysign(q, t).view(rows, -1)[:, :cols]
    return q, s.squeeze(2).float(), _power(top - 10).float()


def _spread_scales(q, s, block):
    return q * s.repeat_interleave(block, dim=1)[:, : q.shape[1]]


def _unpacked(p):
    """Values times block scales of a packed operand, fp32."""
    rows, cols, block = p["values"].shape[0], p["cols"], p["block"]
    table = torch.tensor(_E2M1 + [-v for v in _E2M1], device="cuda")
    code = torch.stack((p["values"] & 15, p["values"] >> 4), dim=2).view(rows, -1)[:, :cols]
    byte = p["scales"][_scale_place(rows, cols, block)][:, : (cols + block - 1) // block]
    s = byte.contiguous().view(torch.float8_e4m3fn).float() if block == 16 else _power(byte.int() - 127).float()
    return _spread_scales(table[code.int()], s, block)


def _plain_product(s, a, a_row):
    """bias, residual and row scales around the sums of a . w^T."""
    y = torch.matmul(a, _unpacked(s["w"]).t()) * a_row * s["w"]["row_scale"][None, :]
    if s.get("bias") is not None:
        y = y + s["bias"].float()
    if s.get("residual") is not None:
        y = y + s["residual"].float()
    return y.to(getattr(torch, s["case"]["dtype"]))


def _normed(v):
    """Rows of fp32 `v` over their root mean square; the mean in 64 bits."""
    r = (1.0 / (v.double().square().mean(dim=1, keepdim=True) + _EPS).sqrt()).float()
    return v * r, r


def _plain_norm(s):
    z = s["y"].float()
    if s["post"] is not None:
        z = _normed(z)[0] * s["post"].float()
    z = z * (s["scale"] if s["gate"] is None else s["gate"].float() * s["scale"])
    x = (s["x"].float() + z).to(s["x"].dtype)
    return x, _normed(x.float())[0] * s["weight"].float()


def _plain_norm_backward(s):
    out = {}
    dh = s["dh"].float()
    n, r = _normed(s["x"].float())
    dn = dh * s["weight"].float()
    g = s["dx"].float() + r * (dn - n * (dn * n).double().mean(dim=1, keepdim=True).float())
    out["dx"] = g.to(s["x"].dtype)
    out["dweight"] = (dh * n).double().sum(dim=0).float()
    y, post, gate = s["y"].float(), s["post"], s["gate"]
    n, r = _normed(y) if post is not None else (y, None)
    z = n * post.float() if post is not None else n
    if gate is not None:
        dgate = g * z * s["scale"]
        out["dgate"] = dgate.double().sum(dim=0).float() if gate.dim() == 1 else dgate.to(s["x"].dtype)
    dz = g * (s["scale"] if gate is None else gate.float() * s["scale"])
    if post is not None:
        out["dpost"] = (dz * n).double().sum(dim=0).float()
        dz = dz * post.float()
        dz = r * (dz - n * (dz * n).double().mean(dim=1, keepdim=True).float())
    out["dy"] = dz.to(s["x"].dtype)
    return out


def _plain(s):
    op, dtype = s["case"]["op"], getattr(torch, s["case"]["dtype"])
    if op == "quantize":
        q, scale, row = _quantized(s["x"], s["case"]["block"])
        return {"x": (_spread_scales(q, scale, s["case"]["block"]) * row).to(dtype), "row_scale": row.reshape(-1)}
    if op == "norm":
        x, h = _plain_norm(s)
        return {"x": x, "h": h.to(dtype)}
    if op == "norm_backward":
        return _plain_norm_backward(s)
    if op == "product":
        return _plain_product(s, _unpacked(s["x"]), s["x"]["row_scale"][:, None])
    x, h = (None, s["x"]) if op == "linear" else _plain_norm(s)
    q, scale, row = _quantized(h, s["case"]["block"])
    y = _plain_product(s, _spread_scales(q, scale, s["case"]["block"]), row)
    return y if x is None else {"x": x, "y": y}


def _operand(p):
    return _pkg().Fp4(p["values"], p["scales"], p["row_scale"], p["cols"], p["block"])


def run(state):
    if not own:
        return _plain(state)
    s, case, pkg = state, state["case"], _pkg()
    op, dtype = case["op"], getattr(torch, case["dtype"])
    if op == "quantize":
        q = pkg.quantize_fp4(s["x"], block=case["block"])
        return {"x": pkg.dequantize_fp4(q, dtype=dtype), "row_scale": q.row_scale}
    if op == "linear":
        return pkg.linear_fp4(s["x"], _operand(s["w"]), bias=s["bias"], residual=s["residual"])
    if op == "product":
        return pkg.gemm_fp4(_operand(s["x"]), _operand(s["w"]), bias=s["bias"], residual=s["residual"], out_dtype=dtype)
    around = dict(weight=s["weight"], post_weight=s["post"], gate=s["gate"], scale=s["scale"], eps=_EPS)
    if op == "norm":
        x, h = pkg.residual_norm(s["x"], s["y"], **around)
        return {"x": x, "h": h}
    if op == "norm_product":
        x, h = pkg.residual_norm(s["x"], s["y"], fp4=case["block"], **around)
        return {"x": x, "y": pkg.gemm_fp4(h, _operand(s["w"]), out_dtype=dtype)}
    g = pkg.residual_norm_backward(s["dh"], s["dx"], s["x"], s["y"], **around)
    out = {"dx": g.dx, "dy": g.dy, "dweight": g.dweight}
    if s["post"] is not None:
        out["dpost"] = g.dpost_weight
    if s["gate"] is not None:
        out["dgate"] = g.dgate
    return out


# ------------------------------------------------------------------ the definition, in 64 bits
def _exact_values(x, block):
    """What the 4-bit form of each row of fp64 `x` stands for, from tables of the numbers there are."""
    rows, cols = x.shape
    grid = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)
    if block == 16:
        scales = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
    else:
        scales = torch.tensor([2.0 ** i for i in range(-126, 12)], dtype=torch.float64, device=x.device)
    units = torch.tensor([2.0 ** i for i in range(-126, 118)], dtype=torch.float64, device=x.device)
    most = torch.clamp(x.abs().max(dim=1, keepdim=True).values, min=2.0 ** -116)
    unit = units[torch.searchsorted(units * 1024, most, right=True) - 1]      # the largest with 1024 unit <= most
    full = torch.zeros((rows, -(-cols // block) * block), dtype=torch.float64, device=x.device)
    full[:, :cols] = x / unit
    full = full.reshape(rows, -1, block)
    need = full.abs().max(dim=2, keepdim=True).values
    s = scales[torch.searchsorted(scales * 6, need)]
    edge = (grid[1:] + grid[:-1]) / 2
    size = full.abs()
    low = torch.zeros_like(size, dtype=torch.uint8)
    for i in range(7):                       # borders 0, 2, 4, 6 lie above an even code and stay below when hit
        at = edge[i] * s
        low += (size > at if i % 2 == 0 else size >= at).to(torch.uint8)
    value = torch.sign(full) * grid[low.int()] * s
    return value.reshape(rows, -1)[:, :cols] * unit, unit


def _exact_packed(p):
    """The numbers of a packed operand, fp64, read element by element from its bytes."""
    rows, cols, block = p["values"].shape[0], p["cols"], p["block"]
    j = torch.arange(cols, device="cuda")
    code = (p["values"][:, j // 2] >> (j % 2 * 4).to(torch.uint8)) & 15
    size = (code & 7).double()
    exponent = torch.floor(size / 2)
    powers = torch.tensor([2.0 ** i for i in range(-127, 129)], dtype=torch.float64, device="cuda")
    value = torch.where(size < 2, size / 2, (1 + (size % 2) / 2) * powers[(exponent + 126).long()])
    value = torch.where(code > 7, -value, value)
    r = torch.arange(rows, device="cuda")
    tiles = (cols + 255) // 256 * (64 // block)
    byte = p["scales"].view(-1, tiles, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, tiles * 4)[r].double()
    if block == 16:
        up = torch.floor(byte / 8)
        scale = torch.where(up > 0, (1 + (byte % 8) / 8) * powers[(up + 120).long()], byte % 8 * 2.0 ** -9)
    else:
        scale = powers[byte.long()]
    return value * scale[:, j // block] * p["row_scale"].double()[:, None]


def _exact_rms(v):
    return v / torch.sqrt((v * v).sum(dim=1, keepdim=True) / v.shape[1] + _EPS)


def _exact_stream(x, y, weight, post, gate, scale, dtype=None):
    """The residual stream after a block, rounded to its type unless that is None, and its norm."""
    z = y if post is None else _exact_rms(y) * post
    x = x + z * scale * (1.0 if gate is None else gate)
    if dtype is not None:
        x = x.to(dtype).double()
    return x, _exact_rms(x) * weight


def exact(case, seed):
    s = prepare(case, seed)
    op, dtype = case["op"], getattr(torch, case["dtype"])
    wide = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if op == "quantize":
        value, unit = _exact_values(wide["x"], case["block"])
        return {"x": value, "row_scale": unit.reshape(-1)}
    if op == "norm_backward":
        # The gradient of the definition itself, from the stream after the block as it is held.
        names = [n for n in ("y", "post", "gate") if n in wide]
        weight = wide["weight"].requires_grad_()
        x = wide["x"].requires_grad_()
        h = _exact_rms(x) * weight
        gx, gw = torch.autograd.grad(h, (x, weight), wide["dh"])
        total = gx + wide["dx"]
        del h, gx
        for n in names:
            wide[n].requires_grad_()
        z = wide["y"] if s["post"] is None else _exact_rms(wide["y"]) * wide["post"]
        t = z * s["scale"] * (1.0 if s["gate"] is None else wide["gate"])
        grads = torch.autograd.grad(t, [wide[n] for n in names], total)
        return {"dx": total.detach(), "dweight": gw, **{"d" + n: v for n, v in zip(names, grads)}}
    if op in ("norm", "norm_product"):
        x, h = _exact_stream(wide["x"], wide["y"], wide["weight"], wide.get("post"), wide.get("gate"), s["scale"], dtype)
        if op == "norm":
            return {"x": x, "h": h}
        return {"x": x, "y": _exact_values(h, case["block"])[0] @ _exact_packed(s["w"]).t()}
    a = _exact_packed(s["x"]) if op == "product" else _exact_values(wide["x"], case["block"])[0]
    y = a @ _exact_packed(s["w"]).t()
    if s["bias"] is not None:
        y += wide["bias"]
    if s["residual"] is not None:
        y += wide["residual"]
    return y
