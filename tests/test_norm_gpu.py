"""The norms around a block on the GPU against their definitions in 64 bits: forward, into a 4-bit operand,
backward (against the formulas and against differences), and a run of them with the 4-bit products."""
import pytest
import torch

from test_fp4_gpu import E2M1, check_sum, decode, normal, ref_quantize, stands_for

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
U32 = 2.0 ** -24


def half_step(t):
    fi = torch.finfo(t.dtype)
    return fi.eps / 2, fi.smallest_normal * fi.eps


def close(got, want, err):
    """|got - want| <= half a step of got's type + err."""
    rel, least = half_step(got)
    tol = rel * want.abs() + err + least
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (bad.sum().item(), ((got.double() - want).abs() / tol).max().item())


def rms(v, eps):
    return 1.0 / torch.sqrt((v * v).mean(dim=1, keepdim=True) + eps)


def case(rows, cols, dtype, post=True, gate="vector", params=None, seed=0, scale=0.5, y=True):
    params = params or dtype
    s = dict(x=normal((rows, cols), seed + 1, dtype), weight=normal((cols,), seed + 2, params, 0.3) + 1)
    if y:
        s["y"] = normal((rows, cols), seed + 3, dtype, 0.7)
        s["post"] = normal((cols,), seed + 4, params, 0.3) + 1 if post else None
        s["gate"] = {"none": None, "vector": normal((cols,), seed + 5, params, 0.5),
                     "matrix": torch.sigmoid(normal((rows, cols), seed + 6)).to(dtype)}[gate]
    else:
        s["y"] = s["post"] = s["gate"] = None
    s["scale"] = scale
    return s


def call(pkg, s, **more):
    return pkg.residual_norm(s["x"], s["y"], weight=s["weight"], post_weight=s["post"], gate=s["gate"], scale=s["scale"], **more)


def want_stream(s, eps=1e-6):
    """x_out before its rounding, and the bound of its fp32 error: r has 8 U32 from 16 fp32 additions of squares
    and one of its own, three products and the factor gate * scale one each, the sum one."""
    x = s["x"].double()
    if s["y"] is None:
        return x, torch.zeros_like(x)
    z = s["y"].double()
    if s["post"] is not None:
        z = z * rms(z, eps) * s["post"].double()
    t = z * s["scale"] * (1.0 if s["gate"] is None else s["gate"].double())
    return x + t, 14 * U32 * t.abs() + U32 * (x + t).abs()


def check_forward(pkg, s, got, eps=1e-6):
    x_out, h = got
    want, err = want_stream(s, eps)
    close(x_out, want, err)
    w = 1.0 if s["weight"] is None else s["weight"].double()
    want = x_out.double() * rms(x_out.double(), eps) * w
    close(h, want, 12 * U32 * want.abs())


SHAPES = [(1, 1), (1, 8192), (3, 7), (5, 16), (33, 255), (40, 1001), (7, 4099), (130, 512), (2, 16384), (3, 16383), (1, 9001), (300, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(pkg, cuda, dtype, rows, cols):
    for post in (True, False):
        for gate in ("none", "vector", "matrix"):
            s = case(rows, cols, dtype, post, gate, seed=rows + cols)
            check_forward(pkg, s, call(pkg, s))
    s = case(rows, cols, dtype, y=False)
    got = call(pkg, s)
    assert got[0] is s["x"]
    check_forward(pkg, s, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(3, 1001), (5, 4096), (2, 16384)])
def test_forward_fp32_weights(pkg, cuda, dtype, rows, cols):
    for gate in ("vector", "matrix"):
        s = case(rows, cols, dtype, True, gate, params=torch.float32)
        check_forward(pkg, s, call(pkg, s))
    s["weight"] = None
    check_forward(pkg, s, call(pkg, s))


@pytest.mark.parametrize("dtype", TYPES)
def test_forward_strides_and_in_place(pkg, cuda, dtype):
    for rows, cols, shift in ((9, 300, 0), (9, 301, 1), (4, 1001, 3)):
        s = case(rows, cols, dtype, True, "matrix")
        want = call(pkg, s)
        wide = {}
        for i, name in enumerate(("x", "y", "gate")):
            buf = torch.full((rows + 1, cols + 24), 7.0, dtype=dtype, device="cuda")
            wide[name] = buf[:rows, shift + i:shift + i + cols]
            wide[name].copy_(s[name])
        out = torch.full((rows + 2, cols + 9), 7.0, dtype=dtype, device="cuda")
        got = call(pkg, {**s, **wide}, out=out[1:rows + 1, 5:5 + cols])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        out[1:rows + 1, 5:5 + cols] = 7.0
        assert (out == 7.0).all()
        for name in ("x", "y"):
            t = {**s, name: s[name].clone()}
            got = call(pkg, t, out=t[name])
            assert got[0] is t[name] and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            t = {**s, name: wide[name]}
            got = call(pkg, t, out=wide[name])
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            buf = wide[name]._base
            buf[:rows, shift + ["x", "y"].index(name):][:, :cols] = 7.0
            assert (buf == 7.0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_forward_ranges(pkg, cuda, dtype):
    """Rows of zeros, of numbers whose squares leave fp32, a row with NaN and one with Inf between ordinary ones."""
    cols = 300
    s = case(8, cols, dtype, True, "none", seed=3)
    big, tiny = (6e4, 6e-8) if dtype == torch.float16 else (1e25, 1e-25)
    for name in ("x", "y"):
        s[name][1] = 0
        s[name][2] *= big / 10
        s[name][3] *= tiny * 10
    check_forward(pkg, s, call(pkg, s))
    s["x"][2:4] = s["y"][2:4] = 1.0
    s["y"][1] = 1.0
    s["x"][1] = tiny
    for eps in (0.0, 1e-12, 0.5):
        check_forward(pkg, s, call(pkg, s, eps=eps), eps)
    want = call(pkg, s)
    s["x"][4, 7], s["y"][6, 299] = float("nan"), float("inf")
    got = call(pkg, s)
    fine = [0, 1, 2, 3, 5, 7]
    for a, b in zip(got, want):
        assert torch.equal(a[fine], b[fine])
    assert got[0][4, 7].isnan() and got[1][4].isnan().all() and got[1][6].isnan().any()


def check_four_bits(f, h, block):
    """A correct 4-bit form of a matrix that differs from fp64 `h` by 12 U32 relative: row scales as for h, block scales
    the least that do, every value one of the nearest."""
    d = 12 * U32
    q, s, g = decode(f, None)
    top = h.abs().amax(dim=1)
    assert (1024 * g <= top * (1 + d)).all() and (2048 * g > top * (1 - d)).all()
    rows, cols = h.shape
    n = -(-cols // block)
    y = torch.zeros((rows, n * block), dtype=torch.float64, device="cuda")
    y[:, :cols] = h / g[:, None]
    y = y.view(rows, n, block)
    most = y.abs().amax(dim=2)
    if block == 16:
        less = torch.where(s > 2.0 ** -6, s - torch.pow(2.0, torch.floor(torch.log2(s * 0.99999999)) - 3), s - 2.0 ** -9)
    else:
        less = s / 2
    assert (6 * s >= most * (1 - d)).all() and ((6 * less < most * (1 + d)) | (s <= (2.0 ** -126 if block == 32 else 0.0))).all()
    grid = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
    full = s.repeat_interleave(block, dim=1)[:, :cols]
    y = y.view(rows, -1)[:, :cols]
    i = torch.searchsorted(grid, q.abs())
    up = torch.where(i < 7, (grid[i] + grid[(i + 1).clamp(max=7)]) / 2, 6.0 + 1e-6) * full
    down = torch.where(i > 0, (grid[i] + grid[(i - 1).clamp(min=0)]) / 2, 0.0) * full
    a = y.abs()
    assert ((a * (1 - d) <= up) & (a * (1 + d) >= down)).all()
    assert ((torch.sign(q) * torch.sign(y) >= 0)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (1, 8192), (40, 1001), (130, 512), (2, 16384), (5, 8200), (300, 33)])
def test_into_four_bits(pkg, cuda, dtype, block, rows, cols):
    for post, gate in ((True, "vector"), (False, "matrix")):
        s = case(rows, cols, dtype, post, gate)
        x_out, f = call(pkg, s, fp4=block)
        plain, _ = call(pkg, s)
        assert torch.equal(x_out, plain)
        assert f.block == block and f.cols == cols and f.values.shape == (rows, (cols + 1) // 2)
        check_four_bits(f, x_out.double() * rms(x_out.double(), 1e-6) * s["weight"].double(), block)
    s = case(rows, cols, dtype, y=False)
    _, f = call(pkg, s, fp4=block)
    check_four_bits(f, s["x"].double() * rms(s["x"].double(), 1e-6) * s["weight"].double(), block)


def test_fp32_norm_and_quantiser_agree(pkg, cuda):
    """Of fp32 rows, h as a matrix and then quantised is h as a 4-bit operand, bit for bit."""
    for rows, cols in ((50, 1000), (3, 16384)):
        s = case(rows, cols, torch.float32)
        _, h = call(pkg, s)
        for block in (16, 32):
            _, f = call(pkg, s, fp4=block)
            want = pkg.quantize_fp4(h, block=block)
            assert torch.equal(f.values, want.values) and torch.equal(f.row_scale, want.row_scale)
            assert torch.equal(decode(f, pkg)[1], decode(want, pkg)[1])


def test_four_bits_of_nan_rows(pkg, cuda):
    s = case(5, 300, torch.bfloat16)
    _, want = call(pkg, s, fp4=16)
    s["x"][3, 17] = float("nan")
    _, f = call(pkg, s, fp4=16)
    fine = [0, 1, 2, 4]
    assert torch.equal(f.values[fine], want.values[fine]) and torch.equal(f.row_scale[fine], want.row_scale[fine])
    assert f.row_scale[3].isnan() and not (f.values[3] & 0x77).any()


# ------------------------------------------------------------------ backward
def want_grads(s, dh, dx_out, x_out, eps=1e-6):
    """fp64 gradients by the formulas, and bounds of what fp32 makes of them: C U32 of the magnitudes, C = 64 for
    the operations of one element, the statistics (10) and row sums of 16 products a thread and a tree of adds."""
    n = x_out.shape[1]
    x = x_out.double()
    r = rms(x, eps)
    dn = dh.double() * (1.0 if s["weight"] is None else s["weight"].double())
    d = torch.zeros_like(x) if dx_out is None else dx_out.double()
    g = d + r * dn - x * r ** 3 * (dn * x).sum(1, keepdim=True) / n
    gs = d.abs() + r * dn.abs() + x.abs() * r ** 3 * (dn * x).abs().sum(1, keepdim=True) / n
    out = {"dx": (g, gs)}
    if s["weight"] is not None:
        out["dweight"] = ((dh.double() * x * r).sum(0), (dh.double() * x * r).abs().sum(0))
    if s["y"] is None:
        return out
    y = s["y"].double()
    k = s["scale"] * (1.0 if s["gate"] is None else s["gate"].double())
    if s["post"] is None:
        z = y
        out["dy"] = (g * k, gs * abs(k))
    else:
        wp = s["post"].double()
        q = rms(y, eps)
        z = y * q * wp
        p = k * wp * g
        out["dy"] = (q * p - y * q ** 3 * (p * y).sum(1, keepdim=True) / n,
                     q * abs(k * wp) * gs + y.abs() * q ** 3 * (abs(k * wp) * gs * y.abs()).sum(1, keepdim=True) / n)
        out["dpost_weight"] = ((g * k * y * q).sum(0), (gs * abs(k) * y.abs() * q).sum(0))
    if s["gate"] is not None:
        v, size = g * z * s["scale"], gs * z.abs() * s["scale"]
        out["dgate"] = (v.sum(0), size.sum(0)) if s["gate"].dim() == 1 else (v, size)
    return out


def check_backward(pkg, s, dh, dx_out, x_out, eps=1e-6):
    got = pkg.residual_norm_backward(dh, dx_out, x_out, s["y"], weight=s["weight"], post_weight=s["post"], gate=s["gate"],
                                     scale=s["scale"], eps=eps)
    want = want_grads(s, dh, dx_out, x_out, eps)
    rows = x_out.shape[0]
    for name in got._fields:
        v = getattr(got, name)
        assert (v is not None) == (name in want)
        if v is None:
            continue
        value, size = want[name]
        # Column sums: up to rows / 148 + 8 in a CTA, 148 of those, one after the other.
        steps = 64 if v.dim() == 2 else 64 + rows / 148 + 170
        assert v.dtype == (x_out.dtype if v.dim() == 2 else torch.float32)
        close(v, value, steps * U32 * size)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES + [(1000, 96), (500, 8192), (200, 12000)])
def test_backward(pkg, cuda, dtype, rows, cols):
    for post in (True, False):
        for gate in ("none", "vector", "matrix"):
            s = case(rows, cols, dtype, post, gate, seed=rows + cols)
            x_out, dh, dx = (normal((rows, cols), 20 + i, dtype) for i in range(3))
            check_backward(pkg, s, dh, dx, x_out)
    check_backward(pkg, s, dh, None, x_out)
    s = case(rows, cols, dtype, y=False)
    check_backward(pkg, s, dh, dx, x_out)
    s["weight"] = None
    check_backward(pkg, s, dh, dx, x_out)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [1, 16, 100, 512, 513, 1024, 2000])
def test_many_short_rows(pkg, cuda, dtype, cols):
    """As many groups to a block as there can be."""
    rows = 148 * 33 + 5
    for gate in ("vector", "matrix"):
        s = case(rows, cols, dtype, True, gate)
        x_out, dh, dx = (normal((rows, cols), 20 + i, dtype) for i in range(3))
        check_forward(pkg, s, call(pkg, s))
        check_backward(pkg, s, dh, dx, x_out)
    _, f = call(pkg, s, fp4=32)
    x_out, _ = call(pkg, s)
    check_four_bits(f, x_out.double() * rms(x_out.double(), 1e-6) * s["weight"].double(), 32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(30, 1001), (170, 8192), (20, 16384)])
def test_backward_fp32_weights(pkg, cuda, dtype, rows, cols):
    s = case(rows, cols, dtype, True, "vector", params=torch.float32)
    x_out, dh, dx = (normal((rows, cols), 20 + i, dtype) for i in range(3))
    check_backward(pkg, s, dh, dx, x_out)


def test_backward_strides(pkg, cuda):
    rows, cols = 50, 333
    for dtype in TYPES:
        s = case(rows, cols, dtype, True, "matrix")
        x_out, dh, dx = (normal((rows, cols + 7), 20 + i, dtype)[:, i:i + cols] for i in range(3))
        s["y"] = normal((rows, cols + 4), 3, dtype)[:, 3:3 + cols]
        check_backward(pkg, s, dh, dx, x_out)


def test_backward_ranges(pkg, cuda):
    """Rows of zeros, squares that leave fp32, and rows with NaN: no other row's dx and dy is touched."""
    for dtype in TYPES:
        s = case(6, 300, dtype)
        x_out, dh, dx = (normal((6, 300), 20 + i, dtype) for i in range(3))
        x_out[1] = s["y"][2] = 0
        x_out[4] *= 1e3 if dtype == torch.float16 else 1e20
        want = check_backward(pkg, s, dh, dx, x_out)
        dh[3, 5] = float("nan")
        got = pkg.residual_norm_backward(dh, dx, x_out, s["y"], weight=s["weight"], post_weight=s["post"], gate=s["gate"], scale=s["scale"])
        fine = [0, 1, 2, 4, 5]
        assert torch.equal(got.dx[fine], want.dx[fine]) and torch.equal(got.dy[fine], want.dy[fine])
        assert got.dx[3].isnan().all()


def test_backward_is_the_derivative(pkg, cuda):
    """Directional derivatives of the forward call: central differences of a weighted sum of its outputs."""
    rows, cols = 6, 200
    for post, gate in ((True, "vector"), (True, "matrix"), (False, "vector"), (True, "none")):
        s = case(rows, cols, torch.float32, post, gate)
        gx, gh = normal((rows, cols), 30), normal((rows, cols), 31)

        def loss(t):
            x_out, h = call(pkg, t)
            return (x_out.double() * gx.double()).sum() + (h.double() * gh.double()).sum()

        grads = pkg.residual_norm_backward(gh, gx, call(pkg, s)[0], s["y"], weight=s["weight"], post_weight=s["post"], gate=s["gate"], scale=s["scale"])
        for name, grad in (("x", grads.dx), ("y", grads.dy), ("weight", grads.dweight), ("post", grads.dpost_weight), ("gate", grads.dgate)):
            if s[name] is None:
                assert grad is None
                continue
            v = normal(tuple(s[name].shape), 40)
            step = 2.0 ** -7
            moved = [loss({**s, name: s[name] + sign * step * v}) for sign in (1, -1)]
            want = (moved[0] - moved[1]).item() / (2 * step)
            got = (grad.double() * v.double()).sum().item()
            # Third derivatives of order one times step^2 / 6 = 1e-5, and fp32 outputs (1e-7 of some 50) over the step.
            size = (grad.double() * v.double()).abs().sum().item()
            assert abs(got - want) <= 1e-3 * size ** 0.5 + 1e-4 * size, (name, got, want, size)


def test_backward_is_the_same_twice(pkg, cuda):
    s = case(700, 1000, torch.bfloat16)
    x_out, dh, dx = (normal((700, 1000), 20 + i, torch.bfloat16) for i in range(3))
    one, two = (pkg.residual_norm_backward(dh, dx, x_out, s["y"], weight=s["weight"], post_weight=s["post"], gate=s["gate"]) for _ in range(2))
    for a, b in zip(one, two):
        assert torch.equal(a, b)


def test_empty(pkg, cuda):
    s = case(0, 50, torch.bfloat16)
    x_out, h = call(pkg, s)
    assert x_out.shape == h.shape == (0, 50)
    g = pkg.residual_norm_backward(s["x"], s["x"], s["x"], s["y"], weight=s["weight"], post_weight=s["post"], gate=s["gate"])
    assert g.dx.shape == (0, 50) and all((v == 0).all() and v.shape == (50,) for v in (g.dweight, g.dpost_weight, g.dgate))


# ------------------------------------------------------------------ a run of them
def test_a_block_of_four_bit_layers(pkg, cuda):
    """Norm into 4 bits, up projection, down projection with its tokens quantised inside, norm after: each step against
    its definition on the step before it; one token and many, eager and from a graph."""
    k, n = 1024, 1400
    up, down = (pkg.quantize_fp4(normal(s, i, scale=0.03)) for i, s in enumerate(((n, k), (k, n))))
    w, wp = (normal((k,), i, torch.bfloat16, 0.2) + 1 for i in (5, 6))
    for m in (1, 6, 300):
        x, y = normal((m, k), 7, torch.bfloat16), normal((m, k), 8, torch.bfloat16)

        def block():
            x1, h = pkg.residual_norm(x, y, weight=w, post_weight=wp, fp4=16)
            a = pkg.gemm_fp4(h, up)
            b = pkg.linear_fp4(a, down)
            x2, o = pkg.residual_norm(x1, b, weight=w, post_weight=wp)
            return x1, h, a, b, x2, o

        x1, h, a, b, x2, o = block()
        s = dict(x=x, y=y, weight=w, post=wp, gate=None, scale=1.0)
        close(x1, *want_stream(s))
        check_four_bits(h, x1.double() * rms(x1.double(), 1e-6) * w.double(), 16)
        check_sum(a, stands_for(h, pkg), stands_for(up, pkg))
        q, sc, g = ref_quantize(a, 16)
        check_sum(b, q * sc.repeat_interleave(16, dim=1)[:, :n] * g[:, None], stands_for(down, pkg))
        check_forward(pkg, {**s, "x": x1, "y": b}, (x2, o))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            again = block()
        x.copy_(normal((m, k), 9, torch.bfloat16))
        graph.replay()
        for u, v in zip(again, block()):
            if isinstance(u, torch.Tensor):
                assert torch.equal(u, v)


def test_training_calls_in_a_graph(pkg, cuda):
    s = case(64, 500, torch.bfloat16)
    dh, dx = normal((64, 500), 20, torch.bfloat16), normal((64, 500), 21, torch.bfloat16)

    def both():
        x_out, h = call(pkg, s)
        return (x_out, h, *pkg.residual_norm_backward(dh, dx, x_out, s["y"], weight=s["weight"], post_weight=s["post"], gate=s["gate"], scale=0.5))

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    s["x"].copy_(normal((64, 500), 33, torch.bfloat16))
    graph.replay()
    for u, v in zip(got, both()):
        assert torch.equal(u, v)


def test_two_streams(pkg, cuda):
    cases = [case(300, 1000, torch.bfloat16, seed=i) for i in range(2)]
    grads = [(normal((300, 1000), 50, torch.bfloat16), normal((300, 1000), 51, torch.bfloat16))] * 2

    def both(s, g):
        x_out, h = call(pkg, s)
        return (x_out, h, *pkg.residual_norm_backward(g[0], g[1], x_out, s["y"], weight=s["weight"], post_weight=s["post"], gate=s["gate"], scale=0.5))

    want = [both(s, g) for s, g in zip(cases, grads)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(both(cases[i], grads[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))


def test_operands_that_are_one_tensor(pkg, cuda):
    """The same matrix as x, y and gate, and replaced in place; the same vector everywhere."""
    for cols in (512, 1001):
        x, w = normal((200, cols), 1, torch.bfloat16), normal((cols,), 2, torch.bfloat16, 0.2) + 1
        want = pkg.residual_norm(x, x.clone(), weight=w, post_weight=w.clone(), gate=x.clone())
        got = pkg.residual_norm(x, x, weight=w, post_weight=w, gate=x)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        want = pkg.residual_norm(x, x.clone(), weight=w, post_weight=w)
        z = x.clone()
        got = pkg.residual_norm(z, z, weight=w, post_weight=w, out=z)
        assert got[0] is z and torch.equal(z, want[0]) and torch.equal(got[1], want[1])
        with pytest.raises(pkg.GemmError):
            pkg.residual_norm(x, x, weight=w, gate=z, out=z)
        a = pkg.residual_norm_backward(x, x, x, x, weight=w, post_weight=w, gate=x)
        b = pkg.residual_norm_backward(x.clone(), x.clone(), x.clone(), x.clone(), weight=w, post_weight=w, gate=x.clone())
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_offsets_beyond_32_bits(pkg, cuda):
    """The last rows of matrices of more than 2^31 elements are those of a small call."""
    rows, cols = 131080, 16392 - 8
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
    x[-3:] = normal((3, cols), 1, torch.bfloat16)
    w = normal((cols,), 2, torch.bfloat16, 0.2) + 1
    want = pkg.residual_norm(x[-3:], x[-3:].clone(), weight=w, post_weight=w)
    grads = pkg.residual_norm_backward(x[-3:], x[-3:], x[-3:], x[-3:], weight=w, post_weight=w)
    got = pkg.residual_norm_backward(x, x, x, x, weight=w, post_weight=w)
    size = grads.dx.float().abs().max()
    assert (got.dx[-3:].float() - grads.dx.float()).abs().max() <= 2 ** -7 * size and (got.dy[-3:].float() - grads.dy.float()).abs().max() <= 2 ** -7 * grads.dy.float().abs().max()
    assert (got.dweight - grads.dweight).abs().max() <= 1e-5 * grads.dweight.abs().max()
    del got
    got = pkg.residual_norm(x, x, weight=w, post_weight=w, out=x)
    assert (x[-3:].float() - want[0].float()).abs().max() <= 2 ** -7 * want[0].float().abs().max()
    assert (got[1][-3:].float() - want[1].float()).abs().max() <= 2 ** -7 * want[1].float().abs().max() and not got[1][:100].any()


def test_refusals_in_python(pkg, cuda):
    s = case(4, 64, torch.bfloat16)
    x, y, w = s["x"], s["y"], s["weight"]
    for run, error in [
        (lambda: pkg.residual_norm(x, y[:3], weight=w), "shape"),
        (lambda: pkg.residual_norm(x, y.float(), weight=w), "BFloat16"),
        (lambda: pkg.residual_norm(x, weight=w[:60]), "weight"),
        (lambda: pkg.residual_norm(x, weight=w.half()), "x's type or be float32"),
        (lambda: pkg.residual_norm(x, y, weight=w, post_weight=w.float()), "one type"),
        (lambda: pkg.residual_norm(x, gate=w), "need y"),
        (lambda: pkg.residual_norm(x, post_weight=w), "need y"),
        (lambda: pkg.residual_norm(x, out=x), "need y"),
        (lambda: pkg.residual_norm(x, y, gate=x[:1].expand(4, 64)), "overlapping"),
        (lambda: pkg.residual_norm(x, y, gate=x.float()), "gate"),
        (lambda: pkg.residual_norm(x, fp4=8), "fp4"),
        (lambda: pkg.residual_norm(x.t()), "unit stride"),
        (lambda: pkg.residual_norm_backward(x[:2], None, x), "shape"),
        (lambda: pkg.residual_norm_backward(x, None, x, gate=w), "need y"),
    ]:
        with pytest.raises(ValueError, match=error):
            run()
    buf = torch.zeros((5, 64), dtype=torch.bfloat16, device="cuda")
    for run in (lambda: pkg.residual_norm(torch.zeros((2, 16385), device="cuda")),
                lambda: pkg.residual_norm(x, eps=-1.0),
                lambda: pkg.residual_norm(x, eps=float("nan")),
                lambda: pkg.residual_norm(buf[:4], y, out=buf[1:]),
                lambda: pkg.residual_norm(torch.zeros((2, 0), device="cuda"))):
        with pytest.raises(pkg.GemmError):
            run()
