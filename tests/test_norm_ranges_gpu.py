"""The norms around a block where their statistics and coefficients are hard to hold: rows with outlying channels,
magnitudes far from one, updates in place of many rows."""
import pytest
import torch

from test_fp4_gpu import normal
from test_norm_gpu import TYPES, case, check_backward

pytestmark = pytest.mark.gpu

HALVES = [torch.bfloat16, torch.float16]


def uneven(rows, cols, seed, dtype, kind):
    x = normal((rows, cols), seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 99)
    if kind == "some":
        x *= torch.where(torch.rand((cols,), generator=g, device="cuda") > 0.995, 8.0, 1.0)
    elif kind == "channel":
        x[:, cols // 3] *= 100.0
    elif kind == "one":
        x[:, cols // 2] = 3000.0
    elif kind == "spread":
        x *= 2.0 ** torch.randint(-12, 13, (rows, cols), generator=g, device="cuda").float()
    return x.to(dtype)


def inverse_roots(v, eps):
    """fp32 1 / sqrt(mean v^2 + eps) of 16-bit rows, from below and from above: the mean is held to 2^-40, its inverse
    root to half of that and 2^-43 of its own, so that both are the same but next to the middle of two fp32 numbers."""
    r = 1.0 / torch.sqrt((v.double() ** 2).mean(dim=1, keepdim=True) + eps)
    return (r * (1 - 2.0 ** -36)).float(), (r * (1 + 2.0 ** -36)).float()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("kind", ["even", "some", "channel", "one", "spread"])
@pytest.mark.parametrize("rows,cols", [(500, 8192), (9, 8192), (300, 1000), (200, 16384), (700, 24), (600, 4001)])
def test_statistics_of_uneven_rows(pkg, cuda, dtype, kind, rows, cols):
    """x_out, h and its 4-bit form from statistics in 64 bits and one fp32 operation after the other: equal."""
    y = uneven(rows, cols, rows + cols, dtype, kind)
    x = torch.zeros_like(y)
    w, wp = (normal((cols,), i, torch.float32, 0.3) + 1 for i in (2, 3))
    x_out, h = pkg.residual_norm(x, y, weight=w, post_weight=wp)
    ways = [(y.float() * q * wp).to(dtype) for q in inverse_roots(y, 1e-6)]
    assert ((x_out == ways[0]) | (x_out == ways[1])).all(), (x_out != ways[0]).sum().item()
    exact = [x_out.float() * r * w for r in inverse_roots(x_out, 1e-6)]
    ways = [e.to(dtype) for e in exact]
    assert ((h == ways[0]) | (h == ways[1])).all(), (h != ways[0]).sum().item()
    for block in (16, 32):
        again, f = pkg.residual_norm(x, y, weight=w, post_weight=wp, fp4=block)
        assert torch.equal(again, x_out)
        ways = [pkg.quantize_fp4(e, block=block) for e in exact]
        assert ((f.values == ways[0].values).all(1) | (f.values == ways[1].values).all(1)).all()
        assert ((f.row_scale == ways[0].row_scale) | (f.row_scale == ways[1].row_scale)).all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("rows,cols", [(300, 16384), (300, 14337), (300, 13313), (170, 12288), (90, 1001), (4, 8192)])
def test_the_gate_comes_after_the_weight(pkg, cuda, dtype, wide, rows, cols):
    """z times gate * scale in that order for every number of columns, also where weight times gate leaves fp32's range."""
    y = normal((rows, cols), 5, dtype)
    x = torch.zeros_like(y)
    wp, gate = (normal((cols,), i, torch.float32 if wide else dtype, 0.3) + 1 for i in (3, 4))
    if wide:
        y[:, 7] *= 2.0 ** -13
        wp[7], gate[7] = 1e20, 1e20 if dtype == torch.bfloat16 else 1e-16
        gate[8], wp[9] = 1e-30, 1e-20
    for shift in (0, 1):      # vectors off 16-byte boundaries
        v = [torch.nn.functional.pad(t, (shift, 0))[shift:] for t in (wp, gate)]
        x_out, _ = pkg.residual_norm(x, y, post_weight=v[0], gate=v[1], scale=0.3)
        k = gate.float() * torch.tensor(0.3, device="cuda")
        ways = [(((y.float() * q) * wp.float()) * k).to(dtype) for q in inverse_roots(y, 1e-6)]
        assert ((x_out == ways[0]) | (x_out == ways[1])).all(), (x_out != ways[0]).sum().item()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gate", ["vector", "matrix", "none"])
@pytest.mark.parametrize("rows,cols", [(900, 4096), (700, 1001), (5, 8192), (200, 16384)])
def test_the_product_is_rounded_before_the_sum(pkg, cuda, dtype, gate, rows, cols):
    s = case(rows, cols, dtype, False, gate)
    k = torch.tensor(0.3, device="cuda") * (1.0 if s["gate"] is None else s["gate"].float())
    x_out, _ = pkg.residual_norm(s["x"], s["y"], gate=s["gate"], scale=0.3)
    assert torch.equal(x_out, (s["x"].float() + s["y"].float() * k).to(dtype))


# ------------------------------------------------------------------ gradients of rows far from one
FAR = [1.0, 1e14, 1e16, 1e20, 1e-13, 1e-20]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(72, 1000), (180, 304), (36, 9000), (36, 24)])
@pytest.mark.parametrize("eps", [1e-6, 0.0, 1e-30, 0.5])
def test_gradients_of_rows_far_from_one(pkg, cuda, dtype, rows, cols, eps):
    """Rows of x_out and of y in every pair of magnitudes, within the bounds of ordinary rows: gradients of h about as
    large as x_out (so that dx is about one where eps does not outweigh the row), and about one; with and without a gradient of x_out."""
    far = torch.tensor(FAR, device="cuda").repeat((rows + 5) // 6)[:rows, None]
    other = torch.tensor(FAR, device="cuda").repeat_interleave(6).repeat((rows + 35) // 36)[:rows, None]
    for gate, post in (("vector", True), ("matrix", True), ("none", False)):
        s = case(rows, cols, dtype, post, gate, params=torch.float32)
        s["y"] = (normal((rows, cols), 3) * other).to(dtype)
        x_out = (normal((rows, cols), 20) * far).to(dtype)
        dh = normal((rows, cols), 21)
        check_backward(pkg, s, (dh * far).to(dtype), None, x_out, eps)
        check_backward(pkg, s, (dh * far).to(dtype), normal((rows, cols), 22, dtype), x_out, eps)
        # dh about one: r dh y's way leaves the type where both rows are small and eps too.
        if eps > 1e-9:
            check_backward(pkg, s, dh.to(dtype), None, x_out, eps)
            check_backward(pkg, s, dh.to(dtype), (normal((rows, cols), 22) / far.clamp(min=1.0)).to(dtype), x_out, eps)


@pytest.mark.parametrize("rows,cols", [(9, 700), (200, 700), (4, 10000)])
def test_gradients_of_far_fp16_rows(pkg, cuda, rows, cols):
    """The ends of fp16, with an eps that outweighs none of it."""
    far = torch.tensor([1.0, 1e4, 2e-6], device="cuda").repeat(rows)[:rows, None]
    for eps in (0.0, 1e-6):
        s = case(rows, cols, torch.float16, True, "vector", scale=2.0 ** -10)
        s["y"] = (normal((rows, cols), 3) * far.flip(0)).clamp(-6e4, 6e4).half()
        x_out = (normal((rows, cols), 20) * far).clamp(-6e4, 6e4).half()
        check_backward(pkg, s, (normal((rows, cols), 21) * far * 2.0 ** -6).clamp(-6e4, 6e4).half(), None, x_out, eps)


def test_large_gradients_of_ordinary_rows(pkg, cuda):
    """Row sums that leave fp32 though the rows' squares do not."""
    s = case(3, 600, torch.float32)
    x_out, dh = normal((3, 600), 20) * 1e8, normal((3, 600), 21)
    dh[1] *= 1e32
    check_backward(pkg, s, dh, None, x_out)


# ------------------------------------------------------------------ many rows in place
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(5000, 512), (4001, 1001), (3000, 4096), (1200, 8192), (700, 16384), (20000, 24)])
def test_many_rows_in_place(pkg, cuda, dtype, rows, cols):
    """Groups that walk down many rows with the coming ones copied ahead: x_out over x or y, aligned and off 16-byte
    boundaries, is that of a call apart."""
    s = case(rows, cols, dtype, True, "vector")
    for shift in (0, 3):
        for name in ("x", "y"):
            store = torch.full((rows + 1, cols + 8 + shift), 7.0, dtype=dtype, device="cuda")
            t = dict(x=s["x"], y=s["y"])
            t[name] = store[:rows, shift:shift + cols]
            t[name].copy_(s[name])
            around = dict(weight=s["weight"], post_weight=s["post"], gate=s["gate"], scale=0.5)
            want = pkg.residual_norm(t["x"], t["y"], **around)
            want4 = pkg.residual_norm(t["x"], t["y"], fp4=16, **around)[1]
            got = pkg.residual_norm(t["x"], t["y"], out=t[name], **around)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            t[name].copy_(s[name])
            _, four = pkg.residual_norm(t["x"], t["y"], fp4=16, out=t[name], **around)
            assert torch.equal(t[name], want[0])
            assert torch.equal(four.values, want4.values) and torch.equal(four.row_scale, want4.row_scale)
            store[:rows, shift:shift + cols] = 7.0
            assert (store == 7.0).all()
