"""The norms around a block where their statistics and coefficients are hard to hold: rows with outlying channels,
magnitudes far from one, updates in place of many rows."""
import pytest
import torch

from test_fp4_gpu import normal
from test_norm_gpu import TYPES

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
