"""Tensors that a call overwrites count as changed: autograd refuses to use what it had saved of them."""
import pytest
import torch

from test_fp4_gpu import normal

pytestmark = pytest.mark.gpu


def overwriting(pkg, w8, w4, t):
    """Calls that write `t`, bf16 (64, 64)."""
    x = normal((64, 64), 2, torch.bfloat16)
    return [
        lambda: pkg.residual_norm(x, x, out=t),
        lambda: pkg.residual_norm(t, x, out=t, fp4=16),
        lambda: pkg.linear_fp4(x, w4, out=t),
        lambda: pkg.gemm_fp4(pkg.quantize_fp4(x), w4, out=t),
        lambda: pkg.dequantize_fp4(w4, out=t),
        lambda: pkg.linear_int8(x, *w8, out=t),
        lambda: pkg.dropout(x, pkg.Dropout(0.5, 1), out=t),
    ]


@pytest.mark.parametrize("which", range(7))
def test_outputs_raise_their_version(pkg, cuda, which):
    w = normal((64, 64), 1, torch.bfloat16)
    w8, w4 = pkg.quantize_int8(w), pkg.quantize_fp4(w)
    leaf = normal((64, 64), 3, torch.bfloat16).requires_grad_()
    t = leaf * 2
    loss = (t * t).sum()
    before = t._version
    overwriting(pkg, w8, w4, t.detach())[which]()
    assert t._version > before
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    with torch.inference_mode():
        t = normal((64, 64), 3, torch.bfloat16) * 2
        overwriting(pkg, w8, w4, t)[which]()


def test_a_norm_without_a_block_changes_nothing(pkg, cuda):
    x = normal((8, 64), 3, torch.bfloat16)
    before = x._version
    assert pkg.residual_norm(x)[0] is x and x._version == before
