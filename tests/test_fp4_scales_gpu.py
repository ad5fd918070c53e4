"""Products whose scales change from one step of K to the next by powers of two, so that a scale that is another step's shows in
the result."""
import pytest
import torch

from test_fp4_gpu import check_sum, stands_for

pytestmark = pytest.mark.gpu


def whole(rows, steps, seed):
    """Whole numbers up to 24: one to three times a power of two that the row's 256 elements of a step share."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randint(1, 4, (rows, steps, 256), generator=g, device="cuda") * (2 * torch.randint(0, 2, (rows, steps, 256), generator=g, device="cuda") - 1)
    return (x * 2 ** torch.randint(0, 4, (rows, steps, 1), generator=g, device="cuda")).reshape(rows, steps * 256).float()


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("cg,bn", [(2, 256), (2, 128), (1, 128), (1, 64)])
def test_scales_of_neighbouring_steps(pkg, cuda, block, cg, bn):
    for m, n, steps in ((min(bn, 500) if bn < 128 else 700, 1500, 33), (min(bn, 300), 20000, 7), (min(bn, 256), 256, 2)):
        x, w = whole(m, steps, 1), whole(n, steps, 2)
        a, b = pkg.quantize_fp4(x, block=block), pkg.quantize_fp4(w, block=block)
        # Blocks of 16 without a 3 have a scale that is no power of two (2 / 6 rounded up to 11 / 32), so sums need not be whole numbers.
        fa, fb = stands_for(a, pkg), stands_for(b, pkg)
        for _ in range(3):
            check_sum(pkg.gemm_fp4(a, b, cta_group=cg, tile_n=bn), fa, fb)
