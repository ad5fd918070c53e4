"""The 4-bit operators on the GPU against their definitions in 64 bits: the quantiser (exact), its way
back (exact), the product and its epilogue in every tile and split, and the linear layer."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
HALVES = [torch.bfloat16, torch.float16]
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
U32 = 2.0 ** -24


# ------------------------------------------------------------------ the definitions, in 64 bits
def powers(low, high):
    return torch.tensor([2.0 ** i for i in range(low, high)], dtype=torch.float64, device="cuda")


def ref_quantize(x, block):
    """Values, block scales and row scales (fp64) of finite rows."""
    x = x.double()
    rows, cols = x.shape
    unit = powers(-126, 118)
    top = x.abs().amax(dim=1).clamp(min=2.0 ** -116)
    g = unit[torch.searchsorted(unit * 1024, top, right=True) - 1]
    n = -(-cols // block)
    y = torch.zeros((rows, n * block), dtype=torch.float64, device="cuda")
    y[:, :cols] = (x / g[:, None]).float()       # exact, but for numbers below 2^-126
    y = y.view(rows, n, block)
    if block == 16:
        grid = torch.arange(127, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()
    else:
        grid = powers(-126, 12)
    s = grid[torch.searchsorted(grid * 6, y.abs().amax(dim=2))]
    e2m1 = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
    edges = (e2m1[1:] + e2m1[:-1]) / 2
    code = torch.zeros(y.shape, dtype=torch.int64, device="cuda")
    for i in range(7):
        at = edges[i] * s[:, :, None]
        code += (y.abs() > at) if i % 2 == 0 else (y.abs() >= at)
    q = torch.sign(y) * e2m1[torch.where(s[:, :, None] > 0, code, 0)]
    return q.view(rows, -1)[:, :cols], s, g


def decode(f, pkg):
    """Values, block scales and row scales (fp64) of an Fp4, from its bytes."""
    rows = f.values.shape[0]
    code = torch.stack((f.values & 15, f.values >> 4), dim=2).reshape(rows, -1)[:, :f.cols].long()
    e2m1 = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device="cuda")
    tiles = (f.cols + 255) // 256 * 64 // f.block
    r = torch.arange(rows, device="cuda")[:, None]
    c = torch.arange((f.cols + f.block - 1) // f.block, device="cuda")[None, :]
    byte = f.scales[(r // 128 * tiles + c // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + c % 4].contiguous()
    s = byte.view(torch.float8_e4m3fn).double() if f.block == 16 else powers(-127, 128)[byte.long()]
    return e2m1[code], s, f.row_scale.double()


def stands_for(f, pkg):
    q, s, g = decode(f, pkg)
    return q * s.repeat_interleave(f.block, dim=1)[:, :f.cols] * g[:, None]


def normal(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def check_sum(got, a, b, bias=None, residual=None):
    """|got - want| <= half a step of got's type + the tensor cores' sum (each of the steps of 64 along K leaves at
    most a step of fp32 of the magnitudes added so far, a few more where parts of a split are added) + the four fp32
    operations of the epilogue.  a, b: fp64 matrices."""
    want = a @ b.t()
    size = a.abs() @ b.abs().t()
    steps = a.shape[1] / 64 + 16
    err = size * steps * 2 * U32
    if bias is not None:
        want = want + bias.double()
        size = size + bias.double().abs()
    if residual is not None:
        want = want + residual.double()
        size = size + residual.double().abs()
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * want.abs() + err + 4 * U32 * size + fi.smallest_normal * fi.eps
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (bad.sum().item(), ((got.double() - want).abs() / tol).max().item())


# ------------------------------------------------------------------ quantiser
def check_quantized(f, x, pkg):
    assert f.cols == x.shape[1] and f.values.stride(0) % 16 == 0
    q, s, g = decode(f, pkg)
    want_q, want_s, want_g = ref_quantize(x, f.block)
    assert torch.equal(g, want_g)
    assert torch.equal(s, want_s)
    assert torch.equal(q, want_q)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (1, 16), (5, 33), (2, 255), (33, 257), (129, 1000), (300, 128), (2, 40001), (1, 70000)])
def test_quantize_exact(pkg, cuda, dtype, block, rows, cols):
    x = normal((rows, cols), rows * 7 + cols, dtype, 3.0)
    check_quantized(pkg.quantize_fp4(x, block=block), x, pkg)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(148 * 40, 600), (20000, 250), (3000, 1024), (400, 8192), (300, 8193), (200, 20000), (160, 32768), (150, 40000)])
def test_quantize_many_rows(pkg, cuda, dtype, rows, cols):
    """Rows that groups of threads go down, with as many groups to a block as there can be."""
    x = normal((rows, cols), rows + cols, dtype, 3.0)
    check_quantized(pkg.quantize_fp4(x, block=16 if rows % 3 else 32), x, pkg)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_borders(pkg, cuda, dtype, block):
    """Values on the borders between codes under every block scale, one step beside them, and block maxima that
    are exactly six times a scale: the first element fixes the row's scale, the second of a block its own."""
    step = torch.finfo(dtype).eps
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    rows = []
    for m in range(8):                                     # significands 8/8 .. 15/8 of an e4m3 scale
        for e in (-9, -3, 0, 4):
            s = (1 + m / 8) * 2.0 ** e
            for bump in (0.0, step, -step):
                row = torch.zeros(16 * block, dtype=torch.float64)
                row[0] = 1024.0
                for b in range(1, 8):
                    row[b * block] = 6 * s * (1 + (bump if b > 3 else 0.0))
                    for j, mid in enumerate(mids):
                        row[b * block + 1 + j] = mid * s * (1 + bump) * (-1) ** b
                rows.append(row)
    x = torch.stack(rows).cuda().to(dtype)
    check_quantized(pkg.quantize_fp4(x, block=block), x, pkg)


@pytest.mark.parametrize("block", [16, 32])
def test_quantize_far_ranges(pkg, cuda, block):
    """Zeros, subnormals, the largest numbers, and rows whose elements are far apart."""
    rows = [torch.zeros(100), torch.full((100,), 2.0 ** -149), torch.full((100,), 3.4e38), torch.full((100,), -(2.0 ** -130)),
            torch.logspace(-45, 38, 100), -torch.logspace(-45, 38, 100), torch.tensor([1e-30] * 99 + [1e30])]
    x = torch.stack([r.float() for r in rows]).cuda()
    check_quantized(pkg.quantize_fp4(x, block=block), x, pkg)
    x = x.bfloat16()
    x = torch.where(x.isinf(), 3e38, x)
    check_quantized(pkg.quantize_fp4(x, block=block), x, pkg)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_nan_and_inf_keep_to_their_rows(pkg, cuda, dtype, block):
    x = normal((6, 300), 1, dtype)
    x[1, 7], x[3, 299], x[4, 0] = float("nan"), float("inf"), float("-inf")
    f = pkg.quantize_fp4(x, block=block)
    fine = torch.tensor([0, 2, 5], device="cuda")
    q, s, g = decode(f, pkg)
    want_q, want_s, want_g = ref_quantize(x[fine], block)
    assert torch.equal(q[fine], want_q) and torch.equal(s[fine], want_s) and torch.equal(g[fine], want_g)
    assert g[1].isnan() and g[3].isinf() and g[4].isinf() and not q[[1, 3, 4]].any()
    w = pkg.quantize_fp4(normal((40, 300), 2), block=block)
    y = pkg.gemm_fp4(f, w)
    assert y[[1, 3, 4]].isnan().all() and y[fine].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_strided_rows_and_odd_bases(pkg, cuda, dtype):
    base = normal((50, 333), 3, dtype)
    for x in (base[:, 5:300], base[1::3, :77], base.view(-1)[1:1 + 40 * 333].view(40, 333)):
        check_quantized(pkg.quantize_fp4(x), x, pkg)


def test_bytes_behind_a_row_are_left(pkg, cuda):
    """Through the C ABI: a buffer with room behind each row and behind the last scale tile."""
    import ctypes as C
    for cols, block in ((7, 16), (250, 32), (257, 16)):
        x = normal((5, cols), cols, torch.bfloat16)
        ld = (cols + 1) // 2 // 16 * 16 + 32
        values = torch.full((6, ld), 0xAA, dtype=torch.uint8, device="cuda")
        need = pkg.fp4_scale_bytes(5, cols, block)
        scales = torch.full((need + 64,), 0xAA, dtype=torch.uint8, device="cuda")
        rows = torch.full((8,), 7.0, device="cuda")
        a = pkg.Fp4QuantArgs(C.sizeof(pkg.Fp4QuantArgs), 0, 5, cols, x.data_ptr(), cols, values.data_ptr(), ld, scales.data_ptr(),
                             rows.data_ptr(), block, 0)
        assert pkg.lib().gemm_sm100a_quantize_fp4(bytes(a), None) == pkg.OK
        torch.cuda.synchronize()
        assert (values[:5, (cols + 1) // 2:] == 0xAA).all() and (values[5] == 0xAA).all()
        assert (scales[need:] == 0xAA).all() and (rows[5:] == 7.0).all()
        check_quantized(pkg.Fp4(values[:5, :(cols + 1) // 2], scales, rows[:5], cols, block), x, pkg)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 33), (130, 1000), (3, 20001)])
def test_dequantize(pkg, cuda, dtype, block, rows, cols):
    x = normal((rows, cols), rows + cols, torch.float32, 2.0)
    f = pkg.quantize_fp4(x, block=block)
    want = stands_for(f, pkg).to(dtype)
    assert torch.equal(pkg.dequantize_fp4(f, dtype=dtype), want)
    out = torch.full((rows, cols + 3), 5.0, dtype=dtype, device="cuda")
    pkg.dequantize_fp4(f, out=out[:, 1:cols + 1])
    assert torch.equal(out[:, 1:cols + 1], want) and (out[:, 0] == 5).all() and (out[:, cols + 1:] == 5).all()
    plain = pkg.dequantize_fp4(f._replace(row_scale=None), dtype=torch.float32)
    assert torch.equal(plain.double() * f.row_scale.double()[:, None], stands_for(f, pkg))


# ------------------------------------------------------------------ product
KNOBS = [dict()] + [dict(cta_group=1, tile_n=bn, split_k=s) for bn in (16, 32, 64, 128) for s in (1, 2, 4)] + \
        [dict(cta_group=2, tile_n=bn) for bn in (128, 256)]


def operands(pkg, m, n, k, block, seed=0, dtype=torch.float32):
    a = pkg.quantize_fp4(normal((m, k), seed + 1, dtype), block=block)
    b = pkg.quantize_fp4(normal((n, k), seed + 2, dtype, 0.05), block=block)
    return a, b, stands_for(a, pkg), stands_for(b, pkg)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("knobs", KNOBS)
def test_product_tiles(pkg, cuda, block, knobs):
    for m, n, k in ((13, 200, 1100), (16, 128, 1024), (1, 1, 1025)):
        a, b, fa, fb = operands(pkg, m, n, k, block)
        check_sum(pkg.gemm_fp4(a, b, **knobs), fa, fb)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("knobs", [k for k in KNOBS if k.get("tile_n", 0) not in (16, 32, 64)])
def test_product_many_tiles(pkg, cuda, block, knobs):
    for m, n, k in ((700, 520, 2000), (257, 1025, 600)):
        if knobs.get("split_k", 1) > -(-k // 256):      # refused: no more parts than blocks of K
            continue
        a, b, fa, fb = operands(pkg, m, n, k, block)
        for dtype in HALVES:
            check_sum(pkg.gemm_fp4(a, b, out_dtype=dtype, **knobs), fa, fb)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("cg,bn", [(1, 16), (1, 32), (1, 64), (1, 128), (2, 128), (2, 256)])
def test_each_scale_reaches_its_elements(pkg, cuda, block, cg, bn):
    """One non-zero element per token and channel: every output is one product of known scales, exact."""
    m, n, k = min(bn, 250), 300, 700
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    x = torch.zeros((m, k), device="cuda")
    w = torch.zeros((n, k), device="cuda")
    pick = torch.randint(0, k, (m,), generator=g, device="cuda")
    x[torch.arange(m, device="cuda"), pick] = 2.0 ** torch.randint(-3, 4, (m,), generator=g, device="cuda").float()
    w.copy_(2.0 ** torch.randint(-6, 7, (n, k), generator=g, device="cuda").float())
    a, b = pkg.quantize_fp4(x, block=block), pkg.quantize_fp4(w, block=block)
    want = stands_for(a, pkg) @ stands_for(b, pkg).t()
    got = pkg.gemm_fp4(a, b, cta_group=cg, tile_n=bn)
    assert torch.equal(got.double(), want.to(torch.bfloat16).double())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n", [264, 301])
@pytest.mark.parametrize("m", [3, 100, 300])
@pytest.mark.parametrize("knobs", [dict(), dict(cta_group=1, tile_n=128), dict(cta_group=1, tile_n=128, split_k=2), dict(cta_group=2, tile_n=256)])
def test_bias_and_residual(pkg, cuda, dtype, n, m, knobs):
    a, b, fa, fb = operands(pkg, m, n, 777, 16)
    residual = normal((m, n), 5, dtype)
    for bias_type in TYPES:
        bias = normal((n,), 6, bias_type)
        check_sum(pkg.gemm_fp4(a, b, bias=bias, residual=residual, out_dtype=dtype, **knobs), fa, fb, bias, residual)
    inplace = residual.clone()
    out = pkg.gemm_fp4(a, b, residual=inplace, out=inplace, **knobs)
    assert out is inplace
    assert torch.equal(out, pkg.gemm_fp4(a, b, residual=residual, out_dtype=dtype, **knobs))


def test_outputs_in_a_wider_buffer(pkg, cuda):
    a, b, fa, fb = operands(pkg, 200, 300, 512, 16)
    for start in (0, 1, 8):
        store = torch.full((202, 320), 9.0, dtype=torch.bfloat16, device="cuda")
        out = store[1:201, start:start + 300]
        pkg.gemm_fp4(a, b, out=out)
        check_sum(out, fa, fb)
        store[1:201, start:start + 300] = 9.0
        assert (store == 9.0).all()


def test_more_tiles_than_ctas_in_pairs(pkg, cuda):
    """Several tiles per CTA pair: the accumulator's two positions and the chunks of C in order."""
    m, n, k = 1500, 4200, 520
    a, b, fa, fb = operands(pkg, m, n, k, 16)
    residual = normal((m, n), 7, torch.bfloat16)
    for bn in (128, 256):
        check_sum(pkg.gemm_fp4(a, b, cta_group=2, tile_n=bn), fa, fb)
        check_sum(pkg.gemm_fp4(a, b, residual=residual, cta_group=2, tile_n=bn), fa, fb, residual=residual)


def test_large_and_small_row_scales(pkg, cuda):
    """Token scales that alone would take the sum out of range, against weights that bring it back."""
    x, w = normal((3, 512), 8), normal((64, 512), 9)
    for e in (100, -90):
        a = pkg.quantize_fp4(x * 2.0 ** e)
        b = pkg.quantize_fp4(w * 2.0 ** -e)
        for knobs in (dict(), dict(cta_group=1, tile_n=16), dict(cta_group=1, tile_n=16, split_k=2)):
            check_sum(pkg.gemm_fp4(a, b, **knobs), stands_for(a, pkg), stands_for(b, pkg))
        check_sum(pkg.linear_fp4((x * 2.0 ** e).bfloat16(), b), stands_for(pkg.quantize_fp4((x * 2.0 ** e).bfloat16()), pkg), stands_for(b, pkg))


def test_no_row_scale_is_one(pkg, cuda):
    a, b, _, _ = operands(pkg, 20, 150, 256, 32)
    a, b = a._replace(row_scale=None), b._replace(row_scale=None)
    one = [f._replace(row_scale=torch.ones(f.values.shape[0], device="cuda")) for f in (a, b)]
    got = pkg.gemm_fp4(a, b)
    assert torch.equal(got, pkg.gemm_fp4(*one)) and got.isfinite().all()


# ------------------------------------------------------------------ linear layer
@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 300, 16), (1, 1024, 16384), (1, 1000, 8000), (2, 520, 4099), (5, 130, 3000), (8, 257, 2048),
                                   (8, 4096, 2048), (9, 300, 2048), (8, 300, 2049), (3, 20000, 600), (200, 300, 1000), (1, 128, 20000)])
def test_linear_is_quantise_and_product(pkg, cuda, block, dtype, m, n, k):
    x = normal((m, k), 11, dtype)
    w = pkg.quantize_fp4(normal((n, k), 12, scale=0.05), block=block)
    q = pkg.quantize_fp4(x, block=block)
    bias, residual = normal((n,), 13, dtype), normal((m, n), 14, dtype)
    fx, fw = stands_for(q, pkg), stands_for(w, pkg)
    check_sum(pkg.linear_fp4(x, w), fx, fw)
    check_sum(pkg.linear_fp4(x, w, bias=bias, residual=residual), fx, fw, bias, residual)
    # The residual's row strides and the result's own.
    store = torch.full((m, n + 5), 3.0, dtype=dtype, device="cuda")
    pkg.linear_fp4(x, w, out=store[:, 2:n + 2])
    assert torch.equal(store[:, 2:n + 2], pkg.linear_fp4(x, w)) and (store[:, :2] == 3).all() and (store[:, n + 2:] == 3).all()


def test_linear_of_fp32_tokens(pkg, cuda):
    w = pkg.quantize_fp4(normal((100, 300), 1))
    x = normal((4, 300), 2)
    with pytest.raises(pkg.GemmError, match="bf16 or fp16"):
        pkg.linear_fp4(x, w)
    y = pkg.linear_fp4(x, w, out_dtype=torch.float16)
    assert y.dtype == torch.float16
    check_sum(y, stands_for(pkg.quantize_fp4(x), pkg), stands_for(w, pkg))


@pytest.mark.parametrize("m", [1, 7, 40])
def test_linear_over_its_tokens(pkg, cuda, m):
    w = pkg.quantize_fp4(normal((512, 512), 1, scale=0.05))
    x = normal((m, 512), 2, torch.bfloat16)
    want = pkg.linear_fp4(x, w, residual=x, cta_group=1, tile_n=64)
    y = x.clone()
    got = pkg.linear_fp4(y, w, residual=y, out=y)
    assert got is y
    check_sum(got, stands_for(pkg.quantize_fp4(x), pkg), stands_for(w, pkg), residual=x)
    check_sum(want, stands_for(pkg.quantize_fp4(x), pkg), stands_for(w, pkg), residual=x)


def test_a_row_of_nan_touches_no_other_in_the_fused_form(pkg, cuda):
    w = pkg.quantize_fp4(normal((300, 600), 1))
    x = normal((4, 600), 2, torch.bfloat16)
    want = pkg.linear_fp4(x, w)
    x[2, 599] = float("inf")
    got = pkg.linear_fp4(x, w)
    assert got[2].isnan().all() and torch.equal(got[[0, 1, 3]], want[[0, 1, 3]])


def test_empty_sizes(pkg, cuda):
    w = pkg.quantize_fp4(normal((30, 64), 1))
    assert pkg.linear_fp4(normal((0, 64), 2, torch.bfloat16), w).shape == (0, 30)
    none = pkg.quantize_fp4(normal((0, 64), 2))
    assert pkg.gemm_fp4(none, w).shape == (0, 30)
    assert pkg.dequantize_fp4(none).shape == (0, 64)


def test_the_nvfp4_gemm_reads_quantised_matrices(pkg, cuda):
    """Blocks of 16 with K in multiples of 256 are in the layout of the benchmark's NVFP4 product."""
    m, n, k = 256, 256, 512
    a = pkg.quantize_fp4(normal((m, k), 1))
    b = pkg.quantize_fp4(normal((n, k), 2))
    d = torch.empty((n, m), dtype=torch.bfloat16, device="cuda")
    args = pkg.make_args(dtype=pkg.NVFP4, m=m, n=n, k=k, a=a.values.data_ptr(), b=b.values.data_ptr(), d=d.data_ptr(),
                         lda=2 * a.values.stride(0), ldb=2 * b.values.stride(0), sfa=a.scales.data_ptr(), sfb=b.scales.data_ptr())
    pkg.launch(args, torch.cuda.current_stream().cuda_stream)
    ones = [f._replace(row_scale=torch.ones_like(f.row_scale)) for f in (a, b)]
    check_sum(d.t(), stands_for(ones[0], pkg), stands_for(ones[1], pkg))


# ------------------------------------------------------------------ streams, graphs, failures
def test_graph_replays(pkg, cuda):
    w = pkg.quantize_fp4(normal((700, 1024), 1, scale=0.05))
    for m in (1, 4, 50, 300):
        x = normal((m, 1024), 2, torch.bfloat16)
        pkg.linear_fp4(x, w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = pkg.linear_fp4(x, w)
            back = pkg.dequantize_fp4(pkg.quantize_fp4(y))
        for seed in (3, 4):
            x.copy_(normal((m, 1024), seed, torch.bfloat16))
            graph.replay()
            want = pkg.linear_fp4(x, w)
            assert torch.equal(y, want) and torch.equal(back, pkg.dequantize_fp4(pkg.quantize_fp4(want)))


def test_calls_on_two_streams(pkg, cuda):
    """Products of two streams at once: CTAs of one wait for no CTA of the other."""
    w = pkg.quantize_fp4(normal((4096, 2048), 1, scale=0.05))
    xs = [normal((m, 2048), m, torch.bfloat16) for m in (1, 300)]
    want = [pkg.linear_fp4(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(pkg.linear_fp4(xs[i], w))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


@pytest.mark.parametrize("knobs", [dict(cta_group=1, tile_n=64), dict(cta_group=1, tile_n=64, split_k=2), dict(cta_group=2, tile_n=256)])
def test_a_wait_that_runs_out_is_reported(pkg, cuda, knobs):
    a, b, fa, fb = operands(pkg, 64, 256, 2048, 16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    pkg.gemm_fp4(a, b, status=status, timeout_ms=20, flags=pkg.FLAG_INJECT_STALL, **knobs)
    rc, detail = pkg.read_status(status.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == pkg.ERR_TIMEOUT and detail & 0xFF == 3
    status.zero_()
    check_sum(pkg.gemm_fp4(a, b, status=status, **knobs), fa, fb)
    assert pkg.read_status(status.data_ptr(), torch.cuda.current_stream().cuda_stream)[0] == pkg.OK


def test_offsets_beyond_32_bits(pkg, cuda):
    """The last rows of matrices of more than 2^31 elements are those of a small call."""
    x = torch.zeros((140000, 16384), dtype=torch.bfloat16, device="cuda")
    x[-5:] = normal((5, 16384), 1, torch.bfloat16)
    f = pkg.quantize_fp4(x)
    small = pkg.quantize_fp4(x[-5:])
    assert torch.equal(f.values[-5:], small.values) and torch.equal(f.row_scale[-5:], small.row_scale)
    del x
    y = pkg.dequantize_fp4(f)
    assert torch.equal(y[-5:], pkg.dequantize_fp4(small)) and not y[:100].any()
    del y, f
    w = pkg.quantize_fp4(normal((32776, 256), 2), block=32)
    a = pkg.quantize_fp4(normal((70001, 256), 3), block=32)
    d = pkg.gemm_fp4(a, w)
    last = pkg.quantize_fp4(normal((70001, 256), 3)[-6:], block=32)
    check_sum(d[-6:], stands_for(last, pkg), stands_for(w, pkg))


def test_a_graph_captured_before_any_other_call_of_its_size(pkg, cuda):
    w = pkg.quantize_fp4(normal((333, 1777), 1, scale=0.05), block=32)
    for m in (3, 77):
        x = normal((m, 1777), 2, torch.float16)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = pkg.linear_fp4(x, w)
        graph.replay()
        check_sum(y, stands_for(pkg.quantize_fp4(x, block=32), pkg), stands_for(w, pkg))


def test_refusals_in_python(pkg, cuda):
    w = pkg.quantize_fp4(normal((30, 64), 1))
    x = normal((4, 64), 2, torch.bfloat16)
    a = pkg.quantize_fp4(x)
    for call, error in [
        (lambda: pkg.quantize_fp4(x, block=64), "block"),
        (lambda: pkg.quantize_fp4(x.cpu()), "CUDA"),
        (lambda: pkg.quantize_fp4(x.long()), "bfloat16"),
        (lambda: pkg.quantize_fp4(x.t()), "unit stride"),
        (lambda: pkg.gemm_fp4(a, pkg.quantize_fp4(normal((30, 65), 1))), "columns"),
        (lambda: pkg.gemm_fp4(a, pkg.quantize_fp4(normal((30, 64), 1), block=32)), "blocks"),
        (lambda: pkg.gemm_fp4(a._replace(scales=a.scales[:100]), w), "scales"),
        (lambda: pkg.gemm_fp4(a._replace(values=a.values[:, 1:]), w), "columns"),
        (lambda: pkg.gemm_fp4(a._replace(row_scale=a.row_scale[1:]), w), "row_scale"),
        (lambda: pkg.gemm_fp4(x, w), "Fp4"),
        (lambda: pkg.linear_fp4(x, w, bias=normal((31,), 1)), "bias"),
        (lambda: pkg.linear_fp4(x, w, residual=normal((4, 30), 1)), "residual"),
        (lambda: pkg.dequantize_fp4(a, dtype=torch.int8), "dtype"),
    ]:
        with pytest.raises(ValueError, match=error):
            call()
    for call, error in [
        (lambda: pkg.gemm_fp4(a, w, out_dtype=torch.float32), "bf16 or fp16"),
        (lambda: pkg.gemm_fp4(a, w, tile_n=48), "tile_n"),
        (lambda: pkg.gemm_fp4(pkg.quantize_fp4(normal((40, 64), 1)), w, tile_n=32, cta_group=1), "must hold all"),
        (lambda: pkg.gemm_fp4(a, w, split_k=4), "split_k"),
    ]:
        with pytest.raises(pkg.GemmError, match=error):
            call()
