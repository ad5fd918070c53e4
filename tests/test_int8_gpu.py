"""The int8 operators on the GPU against their definitions in 64 bits: the
quantiser (exact), the product and its epilogue, dropout (exact mask), the
linear layer forward and backward, and a training step made of them."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
TINY = 2.0 ** -126
U32 = 2.0 ** -24     # half a unit in the last place of an fp32 operation, relative


# ------------------------------------------------------------------ the definitions, in 64 bits
def ref_quantize(x):
    """q and scale of the rows of x (finite rows)."""
    x = x.double()
    amax = x.abs().amax(dim=1).clamp(min=127.0 * TINY)
    return torch.round(x * 127.0 / amax[:, None]), amax / 127.0


def ref_words(rows, cols, drop):
    """The 32-bit word of every element, with unsigned numpy integers."""
    row_elems = drop.col0 + cols if drop.row_elems is None else drop.row_elems
    seed = int(drop.seed.item()) if isinstance(drop.seed, torch.Tensor) else drop.seed
    g, u = np.uint64(0x9E3779B97F4A7C15), np.uint64

    def mix(z):
        z = (z ^ (z >> u(30))) * u(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> u(27))) * u(0x94D049BB133111EB)
        return z ^ (z >> u(31))

    with np.errstate(over="ignore"):
        key = mix(np.array([seed % 2 ** 64], np.uint64) + mix(np.array([drop.stream_id % 2 ** 64], np.uint64) + g))
        r = np.arange(rows, dtype=np.uint64)[:, None] + u(drop.row0)
        c = np.arange(cols, dtype=np.uint64)[None, :] + u(drop.col0)
        index = r * u(row_elems) + c
        h = mix(key + (index // u(2) + u(1)) * g)
    return np.where(index % u(2) == u(1), h >> u(32), h & u(0xFFFFFFFF))


def ref_keep(rows, cols, drop):
    if drop is None or drop.p == 0.0:
        return torch.ones((rows, cols), dtype=torch.bool)
    return torch.from_numpy(ref_words(rows, cols, drop) >= np.uint64(round(drop.p * 2 ** 32)))


def ref_product(a, sa, b, sb, bias=None, residual=None, drop=None):
    """(value, magnitude of the fp32 terms it is made of)."""
    t = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()[None, :]
    size = t.abs()
    if bias is not None:
        t = t + bias.double()
        size = size + bias.double().abs()
    if drop is not None and drop.p > 0.0:
        keep = ref_keep(t.shape[0], t.shape[1], drop).to(t.device)
        grow = 0.0 if drop.p == 1.0 else 1.0 / (1.0 - drop.p)
        t = torch.where(keep, t * grow, 0.0)
        size = torch.where(keep, size * grow, 0.0)
    if residual is not None:
        t = t + residual.double()
        size = size + residual.double().abs()
    return t, size


def check_close(got, want, size, scale_err=0.0):
    """|got - want| <= half a step of got's type + the fp32 operations before it (conversion of the
    sum, two scales, bias, 1/(1-p) and its rounding, residual: 7 roundings of at most U32 * size)."""
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * want.abs() + (8 * U32 + scale_err) * size + fi.smallest_normal * fi.eps
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (bad.sum().item(), ((got.double() - want).abs() / tol.clamp(min=1e-300)).max().item())


def normal(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def int8s(pkg, rows, cols, seed):
    """Random int8 values, the extremes -128 and 127 among them, in padded rows."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    q = pkg.empty_int8(rows, cols, "cuda")
    q.copy_(torch.randint(-128, 128, (rows, cols), generator=g, device="cuda", dtype=torch.int16).to(torch.int8))
    return q


def scales(n, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.rand((n,), generator=g, device="cuda") * 0.05 + 0.001


# ------------------------------------------------------------------ quantiser
def check_quantized(q, scale, x):
    want_q, want_s = ref_quantize(x)
    assert torch.equal(q.double(), want_q)
    assert ((scale.double() - want_s).abs() <= U32 * want_s + 2.0 ** -150).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8192), (3, 7), (5, 1000), (33, 4099), (300, 128), (2, 40000), (1, 70001)])
@pytest.mark.parametrize("transpose", [False, True])
def test_quantize_exact(pkg, cuda, dtype, rows, cols, transpose):
    x = normal((rows, cols), rows * 7 + cols, dtype, 3.0)
    q, scale = pkg.quantize_int8(x, transpose=transpose)
    assert q.stride(0) % 16 == 0
    check_quantized(q, scale, x.t() if transpose else x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [31, 257, 3000, 20000])
def test_quantize_transposed_long_columns(pkg, cuda, dtype, rows):
    """Columns longer than a cluster's shared memory are read again."""
    x = normal((rows, 70), rows, dtype)
    q, scale, sums = pkg.quantize_int8(x, transpose=True, column_sums=True)
    check_quantized(q, scale, x.t())
    want = x.double().sum(0)
    # fp32 sums of at most 20000 / 8 / 16 consecutive terms, then 32 + 8 partial sums: 200 roundings of partial
    # sums that stay below the sum of magnitudes.
    assert ((sums.double() - want).abs() <= 200 * U32 * x.double().abs().sum(0)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [255, 272, 500, 700, 1000, 1025, 1290, 1300, 1537, 1792, 1793, 2040])
def test_quantize_transposed_every_cluster_size(pkg, cuda, dtype, rows):
    """One to eight CTAs per strip, rows that fill the last 16-row sets of a warp unevenly, strips that
    end inside 64 bytes."""
    x = normal((rows, 83), rows + 1, dtype)
    q, scale, sums = pkg.quantize_int8(x, transpose=True, column_sums=True)
    check_quantized(q, scale, x.t())
    # A thread adds at most ceil(256 / 32) rows of a CTA, then 3 + 4 + 8 partial sums of lanes, warps and CTAs.
    assert ((sums.double() - x.double().sum(0)).abs() <= 24 * U32 * x.double().abs().sum(0)).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_ties_go_to_even(pkg, cuda, dtype):
    """amax = 254 makes every odd value a tie: 127 x / 254 = x / 2."""
    x = torch.arange(-254, 255, device="cuda", dtype=torch.float32)
    x = torch.stack([x, x * 2.0 ** -10, x * 2.0 ** -20 if dtype != torch.float16 else -x]).to(dtype)
    if dtype == torch.bfloat16:
        assert torch.equal(x.float()[0], torch.arange(-254, 255, device="cuda").float())
    for t in (False, True):
        src = x.t().contiguous() if t else x
        q, scale = pkg.quantize_int8(src, transpose=t)
        check_quantized(q, scale, x)
    assert q[0, 255].item() == 0 and q[0, 257].item() == 2     # 0.5 -> 0, 1.5 -> 2


def test_quantize_fp32_next_to_ties(pkg, cuda):
    """fp32 values one unit around (n + 1/2) amax / 127 for many amax."""
    g = torch.Generator().manual_seed(3)
    amax = torch.rand((200,), generator=g, dtype=torch.float64).float() * 10 + 1
    n = torch.arange(-127, 127, dtype=torch.float64) + 0.5
    mid = (n[None, :] * amax.double()[:, None] / 127.0).float()
    x = torch.cat([amax[:, None], mid, torch.nextafter(mid, torch.full_like(mid, 1e9)),
                   torch.nextafter(mid, torch.full_like(mid, -1e9))], dim=1).cuda()
    for t in (False, True):
        q, scale = pkg.quantize_int8(x.t().contiguous() if t else x, transpose=t)
        check_quantized(q, scale, x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [1e-45, 1e-39, 1e-37, 1e-30, 1e-19, 1e19, 1e30, 1e37])
def test_quantize_extreme_ranges(pkg, cuda, dtype, scale):
    x = (normal((4, 333), 5).clamp(-3, 3).double() * scale).to(dtype)
    for t in (False, True):
        q, s = pkg.quantize_int8(x.t().contiguous() if t else x, transpose=t)
        check_quantized(q, s, x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("transpose", [False, True])
def test_quantize_zero_nan_inf_rows(pkg, cuda, dtype, transpose):
    x = normal((6, 100), 1, dtype)
    x[1] = 0.0
    x[2, 17] = float("nan")
    x[3, 99] = float("-inf")
    x[4, 5], x[4, 6] = float("inf"), float("nan")
    q, s = pkg.quantize_int8(x.t().contiguous() if transpose else x, transpose=transpose)
    assert (q[1:5] == 0).all()
    assert s[1].item() == TINY and math.isnan(s[2].item()) and s[3].item() == math.inf and math.isnan(s[4].item())
    fine = [0, 5]
    check_quantized(q[fine], s[fine], x[fine])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("transpose", [False, True])
def test_quantize_strided_and_unaligned(pkg, cuda, dtype, transpose):
    big = normal((50, 300), 2, dtype)
    for x in (big[:, 1:200], big[3:40, 8:280], big[::2, :129], big[:1, 5:6]):
        q, s = pkg.quantize_int8(x, transpose=transpose)
        check_quantized(q, s, x.t() if transpose else x)


def test_quantize_leaves_the_padding_alone(pkg, cuda):
    x = normal((9, 21), 4, torch.bfloat16)
    L = pkg.lib()
    for transpose, rows, cols in ((0, 9, 21), (1, 21, 9)):
        q = torch.full((rows + 2, 48), 77, dtype=torch.int8, device="cuda")
        s = torch.full((rows + 2,), 77.0, device="cuda")
        a = pkg.Int8QuantArgs(struct_size=136, x_type=0, rows=9, cols=21, x=x.data_ptr(), ldx=21, q=q.data_ptr(), ldq=48,
                              scale=s.data_ptr(), transpose=transpose)
        assert L.gemm_sm100a_quantize_int8(bytes(a), torch.cuda.current_stream().cuda_stream) == pkg.OK
        check_quantized(q[:rows, :cols], s[:rows], x.t() if transpose else x)
        assert (q[rows:] == 77).all() and (q[:, cols:] == 77).all() and (s[rows:] == 77).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("p", [0.25, 0.9, 1.0])
def test_quantize_with_dropout(pkg, cuda, dtype, transpose, p):
    rows, cols = 300, 133
    drop = pkg.Dropout(p, seed=2 ** 63 + 11, stream_id=3, row0=5, col0=3, row_elems=141)
    x = normal((rows, cols), 9, dtype)
    keep = ref_keep(rows, cols, drop).cuda()
    x[~keep] = float("nan")                       # a dropped NaN is a zero
    masked = torch.where(keep, x.double(), 0.0)
    out = pkg.quantize_int8(x, transpose=transpose, dropout=drop, column_sums=transpose)
    q, s = out[:2]
    want_q, want_s = ref_quantize(masked.t() if transpose else masked)
    grow = 0.0 if p == 1.0 else 1.0 / (1.0 - p)
    assert torch.equal(q.double(), want_q)
    assert ((s.double() - want_s * grow).abs() <= 3 * U32 * want_s * grow).all()
    if transpose:
        assert ((out[2].double() - masked.sum(0) * grow).abs() <= 60 * U32 * masked.abs().sum(0) * grow).all()


def test_quantize_empty(pkg, cuda):
    q, s, c = pkg.quantize_int8(torch.empty((0, 5), device="cuda"), transpose=True, column_sums=True)
    assert q.shape == (5, 0) and (s == TINY).all() and (c == 0).all()
    q, s = pkg.quantize_int8(torch.empty((0, 5), device="cuda"))
    assert q.shape == (0, 5) and s.shape == (0,)
    with pytest.raises(ValueError):
        pkg.quantize_int8(torch.empty((5, 0), device="cuda"))


# ------------------------------------------------------------------ product
PRODUCT_SHAPES = [(1, 1, 1), (1, 16, 16), (2, 3, 5), (1, 4099, 1000), (8, 130, 129), (9, 257, 4096), (16, 128, 8192),
                  (17, 1000, 2056), (33, 640, 384), (64, 256, 257), (65, 129, 8191), (127, 1025, 640),
                  (128, 128, 128), (200, 3000, 160), (256, 512, 1024), (300, 1111, 777), (513, 2049, 300), (1200, 1300, 272)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", PRODUCT_SHAPES)
def test_product(pkg, cuda, dtype, m, n, k):
    a, b = int8s(pkg, m, k, m + k), int8s(pkg, n, k, n + 2 * k)
    sa, sb = scales(m, 1), scales(n, 2)
    if dtype == torch.float16:
        sa = sa * 0.02          # keeps the largest values below 65504
    d = pkg.gemm_int8(a, sa, b, sb, out_dtype=dtype)
    check_close(d, *ref_product(a, sa, b, sb))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 257, 640), (7, 100, 1000), (40, 333, 512), (300, 777, 400), (700, 1024, 256)])
@pytest.mark.parametrize("bias_dtype", [torch.float32, None])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_product_epilogue(pkg, cuda, dtype, m, n, k, bias_dtype, p):
    a, b = int8s(pkg, m, k, m), int8s(pkg, n, k, n)
    sa, sb = scales(m, 1) * 0.01, scales(n, 2)
    bias = normal((n,), 3, bias_dtype or dtype)
    residual = normal((m, n), 4, dtype)
    drop = pkg.Dropout(p, seed=77, stream_id=5, row0=2, col0=1, row_elems=n + 4) if p else None
    d = pkg.gemm_int8(a, sa, b, sb, bias=bias, residual=residual, dropout=drop, out_dtype=dtype)
    check_close(d, *ref_product(a, sa, b, sb, bias, residual, drop))
    # the residual may be the output
    out = residual.clone()
    got = pkg.gemm_int8(a, sa, b, sb, bias=bias, residual=out, dropout=drop, out=out)
    assert got is out and torch.equal(out, d)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(9, 131, 200), (70, 131, 200), (300, 515, 200), (700, 1031, 200), (40, 131, 4096)])
@pytest.mark.parametrize("row0,col0", [(0, 0), (1, 0), (0, 1), (1, 1)])
def test_product_dropout_with_rows_of_an_odd_length(pkg, cuda, dtype, m, n, k, row0, col0):
    """Draws' pairs begin at even channels in one token and at odd ones in the next."""
    a, b = int8s(pkg, m, k, m), int8s(pkg, n, k, n)
    sa, sb = scales(m, 1) * 0.01, scales(n, 2)
    drop = pkg.Dropout(0.4, seed=9, stream_id=1, row0=row0, col0=col0, row_elems=n + 2)
    got = pkg.gemm_int8(a, sa, b, sb, dropout=drop, out_dtype=dtype)
    keep = ref_keep(m, n, drop).to(got.device)
    assert (got[~keep] == 0).all()
    want, size = ref_product(a, sa, b, sb, None, None, drop)
    check_close(got, want, size)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", [(3, 131), (50, 131), (300, 515), (600, 777)])
def test_product_writes_only_its_output(pkg, cuda, dtype, m, n):
    """D inside a larger buffer, at an odd column (element alignment) and at an aligned one."""
    k = 320
    a, b, sa, sb = int8s(pkg, m, k, 1), int8s(pkg, n, k, 2), scales(m, 3) * 0.01, scales(n, 4)
    want = pkg.gemm_int8(a, sa, b, sb, out_dtype=dtype)
    for c0, width in ((1, n + 6), (8, (n + 31) // 16 * 16)):
        buf = torch.full((m + 3, width), 123.0, dtype=dtype, device="cuda")
        out = buf[1:m + 1, c0:c0 + n]
        pkg.gemm_int8(a, sa, b, sb, out=out)
        assert torch.equal(out, want)
        out.fill_(123.0)
        assert (buf == 123.0).all()


VARIANTS = ([dict(cta_group=1, tile_n=bn, split_k=s) for bn in (16, 32, 64, 128) for s in (1, 2, 4, 8)]
            + [dict(cta_group=2, tile_n=bn) for bn in (128, 256)])


@pytest.mark.parametrize("knobs", VARIANTS, ids=lambda v: "-".join(str(x) for x in v.values()))
def test_every_tile_and_split_gives_the_same_bits(pkg, cuda, knobs):
    """Each variant on ragged problems, with and without TMA stores (odd n), every epilogue term."""
    for m, n, k, dtype in ((1, 200, 1100, torch.bfloat16), (75, 333, 2000, torch.float16), (301, 648, 1024, torch.float32),
                           (530, 1100, 1500, torch.bfloat16)):
        a, b, sa, sb = int8s(pkg, m, k, 1), int8s(pkg, n, k, 2), scales(m, 3) * 0.01, scales(n, 4)
        bias, residual = normal((n,), 5, dtype), normal((m, n), 6, dtype)
        drop = pkg.Dropout(0.3, seed=3)
        for kw in (dict(), dict(bias=bias, residual=residual, dropout=drop)):
            want = pkg.gemm_int8(a, sa, b, sb, out_dtype=dtype, **kw)
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            out = torch.full((m + 2, n), 77.0, dtype=dtype, device="cuda")
            pkg.gemm_int8(a, sa, b, sb, out=out[1:m + 1], status=status, **kw, **knobs)
            assert status.item() == 0
            assert torch.equal(out[1:m + 1], want)
            assert (out[0] == 77.0).all() and (out[m + 1] == 77.0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(300, 600, 6000), (700, 1040, 700)])
def test_pairs_with_long_and_short_main_loops(pkg, cuda, dtype, m, n, k):
    """One and two epilogue groups, several tiles per pair, the residual staged, unaligned and in place."""
    a, b, sa, sb = int8s(pkg, m, k, 1), int8s(pkg, n, k, 2), scales(m, 3) * 0.01, scales(n, 4)
    bias, residual = normal((n,), 5, dtype), normal((m, n), 6, dtype)
    drop = pkg.Dropout(0.3, seed=3, row0=1, col0=2, row_elems=n + 2)
    want = ref_product(a, sa, b, sb, bias, residual, drop)
    shifted = torch.empty((m, n + 3), dtype=dtype, device="cuda")[:, 1:n + 1]
    shifted.copy_(residual)
    first = None
    for kw in (dict(), dict(cta_group=2, tile_n=128), dict(cta_group=2, tile_n=256)):
        for res in (residual, shifted):
            d = pkg.gemm_int8(a, sa, b, sb, bias=bias, residual=res, dropout=drop, out_dtype=dtype, **kw)
            first = d if first is None else first
            assert torch.equal(d, first)
        out = residual.clone()
        pkg.gemm_int8(a, sa, b, sb, bias=bias, residual=out, dropout=drop, out=out, **kw)
        assert torch.equal(out, first)
        odd = drop._replace(col0=1)                       # pairs of a draw begin at odd channels
        check_close(pkg.gemm_int8(a, sa, b, sb, dropout=odd, out_dtype=dtype, **kw), *ref_product(a, sa, b, sb, drop=odd))
    check_close(first, *want)


def test_refused_knobs(pkg, cuda):
    a, b, sa, sb = int8s(pkg, 4, 512, 1), int8s(pkg, 6, 512, 2), scales(4, 3), scales(6, 4)
    for knobs in (dict(tile_n=48), dict(cta_group=3), dict(cta_group=2, tile_n=64), dict(split_k=3),
                  dict(cta_group=2, tile_n=256, split_k=2), dict(split_k=8)):       # 4 K blocks, 8 CTAs
        with pytest.raises(pkg.GemmError):
            pkg.gemm_int8(a, sa, b, sb, **knobs)


def test_a_stalled_load_ends_with_a_status(pkg, cuda):
    """The injected stall makes every wait run out: the status says so, nothing hangs, and the next
    product is right."""
    a, b, sa, sb = int8s(pkg, 300, 1024, 1), int8s(pkg, 600, 1024, 2), scales(300, 3), scales(600, 4)
    want = pkg.gemm_int8(a, sa, b, sb)
    for knobs in (dict(cta_group=1, tile_n=64, split_k=1), dict(cta_group=1, tile_n=64, split_k=4),
                  dict(cta_group=2, tile_n=256)):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        pkg.gemm_int8(a, sa, b, sb, status=status, timeout_ms=20, flags=pkg.FLAG_INJECT_STALL, **knobs)
        rc, detail = pkg.read_status(status.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert rc == pkg.ERR_TIMEOUT and detail != 0
        assert torch.equal(pkg.gemm_int8(a, sa, b, sb, **knobs), want)


def test_product_extreme_sums(pkg, cuda):
    """The largest sums of 8-bit products, at the longest K: -128 * -128 * 131071 < 2^31."""
    k = pkg.MAX_INT8_K
    for m, n in ((1, 130), (130, 130)):
        a, b = pkg.empty_int8(m, k, "cuda"), pkg.empty_int8(n, k, "cuda")
        a.fill_(-128)
        b.fill_(-128)
        b[1::2] = 127
        d = pkg.gemm_int8(a, None, b, None, out_dtype=torch.float32)
        want = torch.where(torch.arange(n, device="cuda") % 2 == 0, 16384.0 * k, -16256.0 * k).double().expand(m, n)
        check_close(d, want, want.abs())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("knobs", [dict()] + [dict(cta_group=1, tile_n=64, split_k=s) for s in (1, 4)]
                         + [dict(cta_group=2, tile_n=bn) for bn in (128, 256)], ids=str)
def test_product_scales_far_from_one(pkg, cuda, dtype, knobs):
    """Outputs of ordinary size from scales whose product with the sum alone would leave fp32, some tokens'
    large, some channels', zero channels among them."""
    m, n, k = 301, 520, 1024
    a, b, bias, residual = int8s(pkg, m, k, 1), int8s(pkg, n, k, 2), normal((n,), 3), normal((m, n), 4, dtype)
    for rows, lift in ((m, 2.0 ** 120), (m, 2.0 ** -110), (5, 2.0 ** 120), (1, 2.0 ** 96)):
        sa, sb = scales(m, 3) * 0.01 * lift, scales(n, 4) / lift
        sb[::7] = 0.0
        if rows == m:
            sa[::3] /= min(lift, 2.0 ** 100)           # ordinary tokens in the same tile
        for kw in (dict(), dict(bias=bias, residual=residual[:rows], dropout=pkg.Dropout(0.25, seed=2))):
            d = pkg.gemm_int8(a[:rows], sa[:rows].contiguous(), b, sb, out_dtype=dtype, **kw, **knobs)
            want, size = ref_product(a[:rows], sa[:rows], b, sb, kw.get("bias"), kw.get("residual"), kw.get("dropout"))
            # Ordinary tokens with large channels: what lies half a step beyond the type's largest value rounds to Inf
            # (fp16 from 65520; the step above a value v <= 65504 is at least eps v / 2).
            top = torch.finfo(dtype).max
            over = want.abs() > top * (1 + torch.finfo(dtype).eps)
            assert torch.equal(d[over].double(), want[over].sign() * math.inf)
            check_close(torch.where(over, 0.0, d).to(dtype), torch.where(over, 0.0, want), size.clamp(max=top))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 512), (1, 16000), (8, 2048), (8, 130), (60, 512), (400, 640)])
def test_linear_of_tokens_far_from_one(pkg, cuda, dtype, m, k):
    """Tokens next to the end of fp32's range, and small weights: whole-K, split and one-launch forms."""
    x, n = (normal((m, k), 1).double().clamp(-3, 3) * 1e37).to(dtype), 300
    w, ws = pkg.quantize_int8((normal((n, k), 2).double() * 1e-34).float())
    y = pkg.linear_int8(x, w, ws)
    check_close(y, *ref_product(*ref_quantize(x), w, ws), scale_err=U32)
    q, s = pkg.quantize_int8(x)
    assert torch.equal(y, pkg.gemm_int8(q, s, w, ws, out_dtype=dtype))


def test_product_nan_rows_touch_only_themselves(pkg, cuda):
    m, n, k = 40, 200, 256
    a, b, sa, sb = int8s(pkg, m, k, 1), int8s(pkg, n, k, 2), scales(m, 3), scales(n, 4)
    want = pkg.gemm_int8(a, sa, b, sb)
    sa[7], sb[150] = float("nan"), float("nan")
    d = pkg.gemm_int8(a, sa, b, sb)
    assert torch.isnan(d[7]).all() and torch.isnan(d[:, 150]).all()
    rows = [i for i in range(m) if i != 7]
    cols = [j for j in range(n) if j != 150]
    assert torch.equal(d[rows][:, cols], want[rows][:, cols])


def test_product_empty(pkg, cuda):
    b, sb = int8s(pkg, 20, 32, 2), scales(20, 4)
    assert pkg.gemm_int8(pkg.empty_int8(0, 32, "cuda"), torch.empty(0, device="cuda"), b, sb).shape == (0, 20)
    assert pkg.linear_int8(torch.empty((0, 32), device="cuda"), b, sb).shape == (0, 20)
    with pytest.raises(pkg.GemmError):
        pkg.gemm_int8(pkg.empty_int8(4, 0, "cuda"), None, pkg.empty_int8(4, 0, "cuda"), None)


def test_refused_tensors(pkg, cuda):
    a, b, sa, sb = int8s(pkg, 4, 32, 1), int8s(pkg, 6, 32, 2), scales(4, 3), scales(6, 4)
    with pytest.raises(ValueError):
        pkg.gemm_int8(a, sa, b[:, :16], sb)                  # other k
    with pytest.raises(ValueError):
        pkg.gemm_int8(a, sb, b, sb)                          # scales of another length
    with pytest.raises(ValueError):
        pkg.gemm_int8(a, sa, b, sb, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        pkg.gemm_int8(a, sa, b, sb, residual=torch.zeros((4, 6), device="cuda"))     # not D's type
    with pytest.raises(ValueError):
        pkg.gemm_int8(a, sa, b, sb, out=torch.zeros((6, 4), device="cuda").t())      # column-major
    with pytest.raises(ValueError):
        pkg.gemm_int8(torch.zeros((4, 40), dtype=torch.int8, device="cuda")[:, :32], sa, b, sb)   # stride 40
    with pytest.raises(pkg.GemmError):
        pkg.gemm_int8(a[:, 1:17], sa, b[:, :16], sb)         # base not 16-byte aligned
    with pytest.raises(TypeError):
        pkg.gemm_int8(a, sa, b, sb, tile_q=3)
    with pytest.raises(pkg.GemmError):
        pkg.gemm_int8(a, sa, b, sb, dropout=pkg.Dropout(1.5))
    with pytest.raises(ValueError):
        pkg.dropout(torch.zeros((4, 4), device="cuda"), pkg.Dropout(0.5, seed=torch.zeros(1, device="cuda")))


# ------------------------------------------------------------------ linear layer
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 100, 64), (1, 2051, 8192), (4, 300, 1001), (8, 129, 28672), (20, 1000, 515),
                                   (64, 128, 4096), (100, 700, 333), (513, 1030, 640)])
def test_linear_is_quantise_then_product(pkg, cuda, dtype, m, n, k):
    """Bit for bit, and against 64 bits."""
    x = normal((m, k), m + n, dtype)
    w, ws = pkg.quantize_int8(normal((n, k), 5, scale=0.02))
    bias = normal((n,), 6, dtype)
    drop = pkg.Dropout(0.2, seed=9)
    residual = normal((m, n), 7, dtype)
    q, s = pkg.quantize_int8(x)
    for kw in (dict(), dict(bias=bias), dict(bias=bias, dropout=drop, residual=residual)):
        y = pkg.linear_int8(x, w, ws, **kw)
        assert y.dtype == dtype
        assert torch.equal(y, pkg.gemm_int8(q, s, w, ws, out_dtype=dtype, **kw))
        want = ref_product(*ref_quantize(x), w, ws, kw.get("bias"), kw.get("residual"), kw.get("dropout"))
        check_close(y, *want, scale_err=U32)


def test_linear_refuses_knobs_before_it_quantises(pkg, cuda):
    """A refused call launches nothing: the workspace and the output stay as they were."""
    import ctypes
    m, n, k = 20, 64, 512
    x = normal((m, k), 1, torch.bfloat16)
    w, ws = pkg.quantize_int8(normal((n, k), 2))
    work, scale = torch.full((m, k), 77, dtype=torch.int8, device="cuda"), torch.full((m,), 77.0, device="cuda")
    out = torch.full((m, n), 77.0, dtype=torch.bfloat16, device="cuda")
    for knobs in (dict(tile_n=48), dict(cta_group=3), dict(cta_group=2, tile_n=64), dict(split_k=3), dict(split_k=8),
                  dict(cta_group=2, tile_n=256, split_k=2)):
        a = pkg.Int8GemmArgs(struct_size=0, d_type=0, m=m, n=n, k=k, a=work.data_ptr(), lda=k, b=w.data_ptr(),
                             ldb=w.stride(0), d=out.data_ptr(), ldd=n, scale_a=scale.data_ptr(), scale_b=ws.data_ptr(), **knobs)
        a.struct_size = ctypes.sizeof(a)
        rc = pkg.lib().gemm_sm100a_int8_linear(bytes(a), x.data_ptr(), 0, k, torch.cuda.current_stream().cuda_stream)
        assert rc == pkg.ERR_CANNOT_IMPLEMENT
        assert (work == 77).all() and (scale == 77).all() and (out == 77).all()
        with pytest.raises(pkg.GemmError):
            pkg.linear_int8(x, w, ws, **knobs)


@pytest.mark.parametrize("m", [1, 8, 40])
def test_linear_names_the_reason_of_a_refusal(pkg, cuda, m):
    """The same one with and without a workspace for the tokens."""
    w, ws = pkg.quantize_int8(normal((50, 64), 2))
    x = normal((m, 64), 1)
    for reason, call in (("16-byte aligned", lambda: pkg.linear_int8(x[:, 1:17], w[:, 1:17], ws)),
                         ("empty problem", lambda: pkg.linear_int8(x[:, :0], w[:, :0], ws)),
                         ("dropout p", lambda: pkg.linear_int8(x, w, ws, dropout=pkg.Dropout(1.5))),
                         ("row_elems", lambda: pkg.linear_int8(x, w, ws, dropout=pkg.Dropout(0.5, row_elems=49)))):
        with pytest.raises(pkg.GemmError, match=reason):
            call()


def test_linear_strided_tokens(pkg, cuda):
    big = normal((70, 700), 1, torch.bfloat16)
    w, ws = pkg.quantize_int8(normal((300, 513), 5, scale=0.02))
    for x in (big[:, 1:514], big[::3, 8:521], big[5:6, :513]):
        y = pkg.linear_int8(x, w, ws)
        assert torch.equal(y, pkg.linear_int8(x.contiguous(), w, ws))
        check_close(y, *ref_product(*ref_quantize(x), w, ws), scale_err=U32)


@pytest.mark.parametrize("m", [1, 3, 40, 300])
def test_linear_non_finite_tokens(pkg, cuda, m):
    x = normal((m, 512), 1, torch.bfloat16)
    w, ws = pkg.quantize_int8(normal((200, 512), 5, scale=0.02))
    want = pkg.linear_int8(x, w, ws)
    x[m - 1, 3] = float("inf")
    y = pkg.linear_int8(x, w, ws)
    assert torch.isnan(y[m - 1]).all()
    assert torch.equal(y[:m - 1], want[:m - 1])


def test_a_token_does_not_depend_on_its_batch(pkg, cuda):
    """The same token gives the same bits alone and inside any batch."""
    x = normal((400, 1024), 1, torch.bfloat16)
    w, ws = pkg.quantize_int8(normal((1500, 1024), 5, scale=0.02))
    full = pkg.linear_int8(x, w, ws)
    for m in (1, 2, 8, 9, 16, 33, 64, 65, 128, 129, 257):
        assert torch.equal(pkg.linear_int8(x[:m], w, ws), full[:m]), m


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 3, 8, 9, 40])
def test_linear_in_place(pkg, cuda, dtype, m):
    """The result replaces the tokens, alone and added to them, while other streams keep SMs busy; and
    out beside the tokens in one buffer, or a row further down in it."""
    k = 1024
    first = normal((m, k), 1, dtype)
    w, ws = pkg.quantize_int8(normal((k, k), 2, scale=0.05))
    plain, added = pkg.linear_int8(first, w, ws), pkg.linear_int8(first, w, ws, residual=first)
    big, side = normal((4096, 4096), 3), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        x, y = first.clone(), first.clone()
        with torch.cuda.stream(side):
            pkg.dropout(big, pkg.Dropout(0.5), out=big)
        assert pkg.linear_int8(x, w, ws, out=x) is x
        pkg.linear_int8(y, w, ws, residual=y, out=y)
        assert torch.equal(x, plain) and torch.equal(y, added)
    both = torch.zeros((m, 2 * k), dtype=dtype, device="cuda")
    both[:, :k] = first
    pkg.linear_int8(both[:, :k], w, ws, out=both[:, k:])
    assert torch.equal(both[:, k:], plain) and torch.equal(both[:, :k], first)
    rows = torch.zeros((m + 1, k), dtype=dtype, device="cuda")
    rows[:m] = first
    pkg.linear_int8(rows[:m], w, ws, out=rows[1:])
    assert torch.equal(rows[1:], plain) and torch.equal(rows[0], first[0])


# ------------------------------------------------------------------ backward
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 64, 100), (5, 33, 7), (77, 300, 130), (333, 1000, 250), (600, 129, 1000)])
@pytest.mark.parametrize("p", [0.0, 0.25])
def test_backward(pkg, cuda, dtype, m, n, k, p):
    dy, x = normal((m, n), 1, dtype), normal((m, k), 2, dtype)
    w = normal((n, k), 3, scale=0.02)
    wt, wts = pkg.quantize_int8(w, transpose=True)
    drop = pkg.Dropout(p, seed=31, stream_id=2) if p else None
    dx, dw, db = pkg.linear_int8_backward(dy, x, wt, wts, dropout=drop)
    assert dx.dtype == dtype and dw.dtype == torch.float32 and db.dtype == torch.float32
    grow = 1.0 / (1.0 - p)
    dz = torch.where(ref_keep(m, n, drop).cuda(), dy.double(), 0.0)
    qz, sz = ref_quantize(dz)
    check_close(dx, *ref_product(qz, sz * grow, wt, wts), scale_err=4 * U32)
    qt, st = ref_quantize(dz.t())
    qx, sx = ref_quantize(x.t())
    check_close(dw, *ref_product(qt, st * grow, qx, sx), scale_err=4 * U32)
    assert ((db.double() - dz.sum(0) * grow).abs() <= 100 * U32 * dz.abs().sum(0) * grow + 1e-30).all()


def test_backward_is_near_the_gradient_of_the_linear_map(pkg, cuda):
    """Against the unquantised gradient and against differences of the unquantised layer: each
    product differs by the rounding of its two operands, at most half a step (amax / 254) each."""
    m, n, k = 64, 96, 80
    dy, x, w = normal((m, n), 1).double(), normal((m, k), 2).double(), normal((n, k), 3, scale=0.05).double()
    wt, wts = pkg.quantize_int8(w.float(), transpose=True)
    dx, dw, db = pkg.linear_int8_backward(dy.float(), x.float(), wt, wts)

    def bound(a, b):      # sum over the contracted axis of |da| |b| + |a| |db| + |da| |db|, rows of a and b contracted
        ha, hb = a.abs().amax(1, keepdim=True) / 254, b.abs().amax(1, keepdim=True) / 254
        return (ha * b.abs().sum(1)[None, :] + a.abs().sum(1)[:, None] * hb.t() + a.shape[1] * ha * hb.t()) * (1 + 1e-4)

    assert ((dx.double() - dy @ w).abs() <= bound(dy, w.t())).all()
    assert ((dw.double() - dy.t() @ x).abs() <= bound(dy.t(), x.t())).all()
    # differences of f(x, w, b) = sum(dy * (x w^T + b)), which is linear in each argument
    f = lambda x, w, b: (dy * (x @ w.t() + b)).sum()   # noqa: E731
    zero = torch.zeros(n, device="cuda", dtype=torch.float64)
    for i, j in ((0, 0), (13, 57), (63, 79)):
        e = torch.zeros_like(x)
        e[i, j] = 0.5
        diff = f(x + e, w, zero) - f(x - e, w, zero)
        assert abs(dx[i, j].item() - diff.item()) <= bound(dy, w.t())[i, j] + 1e-9
        e = torch.zeros_like(w)
        e[i, j] = 0.5
        diff = f(x, w + e, zero) - f(x, w - e, zero)
        assert abs(dw[i, j].item() - diff.item()) <= bound(dy.t(), x.t())[i, j] + 1e-9
        b = zero.clone()
        b[i] = 0.5
        assert abs(db[i].item() - (f(x, w, b) - f(x, w, -b)).item()) <= 100 * U32 * dy.abs().sum(0)[i]


@pytest.mark.parametrize("wanted", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)])
def test_backward_of_some_gradients(pkg, cuda, wanted):
    """NULL outputs are not computed; the others have the same bits, and nothing else is written."""
    m, n, k = 50, 70, 90
    dy, x = normal((m, n), 1), normal((m, k), 2)
    wt, wts = pkg.quantize_int8(normal((n, k), 3, scale=0.02), transpose=True)
    full = pkg.linear_int8_backward(dy, x, wt, wts)
    out = [torch.full((m + 1, k + 3), 5.0, device="cuda"), torch.full((n + 1, k + 3), 5.0, device="cuda"),
           torch.full((n + 1,), 5.0, device="cuda")]
    need = pkg.lib().gemm_sm100a_int8_backward_workspace(m, n, k)
    work = torch.full((need + 64,), 77, dtype=torch.uint8, device="cuda")
    a = pkg.Int8BackwardArgs(struct_size=0, type=2, m=m, n=n, k=k, dy=dy.data_ptr(), lddy=n,
                             x=x.data_ptr() if wanted[1] else None, ldx=k, wt=wt.data_ptr() if wanted[0] else None,
                             ldwt=wt.stride(0), wt_scale=wts.data_ptr() if wanted[0] else None, lddx=k + 3, lddw=k + 3,
                             dw_type=2, workspace=work.data_ptr(), workspace_bytes=need)
    import ctypes
    a.struct_size = ctypes.sizeof(a)
    for name, want, o in zip(("dx", "dw", "dbias"), wanted, out):
        setattr(a, name, o.data_ptr() if want else None)
    assert pkg.lib().gemm_sm100a_int8_linear_backward(bytes(a), torch.cuda.current_stream().cuda_stream) == pkg.OK
    for want, o, f in zip(wanted, out, full):
        part = o[tuple(slice(0, s) for s in f.shape)]
        if want:
            assert torch.equal(part, f)
            part.fill_(5.0)
        assert (o == 5.0).all()
    assert (work[need:] == 77).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("over", ["x", "dy", "dw"])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_backward_over_its_inputs(pkg, cuda, dtype, over, p):
    """dX in the place of X or of dY, and dX in the place of dY with dW in the place of X."""
    import ctypes
    m = n = k = 96
    dy, x = normal((m, n), 1, dtype), normal((m, k), 2, dtype)
    wt, wts = pkg.quantize_int8(normal((n, k), 3, scale=0.02), transpose=True)
    drop = pkg.Dropout(p, seed=8) if p else None
    want = pkg.linear_int8_backward(dy, x, wt, wts, dropout=drop, dw_dtype=dtype)
    dx = x if over == "x" else dy
    dw = x if over == "dw" else torch.empty((n, k), dtype=dtype, device="cuda")
    db = torch.empty((n,), device="cuda")
    need = pkg.lib().gemm_sm100a_int8_backward_workspace(m, n, k)
    work = torch.empty((need,), dtype=torch.uint8, device="cuda")
    code = TYPES.index(dtype)
    a = pkg.Int8BackwardArgs(struct_size=0, type=code, m=m, n=n, k=k, dy=dy.data_ptr(), lddy=n, x=x.data_ptr(), ldx=k,
                             wt=wt.data_ptr(), ldwt=wt.stride(0), wt_scale=wts.data_ptr(), dx=dx.data_ptr(), lddx=k,
                             dw=dw.data_ptr(), lddw=k, dbias=db.data_ptr(), dw_type=code, workspace=work.data_ptr(),
                             workspace_bytes=need)
    a.struct_size = ctypes.sizeof(a)
    a.drop.p, a.drop.seed, a.drop.row_elems = p, 8, n
    assert pkg.lib().gemm_sm100a_int8_linear_backward(bytes(a), torch.cuda.current_stream().cuda_stream) == pkg.OK
    for got, t in zip((dx, dw, db), want):
        assert torch.equal(got, t)


def test_backward_of_no_tokens(pkg, cuda):
    wt, wts = pkg.quantize_int8(normal((20, 30), 3), transpose=True)
    dx, dw, db = pkg.linear_int8_backward(torch.empty((0, 20), device="cuda"), torch.empty((0, 30), device="cuda"), wt, wts)
    assert dx.shape == (0, 30) and (dw == 0).all() and dw.shape == (20, 30) and (db == 0).all()


# ------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (33, 1001), (5, 8192), (1000, 24), (2, 30000), (70000, 3)])
@pytest.mark.parametrize("p", [0.1, 0.5, 1.0])
def test_dropout(pkg, cuda, dtype, rows, cols, p):
    x, residual = normal((rows, cols), 1, dtype), normal((rows, cols), 2, dtype)
    drop = pkg.Dropout(p, seed=123456789, stream_id=1)
    keep = ref_keep(rows, cols, drop).cuda()
    grow = 0.0 if p == 1.0 else 1.0 / (1.0 - p)
    y = pkg.dropout(x, drop)
    want = torch.where(keep, x.double() * grow, 0.0)
    assert ((y == 0) | keep).all()
    check_close(y, want, want.abs())
    check_close(pkg.dropout(x, drop, residual=residual), want + residual.double(), want.abs() + residual.double().abs())


@pytest.mark.parametrize("p,kept", [(1e-12, True), (1.0 - 1e-12, False)])
def test_dropout_next_to_none_and_all(pkg, cuda, p, kept):
    """Probabilities that round to 0 and to 1 in steps of 2^-32."""
    x = normal((30, 50), 1)
    x[0, 0] = float("nan")
    y = pkg.dropout(x, pkg.Dropout(p))
    q, s = pkg.quantize_int8(x[1:], dropout=pkg.Dropout(p))
    d = pkg.gemm_int8(q, None, q, None, dropout=pkg.Dropout(p))
    if kept:
        assert torch.equal(y[1:], x[1:]) and torch.isnan(y[0, 0])
        assert torch.equal(q, pkg.quantize_int8(x[1:])[0]) and torch.equal(d, pkg.gemm_int8(q, None, q, None))
    else:
        assert (y == 0).all() and (q == 0).all() and (d == 0).all()


def test_dropout_rate(pkg, cuda):
    """Kept words are uniform: 4e6 draws, five standard deviations of the binomial."""
    n = 4_000_000
    y = pkg.dropout(torch.ones((2000, 2000), device="cuda"), pkg.Dropout(0.3, seed=5))
    kept = (y != 0).sum().item()
    assert abs(kept - 0.7 * n) <= 5 * math.sqrt(n * 0.3 * 0.7)


def test_dropout_slices_are_parts_of_one_mask(pkg, cuda):
    """Ranks that own column or row slices draw exactly their part."""
    x = normal((100, 640), 1)
    whole = pkg.dropout(x, pkg.Dropout(0.4, seed=8))
    for c0, c1 in ((0, 320), (320, 640), (1, 4), (333, 640)):
        part = pkg.dropout(x[:, c0:c1], pkg.Dropout(0.4, seed=8, col0=c0, row_elems=640))
        assert torch.equal(part, whole[:, c0:c1])
    part = pkg.dropout(x[37:], pkg.Dropout(0.4, seed=8, row0=37))
    assert torch.equal(part, whole[37:])
    assert not torch.equal(pkg.dropout(x, pkg.Dropout(0.4, seed=9)), whole)
    assert not torch.equal(pkg.dropout(x, pkg.Dropout(0.4, seed=8, stream_id=1)), whole)


def test_dropout_far_indices(pkg, cuda):
    """Element indices beyond 32 and close to 62 bits."""
    x = normal((4, 100), 1)
    for drop in (pkg.Dropout(0.5, seed=1, row0=2 ** 40, col0=7, row_elems=2 ** 21 + 1),
                 pkg.Dropout(0.5, seed=2 ** 64 - 1, stream_id=2 ** 64 - 1, row0=2 ** 33, row_elems=101)):
        keep = ref_keep(4, 100, drop).cuda()
        assert torch.equal(pkg.dropout(x, drop) != 0, keep)


def test_dropout_masks_nan_and_inf(pkg, cuda):
    drop = pkg.Dropout(0.5, seed=4)
    keep = ref_keep(16, 64, drop).cuda()
    for bad in (float("nan"), float("inf")):
        y = pkg.dropout(torch.full((16, 64), bad, device="cuda"), drop)
        assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()


def test_dropout_in_place_strided_and_empty(pkg, cuda):
    base = normal((40, 130), 1, torch.bfloat16)
    drop = pkg.Dropout(0.3, seed=4)
    x = base[:, 1:102]
    want = pkg.dropout(x.contiguous(), drop)
    assert torch.equal(pkg.dropout(x, drop), want)
    before = base.clone()
    pkg.dropout(x, drop, out=x)
    assert torch.equal(x, want)
    assert torch.equal(base[:, :1], before[:, :1]) and torch.equal(base[:, 102:], before[:, 102:])
    assert pkg.dropout(torch.empty((0, 5), device="cuda"), drop).shape == (0, 5)
    assert torch.equal(pkg.dropout(before, pkg.Dropout(0.0)), before)


def test_outputs_beside_and_over_other_operands(pkg, cuda):
    """Columns of one buffer and rows behind one another are apart; a shifted overlap is refused and
    leaves everything as it was."""
    drop = pkg.Dropout(0.3, seed=4)
    m, n, k = 20, 64, 128
    buf = normal((m, 3 * n), 1, torch.bfloat16)
    first = buf.clone()
    x, y, z = buf[:, :n], buf[:, n:2 * n], buf[:, 2 * n:]
    want = pkg.dropout(x.contiguous(), drop, residual=z.contiguous())
    assert torch.equal(pkg.dropout(x, drop, residual=z, out=y), want)
    a, b, sa, sb = int8s(pkg, m, k, 1), int8s(pkg, n, k, 2), scales(m, 3), scales(n, 4)
    want = pkg.gemm_int8(a, sa, b, sb, residual=z.contiguous())
    assert torch.equal(pkg.gemm_int8(a, sa, b, sb, residual=z, out=y), want)
    assert torch.equal(buf[:, :n], first[:, :n]) and torch.equal(buf[:, 2 * n:], first[:, 2 * n:])
    rows = first.clone()
    w, ws = pkg.quantize_int8(normal((n, n), 5))
    for call in (lambda: pkg.dropout(rows[:, :n], drop, out=rows[:, 1:n + 1]),
                 lambda: pkg.dropout(rows[:-1], drop, out=rows[1:]),
                 lambda: pkg.dropout(rows[:, n:2 * n], drop, residual=rows[:, :n], out=rows[:, 8:n + 8]),
                 lambda: pkg.gemm_int8(a, sa, b, sb, residual=rows[:, :n], out=rows[:, 8:n + 8]),
                 lambda: pkg.linear_int8(rows[:8, :n], w, ws, residual=rows[:8, :n], out=rows[1:9, :n])):
        with pytest.raises(pkg.GemmError):
            call()
    assert torch.equal(rows, first)


def test_dropout_seed_from_the_device(pkg, cuda):
    x = normal((50, 100), 1)
    word = torch.tensor([41], dtype=torch.int64, device="cuda")
    y = pkg.dropout(x, pkg.Dropout(0.5, seed=word))
    assert torch.equal(y, pkg.dropout(x, pkg.Dropout(0.5, seed=41)))
    word += 1
    assert torch.equal(pkg.dropout(x, pkg.Dropout(0.5, seed=word)), pkg.dropout(x, pkg.Dropout(0.5, seed=42)))


def test_dropout_gradient_against_differences(pkg, cuda):
    """y is linear in x: the gradient of sum(dy * y) is the same map of dy."""
    x, dy = normal((8, 33), 1), normal((8, 33), 2)
    drop = pkg.Dropout(0.3, seed=6)
    dx = pkg.dropout(dy, drop).double()
    for i, j in ((0, 0), (3, 32), (7, 16), (5, 5)):
        e = torch.zeros_like(x)
        e[i, j] = 1.0
        diff = (dy.double() * (pkg.dropout(x + e, drop).double() - pkg.dropout(x - e, drop).double())).sum() / 2
        # x + e and its product each round once: 2^-24 of values below 8 / (1 - p), times |dy|
        assert abs(dx[i, j].item() - diff.item()) <= 16 * U32 * 8 / 0.7 * dy.abs().max().item()


# ------------------------------------------------------------------ together
def test_training_step_of_a_residual_block(pkg, cuda):
    """quantise -> product with bias, dropout and residual -> gradients -> update, then a decoding
    step with the new weights: each call against 64 bits on the same intermediate values."""
    m, n, k = 150, 256, 320
    x = normal((m, k), 1, torch.bfloat16)
    w = normal((n, k), 2, scale=0.05)
    bias = normal((n,), 3)
    residual = normal((m, n), 4, torch.bfloat16)
    dy = normal((m, n), 5, torch.bfloat16)
    for step in range(2):
        drop = pkg.Dropout(0.1, seed=100 + step)
        wq, ws = pkg.quantize_int8(w)
        wt, wts = pkg.quantize_int8(w, transpose=True)
        check_quantized(wq, ws, w)
        check_quantized(wt, wts, w.t())
        y = pkg.linear_int8(x, wq, ws, bias=bias, dropout=drop, residual=residual)
        check_close(y, *ref_product(*ref_quantize(x), wq, ws, bias, residual, drop), scale_err=U32)
        dx, dw, db = pkg.linear_int8_backward(dy, x, wt, wts, dropout=drop)
        dz = torch.where(ref_keep(m, n, drop).cuda(), dy.double(), 0.0)
        qz, sz = ref_quantize(dz)
        check_close(dx, *ref_product(qz, sz / 0.9, wt, wts), scale_err=4 * U32)
        qt, st = ref_quantize(dz.t())
        qx, sx = ref_quantize(x.t())
        check_close(dw, *ref_product(qt, st / 0.9, qx, sx), scale_err=4 * U32)
        w = w - 0.01 * dw
        bias = bias - 0.01 * db
    wq, ws = pkg.quantize_int8(w)
    full = pkg.linear_int8(x, wq, ws, bias=bias)
    for t in (0, 77, m - 1):
        assert torch.equal(pkg.linear_int8(x[t:t + 1], wq, ws, bias=bias), full[t:t + 1])


def test_graph_capture_with_device_seed(pkg, cuda):
    """A captured forward and backward pass replays the direct result, and the next seed's mask."""
    m, n, k = 96, 300, 256
    x, dy = normal((m, k), 1, torch.bfloat16), normal((m, n), 2, torch.bfloat16)
    w = normal((n, k), 3, scale=0.05)
    wq, ws = pkg.quantize_int8(w)
    wt, wts = pkg.quantize_int8(w, transpose=True)
    word = torch.tensor([7], dtype=torch.int64, device="cuda")

    def step(seed):
        drop = pkg.Dropout(0.2, seed=seed)
        y = pkg.linear_int8(x, wq, ws, dropout=drop)
        one = pkg.linear_int8(x[:1], wq, ws)
        return (y, one, pkg.dropout(y, drop)) + pkg.linear_int8_backward(dy, x, wt, wts, dropout=drop)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        direct = [step(7), step(8)]
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step(word)
    for want in direct:
        for t in out:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for t, v in zip(out, want):
            assert torch.equal(t, v)
        word += 1
    del graph


def test_two_streams_at_once(pkg, cuda):
    x = normal((64, 2048), 1, torch.bfloat16)
    w, ws = pkg.quantize_int8(normal((4096, 2048), 2, scale=0.05))
    want = pkg.linear_int8(x, w, ws)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(pkg.linear_int8(x, w, ws))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_each_call_sees_the_call_before_it(pkg, cuda):
    """Launches overlap: every operand is written by the kernel just before the one that reads it
    (weights, tokens, scales, residual, output read by torch), over and over in the same buffers."""
    m, n, k = 24, 640, 768
    w = torch.empty((n, k), device="cuda")
    x = torch.empty((m, k), device="cuda", dtype=torch.bfloat16)
    ws, xs, outs = [normal((n, k), 10 + i, scale=0.05) for i in range(6)], [normal((m, k), 20 + i, torch.bfloat16) for i in range(6)], []
    for rows in (m, 2):
        direct = []
        for i in range(6):
            q, s = pkg.quantize_int8(ws[i])
            torch.cuda.synchronize()
            y = pkg.linear_int8(xs[i][:rows], q, s)
            torch.cuda.synchronize()
            y = pkg.dropout(y, pkg.Dropout(0.5, seed=i))
            z, zs = pkg.quantize_int8(y, transpose=True)
            torch.cuda.synchronize()
            direct.append((y.clone(), z.clone(), zs.clone()))
        torch.cuda.synchronize()
        outs = []
        for _ in range(20):
            for i in range(6):
                w.copy_(ws[i])
                x.copy_(xs[i])
                q, s = pkg.quantize_int8(w)
                y = pkg.linear_int8(x[:rows], q, s)
                pkg.dropout(y, pkg.Dropout(0.5, seed=i), out=y)
                z, zs = pkg.quantize_int8(y, transpose=True)
                outs.append((y.clone(), z.clone(), zs.clone()))
                del q, s, y, z, zs
        for j, got in enumerate(outs):
            for a, b in zip(got, direct[j % 6]):
                assert torch.equal(a, b), (rows, j)


def test_capture_across_streams(pkg, cuda):
    """Calls captured on two streams that fork and join, and a graph whose nodes are other kernels
    between them."""
    x = normal((40, 512), 1, torch.bfloat16)
    wq, ws = pkg.quantize_int8(normal((300, 512), 2, scale=0.05))
    drop = pkg.Dropout(0.3, seed=1)

    def step(side):
        main = torch.cuda.current_stream()
        a = pkg.linear_int8(x, wq, ws)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            b = pkg.dropout(a, drop)
            qb, sb = pkg.quantize_int8(b, transpose=True)
        c = pkg.linear_int8(x[:3], wq, ws)
        d = (a * 2).contiguous()
        main.wait_stream(side)
        e = pkg.dropout(d, drop, residual=b)
        return a, b, qb, sb, c, e

    side, stream = torch.cuda.Stream(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = [t.clone() for t in step(side)]
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step(side)
    for _ in range(3):
        for t in out:
            t.fill_(1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    del graph


def test_strides_beyond_32_bits(pkg, cuda):
    """Rows 2^30 elements apart: offsets of 2^31 elements and more in every operand."""
    m, n, k, far = 3, 150, 160, 2 ** 30
    big = torch.empty((2 * far + 512,), dtype=torch.bfloat16, device="cuda")
    big8 = torch.empty((2 * far + 512,), dtype=torch.int8, device="cuda")

    def spread(t, store):
        v = store.as_strided((t.shape[0], t.shape[1]), (far, 1))
        v.copy_(t)
        return v

    x = normal((m, k), 1, torch.bfloat16)
    q, s = pkg.quantize_int8(x)
    qt, st = pkg.quantize_int8(x, transpose=True)
    fx = spread(x, big)
    for t, want, scale in ((False, q, s), (True, qt, st)):
        got = pkg.quantize_int8(fx, transpose=t)
        assert torch.equal(got[0], want) and torch.equal(got[1], scale)
    drop = pkg.Dropout(0.4, seed=2, row_elems=far)
    want = pkg.dropout(x, drop)
    assert torch.equal(pkg.dropout(fx, drop), want)
    pkg.dropout(fx, drop, out=fx)
    assert torch.equal(fx, want)
    w, ws = pkg.quantize_int8(normal((n, k), 3, scale=0.05))
    y = pkg.gemm_int8(q, s, w, ws)
    fq = spread(q, big8)
    assert torch.equal(pkg.gemm_int8(fq, s, w, ws), y)
    for kn in (dict(), dict(cta_group=2, tile_n=128), dict(cta_group=1, tile_n=16, split_k=2)):
        out = spread(torch.zeros((m, n), dtype=torch.bfloat16, device="cuda"), big)
        pkg.gemm_int8(q, s, w, ws, residual=out, out=out, **kn)
        assert torch.equal(out, y), kn
    assert torch.equal(pkg.linear_int8(spread(x, big), w, ws), pkg.linear_int8(x, w, ws))
    w3, ws3 = w[:3], ws[:3]
    assert torch.equal(pkg.gemm_int8(q, s, spread(w3, big8), ws3), y[:, :3])


def test_host_memory_is_refused(pkg, cuda):
    """A pointer to host memory is an error of the call, before any launch."""
    L = pkg.lib()
    host = torch.zeros((64,), dtype=torch.bfloat16)
    x = normal((2, 16), 1, torch.bfloat16)
    a = pkg.DropoutOpArgs(struct_size=128, type=0, rows=2, cols=16, x=x.data_ptr(), ldx=16, y=host.data_ptr(), ldy=16)
    assert L.gemm_sm100a_dropout(bytes(a), torch.cuda.current_stream().cuda_stream) == pkg.ERR_LAUNCH
    torch.cuda.synchronize()
    assert torch.equal(pkg.dropout(x, pkg.Dropout(0.0)), x)


@pytest.mark.parametrize("dtype", [torch.float64, torch.int8, torch.int32, torch.bool, torch.complex64, torch.float8_e4m3fn])
def test_other_types_are_refused(pkg, cuda, dtype):
    """Tensors on the device, of types that no kernel reads."""
    bad, good = torch.zeros((4, 64), device="cuda").to(dtype), torch.zeros((4, 64), device="cuda")
    w, ws = pkg.quantize_int8(torch.ones((64, 64), device="cuda"))
    for call in (lambda: pkg.quantize_int8(bad), lambda: pkg.quantize_int8(bad, transpose=True),
                 lambda: pkg.linear_int8(bad, w, ws), lambda: pkg.linear_int8(good, w, ws, bias=bad[0]),
                 lambda: pkg.linear_int8(good, w, ws, residual=bad), lambda: pkg.linear_int8(good, w, ws, out=bad),
                 lambda: pkg.linear_int8(good, w, bad[0]), lambda: pkg.dropout(bad, pkg.Dropout(0.5)),
                 lambda: pkg.dropout(good, pkg.Dropout(0.5), residual=bad), lambda: pkg.dropout(good, pkg.Dropout(0.5), out=bad),
                 lambda: pkg.linear_int8_backward(bad, good, w, ws), lambda: pkg.linear_int8_backward(good, bad, w, ws),
                 lambda: pkg.linear_int8_backward(good, good, w, ws, dw_dtype=dtype),
                 lambda: pkg.gemm_int8(w, ws, w, ws, out_dtype=dtype)):
        with pytest.raises(ValueError):
            call()
    if dtype != torch.int8:
        with pytest.raises(ValueError):
            pkg.linear_int8(good, torch.zeros((64, 64), device="cuda").to(dtype), ws)


def test_out_of_memory_is_the_frameworks_own_error(pkg, cuda):
    with pytest.raises(torch.OutOfMemoryError):
        pkg.empty_int8(1 << 20, 1 << 22, cuda)


def test_knobs_beyond_32_bits_are_refused(pkg, cuda):
    a, b = int8s(pkg, 4, 64, 0), int8s(pkg, 5, 64, 1)
    for knob in ("tile_n", "cta_group", "split_k", "timeout_ms", "flags"):
        for value in (2 ** 32, -1):
            with pytest.raises(ValueError, match=knob):
                pkg.gemm_int8(a, None, b, None, **{knob: value})
