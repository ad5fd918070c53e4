"""CPU tests of the int8 operators' argument checks (no kernel launches): every
refusal happens before any CUDA call, with a reason."""
import ctypes as C

import pytest
import torch


def _gemm(pkg, **kw):
    a = pkg.Int8GemmArgs()
    a.struct_size = C.sizeof(pkg.Int8GemmArgs)
    base = dict(d_type=0, m=64, n=128, k=256, a=0x10000, lda=256, b=0x20000, ldb=256, d=0x30000, ldd=128,
                scale_a=0x40000, scale_b=0x50000)
    base.update(kw)
    for name, v in base.items():
        if name.startswith("drop_"):
            setattr(a.drop, name[5:], v)
        else:
            setattr(a, name, v)
    return a


def test_structs_have_the_sizes_of_the_header(pkg, tmp_path):
    """The ctypes views against a C compiler's layout of the header."""
    import subprocess
    from pathlib import Path
    names = ["DropoutArgs", "Int8GemmArgs", "Int8QuantArgs", "Int8BackwardArgs", "DropoutOpArgs"]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "gemm_sm100a.h"\nint main(void) {'
                   + "".join(f' printf("%zu ", sizeof({n}));' for n in names)
                   + ' printf("%zu %zu %zu", offsetof(Int8GemmArgs, drop), offsetof(Int8QuantArgs, drop),'
                     ' offsetof(Int8BackwardArgs, drop)); return 0; }\n')
    root = Path(__file__).resolve().parent.parent
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", f"-I{root / 'include'}", str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got[:5] == [C.sizeof(getattr(pkg, n)) for n in names]
    assert got[5:] == [pkg.Int8GemmArgs.drop.offset, pkg.Int8QuantArgs.drop.offset, pkg.Int8BackwardArgs.drop.offset]


def test_a_plain_problem_is_accepted(pkg):
    rc, info = pkg.query_int8(_gemm(pkg))
    assert rc == pkg.OK and info.can_implement == 1


@pytest.mark.parametrize("kw,rc,frag", [
    (dict(struct_size=8), "bad", b"struct_size"),
    (dict(a=None), "bad", b"null"),
    (dict(d=None), "bad", b"null"),
    (dict(d_type=3), "no", b"d_type"),
    (dict(bias=0x60000, bias_type=7), "no", b"bias_type"),
    (dict(k=0), "no", b"empty"),
    (dict(m=-1), "no", b"empty"),
    (dict(k=131072, lda=131072, ldb=131072), "no", b"131071"),
    (dict(m=1 << 31), "no", b"too large"),
    (dict(a=0x10008), "no", b"16-byte"),
    (dict(lda=240), "no", b"lda"),
    (dict(k=250, lda=250, ldb=256), "no", b"multiples of 16"),
    (dict(ldd=127), "no", b"ldd"),
    (dict(d=0x30001), "no", b"element"),
    (dict(c=0x60000, ldc=100), "no", b"ldc"),
    (dict(scale_a=0x40002), "no", b"scales"),
    (dict(bias=0x60001), "no", b"bias"),
    (dict(flags=2), "no", b"flags"),
    (dict(drop_p=-0.1), "no", b"dropout p"),
    (dict(drop_p=float("nan")), "no", b"dropout p"),
    (dict(drop_p=0.5, drop_row_elems=127), "no", b"row_elems"),
    (dict(drop_p=0.5, drop_row_elems=200, drop_col0=100), "no", b"row_elems"),
    (dict(drop_p=0.5, drop_row_elems=128, drop_row0=-1), "no", b"row0"),
    (dict(drop_p=0.5, drop_row_elems=128, drop_row0=1 << 60), "no", b"2^62"),
    (dict(drop_p=0.5, drop_row_elems=128, drop_seed_offset=0x60004), "no", b"seed_offset"),
])
def test_refused_products(pkg, kw, rc, frag):
    got, info = pkg.query_int8(_gemm(pkg, **kw))
    assert got == (pkg.ERR_BAD_ARGS if rc == "bad" else pkg.ERR_CANNOT_IMPLEMENT)
    assert frag in info.reason, info.reason
    assert info.can_implement == 0
    L = pkg.lib()
    assert L.gemm_sm100a_int8_launch(bytes(_gemm(pkg, **kw)), None) == got
    assert L.gemm_sm100a_int8_linear(bytes(_gemm(pkg, **kw)), C.c_void_p(0x70000), 0, 256, None) == got


@pytest.mark.parametrize("d_type", [0, 1, 2])
@pytest.mark.parametrize("knobs", [dict()] + [dict(cta_group=1, tile_n=bn, split_k=s) for bn in (16, 32, 64, 128)
                                              for s in (1, 2, 4, 8)] + [dict(cta_group=2, tile_n=bn) for bn in (128, 256)])
def test_one_cta_per_sm(pkg, d_type, knobs):
    """CTAs of a split or a pair wait for one another and, without a limit, for tensor memory: two kernels must
    not share SMs, or each could hold what the other one waits for.  An SM has 228 KiB of shared memory."""
    for k in (1024, 1152, 4096, 20000):
        for c in (None, 0x60000):
            rc, info = pkg.query_int8(_gemm(pkg, k=k, lda=20480, ldb=20480, d_type=d_type, c=c, ldc=128, **knobs))
            assert rc == pkg.OK and 2 * info.smem_bytes > 228 * 1024 and info.smem_bytes <= 227 * 1024


# (offset of the output behind the operand in elements, its stride, whether they share an element), for 4 rows of
# 32 elements with a stride of 80: in place, shifted by less than a row, side by side, one element too near, one or
# more rows further down, right behind, and with a stride of its own.
OVERLAPS = [(0, 80, False), (1, 80, True), (-1, 80, True), (31, 80, True), (32, 80, False), (48, 80, False), (49, 80, True),
            (80, 80, True), (-80, 80, True), (240, 80, True), (241, 80, True), (272, 80, False), (320, 80, False),
            (-240, 80, True), (-272, 80, False), (-271, 80, True), (0, 88, True), (32, 88, False), (32, 160, False),
            (32, 112, True), (272, 88, False)]


def _rows(start, ld):
    return {start + i * ld + j for i in range(4) for j in range(32)}


@pytest.mark.parametrize("offset,ld,meet", OVERLAPS)
def test_outputs_over_other_operands(pkg, offset, ld, meet):
    """In place or apart; anything between is refused.  (No device memory is behind the addresses: what is
    accepted ends at the search for the output's device.)"""
    assert meet == (offset != 0 and not _rows(0, 80).isdisjoint(_rows(offset, ld)) or (offset == 0 and ld != 80))
    L, at, out = pkg.lib(), 0x100000, 0x100000 + 2 * offset
    want = pkg.ERR_CANNOT_IMPLEMENT if meet else pkg.ERR_LAUNCH
    far = dict(residual=0x400000, ldr=32)
    assert L.gemm_sm100a_dropout(bytes(_drop(pkg, rows=4, x=at, ldx=80, y=out, ldy=ld)), None) == want
    assert L.gemm_sm100a_dropout(bytes(_drop(pkg, rows=4, x=at, ldx=80, y=out, ldy=ld, **far)), None) == want
    assert L.gemm_sm100a_dropout(bytes(_drop(pkg, rows=4, x=0x400000, ldx=32, residual=at, ldr=80, y=out, ldy=ld)), None) == want
    args = _gemm(pkg, m=4, n=32, c=at, ldc=80, d=out, ldd=ld)
    rc, info = pkg.query_int8(args)
    assert (rc, b"apart" in info.reason) == ((pkg.ERR_CANNOT_IMPLEMENT, True) if meet else (pkg.OK, False))
    assert L.gemm_sm100a_int8_launch(bytes(args), None) == want


def test_overlap_against_sets_of_elements(pkg):
    """The refusal of C over D for random small matrices in one buffer, equal strides and others."""
    import random
    rng = random.Random(5)
    seen = [0, 0]
    for _ in range(4000):
        m, n = rng.randint(1, 6), rng.randint(1, 9)
        ldc = n + rng.choice([0, 1, 3, n, 2 * n])
        ldd = ldc if rng.random() < 0.5 else n + rng.choice([0, 1, 2, n, 3 * n])
        shift = rng.randint(-m * ldd - 2, m * ldc + 2)
        c = {i * ldc + j for i in range(m) for j in range(n)}
        d = {shift + i * ldd + j for i in range(m) for j in range(n)}
        same = shift == 0 and (ldc == ldd or m == 1)
        rc, _ = pkg.query_int8(_gemm(pkg, m=m, n=n, c=0x100000, ldc=ldc, d=0x100000 + 2 * shift, ldd=ldd))
        fine = same or c.isdisjoint(d)
        assert rc == (pkg.OK if fine else pkg.ERR_CANNOT_IMPLEMENT), (m, n, ldc, ldd, shift)
        seen[fine] += 1
    assert min(seen) > 500


def test_null_argument_blocks(pkg):
    L = pkg.lib()
    assert L.gemm_sm100a_int8_launch(None, None) == pkg.ERR_BAD_ARGS
    assert L.gemm_sm100a_quantize_int8(None, None) == pkg.ERR_BAD_ARGS
    assert L.gemm_sm100a_dropout(None, None) == pkg.ERR_BAD_ARGS
    assert L.gemm_sm100a_int8_linear_backward(None, None) == pkg.ERR_BAD_ARGS


def test_empty_products_launch_nothing(pkg):
    L = pkg.lib()
    for kw in (dict(m=0), dict(n=0)):
        assert L.gemm_sm100a_int8_launch(bytes(_gemm(pkg, **kw)), None) == pkg.OK
        assert L.gemm_sm100a_int8_linear(bytes(_gemm(pkg, **kw)), C.c_void_p(0x70000), 0, 256, None) == pkg.OK


@pytest.mark.parametrize("x,x_type,ldx", [(None, 0, 256), (0x70000, 5, 256), (0x70000, 0, 255), (0x70001, 0, 256)])
def test_linear_refuses_bad_tokens(pkg, x, x_type, ldx):
    assert pkg.lib().gemm_sm100a_int8_linear(bytes(_gemm(pkg)), C.c_void_p(x), x_type, ldx, None) in (
        pkg.ERR_BAD_ARGS, pkg.ERR_CANNOT_IMPLEMENT)


def _linear(pkg, x, ldx, **kw):
    """A linear layer of few tokens without a workspace.  No device memory is behind the addresses, so a call
    that is accepted ends at the search for D's device."""
    args = _gemm(pkg, a=None, scale_a=None, **kw)
    return pkg.lib().gemm_sm100a_int8_linear(bytes(args), C.c_void_p(x), 0, ldx, None)


def test_linear_over_its_tokens_needs_a_workspace(pkg):
    """In one launch a CTA would store D where another one still reads its tokens."""
    kw = dict(m=3, n=256, k=256, d=0x100000, ldd=256)
    assert _linear(pkg, 0x200000, 256, **kw) == pkg.ERR_LAUNCH                # apart
    assert _linear(pkg, 0x100000 + 3 * 512, 256, **kw) == pkg.ERR_LAUNCH      # right behind D
    assert _linear(pkg, 0x100000, 256, **kw) == pkg.ERR_BAD_ARGS              # in place
    assert _linear(pkg, 0x100000 + 3 * 512 - 2, 256, **kw) == pkg.ERR_BAD_ARGS
    assert _linear(pkg, 0x100000 - 3 * 512 + 2, 256, **kw) == pkg.ERR_BAD_ARGS
    assert _linear(pkg, 0x100000 - 3 * 512, 256, **kw) == pkg.ERR_LAUNCH
    # columns of one buffer: side by side, and one element too near
    assert _linear(pkg, 0x100000 - 8, 256, **dict(kw, n=0, ldd=0)) == pkg.OK   # no D at all
    kw["ldd"] = 600
    assert _linear(pkg, 0x100000 + 512, 600, **kw) == pkg.ERR_LAUNCH
    assert _linear(pkg, 0x100000 + 510, 600, **kw) == pkg.ERR_BAD_ARGS
    assert _linear(pkg, 0x100000 + 688, 600, **kw) == pkg.ERR_LAUNCH
    assert _linear(pkg, 0x100000 + 690, 600, **kw) == pkg.ERR_BAD_ARGS        # its rows end in D's next ones


def _quant(pkg, **kw):
    a = pkg.Int8QuantArgs()
    a.struct_size = C.sizeof(pkg.Int8QuantArgs)
    base = dict(x_type=0, rows=8, cols=32, x=0x10000, ldx=32, q=0x20000, ldq=32, scale=0x30000)
    base.update(kw)
    for name, v in base.items():
        if name.startswith("drop_"):
            setattr(a.drop, name[5:], v)
        else:
            setattr(a, name, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(struct_size=4), dict(x_type=3), dict(x_type=-1), dict(rows=-1), dict(cols=1 << 31), dict(x=None), dict(q=None),
    dict(scale=None), dict(col_sums=0x40000), dict(ldx=31), dict(x=0x10001), dict(ldq=40), dict(ldq=16), dict(q=0x20008),
    dict(scale=0x30002), dict(drop_p=2.0), dict(drop_p=0.5, drop_row_elems=31), dict(transpose=1, rows=40, ldq=32),
])
def test_refused_quantisations(pkg, kw):
    rc = pkg.lib().gemm_sm100a_quantize_int8(bytes(_quant(pkg, **kw)), None)
    assert rc in (pkg.ERR_BAD_ARGS, pkg.ERR_CANNOT_IMPLEMENT)


def _backward(pkg, **kw):
    a = pkg.Int8BackwardArgs()
    a.struct_size = C.sizeof(pkg.Int8BackwardArgs)
    base = dict(type=0, m=8, n=32, k=48, dy=0x10000, lddy=32, x=0x20000, ldx=48, wt=0x30000, ldwt=32, wt_scale=0x40000,
                dx=0x50000, lddx=48, dw=0x60000, lddw=48, dbias=0x70000, dw_type=2, workspace=0x80000,
                workspace_bytes=1 << 20)
    base.update(kw)
    for name, v in base.items():
        if name.startswith("drop_"):
            setattr(a.drop, name[5:], v)
        else:
            setattr(a, name, v)
    return a


def test_backward_workspace(pkg):
    size = pkg.lib().gemm_sm100a_int8_backward_workspace
    assert size(8, 32, 48) >= 8 * 32 + 32 * 8 + 48 * 8 + 4 * (8 + 32 + 48)
    assert size(131071, 131071, 1) > 0
    assert size(131072, 1, 1) == -1 and size(1, 131072, 1) == -1 and size(-1, 1, 1) == -1


@pytest.mark.parametrize("kw", [
    dict(struct_size=4), dict(type=3), dict(dw_type=-1), dict(m=-1), dict(n=0), dict(k=0), dict(m=131072), dict(n=131072),
    dict(dy=None), dict(x=None), dict(wt=None), dict(wt_scale=None), dict(workspace=None), dict(workspace_bytes=100),
    dict(dy=0x10001), dict(x=0x20001), dict(wt=0x30008), dict(dx=0x50001), dict(dw=0x60002), dict(dbias=0x70002),
    dict(workspace=0x80008), dict(lddy=31), dict(ldx=47), dict(ldwt=31), dict(ldwt=40), dict(lddx=47), dict(lddw=47),
    dict(drop_p=1.5), dict(drop_p=0.5, drop_row_elems=8),
])
def test_refused_backward_passes(pkg, kw):
    rc = pkg.lib().gemm_sm100a_int8_linear_backward(bytes(_backward(pkg, **kw)), None)
    assert rc in (pkg.ERR_BAD_ARGS, pkg.ERR_CANNOT_IMPLEMENT)


def test_a_backward_pass_of_nothing_launches_nothing(pkg):
    assert pkg.lib().gemm_sm100a_int8_linear_backward(bytes(_backward(pkg, dx=None, dw=None, dbias=None)), None) == pkg.OK


def _drop(pkg, **kw):
    a = pkg.DropoutOpArgs()
    a.struct_size = C.sizeof(pkg.DropoutOpArgs)
    base = dict(type=0, rows=8, cols=32, x=0x10000, ldx=32, y=0x20000, ldy=32, drop_p=0.5, drop_row_elems=32)
    base.update(kw)
    for name, v in base.items():
        if name.startswith("drop_"):
            setattr(a.drop, name[5:], v)
        else:
            setattr(a, name, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(struct_size=4), dict(type=3), dict(rows=-1), dict(x=None), dict(y=None), dict(ldx=31), dict(ldy=16),
    dict(residual=0x30000, ldr=8), dict(residual=0x30001, ldr=32), dict(x=0x10001), dict(drop_p=1.5),
    dict(drop_row_elems=16), dict(drop_col0=-2), dict(drop_seed_offset=0x50001),
])
def test_refused_dropouts(pkg, kw):
    rc = pkg.lib().gemm_sm100a_dropout(bytes(_drop(pkg, **kw)), None)
    assert rc in (pkg.ERR_BAD_ARGS, pkg.ERR_CANNOT_IMPLEMENT)


def test_python_helpers_refuse_host_tensors(pkg):
    """There is no CPU path: a host tensor is an error, not a fallback."""
    x = torch.zeros((4, 32))
    q = torch.zeros((4, 32), dtype=torch.int8)
    s = torch.ones(4)
    with pytest.raises(ValueError):
        pkg.quantize_int8(x)
    with pytest.raises(ValueError):
        pkg.gemm_int8(q, s, q, s)
    with pytest.raises(ValueError):
        pkg.linear_int8(x, q, s)
    with pytest.raises(ValueError):
        pkg.linear_int8_backward(x, x, q, s)
    with pytest.raises(ValueError):
        pkg.dropout(x, pkg.Dropout(0.5))
    with pytest.raises(ValueError):
        pkg.quantize_int8(x.to(torch.float64))
    with pytest.raises(ValueError):
        pkg.quantize_int8(x[0])


@pytest.mark.parametrize("device", ["cpu", "meta", torch.device("cpu")])
def test_int8_matrices_are_on_cuda_devices(pkg, device):
    """A device of another kind is refused, not replaced by the current CUDA device."""
    with pytest.raises(ValueError, match="CUDA"):
        pkg.empty_int8(4, 32, device)
