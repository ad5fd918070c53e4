"""CPU tests of the argument checks of the 4-bit operators and the norms (no kernel launches): every refusal happens
before any CUDA call."""
import ctypes as C

import pytest


def _fill(struct, base, kw):
    a = struct()
    a.struct_size = C.sizeof(struct)
    for name, v in {**base, **kw}.items():
        setattr(a, name, v)
    return a


def _gemm(pkg, **kw):
    return _fill(pkg.Fp4GemmArgs, dict(d_type=0, m=64, n=128, k=512, a=0x10000, lda=256, a_scales=0x20000, a_row_scale=0x30000,
                                       b=0x40000, ldb=256, b_scales=0x50000, b_row_scale=0x60000, d=0x70000, ldd=128, block=16), kw)


def _quant(pkg, **kw):
    return _fill(pkg.Fp4QuantArgs, dict(x_type=0, rows=8, cols=100, x=0x10000, ldx=100, values=0x20000, ldv=64, scales=0x30000,
                                        row_scale=0x40000, block=16), kw)


def _dequant(pkg, **kw):
    return _fill(pkg.Fp4DequantArgs, dict(y_type=0, rows=8, cols=100, y=0x10000, ldy=100, values=0x20000, ldv=64, scales=0x30000,
                                          row_scale=0x40000, block=16), kw)


def _norm(pkg, **kw):
    return _fill(pkg.ResidualNormArgs, dict(type=0, rows=8, cols=100, x=0x10000, ldx=100, y=0x20000, ldy=100, x_out=0x30000, ldo=100,
                                            h=0x40000, ldh=100, weight=0x50000, post_weight=0x60000, gate=0x70000, param_type=0, eps=1e-6, scale=1.0), kw)


def _back(pkg, **kw):
    ws = pkg.lib().gemm_sm100a_residual_norm_workspace(8, 100)
    return _fill(pkg.ResidualNormBackwardArgs, dict(type=0, rows=8, cols=100, dh=0x10000, lddh=100, dx_out=0x20000, lddo=100, x_out=0x30000,
                                                    ldo=100, y=0x40000, ldy=100, weight=0x50000, post_weight=0x60000, gate=0x70000, param_type=0,
                                                    scale=1.0, eps=1e-6, dx=0x80000, lddx=100, dy=0x90000, lddy=100, dweight=0xA0000,
                                                    dpost_weight=0xB0000, dgate=0xC0000, lddg=100, workspace=0xD0000, workspace_bytes=ws), kw)


def test_structs_have_the_sizes_of_the_header(pkg, tmp_path):
    """The ctypes views against a C compiler's layout of the header, field by field."""
    import subprocess
    from pathlib import Path
    structs = [pkg.Fp4GemmArgs, pkg.Fp4QuantArgs, pkg.Fp4DequantArgs, pkg.ResidualNormArgs, pkg.ResidualNormBackwardArgs]
    lines = []
    for s in structs:
        lines.append(f'printf("%zu ", sizeof({s.__name__}));')
        lines += [f'printf("%zu ", offsetof({s.__name__}, {name}));' for name, _ in s._fields_]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "gemm_sm100a.h"\nint main(void) {' + "\n".join(lines) + " return 0; }\n")
    root = Path(__file__).resolve().parent.parent
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", f"-I{root / 'include'}", str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for s in structs:
        want.append(C.sizeof(s))
        want += [getattr(s, name).offset for name, _ in s._fields_]
    assert got == want


@pytest.mark.parametrize("rows,cols,block,want", [(0, 100, 16, 0), (1, 1, 16, 4 * 512), (128, 256, 16, 4 * 512), (129, 257, 16, 2 * 8 * 512),
                                                  (1, 1, 32, 2 * 512), (300, 1000, 32, 3 * 8 * 512), (10, 100, 64, -1), (-1, 5, 16, -1), (5, 1 << 31, 16, -1)])
def test_scale_bytes(pkg, rows, cols, block, want):
    assert pkg.fp4_scale_bytes(rows, cols, block) == want
    if want >= 0 and block == 16 and cols % 256 == 0:
        assert want == pkg.sf_bytes(rows, cols)


def test_a_plain_product_is_accepted(pkg):
    for block in (16, 32):
        for kw in (dict(), dict(m=1), dict(m=5000, n=9000), dict(k=511), dict(a_row_scale=None, b_row_scale=None), dict(bias=0x80000, bias_type=2)):
            rc, info = pkg.query_fp4(_gemm(pkg, block=block, **{"lda": 4096, "ldb": 4096, "ldd": 9000, **kw}))
            assert rc == pkg.OK and info.can_implement == 1, info.reason


@pytest.mark.parametrize("kw,rc,frag", [
    (dict(struct_size=8), "bad", b"struct_size"),
    (dict(a=None), "bad", b"null"),
    (dict(b_scales=None), "bad", b"null"),
    (dict(d=None), "bad", b"null"),
    (dict(d_type=2), "no", b"bf16 or fp16"),
    (dict(d_type=-1), "no", b"bf16 or fp16"),
    (dict(block=8), "no", b"block"),
    (dict(bias=0x80000, bias_type=7), "no", b"bias_type"),
    (dict(k=0), "no", b"empty"),
    (dict(n=-1), "no", b"empty"),
    (dict(m=1 << 31), "no", b"too large"),
    (dict(b=0x40008), "no", b"16-byte"),
    (dict(b_scales=0x50004), "no", b"16-byte"),
    (dict(ldb=240), "no", b"lda"),
    (dict(ldb=264), "no", b"multiples of 16"),
    (dict(ldd=127), "no", b"ldd"),
    (dict(d=0x70001), "no", b"element"),
    (dict(c=0x90000, ldc=100), "no", b"ldc"),
    (dict(c=0x70002, ldc=128), "no", b"apart"),
    (dict(c=0x70000, ldc=130), "no", b"apart"),
    (dict(b_row_scale=0x60002), "no", b"row scales"),
    (dict(bias=0x80001), "no", b"bias"),
    (dict(flags=2), "no", b"flags"),
    (dict(tile_n=48), "no", b"tile_n"),
    (dict(tile_n=32, cta_group=1), "no", b"must hold all"),
    (dict(split_k=3), "no", b"split_k"),
    (dict(split_k=4), "no", b"split_k"),
    (dict(cta_group=2, tile_n=128, split_k=2), "no", b"split_k"),
])
def test_refused_products(pkg, kw, rc, frag):
    got, info = pkg.query_fp4(_gemm(pkg, **kw))
    assert got == (pkg.ERR_BAD_ARGS if rc == "bad" else pkg.ERR_CANNOT_IMPLEMENT)
    assert frag in info.reason, info.reason
    # (A product that only its knobs refuse is refused after the search for D's device, where there is one.)
    assert pkg.lib().gemm_sm100a_fp4_launch(bytes(_gemm(pkg, **kw)), None) in (got, pkg.ERR_LAUNCH)
    if "a" not in kw:
        assert pkg.lib().gemm_sm100a_fp4_linear(bytes(_gemm(pkg, **kw)), C.c_void_p(0xA0000), 0, 512, None) in (got, pkg.ERR_LAUNCH)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("knobs", [dict()] + [dict(cta_group=1, tile_n=bn, split_k=s) for bn in (16, 32, 64, 128) for s in (1, 2, 4, 8)]
                         + [dict(cta_group=2, tile_n=bn) for bn in (128, 256)])
def test_one_cta_per_sm(pkg, block, knobs):
    """CTAs of a split or a pair wait for one another and, without a limit, for tensor memory: two kernels must
    not share SMs, or each could hold what the other one waits for.  An SM has 228 KiB of shared memory."""
    for k in (2048, 2304, 8192, 40000):
        for c in (None, 0x90000):
            rc, info = pkg.query_fp4(_gemm(pkg, m=16, k=k, lda=20480, ldb=20480, c=c, ldc=128, block=block, **knobs))
            assert rc == pkg.OK and 2 * info.smem_bytes > 228 * 1024 and info.smem_bytes <= 227 * 1024 and info.stages >= 1, (k, info.reason)


def test_which_linear_layers_need_a_workspace(pkg):
    L, far = pkg.lib(), 0x900000

    def need(x=far, x_type=0, ldx=4096, **kw):
        return L.gemm_sm100a_fp4_linear_workspace(bytes(_gemm(pkg, **{"ldb": 8192, **kw})), C.c_void_p(x), x_type, ldx)

    assert need(m=1, k=512) == 0 and need(m=8, k=2048) == 0 and need(m=1, k=16384, ldx=16384) == 0
    assert need(m=9, k=512) == 1 and need(m=8, k=2049) == 1 and need(m=1, k=16385, ldx=20000) == 1
    assert need(m=1, k=512, x_type=2) == 1 and need(m=1, k=512, tile_n=16) == 1 and need(m=1, k=512, flags=1) == 1
    assert need(m=1, k=512, x=0x70000) == 1 and need(m=2, k=128, x=0x70000 + 2 * 127, ldx=128) == 1 and need(m=2, k=128, x=0x70000 + 2 * 256, ldx=128) == 0
    # One that needs a workspace is refused without it.
    assert L.gemm_sm100a_fp4_linear(bytes(_gemm(pkg, a=None, m=64)), C.c_void_p(far), 0, 512, None) == pkg.ERR_BAD_ARGS
    assert L.gemm_sm100a_fp4_linear(bytes(_gemm(pkg, a_row_scale=None, m=64)), C.c_void_p(far), 0, 512, None) == pkg.ERR_BAD_ARGS
    assert L.gemm_sm100a_fp4_linear(bytes(_gemm(pkg)), None, 0, 512, None) == pkg.ERR_BAD_ARGS
    assert L.gemm_sm100a_fp4_linear(bytes(_gemm(pkg)), C.c_void_p(far), 0, 500, None) == pkg.ERR_CANNOT_IMPLEMENT
    assert L.gemm_sm100a_fp4_linear(bytes(_gemm(pkg)), C.c_void_p(far), 5, 512, None) == pkg.ERR_CANNOT_IMPLEMENT


@pytest.mark.parametrize("kw,rc", [
    (dict(struct_size=4), "bad"), (dict(x=None), "bad"), (dict(values=None), "bad"), (dict(scales=None), "bad"), (dict(row_scale=None), "bad"),
    (dict(x_type=3), "no"), (dict(block=24), "no"), (dict(rows=-1), "no"), (dict(cols=1 << 31), "no"), (dict(ldx=99), "no"), (dict(x=0x10001), "no"),
    (dict(ldv=48), "no"), (dict(ldv=72), "no"), (dict(values=0x20008), "no"), (dict(scales=0x30008), "no"), (dict(row_scale=0x40002), "no"),
])
def test_refused_quantisations(pkg, kw, rc):
    assert pkg.lib().gemm_sm100a_quantize_fp4(bytes(_quant(pkg, **kw)), None) == (pkg.ERR_BAD_ARGS if rc == "bad" else pkg.ERR_CANNOT_IMPLEMENT)


@pytest.mark.parametrize("kw,rc", [
    (dict(struct_size=4), "bad"), (dict(y=None), "bad"), (dict(values=None), "bad"), (dict(scales=None), "bad"), (dict(y_type=4), "no"),
    (dict(block=0), "no"), (dict(ldy=99), "no"), (dict(y=0x10001), "no"), (dict(ldv=49), "no"), (dict(row_scale=0x40001), "no"),
])
def test_refused_dequantisations(pkg, kw, rc):
    assert pkg.lib().gemm_sm100a_dequantize_fp4(bytes(_dequant(pkg, **kw)), None) == (pkg.ERR_BAD_ARGS if rc == "bad" else pkg.ERR_CANNOT_IMPLEMENT)


@pytest.mark.parametrize("kw,rc", [
    (dict(struct_size=4), "bad"), (dict(x=None), "bad"), (dict(h=None), "bad"), (dict(x_out=None), "bad"), (dict(y=None), "bad"),
    (dict(y=None, x_out=None), "bad"), (dict(block=16), "bad"), (dict(block=16, h=None, values=0x80000, scales=0x90000), "bad"),
    (dict(type=3), "no"), (dict(param_type=1), "no"), (dict(cols=0), "no"), (dict(cols=16385, ldx=20000, ldy=20000, ldo=20000, ldh=20000), "no"),
    (dict(rows=-1), "no"), (dict(eps=-1e-6), "no"), (dict(eps=float("nan")), "no"), (dict(block=8), "no"),
    (dict(ldx=99), "no"), (dict(ldy=99), "no"), (dict(ldo=99), "no"), (dict(ldh=99), "no"), (dict(ldg=99), "no"),
    (dict(x=0x10001), "no"), (dict(weight=0x50001), "no"), (dict(weight=0x50002, param_type=2), "no"), (dict(gate=0x70001), "no"),
    (dict(x_out=0x10002), "no"), (dict(x_out=0x10000, ldo=101), "no"), (dict(x_out=0x20002), "no"), (dict(h=0x10000), "no"), (dict(h=0x20004), "no"),
    (dict(h=0x30000), "no"), (dict(gate=0x30000, ldg=100), "no"), (dict(gate=0x40000, ldg=100), "no"),
    (dict(block=16, h=None, values=0x80008, ldv=64, scales=0x90000, row_scale=0xA0000), "no"),
    (dict(block=16, h=None, values=0x80000, ldv=48, scales=0x90000, row_scale=0xA0000), "no"),
    (dict(block=16, h=None, values=0x80000, ldv=64, scales=0x90004, row_scale=0xA0000), "no"),
])
def test_refused_norms(pkg, kw, rc):
    assert pkg.lib().gemm_sm100a_residual_norm(bytes(_norm(pkg, **kw)), None) == (pkg.ERR_BAD_ARGS if rc == "bad" else pkg.ERR_CANNOT_IMPLEMENT)


def test_accepted_norms_end_at_the_search_for_the_device(pkg):
    """No device memory is behind the addresses."""
    four = dict(block=32, h=None, values=0x80000, ldv=64, scales=0x90000, row_scale=0xA0000)
    for kw in (dict(), dict(x_out=0x10000), dict(x_out=0x20000), dict(gate=0x90000, ldg=100), dict(param_type=2), dict(weight=None, gate=None, post_weight=None),
               dict(y=None, x_out=None, gate=None, post_weight=None), four):
        assert pkg.lib().gemm_sm100a_residual_norm(bytes(_norm(pkg, **kw)), None) == pkg.ERR_LAUNCH
    for kw in (dict(), dict(dx_out=None), dict(y=None, dy=None, post_weight=None, gate=None, dpost_weight=None, dgate=None), dict(gate=0x100000, ldg=100),
               dict(dweight=None, dpost_weight=None, dgate=None)):
        assert pkg.lib().gemm_sm100a_residual_norm_backward(bytes(_back(pkg, **kw)), None) == pkg.ERR_LAUNCH
    assert pkg.lib().gemm_sm100a_residual_norm(bytes(_norm(pkg, rows=0, x=None, h=None)), None) == pkg.OK


@pytest.mark.parametrize("kw,rc", [
    (dict(struct_size=4), "bad"), (dict(dh=None), "bad"), (dict(x_out=None), "bad"), (dict(dx=None), "bad"), (dict(dy=None), "bad"),
    (dict(workspace=None), "bad"), (dict(workspace_bytes=10), "bad"), (dict(y=None), "bad"), (dict(weight=None), "bad"), (dict(gate=None), "bad"),
    (dict(post_weight=None), "bad"), (dict(type=5), "no"), (dict(cols=20000), "no"), (dict(param_type=1), "no"), (dict(eps=-1.0), "no"),
    (dict(lddh=99), "no"), (dict(lddx=99), "no"), (dict(dh=0x10001), "no"), (dict(dweight=0xA0002), "no"), (dict(workspace=0xD0008), "no"),
    (dict(dx=0x10000), "no"), (dict(dx=0x30010), "no"), (dict(dy=0x80008), "no"), (dict(dy=0x40000), "no"),
    (dict(gate=0x100000, ldg=100, dgate=0x100000), "no"), (dict(gate=0x100000, ldg=100, dgate=0x90000), "no"),
])
def test_refused_norm_gradients(pkg, kw, rc):
    assert pkg.lib().gemm_sm100a_residual_norm_backward(bytes(_back(pkg, **kw)), None) == (pkg.ERR_BAD_ARGS if rc == "bad" else pkg.ERR_CANNOT_IMPLEMENT)


def test_norm_workspace(pkg):
    L = pkg.lib()
    assert L.gemm_sm100a_residual_norm_workspace(0, 100) == 0
    for rows, cols in ((-1, 5), (5, 0), (5, 16385)):
        assert L.gemm_sm100a_residual_norm_workspace(rows, cols) == -1
    for rows, cols in ((1, 1), (5, 8192), (10000, 64), (16384, 16384)):
        assert 8 * cols <= L.gemm_sm100a_residual_norm_workspace(rows, cols) <= 8 * cols * min(rows, 148 * 16)
