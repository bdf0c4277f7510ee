"""Host-side checks of the 4-bit and mixture-of-experts entry points: sizes and refusals, before anything is launched."""
import ctypes

import pytest

BAD = 0x1000  # a non-null, aligned address that is never dereferenced on these paths


def status(fn, *a, **kw):
    from gemm_mmbo_b200 import MmboError
    try:
        fn(*a, **kw)
    except MmboError as e:
        return e.status
    return 0


def test_packed_sizes(mm):
    # 16 x 128 tiles: 1024 bytes of codes, 32 of scales and 16 of zero points a group
    assert mm.w4_bytes(16, 128, 128, False) == 1056
    assert mm.w4_bytes(16, 128, 128, True) == 1072
    assert mm.w4_bytes(17, 129, 32, True) == 4 * (1024 + 4 * 48)
    assert mm.w4_bytes(0, 128) == 0 and mm.w4_bytes(5, 0) == 0
    assert mm.w4_bytes(2 ** 31 - 1, 2 ** 31 - 1, 64, False) > 2 ** 60
    assert status(mm.w4_bytes, 16, 128, 16) == -21 and status(mm.w4_bytes, 16, 128, 256) == -21
    assert status(mm.w4_bytes, 2 ** 31, 1) == -2
    from gemm_mmbo_b200._lib import LIB
    assert LIB.mmbo_w4_bytes(16, 16, 64, 2, ctypes.byref(ctypes.c_size_t())) == -21
    assert LIB.mmbo_w4_bytes(16, 16, 64, 0, None) == -3


def test_status_strings_of_the_new_codes(mm):
    for code in (-21, -22):
        assert mm.status_string(code) not in ("", "unknown status")


def test_gemm_w4_refusals(mm):
    def call(dtype="f16", m=64, n=3, k=256, packed=BAD, group=64, zeros=False, B=BAD, ldb=256, C=BAD, ldc=64):
        return status(mm.gemm_w4, dtype, m, n, k, 1.0, packed, group, zeros, B, ldb, 0.0, C, ldc, stream=0)

    assert call(group=48) == -21
    assert call(ldb=255) == -5 and call(ldc=63) == -6
    assert call(m=2 ** 31) == -2 and call(n=2 ** 31) == -2 and call(k=2 ** 31) == -2
    assert call(packed=None) == -3 and call(B=None) == -3 and call(C=None) == -3
    assert call(packed=BAD + 8) == -22 and call(B=BAD + 1) == -22 and call(C=BAD + 1) == -22
    assert call(m=0) == 0 and call(n=0) == 0
    with pytest.raises(KeyError):
        call(dtype="f32")
    from gemm_mmbo_b200._lib import LIB
    one = ctypes.c_float(1)
    for dt in (0, 2, 7):
        assert LIB.mmbo_gemm_w4(dt, 64, 1, 64, one, BAD, 64, 0, BAD, 64, one, BAD, 64, None) == -9
    assert LIB.mmbo_gemm_w4(1, 64, 1, 64, None, BAD, 64, 0, BAD, 64, one, BAD, 64, None) == -3
    assert LIB.mmbo_gemm_w4(1, 64, 1, 64, one, BAD, 64, 0, BAD, 64, None, BAD, 64, None) == -3


def test_quantize_pack_unpack_refusals(mm):
    q = lambda **kw: status(mm.w4_quantize, "bf16", **{**dict(m=8, k=100, group=32, zeros=True, W=BAD, ldw=100, packed=BAD,
                                                              stream=0), **kw})
    u = lambda **kw: status(mm.w4_unpack, "bf16", **{**dict(m=8, k=100, group=32, zeros=True, W=BAD, ldw=100, packed=BAD,
                                                            stream=0), **kw})
    for f in (q, u):
        assert f(group=0) == -21 and f(ldw=99) == -4 and f(W=None) == -3 and f(packed=None) == -3
        assert f(W=BAD + 1) == -22 and f(packed=BAD + 4) == -22
        assert f(m=0) == 0 and f(k=0) == 0
    p = lambda **kw: status(mm.w4_pack, "f16", **{**dict(m=8, k=101, group=32, codes=BAD, ldcodes=51, scales=BAD, ldscales=4,
                                                         zero_points=BAD, ldzeros=4, packed=BAD, stream=0), **kw})
    assert p(ldcodes=50) == -4 and p(ldscales=3) == -5 and p(ldzeros=3) == -5
    assert p(codes=None) == -3 and p(scales=None) == -3 and p(packed=None) == -3
    assert p(scales=BAD + 1) == -22 and p(packed=BAD + 8) == -22
    assert p(group=100) == -21 and p(m=0) == 0


def test_moe_refusals(mm):
    need = mm.moe_workspace_bytes("f16", 4, 128, 64, 8, 2)
    assert need > 0

    def call(dtype="f16", tokens=4, d=128, f=64, experts=8, topk=2, **kw):
        a = dict(X=BAD, ldx=128, router=BAD, ldr=128, gate=BAD, up=BAD, ldg=128, strideG=128 * 64, down=BAD, ldd=64,
                 strideD=64 * 128, Y=BAD, ldy=128, workspace=BAD, workspace_bytes=need, stream=0)
        a.update(kw)
        return status(mm.moe, dtype, tokens, d, f, experts, topk, **a)

    assert call(topk=0) == -2 and call(topk=9) == -2 and call(experts=0) == -2 and call(experts=1025) == -2
    assert call(experts=64, topk=33) == -2 and call(tokens=257) == -2
    assert call(d=0) == -2 and call(f=0) == -2 and call(d=65537) == -2 and call(f=65537) == -2
    assert call(ldx=127) == -5 and call(ldy=127) == -6 and call(ldr=127) == -4
    assert call(ldg=127) == -4 and call(ldd=63) == -4 and call(strideG=64 * 128 - 1) == -4 and call(strideD=100) == -4
    for name in ("X", "router", "gate", "up", "down", "Y", "workspace"):
        assert call(**{name: None}) == -3, name
        assert call(**{name: BAD + 1}) == -22, name
    assert call(ids=BAD + 2) == -22 and call(gates=BAD + 2) == -22 and call(workspace=BAD + 128) == -22
    assert call(workspace_bytes=need - 1) == -15
    assert call(group=16) == -21 and call(group=0, zeros=True) == -21
    size = mm.w4_bytes(64, 128, 64, False)
    assert call(group=64, strideG=size - 16, strideD=10 ** 6) == -4
    assert call(group=64, strideG=size + 8, strideD=10 ** 6) == -22
    assert call(group=64, gate=BAD + 2, strideG=10 ** 6, strideD=10 ** 6) == -22
    assert call(tokens=0) == 0
    assert status(mm.moe_workspace_bytes, "f16", 4, 0, 64, 8, 2) == -2
    from gemm_mmbo_b200._lib import LIB
    out = ctypes.c_size_t()
    assert LIB.mmbo_moe_workspace_bytes(0, 4, 128, 64, 8, 2, ctypes.byref(out)) == -9
    assert LIB.mmbo_moe_workspace_bytes(1, 4, 128, 64, 8, 2, None) == -3
