"""What the 8-bit operators refuse: checks that need no GPU."""
import ctypes

import pytest
import torch

from deers_b200 import _lib, q8
from deers_b200.errors import DeviceMismatch, DTypeMismatch, LayoutMismatch

E4M3 = torch.float8_e4m3fn


def test_the_mirror_refuses():
    x = torch.zeros(4, 32)
    for call in (q8.rms_norm_add_q8, q8.quantize_q8):
        with pytest.raises(DeviceMismatch):
            call(x)
        with pytest.raises(DTypeMismatch):
            call(x.double())
        with pytest.raises(DTypeMismatch):
            call(x, dtype=torch.uint8)
        with pytest.raises(LayoutMismatch):
            call(torch.zeros(()))
        with pytest.raises(LayoutMismatch):
            call(torch.zeros(3, 0))
    with pytest.raises(LayoutMismatch):
        q8.quantize_weight_q8(torch.zeros(3))
    rows, w = q8.RowsQ8(torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4)), q8.RowsQ8(torch.zeros(8, 32, dtype=torch.int8), torch.zeros(8))
    for bad, error in (((rows, w), DeviceMismatch), ((rows, q8.RowsQ8(w.codes[:, :16], w.scale)), LayoutMismatch), ((rows, q8.RowsQ8(w.codes, w.scale[:3])), LayoutMismatch),
                       ((q8.RowsQ8(rows.codes, rows.scale[:1]), w), LayoutMismatch), ((rows, q8.RowsQ8(w.codes.to(E4M3), w.scale)), DTypeMismatch),
                       ((q8.RowsQ8(rows.codes, rows.scale.double()), w), DTypeMismatch), ((q8.RowsQ8(x, rows.scale), w), DTypeMismatch)):
        with pytest.raises(error):
            q8.linear_q8(*bad)
    with pytest.raises(DTypeMismatch):
        q8.linear_q8(rows, w, torch.bfloat16)


def test_the_cache_refuses():
    codes, scale = torch.zeros(2, 3, 40, 32).to(E4M3), torch.zeros(2, 3, 2)
    with pytest.raises(DeviceMismatch):
        q8.CacheQ8(codes, codes, scale, scale)
    with pytest.raises(LayoutMismatch):
        q8.CacheQ8(codes, codes, scale[..., :1], scale)
    with pytest.raises(LayoutMismatch):
        q8.CacheQ8(codes, codes[:, :2], scale, scale)
    with pytest.raises(LayoutMismatch):
        q8.CacheQ8(codes[..., :24], codes[..., :24], scale, scale)
    with pytest.raises(LayoutMismatch):
        q8.CacheQ8(codes.transpose(2, 3), codes.transpose(2, 3), scale[..., :1], scale[..., :1])
    with pytest.raises(DTypeMismatch):
        q8.CacheQ8(codes.float(), codes.float(), scale, scale)
    with pytest.raises(DTypeMismatch):
        q8.CacheQ8(codes, codes, scale.double(), scale)
    for bad in ((0, 1, 1, 16), (1, 1, 1, 20), (1, 1, 0, 16), (1, 1, 8, 272)):
        with pytest.raises(LayoutMismatch):
            q8.CacheQ8.new(*bad)
    with pytest.raises(DeviceMismatch):
        q8.CacheQ8.new(1, 1, 8, 16, device="cpu")


# ---- the C entries: their checks come before anything is done with the context, for which a block of zeros stands here
CTX = ctypes.create_string_buffer(1 << 16)
P = 1 << 20                                                       # a pointer on every boundary, never followed


def desc(**more):
    d = _lib.QuantizeDesc(4, 32, _lib.F16, _lib.I8, 1, 0, 1e-5, 32, 32, 32, 32)
    for k, v in more.items():
        setattr(d, k, v)
    return ctypes.byref(d)


def test_quantize_rows_refuses():
    f = _lib.lib().deers_b200_quantize_rows
    assert f(None, desc(), P, None, None, P, P) == _lib.ERR_NULL
    assert f(CTX, None, P, None, None, P, P) == _lib.ERR_NULL
    assert f(CTX, desc(), None, None, None, P, P) == _lib.ERR_NULL
    assert f(CTX, desc(), P, P, None, P, P) == _lib.ERR_NULL            # a residual without a place for the sum
    assert f(CTX, desc(), P, None, P, P, P) == _lib.ERR_UNSUPPORTED
    assert f(CTX, desc(rows=0), None, None, None, None, None) == _lib.OK
    for bad in (dict(rows=-1), dict(C=0), dict(rows=1 << 31)):
        assert f(CTX, desc(**bad), P, None, None, P, P) == _lib.ERR_SHAPE
    assert f(CTX, desc(C=(1 << 30) + 1, ld_codes=(1 << 30) + 16), P, None, None, P, P) == _lib.ERR_UNSUPPORTED
    for bad in (dict(dtype=2), dict(code=0)):
        assert f(CTX, desc(**bad), P, None, None, P, P) == _lib.ERR_DTYPE
    assert f(CTX, desc(relu_squared=1), P, None, None, P, P) == _lib.ERR_UNSUPPORTED
    for bad in (dict(ld_codes=24), dict(ld_codes=16), dict(ld_x=-1)):
        assert f(CTX, desc(**bad), P, None, None, P, P) == _lib.ERR_LAYOUT
    assert f(CTX, desc(ld_sum=31), P, P, P, P, P) == _lib.ERR_LAYOUT
    for bad in ((P + 1, P, P), (P, P + 8, P), (P, P, P + 2)):
        assert f(CTX, desc(), bad[0], None, None, bad[1], bad[2]) == _lib.ERR_LAYOUT


def test_gemm_q8_refuses():
    f = _lib.lib().deers_b200_gemm_q8
    ok = dict(M=4, N=8, K=32, code=_lib.I8, a=P, lda=32, sa=P, b=P, ldb=32, sb=P, out=_lib.F16, c=P, ldc=8)
    call = lambda ctx=CTX, **more: f(ctx, *{**ok, **more}.values())  # noqa: E731
    assert call(ctx=None) == _lib.ERR_NULL and call(M=0, a=None) == _lib.OK
    for n in ("a", "sa", "b", "sb", "c"):
        assert call(**{n: None}) == _lib.ERR_NULL
    for bad in (dict(M=-1), dict(N=0), dict(K=0)):
        assert call(**bad) == _lib.ERR_SHAPE
    for bad in (dict(code=_lib.F16), dict(out=_lib.I8)):
        assert call(**bad) == _lib.ERR_DTYPE
    for K in (131072, 131073):                                   # 131072 products of -128 and -128 leave 32 bits
        assert call(K=K, lda=1 << 18, ldb=1 << 18) == _lib.ERR_UNSUPPORTED
    for bad in (dict(lda=31), dict(lda=16), dict(ldb=40), dict(ldc=7), dict(a=P + 8), dict(b=P + 1), dict(c=P + 1), dict(sa=P + 2), dict(sb=P + 1)):
        assert call(**bad) == _lib.ERR_LAYOUT


def cache(**more):
    c = _lib.CacheQ8(2, 3, 40, 32, P, P, P, P, *((ctypes.c_int64 * 3)(3 * 40 * 32, 40 * 32, 32) for _ in range(2)), *((ctypes.c_int64 * 2)(6, 2) for _ in range(2)))
    for k, v in more.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [(dict(B=0), "SHAPE"), (dict(capacity=0), "SHAPE"), (dict(D=24), "UNSUPPORTED"), (dict(D=272), "UNSUPPORTED"), (dict(B=40000), "UNSUPPORTED"), (dict(k=None), "NULL"),
              (dict(v_scale=None), "NULL"), (dict(k=P + 8), "LAYOUT"), (dict(k_scale=P + 2), "LAYOUT"), (dict(k_strides=(ctypes.c_int64 * 3)(3840, 1280, 8)), "LAYOUT"),
              (dict(v_strides=(ctypes.c_int64 * 3)(3840, 1280, 16)), "LAYOUT"), (dict(v_strides=(ctypes.c_int64 * 3)(-16, 1280, 32)), "LAYOUT"),
              (dict(k_scale_strides=(ctypes.c_int64 * 2)(-1, 2)), "LAYOUT")]


def test_cache_append_refuses():
    f = _lib.lib().deers_b200_cache_q8_append
    good = (ctypes.c_int64 * 4)(3 * 5 * 32, 5 * 32, 32, 1)
    call = lambda c=None, T=5, dtype=_lib.F16, k=P, ks=good, v=P, vs=good, start=P, count=None, ctx=CTX: f(ctx, ctypes.byref(c or cache()), T, dtype, k, ks, v, vs, start, count)  # noqa: E731
    for more, error in BAD_CACHES:
        assert call(cache(**more)) == getattr(_lib, "ERR_" + error), more
    assert call(ctx=None) == _lib.ERR_NULL and call(T=0, k=None) == _lib.OK
    for bad in (dict(k=None), dict(v=None), dict(start=None), dict(ks=None)):
        assert call(**bad) == _lib.ERR_NULL
    assert call(dtype=_lib.E4M3) == _lib.ERR_DTYPE and call(T=-1) == _lib.ERR_SHAPE and call(T=41) == _lib.ERR_SHAPE
    for bad in (dict(ks=(ctypes.c_int64 * 4)(480, 160, 32, 2)), dict(vs=(ctypes.c_int64 * 4)(480, -160, 32, 1)), dict(k=P + 1), dict(start=P + 2), dict(count=P + 1),
                dict(c=cache(k_strides=(ctypes.c_int64 * 3)(0, 1280, 32))), dict(c=cache(v_scale_strides=(ctypes.c_int64 * 2)(6, 0)))):
        assert call(**bad) == _lib.ERR_LAYOUT


def test_attn_decode_q8_refuses():
    L = _lib.lib()

    def d(c=None, **more):
        s = (ctypes.c_int64 * 4)(6 * 32, 32, 32, 1)
        x = _lib.DecodeQ8Desc(c or cache(), 6, 1, _lib.F16, 1, 0.1, s, s)
        for k, v in more.items():
            setattr(x, k, v)
        return ctypes.byref(x)

    call = lambda x, q=P, n=P, o=P, lse=None, ws=None, size=0, ctx=CTX: L.deers_b200_attn_decode_q8(ctx, x, q, n, o, lse, ws, size)  # noqa: E731
    for more, error in BAD_CACHES:
        assert call(d(cache(**more))) == getattr(_lib, "ERR_" + error), more
        assert L.deers_b200_attn_decode_q8_workspace_bytes(d(cache(**more))) == 0
    assert call(d(), ctx=None) == _lib.ERR_NULL and call(None) == _lib.ERR_NULL
    for bad in (dict(q=None), dict(n=None), dict(o=None)):
        assert call(d(), **bad) == _lib.ERR_NULL
    assert call(d(dtype=_lib.I8)) == _lib.ERR_DTYPE
    for bad in (dict(H=7), dict(H=0), dict(Tq=0), dict(scale=float("nan"))):
        assert call(d(**bad)) == _lib.ERR_SHAPE
    assert call(d(Tq=41)) == _lib.ERR_UNSUPPORTED and call(d(Tq=129)) == _lib.ERR_UNSUPPORTED
    for bad in (dict(q=P + 1), dict(o=P + 1), dict(n=P + 2), dict(lse=P + 1)):
        assert call(d(), **bad) == _lib.ERR_LAYOUT
    for bad in (dict(q_strides=(ctypes.c_int64 * 4)(192, 32, 32, 2)), dict(o_strides=(ctypes.c_int64 * 4)(192, -32, 32, 1))):
        assert call(d(**bad)) == _lib.ERR_LAYOUT
    long = cache(B=1, H=1, capacity=1 << 20)
    need = L.deers_b200_attn_decode_q8_workspace_bytes(d(long, H=1))
    assert need > 0
    assert call(d(long, H=1)) == _lib.ERR_WORKSPACE and call(d(long, H=1), ws=P, size=need - 1) == _lib.ERR_WORKSPACE
    assert call(d(long, H=1), ws=P + 8, size=need) == _lib.ERR_WORKSPACE
    for strides in ((0, 1280, 32), (3840, 0, 32)):               # a cache that several sequences or heads share
        assert call(d(cache(k_strides=(ctypes.c_int64 * 3)(*strides)))) == _lib.ERR_LAYOUT
    size = lambda **c: L.deers_b200_attn_decode_q8_workspace_bytes(d(cache(**c), H=2))  # noqa: E731
    assert size(B=64, H=1, capacity=16384) > 0 and size(B=65, H=1, capacity=16384) == 0 and size(B=1, H=1, capacity=16383) == 0


def test_gemm_q8_refuses_sizes_whose_tiles_leave_32_bits():
    """Up to 2^31 - 513 rows, columns and summands: the last tile's places are whole numbers of 32 bits too."""
    f = _lib.lib().deers_b200_gemm_q8
    most = 0x7fffffff
    for M, N, K in ((most, 8, 32), (most - 511, 8, 32), (4, most, 32), (4, most - 511, 32), (4, 8, most), (4, 8, most - 511)):
        ld = (K + 15) // 16 * 16
        assert f(CTX, M, N, K, _lib.E4M3, P, ld, P, P, ld, P, _lib.F16, P, N) == _lib.ERR_UNSUPPORTED, (M, N, K)
