"""The 8-bit operators of cached decoding against their definition in 64 bits."""
import ctypes
import math

import pytest
import torch

from tests import q8_util as ref

pytestmark = pytest.mark.gpu

E4M3, I8 = ref.E4M3, ref.I8
CODES = pytest.mark.parametrize("codes", [I8, E4M3], ids=["i8", "e4m3"])
TYPES = pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])


def q8():
    from deers_b200 import q8 as m
    return m


def sync():
    from deers_b200 import ops
    ops.Context.current(torch.device("cuda", 0)).sync()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def same(got, want):
    """Equal values, NaN where NaN."""
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want)), f"{(got - want).abs().max()}"


def near(got, want, tol):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    fine = torch.isfinite(want)
    off = (got - want).abs()[fine] - (tol.expand_as(want)[fine] if isinstance(tol, torch.Tensor) else tol)
    assert off.numel() == 0 or float(off.max()) <= 0, f"over the tolerance by {float(off.max())}"


def check_rows(rows, h, x, residual, norm, relu, eps, codes):
    wh, wq, ws = ref.quantize(x, residual, norm, relu, eps, codes)
    if h is not None:
        same(h, wh)
    same(rows.codes.float(), wq)
    near(rows.scale, ws, ws.abs() * ref.scale_tolerance(x.shape[-1]) + 1e-45)


# ---- rows ---------------------------------------------------------------------------------------------------------------
SIZES = [(1, 1), (3, 7), (5, 16), (17, 100), (2, 255), (9, 768), (2, 1024), (3, 1025), (2, 2048), (5, 3000), (2, 4100), (2, 8192), (2, 9001), (2, 17001)]


@CODES
@TYPES
@pytest.mark.parametrize("rows,C", SIZES, ids=lambda v: str(v))
def test_rows_with_norm_and_residual(rows, C, dtype, codes):
    g = gen(rows * 10007 + C)
    x, r = torch.randn(rows, C, generator=g).to(dtype), (torch.randn(rows, C, generator=g) * 3).to(dtype)
    h, got = q8().rms_norm_add_q8(x.cuda(), r.cuda(), 1e-5, codes)
    sync()
    assert h.dtype == dtype and got.codes.dtype == codes and got.codes.shape == x.shape
    check_rows(got, h, x, r, True, False, 1e-5, codes)
    h, got = q8().rms_norm_add_q8(x.cuda(), None, 1e-6, codes)
    check_rows(got, h, x, None, True, False, 1e-6, codes)


@CODES
@TYPES
@pytest.mark.parametrize("relu", [False, True])
def test_rows_of_many_axes_and_strides(relu, dtype, codes):
    x = torch.randn(3, 4, 50, generator=gen(1)).to(dtype)
    check_rows(q8().quantize_q8(x.cuda(), codes, relu), None, x, None, False, relu, 0.0, codes)
    wide = torch.randn(6, 200, generator=gen(2)).to(dtype)
    for a, b in ((0, 64), (3, 133), (8, 200)):                   # aligned and unaligned columns of wider rows
        check_rows(q8().quantize_q8(wide.cuda()[:, a:b], codes, relu), None, wide[:, a:b], None, False, relu, 0.0, codes)
    check_rows(q8().quantize_q8(wide.cuda().t(), codes, relu), None, wide.t(), None, False, relu, 0.0, codes)
    one = wide[0]
    got = q8().quantize_q8(one.cuda(), codes, relu)
    assert got.scale.shape == ()
    check_rows(got, None, one, None, False, relu, 0.0, codes)
    assert q8().quantize_q8(x[:0].cuda(), codes, relu).codes.shape == (0, 4, 50)


@CODES
def test_rows_at_borders_are_rounded_to_even(codes):
    # quotients that lie on borders between codes: the row's largest value is the largest code, so value and quotient are one
    if codes is I8:
        x = torch.cat([torch.arange(-126, 127).double() + 0.5, torch.tensor([127.0])])
    else:
        v = torch.arange(127, dtype=torch.uint8).view(E4M3).double()
        x = torch.cat([(v[1:] + v[:-1]) / 2, -(v[1:] + v[:-1]) / 2, torch.tensor([448.0])])
    for dtype in (torch.float16, torch.float32):
        for f in (1.0, 2.0 ** -7, 2.0 ** 5):
            t = (x * f).to(dtype)[None]
            if not torch.equal(t.double()[0], x * f):
                continue
            check_rows(q8().quantize_q8(t.cuda(), codes), None, t, None, False, False, 0.0, codes)
    # and next to them, to either side
    t = (x * 0.7).float()
    t = torch.stack([t, torch.nextafter(t, torch.full_like(t, math.inf)), torch.nextafter(t, torch.full_like(t, -math.inf))])
    check_rows(q8().quantize_q8(t.cuda(), codes), None, t, None, False, False, 0.0, codes)


@CODES
def test_rows_of_zeros_and_of_no_numbers(codes):
    x = torch.randn(6, 300, generator=gen(4))
    x[0] = 0
    x[1, 7] = math.inf
    x[2, 299] = math.nan
    x[3, 0] = -math.inf
    x[4] = -x[4].abs()
    for dtype in (torch.float16, torch.float32):
        t = x.to(dtype)
        check_rows(q8().rms_norm_add_q8(t.cuda(), None, 1e-5, codes)[1], None, t, None, True, False, 1e-5, codes)
        check_rows(q8().quantize_q8(t.cuda(), codes, relu_squared=True), None, t, None, False, True, 0.0, codes)
    # a sum that leaves f16
    big = torch.full((2, 64), 60000.0, dtype=torch.float16)
    h, got = q8().rms_norm_add_q8(big.cuda(), big.cuda(), 1e-5, codes)
    assert torch.isinf(h).all() and torch.isnan(got.scale).all() and not got.codes.float().any()


@CODES
def test_rows_of_the_smallest_and_largest_numbers(codes):
    base = torch.randn(4, 64, generator=gen(5))
    x = torch.stack([base[0] * 1e-38, base[1] * 1e-40, base[2] * 1e-43, base[3] / base[3].abs().max() * 3e38]).float()
    got = q8().quantize_q8(x.cuda(), codes)
    _, wq, ws = ref.quantize(x, codes=codes)
    same(got.codes.float(), wq)
    # (a scale among the subnormals is off by half of their step)
    near(got.scale, ws, ws.abs() * 2.0 ** -23 + 2.0 ** -149)


def test_rows_into_a_callers_buffers():
    """The C entry: the sum may be the residual, codes may have longer rows, whose ends stay as they are."""
    from deers_b200 import _lib, ops
    ctx = ops.Context.current(torch.device("cuda", 0))
    x, r = (torch.randn(5, 100, generator=gen(s)).half() for s in (6, 7))
    dx, dr = x.cuda(), r.cuda()
    codes = torch.full((5, 128), 77, dtype=torch.int8, device="cuda")
    scale = torch.empty(5, device="cuda")
    d = _lib.QuantizeDesc(5, 100, _lib.F16, _lib.I8, 1, 0, 1e-5, 100, 100, 100, 128)
    _lib.check(_lib.lib().deers_b200_quantize_rows(ctx.handle, ctypes.byref(d), dx.data_ptr(), dr.data_ptr(), dr.data_ptr(), codes.data_ptr(), scale.data_ptr()))
    wh, wq, _ = ref.quantize(x, r, True, False, 1e-5, I8)
    same(dr, wh)
    same(codes[:, :100], wq)
    assert (codes[:, 100:] == 77).all()


# ---- products -----------------------------------------------------------------------------------------------------------
def make_rows(g, n, K, codes, size=1.0):
    x = torch.randn(n, K, generator=g) * size
    _, q, s = ref.quantize(x, codes=codes)
    return q, s.float()


def check_linear(a, sa, b, sb, codes, out=torch.float16, lead=None):
    m = q8()
    rows = m.RowsQ8(a.to(codes).cuda(), sa.cuda())
    if lead:
        rows = m.RowsQ8(rows.codes.reshape(*lead, -1), rows.scale.reshape(lead))
    y = m.linear_q8(rows, m.RowsQ8(b.to(codes).cuda(), sb.cuda()), out)
    sync()
    assert y.dtype == out and y.shape == (*(lead or a.shape[:1]), b.shape[0])
    both = sa.double()[:, None] * sb.double()[None]
    want, size = (a @ b.t()) * both, (a.abs() @ b.abs().t()) * both.abs()
    K = a.shape[1]
    # a sum in whole numbers is exact; in f32 every one of K / 32 steps may cut off 2^-23 of what there is, and 2^-18 of its own 32 products
    sums = 0.0 if codes is I8 else (K / 32 + 32) * 2.0 ** -23
    near(y.reshape(-1, b.shape[0]), want, ref.half_step(want, out) * (1 + 2.0 ** -10) + 2.0 ** -22 * want.abs() + sums * torch.nan_to_num(size))


LINEAR = [(1, 16, 16), (1, 768, 2304), (2, 32, 1), (3, 33, 7), (7, 100, 130), (16, 512, 100), (17, 640, 257), (33, 1000, 129), (64, 2048, 500), (65, 4096, 96),
          (100, 96, 1000), (129, 130, 300), (200, 2731, 1001), (256, 256, 512), (300, 64, 2000), (513, 1024, 520), (1, 16384, 40), (5, 9000, 33)]


@CODES
@pytest.mark.parametrize("M,K,N", LINEAR, ids=lambda v: str(v))
def test_linear(M, K, N, codes):
    g = gen(M * 31 + K * 7 + N)
    check_linear(*make_rows(g, M, K, codes), *make_rows(g, N, K, codes, 1 / math.sqrt(K)), codes)


@CODES
@pytest.mark.parametrize("M,K,N", [(1, 48, 9), (5, 768, 260), (70, 300, 131), (257, 520, 384)], ids=lambda v: str(v))
def test_linear_to_f32(M, K, N, codes):
    g = gen(M + K + N)
    check_linear(*make_rows(g, M, K, codes), *make_rows(g, N, K, codes), codes, torch.float32)


@CODES
def test_linear_of_many_axes_and_of_rows_as_the_quantiser_leaves_them(codes):
    g = gen(11)
    check_linear(*make_rows(g, 24, 64, codes), *make_rows(g, 48, 64, codes), codes, lead=(2, 3, 4))
    x, w = torch.randn(2, 9, 150, generator=g), torch.randn(150, 70, generator=g)
    rows, weight = q8().quantize_q8(x.cuda(), codes), q8().quantize_weight_q8(w.cuda(), codes)
    y = q8().linear_q8(rows, weight, torch.float32)
    a, b = rows.codes.float().cpu().double(), weight.codes.float().cpu().double()
    same(b, ref.quantize(w.t().contiguous(), codes=codes)[1])
    both = rows.scale.cpu().double()[..., None] * weight.scale.cpu().double()
    near(y, (a @ b.t()) * both, 40 * 2.0 ** -23 * (a.abs() @ b.abs().t()) * both)
    assert q8().linear_q8(q8().quantize_q8(x[:0].cuda(), codes), weight).shape == (0, 9, 70)


def test_linear_with_the_largest_codes_and_scales_of_no_number():
    # 16384 products of 127 * 127 are beyond f32's whole numbers
    a, b = torch.full((3, 16384), 127.0).double(), torch.full((130, 16384), -127.0).double()
    a[1, 0], b[5, 3] = 126.0, -1.0
    check_linear(a, torch.tensor([1.0, 0.5, math.nan]), b, torch.linspace(1e-9, 1e-5, 130), I8, torch.float32)
    # e4m3: a NaN code reaches its row, a scale of NaN its channel
    g = gen(12)
    a, sa = make_rows(g, 4, 64, E4M3)
    b, sb = make_rows(g, 40, 64, E4M3)
    a[2, 9], sb[7] = math.nan, math.nan
    check_linear(a, sa, b, sb, E4M3)


def test_linear_with_the_longest_sums_of_whole_numbers():
    # 131071 products of -128 and -128, the last that fit 32 bits (quantised rows have no -128, a caller's may)
    a, b = torch.full((2, 131071), -128.0).double(), torch.full((3, 131071), -128.0).double()
    a[1] = 127.0
    check_linear(a, torch.tensor([1e-3, 1.0]), b, torch.tensor([1e-4, 1e-5, 1.0]), I8, torch.float32)


# ---- the cache ----------------------------------------------------------------------------------------------------------
def cache_values(c):
    return c.k.float().cpu().double(), c.k_scale.cpu(), c.v.float().cpu().double(), c.v_scale.cpu()


@TYPES
@pytest.mark.parametrize("B,H,cap,D", [(1, 1, 1, 16), (2, 3, 70, 32), (3, 5, 100, 80), (2, 2, 200, 128), (1, 4, 96, 256)], ids=lambda v: str(v))
def test_append_in_pieces(B, H, cap, D, dtype):
    """Rows that arrive in pieces of any length at any place, larger ones behind smaller ones and the other way round."""
    g = gen(B + H + cap + D)
    c = q8().CacheQ8.new(B, H, cap, D)
    k, ks, v, vs = cache_values(c)
    at = torch.zeros(B, dtype=torch.int32)
    for T in (1, 1, 5, 31, 33, 1, 64, 2, 1):
        if T > cap:
            continue
        size = float(torch.rand(1, generator=g)) * 10
        kn, vn = ((torch.randn(B, H, T, D, generator=g) * size).to(dtype) for _ in range(2))
        count = torch.minimum(torch.randint(0, T + 1, (B,), generator=g) if T > 1 else torch.ones(B), cap - at).to(torch.int32)
        c.append(kn.cuda(), vn.cuda(), at.cuda(), count.cuda())
        ref.append(k, ks, kn, at, count)
        ref.append(v, vs, vn, at, count)
        for got, want in zip(cache_values(c), (k, ks, v, vs)):
            same(got, want)
        at += count
    sync()


def test_append_of_whole_batches_from_views():
    """Without counts, from head-major views of a fused projection, into views of a larger cache; a long prompt; again; and anew."""
    g = gen(21)
    B, H, T, D, cap = 2, 3, 300, 64, 320
    big = q8().CacheQ8.new(B + 1, H + 2, cap, D)
    views = (big.k[1:, 1:1 + H], big.v[1:, 1:1 + H], big.k_scale[1:, 1:1 + H], big.v_scale[1:, 1:1 + H])
    c = q8().CacheQ8(*views)
    for dtype, shift in ((torch.float16, 0), (torch.float32, 0), (torch.float16, 1)):
        flat = torch.randn(B, T, 3 * H * D + shift, generator=g).to(dtype)
        kn, vn = (flat[..., shift + i * H * D:shift + (i + 1) * H * D].unflatten(-1, (H, D)).permute(0, 2, 1, 3) for i in (1, 2))
        dev = flat.cuda()
        dk, dv = (dev[..., shift + i * H * D:shift + (i + 1) * H * D].unflatten(-1, (H, D)).permute(0, 2, 1, 3) for i in (1, 2))
        start = torch.tensor([0, 20], dtype=torch.int32)
        k, ks, v, vs = (t.clone() for t in cache_values(c))
        ref.append(k, ks, kn, start, [T, T])
        ref.append(v, vs, vn, start, [T, T])
        for _ in range(2):                                       # the same rows again change nothing
            c.append(dk, dv, start.cuda())
            for got, want in zip(cache_values(c), (k, ks, v, vs)):
                same(got, want)
    assert not big.k[0].float().any() and not big.k[:, 0].float().any() and not big.k_scale[0].any()


def test_append_of_no_numbers_and_zeros():
    c = q8().CacheQ8.new(1, 1, 40, 16)
    k, ks, v, vs = cache_values(c)
    rows = torch.zeros(1, 1, 4, 16)
    rows[0, 0, 1], rows[0, 0, 2, 3], rows[0, 0, 3, 5], rows[0, 0, 3, 6] = 2.0, math.nan, math.inf, -math.inf
    tiny = torch.randn(1, 1, 3, 16, generator=gen(3)) * 1e-41
    for n, (new, at) in enumerate(((torch.zeros(1, 1, 2, 16), 0), (rows, 2), (torch.zeros(1, 1, 1, 16), 6), (rows * 100, 30), (tiny, 34), (tiny, 0))):
        start = torch.tensor([at], dtype=torch.int32)
        c.append(new.cuda(), (new * 2).cuda(), start.cuda())
        ref.append(k, ks, new, start, [new.shape[2]])
        ref.append(v, vs, new * 2, start, [new.shape[2]])
        for got, want in zip(cache_values(c), (k, ks, v, vs)):
            same(got, want)
    sync()


@TYPES
def test_append_of_values_at_borders_between_codes(dtype):
    """Quotients on borders between codes and next to them, at scales that are powers of two and at others, tiny ones among them; and the earlier
    rows of a block, rounded again to a scale that brings codes onto borders."""
    every = torch.arange(127, dtype=torch.uint8).view(E4M3).double()
    mid = (every[1:] + every[:-1]) / 2
    x = torch.cat([mid, -mid, torch.tensor([448.0, 0.0, -0.0, 448.0])])          # 256
    for f in (1.0, 2.0 ** -7, 0.7, 3.3) + ((1e-22, 1e25) if dtype is torch.float32 else ()):
        t = (x * f).to(dtype)
        rows = torch.stack([t, torch.nextafter(t, torch.full_like(t, math.inf)), torch.nextafter(t, torch.full_like(t, -math.inf))])[None, None]
        c = q8().CacheQ8.new(1, 1, 40, 256)
        k, ks, v, vs = cache_values(c)
        for new, at in ((rows, 0), (rows * 2, 3), (rows * 3, 30)):
            start = torch.tensor([at], dtype=torch.int32)
            c.append(new.cuda(), new.flip(-1).cuda(), start.cuda())
            ref.append(k, ks, new, start, [3])
            ref.append(v, vs, new.flip(-1), start, [3])
            for got, want in zip(cache_values(c), (k, ks, v, vs)):
                same(got, want)
    sync()


def test_append_outside_of_the_cache_is_left_out_and_told():
    from deers_b200 import _lib
    from deers_b200.errors import CudaError
    for at, count, kept in ((7, 4, 3), (10, 1, 0), (-1, 2, 0), (2 ** 31 - 1, 4, 0), (0, -3, 0), (3, 9, 4)):
        c = q8().CacheQ8.new(1, 1, 10, 16)
        new = torch.ones(1, 1, 4, 16).cuda()
        c.append(new, new, torch.tensor([at], dtype=torch.int32).cuda(), torch.tensor([count], dtype=torch.int32).cuda())
        with pytest.raises(CudaError) as e:
            sync()
        assert e.value.status == _lib.ERR_KERNEL
        assert int((c.k.float()[0, 0, :, 0] != 0).sum()) == kept
    sync()


# ---- attention over the cache -------------------------------------------------------------------------------------------
def filled(g, B, H, cap, D):
    """A cache with codes everywhere and a NaN behind nothing that is read: code values, scales and the library's object."""
    x = [torch.randn(B, H, cap, D, generator=g) * (0.1 + 3 * torch.rand(B, H, cap, 1, generator=g)) for _ in range(2)]
    out = []
    for t in x:
        n = -(-cap // 32)
        p = torch.nn.functional.pad(t, (0, 0, 0, n * 32 - cap)).reshape(B, H, n, 32, D)
        s = p.abs().amax((-1, -2)) / 448
        out += [ref.nearest(p.double() / s.double()[..., None, None], E4M3).reshape(B, H, n * 32, D)[:, :, :cap].clone(), s]
    return out[0], out[1], out[2], out[3]


def on_device(k, ks, v, vs):
    return q8().CacheQ8(k.float().to(E4M3).cuda(), v.float().to(E4M3).cuda(), ks.cuda(), vs.cuda())


def check_decode(q, cache, lengths, causal=True, scale=None, got=None):
    k, ks, v, vs = cache
    if got is None:
        got = q8().attention_decode_q8(q.cuda(), on_device(*cache), lengths.cuda(), scale, causal, want_lse=True)
        sync()
    s = 1 / math.sqrt(q.shape[3]) if scale is None else scale
    o, lse, err_o, err_l = ref.decode(q, k, ks, v, vs, lengths, s, causal)
    near(got[0], o, err_o[..., None] + ref.half_step(o, q.dtype))
    near(got[1], lse, err_l)


DECODE = [  # B, H, G, Tq, D, cap, lengths
    (1, 1, 1, 1, 16, 1, [1]), (1, 12, 1, 1, 64, 800, [777]), (2, 4, 2, 1, 32, 100, [0, 100]), (3, 6, 3, 2, 80, 300, [1, 2, 299]),
    (2, 8, 8, 1, 128, 513, [512, 33]), (2, 16, 8, 2, 96, 400, [400, 31]), (1, 8, 4, 5, 256, 130, [130]), (2, 3, 1, 7, 48, 64, [3, 64]),
    (1, 2, 1, 1, 64, 20000, [19999]), (1, 1, 1, 3, 128, 40000, [39000]), (5, 2, 2, 8, 112, 257, [5, 8, 100, 256, 257]), (1, 32, 32, 2, 64, 600, [555]),
    (40, 8, 1, 1, 128, 96, list(range(57, 97))), (1, 4, 4, 3, 32, 90, [77]), (2, 2, 1, 1, 96, 500, [311, 500]), (20, 16, 1, 1, 64, 40, list(range(1, 41, 2))),
    # (up to 64 slices of 16384 keys and more are walked in even shares of all keys)
    (3, 8, 4, 3, 96, 17000, [0, 17000, 5]), (2, 4, 4, 1, 256, 16384, [16384, 7]), (40, 1, 1, 1, 16, 16384, [(i * i * 37) % 1700 for i in range(39)] + [16384]),
    (3, 2, 2, 8, 32, 16385, [16385, 9, 16384]), (2, 2, 2, 2, 64, 16400, [0, 0]), (65, 2, 2, 1, 16, 16384, [(i * i * 37) % 1700 for i in range(64)] + [16384])]


@TYPES
@pytest.mark.parametrize("B,H,G,Tq,D,cap,lengths", DECODE, ids=lambda v: str(v) if not isinstance(v, list) else "")
def test_decode(B, H, G, Tq, D, cap, lengths, dtype):
    g = gen(B * 3 + H + G + Tq + D + cap)
    cache = filled(g, B, H // G, cap, D)
    q = torch.randn(B, H, Tq, D, generator=g).to(dtype)
    n = torch.tensor(lengths, dtype=torch.int32)
    check_decode(q, cache, n)
    if Tq > 1:
        check_decode(q, cache, n, causal=False)
    check_decode(q * 20, cache, n, scale=0.3)


@TYPES
def test_decode_of_views_and_token_major_queries(dtype):
    g = gen(31)
    k, ks, v, vs = filled(g, 3, 4, 150, 64)
    dev = [t.float().to(E4M3).cuda() for t in (k, v)]
    c = q8().CacheQ8(dev[0][1:, 1:3, 32:], dev[1][1:, 1:3, 32:], ks.cuda()[1:, 1:3, 1:], vs.cuda()[1:, 1:3, 1:])
    flat = torch.randn(2, 2, 4 * 64 + 1, generator=g).to(dtype)
    n = torch.tensor([118, 60], dtype=torch.int32)
    for shift in (0, 1):
        q = flat[..., shift:shift + 256].unflatten(-1, (4, 64)).permute(0, 2, 1, 3)
        dq = flat.cuda()[..., shift:shift + 256].unflatten(-1, (4, 64)).permute(0, 2, 1, 3)
        got = q8().attention_decode_q8(dq, c, n.cuda(), want_lse=True)
        check_decode(q, (k[1:, 1:3, 32:], ks[1:, 1:3, 1:], v[1:, 1:3, 32:], vs[1:, 1:3, 1:]), n, got=got)


@TYPES
@pytest.mark.parametrize("D,cap", [(64, 90), (128, 700), (256, 5000), (96, 17000), (32, 75)])
def test_decode_is_not_reached_by_what_it_does_not_see(D, cap, dtype):
    """NaN codes behind the last row, and in keys that some of a call's rows see and others do not."""
    g = gen(D)
    k, ks, v, vs = filled(g, 2, 2, cap, D)
    n = torch.tensor([cap - 5, cap // 2], dtype=torch.int32)
    for b in range(2):
        k[b, :, int(n[b]):] = math.nan
        v[b, :, int(n[b]):] = math.nan
        if int(n[b]) % 32 == 0:
            continue
        ks[b, :, -(-int(n[b]) // 32):] = math.nan
        vs[b, :, -(-int(n[b]) // 32):] = math.nan
    q = torch.randn(2, 4, 3, D, generator=g).to(dtype)
    check_decode(q, (k, ks, v, vs), n)
    v[0, 0, int(n[0]) - 1, 3] = math.nan                         # seen by the last of three rows
    v[1, 1, int(n[1]) - 2, 0] = math.nan                         # by the last two
    k[1, 0, int(n[1]) - 1, 5] = math.nan
    check_decode(q, (k, ks, v, vs), n)
    v[0, 1, 2, 7] = math.nan                                     # by all
    check_decode(q, (k, ks, v, vs), n)
    q[0, 0, 1, 0], q[1, 3, 0, 2] = math.nan, math.inf            # a query of no number is its own row's alone
    got = q8().attention_decode_q8(q.cuda(), on_device(k, ks, v, vs), n.cuda(), want_lse=True)
    o = got[0].cpu()
    assert torch.isnan(o[0, 0, 1]).all() and torch.isnan(o[1, 3, 0]).all()
    want = ref.decode(torch.nan_to_num(q, 0, 0, 0), k, ks, v, vs, n, 1 / math.sqrt(D))
    keep = torch.ones(2, 4, 3, dtype=torch.bool)
    keep[0, 0, 1] = keep[1, 3, 0] = False
    near(o[keep], want[0][keep], (want[2][..., None] + ref.half_step(torch.nan_to_num(want[0]), dtype))[keep])


def test_decode_with_scales_of_all_sizes():
    """Blocks whose scales differ by powers of ten, blocks of zeros, and values that are all tiny or all large."""
    g = gen(41)
    for f in (1.0, 1e-30, 1e30):
        k, ks, v, vs = filled(g, 1, 2, 256, 64)
        vs *= f * torch.tensor([1.0, 1e-6, 0.0, 1e3, 1e-12, 1.0, 1e-3, 1.0])
        v[:, :, 64:96] = 0
        ks[..., 5], k[:, :, 160:192] = 0.0, 0
        check_decode(torch.randn(1, 2, 1, 64, generator=g), (k, ks, v, vs), torch.tensor([250], dtype=torch.int32))
    # queries of all sizes in f32
    k, ks, v, vs = filled(g, 1, 2, 256, 64)
    for f in (1e-30, 1e-6, 1e4):
        check_decode(torch.randn(1, 2, 1, 64, generator=g) * f, (k, ks, v, vs), torch.tensor([256], dtype=torch.int32), scale=0.1 / f if f > 1e-20 else 1.0)


def test_decode_of_the_smallest_and_largest_numbers():
    """f32: values next to the subnormals keep their bits, queries beyond f16's largest times 2^100 are scaled into its range."""
    g = gen(43)
    n = torch.tensor([250], dtype=torch.int32)
    k, ks, v, vs = filled(g, 1, 2, 256, 64)
    check_decode(torch.zeros(1, 2, 1, 64), (k, ks, v, vs * 1e-35), n)        # (equal weights: nothing but the values' own error)
    check_decode(torch.randn(1, 2, 1, 64, generator=g) * 1e36, (k, ks, v, vs), n, scale=1e-37)


def test_decode_of_lengths_outside_of_the_cache_is_told():
    from deers_b200.errors import CudaError
    g = gen(51)
    cache = filled(g, 2, 1, 40, 32)
    q = torch.randn(2, 1, 1, 32, generator=g)
    got = q8().attention_decode_q8(q.cuda(), on_device(*cache), torch.tensor([41, -1], dtype=torch.int32).cuda(), want_lse=True)
    with pytest.raises(CudaError):
        sync()
    check_decode(q, cache, torch.tensor([40, 0]), got=got)


# ---- together -----------------------------------------------------------------------------------------------------------
class Block:
    """Attention and MLP of one block, as a served model calls them."""

    def __init__(self, g, C, H, Hkv, hidden, codes):
        D = C // H
        self.H, self.Hkv, self.D, self.codes = H, Hkv, D, codes
        sizes = {"qkv": (C, (H + 2 * Hkv) * D), "out": (C, C), "up": (C, hidden), "down": (hidden, C)}
        self.plain = {n: (torch.randn(s, generator=g) / math.sqrt(s[0])).half() for n, s in sizes.items()}
        self.w = {n: q8().quantize_weight_q8(w.cuda(), codes) for n, w in self.plain.items()}

    def step(self, x, residual, cache, start, lengths):
        """x, residual [B, T, C] -> (the stream, what is to be added to it)."""
        m = q8()
        B, T, C = x.shape
        h, rows = m.rms_norm_add_q8(x, residual, 1e-5, self.codes)
        qkv = m.linear_q8(rows, self.w["qkv"]).unflatten(-1, (self.H + 2 * self.Hkv, self.D)).permute(0, 2, 1, 3)
        q, k, v = qkv.split([self.H, self.Hkv, self.Hkv], 1)
        cache.append(k, v, start)
        o = m.attention_decode_q8(q, cache, lengths)
        y = m.linear_q8(m.quantize_q8(o.permute(0, 2, 1, 3).reshape(B, T, C), self.codes), self.w["out"])
        h, rows = m.rms_norm_add_q8(y, h, 1e-5, self.codes)
        u = m.linear_q8(rows, self.w["up"])
        return h, m.linear_q8(m.quantize_q8(u, self.codes, relu_squared=True), self.w["down"])

    def want(self, x, residual, past):
        """The same block in f64 without any 8 bits: what the 8-bit one approximates.  past: (k, v) [B,Hkv,n,D]."""
        w = {n: t.double() for n, t in self.plain.items()}
        B, T, C = x.shape
        h = x.double() + residual.double()
        norm = lambda t: t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-5)  # noqa: E731
        qkv = (norm(h) @ w["qkv"]).unflatten(-1, (self.H + 2 * self.Hkv, self.D)).permute(0, 2, 1, 3)
        q, k, v = qkv.split([self.H, self.Hkv, self.Hkv], 1)
        k, v = (torch.cat([p, n], 2) for p, n in zip(past, (k, v)))
        G, n = self.H // self.Hkv, k.shape[2]
        s = q @ k.repeat_interleave(G, 1).transpose(-1, -2) / math.sqrt(self.D)
        s = s.masked_fill(torch.arange(n)[None] > torch.arange(T)[:, None] + n - T, -math.inf)
        o = (torch.softmax(s, -1) @ v.repeat_interleave(G, 1)).permute(0, 2, 1, 3).reshape(B, T, C)
        h = h + o @ w["out"]
        return h, torch.relu(norm(h) @ w["up"]).square() @ w["down"], (k, v)


@CODES
def test_a_block_decodes_step_by_step(codes):
    """A prompt and single tokens through cache and attention, against the block without 8 bits.  A value loses at most half a step where it
    becomes a code: e4m3 2^-4 of itself, int8 1/254 of its row's largest; errors of thousands of values add up as their root, so the
    outputs are within a tenth (e4m3) or a twentieth (int8 rows, cache in e4m3) of their norm."""
    g = gen(61)
    B, C, H, Hkv, T0, steps = 2, 256, 4, 2, 37, 4
    block = Block(g, C, H, Hkv, 640, codes)
    cache = q8().CacheQ8.new(B, Hkv, 64, C // H)
    past = tuple(torch.zeros(B, Hkv, 0, C // H, dtype=torch.float64) for _ in range(2))
    at = 0
    for T in [T0] + [1] * steps:
        x, r = (torch.randn(B, T, C, generator=g).half() for _ in range(2))
        start = torch.full((B,), at, dtype=torch.int32, device="cuda")
        got = block.step(x.cuda(), r.cuda(), cache, start, start + T)
        h, y, past = block.want(x, r, past)
        for a, b in zip(got, (h, y)):
            off = float((a.cpu().double() - b).norm() / b.norm())
            assert off < (0.1 if codes is E4M3 else 0.05), off
        at += T
    sync()


def test_a_padded_batch_of_prompts():
    """Prompts of unlike lengths, padded at the back: query t of every sequence sees rows up to its own when the lengths are start + T; what the
    padding's queries see is nobody's."""
    g = gen(67)
    B, H, T, D = 3, 2, 45, 64
    counts = torch.tensor([45, 1, 33], dtype=torch.int32)
    k, v = (torch.randn(B, H, T, D, generator=g).half() for _ in range(2))
    q = torch.randn(B, 2 * H, T, D, generator=g).half()
    cache = q8().CacheQ8.new(B, H, 64, D)
    start = torch.tensor([0, 16, 2], dtype=torch.int32)
    cache.append(k.cuda(), v.cuda(), start.cuda(), counts.cuda())
    got = q8().attention_decode_q8(q.cuda(), cache, (start + T).cuda(), want_lse=True)
    sync()
    values = cache_values(cache)
    for i in range(B):
        n = int(counts[i])
        one = [t[i:i + 1] for t in values]
        check_decode(q[i:i + 1, :, :n], (one[0], one[1], one[2], one[3]), start[i:i + 1] + n, got=[t[i:i + 1, :, :n] for t in got])


def test_a_captured_step_serves_every_length():
    """The chain recorded once and replayed at growing lengths equals the same calls made one by one, beside a second captured chain."""
    g = gen(71)
    B, C, H = 2, 128, 2
    block = Block(g, C, H, H, 320, I8)
    side = torch.cuda.Stream()
    chains = []
    for n in range(2):
        c = {"cache": q8().CacheQ8.new(B, H, 400, C // H), "start": torch.zeros(B, dtype=torch.int32, device="cuda"),
             "x": torch.zeros(B, 1, C, dtype=torch.float16, device="cuda"), "r": torch.zeros(B, 1, C, dtype=torch.float16, device="cuda")}
        with torch.cuda.stream(side):
            for _ in range(2):
                block.step(c["x"], c["r"], c["cache"], c["start"], c["start"] + 1)
            side.synchronize()
            c["graph"] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(c["graph"], stream=side):
                c["out"] = block.step(c["x"], c["r"], c["cache"], c["start"], c["start"] + 1)
        chains.append(c)
    plain = [q8().CacheQ8.new(B, H, 400, C // H) for _ in chains]
    for step in range(40):
        xs = [[torch.randn(B, 1, C, generator=g).half().cuda() for _ in range(2)] for _ in chains]
        for c, (x, r) in zip(chains, xs):                        # both replayed before either is looked at
            c["x"].copy_(x)
            c["r"].copy_(r)
            c["start"].fill_(step * 7)
            c["graph"].replay()
        for c, p, (x, r) in zip(chains, plain, xs):
            start = torch.full((B,), step * 7, dtype=torch.int32, device="cuda")
            want = block.step(x, r, p, start, start + 1)
            torch.cuda.synchronize()
            for a, b in zip(c["out"], want):
                assert torch.equal(a, b)
    for c, p in zip(chains, plain):
        assert torch.equal(c["cache"].k.view(torch.uint8), p.k.view(torch.uint8)) and torch.equal(c["cache"].v_scale, p.v_scale)


def test_results_do_not_change_from_run_to_run():
    g = gen(81)
    cache = on_device(*filled(g, 2, 2, 3000, 128))
    q = torch.randn(2, 4, 2, 128, generator=g).half().cuda()
    n = torch.tensor([3000, 1700], dtype=torch.int32).cuda()
    rows, w = (q8().quantize_q8(torch.randn(s, 4096, generator=g).cuda(), E4M3) for s in (33, 200))
    first = q8().attention_decode_q8(q, cache, n), q8().linear_q8(rows, w)
    for _ in range(20):
        assert torch.equal(q8().attention_decode_q8(q, cache, n), first[0])
        assert torch.equal(q8().linear_q8(rows, w), first[1])


def test_another_stream_and_the_current_device_stay():
    g = gen(91)
    x = torch.randn(64, 512, generator=g).cuda()
    want = q8().quantize_q8(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = q8().quantize_q8(x)
        y = q8().linear_q8(got, got)
    torch.cuda.synchronize()
    assert torch.equal(got.codes, want.codes) and torch.equal(y, q8().linear_q8(want, want))
    assert torch.cuda.current_device() == 0
