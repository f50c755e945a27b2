"""The 8-bit operators where they can go wrong: places outside of a cache in front of other operators, scales of unlike sizes, rows whose squares leave
f32, every form of the products, layouts and lengths at the ends of what is taken."""
import ctypes
import math

import pytest
import torch

from tests import q8_util as ref
from tests.test_q8_gpu import CODES, TYPES, E4M3, I8, cache_values, check_linear, check_rows, filled, gen, make_rows, near, on_device, q8, same, sync

pytestmark = pytest.mark.gpu


# ---- places and lengths outside of a cache, and what runs behind them ------------------------------------------------------
def _behind_a_report(call):
    """What products give behind a call that reports a place or length, before the context is asked: the same as without it."""
    from deers_b200 import ops
    from deers_b200.errors import CudaError
    g = gen(7)
    rows, w = q8().quantize_q8(torch.randn(40, 300, generator=g).cuda()), q8().quantize_q8(torch.randn(90, 300, generator=g).cuda())
    many, wide = (q8().quantize_q8(torch.randn(n, 64, generator=g).cuda(), E4M3) for n in (4000, 600))
    x, lin = torch.randn(130, 64, generator=g).half().cuda(), torch.randn(64, 136, generator=g).half().cuda()
    t = torch.randn(1, 2, 200, 64, generator=g).half().cuda()
    run = lambda: [q8().linear_q8(rows, w), q8().linear_q8(many, wide), ops._gemm(130, 136, 64, x, 0, lin, 1), ops.CausalAttention.new(t, t, t).forward()]  # noqa: E731
    flat = lambda ts: [u for t in ts for u in (t if isinstance(t, (tuple, list)) else [t])]  # noqa: E731
    want = flat(run())
    sync()
    del_me = [torch.full_like(t, math.nan) for t in want]        # what a call that writes nothing would find in its memory
    torch.cuda.synchronize()
    del del_me
    call()
    got = flat(run())
    with pytest.raises(CudaError):
        sync()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    sync()                                                       # told once


def test_append_outside_of_the_cache_leaves_other_operators_alone():
    c = q8().CacheQ8.new(2, 1, 10, 16)
    new = torch.ones(2, 1, 4, 16).cuda()
    start = torch.tensor([2, 9], dtype=torch.int32).cuda()
    _behind_a_report(lambda: c.append(new, new, start))
    assert (c.k.float()[0, 0, 2:6] == 448).all() and (c.k.float()[1, 0, 9] == 448).all()


def test_decode_of_a_length_outside_of_the_cache_leaves_other_operators_alone():
    g = gen(8)
    c, q = on_device(*filled(g, 2, 1, 40, 32)), torch.randn(2, 1, 1, 32, generator=g).cuda()
    n = torch.tensor([41, 20], dtype=torch.int32).cuda()
    _behind_a_report(lambda: q8().attention_decode_q8(q, c, n))


def test_a_sequence_that_brings_no_rows_is_no_report():
    """Idle sequences, wherever they are said to stand."""
    c = q8().CacheQ8.new(4, 1, 10, 16)
    new = torch.ones(4, 1, 4, 16).cuda()
    start, count = (torch.tensor(t, dtype=torch.int32).cuda() for t in ([-1, 11, 10, 6], [0, 0, 0, 4]))
    c.append(new, new, start, count)
    sync()
    assert not c.k.float()[:3].any() and not c.k_scale[:3].any() and (c.k.float()[3, 0, 6:] == 448).all()


def test_a_captured_step_with_a_full_sequence_serves_the_others():
    """Replays of append, attention and a product where one sequence has run out of its cache: the others' rows, every time."""
    from deers_b200.errors import CudaError
    g = gen(9)
    D = 32
    c, p = (q8().CacheQ8.new(2, 1, 40, D) for _ in range(2))
    w = q8().quantize_weight_q8(torch.randn(D, 50, generator=g).cuda())
    x = torch.zeros(2, 1, 1, D, dtype=torch.float16, device="cuda")
    start = torch.zeros(2, dtype=torch.int32, device="cuda")

    def step(cache):
        cache.append(x, x, start)
        o = q8().attention_decode_q8(x, cache, start + 1)
        return q8().linear_q8(q8().quantize_q8(o[:, 0, 0]), w)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(c)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(c)
    torch.cuda.synchronize()
    for at in range(3):
        x.copy_(torch.randn(2, 1, 1, D, generator=g))
        start.copy_(torch.tensor([at, 39 + at], dtype=torch.int32))
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        start.copy_(torch.tensor([at, 0], dtype=torch.int32))
        assert torch.equal(out[0], step(p)[0])
    from deers_b200 import ops
    with torch.cuda.stream(side), pytest.raises(CudaError):
        ops.Context.current(torch.device("cuda", 0)).sync()
    sync()


# ---- attention over blocks whose scales and weights are far apart ----------------------------------------------------------
def _weighed(q, cache, lengths, scale, dtype, causal=True):
    """(o, lse) by definition, and how far an f32 computation of o may be off: every key's share of o by the error of its own score (a sum of as many products
    as q has channels, 2^-23 of their sizes each, and the roundings behind it), of its weight (two f16 and exp2, 2^-21) and of the sums over the keys."""
    k, ks, v, vs = cache
    B, H, Tq, D = q.shape
    G, q = H // k.shape[1], q.double()
    o, lse, err = torch.zeros_like(q), torch.full((B, H, Tq), -math.inf, dtype=torch.float64), torch.zeros_like(q)
    for b in range(B):
        n = int(lengths[b])
        of = torch.arange(n) // 32
        for h in range(H):
            kk, vv = (t[b, h // G, :n].double() * s[b, h // G].double()[of][:, None] for t, s in ((k, ks), (v, vs)))
            for i in range(Tq):
                m = n - (Tq - 1 - i) if causal else n
                if m <= 0:
                    continue
                s = kk[:m] @ q[b, h, i] * scale
                p, ds = torch.softmax(s, 0), (int((q[b, h, i] != 0).sum()) + 16) * 2.0 ** -23 * (kk[:m].abs() @ q[b, h, i].abs()) * abs(scale)
                lse[b, h, i], o[b, h, i] = torch.logsumexp(s, 0), p @ vv[:m]
                # (the weights' sum is off by the weighed errors of the scores)
                each = ds + float(p @ ds) + 2 * 2.0 ** -21 + 2 * (m / 8 + 64) * 2.0 ** -23
                err[b, h, i] = (p * each) @ vv[:m].abs()
    return o, lse, err + ref.half_step(o, dtype)


def _far_apart(g, H, cap, D, ratio, dip, at):
    """A cache whose keys score within a tenth of 0 along channel 0, but those of block `at`, whose scores are `dip` and whose values are `ratio` larger."""
    k = torch.randn(1, H, cap, D, generator=g)
    k[..., 0] = (torch.rand(1, H, cap, generator=g) - 0.5) * 0.2
    v = torch.randn(1, H, cap, D, generator=g)
    lo, hi = 32 * at, min(cap, 32 * at + 32)
    k[:, :, lo:hi, 0] = dip * (1 + 0.05 * torch.rand(1, H, hi - lo, generator=g))
    v[:, :, lo:hi] *= ratio
    out = []
    for t in (k, v):
        n = -(-cap // 32)
        p = torch.nn.functional.pad(t, (0, 0, 0, n * 32 - cap)).reshape(1, H, n, 32, D)
        s = p.abs().amax((-1, -2)) / 448
        out += [ref.nearest(p.double() / s.double()[..., None, None], E4M3).reshape(1, H, n * 32, D)[:, :, :cap].clone(), s]
    return out


# heads, query heads a head, rows, width, capacity, keys: whole slices, clusters, even shares; eight and sixteen query rows
FAR = [(1, 1, 1, 64, 128, 100), (150, 1, 1, 64, 640, 640), (2, 1, 1, 32, 90, 90), (1, 4, 2, 128, 2048, 1500), (1, 16, 1, 96, 1000, 999), (1, 2, 1, 256, 700, 650), (1, 8, 2, 64, 16384, 3000)]


@TYPES
@pytest.mark.parametrize("H,G,Tq,D,cap,n", FAR, ids=lambda v: str(v))
@pytest.mark.parametrize("ratio", [1e7, 1e9, 1e12, 1e-12], ids=lambda v: f"{v:g}")
def test_decode_with_large_values_of_no_weight(H, G, Tq, D, cap, n, ratio, dtype):
    """A block with values far larger than the others' and a softmax weight of e^-60: the outputs are the others', with all their bits.  In front, in the middle
    and at the end; and values far smaller that have all the weight."""
    g = gen(D + cap + Tq)
    q = torch.zeros(1, H * G, Tq, D)
    q[..., 0] = 1.0 + 0.1 * torch.rand(1, H * G, Tq, generator=g)
    q = q.to(dtype)
    dip = -60.0 if ratio > 1 else 60.0
    lengths = torch.tensor([n], dtype=torch.int32)
    for at in (0, 1, (n - 1) // 32):
        cache = _far_apart(g, H, cap, D, ratio, dip, at)
        got = q8().attention_decode_q8(q.cuda(), on_device(*cache), lengths.cuda(), 1.0, want_lse=True)
        sync()
        o, lse, err = _weighed(q, cache, lengths, 1.0, dtype)
        near(got[0], o, err)


@TYPES
def test_decode_rows_weigh_large_values_each_for_itself(dtype):
    """Of the query rows of a head some have all their weight on a block of large values and others none there; rows that do not see the block at all."""
    g = gen(77)
    for D, cap, n, at in ((64, 97, 97, 3), (128, 1025, 1025, 32), (64, 640, 640, 0), (128, 1025, 1025, 4)):      # (1025 and 97: the last key is a block of its own)
        cache = _far_apart(g, 1, cap, D, 1e4, 10.0, at)
        q = torch.zeros(1, 4, 3, D)
        q[..., 0] = torch.tensor([1.0, -1.0, 0.0, -6.0])[None, :, None]
        q = q.to(dtype)
        cache[3][0, 0, at] *= 2.0 ** 30                          # values 1e13 of the others'
        lengths = torch.tensor([n], dtype=torch.int32)
        got = q8().attention_decode_q8(q.cuda(), on_device(*cache), lengths.cuda(), 1.0, want_lse=True)
        sync()
        o, lse, err = _weighed(q, cache, lengths, 1.0, torch.float32)
        if dtype is torch.float16:                               # (values that f16 holds; the others become infinite, as they should)
            err = err + ref.half_step(o, dtype)
            o = torch.where(o.abs() > 65519.0, o.sign() * math.inf, o)
        near(got[0], o, torch.where(torch.isfinite(err), err, torch.zeros_like(err)))


def test_decode_with_values_of_every_size_beside_one_another():
    """f32: scales from 2^-100 to 2^4 in the blocks of one walk, weights from 1 to 2^-99."""
    g = gen(79)
    for D, cap in ((64, 448), (128, 448)):
        cache = _far_apart(g, 1, cap, D, 1.0, 0.0, 0)
        n = -(-cap // 32)
        for order in (range(n), range(n - 1, -1, -1)):
            for i, j in enumerate(order):                        # block j: values 2^(8 i) of the smallest, scores -5.3 i (2^-7.6 i)
                cache[3][0, 0, j] = 2.0 ** (-100 + 8 * i)
                rows = cache[0][0, 0, 32 * j:32 * j + 32]
                rows[:, 0] = -448.0
                cache[1][0, 0, j] = 5.3 * i / 448 if i else 0.01 / 448
            q = torch.zeros(1, 2, 1, D)
            q[..., 0] = 1.0
            lengths = torch.tensor([cap], dtype=torch.int32)
            got = q8().attention_decode_q8(q.cuda(), on_device(*cache), lengths.cuda(), 1.0, want_lse=True)
            sync()
            o, lse, err = _weighed(q, cache, lengths, 1.0, torch.float32)
            near(got[0], o, err)


def test_decode_refuses_queries_of_other_shapes():
    from deers_b200.errors import LayoutMismatch
    c, n = q8().CacheQ8.new(2, 3, 40, 32), torch.zeros(2, dtype=torch.int32, device="cuda")
    for shape in ((2, 3, 1, 0), (2, 3, 0, 32), (2, 0, 1, 32), (1, 3, 1, 32), (2, 4, 1, 32), (2, 3, 41, 32), (2, 3, 32), (2, 3, 1, 48)):
        with pytest.raises(LayoutMismatch):
            q8().attention_decode_q8(torch.zeros(shape, device="cuda"), c, n)


# ---- the norm of rows whose squares leave f32 --------------------------------------------------------------------------------
@CODES
@pytest.mark.parametrize("C", [5, 64, 300, 1025, 2048, 5000, 9001, 16000])
def test_norm_of_the_smallest_and_largest_rows(C, codes):
    """Rows of every size of f32; the norm of one does not depend on its size (without eps)."""
    base = torch.randn(7, C, generator=gen(C))
    size = torch.tensor([1e36, 1e25, 3e18, 1e-18, 1e-23, 1e-30, 1e-41])
    x = (base / base.abs().amax(1, keepdim=True) * size[:, None]).float()
    for eps in (0.0, 1e-5):
        h, got = q8().rms_norm_add_q8(x.cuda(), None, eps, codes)
        sync()
        check_rows(got, h, x, None, True, False, eps, codes)
    x, r = (x * 0.75).float(), (x.flip(1) * 0.25).float()
    h, got = q8().rms_norm_add_q8(x.cuda(), r.cuda(), 0.0, codes)
    check_rows(got, h, x, r, True, False, 0.0, codes)


@pytest.mark.parametrize("C", [40, 5000, 9001])
def test_norm_of_the_largest_rows_into_a_callers_buffers(C):
    """The sum in the residual's place, or in x's."""
    from deers_b200 import _lib, ops
    ctx = ops.Context.current(torch.device("cuda", 0))
    x, r = (torch.randn(6, C, generator=gen(C + s)) * 1e25 for s in range(2))
    wh, wq, ws = ref.quantize(x, r, True, False, 0.0, E4M3)
    ld = -(-C // 16) * 16
    for into in (0, 1):
        dev = [x.cuda(), r.cuda()]
        codes, scale = torch.empty(6, ld, dtype=E4M3, device="cuda"), torch.empty(6, device="cuda")
        d = _lib.QuantizeDesc(6, C, _lib.F32, _lib.E4M3, 1, 0, 0.0, C, C, C, ld)
        _lib.check(_lib.lib().deers_b200_quantize_rows(ctx.handle, ctypes.byref(d), dev[0].data_ptr(), dev[1].data_ptr(), dev[into].data_ptr(), codes.data_ptr(),
                                                       scale.data_ptr()))
        sync()
        same(dev[into], wh)
        same(codes[:, :C].float(), wq)
        near(scale, ws, ws.abs() * ref.scale_tolerance(C))


# ---- products: scales of another shape ---------------------------------------------------------------------------------------
def test_linear_refuses_scales_of_another_shape():
    from deers_b200.errors import LayoutMismatch
    m = q8()
    a, w = torch.zeros(2, 3, 32, dtype=torch.int8, device="cuda"), torch.zeros(8, 32, dtype=torch.int8, device="cuda")
    sa, sw = torch.zeros(2, 3, device="cuda"), torch.zeros(8, device="cuda")
    assert m.linear_q8(m.RowsQ8(a, sa), m.RowsQ8(w, sw)).shape == (2, 3, 8)
    for bad in (sa.t().contiguous(), sa.reshape(6), sa[..., None], sa[None]):
        with pytest.raises(LayoutMismatch):
            m.linear_q8(m.RowsQ8(a, bad), m.RowsQ8(w, sw))
    for bad in (sw[:, None], sw[None], sw.reshape(2, 4)):
        with pytest.raises(LayoutMismatch):
            m.linear_q8(m.RowsQ8(a, sa), m.RowsQ8(w, bad))


# ---- products: scales of every size ------------------------------------------------------------------------------------------
@CODES
@pytest.mark.parametrize("M,N,K", [(3, 40, 100), (300, 70, 130), (300, 70, 2400), (2500, 40, 64)], ids=lambda v: str(v))
def test_linear_with_scales_of_every_size(M, N, K, codes):
    """Scales whose product is in range where that of one of them and a sum is not."""
    g = gen(M + K)
    a, b = make_rows(g, M, K, codes)[0], make_rows(g, N, K, codes)[0]
    for f, other in ((1e36, 1e-36), (1e-36, 1e36), (1e-42, 1e37), (1e38, 1e-30), (1e38, 1e-41)):
        sa, sb = (((0.5 + torch.rand(n, generator=g)) * s).float() for n, s in ((M, f), (N, other)))
        check_linear(a, sa, b, sb, codes, torch.float32)
        if f * other <= 2:
            check_linear(a, sa, b, sb * 2.0 ** -9, codes)
    sa = torch.full((M,), 2.0 ** -100)
    sa[::2] = 2.0 ** 100
    sa[1] = 0.0
    check_linear(a, sa, b, torch.full((N,), 2.0 ** -110), codes, torch.float32)


# ---- products: every kernel --------------------------------------------------------------------------------------------------
# M, N, K; kernel that takes them (persistent, by pairs), columns of its tile, its rows and columns swapped, parts of K
FORMS = [((2137, 37, 54), (True, False, 256, False, 1)), ((20001, 513, 70), (True, False, 256, False, 1)), ((5454, 1573, 609), (True, False, 256, False, 1)),
         ((2415, 38, 3597), (True, True, 256, False, 1)), ((5423, 1541, 900), (True, True, 256, False, 1)),
         ((138, 16196, 674), (False, False, 256, False, 1)), ((132, 6760, 6479), (False, False, 256, False, 2)), ((154, 2070, 12753), (False, False, 256, False, 7)),
         ((513, 520, 1024), (False, False, 128, False, 1)), ((778, 777, 2879), (False, False, 128, False, 2)), ((649, 645, 2464), (False, False, 128, False, 3)),
         ((1697, 132, 2806), (False, False, 128, False, 4)), ((333, 1001, 2731), (False, False, 128, False, 5)), ((273, 5, 2236), (False, False, 128, False, 6)),
         ((297, 34, 2368), (False, False, 128, False, 7)), ((262, 1, 2787), (False, False, 128, False, 8)),
         ((34, 130, 1641), (False, False, 64, True, 7)), ((35, 2395, 912), (False, False, 64, True, 4)), ((18, 3969, 1094), (False, False, 32, True, 3)),
         ((19, 77, 916), (False, False, 32, True, 8)), ((1, 2159, 1834), (False, False, 16, True, 5))]


@CODES
@pytest.mark.parametrize("out", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("size,form", FORMS, ids=lambda v: "-".join(map(str, v)))
def test_linear_by_every_kernel(size, form, out, codes):
    """One size or more for every kernel, with remainders in rows, columns and K, several tiles a block, more K blocks than stages and fewer."""
    from deers_b200 import _lib, ops
    M, N, K = size
    r = ops.Context.current(torch.device("cuda", 0)).product_route(_lib.PRODUCT_Q8, [(M, N)], K)
    assert (bool(r.persistent), bool(r.pair), r.tile_m if r.swapped else r.tile_n, bool(r.swapped), r.parts) == form
    g = gen(M + N + K)
    a, sa = make_rows(g, M, K, codes)
    b, sb = make_rows(g, N, K, codes, 1 / math.sqrt(K))
    m = q8()
    y = m.linear_q8(m.RowsQ8(a.to(codes).cuda(), sa.cuda()), m.RowsQ8(b.to(codes).cuda(), sb.cuda()), out)
    sync()
    a, b, both = a.cuda(), b.cuda(), (sa.double()[:, None] * sb.double()[None]).cuda()
    want, size = (a @ b.t()) * both, (a.abs() @ b.abs().t()) * both
    sums = 0.0 if codes is I8 else (K / 32 + 32) * 2.0 ** -23     # (as in check_linear)
    near(y, want.cpu(), (ref.half_step(want, out) * (1 + 2.0 ** -10) + 2.0 ** -22 * want.abs() + sums * size).cpu())


# ---- a cache with tokens in front of heads -----------------------------------------------------------------------------------
@TYPES
@pytest.mark.parametrize("B,H,G,Tq,D,cap", [(2, 3, 2, 1, 64, 70), (1, 5, 1, 2, 80, 300), (3, 2, 4, 4, 256, 100), (2, 1, 2, 1, 128, 90)], ids=lambda v: str(v))
def test_a_cache_with_tokens_in_front_of_heads(B, H, G, Tq, D, cap, dtype):
    """Codes [B, capacity, H, D] seen as [B, H, capacity, D]: append into them and attention over them."""
    g = gen(B + H + D + cap)
    codes = [torch.zeros(B, cap, H, D).to(E4M3).cuda().permute(0, 2, 1, 3) for _ in range(2)]
    scales = [torch.zeros(B, H, -(-cap // 32)).cuda() for _ in range(2)]
    c = q8().CacheQ8(codes[0], codes[1], scales[0], scales[1])
    k, ks, v, vs = cache_values(c)
    at = torch.zeros(B, dtype=torch.int32)
    for T in (cap - 20, 5, Tq):
        kn, vn = (torch.randn(B, H, T, D, generator=g).to(dtype) for _ in range(2))
        c.append(kn.cuda(), vn.cuda(), at.cuda())
        ref.append(k, ks, kn, at, [T] * B)
        ref.append(v, vs, vn, at, [T] * B)
        at += T
    for got, want in zip(cache_values(c), (k, ks, v, vs)):
        same(got, want)
    q = torch.randn(B, H * G, Tq, D, generator=g).to(dtype)
    got = q8().attention_decode_q8(q.cuda(), c, at.cuda(), want_lse=True)
    sync()
    o, lse, err_o, err_l = ref.decode(q, k, ks, v, vs, at, 1 / math.sqrt(D))
    near(got[0], o, err_o[..., None] + ref.half_step(o, dtype))
    near(got[1], lse, err_l)


# ---- wide rows ---------------------------------------------------------------------------------------------------------------
@CODES
@TYPES
@pytest.mark.parametrize("C", [8192, 12000, 16384, 16392, 20000])
def test_wide_rows_on_16_byte_boundaries(C, dtype, codes):
    g = gen(C)
    x, r = torch.randn(3, C, generator=g).to(dtype), (torch.randn(3, C, generator=g) * 3).to(dtype)
    h, got = q8().rms_norm_add_q8(x.cuda(), r.cuda(), 1e-5, codes)
    sync()
    check_rows(got, h, x, r, True, False, 1e-5, codes)
    check_rows(q8().quantize_q8(x.cuda(), codes, True), None, x, None, False, True, 0.0, codes)
