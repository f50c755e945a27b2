"""The 8-bit operators where they can go wrong: places outside of a cache in front of other operators, scales of unlike sizes, rows whose squares leave
f32, every form of the products, layouts and lengths at the ends of what is taken."""
import math

import pytest
import torch

from tests.test_q8_gpu import E4M3, filled, gen, on_device, q8, same, sync

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
