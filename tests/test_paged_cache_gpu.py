"""GPU: PagedKVCache beside other work of its stream, in graphs, and after refused calls."""

import pytest
import torch

import fastkernels_b200 as fk
from tests import paged_oracle as O
from tests.test_kv_cache_gpu import BF, E4, gen

pytestmark = pytest.mark.gpu


def rows(n, g, heads=2):
    return torch.randn(n, heads, 128, generator=g).to(BF).cuda()


@pytest.mark.parametrize("cache", [BF, E4])
def test_the_host_does_not_wait(cache):
    """Calls return while earlier work of their stream still runs, those that take pages and those that do not."""
    g = gen(1)
    k, v, q = rows(31, g), rows(31, g), rows(31, g, 8)
    big = torch.randn(8192, 8192, device="cuda", dtype=BF)
    for busy in (False, True):                        # first without other work: kernels are loaded and memory is taken once
        c = fk.PagedKVCache(60, 2, 128, seqs=3, dtype=cache)
        c.append(k[:21], v[:21], [15, 0, 6])
        c.attend(q[:21])
        torch.cuda.synchronize()
        for _ in range(60 if busy else 1):            # some 50 ms
            big = big @ big * 1e-2
        over = torch.cuda.Event()
        over.record()
        for new in ([5, 3, 2], [1, 1, 1], [1, 1, 1]):
            n = sum(new)
            c.append(k[:n], v[:n], new)
            out = c.attend(q[:n])
        read = c.read()
        c.release(2)
        assert not (busy and over.query())
    torch.cuda.synchronize()
    assert torch.isfinite(out).all() and read[0].shape[0] == 22 + 5 + 10 and c.lengths.tolist() == c.host_lengths == [22, 5, 0]


@pytest.mark.parametrize("ring", [None, 16, 7])
def test_many_appends_in_flight_keep_their_own_lengths(ring):
    """The host runs ahead by many appends: each attention sees the lengths and pages of its own append, also where the words that they are
    copied from are used again and again."""
    c = fk.PagedKVCache(200, 2, 128, seqs=2, page_size=2)
    if ring:
        c._ring = c._ring[:ring]
    g = gen(2)
    k, v, q = rows(200, g), rows(200, g), rows(200, g, 4)
    big = torch.randn(8192, 8192, device="cuda", dtype=BF)
    for _ in range(20):
        big = big @ big * 1e-2
    got = []
    for i in range(100):
        c.append(k[2 * i:2 * i + 2], v[2 * i:2 * i + 2])
        got.append(c.attend(q[2 * i:2 * i + 2]))
    torch.cuda.synchronize()
    order = torch.arange(100, dtype=torch.int32).repeat(2, 1) + torch.tensor([[0], [100]], dtype=torch.int32)
    flat = [torch.cat([x.cpu()[0::2], x.cpu()[1::2]]).unsqueeze(2) for x in (k, v)]
    for i in (0, 1, 2, 50, 99):
        out, mag, size, count = O.attention(q[2 * i:2 * i + 2].cpu(), *flat, order, [i + 1, i + 1], None, scale=128 ** -0.5)
        assert ((got[i].cpu().double() - out).abs() <= O.bound(BF, out, mag, size, count, 128)).all()


def test_growing_is_refused_in_a_capture_and_attend_is_not():
    c = fk.PagedKVCache(20, 2, 128, seqs=2)
    g = gen(3)
    k, q = rows(2, g), rows(2, g, 4)
    c.append(k, k)
    want = c.attend(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: c.append(k, k), lambda: c.read(), lambda: c.release(0)):
            with pytest.raises(RuntimeError, match="captured"):
                call()
        got = c.attend(q)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and c.host_lengths == [1, 1]
    c.append(k, k)                                    # the captured attention follows the cache
    want = c.attend(q)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_an_append_after_a_refused_one():
    c = fk.PagedKVCache(20, 2, 128, seqs=2)
    g = gen(4)
    k, v, q = rows(5, g), rows(5, g), rows(5, g, 4)
    for key, value in ((k.float(), v.float()), (k.cpu(), v.cpu()), (k, v.half()), (k.transpose(1, 2).contiguous().transpose(1, 2)[:, :, ::2], v)):
        with pytest.raises(ValueError):
            c.append(key, value, [2, 3])
        assert c.host_lengths == [0, 0] and c.lengths.tolist() == [0, 0] and (c.page_table == -1).all()
    c.append(k, v, [2, 3])
    fresh = fk.PagedKVCache(20, 2, 128, seqs=2)
    fresh.append(k, v, [2, 3])
    assert torch.equal(c.attend(q), fresh.attend(q)) and torch.equal(c.read()[0], k)


@pytest.mark.parametrize("scale", [1e39, -1e39, 2.4e38, float("inf"), float("nan")])
def test_scales_that_fp32_does_not_hold_are_refused(scale):
    c = fk.PagedKVCache(4, 2, 128)
    k, q = rows(1, gen(5)), rows(1, gen(5), 4)
    c.append(k, k)
    with pytest.raises(ValueError, match="finite"):
        c.attend(q, scale=scale)
    assert torch.equal(c.attend(q), c.attend(q, scale=128 ** -0.5))


def test_more_heads_than_a_block_counts_are_refused():
    cache = [torch.zeros(2, 1025, 1, 8, device="cuda", dtype=BF) for _ in range(2)]
    where = (torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda"))
    row = torch.zeros(1, 1025, 8, device="cuda", dtype=BF)
    with pytest.raises(ValueError, match="at most 1024 heads"):
        fk.paged_kv_append(row, row, *cache, *where)
    with pytest.raises(ValueError, match="at most 1024 heads"):
        fk.paged_kv_gather(*cache, *where, None, 1)
    assert (fk.paged_attention(row, *cache, *where) == 0).all()          # the attention takes them
    fit = [t[:, :1024].contiguous() for t in cache]
    ones = torch.ones(1, 1024, 8, device="cuda", dtype=BF)
    fk.paged_kv_append(ones, ones, *fit, *where)
    assert all((t == 1).all() for t in fk.paged_kv_gather(*fit, *where, None, 1)) and (fit[0][1] == 0).all()


def test_expanded_tensors_are_read_and_not_written():
    """Rows, queries and caches that repeat one element's memory are fine to read; as outputs they are refused."""
    g = gen(6)
    cache = [torch.zeros(3, 2, 16, 128, device="cuda", dtype=BF) for _ in range(2)]
    where = (torch.tensor([[2, 0]], dtype=torch.int32, device="cuda"), torch.tensor([4], dtype=torch.int32, device="cuda"), torch.tensor([0, 4], dtype=torch.int32, device="cuda"))
    one = rows(1, g)
    fk.paged_kv_append(one.expand(4, 2, 128), one.expand(4, 2, 128), *cache, *where)
    got = fk.paged_kv_gather(*cache, *where, 4)
    assert torch.equal(got[0], one.expand(4, 2, 128)) and torch.equal(got[1], got[0])
    q = rows(1, g, 4)
    out = fk.paged_attention(q.expand(4, 4, 128), *cache, *where)
    want = one.repeat_interleave(2, dim=1).expand(4, 4, 128)
    assert ((out - want).abs() <= 2.0 ** -7 * want.abs()).all()          # equal values: one rounding of the weights, one of the result
    wide = [t[:, :1].expand(3, 2, 16, 128) for t in cache]
    fk.paged_attention(q.expand(4, 4, 128), *wide, *where)
    empty = torch.zeros(1, 4, 128, device="cuda", dtype=BF)
    for call in (lambda: fk.paged_kv_append(one.expand(4, 2, 128), one.expand(4, 2, 128), *wide, *where),
                 lambda: fk.paged_kv_gather(*cache, *where, 4, out=(empty[:, :2].expand(4, 2, 128), got[1])),
                 lambda: fk.paged_attention(q.expand(4, 4, 128), *cache, *where, out=empty.expand(4, 4, 128))):
        with pytest.raises(ValueError, match="expanded"):
            call()
