"""GPU: a wait of the attention kernels that runs out.  Nothing here traps, faults or spins without a limit: the wait limit is set to
(almost) nothing, the kernels give up their waits at once and end by themselves, what depended on a wait is NaN, and the next call is
right again."""

import pytest
import torch

import fastkernels_b200 as fk
from fastkernels_b200 import _lib
from tests.test_kv_cache_gpu import BF, E4, F16, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [[1, 1, 1], [200, 1, 64], [900]])
@pytest.mark.parametrize("dim,dtype,cache,page", [(256, BF, BF, 16), (128, F16, F16, 12), (256, BF, E4, 16), (128, F16, E4, 32)])
def test_rows_of_a_wait_that_ran_out_are_nan_and_no_other_number_is_wrong(new, dim, dtype, cache, page):
    lib = _lib.load()
    b = Batch(dim + page, new, [900, 400, 700][:len(new)], kv_heads=2, heads=16, dim=dim, page=page, dtype=dtype, cache=cache)
    want = b.attend(max_query=max(new))
    torch.cuda.synchronize()
    try:
        assert lib.fk_set_wait_limit_cycles(1) == 0
        got = b.attend(max_query=max(new))
        torch.cuda.synchronize()
    finally:
        assert lib.fk_set_wait_limit_cycles(0) == 0
    lost = torch.isnan(got)
    assert torch.equal(torch.where(lost, want, got), want)
    if max(new) > 1:                                 # a decode warp's copies may land while its queries are loaded: then it has nothing to wait for
        assert lost.any()
    assert torch.equal(b.attend(max_query=max(new)), want)


@pytest.mark.parametrize("dim,dtype,cache,page", [(256, BF, BF, 16), (128, F16, F16, 12), (256, BF, E4, 16), (64, BF, BF, 64)])
def test_a_limit_below_the_time_of_a_call_stops_nothing_that_moves(dim, dtype, cache, page):
    """100000 clocks, some 50 us, where an item alone takes hundreds: waits that last from one edge of the mask to the next count from
    what moved last."""
    lib = _lib.load()
    g = torch.Generator(device="cuda").manual_seed(dim)
    pages = -(-40000 // page)
    k, v = (torch.randn(pages, 1, page, dim, generator=g, device="cuda").to(cache) for _ in range(2))
    scales = {} if cache != E4 else {name: torch.ones(pages, 1, page, device="cuda") for name in ("key_scale", "value_scale")}
    q = torch.randn(1500, 8, dim, generator=g, device="cuda").to(dtype)
    where = (torch.randperm(pages, generator=g, device="cuda").to(torch.int32).view(1, -1), torch.tensor([40000], dtype=torch.int32, device="cuda"),
             torch.tensor([0, 1500], dtype=torch.int32, device="cuda"))

    def call():
        return fk.paged_attention(q, k, v, *where, max_query=1500, **scales)
    want = call()
    torch.cuda.synchronize()
    try:
        assert lib.fk_set_wait_limit_cycles(100000) == 0
        got = [call() for _ in range(5)]
        torch.cuda.synchronize()
    finally:
        assert lib.fk_set_wait_limit_cycles(0) == 0
    assert torch.isfinite(want).all() and all(torch.equal(x, want) for x in got)


@pytest.mark.parametrize("limit", [50, 400, 1000, 2000])
@pytest.mark.parametrize("dim,kv_heads,group,dtype,cache,page,new", [(256, 2, 8, BF, BF, 16, [700, 1, 300]), (128, 8, 4, F16, F16, 32, [300, 1, 200]), (128, 8, 4, F16, F16, 12, [300, 1, 200]),
                                                                     (128, 8, 4, BF, E4, 16, [300, 1, 200]), (256, 2, 8, BF, BF, 16, [1] * 40), (128, 8, 4, BF, E4, 16, [2] * 20)])
def test_waits_that_run_out_somewhere_on_the_way(dim, kv_heads, group, dtype, cache, page, new, limit):
    """Limits about as long as the waits: some warps give up in the middle of their run.  What is a number is the right one."""
    lib = _lib.load()
    g = torch.Generator().manual_seed(limit)
    lengths = [max(n, int(x)) for n, x in zip(new, torch.randint(700, 3000, (len(new),), generator=g))]
    b = Batch(dim + page, new, lengths, kv_heads=kv_heads, heads=kv_heads * group, dim=dim, page=page, dtype=dtype, cache=cache)
    args = (b.q.cuda(), *b.dev())
    want = fk.paged_attention(*args, max_query=max(new), **b.scales)
    torch.cuda.synchronize()
    try:
        assert lib.fk_set_wait_limit_cycles(limit) == 0
        got = [fk.paged_attention(*args, max_query=max(new), **b.scales) for _ in range(4)]
        torch.cuda.synchronize()
    finally:
        assert lib.fk_set_wait_limit_cycles(0) == 0
    for x in got:
        assert torch.equal(torch.where(torch.isnan(x), want, x), want)
    assert torch.equal(fk.paged_attention(*args, max_query=max(new), **b.scales), want)
