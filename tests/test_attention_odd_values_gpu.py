"""GPU: values that are not finite.  A row that sees one gets what the formula gives; one that does not is not touched, whoever shares
its tile; neither costs more than the pass over the keys."""

import pytest
import torch

import fastkernels_b200 as fk
from tests import paged_oracle as O
from tests.test_kv_cache_gpu import BF, E4, F16, Batch

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def spot(b, seq, pos):
    return O.place(b.table, b.page, b.k.shape[0], seq, pos)


def check_patterns(b, got, **kw):
    """Infinities and NaN where the formula has them, everything else within the bound."""
    out, mag, size, count = O.attention(b.q, b.k, b.v, b.table, b.lengths, b.starts, scale=b.q.shape[2] ** -0.5, k_scale=b.k_scale, v_scale=b.v_scale, **kw)
    got = got.cpu().double()
    odd = ~torch.isfinite(out)
    assert odd.any() and not odd.all()
    assert torch.equal(torch.isnan(got), torch.isnan(out))
    assert torch.equal(got[odd & ~torch.isnan(out)], out[odd & ~torch.isnan(out)])
    tol = O.bound(b.dtype, out, mag, size, count, b.q.shape[2])
    assert ((got - out).abs()[~odd] <= tol[~odd]).all()


@pytest.mark.parametrize("dim,kv_heads,group,dtype,cache,page", [(256, 2, 8, BF, BF, 16), (128, 8, 4, F16, F16, 12), (128, 4, 4, F16, F16, 32), (128, 8, 4, BF, E4, 16), (64, 2, 2, BF, BF, 16)])
@pytest.mark.parametrize("new,lengths", [([40] * 8, [100, 128, 90, 60, 100, 128, 200, 40]), ([70, 1, 130], [300, 90, 140]), ([2, 2, 2], [300, 90, 31])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2)])
def test_rows_see_what_is_not_finite_only_where_they_may(dim, kv_heads, group, dtype, cache, page, new, lengths, window, sinks):
    """NaN, infinities of both signs and pairs of them in single columns: early, behind the window, within the chunk and at its end."""
    b = Batch(dim + len(new), new, lengths, kv_heads=kv_heads, heads=kv_heads * group, dim=dim, dtype=dtype, cache=cache, page=page)
    for s, (n, length) in enumerate(zip(new, lengths)):
        bads = [(length - 1, 3, NAN), (length - 1, 5, INF), (max(0, length - n - 8), 5, -INF), (length - n // 2 - 1, 7, NAN), (max(0, length - 25), 9, INF), (0, 3, INF), (1, 11, -INF)]
        for pos, column, bad in bads:
            if s % 2 and bad != bad:
                continue
            pg, rw = spot(b, s, pos)
            b.v[pg, s % kv_heads, rw, column] = NAN if cache == E4 else bad       # codes hold no infinities
    check_patterns(b, b.attend(max_query=max(new), window=window, sinks=sinks), window=window, sinks=sinks)


@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("cache", [BF, E4])
def test_an_early_value_that_is_not_finite_costs_no_second_pass(bad, cache):
    """One such row at the start of a long context: every row of the chunk sees it, clean sequences of the call stay as they are, and the call takes
    about the time that it takes without it."""
    g = torch.Generator(device="cuda").manual_seed(5)
    new, lengths, heads, dim, page = [512, 64, 1], [16384, 3000, 5000], 16, 256, 16
    need = [-(-n // page) for n in lengths]
    table = torch.full((3, max(need)), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = torch.arange(at, at + n)
        at += n
    k, v = (torch.randn(at, 2, page, dim, generator=g, device="cuda").to(BF) for _ in range(2))
    scales = {}
    if cache == E4:
        k, v = k.to(E4), v.to(E4)
        scales = {name: torch.ones(at, 2, page, device="cuda") for name in ("key_scale", "value_scale")}
    q = torch.randn(sum(new), heads, dim, generator=g, device="cuda").to(BF)
    where = (table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.tensor([0, 512, 576, 577], dtype=torch.int32, device="cuda"))

    def timed():
        out = [fk.paged_attention(q, k, v, *where, max_query=512, **scales) for _ in range(3)][-1]
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(3):
            fk.paged_attention(q, k, v, *where, max_query=512, **scales)
        b.record()
        torch.cuda.synchronize()
        return out, a.elapsed_time(b) / 3
    clean, before = timed()
    if cache == E4:
        scales["value_scale"][0, :, 0] = bad
    else:
        v[0, :, 0] = bad
    got, after = timed()
    assert not torch.isfinite(got[:512]).any() and torch.equal(got[512:], clean[512:])
    # the rows of a pass over 16384 keys by one warp each, eight to a warp, would take tens of milliseconds
    assert after <= 2 * before + 1.0, (before, after)


@pytest.mark.parametrize("dim,kv_heads,group,dtype,cache,page,new,length", [(128, 8, 4, F16, F16, 32, [40] * 16, 520), (256, 4, 8, BF, BF, 16, [20] * 32, 400), (128, 8, 4, BF, E4, 16, [70, 1, 40] * 8, 520),
                                                                            (128, 8, 4, F16, F16, 12, [70, 1, 40] * 8, 520), (128, 8, 4, BF, BF, 16, [3] * 64, 700)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 2), (9, 0)])
def test_items_of_several_tiles_in_a_row(dim, kv_heads, group, dtype, cache, page, new, length, window, sinks):
    """Whole items among what a pair of SMs (or a warp) walks, next to items in parts: expected infinities and NaN are counted, the rest is
    the definition in 64 bits without them."""
    b = Batch(dim + len(new), new, [length] * len(new), kv_heads=kv_heads, heads=kv_heads * group, dim=dim, dtype=dtype, cache=cache, page=page)
    for s, n in enumerate(new):
        for pos, column, bad in [(length - 1, 3, NAN), (length - 1, 5, INF), (length - n - 8, 5, -INF), (length - n // 2 - 1, 7, INF), (length - 30, 9, NAN), (0, 3, INF), (1, 11, -INF), (200, 13, NAN)]:
            if s % 3 or bad == bad:
                pg, rw = spot(b, s, pos)
                b.v[pg, s % kv_heads, rw, column] = NAN if cache == E4 else bad
    got = b.attend(max_query=max(new), window=window, sinks=sinks)
    clean = 0
    for s, n in enumerate(new):
        a, at = int(b.starts[s]), torch.arange(length)
        pg, rw = b.table[s, at // page].long(), at % page
        k, v = b.k.float()[pg, :, rw].double(), b.v.float()[pg, :, rw].double()
        if cache == E4:
            k, v = k * b.k_scale[pg, :, rw].double().unsqueeze(-1), v * b.v_scale[pg, :, rw].double().unsqueeze(-1)
        q, k, v, at = b.q[a:a + n].cuda().double(), k.cuda().repeat_interleave(group, 1), v.cuda().repeat_interleave(group, 1), at.cuda()
        pos = torch.arange(length - n, length, device="cuda").view(-1, 1)
        seen = (at <= pos) & ((at > pos - window) | (at < sinks)) if window else at <= pos
        nans, ups, downs = (torch.einsum("rj,jhd->rhd", seen.double(), x.double()) > 0 for x in (v.isnan(), v == INF, v == -INF))
        nans = nans | (ups & downs)
        flat = v.nan_to_num(0.0, 0.0, 0.0)
        w = torch.softmax((torch.einsum("rhd,jhd->rhj", q, k) * dim ** -0.5).masked_fill(~seen.unsqueeze(1), -INF), -1)
        out, mag = torch.einsum("rhj,jhd->rhd", w, flat), torch.einsum("rhj,jhd->rhd", w, flat.abs())
        size = (torch.einsum("rhd,jhd->rhj", q.abs(), k.abs()) * dim ** -0.5).masked_fill(~seen.unsqueeze(1), 0.0).amax(-1)
        mine = got[a:a + n].double()
        assert torch.equal(mine.isnan(), nans) and torch.equal(mine == INF, ups & ~nans) and torch.equal(mine == -INF, downs & ~nans)
        fine = ~(nans | ups | downs)
        tol = O.bound(dtype, out, mag, size, seen.sum(-1).double().view(-1, 1).expand_as(size), dim)
        assert ((mine - out).abs()[fine] <= tol[fine]).all()
        clean += int((~fine).sum() == 0)
    assert clean < len(new)
