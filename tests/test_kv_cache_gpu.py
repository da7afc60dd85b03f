"""GPU: the paged key/value cache (append, gather) and the attention over it against their definitions in 64 bits."""

import pytest
import torch

import fastkernels_b200 as fk
from tests import paged_oracle as O

pytestmark = pytest.mark.gpu

BF, F16, F32, E4 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def gen(seed):
    return torch.Generator().manual_seed(seed)


class Batch:
    """A ragged batch over a shuffled pool of pages, its tensors on the GPU and copies on the CPU."""

    def __init__(self, seed, new, lengths, *, kv_heads=2, heads=4, dim=64, page=16, dtype=BF, cache=None, nhd=False, spare=3, fill=None):
        g = gen(seed)
        cache = cache or dtype
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g).to(torch.int32)
        self.table = torch.full((len(new), max(need + [1]) + 1), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.new, self.rows, self.dtype, self.cache, self.page = new, starts[-1], dtype, cache, page
        self.starts, self.lengths = torch.tensor(starts, dtype=torch.int32), torch.tensor(lengths, dtype=torch.int32)
        shape = (pages, kv_heads, page, dim)
        k, v = (torch.randn(shape, generator=g) * torch.exp2(2 * torch.rand(*shape[:3], 1, generator=g) - 1) for _ in range(2))
        self.k_scale = self.v_scale = None
        if cache == E4:
            (k, self.k_scale), (v, self.v_scale) = O.quantised(k), O.quantised(v)
            k, v = k.float(), v.float()
        self.k, self.v = k.to(cache), v.to(cache)
        self.q = torch.randn(self.rows, heads, dim, generator=g).to(dtype)
        self.nhd = nhd

    def dev(self):
        def put(t):
            if t is None:
                return None
            if self.nhd and t.ndim >= 3:            # [pages, page_size, kv_heads, ...] in memory
                return t.transpose(1, 2).contiguous().cuda().transpose(1, 2)
            return t.cuda()
        self.dk, self.dv = put(self.k), put(self.v)
        self.scales = {"key_scale": put(self.k_scale), "value_scale": put(self.v_scale)}
        self.where = (self.table.cuda(), self.lengths.cuda(), self.starts.cuda())
        return self.dk, self.dv, *self.where

    def attend(self, **kw):
        return fk.paged_attention(self.q.cuda(), *self.dev(), **self.scales, **kw)

    def check(self, got, *, scale=None, window=0, sinks=0):
        scale = self.q.shape[2] ** -0.5 if scale is None else scale
        out, mag, size, count = O.attention(self.q, self.k, self.v, self.table, self.lengths, self.starts, scale=scale, window=window, sinks=sinks,
                                            k_scale=self.k_scale, v_scale=self.v_scale)
        tol = O.bound(self.dtype, out, mag, size, count, self.q.shape[2])
        err = (got.cpu().double() - out).abs()
        assert torch.isfinite(got).all()
        assert (err <= tol).all(), f"error {err.max():.3e}, {(err / tol).max():.2f} times the bound"
        return out


# ---------------------------------------------------------------------------------------------- append and gather

@pytest.mark.parametrize("dtype,cache", [(BF, BF), (F16, F16), (F32, F32), (BF, E4), (F16, E4), (F32, E4)])
@pytest.mark.parametrize("dim,page,kv_heads,nhd", [(128, 16, 2, False), (256, 16, 1, True), (80, 12, 3, False), (7, 1, 2, True), (1, 5, 1, False), (64, 32, 5, True)])
def test_append_then_gather(dtype, cache, dim, page, kv_heads, nhd):
    b = Batch(dim + page, [3, 0, 1, 18], [40, 9, 1, 18], kv_heads=kv_heads, heads=kv_heads, dim=dim, page=page, dtype=dtype, cache=cache, nhd=nhd)
    dk, dv, table, lengths, starts = b.dev()
    g = gen(5)
    key, value = (torch.randn(b.rows + 2, kv_heads, dim, generator=g) * torch.exp2(20 * torch.rand(b.rows + 2, kv_heads, 1, generator=g) - 10) for _ in range(2))
    key[1] = 0.0
    key, value = key.to(dtype), value.to(dtype)
    fk.paged_kv_append(key.cuda(), value.cuda(), dk, dv, table, lengths, starts, **b.scales)
    for x, before, after, scale_before, scale in ((key, b.k, dk, b.k_scale, b.scales["key_scale"]), (value, b.v, dv, b.v_scale, b.scales["value_scale"])):
        want, want_scale = before.float().double(), None if scale is None else scale_before.clone()
        codes, scales = O.quantised(x) if cache == E4 else (x.double(), None)
        for r, s, p in O.rows_of(b.starts, b.lengths, b.rows):
            pg, rw = O.place(b.table, page, before.shape[0], s, p)
            want[pg, :, rw] = codes[r]
            if scale is not None:
                want_scale[pg, :, rw] = scales[r]
        assert torch.equal(after.cpu().float().double(), want)                    # other rows stay; codes are exact
        if scale is not None:
            assert torch.equal(scale.cpu(), want_scale)
    out_k, out_v = fk.paged_kv_gather(dk, dv, table, lengths, starts, b.rows + 2, dtype=dtype, **b.scales)
    for x, out in ((key, out_k), (value, out_v)):
        assert out.dtype == dtype and (out[b.rows:] == 0).all()
        want = x[:b.rows]
        if cache == E4:
            codes, scales = O.quantised(want)
            want = (codes.float() * scales.unsqueeze(-1)).to(dtype)                 # one product in fp32, one rounding
        assert torch.equal(out[:b.rows].cpu(), want)


def test_append_keeps_codes_half_way_between_two():
    """Quotients that lie exactly half way between two codes go to the even one; others of the same magnitude do not."""
    x = torch.zeros(1, 1, 64)
    x[0, 0, 0] = 448.0
    x[0, 0, 1:17] = torch.tensor([17.0, 19.0, 21.0, 23.0, 25.0, 27.0, 29.0, 31.0, -17.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -11, 433.0, 432.0, 431.0, 416.0])
    for factor in (1.0, 2.0 ** -90, 3.0, 2.0 ** 100):
        b = Batch(1, [1], [1], kv_heads=1, heads=1, dim=64, dtype=F32, cache=E4)
        dk, dv, table, lengths, starts = b.dev()
        y = x * factor
        fk.paged_kv_append(y.cuda(), y.cuda(), dk, dv, table, lengths, starts, **b.scales)
        codes, scales = O.quantised(y)
        pg, rw = O.place(b.table, 16, b.k.shape[0], 0, 0)
        assert torch.equal(dk[pg, 0, rw].cpu().float().double(), codes[0, 0]) and torch.equal(b.scales["key_scale"][pg, 0, rw].cpu(), scales[0, 0])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_row_that_is_not_finite_reads_back_as_nan_and_no_other_does(bad):
    b = Batch(2, [4], [4], kv_heads=2, heads=2, dim=128, cache=E4)
    dk, dv, table, lengths, starts = b.dev()
    key = torch.randn(4, 2, 128, generator=gen(3)).to(BF)
    key[2, 1, 77] = bad
    fk.paged_kv_append(key.cuda(), key.cuda(), dk, dv, table, lengths, starts, **b.scales)
    out, _ = fk.paged_kv_gather(dk, dv, table, lengths, starts, 4, **b.scales)
    nan = torch.isnan(out).all(-1).cpu()
    assert nan[2, 1] and nan.sum() == 1 and torch.isnan(out).sum() == 128


def test_gather_into_given_tensors_keeps_the_rows_behind_the_last_sequence():
    b = Batch(4, [2, 3], [20, 3], kv_heads=3, heads=3, dim=64)
    dk, dv, table, lengths, starts = b.dev()
    big = torch.full((9, 3, 2, 64), 7.0, device="cuda", dtype=BF)
    out = (big[:, :, 0], big[:, :, 1])
    fk.paged_kv_gather(dk, dv, table, lengths, starts, 9, out=out)
    assert (big[5:] == 7).all()
    for r, s, p in O.rows_of(b.starts, b.lengths, 5):
        pg, rw = O.place(b.table, 16, b.k.shape[0], s, p)
        assert torch.equal(out[0][r].cpu(), b.k[pg, :, rw]) and torch.equal(out[1][r].cpu(), b.v[pg, :, rw])


# ---------------------------------------------------------------------------------------------- attention

SHAPES = [  # new, lengths
    ([1], [1]), ([1], [2]), ([1, 1, 1], [17, 1, 300]), ([1] * 5, [64, 65, 63, 128, 129]), ([5], [5]), ([3, 1, 0, 40], [33, 70, 12, 41]), ([130], [200]),
]


@pytest.mark.parametrize("new,lengths", SHAPES)
@pytest.mark.parametrize("dim,kv_heads,group,page", [(256, 2, 8, 16), (128, 2, 4, 32), (64, 1, 7, 8), (80, 2, 3, 12), (128, 1, 16, 1), (33, 3, 1, 5)])
@pytest.mark.parametrize("dtype,cache", [(BF, BF), (F16, F16), (BF, E4), (F16, E4), (F32, F32), (F32, E4)])
def test_attention(new, lengths, dim, kv_heads, group, page, dtype, cache):
    b = Batch(len(new) + dim, new, lengths, kv_heads=kv_heads, heads=kv_heads * group, dim=dim, page=page, dtype=dtype, cache=cache)
    got = b.attend(max_query=max(new))
    assert got.dtype == dtype
    b.check(got)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (16, 4), (17, 16), (50, 0), (50, 40), (1000, 4)])
@pytest.mark.parametrize("new,lengths", [([1, 1, 1], [300, 20, 1]), ([70, 1, 9], [200, 129, 9])])
@pytest.mark.parametrize("dim,group,dtype,cache", [(256, 8, BF, BF), (128, 4, F16, E4), (64, 2, BF, E4), (48, 2, F32, F32)])
def test_attention_window_and_sinks(window, sinks, new, lengths, dim, group, dtype, cache):
    b = Batch(window + sinks, new, lengths, kv_heads=2, heads=2 * group, dim=dim, dtype=dtype, cache=cache)
    b.check(b.attend(window=window, sinks=sinks), window=window, sinks=sinks)


@pytest.mark.parametrize("dtype,cache", [(BF, BF), (F16, F16), (BF, E4), (F32, F32)])
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_attention_scale(dtype, cache, scale):
    b = Batch(7, [4, 1], [90, 33], dim=128, heads=8, dtype=dtype, cache=cache)
    b.check(b.attend(scale=scale), scale=scale)


@pytest.mark.parametrize("dtype,cache", [(BF, BF), (F16, E4), (F32, F32)])
@pytest.mark.parametrize("dim", [64, 128, 256, 40])
def test_attention_strided_and_shifted_tensors(dtype, cache, dim):
    """Cache rows before heads in memory; queries cut out of a wider tensor, shifted by one element; output rows with gaps."""
    b = Batch(11, [1, 20, 3], [50, 20, 77], kv_heads=2, heads=8, dim=dim, dtype=dtype, cache=cache, nhd=True)
    args = b.dev()
    wide = torch.zeros(b.rows, 8, 2 * dim + 3, dtype=dtype, device="cuda")
    wide[:, :, 1:dim + 1] = b.q.cuda()
    out = torch.full((b.rows, 8, dim + 5), 3.0, dtype=dtype, device="cuda")
    got = fk.paged_attention(wide[:, :, 1:dim + 1], *args, out=out[:, :, :dim], **b.scales)
    assert (out[:, :, dim:] == 3).all()
    b.check(got)
    # a cache whose rows start on odd elements
    one = [torch.zeros(*t.shape[:3], dim + 1, dtype=torch.uint8, device="cuda").view(t.dtype) if t.dtype == E4 else
           torch.zeros(*t.shape[:3], dim + 1, dtype=t.dtype, device="cuda") for t in args[:2]]
    for x, t in zip(one, args):
        (x.view(torch.uint8) if t.dtype == E4 else x)[..., 1:] = t.view(torch.uint8) if t.dtype == E4 else t
    b.check(fk.paged_attention(b.q.cuda(), one[0][..., 1:], one[1][..., 1:], *args[2:], **b.scales))


@pytest.mark.parametrize("dtype,cache", [(BF, BF), (F16, F16), (F16, E4), (F32, F32)])
@pytest.mark.parametrize("dim,new,window,sinks", [(256, [1, 1], 0, 0), (128, [1, 1], 20, 2), (128, [40, 3], 0, 0), (256, [40, 2], 20, 2), (64, [40, 2], 7, 1)])
def test_masked_places_have_no_influence(dtype, cache, dim, new, window, sinks):
    """Not-a-number and infinities in rows of the pages that no row sees, and in later tokens of the same chunk."""
    b = Batch(21, new, [90, 47], kv_heads=2, heads=8, dim=dim, dtype=dtype, cache=cache)
    clean = b.attend(window=window, sinks=sinks, max_query=max(new))
    b.check(clean, window=window, sinks=sinks)
    used = torch.zeros(b.k.shape[0], b.page, dtype=torch.bool)
    for _, s, p in O.rows_of(b.starts, b.lengths, b.rows):
        for j in range(p + 1):
            if not window or j > p - window or j < sinks:
                pg, rw = O.place(b.table, b.page, b.k.shape[0], s, j)
                used[pg, rw] = True
    poison = torch.tensor([float("nan"), float("inf"), float("-inf")])
    pick = torch.randint(0, 3, (int((~used).sum()),), generator=gen(1))
    for t, scale in ((b.k, b.k_scale), (b.v, b.v_scale)):
        if scale is None:
            t.transpose(1, 2)[~used] = poison[pick][:, None, None].to(dtype).expand(-1, 2, dim)
        else:
            scale.transpose(1, 2)[~used] = poison[pick][:, None].expand(-1, 2)
    again = b.attend(window=window, sinks=sinks, max_query=max(new))
    assert torch.equal(clean, again)
    # the last token of the longest chunk: only its own row may notice
    if max(new) > 1:
        s = new.index(max(new))
        pg, rw = O.place(b.table, b.page, b.k.shape[0], s, int(b.lengths[s]) - 1)
        for bad in (float("nan"), float("inf")):
            (b.v if b.v_scale is None else b.v_scale)[pg, :, rw] = bad
            got = b.attend(window=window, sinks=sinks, max_query=max(new))
            mine = int(b.starts[s + 1]) - 1
            others = [r for r in range(b.rows) if r != mine]
            assert not torch.isfinite(got[mine]).any()
            out, mag, size, count = O.attention(b.q[:mine], b.k, b.v, b.table, b.lengths, b.starts, scale=dim ** -0.5, window=window, sinks=sinks,
                                                k_scale=b.k_scale, v_scale=b.v_scale)
            err = (got[:mine].cpu().double() - out).abs()
            assert torch.isfinite(got[others]).all() and (err <= O.bound(dtype, out, mag, size, count, dim)).all()


def test_rows_that_see_nothing_are_zero_and_rows_behind_the_last_sequence_stay():
    for dim, cache, max_query in ((256, BF, 1), (128, E4, 40), (80, BF, 0), (64, BF, 3)):
        b = Batch(31, [2, 1, 3], [2, 0, 1], kv_heads=1, heads=4, dim=dim, cache=cache)          # lengths shorter than the rows
        args = b.dev()
        q = torch.randn(10, 4, dim, generator=gen(2)).to(BF)
        out = torch.full((10, 4, dim), 5.0, device="cuda", dtype=BF)
        fk.paged_attention(q.cuda(), *args, out=out, max_query=max_query, **b.scales)
        assert (out[6:] == 5).all() and (out[2] == 0).all() and (out[3:5] == 0).all() and (out[5] != 0).any()
        fresh = fk.paged_attention(q.cuda(), *args, max_query=max_query, **b.scales)
        assert torch.equal(fresh[:6], out[:6]) and (fresh[6:] == 0).all()
        one = fk.paged_attention(q.cuda()[:2], *args[:4], **b.scales)                            # no starts: one token per sequence
        assert torch.isfinite(one).all() and (one[1] == 0).all()


@pytest.mark.parametrize("dim,cache,dtype", [(256, BF, BF), (128, E4, F16), (80, F32, F32)])
@pytest.mark.parametrize("max_query", [0, 1, 100])
def test_bad_page_tables_lengths_and_starts_stay_in_bounds(dim, cache, dtype, max_query):
    """Pages outside the cache, lengths beyond the table, starts out of order or beyond the rows: skipped, zero, not visible."""
    b = Batch(41, [1, 30, 1], [60, 90, 20], kv_heads=2, heads=4, dim=dim, dtype=dtype, cache=cache)
    b.table[0, 1], b.table[1, 0], b.table[1, 3], b.table[2, 1] = -1, 2 ** 31 - 1, -2 ** 31, b.k.shape[0]
    b.check(b.attend(max_query=max_query))
    key = torch.ones(b.rows, 2, dim, dtype=dtype)
    before = b.k.float()
    dk, dv, table, lengths, starts = b.dev()
    fk.paged_kv_append(key.cuda(), key.cuda(), dk, dv, table, lengths, starts, **b.scales)
    out, _ = fk.paged_kv_gather(dk, dv, table, lengths, starts, b.rows, dtype=dtype, **b.scales)
    for r, s, p in O.rows_of(b.starts, b.lengths, b.rows):
        at = O.place(b.table, 16, b.k.shape[0], s, p)
        want = 0.0 if at is None else 1.0
        assert (out[r].float() == want).all()
        if at is not None:
            before[at[0], :, at[1]] = 448.0 if cache == E4 else 1.0
    assert torch.equal(dk.cpu().float(), before)
    for lens, sts in (([2 ** 31 - 1, 0, 20], [0, 1, 31, 32]), ([-5, -2 ** 31, 500], [0, 1, 31, 32]), ([60, 90, 20], [0, 40, 2, 32]), ([60, 90, 20], [-7, 1, 500, 900]),
                      ([60, 90, 20], [5, 5, 5, 5]), ([60, 90, 20], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 0])):
        ls, st = torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(sts, dtype=torch.int32).cuda()
        got = fk.paged_attention(b.q.cuda(), dk, dv, table, ls, st, max_query=max_query, **b.scales)
        torch.cuda.synchronize()
        assert torch.isfinite(got).all()
        fk.paged_kv_append(key.cuda(), key.cuda(), dk, dv, table, ls, st, **b.scales)
        fk.paged_kv_gather(dk, dv, table, ls, st, b.rows, dtype=dtype, **b.scales)
        torch.cuda.synchronize()


@pytest.mark.parametrize("new", [1, 24])
@pytest.mark.parametrize("dtype,cache", [(BF, E4), (BF, BF)])
def test_offsets_beyond_32_bits(new, dtype, cache):
    """A cache of more than 2^32 elements (over 2^31 pages x heads x rows x dim), of which the last pages are used."""
    dim, page, heads = 256, 16, 2
    pages = 2 ** 32 // (heads * page * dim) + 600
    small = Batch(51, [new], [500], kv_heads=heads, heads=16, dim=dim, page=page, dtype=dtype, cache=cache)
    n = small.k.shape[0]
    big = []
    for t in (small.k, small.v):
        x = torch.empty(pages, heads, page, dim, dtype=torch.uint8 if cache == E4 else dtype, device="cuda")
        x[pages - n:] = (t.view(torch.uint8) if cache == E4 else t).cuda()
        big.append(x.view(cache))
    scales = {}
    if cache == E4:
        for name, t in (("key_scale", small.k_scale), ("value_scale", small.v_scale)):
            scales[name] = torch.empty(pages, heads, page, device="cuda")
            scales[name][pages - n:] = t.cuda()
    table = torch.where(small.table >= 0, small.table + (pages - n), small.table).cuda()
    lengths, starts = small.lengths.cuda(), small.starts.cuda()
    small.check(fk.paged_attention(small.q.cuda(), *big, table, lengths, starts, max_query=new, **scales))
    key = torch.randn(new, heads, dim, generator=gen(1)).to(dtype).cuda()
    fk.paged_kv_append(key, key, *big, table, lengths, starts, **scales)
    out, _ = fk.paged_kv_gather(*big, table, lengths, starts, new, **scales)
    codes, s = O.quantised(key.cpu()) if cache == E4 else (None, None)
    assert torch.equal(out.cpu(), (codes.float() * s.unsqueeze(-1)).to(dtype) if cache == E4 else key.cpu())


@pytest.mark.parametrize("new,lengths", [([1] * 7, [900, 30, 1, 64, 500, 77, 128]), ([40, 1, 200], [700, 300, 200])])
@pytest.mark.parametrize("dim,cache", [(256, BF), (128, E4), (80, BF)])
def test_the_same_call_twice_gives_the_same_bits(new, lengths, dim, cache):
    b = Batch(61, new, lengths, kv_heads=2, heads=8, dim=dim, cache=cache)
    first = b.attend(max_query=max(new))
    for _ in range(5):
        assert torch.equal(first, b.attend(max_query=max(new)))


def test_captured_calls_follow_the_lengths_and_do_not_share_scratch():
    """Append, attention and read-back in a graph, replayed with grown sequences; two such graphs replayed at once on two
    streams, with an eager call between, give what they give alone."""
    graphs = []
    for seed in (71, 72):
        b = Batch(seed, [1, 1, 6], [400, 90, 300], kv_heads=2, heads=16, dim=256)
        dk, dv, table, lengths, starts = b.dev()
        q = b.q.cuda()
        kv = torch.randn(b.rows, 2, 256, generator=gen(seed)).to(BF).cuda()

        def call(q=q, kv=kv, dk=dk, dv=dv, table=table, lengths=lengths, starts=starts):
            fk.paged_kv_append(kv, kv, dk, dv, table, lengths, starts)
            return fk.paged_attention(q, dk, dv, table, lengths, starts, max_query=6), fk.paged_kv_gather(dk, dv, table, lengths, starts, 8)[0]
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = call()
        graphs.append((g, res, call, lengths))
    for step in range(3):
        alone = []
        for g, res, call, lengths in graphs:
            lengths -= 3
            g.replay()
            torch.cuda.synchronize()
            alone.append([t.clone() for t in res])
            for a, e in zip(alone[-1], call()):
                assert torch.equal(a, e)
        for _ in range(10):
            streams = [torch.cuda.Stream() for _ in graphs]
            for (g, *_), s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            eager = graphs[0][2]()[0] if step == 0 else None
            torch.cuda.synchronize()
            for (g, res, *_), a in zip(graphs, alone):
                assert all(torch.equal(x, y) for x, y in zip(res, a))
            if eager is not None:
                assert torch.equal(eager, alone[0][0])


def test_calls_run_on_the_current_stream_and_on_the_tensors_device():
    b = Batch(81, [1, 5], [100, 200], kv_heads=2, heads=8, dim=128)
    want = b.attend()
    s = torch.cuda.Stream()
    args, q = b.dev(), b.q.cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        busy = torch.randn(4096, 4096, device="cuda")
        for _ in range(5):
            busy = busy @ busy
        q2 = q + 0 * busy[:1, :1].nan_to_num(0, 0, 0).to(BF)
        got = fk.paged_attention(q2, *args)
    s.synchronize()
    assert torch.equal(got, want)
    if torch.cuda.device_count() > 1:
        moved = [t.to("cuda:1") for t in (q, *args)]
        assert torch.equal(fk.paged_attention(*moved).cpu(), want.cpu())


@pytest.mark.parametrize("cache", [BF, E4])
def test_a_cache_grows_from_prompt_to_decode(cache):
    """Append, attention and read-back together as a model uses them: prompts of three sequences, then single tokens, one
    sequence released and started anew."""
    c = fk.PagedKVCache(40, 2, 128, seqs=3, dtype=cache)
    g = gen(91)
    held = [[[], []] for _ in range(3)]
    for step, new in enumerate([[33, 5, 0], [1, 1, 1], [1, 0, 17], [1, 1, 1], [2, 3, 1]]):
        if step == 3:
            c.release(0)
            held[0] = [[], []]
        rows = sum(new)
        k, v = (torch.randn(rows, 2, 128, generator=g).to(BF) for _ in range(2))
        q = torch.randn(rows, 8, 128, generator=g).to(BF)
        c.append(k.cuda(), v.cuda(), new)
        got = c.attend(q.cuda(), window=40 if step == 4 else 0, sinks=2 if step == 4 else 0)
        at = 0
        for s, n in enumerate(new):
            for i in range(n):
                held[s][0].append(k[at + i])
                held[s][1].append(v[at + i])
            at += n
        assert c.host_lengths == [len(h[0]) for h in held]
        flat = [torch.stack([t for h in held for t in h[i]]) for i in (0, 1)]
        stored = c.read(dtype=F32 if cache == E4 else None)
        want = []
        for x, y in zip(flat, stored):
            if cache == E4:
                codes, scales = O.quantised(x)
                x = codes.float() * scales.unsqueeze(-1)
            assert torch.equal(y.cpu(), x)
            want.append(x)
        # the oracle over one page per token
        table = torch.full((3, max(c.host_lengths) + 1), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(c.host_lengths):
            table[s, :n] = torch.arange(at, at + n)
            at += n
        starts = torch.tensor([0, new[0], new[0] + new[1], rows])
        out, mag, size, count = O.attention(q, want[0].unsqueeze(2), want[1].unsqueeze(2), table, c.host_lengths, starts, scale=128 ** -0.5,
                                            window=40 if step == 4 else 0, sinks=2 if step == 4 else 0)
        assert ((got.cpu().double() - out).abs() <= O.bound(BF, out, mag, size, count, 128)).all()
    with pytest.raises(ValueError, match="no pages left"):
        c.append(torch.zeros(1000, 2, 128, device="cuda", dtype=BF), torch.zeros(1000, 2, 128, device="cuda", dtype=BF), [1000, 0, 0])


def test_refusals():
    b = Batch(1, [1, 3], [20, 30], kv_heads=2, heads=4, dim=64)
    dk, dv, table, lengths, starts = b.dev()
    q = b.q.cuda()
    e4 = torch.zeros(dk.shape, dtype=torch.uint8, device="cuda").view(E4)
    scale = torch.ones(dk.shape[:3], device="cuda")
    att = fk.paged_attention

    def refused(match, call):
        with pytest.raises(ValueError, match=match):
            call()

    refused("CUDA", lambda: att(b.q, b.k, b.v, b.table, b.lengths, b.starts))
    refused("same shape", lambda: att(q, dk, dv[:-1], table, lengths, starts))
    refused("dtype and device", lambda: att(q, dk, dv.half(), table, lengths, starts))
    refused("float32, bfloat16", lambda: att(q, dk.int(), dv.int(), table, lengths, starts))
    refused("last dimension", lambda: att(q, dk.transpose(2, 3).contiguous().transpose(2, 3), dv, table, lengths, starts))
    refused("page_table must be int32", lambda: att(q, dk, dv, table.long(), lengths, starts))
    refused("lengths must be int32", lambda: att(q, dk, dv, table, lengths[:1], starts))
    refused("query_starts must be int32", lambda: att(q, dk, dv, table, lengths, starts[:-1]))
    refused("on cuda", lambda: att(q, dk, dv, table, lengths.cpu(), starts))
    refused("key_scale is required", lambda: att(q, e4, e4, table, lengths, starts))
    refused("value_scale must be float32", lambda: att(q, e4, e4, table, lengths, starts, key_scale=scale, value_scale=scale.half()))
    refused("belong to a float8", lambda: att(q, dk, dv, table, lengths, starts, key_scale=scale, value_scale=scale))
    refused("multiple of the cache's kv_heads", lambda: att(q[:, :3], dk, dv, table, lengths, starts))
    refused("must have shape", lambda: att(q[:, :, :32], dk, dv, table, lengths, starts))
    refused("cache's dtype", lambda: att(q.half(), dk, dv, table, lengths, starts))
    refused("more rows than there are sequences", lambda: att(q, dk, dv, table, lengths))
    refused("must not be negative", lambda: att(q, dk, dv, table, lengths, starts, window=-1))
    refused("sinks need a window", lambda: att(q, dk, dv, table, lengths, starts, sinks=4))
    refused("finite", lambda: att(q, dk, dv, table, lengths, starts, scale=float("nan")))
    refused("overlap", lambda: att(q, dk, dv, table, lengths, starts, out=q))
    refused("query's dtype|cache's dtype", lambda: att(q, dk, dv, table, lengths, starts, out=q.float()))
    refused("between 1 and 256", lambda: att(torch.zeros(4, 4, 260, device="cuda"), *(torch.zeros(4, 2, 16, 260, device="cuda") for _ in range(2)), table, lengths, starts))
    key = torch.zeros(4, 2, 64, device="cuda", dtype=BF)
    refused("same dtype", lambda: fk.paged_kv_append(key, key.half(), e4, e4, table, lengths, starts, key_scale=scale, value_scale=scale))
    refused("must have shape", lambda: fk.paged_kv_append(key, key[:3], dk, dv, table, lengths, starts))
    refused("must not be negative", lambda: fk.paged_kv_gather(dk, dv, table, lengths, starts, -1))
    refused("overlap", lambda: fk.paged_kv_gather(dk, dv, table, lengths, starts, 4, out=(key, key)))
    refused("dtype", lambda: fk.paged_kv_gather(dk, dv, table, lengths, starts, 4, dtype=F16))
    assert att(q[:0], dk, dv, table, lengths, starts).shape == (0, 4, 64)
    assert fk.paged_kv_gather(dk, dv, table, lengths, starts, 0)[0].shape == (0, 2, 64)
    fk.paged_kv_append(key[:0], key[:0], dk, dv, table, lengths, starts)
    none = (table[:0], lengths[:0], starts[:1])
    assert (att(q, dk, dv, *none) == 0).all() and (fk.paged_kv_gather(dk, dv, *none, 4)[0] == 0).all()


@pytest.mark.parametrize("new,lengths,window,sinks", [([2048], [2048], 0, 0), ([700], [9000], 0, 0), ([1500], [6000], 1024, 4), ([1, 900, 1, 1, 333, 2, 64, 1], [4100, 3000, 999, 2500, 3333, 1800, 64, 4000], 0, 0),
                                                      ([1, 900, 1, 1, 333, 2, 64, 1], [4100, 3000, 999, 2500, 3333, 1800, 64, 4000], 500, 70)])
@pytest.mark.parametrize("dim,kv_heads,group,dtype,cache,page", [(256, 2, 8, BF, BF, 16), (128, 8, 4, F16, F16, 32), (128, 2, 4, BF, BF, 12), (256, 1, 8, BF, E4, 16), (64, 4, 2, F16, E4, 64), (128, 1, 7, BF, BF, 8)])
def test_long_chunks(new, lengths, window, sinks, dim, kv_heads, group, dtype, cache, page):
    """Many key tiles per item and many items per worker: every ring, barrier phase and joined part goes round several times.
    Against the definition in 64 bits on the GPU, and twice with the same bits."""
    g = torch.Generator(device="cuda").manual_seed(sum(lengths) + dim)
    need = [-(-n // page) for n in lengths]
    pages, starts = sum(need) + 2, [0]
    for n in new:
        starts.append(starts[-1] + n)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(new), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    shape = (pages, kv_heads, page, dim)
    k, v = (torch.randn(shape, generator=g, device="cuda") * torch.exp2(4 * torch.rand(*shape[:3], 1, generator=g, device="cuda") - 2) for _ in range(2))
    scales = {}
    if cache == E4:
        for name, x in (("key_scale", k), ("value_scale", v)):
            scales[name] = x.abs().amax(-1) / 448
        k, v = (x / scales[n].unsqueeze(-1) for n, x in (("key_scale", k), ("value_scale", v)))
    k, v = k.to(cache), v.to(cache)
    q = torch.randn(starts[-1], kv_heads * group, dim, generator=g, device="cuda").to(dtype)
    args = (q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.tensor(starts, dtype=torch.int32, device="cuda"))
    got = fk.paged_attention(*args, window=window, sinks=sinks, max_query=max(new), **scales)
    for _ in range(3):
        assert torch.equal(got, fk.paged_attention(*args, window=window, sinks=sinks, max_query=max(new), **scales))
    values = []
    for x, name in ((k, "key_scale"), (v, "value_scale")):
        x = x.float()
        values.append(x * scales[name].unsqueeze(-1) if scales else x)
    for s, (n, length) in enumerate(zip(new, lengths)):
        kk, vv = (x[table[s, :need[s]].long()].transpose(1, 2).reshape(-1, kv_heads, dim)[:length].double() for x in values)
        pos, j = torch.arange(length - n, length, device="cuda").view(n, 1), torch.arange(length, device="cuda")
        seen = (j <= pos) & ((j > pos - window) | (j < sinks)) if window else j <= pos
        for a in range(kv_heads * group):
            x, h = q[starts[s]:starts[s + 1], a].double(), a // group
            w = torch.softmax((x @ kk[:, h].T * dim ** -0.5).masked_fill(~seen, float("-inf")), -1)
            out, mag = w @ vv[:, h], w @ vv[:, h].abs()
            size = (x.abs() @ kk[:, h].abs().T * dim ** -0.5).amax(-1)
            err = (got[starts[s]:starts[s + 1], a].double() - out).abs()
            tol = O.bound(dtype, out, mag, size, seen.sum(-1).double(), dim)
            assert (err <= tol).all(), f"sequence {s} head {a}: {(err / tol).max():.2f} times the bound"


@pytest.mark.parametrize("page", [2, 8, 16, 24, 48, 64, 80, 128, 256])
@pytest.mark.parametrize("dtype,cache,dim", [(BF, BF, 256), (F16, E4, 128), (F16, F16, 64)])
@pytest.mark.parametrize("new", [[1, 1, 1], [70, 1, 300]])
def test_attention_page_sizes(page, dtype, cache, dim, new):
    """Pages smaller and larger than a tile of keys, with and without tensor copies, ending inside of tiles."""
    b = Batch(page, new, [517, 129, 300], kv_heads=2, heads=8, dim=dim, page=page, dtype=dtype, cache=cache)
    b.check(b.attend(max_query=max(new)))
    b.check(b.attend(max_query=max(new), window=100, sinks=3), window=100, sinks=3)


def test_calls_on_two_streams_at_once():
    """Decode and chunk calls of both cache types issued on two streams without waiting give what they give alone."""
    batches = [Batch(s, new, [900, 400, 700], kv_heads=2, heads=16, dim=256, cache=cache) for s, (new, cache) in
               enumerate([([1, 1, 1], BF), ([200, 1, 64], BF), ([1, 1, 1], E4), ([200, 1, 64], E4)])]
    args = [(b.q.cuda(), *b.dev()) for b in batches]

    def call(i):
        return fk.paged_attention(*args[i], max_query=max(batches[i].new), **batches[i].scales)
    alone = [call(i) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for turn in range(10):
        for i in range(4):
            with torch.cuda.stream(streams[(i + turn) % 2]):
                got.append((i, call(i)))
    torch.cuda.synchronize()
    assert all(torch.equal(alone[i], x) for i, x in got)
