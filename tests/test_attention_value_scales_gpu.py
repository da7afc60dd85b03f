"""GPU: 8-bit caches whose values differ in magnitude by far more than 16 bits hold.  A key that a row does not see, or that has no
weight in it, takes nothing from the others, however large its value is."""

import pytest
import torch

from tests import paged_oracle as O
from tests.test_kv_cache_gpu import BF, E4, Batch

pytestmark = pytest.mark.gpu

# decode with and without tensor copies, a few tokens per sequence, tiles
FORMS = [(256, 2, 8, [1, 1, 1]), (128, 8, 4, [1, 1, 1]), (64, 2, 4, [1, 1, 1]), (128, 2, 4, [2, 4, 3]), (64, 2, 4, [2, 4, 3]), (128, 2, 4, [40, 1, 90]), (256, 2, 8, [40, 1, 90])]


def batch(dim, kv_heads, group, new, seed=1):
    return Batch(seed, new, [300, 70, 200], kv_heads=kv_heads, heads=kv_heads * group, dim=dim, dtype=BF, cache=E4)


def spot(b, seq, pos):
    return O.place(b.table, b.page, b.k.shape[0], seq, pos)


def set_key(b, pg, rw, first):
    """A key of one element: its score is what the queries' first element makes of it."""
    b.k[pg, :, rw] = 0.0
    b.k[pg, :, rw, 0] = 448.0 if first >= 0 else -448.0
    b.k_scale[pg, :, rw] = abs(first) / 448.0


@pytest.mark.parametrize("dim,kv_heads,group,new", FORMS)
@pytest.mark.parametrize("exponent", [24, 31, 40, 100])
def test_a_large_value_of_a_later_token(dim, kv_heads, group, new, exponent):
    b = batch(dim, kv_heads, group, new)
    for s, length in enumerate([300, 70, 200]):
        pg, rw = spot(b, s, length - 1)
        b.v_scale[pg, :, rw] *= 2.0 ** exponent
    b.check(b.attend(max_query=max(new)))
    b.check(b.attend(max_query=max(new), window=30, sinks=1), window=30, sinks=1)


@pytest.mark.parametrize("dim,kv_heads,group,new", FORMS)
@pytest.mark.parametrize("exponent", [31, 40, 60])
def test_a_large_value_of_no_weight(dim, kv_heads, group, new, exponent):
    """Scores some 60 powers of two below the others', in an early, a middle and a late key."""
    b = batch(dim, kv_heads, group, new)
    b.q[:, :, 0] = 16.0
    for s, length in enumerate([300, 70, 200]):
        for pos in (1, length // 2, length - max(new) - 1 if length > max(new) else 2):
            pg, rw = spot(b, s, max(pos, 1))
            set_key(b, pg, rw, -30.0 * (dim / 128) ** 0.5)
            b.v_scale[pg, :, rw] *= 2.0 ** exponent
    b.check(b.attend(max_query=max(new)))


@pytest.mark.parametrize("dim,kv_heads,group,new", FORMS)
def test_a_large_value_that_loses_its_weight(dim, kv_heads, group, new):
    """The first key leads, with a large value; later ones outscore it by some 60 powers of two."""
    b = batch(dim, kv_heads, group, new)
    b.q[:, :, 0] = 16.0
    for s, length in enumerate([300, 70, 200]):
        pg, rw = spot(b, s, 0)
        b.v_scale[pg, :, rw] *= 2.0 ** 40
        for pos in range(length // 3, length, 7):
            pg, rw = spot(b, s, pos)
            set_key(b, pg, rw, 30.0 * (dim / 128) ** 0.5)
    b.check(b.attend(max_query=max(new)))


@pytest.mark.parametrize("dim,kv_heads,group,new", FORMS)
@pytest.mark.parametrize("large", [0, 60])
def test_values_of_zero_and_values_of_all_magnitudes(dim, kv_heads, group, new, large):
    b = batch(dim, kv_heads, group, new)
    g = torch.Generator().manual_seed(3)
    for s, length in enumerate([300, 70, 200]):
        for pos in list(range(0, length // 2)) + [length - 2]:
            pg, rw = spot(b, s, pos)
            b.v[pg, :, rw] = 0.0
            b.v_scale[pg, :, rw] = O.LEAST / 448.0
    b.v_scale *= torch.exp2(large * (torch.rand(b.v_scale.shape, generator=g) - 0.5))
    b.check(b.attend(max_query=max(new)))


@pytest.mark.parametrize("dim,kv_heads,group,new", FORMS)
@pytest.mark.parametrize("exponent", [-126, -127, -128, -130, -133, -100, 100])
def test_queries_of_any_magnitude(dim, kv_heads, group, new, exponent):
    """Subnormal bf16 queries among them: their scores are all but zero, the result is nearly the mean of the values."""
    b = batch(dim, kv_heads, group, new, seed=2)
    heads = b.q.shape[1]
    b.q[:, : heads // 2] = (b.q[:, : heads // 2].sign() * 2.0 ** exponent).to(BF)
    scale = 1e-30 if exponent > 0 else None
    b.check(b.attend(max_query=max(new), scale=scale), scale=scale)


@pytest.mark.parametrize("dim,kv_heads,group,new", FORMS)
def test_large_values_stay_finite(dim, kv_heads, group, new):
    """Values up to 2^115: sums over 300 keys stay below 2^124, in whole items and in parts, as long as no factor is left in them."""
    b = batch(dim, kv_heads, group, new, seed=4)
    b.v_scale *= 2.0 ** 115 / (448.0 * b.v_scale.max())
    b.check(b.attend(max_query=max(new)))


@pytest.mark.parametrize("dim,kv_heads,group,new", FORMS)
@pytest.mark.parametrize("zero", [0.0, O.LEAST / 448.0])
@pytest.mark.parametrize("exponent", [-20, -40, -90, 40])
def test_values_of_any_magnitude_behind_zeros(dim, kv_heads, group, new, zero, exponent):
    """The first two tiles of keys and a last one hold zeros, with a scale of zero or the least one; all others are small, or large."""
    b = batch(dim, kv_heads, group, new, seed=6)
    b.v_scale *= 2.0 ** exponent
    for s, length in enumerate([300, 70, 200]):
        for pos in list(range(0, min(260, length - 10))) + [length - 1]:
            pg, rw = spot(b, s, pos)
            b.v[pg, :, rw] = 0.0
            b.v_scale[pg, :, rw] = zero
    b.check(b.attend(max_query=max(new)))


def check_on_gpu(b, got, window=0, sinks=0):
    """`Batch.check`, its definition in 64 bits on the GPU, a sequence at a time: for batches that take the oracle minutes."""
    group = b.q.shape[1] // b.k.shape[1]
    for s, length in enumerate(b.lengths.tolist()):
        a, e = int(b.starts[s]), int(b.starts[s + 1])
        at = torch.arange(length)
        pg, rw = b.table[s, at // b.page].long(), at % b.page
        k, v = ((t.float()[pg, :, rw].double() * scale[pg, :, rw].double().unsqueeze(-1)).cuda().repeat_interleave(group, 1) for t, scale in ((b.k, b.k_scale), (b.v, b.v_scale)))
        q, at, pos = b.q[a:e].cuda().double(), at.cuda(), torch.arange(length - (e - a), length, device="cuda").view(-1, 1)
        seen = ((at <= pos) & ((at > pos - window) | (at < sinks)) if window else at <= pos).unsqueeze(1)
        scale = q.shape[2] ** -0.5
        w = torch.softmax((torch.einsum("rhd,jhd->rhj", q, k) * scale).masked_fill(~seen, float("-inf")), -1)
        out, mag = torch.einsum("rhj,jhd->rhd", w, v), torch.einsum("rhj,jhd->rhd", w, v.abs())
        size = (torch.einsum("rhd,jhd->rhj", q.abs(), k.abs()) * scale).masked_fill(~seen, 0.0).amax(-1)
        tol = O.bound(b.dtype, out, mag, size, seen.sum(-1).double().expand_as(size), q.shape[2])
        err = (got[a:e].double() - out).abs()
        assert torch.isfinite(got[a:e]).all() and (err <= tol).all(), f"sequence {s}: {(err / tol).max():.2f} times the bound"


# several key tiles of one item in a row on every pair of SMs: what a row carries from tile to tile is used
RUNS = [(128, 8, 4, 12, 40), (256, 4, 8, 24, 20)]


@pytest.mark.parametrize("dim,kv_heads,group,seqs,tokens", RUNS)
@pytest.mark.parametrize("case", ["zeros", "least", "small after large", "large of no weight", "large that loses its weight", "large of a later token", "all magnitudes"])
def test_magnitudes_over_many_tiles(dim, kv_heads, group, seqs, tokens, case):
    length = 520
    b = Batch(7, [tokens] * seqs, [length] * seqs, kv_heads=kv_heads, heads=kv_heads * group, dim=dim, dtype=BF, cache=E4)
    b.q[:, :, 0] = 16.0
    g = torch.Generator().manual_seed(8)
    if case in ("zeros", "least"):
        b.v_scale *= 2.0 ** -45
    if case == "all magnitudes":
        b.v_scale *= torch.exp2(40 * (torch.rand(b.v_scale.shape, generator=g) - 0.5))
    for s in range(seqs):
        for pos in range(length):
            pg, rw = spot(b, s, pos)
            if case in ("zeros", "least") and pos < 270:
                b.v[pg, :, rw] = 0.0
                b.v_scale[pg, :, rw] = 0.0 if case == "zeros" else O.LEAST / 448.0
            if case == "small after large" and pos >= 150:
                b.v_scale[pg, :, rw] *= 2.0 ** -12
            if case == "large of no weight" and pos % 100 == 30:
                set_key(b, pg, rw, -30.0 * (dim / 128) ** 0.5)
                b.v_scale[pg, :, rw] *= 2.0 ** 45
            if case == "large that loses its weight" and pos == 3:
                b.v_scale[pg, :, rw] *= 2.0 ** 45
            if case == "large that loses its weight" and pos >= 200 and pos % 7 == 0:
                set_key(b, pg, rw, 30.0 * (dim / 128) ** 0.5)
            if case == "large of a later token" and pos == length - 1:
                b.v_scale[pg, :, rw] *= 2.0 ** 45
    check_on_gpu(b, b.attend(max_query=tokens))
    check_on_gpu(b, b.attend(max_query=tokens, window=300, sinks=5), 300, 5)
