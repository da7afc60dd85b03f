"""CPU: the cache's and the attention's entry points reject bad arguments before touching a GPU, the oracle of their tests
agrees with a formula it does not use."""

import ctypes as C

import pytest
import torch

import fastkernels_b200 as fk
from fastkernels_b200 import _lib
from fastkernels_b200._lib import AttentionCall, KvCache, KvRows
from tests import paged_oracle as O

ARG, UNSUPPORTED, WORKSPACE = 1, 2, 3


def cache(**kw):
    c = KvCache()
    c.pages, c.kv_heads, c.page_size, c.head_dim, c.dtype, c.seqs, c.max_pages, c.table_stride = 10, 2, 16, 128, _lib.FK_BF16, 3, 4, 4
    c.key_stride[:] = c.value_stride[:] = (4096, 2048, 128)
    c.key = c.value = c.page_table = c.lengths = 4096
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [({"pages": 0}, ARG), ({"kv_heads": 0}, ARG), ({"page_size": 0}, ARG), ({"head_dim": 0}, ARG), ({"head_dim": 257}, ARG), ({"seqs": -1}, ARG),
              ({"max_pages": -1}, ARG), ({"max_pages": 2 ** 27}, ARG), ({"dtype": 4}, UNSUPPORTED), ({"dtype": -1}, UNSUPPORTED), ({"key": None}, ARG),
              ({"value": None}, ARG), ({"lengths": None}, ARG), ({"page_table": None}, ARG), ({"dtype": _lib.FK_E4M3}, ARG), ({"table_stride": -4}, ARG)]


@pytest.mark.parametrize("change,status", BAD_CACHES)
def test_bad_caches(change, status):
    lib = _lib.load()
    r = KvRows(key=4096, value=4096, dtype=_lib.FK_BF16, rows=3)
    a = AttentionCall(cache=cache(**change), query=4096, out=4096, dtype=_lib.FK_BF16, rows=3, q_heads=4, scale=1.0)
    assert lib.fk_kv_append(C.byref(cache(**change)), C.byref(r), None) == status
    assert lib.fk_kv_gather(C.byref(cache(**change)), C.byref(r), None) == status
    assert lib.fk_paged_attention(C.byref(a), None) == status


@pytest.mark.parametrize("change,status", [({"rows": -1}, ARG), ({"dtype": _lib.FK_F16}, UNSUPPORTED), ({"dtype": _lib.FK_E4M3}, UNSUPPORTED), ({"dtype": 9}, UNSUPPORTED),
                                           ({"key": None}, ARG), ({"value": None}, ARG)])
def test_bad_rows(change, status):
    lib = _lib.load()
    r = KvRows(key=4096, value=4096, dtype=_lib.FK_BF16, rows=3)
    for k, v in change.items():
        setattr(r, k, v)
    assert lib.fk_kv_append(C.byref(cache()), C.byref(r), None) == status
    assert lib.fk_kv_gather(C.byref(cache()), C.byref(r), None) == status


@pytest.mark.parametrize("change,status", [({"rows": -1}, ARG), ({"q_heads": 0}, ARG), ({"q_heads": 5}, ARG), ({"dtype": _lib.FK_F32}, UNSUPPORTED), ({"dtype": 3}, UNSUPPORTED),
                                           ({"query": None}, ARG), ({"out": None}, ARG), ({"window": -1}, ARG), ({"sinks": -1}, ARG), ({"max_query": -1}, ARG),
                                           ({"scale": float("nan")}, ARG), ({"scale": float("inf")}, ARG), ({"rows": 2 ** 30, "q_heads": 4}, ARG)])
def test_bad_attention_calls(change, status):
    lib = _lib.load()
    a = AttentionCall(cache=cache(), query=4096, out=4096, dtype=_lib.FK_BF16, rows=3, q_heads=4, scale=1.0)
    for k, v in change.items():
        setattr(a, k, v)
    assert lib.fk_paged_attention(C.byref(a), None) == status


def test_workspace_is_checked_and_empty_calls_return():
    lib = _lib.load()
    a = AttentionCall(cache=cache(), query=4096, out=4096, dtype=_lib.FK_BF16, rows=3, q_heads=4, scale=1.0)
    a.cache.max_pages, a.cache.table_stride = 1000, 1000
    need = lib.fk_paged_attention_workspace_bytes(C.byref(a))
    assert need > 0 and lib.fk_paged_attention(C.byref(a), None) == WORKSPACE
    a.workspace, a.workspace_bytes = 4096, need - 1
    assert lib.fk_paged_attention(C.byref(a), None) == WORKSPACE
    a.workspace, a.workspace_bytes = 4097, need
    assert lib.fk_paged_attention(C.byref(a), None) == WORKSPACE
    a.rows = 0
    assert lib.fk_paged_attention(C.byref(a), None) == 0 and lib.fk_paged_attention_workspace_bytes(C.byref(a)) == 0
    assert lib.fk_paged_attention(None, None) == ARG and lib.fk_paged_attention_workspace_bytes(None) == 0
    assert lib.fk_kv_append(None, None, None) == ARG and lib.fk_kv_gather(C.byref(cache()), None, None) == ARG
    r = KvRows(dtype=_lib.FK_BF16, rows=0)
    assert lib.fk_kv_append(C.byref(cache()), C.byref(r), None) == 0


def test_host_tensors_are_refused():
    x = torch.zeros(2, 2, 16, 64)
    with pytest.raises(ValueError, match="CUDA"):
        fk.paged_attention(torch.zeros(1, 2, 64), x, x, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        fk.paged_kv_append(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), x, x, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="positive"):
        fk.PagedKVCache(0, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="float8"):
        fk.PagedKVCache(4, 2, 64, device="cpu", dtype=torch.int8)


def test_oracle_against_a_masked_softmax():
    g = torch.Generator().manual_seed(1)
    q, k, v = torch.randn(9, 2, 8, generator=g), torch.randn(20, 1, 1, 8, generator=g), torch.randn(20, 1, 1, 8, generator=g)
    table = torch.randperm(20, generator=g).to(torch.int32).view(1, 20)
    out, mag, _, count = O.attention(q, k, v, table, torch.tensor([20]), torch.tensor([0, 9]), scale=0.5, window=6, sinks=2)
    order = table[0].long()
    s = 0.5 * torch.einsum("rhd,jd->hrj", q.double(), k[order, 0, 0].double())
    j, p = torch.arange(20), torch.arange(11, 20).view(9, 1)
    s = s.masked_fill((j > p) | ((j <= p - 6) & (j >= 2)), float("-inf"))
    want = torch.softmax(s, -1) @ v[order, 0, 0].double()
    assert torch.allclose(out, want.permute(1, 0, 2), atol=1e-12) and (mag >= out.abs() - 1e-12).all() and (count == 8).all()


def test_oracle_e4m3_is_the_nearest_code():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().double()
    codes = codes[torch.isfinite(codes)].unique()
    x = torch.cat([codes, (codes[1:] + codes[:-1]) / 2, torch.linspace(-448, 448, 5001, dtype=torch.float64), torch.logspace(-4, 2, 500, dtype=torch.float64)])
    got = O.e4m3(x)
    dist = (x.unsqueeze(1) - codes).abs()
    assert torch.equal((got - x).abs(), dist.min(1).values)
    assert torch.equal(got, x.float().to(torch.float8_e4m3fn).double())       # ties to even as the type's own conversion takes them


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_a_refused_append_leaves_the_cache_as_it_was(dtype):
    c = fk.PagedKVCache(4, 2, 64, device="cpu", dtype=dtype)
    rows = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    for key, value, new in ((rows.float(), rows, [3]), (rows, rows.half(), [3]), (rows.int(), rows.int(), [3]), (rows, rows[:2], [3]), (rows[:, :1], rows[:, :1], [3]),
                            (rows, rows, [2]), (rows, rows, [-3]), (rows, rows, [3, 0]), (rows.transpose(1, 2).contiguous().transpose(1, 2), rows, [3]), (rows, rows, [3])):
        with pytest.raises(ValueError):
            c.append(key, value, new)
        assert c.host_lengths == [0] and c.lengths.tolist() == [0] and (c.page_table == -1).all() and len(c._free) == 4 and c._starts is None
    for shape in ((2 ** 20, 1, 1, 2 ** 11), (4, 1025, 1, 16)):                 # caches that no append would take
        with pytest.raises(ValueError, match="positions"):
            fk.PagedKVCache(*shape[:3], page_size=shape[3], device="cpu", dtype=dtype)


@pytest.mark.parametrize("scale,status", [(2.4e38, ARG), (-2.4e38, ARG), (3.4e38, ARG), (2.35e38, WORKSPACE), (-2.35e38, WORKSPACE)])
def test_scales_at_the_end_of_fp32(scale, status):
    """Scores are held as powers of two: the scale times log2(e) has to be a number."""
    a = AttentionCall(cache=cache(max_pages=1000, table_stride=1000), query=4096, out=4096, dtype=_lib.FK_BF16, rows=3, q_heads=4, scale=scale)
    assert _lib.load().fk_paged_attention(C.byref(a), None) == status
