"""The paged key/value cache and the attention that reads it, as cases that can be timed and compared.

Three operators: `paged_kv_append` writes new tokens into the cache (as they are, or in 8 bits with one scale per token
and head), `paged_kv_gather` reads tokens back, `paged_attention` lets a chunk of new tokens (one token in decode) attend
to the cache, causally and optionally with a sliding window and a few first tokens that stay visible.

`run` computes an operator from elementary torch operations in 32 bits, or calls the framework where `own` is true.
A case is one operator at one size: `seqs` sequences that bring `tokens` new tokens in all, the longest of them `context`
tokens long with its new ones.  How the tokens and lengths are dealt to the sequences goes by the case alone, the
values and the order of the pages by the seed.
"""

import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
WIDTH = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}
LEAST = 2.0 ** -100         # a row of zeros gets the scale of this maximum


def listed():
    def case(name, kind, **more):
        return dict({"name": name, "kind": kind, "dtype": "bf16", "cache": "bf16", "seqs": 1, "tokens": 1, "context": 1,
                     "heads": 16, "kv_heads": 2, "dim": 256, "page": 16, "window": 0, "sinks": 0}, **more)
    return [
        # one decode step of 32 conversations writes its 32 rows: the time of a call
        case("append, 32 single tokens, 8 bits", "append", cache="e4m3", seqs=32, tokens=32, context=4000),
        # eight prompts written at once: the time of a stream
        case("append, 16384 tokens, 8 bits", "append", cache="e4m3", seqs=8, tokens=16384, context=4096, kv_heads=8, dim=128),
        # an uneven chunk into a cache that keeps its type
        case("append, 1111 tokens", "append", seqs=3, tokens=1111, context=2500),
        # sequences of a quantised cache read back, as for moving them to another place
        case("gather, 65536 tokens, 8 bits", "gather", cache="e4m3", seqs=16, tokens=65536, context=8192),
        # a few short ones of another layout
        case("gather, 777 tokens, f16", "gather", dtype="f16", cache="f16", seqs=5, tokens=777, context=300, kv_heads=4, dim=128, page=32),
        # decode, one conversation of moderate length: the time of a call
        case("decode, 1 x 1000", "attention", seqs=1, tokens=1, context=1000),
        # decode, a full batch of uneven conversations: the time of the cache's bytes
        case("decode, 64 x 16000", "attention", seqs=64, tokens=64, context=16000),
        # the same with a quantised cache and the head layout of many dense models
        case("decode, 128 x 8000, 8 bits", "attention", cache="e4m3", seqs=128, tokens=128, context=8000, heads=32, kv_heads=8, dim=128),
        # decode far into long documents with a window and first tokens that stay
        case("decode, 16 x 131072, window", "attention", seqs=16, tokens=16, context=131072, page=64, window=4096, sinks=4),
        # a chunk of a long prompt: the time of the products
        case("chunk, 2048 of 16384", "attention", seqs=1, tokens=2048, context=16384),
        # prompts' ends, short continuations and single tokens together, with a window
        case("mixed, 1500 in 12 x 4100, window", "attention", dtype="f16", cache="f16", seqs=12, tokens=1500, context=4100, heads=32, kv_heads=8, dim=128, page=32,
             window=1024, sinks=4),
        # full precision, an odd head size and grouping
        case("mixed, 61 in 4 x 700, f32", "attention", dtype="f32", cache="f32", seqs=4, tokens=61, context=700, heads=6, kv_heads=2, dim=80, page=12),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))
    kind = rng.choice(["append", "gather", "decode", "decode", "chunk", "mixed"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"] if kind not in ("chunk", "mixed") else ["bf16", "bf16", "f16"])
    cache = rng.choice([dtype, "e4m3"])
    kv_heads, group, dim = rng.choice([(2, 8, 256), (2, 8, 256), (8, 4, 128), (4, 8, 128), (1, 7, 128), (8, 1, 64), (3, 5, 256), (4, 2, 64), (2, 6, 80), (1, 16, 128)])
    c = {"kind": kind, "dtype": dtype, "cache": cache, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 16, 32, 64, 8, 12, 1, 128]),
         "window": 0, "sinks": 0}
    if kind in ("append", "gather"):
        seqs, tokens = spread(1, 64), spread(1, 16384)
        return dict(c, seqs=seqs, tokens=max(seqs, tokens), context=max(seqs, tokens) + rng.randrange(0, 2000))
    c["kind"] = "attention"
    if rng.random() < 0.4:
        c["window"], c["sinks"] = spread(16, 4096), rng.choice([0, 1, 4, 64])
    if kind == "decode":
        seqs, context = spread(1, 128), spread(1, 16000)
        context = max(1, min(context, 500_000_000 // (seqs * kv_heads * dim * WIDTH[cache])))
        return dict(c, seqs=seqs, tokens=seqs, context=context)
    seqs = 1 if kind == "chunk" else spread(2, 16)
    tokens = spread(2, 2048) if kind == "chunk" else max(seqs, spread(8, 1500))
    context = tokens + spread(1, 8000)
    context = max(tokens, min(context, 1_000_000_000 // (c["heads"] * tokens * seqs)))
    return dict(c, seqs=seqs, tokens=tokens, context=context)


def _layout(case):
    """New tokens and lengths (with the new ones) of each sequence."""
    sizes = sorted((k, v) for k, v in case.items() if k != "name")
    rng = random.Random(repr(sizes))
    S, T, C = case["seqs"], case["tokens"], case["context"]
    if S == T and case["kind"] != "gather":
        new = [1] * S
    elif S == 1:
        new = [T]
    else:
        cuts = sorted(rng.randrange(0, T + 1) for _ in range(S - 1))
        new = [b - a for a, b in zip([0] + cuts, cuts + [T])]
        if case["kind"] == "attention" and T > 2 * S:      # a running batch: a few chunks, the rest single tokens
            for i in range(0, S, 3):
                if new[i] > 1 and i + 1 < S:
                    new[i], new[i + 1] = 1, new[i + 1] + new[i] - 1
    if max(new) > C:
        C = max(new)
    lengths = [max(n, int(C * (0.12 + 0.88 * rng.random()))) for n in new]
    if case["kind"] == "gather":
        lengths = [max(1, n) for n in new]
    lengths[rng.randrange(S)] = max(C, max(lengths)) if case["kind"] != "gather" else max(lengths)
    lengths = [max(a, b) for a, b in zip(lengths, new)]
    return new, lengths


def _visible(case, new, lengths):
    """Pairs of a new token and a token that it sees, and tokens that some new token of their sequence sees."""
    pairs, seen = 0, 0
    w, n0 = case["window"], case["sinks"]
    for n, length in zip(new, lengths):
        first = length - n
        if not w:
            pairs += sum(range(first + 1, length + 1))
            seen += length if n else 0
            continue
        for p in range(first, length):
            lo = max(0, p - w + 1)
            pairs += p + 1 - lo + min(n0, lo)
        if n:
            lo = max(0, first - w + 1)
            seen += length - lo + min(n0, lo)
    return pairs, seen


def work(case):
    new, lengths = _layout(case)
    row = case["kv_heads"] * case["dim"]
    wide, kept = WIDTH[case["dtype"]], WIDTH[case["cache"]]
    scale = 4 * case["kv_heads"] if case["cache"] == "e4m3" else 0
    T = case["tokens"]
    if case["kind"] == "append":
        there = 2 * T * (row * (wide + kept) + scale)
        return {"bytes": 2 * there if case["cache"] == "e4m3" else there, "flops": 0}      # 8 bits: written and read back
    if case["kind"] == "gather":
        return {"bytes": 2 * T * (row * (wide + kept) + scale), "flops": 0}
    pairs, seen = _visible(case, new, lengths)
    return {"bytes": 2 * seen * (row * kept + scale) + 2 * T * case["heads"] * case["dim"] * wide, "flops": 4 * pairs * case["heads"] * case["dim"]}


def _quantised(x):
    """Rows of [..., dim] in 8 bits, and their scales: the largest magnitude of a row becomes 448.  The quotient is taken in
    64 bits: many of a short type's quotients lie half way between two numbers of 8 bits."""
    most = x.float().abs().amax(-1).clamp_min(LEAST)
    return (x.double() * 448.0 / most.double().unsqueeze(-1)).to(torch.float8_e4m3fn), most / 448.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new, lengths = _layout(case)
    S, H, D, ps = case["seqs"], case["kv_heads"], case["dim"], case["page"]
    dtype, kept = TYPES[case["dtype"]], TYPES[case["cache"]]

    def normal(*shape, dtype=dtype):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    def uneven(x):          # tokens differ in magnitude by up to four times
        return x * torch.exp2(2 * torch.rand(*x.shape[:-1], 1, generator=g, device="cuda") - 1).to(x.dtype)

    most = max(-(-n // ps) for n in lengths)
    need = [-(-n // ps) for n in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    first = torch.tensor([sum(need[:i]) for i in range(S)], device="cuda", dtype=torch.int64)
    count = torch.tensor(need, device="cuda", dtype=torch.int64)
    column = torch.arange(most, device="cuda")
    at = (first.unsqueeze(1) + column).clamp_max(pages - 1)
    table = torch.where(column < count.unsqueeze(1), order[at], torch.full_like(order[at], -1)).contiguous()
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s = {"case": dict(case), "table": table, "lengths": torch.tensor(lengths, device="cuda", dtype=torch.int32),
         "starts": torch.tensor(starts, device="cuda", dtype=torch.int32), "rows": case["tokens"], "max_query": max(new), "max_length": max(lengths)}
    shape = (pages, H, ps, D)
    s["k_scale"] = s["v_scale"] = None
    if case["kind"] == "append":
        s["k"], s["v"] = uneven(normal(case["tokens"], H, D)), uneven(normal(case["tokens"], H, D))
        s["k_cache"], s["v_cache"] = (torch.zeros(shape, device="cuda", dtype=kept) for _ in "kv")
        if case["cache"] == "e4m3":
            s["k_scale"], s["v_scale"] = (torch.zeros(shape[:3], device="cuda", dtype=torch.float32) for _ in "kv")
        return s
    if case["cache"] == "e4m3":
        s["k_cache"], s["k_scale"] = _quantised(uneven(normal(*shape, dtype=torch.bfloat16)))
        s["v_cache"], s["v_scale"] = _quantised(uneven(normal(*shape, dtype=torch.bfloat16)))
    else:
        s["k_cache"], s["v_cache"] = uneven(normal(*shape)), uneven(normal(*shape))
    if case["kind"] == "attention":
        s["q"] = normal(case["tokens"], case["heads"], D)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------

def _places(s):
    """Sequence, page and row in the page of each new token."""
    rows = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["starts"][1:], rows, right=True)
    at = s["lengths"][seq] - s["starts"][1:][seq] + rows
    ps = s["k_cache"].shape[2]
    return s["table"][seq, (at // ps).long()].long(), (at % ps).long()


def _put(cache, page, row, x):
    cache = cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache
    cache[page, :, row] = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _take(cache, scale, page, row):
    if scale is None:
        return cache[page, :, row].float()
    return cache.view(torch.uint8)[page, :, row].view(torch.float8_e4m3fn).float() * scale[page, :, row].unsqueeze(-1)


def _append(s):
    page, row = _places(s)
    if s["k_scale"] is None:
        _put(s["k_cache"], page, row, s["k"])
        _put(s["v_cache"], page, row, s["v"])
        return
    k, s["k_scale"][page, :, row] = _quantised(s["k"])
    v, s["v_scale"][page, :, row] = _quantised(s["v"])
    _put(s["k_cache"], page, row, k)
    _put(s["v_cache"], page, row, v)


def _gather(s, dtype):
    page, row = _places(s)
    return _take(s["k_cache"], s["k_scale"], page, row).to(dtype), _take(s["v_cache"], s["v_scale"], page, row).to(dtype)


def _attention(s):
    case, q = s["case"], s["q"]
    S, H, D, n, L = case["seqs"], case["kv_heads"], case["dim"], s["max_query"], s["max_length"]
    G, ps = case["heads"] // H, case["page"]
    j = torch.arange(L, device="cuda")
    page = s["table"][:, j // ps].clamp_min(0).long()
    k = _take(s["k_cache"], s["k_scale"], page, (j % ps).expand(S, L)).permute(0, 2, 3, 1)              # [S, H, D, L]
    v = _take(s["v_cache"], s["v_scale"], page, (j % ps).expand(S, L)).permute(0, 2, 1, 3)              # [S, H, L, D]
    i = torch.arange(n, device="cuda")
    starts, counts = s["starts"][:-1], s["starts"][1:] - s["starts"][:-1]
    at = (starts.unsqueeze(1) + i).clamp_max(s["rows"] - 1).long()                                      # [S, n]
    qs = q[at].float().reshape(S, n, H, G, D).permute(0, 2, 3, 1, 4).reshape(S, H, G * n, D)
    score = (torch.matmul(qs, k) * D ** -0.5).view(S, H, G, n, L)
    pos = (s["lengths"] - counts).unsqueeze(1) + i
    seen = j <= pos.unsqueeze(-1)
    if case["window"]:
        seen = seen & ((j > pos.unsqueeze(-1) - case["window"]) | (j < case["sinks"]))
    score = score.masked_fill(~seen.view(S, 1, 1, n, L), float("-inf"))
    score = torch.exp(score - score.amax(-1, keepdim=True))
    total = score.sum(-1, keepdim=True)
    out = (torch.matmul(score.view(S, H, G * n, L), v).view(S, H, G, n, D) / total).permute(0, 3, 1, 2, 4)
    rows = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["starts"][1:], rows, right=True)
    return out[seq, (rows - s["starts"][seq]).long()].reshape(s["rows"], H * G, D).to(q.dtype)


def run(s):
    case = s["case"]
    dtype, quantised = TYPES[case["dtype"]], s["k_scale"] is not None
    if own:
        import fastkernels_b200 as fk
        cache = (s["k_cache"], s["v_cache"])
        scales = {"key_scale": s["k_scale"], "value_scale": s["v_scale"]}
        if case["kind"] == "append":
            fk.paged_kv_append(s["k"], s["v"], *cache, s["table"], s["lengths"], s["starts"], **scales)
            if quantised:
                return *fk.paged_kv_gather(*cache, s["table"], s["lengths"], s["starts"], s["rows"], dtype=dtype, **scales), s["k_scale"], s["v_scale"]
            return cache
        if case["kind"] == "gather":
            return fk.paged_kv_gather(*cache, s["table"], s["lengths"], s["starts"], s["rows"], dtype=dtype, **scales)
        return fk.paged_attention(s["q"], *cache, s["table"], s["lengths"], s["starts"], window=case["window"], sinks=case["sinks"], max_query=s["max_query"], **scales)
    if case["kind"] == "append":
        _append(s)
        return (*_gather(s, dtype), s["k_scale"], s["v_scale"]) if quantised else (s["k_cache"], s["v_cache"])
    return _gather(s, dtype) if case["kind"] == "gather" else _attention(s)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------

def _e4m3(x):
    """The nearest number of 4 exponent and 3 mantissa bits, ties to even, for |x| <= 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -7))).clamp_min(-6.0) - 3.0)
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    new, lengths = _layout(case)
    ps, H, D = case["page"], case["kv_heads"], case["dim"]
    table = s["table"].tolist()

    def held(cache, scale, i):
        pages = torch.tensor(table[i][: -(-lengths[i] // ps)], device="cuda")
        x = cache[pages].double() if scale is None else cache.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * scale[pages].double().unsqueeze(-1)
        return x.permute(0, 2, 1, 3).reshape(-1, H, D)[: lengths[i]]              # [length, H, D]

    if case["kind"] == "append":
        kept = [s["k_cache"].double(), s["v_cache"].double()]
        scales = [torch.zeros(x.shape[:3], device="cuda", dtype=torch.float64) for x in kept]
        values = []
        for x, cache, scale in zip((s["k"], s["v"]), kept, scales):
            x = x.double()
            most = x.abs().amax(-1).clamp_min(LEAST)
            one = most / 448.0
            if s["k_scale"] is not None:
                values.append(_e4m3(x * 448.0 / most.unsqueeze(-1)) * one.unsqueeze(-1))
            row = 0
            for i, (n, length) in enumerate(zip(new, lengths)):
                at = torch.arange(length - n, length)
                pages = torch.tensor([table[i][p // ps] for p in at.tolist()], device="cuda", dtype=torch.int64)
                off = (at % ps).cuda()
                cache[pages, :, off] = x[row:row + n]
                scale[pages, :, off] = one[row:row + n]
                row += n
        return (*values, *scales) if s["k_scale"] is not None else tuple(kept)
    if case["kind"] == "gather":
        out = []
        for cache, scale in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])):
            out.append(torch.cat([held(cache, scale, i)[lengths[i] - new[i]:] for i in range(case["seqs"])]))
        return tuple(out)
    out, G, first = [], case["heads"] // H, 0
    for i, (n, length) in enumerate(zip(new, lengths)):
        k, v = held(s["k_cache"], s["k_scale"], i), held(s["v_cache"], s["v_scale"], i)
        q = s["q"][first:first + n].double().reshape(n, H, G, D)
        first += n
        pos = torch.arange(length - n, length, device="cuda").view(n, 1)
        j = torch.arange(length, device="cuda")
        hidden = (j > pos) | ((j <= pos - case["window"]) & (j >= case["sinks"])) if case["window"] else j > pos
        heads = []
        for h in range(H):
            for a in range(G):
                score = (q[:, h, a] @ k[:, h].T / D ** 0.5).masked_fill(hidden, float("-inf"))
                heads.append(torch.softmax(score, -1) @ v[:, h])
        out.append(torch.stack(heads, 1))
    return torch.cat(out)
