"""Paged key/value cache and attention from their definitions in 64 bits on the CPU, one row at a time, and the bounds that
follow from the types' roundings."""

import torch

LEAST = 2.0 ** -100


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def e4m3(x):
    """Nearest e4m3 number (ties to even) of |x| <= 448, in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -7))).clamp_min(-6.0) - 3.0)
    return torch.round(x / step) * step


def quantised(x):
    """(codes as 64-bit values, fp32 scales) of rows [..., dim]."""
    most = x.double().abs().amax(-1).clamp_min(LEAST)
    return e4m3(x.double() * 448.0 / most.unsqueeze(-1)), most.float() / 448.0


def place(table, page_size, pages, seq, pos):
    """(page, row) of a position, or None."""
    if pos < 0 or pos // page_size >= table.shape[1]:
        return None
    page = int(table[seq, pos // page_size])
    return (page, pos % page_size) if 0 <= page < pages else None


def rows_of(starts, lengths, rows):
    """(row, sequence, position) of every row that belongs to a sequence."""
    if starts is None:
        return [(s, s, int(lengths[s]) - 1) for s in range(min(rows, len(lengths)))]
    out = []
    for s in range(len(lengths)):
        for r in range(int(starts[s]), min(int(starts[s + 1]), rows)):
            out.append((r, s, int(lengths[s]) - int(starts[s + 1]) + r))
    return out


def read(cache, scale, page, head, row):
    x = cache[page, head, row].float().double()
    return x if scale is None else x * scale[page, head, row].double()


def attention(q, k_cache, v_cache, table, lengths, starts, *, scale, window=0, sinks=0, k_scale=None, v_scale=None):
    """(out, weighted magnitudes sum p|v| / sum p, largest sum |q||k| scale of a row, visible keys of a row), all of [rows, heads, ..]."""
    rows, heads, dim = q.shape
    pages, kv_heads, ps, _ = k_cache.shape
    group = heads // kv_heads
    out, mag = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    size, count = torch.zeros(rows, heads, dtype=torch.float64), torch.zeros(rows, heads, dtype=torch.float64)
    for r, s, p in rows_of(starts, lengths, rows):
        seen = [j for j in range(p + 1) if not window or j > p - window or j < sinks]
        at = [x for x in (place(table, ps, pages, s, j) for j in seen) if x is not None]
        if not at:
            continue
        pg, rw = torch.tensor([a for a, _ in at]), torch.tensor([b for _, b in at])
        for h in range(kv_heads):
            k, v = k_cache.float()[pg, h, rw].double(), v_cache.float()[pg, h, rw].double()
            if k_scale is not None:
                k, v = k * k_scale[pg, h, rw].double().unsqueeze(-1), v * v_scale[pg, h, rw].double().unsqueeze(-1)
            for g in range(group):
                a = h * group + g
                x = q[r, a].double()
                w = torch.softmax(k @ x * scale, 0)
                out[r, a], mag[r, a] = w @ v, w @ v.abs()
                size[r, a], count[r, a] = (k.abs() @ x.abs()).max() * abs(scale), len(at)
    return out, mag, size, count


def bound(dtype, out, mag, size, count, dim, weights=None):
    """Elementwise bound of an attention output of `dtype`: its own rounding; one rounding of each weight to `weights` (the
    query's type where None; fp32 has none); scores summed in fp32 over dim products (dim + 16 roundings of 2^-24 of
    sum |q||k| scale, twice: numerator and denominator), fp32 sums of the weights and products over `count` keys
    (count roundings of 2^-24 each, pessimistic) and 2^-20 for the powers of two."""
    u = half_step(dtype)
    w = half_step(weights or dtype) if (weights or dtype) != torch.float32 else 0.0
    score = 2.0 * (dim + 16) * 2.0 ** -24 * (size + 1.0) + 2.0 * count * 2.0 ** -24 + 2.0 ** -20
    return u * out.abs() + (1 + u) * (w + score).unsqueeze(-1) * 2.0 * mag + torch.finfo(dtype).tiny
