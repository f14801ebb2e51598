"""CPU oracle of the paged 8-bit cache: append, decode and eviction, a token at a time, from their definitions.

Codes and scales are defined in fp32 arithmetic (each operation rounded to nearest even) and are compared bit for bit; attention is
computed in 64 bits."""
import math

import torch

PAGE = 16
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
LEAST = 2.0 ** -100


def values(codes):
    return codes.to(torch.float32)


def recode(x, dtype):
    """fp32 values in units of the scale as codes."""
    top = TOP[dtype]
    x = x.clamp(-top, top)
    if dtype == torch.int8:
        return torch.where(x.isnan(), 0.0, x).round().to(torch.int8)
    return torch.where(x.isnan(), 0.0, x).to(dtype)


def _put(cache, page, h, slot, codes):
    cache.view(torch.int8)[page, h, slot] = codes.view(torch.int8)


def append(k, v, k_cache, v_cache, scale, table, positions, cu=None):
    """In place; k, v [tokens, H, D] on the CPU.  `cu` None: a token a sequence."""
    dtype, H = k_cache.dtype, k_cache.size(1)
    cu = list(range(k.size(0) + 1)) if cu is None else cu.tolist()
    part = torch.tensor(1.0 / TOP[dtype], dtype=torch.float32)
    for b in range(len(cu) - 1):
        at, n = (0 if positions is None else int(positions[b])), cu[b + 1] - cu[b]
        for p in range(at // PAGE, (at + n + PAGE - 1) // PAGE):
            lo, hi = max(at, p * PAGE), min(at + n, p * PAGE + PAGE)
            if hi <= lo:
                continue
            page, slot = int(table[b, p]), lo - p * PAGE
            for kind, (x, cache) in enumerate(((k, k_cache), (v, v_cache))):
                rows = x[cu[b] + lo - at: cu[b] + hi - at].float()                  # [n, H, D]
                for h in range(H):
                    r = rows[:, h]
                    a = r.abs()
                    most = torch.where(a.isnan(), math.inf, a).max()
                    made = torch.clamp(most * part, min=LEAST)
                    if slot > 0:
                        before = scale[page, h, kind].clone()
                        made = torch.maximum(made, before)
                        if made > before:
                            old = values(cache[page, h, :slot])
                            _put(cache, page, h, slice(0, slot), recode(old * (before / made), dtype))
                    scale[page, h, kind] = made
                    codes = recode(r * (torch.ones(()) / made), dtype) if made < math.inf else torch.zeros(r.shape).to(dtype)
                    _put(cache, page, h, slice(slot, slot + hi - lo), codes)


def rows_of(cache, scale, kind, table_row, h, n):
    """The first n tokens of one head in 64 bits [n, D]."""
    pages = [int(p) for p in table_row[: (n + PAGE - 1) // PAGE]]
    return torch.cat([values(cache[p, h]).double() * scale[p, h, kind].double() for p in pages])[:n] if n else torch.zeros(0, cache.size(3), dtype=torch.float64)


def decode(q, k_cache, v_cache, scale, table, lens, softcap=0.0, mass=None, mass_index=None):
    """(out, sum of weights times magnitudes of values) in 64 bits [B, HQ, T, D]; `mass` (64 bits) in place."""
    B, HQ, T, D = q.shape
    H = k_cache.size(1)
    G = HQ // H
    out, size = torch.zeros(B, HQ, T, D, dtype=torch.float64), torch.zeros(B, HQ, T, D, dtype=torch.float64)
    for b in range(B):
        n = max(0, int(lens[b]))
        row = b if mass_index is None else int(mass_index[b])
        for h in range(H):
            k, v = rows_of(k_cache, scale, 0, table[b], h, n), rows_of(v_cache, scale, 1, table[b], h, n)
            for t in range(T):
                m = n - T + 1 + t
                if m <= 0:
                    continue
                x = q[b, h * G: (h + 1) * G, t].double() @ k[:m].T / math.sqrt(D)
                if softcap:
                    x = softcap * torch.tanh(x / softcap)
                w = torch.softmax(x, 1)
                out[b, h * G: (h + 1) * G, t] = w @ v[:m]
                size[b, h * G: (h + 1) * G, t] = w @ v[:m].abs()
                if mass is not None:
                    mass[row, h, :m] += w.sum(0)
    return out, size


def choose(mass, n, budget, sink, recent):
    """Indices that stay, in order, of one head's n tokens with these sums (a list)."""
    if n <= budget:
        return list(range(n))
    mid = list(range(sink, n - recent))
    worth = [math.nan if math.isnan(x) else x for x in mass]
    mid.sort(key=lambda i: (not math.isnan(worth[i]), -worth[i] if not math.isnan(worth[i]) else 0.0, i))
    return sorted(list(range(sink)) + mid[: budget - sink - recent] + list(range(n - recent, n)))


def evict(mass, k_cache, v_cache, scale, table, lens, new_table, budget, sink=0, recent=0, mass_index=None):
    """In place in the caches; (kept, new lens, new mass)."""
    B, H, dtype = len(lens), k_cache.size(1), k_cache.dtype
    kept = torch.full((B, H, budget), -1, dtype=torch.int32)
    new_mass = torch.zeros(B, H, budget)
    new_lens = torch.tensor([min(max(0, int(n)), budget) for n in lens], dtype=torch.int32)
    for b in range(B):
        n = max(0, int(lens[b]))
        row = b if mass_index is None else int(mass_index[b])
        for h in range(H):
            idx = choose(mass[row, h, :n].tolist(), n, budget, sink, recent)
            kept[b, h, : len(idx)] = torch.tensor(idx, dtype=torch.int32)
            new_mass[b, h, : len(idx)] = mass[row, h, idx]
            for p in range((len(idx) + PAGE - 1) // PAGE):
                to, group = int(new_table[b, p]), idx[p * PAGE: p * PAGE + PAGE]
                src = [int(table[b, i // PAGE]) for i in group]
                for kind, cache in enumerate((k_cache, v_cache)):
                    had = scale[src, h, kind]
                    best = had.max()
                    for j, i in enumerate(group):
                        codes = cache[src[j], h, i % PAGE]
                        if had[j] != best:
                            codes = recode(values(codes) * (had[j] / best), dtype)
                        _put(cache, to, h, j, codes)
                    scale[to, h, kind] = best
    return kept, new_lens, new_mass
