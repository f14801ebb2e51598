"""The operators of the paged 8-bit cache as cases that a timer can run: what writes it, what reads it, and what makes it shorter.

A cache keeps 16 tokens a page, [pages, KV heads, 16, D] codes for keys and for values (int8 or e4m3), with a scale for each page, head and
kind, [pages, KV heads, 2] in fp32: a code stands for code * scale.

    append   rows of keys and values into pages: a token for each sequence of a decode step, or packed prompts (also later parts of them)
    decode   attention of the newest token(s) of each sequence, with or without a cap on the scores and the sums of weights each key got
    evict    the tokens with the largest sums kept, in new pages

    listed()            the cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program has in hand before the call
    run(state)          one pass, and its outputs: in plain torch, or (`own`) by the framework
    exact(case, seed)   the same outputs in 64 bits
    work(case)          bytes and operations that a pass cannot do without
"""
import math

import numpy as np
import torch

own = False

DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}       # largest magnitude of a code
LEAST = 2.0 ** -100                        # least scale
PAGE = 16


def listed():
    return [
        # A serving batch's decode step: one new token of each sequence goes into its page.
        dict(name="append_step", kind="append", dtype="fp16", codes="int8", B=64, HKV=8, D=128, lo=1, hi=1, at=1023),
        # Packed prompts of a serving batch.
        dict(name="append_prompts", kind="append", dtype="bf16", codes="e4m3", B=16, HKV=8, D=128, lo=128, hi=4096, at=0),
        # Parts of a few prompts of a small model that go on in the middle of pages: odd lengths.
        dict(name="append_parts", kind="append", dtype="fp16", codes="int8", B=5, HKV=2, D=64, lo=1, hi=701, at=333),
        # A short conversation with few users: every launch and every microsecond of the call counts.
        dict(name="decode_few", kind="decode", dtype="bf16", codes="int8", B=4, HQ=32, HKV=8, D=128, T=1, lo=1, hi=101, cap=0.0, mass=False),
        # A serving batch's decode step: unequal contexts on scattered pages.
        dict(name="decode_batch", kind="decode", dtype="fp16", codes="int8", B=64, HQ=32, HKV=8, D=128, T=1, lo=512, hi=8192, cap=0.0, mass=False),
        # A decode step of a model with wide heads and capped scores.
        dict(name="decode_capped", kind="decode", dtype="bf16", codes="e4m3", B=32, HQ=16, HKV=2, D=256, T=1, lo=10, hi=8191, cap=50.0, mass=False),
        # One long document.
        dict(name="decode_long", kind="decode", dtype="fp16", codes="e4m3", B=1, HQ=32, HKV=8, D=128, T=1, lo=131071, hi=131071, cap=0.0, mass=False),
        # Four guessed tokens of each sequence checked at once; odd groups, some sequences just begun.
        dict(name="decode_guesses", kind="decode", dtype="bf16", codes="int8", B=16, HQ=40, HKV=8, D=64, T=4, lo=2, hi=4096, cap=0.0, mass=False),
        # A decode step that keeps the sums eviction goes by.
        dict(name="decode_sums", kind="decode", dtype="fp16", codes="int8", B=32, HQ=32, HKV=8, D=128, T=1, lo=1024, hi=8192, cap=0.0, mass=True),
        # Long contexts of a batch cut to a quarter.
        dict(name="evict_batch", kind="evict", codes="int8", B=32, HKV=8, D=128, lo=1024, hi=8192, budget=2048, sink=4, recent=256),
        # One long document cut to an eighth.
        dict(name="evict_long", kind="evict", codes="e4m3", B=1, HKV=8, D=128, lo=131071, hi=131071, budget=16384, sink=4, recent=1024),
        # A few short ones of a small model, some shorter than what is kept.
        dict(name="evict_few", kind="evict", codes="int8", B=4, HKV=2, D=64, lo=1, hi=701, budget=130, sink=1, recent=33),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "evict"])
    hkv, d, b = rng.choice([1, 2, 4, 8, 8]), rng.choice([64, 128, 128, 256]), _log(rng, 1, 64)
    c = dict(kind=kind, codes=rng.choice(["int8", "e4m3"]), B=b, HKV=hkv, D=d)
    # the tokens of all sequences together stay within those of the largest listed case of the kind
    if kind == "append":
        step = rng.random() < 0.5
        most = max(1, min(4096, 34000 * 8 * 128 // (b * hkv * d)))
        hi = 1 if step else _log(rng, 1, most)
        return dict(c, dtype=rng.choice(["fp16", "bf16"]), lo=1 if step else _log(rng, 1, hi), hi=hi, at=_log(rng, 1, 1024) - (0 if step else 1))
    most = max(16, min(131071, (270000 if kind == "decode" else 130000) * 8 * 128 // (b * hkv * d)))
    hi = _log(rng, 16, most)
    lo = _log(rng, 1, hi)
    if kind == "decode":
        group, t = rng.choice([1, 2, 4, 4, 5, 7, 8, 12]), rng.choice([1, 1, 1, 2, 3, 5])
        return dict(c, dtype=rng.choice(["fp16", "bf16"]), HQ=hkv * group, T=t, lo=lo, hi=hi, cap=rng.choice([0.0, 0.0, 30.0]), mass=rng.random() < 0.3)
    budget = _log(rng, 16, max(16, hi // 2))
    sink = rng.randrange(0, min(5, budget))
    return dict(c, lo=lo, hi=hi, budget=budget, sink=sink, recent=rng.randrange(0, budget - sink))


def _spread(lo, hi, n):
    """n whole numbers, evenly spread from hi down to lo."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _lens(c):
    """Tokens of each sequence."""
    return _spread(c["lo"], c["hi"], c["B"])


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _codes(c, shape, g):
    """Codes of normal values under a scale that the largest of a page set."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(TOP[c["codes"]] / 3.5).clamp_(-TOP[c["codes"]], TOP[c["codes"]])
    return x.round_().to(torch.int8) if c["codes"] == "int8" else x.to(torch.float8_e4m3fn)


def prepare(c, seed):
    cpu = torch.Generator().manual_seed(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, H, D = c["B"], c["HKV"], c["D"]
    order = torch.randperm(B, generator=cpu).tolist()
    lens = [_lens(c)[i] for i in order]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    if c["kind"] == "append":
        start = [_spread(0, c["at"], B)[i] for i in order]          # tokens that the cache holds of each already
    total = [n + (start[i] if c["kind"] == "append" else 0) for i, n in enumerate(lens)]
    width = max(_pages(n) for n in total)
    held = sum(_pages(n) for n in total)
    more = sum(_pages(min(n, c["budget"])) for n in lens) if c["kind"] == "evict" else 0
    pages = held + more
    ids = torch.randperm(pages, generator=cpu).tolist()
    table, at = torch.zeros((B, width), dtype=torch.int32), 0
    for i, n in enumerate(total):
        table[i, : _pages(n)] = torch.tensor(ids[at: at + _pages(n)], dtype=torch.int32)
        at += _pages(n)
    s = dict(case=c, table=table.cuda(), width=width, k_cache=_codes(c, (pages, H, PAGE, D), g), v_cache=_codes(c, (pages, H, PAGE, D), g),
             scale=(torch.rand((pages, H, 2), generator=g, device="cuda") + 0.5) * (3.5 / TOP[c["codes"]]))
    if c["kind"] == "append":
        T = DTYPE[c["dtype"]]
        step = c["hi"] == 1
        shape = (B, H, 1, D) if step else (sum(lens), H, D)
        s.update(k=torch.randn(shape, generator=g, device="cuda").to(T), v=torch.randn(shape, generator=g, device="cuda").to(T), start=ints(start),
                 cu=None if step else ints([0] + np.cumsum(lens).tolist()))
        return s
    s["lens"] = ints(lens)
    if c["kind"] == "decode":
        s["q"] = torch.randn((B, c["HQ"], c["T"], D), generator=g, device="cuda").to(DTYPE[c["dtype"]])
    if c["kind"] == "evict" or c["mass"]:
        # sums of weights: heavy tails, and keys that no query has looked at
        m = torch.randn((B, H, width * PAGE), generator=g, device="cuda").mul_(2).exp_().mul_(1e-3)
        s["mass"] = m * (torch.rand(m.shape, generator=g, device="cuda") > 0.1)
    if c["kind"] == "evict":
        new, at = torch.zeros((B, _pages(c["budget"])), dtype=torch.int32), held
        for i, n in enumerate(lens):
            m = _pages(min(n, c["budget"]))
            new[i, :m] = torch.tensor(ids[at: at + m], dtype=torch.int32)
            at += m
        s["new"] = new.cuda()
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------
def _bytes(t):
    return t.view(torch.int8)


def _recode(x, codes):
    """Values in units of the scale as codes."""
    if codes == "int8":
        return x.round().clamp(-127, 127).nan_to_num(0.0).to(torch.int8)
    return x.clamp(-448, 448).nan_to_num(0.0).to(torch.float8_e4m3fn)


def _plain_append(s):
    c, B = s["case"], s["case"]["B"]
    H, D = c["HKV"], c["D"]
    k, v = (s[n].reshape(-1, H, D).float() for n in ("k", "v"))
    n = k.shape[0]
    tok = torch.arange(n, device="cuda")
    seq = tok if s["cu"] is None else torch.searchsorted(s["cu"][1:].long(), tok, right=True)
    first = torch.zeros(B, dtype=torch.long, device="cuda") if s["cu"] is None else s["cu"][:-1].long()
    slot = s["start"].long()[seq] + (tok - first[seq] if s["cu"] is not None else 0)
    page = s["table"].long()[seq, slot // PAGE]
    x = torch.stack((k, v), 2)                                                        # [tokens, H, 2, D]
    new = torch.zeros_like(s["scale"]).index_reduce_(0, page, x.abs().nan_to_num(math.inf, math.inf).amax(3), "amax") / TOP[c["codes"]]
    part = s["start"].long() % PAGE                                                   # rows that the first pages have already
    begun = s["table"].long().gather(1, (s["start"].long() // PAGE).clamp(max=s["width"] - 1)[:, None])[:, 0]
    had = torch.where((part > 0)[:, None, None], s["scale"][begun], torch.zeros((), device="cuda"))
    made = new[begun].clamp(min=LEAST).maximum(had)
    ratio = had / made                                                                # [B, H, 2]
    fit = torch.arange(PAGE, device="cuda")[None] < part[:, None]                     # [B, 16]
    for i, cache in enumerate((s["k_cache"], s["v_cache"])):
        old = _bytes(cache)[begun].view(cache.dtype)
        again = _recode(old.float() * ratio[:, :, i, None, None], c["codes"])
        _bytes(cache)[begun] = torch.where(fit[:, None, :, None] & (made > had)[:, :, i, None, None], _bytes(again), _bytes(old))
    new = new.clamp(min=LEAST)
    new[begun] = made
    s["scale"][page] = new[page]
    inv = (1.0 / new)[page]
    for i, cache in enumerate((s["k_cache"], s["v_cache"])):
        _bytes(cache)[page, :, slot % PAGE] = _bytes(_recode(x[:, :, i] * inv[:, :, i, None], c["codes"]))
    return s["k_cache"], s["v_cache"], s["scale"]


def _gathered(s, i, cache):
    """Values [B, H, tokens, D] in fp32 of the pages of the table."""
    t = s["table"].long()
    x = _bytes(cache)[t].view(cache.dtype).float() * s["scale"][t][..., i, None, None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _plain_decode(s):
    c, q = s["case"], s["q"]
    B, H, D, T = c["B"], c["HKV"], c["D"], c["T"]
    k = _gathered(s, 0, s["k_cache"])
    rows = q.reshape(B, H, -1, D).float()                                            # [B, H, group * T, D]
    x = torch.matmul(rows, k.transpose(2, 3)) / math.sqrt(D)
    del k
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    seen = s["lens"][:, None] - T + 1 + torch.arange(rows.shape[2], device="cuda")[None] % T   # keys that a row sees
    mask = torch.arange(x.shape[3], device="cuda") < seen[:, None, :, None]
    x = x.masked_fill(~mask, -math.inf)
    p = torch.exp(x - x.amax(3, keepdim=True).clamp(min=-1e30))
    p = p / p.sum(3, keepdim=True).clamp(min=1e-30)
    out = torch.matmul(p, _gathered(s, 1, s["v_cache"])).reshape(B, c["HQ"], T, D).to(q.dtype)
    if not c["mass"]:
        return out
    s["mass"] += p.sum(2)
    return out, s["mass"]


def _plain_evict(s):
    c = s["case"]
    B, H, n = s["mass"].shape
    at = torch.arange(n, device="cuda")
    lens = s["lens"].long()[:, None, None]
    short = lens <= c["budget"]
    fixed = (at < lens) & (short | (at < c["sink"]) | (at >= lens - c["recent"]))       # [B, 1, n]
    rest = ((at < lens) & ~fixed).expand(B, H, n)
    rank = torch.where(rest, s["mass"], -math.inf).sort(dim=2, descending=True, stable=True).indices.argsort(2)
    keep = fixed | (rest & (rank < c["budget"] - c["sink"] - c["recent"]))
    slots = _pages(c["budget"]) * PAGE
    to = keep.cumsum(2) - 1
    kept = torch.full((B, H, slots), -1, dtype=torch.int32, device="cuda")
    b, h, j = keep.nonzero(as_tuple=True)
    to = to[b, h, j]
    kept[b, h, to] = j.int()
    new_lens = s["lens"].clamp(max=c["budget"])
    new_mass = torch.where(kept[:, :, : c["budget"]] >= 0, s["mass"].gather(2, kept[:, :, : c["budget"]].long().clamp(min=0)), 0.0)
    src, dst = s["table"].long()[b, j // PAGE], s["new"].long()[b, to // PAGE]
    had = s["scale"][src, h]                                                         # [kept tokens, 2]
    best = torch.zeros_like(s["scale"]).view(-1, 2).index_reduce_(0, dst * H + h, had, "amax").view_as(s["scale"])[dst, h]
    s["scale"][dst, h] = best
    ratio = had / best
    for i, cache in enumerate((s["k_cache"], s["v_cache"])):
        x = _bytes(cache)[src, h, j % PAGE].view(cache.dtype).float() * ratio[:, i, None]
        _bytes(cache)[dst, h, to % PAGE] = _bytes(_recode(x, c["codes"]))
    return kept[:, :, : c["budget"]].contiguous(), new_lens, new_mass, s["k_cache"], s["v_cache"], s["scale"]


def run(s):
    c = s["case"]
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "evict": _plain_evict}[c["kind"]](s)
    import flash_attn_v100_b200 as fa
    if c["kind"] == "append":
        fa.append_paged_kv8(s["k"], s["v"], s["k_cache"], s["v_cache"], s["scale"], s["table"], s["start"], s["width"], cu_seqlens=s["cu"])
        return s["k_cache"], s["v_cache"], s["scale"]
    if c["kind"] == "decode":
        out = fa.forward_paged_decode_gqa_kv8(s["q"], s["k_cache"], s["v_cache"], s["scale"], s["table"], s["lens"], s["width"], softcap=c["cap"],
                                              mass=s.get("mass"))
        return (out, s["mass"]) if c["mass"] else out
    kept, new_lens, new_mass = fa.evict_paged_kv8(s["mass"], s["k_cache"], s["v_cache"], s["scale"], s["table"], s["lens"], s["width"], s["new"],
                                                  c["budget"], c["sink"], c["recent"])
    return kept, new_lens, new_mass, s["k_cache"], s["v_cache"], s["scale"]


# ---- the definition in 64 bits, a sequence at a time ---------------------------------------------------------------------
def exact(c, seed):
    s = prepare(c, seed)
    H, D = c["HKV"], c["D"]
    table = s["table"].tolist()
    if c["kind"] == "append":
        scale, start = s["scale"].double(), s["start"].tolist()
        cu = list(range(c["B"] + 1)) if s["cu"] is None else s["cu"].tolist()
        kv = torch.stack((s["k"].reshape(-1, H, D), s["v"].reshape(-1, H, D)), 2).double().abs().amax(3)      # [tokens, H, 2]
        for b, at in enumerate(start):
            n = cu[b + 1] - cu[b]
            for p in range(at // PAGE, _pages(at + n)):
                lo, hi = max(at, p * PAGE), min(at + n, p * PAGE + PAGE)
                need = kv[cu[b] + lo - at: cu[b] + hi - at].amax(0) / TOP[c["codes"]]
                page = table[b][p]
                scale[page] = torch.maximum(need, scale[page]) if lo > p * PAGE else need
        return None, None, scale
    if c["kind"] == "evict":
        mass, lens = s["mass"].double().cpu().numpy(), s["lens"].tolist()
        new_mass = np.zeros((c["B"], H, c["budget"]))
        scale, old, new = s["scale"].double().cpu().numpy(), s["scale"].double().cpu().numpy(), s["new"].tolist()
        for b, n in enumerate(lens):
            for h in range(H):
                idx = np.arange(n)
                if n > c["budget"]:
                    mid = np.arange(c["sink"], n - c["recent"])
                    best = mid[np.argsort(-mass[b, h, mid], kind="stable")[: c["budget"] - c["sink"] - c["recent"]]]
                    idx = np.concatenate([np.arange(c["sink"]), np.sort(best), np.arange(n - c["recent"], n)])
                new_mass[b, h, : idx.size] = mass[b, h, idx]
                of = old[np.array(table[b])[idx // PAGE], h]
                for p in range(_pages(idx.size)):
                    scale[new[b][p], h] = of[p * PAGE: p * PAGE + PAGE].max(0)
        return None, None, torch.from_numpy(new_mass), None, None, torch.from_numpy(scale)
    out = torch.zeros((c["B"], c["HQ"], c["T"], D), dtype=torch.float64, device="cuda")
    mass = s["mass"].double() if c["mass"] else None
    for b, n in enumerate(s["lens"].tolist()):
        ids = torch.tensor(table[b][: _pages(n)], device="cuda")
        kv = [(cache.view(torch.int8)[ids].view(cache.dtype).to(torch.float64) * s["scale"][ids].double()[:, :, i, None, None]).transpose(0, 1).reshape(H, -1, D)[:, :n]
              for i, cache in enumerate((s["k_cache"], s["v_cache"]))]
        for t in range(c["T"]):
            m = n - c["T"] + 1 + t
            if m <= 0:
                continue
            q = s["q"][b, :, t].double().view(H, -1, D)
            x = torch.einsum("hgd,hnd->hgn", q, kv[0][:, :m]) * D ** -0.5
            if c["cap"]:
                x = torch.tanh(x / c["cap"]) * c["cap"]
            w = torch.softmax(x, 2)
            out[b, :, t] = torch.einsum("hgn,hnd->hgd", w, kv[1][:, :m]).reshape(-1, D)
            if mass is not None:
                mass[b, :, :m] += w.sum(1)
    return out if mass is None else (out, mass)


def work(c):
    lens, H, D = _lens(c), c["HKV"], c["D"]
    tokens, pages = sum(lens), sum(_pages(n) for n in lens)
    if c["kind"] == "append":
        return {"bytes": tokens * H * 2 * (2 * D + D) + (tokens + PAGE - 1) // PAGE * H * 8, "flops": tokens * H * 2 * D * 3}
    if c["kind"] == "decode":
        rows = c["B"] * c["HQ"] * c["T"]
        seen = sum(max(0, n - c["T"] + 1 + t) for n in lens for t in range(c["T"]))
        return {"bytes": tokens * H * 2 * D + pages * (H * 8 + 4) + rows * D * 4 + (tokens * H * 8 if c["mass"] else 0),
                "flops": seen * c["HQ"] * 4 * D}
    kept = sum(min(n, c["budget"]) for n in lens)
    return {"bytes": tokens * H * 4 + kept * H * (4 * D + 8) + (pages + sum(_pages(min(n, c["budget"])) for n in lens)) * H * 8, "flops": kept * H * 4 * D}
