"""Inputs of the tests of the paged 8-bit cache: caches on scattered pages, made on the CPU from a seed."""
import math

import torch

from oracle import kv8_oracle as orc

CODES = (torch.int8, torch.float8_e4m3fn)
PAGE = 16


def tables(lens, pages, seed, width=None):
    """(table [B, width] int32 with -1 behind a sequence's pages, pages handed out) for sequences of these lengths."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(pages, generator=g).tolist()
    need = [(max(0, n) + PAGE - 1) // PAGE for n in lens]
    width = width or max(1, max(need))
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(ids[at: at + n], dtype=torch.int32)
        at += n
    assert at <= pages
    return table, ids[at:]


def cache(pages, H, D, codes, seed, spread=4.0):
    """(k codes, v codes, scale): scales differ between pages by up to `spread`."""
    g = torch.Generator().manual_seed(seed)
    top = orc.TOP[codes]
    kv = [orc.recode(torch.randn(pages, H, PAGE, D, generator=g) * (top / 3), codes) for _ in range(2)]
    scale = torch.exp((torch.rand(pages, H, 2, generator=g) - 0.5) * 2 * math.log(spread)) * (2.0 / top)
    return kv[0], kv[1], scale


def bits(t):
    """Codes as integers that can be compared."""
    return t.view(torch.int8) if t.dtype == torch.float8_e4m3fn else t


def half_step(dtype):
    """Relative error of one rounding to the type."""
    return torch.finfo(dtype).eps / 2


def decode_bound(q, k_cache, scale, out, size, dtype, softcap):
    """How far an output may be from its 64-bit value, element by element.

    The rounding of the result; of every weight to fp16 (2^-11 of its product with the value, 2^-24 of the largest value
    where a weight is below fp16's normal range); and what the score's error does to numerator and denominator.  Scores add D / 16 products of
    tensor cores in fp32, each sum off by at most 2^-22 of sum |q| times the largest code, 127 or 448; base-2 exponentials, the cap's tanh and the
    multiplications: 2^-18 and 2^-21 of the cap."""
    D = q.shape[3]
    most = orc.TOP[k_cache.dtype]
    score = float(q.double().abs().sum(3).max()) * most * float(scale[..., 0].max()) / math.sqrt(D) * (D / 16) * 2.0 ** -22
    delta = score + softcap * 2.0 ** -21 + 2.0 ** -18
    assert delta < 2.0 ** -7
    return out.abs() * half_step(dtype) + size * (2.0 ** -11 + 2 * delta) + float(size.max()) * 2.0 ** -20, delta
