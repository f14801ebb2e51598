"""GPU: the operators on the paged 8-bit cache against the CPU oracle.  Codes, scales, kept tokens and their sums are compared bit for bit;
attention goes by the bound that tests/kv8_cases.py derives."""
import math
import os
import subprocess
import sys

import pytest
import torch

import kv8_cases as kc
from oracle import kv8_oracle as orc

pytestmark = pytest.mark.gpu
CODES = kc.CODES
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def fa():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import flash_attn_v100_b200
    return flash_attn_v100_b200


@pytest.fixture(autouse=True)
def no_errors(fa):
    yield
    torch.cuda.synchronize()
    fa.check_async_errors()


def _same(got, want):
    got = got.cpu()
    assert got.dtype == want.dtype and got.shape == want.shape
    assert torch.equal(kc.bits(got), kc.bits(want)), (kc.bits(got) != kc.bits(want)).sum().item()


def _ints(v):
    return torch.tensor(v, dtype=torch.int32)


# ---- append --------------------------------------------------------------------------------------------------------
def _append_both(fa, k, v, kc0, vc0, sc0, table, positions, cu, mutate=lambda t: t):
    dev = [t.cuda() for t in (kc0, vc0, sc0)]
    fa.append_paged_kv8(mutate(k.cuda()), mutate(v.cuda()), *dev, table.cuda(), None if positions is None else positions.cuda(), table.size(1),
                        cu_seqlens=None if cu is None else cu.cuda())
    ref = [t.clone() for t in (kc0, vc0, sc0)]
    flat = lambda t: t.reshape(-1, t.size(1), t.size(-1)) if cu is None else t
    orc.append(flat(k), flat(v), *ref, table, positions, cu)
    for got, want in zip(dev, ref):
        _same(got, want)
    return dev, ref


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,H", [(64, 2), (128, 3), (256, 1)])
def test_append_packed_prompts(fa, codes, dtype, D, H):
    lens, starts = [1, 0, 15, 16, 17, 40, 0, 3, 33], [0, 5, 1, 0, 16, 30, 2, 14, 15]
    total = [a + n for a, n in zip(starts, lens)]
    table, rest = kc.tables(total, 40, 1)
    g = torch.Generator().manual_seed(D + H)
    k, v = ((torch.randn(sum(lens), H, D, generator=g) * s).to(dtype) for s in (3.0, 0.02))
    cu = _ints([0] + torch.tensor(lens).cumsum(0).tolist())
    _append_both(fa, k, v, *kc.cache(40, H, D, codes, 2), table, _ints(starts), cu)
    _append_both(fa, k, v, *kc.cache(40, H, D, codes, 3), table, None, cu)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_append_steps_grow_the_scale(fa, codes, D):
    """Forty steps of three sequences: a page's scale grows as larger rows come, its codes are rounded again, a new page begins anew."""
    H, B = 2, 3
    table, _ = kc.tables([50, 57, 64], 12, 4)
    state = kc.cache(12, H, D, codes, 5)
    dev, ref = [t.cuda() for t in state], [t.clone() for t in state]
    g = torch.Generator().manual_seed(6)
    for step in range(40):
        k, v = (torch.randn(B, H, 1, D, generator=g).mul(1 + 0.2 * step).half() for _ in range(2))
        pos = _ints([step, step + 7, step + 15])
        fa.append_paged_kv8(k.cuda(), v.cuda(), *dev, table.cuda(), pos.cuda(), table.size(1))
        orc.append(k[:, :, 0], v[:, :, 0], *ref, table, pos)
    for got, want in zip(dev, ref):
        _same(got, want)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_values_at_the_edges(fa, codes, dtype):
    """Zeros, the least and the largest values, infinities and NaN; also into a page that has rows."""
    D, H = 64, 1
    rows = torch.randn(12, H, D, generator=torch.Generator().manual_seed(7)).to(dtype)
    top = torch.finfo(dtype).max
    rows[0] = 0
    rows[1] = torch.finfo(dtype).smallest_normal
    rows[2] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps           # least subnormal
    rows[3, 0, 3] = top
    rows[4, 0, 5] = math.inf
    rows[5, 0, 7] = -math.inf
    rows[6, 0, 9] = math.nan
    rows[7] = -0.0
    rows[8] = torch.arange(D).to(dtype) / D - 0.5
    for start in (0, 3):
        n = rows.size(0)
        table, _ = kc.tables([start + 1] * n, n, 8)
        cu = _ints(range(n + 1))
        _append_both(fa, rows, rows.flip(0), *kc.cache(n, H, D, codes, 9), table, _ints([start] * n), cu)


def test_append_takes_slices_of_a_fused_projection(fa):
    H, D, n = 2, 128, 37
    g = torch.Generator().manual_seed(10)
    fused = torch.randn(n, 4 * H * D, generator=g).half().cuda()
    k, v = fused[:, H * D: 2 * H * D].view(n, H, D), fused[:, 3 * H * D:].view(n, H, D)
    assert not k.is_contiguous()
    table, _ = kc.tables([n], 4, 11)
    state = kc.cache(4, H, D, torch.int8, 12)
    dev, ref = [t.cuda() for t in state], [t.clone() for t in state]
    fa.append_paged_kv8(k, v, *dev, table.cuda(), None, table.size(1), cu_seqlens=_ints([0, n]).cuda())
    orc.append(k.cpu(), v.cpu(), *ref, table, None, _ints([0, n]))
    for got, want in zip(dev, ref):
        _same(got, want)
    # a decode step on one row of a fused projection per sequence
    kd, vd = (t[:3].unsqueeze(2) for t in (k, v))
    table3, _ = kc.tables([16, 20, 1], 4, 13)
    fa.append_paged_kv8(kd, vd, *dev, table3.cuda(), _ints([15, 19, 0]).cuda(), table3.size(1))
    orc.append(kd[:, :, 0].cpu(), vd[:, :, 0].cpu(), *ref, table3, _ints([15, 19, 0]))
    for got, want in zip(dev, ref):
        _same(got, want)


def test_append_leaves_bad_pages_alone(fa):
    H, D = 2, 64
    state = kc.cache(4, H, D, torch.int8, 14)
    table = _ints([[0, 7], [-1, 1], [2, 3]])
    k = torch.randn(3 * 20, H, D, generator=torch.Generator().manual_seed(15)).half()
    dev, ref = [t.cuda() for t in state], [t.clone() for t in state]
    # pages 7 and -1 are outside the cache, and tokens 32 to 39 of the last sequence have no entry of the table
    fa.append_paged_kv8(k.cuda(), k.cuda(), *dev, table.cuda(), _ints([0, 0, 20]).cuda(), 2, cu_seqlens=_ints([0, 20, 40, 60]).cuda())
    with pytest.raises(RuntimeError, match="outside the cache"):
        fa.check_async_errors()
    fa.check_async_errors()
    for rows, page, slot in ((k[:16], 0, 0), (k[36:40], 1, 0), (k[40:52], 3, 4)):
        orc.append(rows, rows, *ref, _ints([[page]]), _ints([slot]), _ints([0, rows.size(0)]))
    for got, want in zip(dev, ref):
        _same(got, want)


@pytest.mark.parametrize("packed", [False, True])
def test_padded_batches(fa, packed):
    """Sequences with a negative position write nothing and report nothing; with a length of 0 they get zeros and add no weights."""
    H, D, B = 2, 64, 5
    state = kc.cache(8, H, D, torch.int8, 16)
    table = torch.full((B, 2), -1, dtype=torch.int32)
    table[1], table[3] = _ints([4, 2]), _ints([7, 0])
    lens = [0, 20, 0, 17, 0]
    g = torch.Generator().manual_seed(17)
    cu = _ints([0, 3, 7, 12, 14, 15]) if packed else None
    k, v = (torch.randn(15, H, D, generator=g).half() if packed else torch.randn(B, H, 1, D, generator=g).half() for _ in range(2))
    pos = _ints([-1, 16 if packed else 19, -7, 15 if packed else 16, -2147483648])
    dev, ref = [t.cuda() for t in state], [t.clone() for t in state]
    fa.append_paged_kv8(k.cuda(), v.cuda(), *dev, table.cuda(), pos.cuda(), 2, cu_seqlens=None if cu is None else cu.cuda())
    flat = lambda t: t.reshape(-1, H, D)
    for b in (1, 3):
        rows = slice(int(cu[b]), int(cu[b + 1])) if packed else slice(b, b + 1)
        n = rows.stop - rows.start
        orc.append(flat(k)[rows], flat(v)[rows], *ref, table[b: b + 1], pos[b: b + 1], _ints([0, n]))
    for got, want in zip(dev, ref):
        _same(got, want)
    q, mass = torch.randn(B, 4, 1, D, generator=g).half(), torch.zeros(B, H, 32)
    sums = mass.cuda()
    out = fa.forward_paged_decode_gqa_kv8(q.cuda(), *dev, table.cuda(), _ints(lens).cuda(), 2, mass=sums)
    want, size = orc.decode(q, *ref, table, lens)
    bound, _ = kc.decode_bound(q, ref[0], ref[2], want, size, torch.float16, 0.0)
    assert bool(((out.cpu().double() - want).abs() <= bound).all())
    assert all(bool((out[b] == 0).all()) and bool((sums[b] == 0).all()) for b in (0, 2, 4))


# ---- decode --------------------------------------------------------------------------------------------------------
def _decode_case(fa, codes, dtype, H, G, D, T, lens, seed, softcap=0.0, mass=False, q_scale=1.0):
    pages = sum((max(0, n) + 15) // 16 for n in lens) + 3
    table, rest = kc.tables(lens, pages, seed)
    k8, v8, scale = kc.cache(pages, H, D, codes, seed + 1)
    for p in rest:                                    # pages of nobody: whoever reads them shows
        scale[p] = math.nan
    g = torch.Generator().manual_seed(seed + 2)
    q = (torch.randn(len(lens), H * G, T, D, generator=g) * q_scale).to(dtype)
    sums = torch.rand(len(lens) + 2, H, table.size(1) * 16 + 5, generator=g) if mass else None
    index = torch.randperm(len(lens) + 2, generator=g)[: len(lens)].int() if mass else None
    dev = sums.cuda() if mass else None
    out = fa.forward_paged_decode_gqa_kv8(q.cuda(), k8.cuda(), v8.cuda(), scale.cuda(), table.cuda(), _ints(lens).cuda(), table.size(1), softcap=softcap,
                                          mass=dev, mass_index=index.cuda() if mass else None)
    assert out.shape == q.shape and out.dtype == dtype
    sums64 = sums.double() if mass else None
    used = scale.clone()
    for p in rest:
        used[p] = 0
    ref, size = orc.decode(q, k8, v8, used, table, lens, softcap, sums64, index)
    bound, delta = kc.decode_bound(q, k8, used, ref, size, dtype, softcap)
    off = (out.cpu().double() - ref).abs()
    assert bool((off <= bound).all()), (off / bound).max().item()
    if mass:
        got = dev.cpu().double()
        added = sums64 - sums.double()
        limit = added * (2 * delta + 2.0 ** -18) + sums64 * 2.0 ** -23
        assert bool(((got - sums64).abs() <= limit).all())
        assert torch.equal(dev.cpu()[added == 0], sums[added == 0])
    return out


LENS = [0, 1, 15, 16, 17, 33, 100, 257]


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G", [1, 4, 8, 12])
def test_decode_shapes(fa, codes, dtype, D, G):
    _decode_case(fa, codes, dtype, 2, G, D, 1, LENS, 20 + G)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("H,G,T", [(1, 1, 1), (3, 5, 1), (2, 20, 1), (1, 4, 4), (2, 5, 3), (2, 1, 40), (1, 3, 17)])
def test_decode_groups_and_guessed_tokens(fa, codes, H, G, T):
    _decode_case(fa, codes, torch.bfloat16, H, G, 128, T, LENS + [40], 30 + G + T, mass=True)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("D,G", [(64, 4), (128, 9), (256, 4)])
@pytest.mark.parametrize("softcap", [0.0, 5.0, 50.0])
def test_decode_capped_and_summed(fa, codes, D, G, softcap):
    _decode_case(fa, codes, torch.float16, 2, G, D, 2, LENS, 40 + G, softcap=softcap, mass=True, q_scale=2.0)


@pytest.mark.parametrize("lens", [[5000], [4097, 3], [31, 3000, 1, 16], [700] * 5, [64] * 160], ids=str)
@pytest.mark.parametrize("codes", CODES)
def test_decode_cut_into_parts(fa, codes, lens):
    """Few long sequences (parts for CTAs of their own), and enough sequences for an even cut through all of them."""
    _decode_case(fa, codes, torch.float16, 2, 4, 128, 1, lens, 50 + len(lens), mass=len(lens) < 100)


def test_decode_even_cut_of_unequal_sequences(fa):
    lens = [(37 * i) % 500 for i in range(200)]
    _decode_case(fa, torch.int8, torch.float16, 2, 2, 64, 1, lens, 60, mass=True)


def test_decode_of_more_sequences_than_a_launch_takes(fa):
    lens = [i % 3 for i in range(4100)]
    _decode_case(fa, torch.int8, torch.float16, 1, 1, 64, 1, lens, 61)


@pytest.mark.parametrize("codes", CODES)
def test_decode_scales_of_all_sizes(fa, codes):
    """Pages whose scales differ by 2^40 and pages of zeros under a scale of 0: the large ones decide the result, all of them the weights."""
    H, D, lens = 1, 64, [100, 64]
    table, _ = kc.tables(lens, 12, 62)
    k8, v8, scale = kc.cache(12, H, D, codes, 63)
    g = torch.Generator().manual_seed(64)
    scale[..., 1] = torch.exp2(torch.randint(-20, 21, (12, H), generator=g).float())
    zero = int(table[0, 2])
    scale[zero] = 0.0
    q = torch.randn(2, 4, 1, D, generator=g).bfloat16()
    out = fa.forward_paged_decode_gqa_kv8(q.cuda(), k8.cuda(), v8.cuda(), scale.cuda(), table.cuda(), _ints(lens).cuda(), table.size(1))
    ref, size = orc.decode(q, k8, v8, scale, table, lens)
    bound, _ = kc.decode_bound(q, k8, scale, ref, size, torch.bfloat16, 0.0)
    assert bool(((out.cpu().double() - ref).abs() <= bound).all())


def test_decode_spoiled_pages_spoil_what_sees_them(fa):
    """An infinite scale (a page that was given NaN) makes the rows that see it NaN and no others; codes behind a sequence's end are not seen."""
    H, D, lens = 1, 64, [40, 40]
    table, _ = kc.tables(lens, 6, 65)
    k8, v8, scale = kc.cache(6, H, D, torch.float8_e4m3fn, 66)
    kc.bits(k8)[int(table[1, 2]), :, 8:] = 0x7F                                  # NaN behind token 39
    kc.bits(v8)[int(table[1, 2]), :, 8:] = 0x7F
    q = torch.randn(2, 4, 1, D, generator=torch.Generator().manual_seed(67)).half()
    args = lambda s: (q.cuda(), k8.cuda(), v8.cuda(), s.cuda(), table.cuda(), _ints(lens).cuda(), table.size(1))
    fine = fa.forward_paged_decode_gqa_kv8(*args(scale))
    assert bool(fine.isfinite().all())
    for kind in (0, 1):
        bad = scale.clone()
        bad[int(table[0, 1]), 0, kind] = math.inf
        kc.bits(k8 if kind == 0 else v8)[int(table[0, 1])] = 0
        out = fa.forward_paged_decode_gqa_kv8(*args(bad))
        assert bool(out[0].isnan().all()) and torch.equal(out[1], fine[1])


def test_decode_reports_bad_pages(fa):
    H, D, lens = 1, 64, [40, 20]
    table, _ = kc.tables(lens, 6, 68)
    table[0, 1] = 6
    q = torch.zeros(2, 1, 1, D).half().cuda()
    k8, v8, scale = (t.cuda() for t in kc.cache(6, H, D, torch.int8, 69))
    out = fa.forward_paged_decode_gqa_kv8(q, k8, v8, scale, table.cuda(), _ints(lens).cuda(), table.size(1))
    assert bool(out[1].isfinite().all())
    with pytest.raises(RuntimeError, match="outside the cache"):
        fa.check_async_errors()


def test_decode_lengths_beyond_the_table_are_cut(fa):
    H, D = 1, 64
    table, _ = kc.tables([32], 4, 70)
    k8, v8, scale = (t.cuda() for t in kc.cache(4, H, D, torch.int8, 71))
    q = torch.randn(1, 2, 1, D, generator=torch.Generator().manual_seed(72)).half().cuda()
    run = lambda n: fa.forward_paged_decode_gqa_kv8(q, k8, v8, scale, table.cuda(), _ints([n]).cuda(), 2)
    assert torch.equal(run(1000), run(32)) and bool((run(-3) == 0).all())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("D,G", [(64, 2), (64, 5), (128, 4), (256, 1)])
@pytest.mark.parametrize("how", ["keys", "values", "outside"])
def test_decode_spoiled_pages_leave_earlier_tokens_alone(fa, codes, D, G, how):
    """Of four new tokens those that do not see a page of an infinite scale, or one outside the cache, come out as if it were fine; those without keys stay zero."""
    H, T, lens = 2, 4, [33, 65, 2, 17, 146]
    seen_from = [3, 3, 2, 4, 2]                                   # the first new token that sees the last page (sequence 3: left fine)
    table, rest = kc.tables(lens, 24, 130)
    k8, v8, scale = kc.cache(24, H, D, codes, 131)
    q = torch.randn(len(lens), H * G, T, D, generator=torch.Generator().manual_seed(132)).half().cuda()
    args = lambda k, v, s, t: (q, k.cuda(), v.cuda(), s.cuda(), t.cuda(), _ints(lens).cuda(), t.size(1))
    fine = fa.forward_paged_decode_gqa_kv8(*args(k8, v8, scale, table))
    assert bool(fine.isfinite().all()) and bool((fine[2, :, :2] == 0).all())
    for b in (0, 1, 2, 4):
        at = (lens[b] - 1) // 16
        if how == "outside":
            table[b, at] = 24
            continue
        kind = 0 if how == "keys" else 1
        scale[int(table[b, at]), :, kind] = math.inf
        kc.bits((k8, v8)[kind])[int(table[b, at])] = 0
    out = fa.forward_paged_decode_gqa_kv8(*args(k8, v8, scale, table))
    for b, t in enumerate(seen_from):
        assert torch.equal(out[b, :, :t], fine[b, :, :t]) and bool(out[b, :, t:].isnan().all())
    if how == "outside":
        with pytest.raises(RuntimeError, match="outside the cache"):
            fa.check_async_errors()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("D,G", [(64, 4), (128, 9), (256, 4)])
@pytest.mark.parametrize("softcap", [1e-30, 0.5, 30.0, 1e3, 1e5, 1e6, 1e30])
def test_decode_caps_of_all_sizes(fa, codes, D, G, softcap):
    """Up to the largest cap that is accepted, which leaves the scores as they are.

    The cap's error goes by the score: 2^-19 of it, from a quarter of the cap on an error of 2^-21 of the cap, and a polynomial's 2^-20 below."""
    H, T, lens = 2, 2, LENS
    table, _ = kc.tables(lens, 40, 133)
    k8, v8, scale = kc.cache(40, H, D, codes, 134)
    g = torch.Generator().manual_seed(135)
    q = (torch.randn(len(lens), H * G, T, D, generator=g) * 2).half()
    sums = torch.zeros(len(lens), H, table.size(1) * 16)
    dev, sums64 = sums.cuda(), sums.double()
    out = fa.forward_paged_decode_gqa_kv8(q.cuda(), k8.cuda(), v8.cuda(), scale.cuda(), table.cuda(), _ints(lens).cuda(), table.size(1), softcap=softcap, mass=dev)
    ref, size = orc.decode(q, k8, v8, scale, table, lens, softcap, sums64)
    _, delta = kc.decode_bound(q, k8, scale, ref, size, torch.float16, 0.0)
    most = 0.0                                                    # the largest score of all
    for b, n in enumerate(lens):
        for h in range(H):
            rows = orc.rows_of(k8, scale, 0, table[b], h, n)
            if n:
                most = max(most, float((q[b, h * G: h * G + G].double().reshape(-1, D) @ rows.T).abs().max()) / math.sqrt(D))
    delta += min(most, softcap) * 2.0 ** -19
    assert delta < 2.0 ** -7
    bound = ref.abs() * kc.half_step(torch.float16) + size * (2.0 ** -11 + 2 * delta) + float(size.max()) * 2.0 ** -20
    off = (out.cpu().double() - ref).abs()
    assert bool((off <= bound).all()), (off / bound).max().item()
    assert bool(((dev.cpu().double() - sums64).abs() <= sums64 * (2 * delta + 2.0 ** -18)).all())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_tails_behind_a_strong_token(fa, codes, D):
    """Weights far below the largest add to the result as they add to the sum: one token takes nearly all of the weight and has no value, the others have 1000.

    Weights times V's scale are fp16 with 2^14 at least for the largest: 2^-28 of that is still a normal number, off by 2^-11."""
    B, n = 2400, 200                                              # (so many that a warp has whole sequences; they share their pages)
    top = orc.TOP[codes]
    k8, v8 = (torch.zeros(13, 1, 16, D) for _ in range(2))
    k8[0, 0, 0, 0] = top
    v8[:] = top
    v8[0, 0, 0] = 0
    scale = torch.empty(13, 1, 2)
    scale[..., 0], scale[..., 1] = 1 / top, 1000 / top
    k8, v8 = k8.to(codes), v8.to(codes)
    below = torch.tensor([18.0, 22.0, 25.5, 28.0])[torch.arange(B) % 4]
    q = torch.zeros(B, 1, 1, D)
    q[:, 0, 0, 0] = below * math.log(2) * math.sqrt(D)
    q = q.half()
    table = torch.arange(13).int()[None].expand(B, -1).contiguous()
    out = fa.forward_paged_decode_gqa_kv8(q.cuda(), k8.cuda(), v8.cuda(), scale.cuda(), table.cuda(), torch.full((B,), n).int().cuda(), 13)
    s = q[:, 0, 0, :1].double() * float(scale[0, 0, 0]) * top / math.sqrt(D)
    tails = (n - 1) * torch.exp(-s)
    ref = 1000.0 * tails / (1 + tails)
    delta = float(s.max()) * 2.0 ** -20 + 2.0 ** -18              # (one product; the factors' and the exponential's roundings)
    off = (out[:, 0, 0].cpu().double() - ref).abs()
    assert bool((off <= ref * (kc.half_step(torch.float16) + 2.0 ** -11 + 2 * delta)).all()), (off / ref).max().item()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("lens", [[100, 64, 17], [3000], [90] * 320], ids=["whole", "parts", "even"])
@pytest.mark.parametrize("power", [-92, -60, 60, 112])
def test_decode_of_values_near_the_ends_of_bfloat16(fa, codes, lens, power):
    """Values around 2^power, as an append stores them."""
    H, G, D = 1, 4, 64
    pages = sum((n + 15) // 16 for n in lens)
    table, _ = kc.tables(lens, pages, 136)
    state = kc.cache(pages, H, D, codes, 137)
    dev, ref = [t.cuda() for t in state], [t.clone() for t in state]
    g = torch.Generator().manual_seed(138)
    k, v = torch.randn(sum(lens), H, D, generator=g).bfloat16(), (torch.randn(sum(lens), H, D, generator=g) * 2.0 ** power).bfloat16()
    cu = _ints([0] + torch.tensor(lens).cumsum(0).tolist())
    fa.append_paged_kv8(k.cuda(), v.cuda(), *dev, table.cuda(), None, table.size(1), cu_seqlens=cu.cuda())
    orc.append(k, v, *ref, table, None, cu)
    q = torch.randn(len(lens), H * G, 1, D, generator=g).bfloat16()
    sums = torch.zeros(len(lens), H, table.size(1) * 16)
    got, sums64 = sums.cuda(), sums.double()
    out = fa.forward_paged_decode_gqa_kv8(q.cuda(), *dev, table.cuda(), _ints(lens).cuda(), table.size(1), mass=got)
    want, size = orc.decode(q, *ref, table, lens, mass=sums64)
    bound, delta = kc.decode_bound(q, ref[0], ref[2], want, size, torch.bfloat16, 0.0)
    off = (out.cpu().double() - want).abs()
    assert bool((off <= bound).all()), (off / bound).max().item()
    assert bool(((got.cpu().double() - sums64).abs() <= sums64 * (2 * delta + 2.0 ** -18)).all())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("lens", [[128, 100], [3000], [192] * 320], ids=["whole", "parts", "even"])
@pytest.mark.parametrize("order", ["rising", "falling", "zeros first", "zeros last", "heavy and small"])
def test_decode_of_pages_whose_scales_are_far_apart(fa, codes, lens, order):
    """Scales that rise or fall from page to page, pages of zero rows (2^-100, as an append makes them) beside others, and small values that take the weight from large ones."""
    H, G, D = 1, 4, 64
    pages = sum((n + 15) // 16 for n in lens)
    table, _ = kc.tables(lens, pages, 139)
    k8, v8, scale = kc.cache(pages, H, D, codes, 140)
    g = torch.Generator().manual_seed(141)
    q = torch.randn(len(lens), H * G, 1, D, generator=g).bfloat16()
    for b, n in enumerate(lens):
        own = table[b, : (n + 15) // 16].long()
        i = torch.arange(own.numel()).float() * (180.0 / own.numel())
        if order == "rising":
            scale[own, 0, 1] = torch.exp2(i - 90)
        elif order == "falling":
            scale[own, 0, 1] = torch.exp2(90 - i)
        elif order.startswith("zeros"):
            zero = own[:3] if order == "zeros first" else own[-3:]
            scale[zero, 0, 1] = 2.0 ** -100
            kc.bits(v8)[zero] = 0
        else:                                                     # every other page: 2^40 larger values, and scores 50 lower in base 2
            kc.bits(k8)[own[::2]] = 0
            kc.bits(k8)[own, :, :, 0] = 0x7F if codes == torch.int8 else 0x7E      # the largest code
            scale[own, 0, 0] = 1 / orc.TOP[codes]
            kc.bits(k8)[own[::2], :, :, 0] = 0
            scale[own[::2], 0, 1] = 2.0 ** 40
            scale[own[1::2], 0, 1] = 1.0
    if order == "heavy and small":
        q *= 0.125
        q[..., 0] = 50 * math.log(2) * math.sqrt(D)
    sums = torch.zeros(len(lens), H, table.size(1) * 16)
    got, sums64 = sums.cuda(), sums.double()
    out = fa.forward_paged_decode_gqa_kv8(q.cuda(), k8.cuda(), v8.cuda(), scale.cuda(), table.cuda(), _ints(lens).cuda(), table.size(1), mass=got)
    want, size = orc.decode(q, k8, v8, scale, table, lens, mass=sums64)
    bound, delta = kc.decode_bound(q, k8, scale, want, size, torch.bfloat16, 0.0)
    off = (out.cpu().double() - want).abs()
    assert bool((off <= bound).all()), (off / bound).max().item()
    assert bool(((got.cpu().double() - sums64).abs() <= sums64 * (2 * delta + 2.0 ** -18)).all())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("power", [-100, 0, 100])
def test_decode_of_queries_with_one_large_element(fa, codes, D, power):
    """Elements 2^22 below a bfloat16 row's largest keep their bits: the keys have nothing where the largest is, and the others decide the scores."""
    H, G, lens = 2, 4, [100, 64]
    table, _ = kc.tables(lens, 12, 142)
    k8, v8, scale = kc.cache(12, H, D, codes, 143)
    kc.bits(k8)[..., 5] = 0
    scale[..., 0] *= 2.0 ** -power
    small = (torch.randn(2, H * G, 1, D, generator=torch.Generator().manual_seed(144)) * 2.0 ** power).bfloat16()
    small[..., 5] = 0
    q = small.clone()
    q[..., 5] = 1.5 * 2.0 ** (22 + power)
    out = fa.forward_paged_decode_gqa_kv8(q.cuda(), k8.cuda(), v8.cuda(), scale.cuda(), table.cuda(), _ints(lens).cuda(), table.size(1))
    ref, size = orc.decode(small, k8, v8, scale, table, lens)
    _, delta = kc.decode_bound(small, k8, scale, ref, size, torch.bfloat16, 0.0)
    # an element is off by at most 2^-39 of the largest (half of fp16's least step, under a largest of 2^14 or more): D of them, each with the largest code
    delta += 1.5 * 2.0 ** (22 + power) * 2.0 ** -39 * D * orc.TOP[codes] * float(scale[..., 0].max()) / math.sqrt(D)
    assert delta < 2.0 ** -8
    bound = ref.abs() * kc.half_step(torch.bfloat16) + size * (2.0 ** -11 + 2 * delta) + float(size.max()) * 2.0 ** -20
    off = (out.cpu().double() - ref).abs()
    assert bool((off <= bound).all()), (off / bound).max().item()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("D,H,G,T", [(64, 1, 4, 64), (128, 2, 2, 100), (256, 1, 3, 70)])
def test_decode_of_many_rows(fa, codes, D, H, G, T):
    """Hundreds of rows of a KV head: many blocks, whose tokens see more and more of the last pages."""
    _decode_case(fa, codes, torch.float16, H, G, D, T, [0, 1, T, T + 30, 300], 145, mass=True)


def test_caches_of_more_than_32_bits(fa):
    """Pages whose codes lie beyond 2^32 bytes."""
    H, D, lens = 8, 256, [50]
    pages = (1 << 32) // (H * 16 * D) + 40
    table = _ints([[pages - 1, pages - 30, pages - 2, pages - 7]])
    k8, v8 = (torch.empty((pages, H, 16, D), dtype=torch.int8, device="cuda") for _ in range(2))
    scale = torch.empty((pages, H, 2), device="cuda")
    g = torch.Generator().manual_seed(73)
    k, v = (torch.randn(50, H, D, generator=g).half() for _ in range(2))
    fa.append_paged_kv8(k.cuda(), v.cuda(), k8, v8, scale, table.cuda(), None, 4, cu_seqlens=_ints([0, 50]).cuda())
    q = torch.randn(1, 16, 1, D, generator=g).half()
    out = fa.forward_paged_decode_gqa_kv8(q.cuda(), k8, v8, scale, table.cuda(), _ints(lens).cuda(), 4)
    mass = torch.rand(1, H, 64, generator=g)
    new = _ints([[pages - 12, pages - 3]])
    kept, _, _ = fa.evict_paged_kv8(mass.cuda(), k8, v8, scale, table.cuda(), _ints(lens).cuda(), 4, new.cuda(), 20, 2, 3)
    small = [torch.zeros((6, H, 16, D), dtype=torch.int8) for _ in range(2)] + [torch.zeros(6, H, 2)]
    near = _ints([[0, 1, 2, 3]])
    orc.append(k, v, *small, near, None, _ints([0, 50]))
    ref, size = orc.decode(q, *small, near, lens)
    bound, _ = kc.decode_bound(q, small[0], small[2], ref, size, torch.float16, 0.0)
    assert bool(((out.cpu().double() - ref).abs() <= bound).all())
    want, _, _ = orc.evict(mass, *small, near, lens, _ints([[4, 5]]), 20, 2, 3)
    assert torch.equal(kept.cpu(), want)
    for i, p in enumerate(new[0].tolist()):
        n = 16 if i == 0 else 4
        assert torch.equal(k8[p, :, :n].cpu(), small[0][4 + i, :, :n]) and torch.equal(v8[p, :, :n].cpu(), small[1][4 + i, :, :n])
        assert torch.equal(scale[p].cpu(), small[2][4 + i])


# ---- eviction -------------------------------------------------------------------------------------------------------
def _evict_case(fa, codes, H, D, lens, budget, sink, recent, seed, mass=None, index=None):
    new_pages = (budget + 15) // 16
    pages = sum((max(0, n) + 15) // 16 for n in lens) + new_pages * len(lens) + 2
    table, rest = kc.tables(lens, pages, seed)
    new = _ints([rest[b * new_pages: (b + 1) * new_pages] for b in range(len(lens))])
    state = kc.cache(pages, H, D, codes, seed + 1)
    if mass is None:
        g = torch.Generator().manual_seed(seed + 2)
        mass = torch.randn(len(lens), H, table.size(1) * 16, generator=g).exp()
        mass *= torch.rand(mass.shape, generator=g) > 0.2
    dev, ref = [t.cuda() for t in state], [t.clone() for t in state]
    got = fa.evict_paged_kv8(mass.cuda(), *dev, table.cuda(), _ints(lens).cuda(), table.size(1), new.cuda(), budget, sink, recent,
                             mass_index=None if index is None else index.cuda())
    want = orc.evict(mass, *ref, table, lens, new, budget, sink, recent, index)
    for a, b in zip(got[:2], want[:2]):
        assert torch.equal(a.cpu(), b)
    assert torch.equal(got[2].cpu().nan_to_num(-1.0), want[2].nan_to_num(-1.0))
    for a, b in zip(dev, ref):
        _same(a, b)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 0), (16, 4, 3), (50, 0, 50), (33, 33, 0), (100, 10, 17)])
def test_evict_sizes(fa, codes, D, budget, sink, recent):
    _evict_case(fa, codes, 2, D, LENS + [101, 99], budget, sink, recent, 80 + budget)


def test_evict_equal_sums_keep_the_first(fa):
    lens, H = [300, 2500], 2
    mass = torch.zeros(2, H, 2512)
    mass[:, 1] = torch.randint(0, 3, (2, 2512), generator=torch.Generator().manual_seed(81)).float()
    mass[0, 0, ::2] = -0.0
    _evict_case(fa, torch.int8, H, 64, lens, 130, 3, 20, 82, mass)


def test_evict_odd_sums(fa):
    """Negative sums, infinities and NaN have their places in the order too."""
    g = torch.Generator().manual_seed(83)
    mass = torch.randn(3, 1, 416, generator=g)
    mass[0, 0, ::7] = math.nan
    mass[1, 0, ::5] = math.inf
    mass[2, 0, ::3] = -math.inf
    mass[2, 0, 1::3] = -1e-42
    _evict_case(fa, torch.float8_e4m3fn, 1, 64, [400, 401, 390], 120, 2, 9, 84, mass)


@pytest.mark.parametrize("lens,budget", [([20000], 3001), ([9000, 8191, 40], 512), ([70000], 5)])
def test_evict_long_sequences(fa, lens, budget):
    """Rows that a cluster of CTAs shares."""
    _evict_case(fa, torch.int8, 2, 64, lens, budget, min(4, budget), 0, 85)


def test_evict_behind_a_table_of_very_many_pages(fa):
    """A table whose rows could hold more tokens than the clusters' shared memory has keys."""
    g = torch.Generator().manual_seed(91)
    lens, width = [3000, 700, 4100], 20600
    table, rest = kc.tables(lens, 520, 92, width=width)
    new = _ints([rest[b * 4: b * 4 + 4] for b in range(3)])
    state = kc.cache(520, 1, 64, torch.int8, 93)
    mass = torch.zeros(3, 1, width * 16)
    mass[:, :, :4200] = torch.randint(0, 50, (3, 1, 4200), generator=g).float()
    dev, ref = [t.cuda() for t in state], [t.clone() for t in state]
    got = fa.evict_paged_kv8(mass.cuda(), *dev, table.cuda(), _ints(lens).cuda(), width, new.cuda(), 60, 1, 9)
    want = orc.evict(mass, *ref, table, lens, new, 60, 1, 9)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
    for a, b in zip(dev, ref):
        _same(a, b)


def test_evict_rows_of_sums_by_index(fa):
    g = torch.Generator().manual_seed(86)
    _evict_case(fa, torch.int8, 2, 64, [100, 60, 80], 40, 1, 5, 87, torch.rand(7, 2, 128, generator=g), _ints([5, 0, 3]))


def test_evict_reports_rows_and_pages_outside(fa):
    H, D = 1, 64
    state = [t.cuda() for t in kc.cache(8, H, D, torch.int8, 88)]
    before = [t.clone() for t in state]
    mass = torch.rand(2, H, 32, generator=torch.Generator().manual_seed(89)).cuda()
    table, lens = _ints([[0, 1], [2, 3]]).cuda(), _ints([32, 32]).cuda()
    _, n, _ = fa.evict_paged_kv8(mass, *state, table, lens, 2, _ints([[4], [9]]).cuda(), 16, mass_index=_ints([2, 0]).cuda())
    assert n.tolist() == [0, 16]
    with pytest.raises(RuntimeError, match="outside the cache"):
        fa.check_async_errors()
    for a, b in zip(state, before):
        _same(a, b.cpu())


# ---- together ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("codes", CODES)
def test_prompts_steps_and_eviction_in_a_row(fa, codes):
    """A short service: prompts in, steps with sums, a cut, more steps on what is left, each held against the oracle on the oracle's own cache."""
    H, G, D, B, budget = 2, 4, 64, 3, 40
    lens = [70, 33, 50]
    pages = 40
    table, rest = kc.tables([96] * B, pages, 90, width=6)
    new = _ints([rest[i * 6: i * 6 + 6] for i in range(B)])
    state = kc.cache(pages, H, D, codes, 91)
    dev, ref = [t.cuda() for t in state], [t.clone() for t in state]
    g = torch.Generator().manual_seed(92)
    rnd = lambda *s: torch.randn(*s, generator=g).bfloat16()
    k, v = rnd(sum(lens), H, D), rnd(sum(lens), H, D)
    cu = _ints([0, 70, 103, 153])
    fa.append_paged_kv8(k.cuda(), v.cuda(), *dev, table.cuda(), None, 6, cu_seqlens=cu.cuda())
    orc.append(k, v, *ref, table, None, cu)
    mass, mass64 = torch.zeros(B, H, 96).cuda(), torch.zeros(B, H, 96, dtype=torch.float64)

    def steps(n, table, lens):
        for _ in range(n):
            k, v, q = rnd(B, H, 1, D), rnd(B, H, 1, D), rnd(B, H * G, 1, D)
            fa.append_paged_kv8(k.cuda(), v.cuda(), *dev, table.cuda(), _ints(lens).cuda(), 6)
            orc.append(k[:, :, 0], v[:, :, 0], *ref, table, _ints(lens))
            lens = [n + 1 for n in lens]
            out = fa.forward_paged_decode_gqa_kv8(q.cuda(), *dev, table.cuda(), _ints(lens).cuda(), 6, mass=mass)
            want, size = orc.decode(q, *ref, table, lens, mass=mass64)
            bound, _ = kc.decode_bound(q, ref[0], ref[2], want, size, torch.bfloat16, 0.0)
            assert bool(((out.cpu().double() - want).abs() <= bound).all())
        for got, want in zip(dev, ref):
            _same(got, want)
        return lens

    lens = steps(5, table, lens)
    sums = mass.cpu()
    assert bool(((sums.double() - mass64).abs() <= 1e-2 * mass64 + 1e-9).all())
    kept, new_lens, new_mass = fa.evict_paged_kv8(mass, *dev, table.cuda(), _ints(lens).cuda(), 6, new.cuda(), budget, 2, 8)
    want = orc.evict(sums, *ref, table, lens, new, budget, 2, 8)
    for a, b in zip((kept, new_lens, new_mass), want):
        assert torch.equal(a.cpu(), b)
    mass.zero_(); mass64.zero_()
    mass[:, :, :budget] = new_mass
    mass64[:, :, :budget] = new_mass.cpu().double()
    lens = steps(20, new, new_lens.tolist())
    assert lens == [60, 58, 60]


@pytest.mark.parametrize("codes", CODES)
def test_sums_of_many_steps(fa, codes):
    """Sums that twenty steps add to stay within what each step's scores and roundings allow."""
    H, G, D, lens = 2, 4, 128, [300, 33, 1]
    table, _ = kc.tables([n + 20 for n in lens], 40, 152)
    state = kc.cache(40, H, D, codes, 153)
    dev, ref = [t.cuda() for t in state], [t.clone() for t in state]
    g = torch.Generator().manual_seed(154)
    mass = torch.zeros(3, H, table.size(1) * 16).cuda()
    mass64, worst = mass.cpu().double(), 0.0
    for _ in range(20):
        k, v, q = (torch.randn(3, n, 1, D, generator=g).bfloat16() for n in (H, H, H * G))
        fa.append_paged_kv8(k.cuda(), v.cuda(), *dev, table.cuda(), _ints(lens).cuda(), table.size(1))
        orc.append(k[:, :, 0], v[:, :, 0], *ref, table, _ints(lens))
        lens = [n + 1 for n in lens]
        fa.forward_paged_decode_gqa_kv8(q.cuda(), *dev, table.cuda(), _ints(lens).cuda(), table.size(1), mass=mass)
        out, size = orc.decode(q, *ref, table, lens, mass=mass64)
        worst = max(worst, kc.decode_bound(q, ref[0], ref[2], out, size, torch.bfloat16, 0.0)[1])
    # a weight's score and the sum it is divided by, each off by `worst`; 2^-18 for logarithm and exponentials; a rounding of fp32 for each step
    assert bool(((mass.cpu().double() - mass64).abs() <= mass64 * (2 * worst + 2.0 ** -18 + 20 * 2.0 ** -24)).all())


def test_calls_on_another_stream_and_in_a_graph(fa):
    """A step captured once (append, attention with sums) and replayed with other inputs does what eager calls do, also beside a second graph on another stream."""
    H, G, D, B = 2, 4, 128, 4
    lens = [900, 33, 16, 250]
    pages = 100
    table, _ = kc.tables([n + 32 for n in lens], pages, 93)
    g = torch.Generator().manual_seed(94)
    rows = lambda: [torch.randn(B, n, 1, D, generator=g).half().cuda() for n in (H, H, H * G)]
    sets = []
    for i in range(2):
        dev = [t.cuda() for t in kc.cache(pages, H, D, torch.int8, 95 + i)]
        sets.append(dict(dev=dev, copy=[t.clone() for t in dev], k=rows(), lens=_ints(lens).cuda(), pos=(_ints(lens) - 1).cuda(),
                         mass=torch.zeros(B, H, table.size(1) * 16).cuda(), graph=torch.cuda.CUDAGraph(), stream=torch.cuda.Stream()))
    bt = table.cuda()

    def step(s, dev, mass):
        fa.append_paged_kv8(s["k"][0], s["k"][1], *dev, bt, s["pos"], bt.size(1))
        return fa.forward_paged_decode_gqa_kv8(s["k"][2], *dev, bt, s["lens"], bt.size(1), mass=mass)

    for s in sets:
        with torch.cuda.stream(s["stream"]):                      # first calls outside the capture
            step(s, [t.clone() for t in s["dev"]], s["mass"].clone())
            s["stream"].synchronize()
            with torch.cuda.graph(s["graph"], stream=s["stream"]):
                s["out"] = step(s, s["dev"], s["mass"])
    torch.cuda.synchronize()
    for round_ in range(3):
        fresh = [rows() for _ in sets]
        for s, f in zip(sets, fresh):
            for a, b in zip(s["k"], f):
                a.copy_(b)
        torch.cuda.synchronize()
        for s in sets:
            with torch.cuda.stream(s["stream"]):
                s["graph"].replay()
        torch.cuda.synchronize()
        for s in sets:
            mass = s.setdefault("mass2", torch.zeros_like(s["mass"]))
            out = step(s, s["copy"], mass)
            torch.cuda.synchronize()
            assert torch.equal(out, s["out"]) and torch.equal(mass, s["mass"])
            for a, b in zip(s["dev"], s["copy"]):
                assert torch.equal(kc.bits(a), kc.bits(b))
        for s in sets:
            s["lens"].add_(1); s["pos"].add_(1)


def test_calls_on_two_streams_at_once(fa):
    """Eager calls of two streams beside each other, each with a cache of its own, give what they give alone."""
    lens = [2000, 40, 700, 1]
    table, rest = kc.tables(lens, 400, 120)
    new = _ints([rest[i * 8: i * 8 + 8] for i in range(4)]).cuda()
    bt, n = table.cuda(), _ints(lens).cuda()
    g = torch.Generator().manual_seed(121)
    sets = [dict(dev=[t.cuda() for t in kc.cache(400, 2, 128, c, 122)], q=torch.randn(4, 8, 1, 128, generator=g).half().cuda(),
                 k=torch.randn(4, 2, 1, 128, generator=g).half().cuda(), s=torch.cuda.Stream()) for c in CODES]

    def run(s):
        dev, mass = [t.clone() for t in s["dev"]], torch.zeros(4, 2, table.size(1) * 16).cuda()
        for _ in range(5):
            fa.append_paged_kv8(s["k"], s["k"], *dev, bt, n - 1, bt.size(1))
            out = fa.forward_paged_decode_gqa_kv8(s["q"], *dev, bt, n, bt.size(1), mass=mass)
            kept, _, _ = fa.evict_paged_kv8(mass, *dev, bt, n, bt.size(1), new, 128, 2, 8)
        return dev + [mass, out, kept]

    alone = [[kc.bits(t).cpu() for t in run(s)] for s in sets]
    torch.cuda.synchronize()
    for _ in range(4):
        both = []
        for s in sets:
            with torch.cuda.stream(s["s"]):
                both.append(run(s))
        torch.cuda.synchronize()
        for got, want in zip(both, alone):
            assert all(torch.equal(kc.bits(a).cpu(), b) for a, b in zip(got, want))


FIRST_CALL_IN_A_GRAPH = """
import torch
import flash_attn_v100_b200 as fa
k8, v8 = (torch.ones(4, 2, 16, 64, dtype=torch.int8, device="cuda") for _ in range(2))
scale, table, lens = torch.ones(4, 2, 2, device="cuda"), torch.arange(4, device="cuda").int()[None], torch.full((1,), 50, device="cuda").int()
k, q = torch.full((1, 2, 1, 64), 2.0, device="cuda").half(), torch.zeros(1, 4, 1, 64, device="cuda").half()
mass, new = torch.zeros(1, 2, 64, device="cuda"), torch.arange(2, 4, device="cuda").int()[None]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    fa.append_paged_kv8(k, k, k8, v8, scale, table, lens - 1, 4)
    out = fa.forward_paged_decode_gqa_kv8(q, k8, v8, scale, table, lens, 4, mass=mass)
    kept, n, _ = fa.evict_paged_kv8(mass, k8, v8, scale, table[:, :2].contiguous(), lens - 18, 2, new, 20)
graph.replay()
torch.cuda.synchronize()
fa.check_async_errors()
assert torch.allclose(out.float(), torch.full_like(out, 1 + 1 / 50).float(), atol=1e-3), out
assert abs(mass.sum().item() - 4) < 1e-3 and n.item() == 20 and kept[0, 0].tolist() == list(range(20))
print("fine")
"""


def test_first_calls_of_a_process_inside_a_capture():
    run = subprocess.run([sys.executable, "-c", FIRST_CALL_IN_A_GRAPH], capture_output=True, text=True, timeout=120, cwd=ROOT)
    assert run.returncode == 0 and "fine" in run.stdout, run.stderr[-2000:]


def test_results_do_not_change_from_call_to_call(fa):
    lens = [3000, 17, 900]
    table, _ = kc.tables(lens, 260, 96)
    k8, v8, scale = (t.cuda() for t in kc.cache(260, 4, 128, torch.int8, 97))
    q = torch.randn(3, 16, 1, 128, generator=torch.Generator().manual_seed(98)).half().cuda()
    outs = []
    for _ in range(20):
        mass = torch.zeros(3, 4, table.size(1) * 16).cuda()
        outs.append((fa.forward_paged_decode_gqa_kv8(q, k8, v8, scale, table.cuda(), _ints(lens).cuda(), table.size(1), mass=mass), mass))
    assert all(torch.equal(a, outs[0][0]) and torch.equal(b, outs[0][1]) for a, b in outs)


def test_empty_calls(fa):
    k8, v8, scale = (t.cuda() for t in kc.cache(2, 1, 64, torch.int8, 99))
    table, none = torch.zeros((0, 1), dtype=torch.int32).cuda(), torch.zeros(0, dtype=torch.int32).cuda()
    assert fa.forward_paged_decode_gqa_kv8(torch.zeros(0, 1, 1, 64).half().cuda(), k8, v8, scale, table, none, 1).shape == (0, 1, 1, 64)
    fa.append_paged_kv8(*[torch.zeros(0, 1, 1, 64).half().cuda()] * 2, k8, v8, scale, table, none, 1)
    fa.append_paged_kv8(*[torch.zeros(0, 1, 64).half().cuda()] * 2, k8, v8, scale, torch.zeros((1, 1), dtype=torch.int32).cuda(), None, 1,
                        cu_seqlens=_ints([0, 0]).cuda())
    kept, n, m = fa.evict_paged_kv8(torch.zeros(1, 1, 16).cuda(), k8, v8, scale, table, none, 1, table, 16)
    assert kept.shape == (0, 1, 16) and n.numel() == 0 and m.shape == (0, 1, 16)


# ---- the cache class -------------------------------------------------------------------------------------------------
def test_cache_class_serves_and_evicts(fa):
    """Prompts, steps, a cut that leaves a shared prefix in place, and steps after it, against the operators' oracle."""
    H, G, D = 2, 2, 64
    c = fa.PagedKVCache8(64, 2, H, D, max_batch=4, max_blocks_per_seq=16, codes=torch.int8)
    g = torch.Generator().manual_seed(100)
    rnd = lambda *s: torch.randn(*s, generator=g).half().cuda()
    prompt = list(range(80))
    c.allocate("a", 80, prompt)
    cu = _ints([0, 80]).cuda()
    turn = lambda n: (torch.ones(n, D).cuda(), torch.zeros(n, D).cuda())      # no rotation
    for layer in range(2):
        q, k, v = rnd(80, H * G, D), rnd(80, H, D), rnd(80, H, D)
        _, kr = c.append_prefill(layer, ["a"], q, k, v, *turn(80), cu)
        assert torch.equal(kr, k)
    c.commit("a", 80)
    assert c.cache_prefix(prompt, "a") == 80
    c.allocate("b", 81, prompt + [7])
    assert c.get_cache_len("b") == 80 and c.position("b") == 80
    shared = c.get_block_table("b")[:5]
    assert shared == c.get_block_table("a")[:5]
    before = [t[shared].clone() for t in c.k_pools]

    def step(names):
        for r in names:
            c.reserve(r, c.get_cache_len(r) + 1)
        for layer in range(2):
            n = len(names)
            q, k, v = rnd(n, H * G, 1, D), rnd(n, H, 1, D), rnd(n, H, 1, D)
            q = c.append_decode(layer, names, q, k, v, *turn(n))
            out = c.attend(layer, names, q)
            state = [t.cpu() for t in (c.k_pools[layer], c.v_pools[layer], c.scales[layer])]
            lens = [c.get_cache_len(r) + 1 for r in names]
            table = torch.full((n, 16), -1, dtype=torch.int32)
            for i, r in enumerate(names):
                t = c.get_block_table(r)
                table[i, : len(t)] = _ints(t)
            ref, size = orc.decode(q.cpu(), *state, table, lens)
            bound, _ = kc.decode_bound(q.cpu(), state[0], state[2], ref, size, torch.float16, 0.0)
            assert bool(((out.cpu().double() - ref).abs() <= bound).all())
        for r in names:
            c.commit(r, 1)

    for _ in range(3):
        step(["b", "a"])
    free = c.get_num_free_blocks()
    freed = c.evict(["b"], 40, sink=4, recent=8)
    assert c.get_num_free_blocks() == free + freed and freed == 1 - 3          # five of b's six blocks are shared, three are new
    assert c.get_cache_len("b") == 40 and c.position("b") == 83
    assert all(torch.equal(t[shared], s) for t, s in zip(c.k_pools, before))
    assert c.cache_prefix(prompt, "b") == 0
    row = c.row_of("b")
    assert bool((c.masses[0][row, :, :40] > 0).any()) and bool((c.masses[0][row, :, 40:] == 0).all())
    for _ in range(3):
        step(["b", "a"])
    assert c.evict(["a", "b"], 100) == 0
    c.release("a"); c.release("b")
    assert c.get_num_free_blocks() == 64


@pytest.mark.parametrize("codes", CODES)
def test_cache_class_takes_rejected_guesses_back(fa, codes):
    """The sums after steps of guesses are those of the tokens that stay; bfloat16, rotated."""
    H, G, D = 2, 4, 64
    lens = {"a": 100, "b": 37}
    turn = lambda at: (torch.cos(at[:, None] * 0.01 * torch.arange(1, D // 2 + 1)), torch.sin(at[:, None] * 0.01 * torch.arange(1, D // 2 + 1)))

    def step(c, names, counts, rows, kept, small=None):
        for r in names:
            c.reserve(r, c.get_cache_len(r) + counts)
        at = torch.cat([torch.arange(counts) + c.position(r) for r in names]).float()
        cos, sin = (torch.cat((t, t), 1).cuda() for t in turn(at))
        cu = (torch.arange(len(names) + 1) * counts).int().cuda()
        for layer, (q, k, v) in enumerate(rows):
            q, k = c.append_prefill(layer, names, q.flatten(0, 1).contiguous(), k.flatten(0, 1).contiguous(), v.flatten(0, 1).contiguous(), cos, sin, cu)
            out = c.attend(layer, names, q.view(len(names), counts, H * G, D).transpose(1, 2).contiguous(), softcap=20.0)
            assert out.dtype == torch.bfloat16 and bool(out[:, :, 0].isfinite().all())
        for r in names:
            c.commit(r, kept[r])

    def run(guesses):
        c = fa.PagedKVCache8(40, 2, H, D, max_batch=3, max_blocks_per_seq=12, codes=codes)
        c.allocate("x", 16)                                       # (so that the batches' rows of the table are gathered)
        g = torch.Generator().manual_seed(150)
        rnd = lambda *s: torch.randn(*s, generator=g).bfloat16().cuda()
        for r, n in lens.items():
            c.allocate(r, n)
            step(c, [r], n, [[rnd(1, n, m, D) for m in (H * G, H, H)] for _ in range(2)], {r: n})
        for kept in ({"a": 1, "b": 3}, {"a": 4, "b": 0}, {"a": 2, "b": 1}):
            rows = [[rnd(2, 4, m, D) for m in (H * G, H, H)] for _ in range(2)]
            for layer in rows:
                for i, r in enumerate(("a", "b")):                # rejected rows ask for no larger scale
                    layer[1][i, kept[r]:] *= 1e-3
                    layer[2][i, kept[r]:] *= 1e-3
            if guesses:
                step(c, ["a", "b"], 4, rows, kept)
            else:
                for i, r in enumerate(("a", "b")):
                    if kept[r]:
                        step(c, [r], kept[r], [[t[i: i + 1, : kept[r]] for t in layer] for layer in rows], kept)
        return c

    got, want = run(True), run(False)
    for layer in range(2):
        # weights of one cache in calls of different batches: each off by 2^-17 at most (scores within 2^-18), the sums of a few of them by no more
        assert bool(((got.masses[layer] - want.masses[layer]).abs() <= want.masses[layer] * 2.0 ** -16).all())
        for r in lens:
            assert bool((got.masses[layer][got.row_of(r), :, got.get_cache_len(r):] == 0).all())
            own = torch.tensor(got.get_block_table(r))[: (got.get_cache_len(r) + 15) // 16]
            other = torch.tensor(want.get_block_table(r))[: own.numel()]
            assert torch.equal(got.scales[layer][own.cuda()], want.scales[layer][other.cuda()])
    assert got._guessed == {} and got.get_cache_len("a") == 107 and got.get_cache_len("b") == 41


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("bad", [40.0, math.nan])
def test_cache_class_gives_begun_blocks_back(fa, codes, bad):
    """Rejected rows that ask for a larger scale, or spoil a block: codes and scales are bit for bit those of a run without them."""
    H, D = 2, 128

    def run(guesses):
        c = fa.PagedKVCache8(40, 2, H, D, max_batch=3, max_blocks_per_seq=12, codes=codes)
        g = torch.Generator().manual_seed(151)
        rnd = lambda *s: torch.randn(*s, generator=g).half().cuda()
        turn = lambda n: (torch.ones(n, D).cuda(), torch.zeros(n, D).cuda())      # no rotation
        put = lambda layer, names, rows, cu: c.append_prefill(layer, names, *rows, *turn(rows[0].size(0)), _ints(cu).cuda())
        for r, n in (("a", 100), ("b", 37)):
            c.allocate(r, n)
            for layer in range(2):
                put(layer, [r], [rnd(n, m, D) for m in (2 * H, H, H)], [0, n])
            c.commit(r, n)
        for kept in ({"a": 1, "b": 2}, {"a": 0, "b": 3}, {"a": 5, "b": 0}):
            for r in "ab":
                c.reserve(r, c.get_cache_len(r) + 5)
            for layer in range(2):
                rows = [rnd(8, m, D) for m in (2 * H, H, H)]
                if guesses:
                    for t in rows[1:]:
                        t[kept["a"]: 5], t[5 + kept["b"]:] = bad, bad
                    put(layer, ["a", "b"], rows, [0, 5, 8])
                else:
                    for r, at in (("a", 0), ("b", 5)):
                        if kept[r]:
                            put(layer, [r], [t[at: at + kept[r]] for t in rows], [0, kept[r]])
            for r in "ab":
                c.commit(r, kept[r])
        return c

    got, want = run(True), run(False)
    for r in "ab":
        n = got.get_cache_len(r)
        assert n == want.get_cache_len(r)
        own, other = (torch.tensor(c.get_block_table(r)[: (n + 15) // 16]).cuda() for c in (got, want))
        for layer in range(2):
            assert torch.equal(got.scales[layer][own], want.scales[layer][other])
            for a, b in ((got.k_pools, want.k_pools), (got.v_pools, want.v_pools)):
                a, b = (kc.bits(t[layer])[at].transpose(1, 2).flatten(0, 1)[:n] for t, at in ((a, own), (b, other)))
                assert torch.equal(a, b)


# ---- the host side -------------------------------------------------------------------------------------------------
def test_native_host_side_and_python_do_the_same(fa, monkeypatch):
    from flash_attn_v100_b200 import kv8_ops
    H, D, lens = 2, 64, [70, 20]
    table, rest = kc.tables(lens, 16, 110)
    g = torch.Generator().manual_seed(111)
    k, v, q = (torch.randn(2, n, 1, D, generator=g).half().cuda() for n in (H, H, 4 * H))
    kp, vp = (torch.randn(25, H, D, generator=g).half().cuda() for _ in range(2))
    new, mass0 = _ints([rest[:2], rest[2:4]]).cuda(), torch.rand(3, H, table.size(1) * 16, generator=g).cuda()
    index, n = _ints([2, 0]).cuda(), _ints(lens).cuda()

    def run():
        dev = [t.cuda() for t in kc.cache(16, H, D, torch.float8_e4m3fn, 112)]
        bt, mass = table.cuda(), mass0.clone()
        fa.append_paged_kv8(kp, vp, *dev, bt, _ints([3, 0]).cuda(), bt.size(1), cu_seqlens=_ints([0, 20, 25]).cuda())
        fa.append_paged_kv8(k, v, *dev, bt, n - 1, bt.size(1))
        outs = [fa.forward_paged_decode_gqa_kv8(q, *dev, bt, n, bt.size(1)),
                fa.forward_paged_decode_gqa_kv8(q, *dev, bt, n, bt.size(1), softcap=7.0, mass=mass, mass_index=index)]
        outs += fa.evict_paged_kv8(mass, *dev, bt, n, bt.size(1), new, 30, 2, 4, mass_index=index)
        return [t.cpu() for t in outs + dev + [mass]]

    calls = []
    module = kv8_ops._native_module()
    assert module is not None
    native = kv8_ops._native
    monkeypatch.setattr(kv8_ops, "_native", lambda name, *a: calls.append((name, native(name, *a))) or calls[-1][1])
    fast = run()
    assert [name for name, _ in calls] == ["kv8_append", "kv8_append", "kv8_decode", "kv8_decode", "kv8_evict"] and all(r is not None for _, r in calls)
    monkeypatch.setattr(kv8_ops, "_native", lambda name, *a: None)
    slow = run()
    for a, b in zip(fast, slow):
        assert torch.equal(kc.bits(a), kc.bits(b))


def test_calls_that_do_not_fit_are_refused(fa):
    H, D = 2, 64
    k8, v8, scale = (t.cuda() for t in kc.cache(4, H, D, torch.int8, 113))
    table, n = _ints([[0, 1]]).cuda(), _ints([20]).cuda()
    q, k = torch.zeros(1, 4, 1, D).half().cuda(), torch.zeros(1, H, 1, D).half().cuda()
    mass, new = torch.zeros(1, H, 32).cuda(), _ints([[2, 3]]).cuda()
    decode = lambda q=q, k8=k8, v8=v8, scale=scale, table=table, n=n, width=2, **kw: fa.forward_paged_decode_gqa_kv8(q, k8, v8, scale, table, n, width, **kw)
    append = lambda k=k, v=k, n=n, **kw: fa.append_paged_kv8(k, v, k8, v8, scale, table, n, 2, **kw)
    evict = lambda mass=mass, new=new, budget=16, **kw: fa.evict_paged_kv8(mass, k8, v8, scale, table, n, 2, new, budget, **kw)
    for call, message in (
            (lambda: decode(q=q.float()), "q must be float16 or bfloat16"),
            (lambda: decode(q=q.transpose(1, 3)), "contiguous"),
            (lambda: decode(q=q[:, :3].contiguous()), "divisible"),
            (lambda: decode(q=torch.zeros(1, 4, 0, D).half().cuda()), "at least one token"),
            (lambda: decode(q=torch.zeros(2, 4, 1, D).half().cuda()), "block_table batch size"),
            (lambda: decode(q=torch.zeros(1, 4, 1, 128).half().cuda()), "head dimension must match"),
            (lambda: decode(k8=k8.half()), "int8 or float8_e4m3fn"),
            (lambda: decode(v8=v8.view(torch.float8_e4m3fn)), "dtype of k_cache"),
            (lambda: decode(v8=v8[:3].contiguous()), "same shape"),
            (lambda: decode(scale=scale[:, :, 0].contiguous()), "kv_scale must be"),
            (lambda: decode(table=table.long()), "2D int32"),
            (lambda: decode(width=0), "must be positive"),
            (lambda: decode(q=torch.zeros(2, 4, 1, D).half().cuda(), n=_ints([1, 1]).cuda(), table=_ints([[0], [1]]).cuda()), "row stride"),
            (lambda: decode(n=n.long()), "seq_lens must be"),
            (lambda: decode(softcap=-1.0), "softcap"),
            (lambda: decode(softcap=math.nan), "softcap"),
            (lambda: decode(softcap=1e-40), "softcap"),
            (lambda: decode(mass=mass[:, :, :31].contiguous()), "room for every token"),
            (lambda: decode(mass=mass.half()), "mass must be float32"),
            (lambda: decode(mass=mass[:0]), "row for each sequence"),
            (lambda: decode(mass_index=n), "goes with mass"),
            (lambda: decode(q=torch.zeros(1, 4, 40000, D).half().cuda()), "query rows"),
            (lambda: append(k=k.float(), v=k.float()), "k must be"),
            (lambda: append(v=k.bfloat16()), "dtype and shape of k"),
            (lambda: append(n=None), "positions is required"),
            (lambda: append(k=k[:, :1].contiguous(), v=k[:, :1].contiguous()), "match k_cache in heads"),
            (lambda: append(k=k.transpose(1, 3).contiguous().transpose(1, 3), v=k), "must be contiguous"),
            (lambda: append(k=k, cu_seqlens=_ints([0, 1]).cuda()), "3D"),
            (lambda: evict(budget=0), "budget"),
            (lambda: evict(budget=33), "room for budget"),
            (lambda: evict(sink=9, recent=8), "budget"),
            (lambda: evict(mass=mass[:, :1].contiguous()), "mass must be")):
        with pytest.raises(RuntimeError, match=message):
            call()
    rows = torch.zeros(3 * H * D + 4).half().cuda()
    with pytest.raises(RuntimeError, match="multiples of 16 bytes"):
        fa.append_paged_kv8(rows[4:].view(3, H, D), rows[4:].view(3, H, D), k8, v8, scale, table, None, 2, cu_seqlens=_ints([0, 3]).cuda())
