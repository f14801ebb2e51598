"""CPU: the C ABI of the paged 8-bit cache, refusals that need no device, the oracle against a plain form, and the cache class's bookkeeping."""
import ctypes
import math
import os
import re

import pytest
import torch

import kv8_cases as kc
from oracle import kv8_oracle as orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from flash_attn_v100_b200 import _lib
    from flash_attn_v100_b200.build import build
    build(library="kv8")
    return _lib.library("kv8")


def test_library_exports_every_declared_symbol(lib):
    from flash_attn_v100_b200 import _lib
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "fa_b200_kv8.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(fak_[a-z0-9_]+)\s*\(", text))
    assert names == set(_lib.KV8_SIGNATURES) and all(hasattr(lib, n) for n in names)


def _cache(**kw):
    from flash_attn_v100_b200 import _lib
    return _lib.Kv8Cache(**dict(dict(k=256, v=256, scale=256, pages=4, heads=2, dim=64, codes=0, table=256, width=2, max_pages=2), **kw))


def test_refusals_before_the_device(lib):
    p = ctypes.c_void_p(256)
    ref = ctypes.byref
    append = lambda c, k=p, stride=128, dtype=0, cu=None, batch=1, total=1: lib.fak_append_paged(ref(c), k, p, stride, stride, dtype, None, cu, batch, total, None)
    assert append(_cache(k=None)) == -1 and b"null" in lib.fak_last_error()
    assert append(_cache(dim=80)) == -2 and b"not built" in lib.fak_last_error()
    for bad in (dict(codes=2), dict(pages=0), dict(heads=0), dict(width=1), dict(max_pages=0), dict(k=260), dict(scale=260)):
        assert append(_cache(**bad)) == -1, bad
    assert append(_cache(), dtype=2) == -1 and append(_cache(), stride=120) == -1 and append(_cache(), stride=130) == -1
    assert append(_cache(), total=2) == -1 and append(_cache(), total=-1, cu=p) == -1
    assert append(_cache(), k=ctypes.c_void_p(264)) == -1 and append(_cache(), k=None) == -1
    assert append(_cache(), total=0, batch=0) == 0
    decode = lambda c, q_heads=4, tokens=1, cap=0.0, mass=None, rows=0, cap_m=0, ws=p, n=1 << 40, dtype=0: lib.fak_decode_paged(
        ref(c), p, p, p, 1, q_heads, tokens, dtype, cap, mass, None, rows, cap_m, ws, n, None)
    for bad in (dict(q_heads=3), dict(q_heads=0), dict(tokens=0), dict(cap=-1.0), dict(cap=1e-31), dict(cap=math.inf), dict(cap=math.nan), dict(mass=p), dict(ws=None), dict(n=16),
                dict(dtype=7), dict(ws=ctypes.c_void_p(264)), dict(tokens=65536)):
        assert decode(_cache(), **bad) == -1, bad
    assert b"query rows" in lib.fak_last_error()
    assert lib.fak_decode_workspace(ref(_cache()), 1, 3, 1, 0) == 0
    assert 0 < lib.fak_decode_workspace(ref(_cache()), 1, 4, 1, 0) < lib.fak_decode_workspace(ref(_cache()), 1, 4, 1, 1)
    evict = lambda c=_cache(), rows=1, width=1, budget=16, sink=0, recent=0, mass=p: lib.fak_evict_paged(
        ref(c), mass, None, rows, 32, p, 1, p, width, budget, sink, recent, p, p, p, None)
    for bad in (dict(budget=0), dict(budget=17), dict(sink=9, recent=8), dict(sink=-1), dict(rows=0), dict(mass=None)):
        assert evict(**bad) == -1, bad


def test_python_refusals():
    import flash_attn_v100_b200 as fa
    k8, v8, scale = kc.cache(2, 1, 64, torch.int8, 0)
    table, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 1, 64).half()
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        fa.forward_paged_decode_gqa_kv8(q, k8, v8, scale, table, n, 1)
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        fa.append_paged_kv8(q, q, k8, v8, scale, table, n, 1)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        fa.evict_paged_kv8(torch.zeros(1, 1, 16), k8, v8, scale, table, n, 1, table, 16)
    with pytest.raises(RuntimeError, match="must be a tensor"):
        fa.forward_paged_decode_gqa_kv8(None, k8, v8, scale, table, n, 1)


@pytest.mark.parametrize("codes", kc.CODES)
def test_oracle_append_is_near_the_rows(codes):
    """Every value comes back within half a step of its page's scale (a step and a half where codes were rounded again)."""
    table, _ = kc.tables([45, 20], 6, 1)
    state = kc.cache(6, 2, 64, codes, 2)
    g = torch.Generator().manual_seed(3)
    k, v = torch.randn(50, 2, 64, generator=g), torch.randn(50, 2, 64, generator=g)
    orc.append(k[:40], v[:40], *state, table, None, torch.tensor([0, 30, 40], dtype=torch.int32))
    orc.append(k[40:], v[40:], *state, table, torch.tensor([30, 10], dtype=torch.int32), torch.tensor([0, 5, 10], dtype=torch.int32))
    want = torch.cat((k[:30], k[40:45]))
    for h in range(2):
        got = orc.rows_of(state[0], state[2], 0, table[0], h, 35)
        a = want[:, h].double()
        if codes == torch.int8:
            limit = torch.full_like(a, 1.5 * float(state[2][table[0, :3].long(), h, 0].max()))
        else:
            limit = a.abs() * 2.0 ** -3 + 1e-3
        assert bool(((got - a).abs() <= limit).all())


def test_oracle_chooses_as_a_sort_does():
    g = torch.Generator().manual_seed(4)
    for n, budget, sink, recent in ((50, 20, 3, 5), (20, 20, 0, 0), (21, 20, 20, 0), (9, 1, 0, 0)):
        mass = torch.randint(0, 5, (n,), generator=g).float()
        got = orc.choose(mass.tolist(), n, budget, sink, recent)
        assert len(got) == min(n, budget) and got == sorted(set(got))
        if n > budget:
            assert set(range(sink)) <= set(got) and set(range(n - recent, n)) <= set(got)
            left = [i for i in range(sink, n - recent) if i not in got]
            taken = [i for i in range(sink, n - recent) if i in got]
            assert all((mass[i], -i) > (mass[j], -j) for i in taken for j in left)
    assert orc.choose([0.0, math.nan, 3.0, -0.0], 4, 2, 0, 0) == [1, 2]
    assert orc.choose([-0.0, 0.0, 0.0], 3, 1, 0, 0) == [0]


def test_cache_class_bookkeeping():
    from flash_attn_v100_b200 import PagedKVCache8
    c = PagedKVCache8(8, 1, 2, 64, max_batch=2, max_blocks_per_seq=4, device="cpu", codes=torch.float8_e4m3fn)
    assert c.k_pools[0].dtype == torch.float8_e4m3fn and c.scales[0].shape == (8, 2, 2) and c.masses[0].shape == (2, 2, 64)
    c.masses[0].fill_(1.0)
    row = c.allocate("a", 20)
    assert bool((c.masses[0][row] == 0).all())
    c.commit("a", 20)
    assert c.position("a") == c.get_cache_len("a") == 20
    assert c.evict(["a"], 20, 0, 0) == 0                          # nothing to cut: no kernel
    for bad in ((0, 0, 0), (10, 6, 5), (10, -1, 0)):
        with pytest.raises(ValueError):
            c.evict(["a"], *bad)
    with pytest.raises(ValueError, match="twice"):
        c.evict(["a", "a"], 10, 0, 0)
    c.allocate("b", 64)
    free = c.get_num_free_blocks()
    c.commit("b", 64)
    with pytest.raises(MemoryError):
        c.evict(["b"], 60, 0, 0)                                  # four new blocks are needed
    assert c.get_num_free_blocks() == free and c.get_cache_len("b") == 64
    c.release("a")
    with pytest.raises(RuntimeError):
        c.evict(["b"], 30, 0, 0)                                  # (no kernel on the CPU: the new blocks go back)
    assert c.get_num_free_blocks() == free + 2 and c.get_cache_len("b") == 64 and c.position("b") == 64
    with pytest.raises(KeyError):
        c.position("a")
    with pytest.raises(RuntimeError, match="no sums"):
        PagedKVCache8(8, 1, 2, 64, 2, 4, device="cpu", eviction=False).evict([], 10)
    with pytest.raises(ValueError):
        PagedKVCache8(8, 1, 2, 64, 2, 4, device="cpu", codes=torch.uint8)


@pytest.fixture
def on_cpu(monkeypatch):
    """The cache class with the oracle in the operators' place and no rotation."""
    from flash_attn_v100_b200 import kv8_ops, ops

    def append(k, v, k_cache, v_cache, scale, table, positions, width, cu_seqlens=None):
        flat = lambda t: t.reshape(-1, t.size(1), t.size(-1)) if cu_seqlens is None else t
        orc.append(flat(k), flat(v), k_cache, v_cache, scale, table, positions, cu_seqlens)

    def decode(q, k_cache, v_cache, scale, table, lens, width, softcap=0.0, mass=None, mass_index=None):
        sums = None if mass is None else mass.double()
        out, _ = orc.decode(q, k_cache, v_cache, scale, table, lens.tolist(), softcap, sums, mass_index)
        if mass is not None:
            mass.copy_(sums)
        return out.to(q.dtype)

    def evict(mass, k_cache, v_cache, scale, table, lens, width, new, budget, sink=0, recent=0, mass_index=None):
        return orc.evict(mass, k_cache, v_cache, scale, table, lens.tolist(), new, budget, sink, recent, mass_index)

    monkeypatch.setattr(kv8_ops, "append_paged_kv8", append)
    monkeypatch.setattr(kv8_ops, "forward_paged_decode_gqa_kv8", decode)
    monkeypatch.setattr(kv8_ops, "evict_paged_kv8", evict)
    monkeypatch.setattr(ops, "rope_append_paged_fp16", lambda q, k, *a, **kw: (q, k))
    return decode


def _serve(c, names, tokens, kept, g, small=1.0, spoiled=None):
    """One step of `tokens` new tokens of each request, of which kept[name] stay; rows that do not are `small` times as large as others, and the query of
    token `spoiled` is NaN."""
    H, G, D = c.num_kv_heads, 2, c.head_dim
    for r in names:
        c.reserve(r, c.get_cache_len(r) + tokens)
    factor = torch.ones(len(names), tokens)
    for i, r in enumerate(names):
        factor[i, kept[r]:] = small
    for layer in range(c.num_layers):
        q, k, v = (torch.randn(len(names) * tokens, n, D, generator=g).half() for n in (H * G, H, H))
        k, v = ((t * factor.reshape(-1, 1, 1)).half() for t in (k, v))
        cu = torch.arange(0, len(names) * tokens + 1, tokens, dtype=torch.int32)
        q, k = c.append_prefill(layer, names, *(t.to(c.device) for t in (q, k, v)), None, None, cu.to(c.device))
        q = q.view(len(names), tokens, H * G, D).transpose(1, 2).contiguous()
        if spoiled is not None:
            q[:, :, spoiled] = math.nan
        c.attend(layer, names, q)
    for r in names:
        c.commit(r, kept[r])


def test_weights_of_rejected_guesses_are_taken_back(on_cpu):
    """Steps of four guesses, of which some stay, leave the sums that the tokens that stay have given alone; also slots that are written again, and a NaN."""
    from flash_attn_v100_b200 import PagedKVCache8
    lens = {"a": 20, "b": 33}

    def run(guesses):
        c = PagedKVCache8(20, 2, 2, 64, max_batch=3, max_blocks_per_seq=6, device="cpu")
        g = torch.Generator().manual_seed(7)
        for r, n in lens.items():
            c.allocate(r, n)
            _serve(c, [r], n, {r: n}, g)
        c.allocate("c", 16)                                       # (a row that nobody touches)
        c.masses[1][c.row_of("c")] = 3.0
        for step, kept in enumerate(({"a": 1, "b": 3}, {"a": 4, "b": 0}, {"a": 0, "b": 1}, {"a": 2, "b": 4})):
            g = torch.Generator().manual_seed(step)
            if guesses:
                _serve(c, ["a", "b"], 4, kept, g, small=1e-3, spoiled=3 if step == 0 else None)
            else:
                # the same tokens, but those that do not stay are never there: a request at a time
                H, G, D = 2, 2, 64
                drawn = [[torch.randn(8, n, D, generator=g).half().view(2, 4, n, D) for n in (H * G, H, H)] for _ in range(2)]
                for i, r in enumerate(("a", "b")):
                    n = kept[r]
                    if n == 0:
                        continue
                    c.reserve(r, c.get_cache_len(r) + n)
                    for layer in range(2):
                        q, k, v = (t[i, :n] for t in drawn[layer])
                        c.append_prefill(layer, [r], q, k, v, None, None, torch.tensor([0, n], dtype=torch.int32))
                        c.attend(layer, [r], q.transpose(0, 1)[None].contiguous())
                    c.commit(r, n)
        return c

    got, want = run(True), run(False)
    assert got._guessed == {} and got.get_cache_len("a") == want.get_cache_len("a") == 27
    for layer in range(2):
        assert bool(got.masses[layer].isfinite().all())
        # the class's sums are fp32: of about ten additions each is off by at most 2^-24 of a sum; the codes are the same, as rejected rows are small
        assert bool(((got.masses[layer] - want.masses[layer]).abs() <= want.masses[layer] * 2.0 ** -20).all())
        for r, n in (("a", 27), ("b", 41)):
            assert bool((got.masses[layer][got.row_of(r), :, n:] == 0).all())
    got.release("a")
    assert "a" not in got._guessed


def test_an_eviction_drops_what_was_not_committed(on_cpu):
    from flash_attn_v100_b200 import PagedKVCache8
    c = PagedKVCache8(20, 1, 2, 64, max_batch=1, max_blocks_per_seq=6, device="cpu")
    g = torch.Generator().manual_seed(8)
    c.allocate("a", 40)
    _serve(c, ["a"], 40, {"a": 40}, g)
    sums = c.masses[0].clone()
    c.reserve("a", 43)
    q, k, v = (torch.randn(3, n, 64, generator=g).half() for n in (4, 2, 2))
    c.append_prefill(0, ["a"], q, k, v, None, None, torch.tensor([0, 3], dtype=torch.int32))
    c.attend(0, ["a"], q.transpose(0, 1)[None].contiguous())
    assert not torch.equal(c.masses[0], sums)
    c.evict(["a"], 20, 2, 4)
    kept = torch.tensor([orc.choose(sums[0, h].tolist(), 40, 20, 2, 4) for h in range(2)])
    assert torch.equal(c.masses[0][0, :, :20], sums[0].gather(1, kept)) and bool((c.masses[0][0, :, 20:] == 0).all()) and c._guessed == {}


@pytest.mark.parametrize("bad", [30.0, math.inf, math.nan])
def test_rejected_guesses_leave_no_trace_in_their_blocks(on_cpu, bad):
    """Rows that do not stay and ask for a larger scale, or spoil a block, leave codes, scales and sums as they are without them; also where a request is evicted instead."""
    from flash_attn_v100_b200 import PagedKVCache8
    H, D = 2, 64

    def run(guesses):
        c = PagedKVCache8(20, 2, H, D, max_batch=2, max_blocks_per_seq=6, device="cpu", codes=torch.float8_e4m3fn)
        for r, n in (("a", 20), ("b", 37)):
            c.allocate(r, n)
            _serve(c, [r], n, {r: n}, torch.Generator().manual_seed(n))
        cu = torch.tensor([0, 5, 8], dtype=torch.int32)
        for step, kept in enumerate(({"a": 1, "b": 2}, {"a": 0, "b": 3}, {"a": 5, "b": 0})):
            g = torch.Generator().manual_seed(step)
            rows = [[torch.randn(8, n, D, generator=g).half() for n in (2 * H, H, H)] for _ in range(2)]
            for r in ("a", "b"):
                c.reserve(r, c.get_cache_len(r) + 5)
            for layer in range(2):
                if guesses:
                    q, k, v = (t.clone() for t in rows[layer])
                    for t in (k, v):
                        t[kept["a"]: 5], t[5 + kept["b"]:] = bad, bad
                    c.append_prefill(layer, ["a", "b"], q, k, v, None, None, cu)
                    v.zero_()                                     # (the caller's rows may change behind the call)
                else:
                    for r, at in (("a", 0), ("b", 5)):
                        q, k, v = (t[at: at + kept[r]] for t in rows[layer])
                        if kept[r]:
                            c.append_prefill(layer, [r], q, k, v, None, None, torch.tensor([0, kept[r]], dtype=torch.int32))
            cu.zero_()                                            # (so may its offsets)
            for r in ("a", "b"):
                c.commit(r, kept[r])
            cu.copy_(torch.tensor([0, 5, 8]))
        return c

    got, want = run(True), run(False)
    assert got._appended == {} and [got.get_cache_len(r) for r in "ab"] == [want.get_cache_len(r) for r in "ab"] == [26, 42]
    for layer in range(2):
        for r in "ab":
            n = got.get_cache_len(r)
            blocks = [c.get_block_table(r)[: (n + 15) // 16] for c in (got, want)]
            for i, name in enumerate(("k_pools", "v_pools")):
                for h in range(H):
                    a, b = (orc.rows_of(getattr(c, name)[layer], c.scales[layer], i, t, h, n) for c, t in zip((got, want), blocks))
                    assert torch.equal(a, b)
            assert torch.equal(got.scales[layer][blocks[0]], want.scales[layer][blocks[1]])
    # tokens that were appended to begun blocks and not committed are gone with an eviction
    c = got
    c.reserve("a", 28)
    rows = [torch.full((2, n, D), bad).half() for n in (2 * H, H, H)]
    for layer in range(2):
        c.append_prefill(layer, ["a"], *rows, None, None, torch.tensor([0, 2], dtype=torch.int32))
    c.evict(["a"], 25, 1, 20)
    t = c.get_block_table("a")
    assert bool(c.scales[0][t].isfinite().all()) and float(c.scales[0][t].max()) < 0.03      # (30 / 448 is more)


def test_an_eviction_that_fails_leaves_the_sums(on_cpu, monkeypatch):
    """A layer that fails behind others: sums, tokens and blocks of all layers are as they were, and a second try cuts as if there had been no first."""
    from flash_attn_v100_b200 import PagedKVCache8, kv8_ops
    c = PagedKVCache8(20, 3, 2, 64, max_batch=2, max_blocks_per_seq=6, device="cpu")
    for r, n in (("a", 40), ("b", 57)):
        c.allocate(r, n)
        _serve(c, [r], n, {r: n}, torch.Generator().manual_seed(n))
    before, free, tables = [m.clone() for m in c.masses], c.get_num_free_blocks(), [c.get_block_table(r) for r in "ab"]
    evict, calls = kv8_ops.evict_paged_kv8, []

    def failing(*a, **kw):
        calls.append(a)
        if len(calls) == 2:
            raise torch.OutOfMemoryError("no room for the second layer")
        return evict(*a, **kw)

    monkeypatch.setattr(kv8_ops, "evict_paged_kv8", failing)
    with pytest.raises(torch.OutOfMemoryError):
        c.evict(["a", "b"], 20, 2, 4)
    assert all(torch.equal(m, b) for m, b in zip(c.masses, before)) and c.get_num_free_blocks() == free
    assert [c.get_block_table(r) for r in "ab"] == tables and (c.get_cache_len("a"), c.get_cache_len("b")) == (40, 57)
    c.evict(["a", "b"], 20, 2, 4)
    for layer in range(3):
        for row, n in ((c.row_of("a"), 40), (c.row_of("b"), 57)):
            kept = torch.tensor([orc.choose(before[layer][row, h].tolist(), n, 20, 2, 4) for h in range(2)])
            assert torch.equal(c.masses[layer][row, :, :20], before[layer][row].gather(1, kept)) and bool((c.masses[layer][row, :, 20:] == 0).all())


def test_an_eviction_of_a_nearly_full_cache_goes_in_turns(on_cpu):
    """Blocks that the first requests give back are those that the next ones move to; where even that does not do, nothing is touched."""
    from flash_attn_v100_b200 import PagedKVCache8
    lens = {"a": 90, "b": 96, "c": 81, "d": 30}

    def filled(blocks):
        c = PagedKVCache8(blocks, 2, 2, 64, max_batch=4, max_blocks_per_seq=6, device="cpu")
        for r, n in lens.items():
            c.allocate(r, n)
            _serve(c, [r], n, {r: n}, torch.Generator().manual_seed(n))
        return c

    got, want = filled(22), filled(60)                            # 20 blocks are held, a cut request takes two
    assert got.evict(list("abcd"), 32, 2, 8) == want.evict(list("abcd"), 32, 2, 8) == 12
    assert got.get_num_free_blocks() == 14 and sum(got._refs) == 8 and sorted(got._free + [b for r in lens for b in got.get_block_table(r)]) == list(range(22))
    for r, n in lens.items():
        n = min(n, 32)
        assert got.get_cache_len(r) == n and got.position(r) == lens[r]
        tables = [c.get_block_table(r) for c in (got, want)]
        assert got.block_table[got.row_of(r)].tolist() == tables[0] + [-1] * (6 - len(tables[0]))
        for layer in range(2):
            assert torch.equal(got.masses[layer], want.masses[layer])
            for i, name in enumerate(("k_pools", "v_pools")):
                a, b = (orc.rows_of(getattr(c, name)[layer], c.scales[layer], i, t, 1, n) for c, t in zip((got, want), tables))
                assert torch.equal(a, b)
    # four blocks for a request and two free ones; and blocks that a prefix holds do not come free
    c = filled(22)
    state = lambda: (c._free[:], {r: c.get_block_table(r) for r in lens}, [m.clone() for m in c.masses])
    before = state()
    with pytest.raises(MemoryError):
        c.evict(list("abcd"), 50, 2, 8)
    assert c.cache_prefix(list(range(90)), "a") == 80
    with pytest.raises(MemoryError):
        c.evict(["a", "b"], 32, 2, 8)
    after = state()
    assert after[:2] == before[:2] and all(torch.equal(x, y) for x, y in zip(after[2], before[2]))
    assert c.evict(["b", "a"], 32, 2, 8) == 4 - 1                  # five of a's six blocks stay held by the prefix


def test_sizes_beyond_32_bits_are_refused(monkeypatch):
    """What the C ABI takes as 32-bit numbers would be cut off: refused before a call (shapes only, no memory)."""
    from flash_attn_v100_b200 import _lib, kv8_ops
    for name in ("_check_input", "_same_device"):
        monkeypatch.setattr(kv8_ops, name, lambda *a: None)
    monkeypatch.setattr(kv8_ops, "_native", lambda *a: None)
    monkeypatch.setattr(_lib, "library", lambda name: pytest.fail("called"))
    meta = lambda shape, dtype: torch.empty(shape, dtype=dtype, device="meta")
    k8, scale, lens = meta((4, 2, 16, 64), torch.int8), meta((4, 2, 2), torch.float32), meta(1, torch.int32)
    table, mass, new = meta((1, 2), torch.int32), meta((1, 2, 32), torch.float32), meta((1, 1), torch.int32)
    big = 2 ** 32 + 64
    evict = lambda mass=mass, width=2, new=new, budget=16: kv8_ops.evict_paged_kv8(mass, k8, k8, scale, table, lens, width, new, budget)
    for call, message in ((lambda: evict(mass=meta((1, 2, big), torch.float32)), "fewer than 2.31 rows"),
                          (lambda: evict(mass=meta((big, 2, 32), torch.float32)), "fewer than 2.31 rows"),
                          (lambda: evict(new=meta((1, big), torch.int32)), "below 2.31"),
                          (lambda: evict(new=meta((1, big), torch.int32), budget=big), "below 2.31"),
                          (lambda: evict(width=big), "below 2.31")):
        with pytest.raises(RuntimeError, match=message):
            call()
