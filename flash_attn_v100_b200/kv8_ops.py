"""Operators on a paged cache in 8 bits (include/fa_b200_kv8.h): what writes it, what reads it and what makes it shorter.

The cache keeps 16 tokens a page: k_cache and v_cache [pages, H_KV, 16, D], int8 (codes -127..127) or float8_e4m3fn (none of them NaN), and kv_scale [pages, H_KV, 2]
fp32 with a scale for each page, head and kind (0: keys, 1: values), from 0 up; a code stands for code * scale.  D is 64, 128 or 256.  block_table [B, *] int32
with row stride `max_num_blocks` holds a sequence's pages in order, as in `forward_paged_decode_gqa_fp16`.  q, k, v are float16 or bfloat16.

Calls go to the current stream of the tensors' device and can be captured in CUDA graphs; there is no CPU path.  A page outside the
cache is never touched, the kernels record it: `check_async_errors` raises."""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import (PAGE_BLOCK_SIZE, SUPPORTED_D, _check_dim, _check_gqa_heads, _check_input, _chk, _native_module, _on, _ptr, _same_device, _stream_ptr,
                  _UNSET)

_ROWS = {torch.float16: 0, torch.bfloat16: 1}
_CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}
_INT = 2 ** 31 - 1      # the C ABI's sizes
_call_mod = _UNSET


def _kv8():
    return _lib.library("kv8")


def _native(name, *args):
    """The call `name` of the native host side (csrc/host/call.cpp); None where the call is anything but the plain case, which the wrappers below then look at."""
    global _call_mod
    if _call_mod is _UNSET:
        module = _native_module()
        if module is not None:
            _lib.bind_kv8(module)
        _call_mod = module
    return None if _call_mod is None else getattr(_call_mod, name)(*args)


def _rc(rc):
    if rc != 0:
        _lib.check(rc, "kv8")


def _cache(k_cache, v_cache, kv_scale, block_table, batch, max_num_blocks):
    """The checked cache as the C ABI takes it."""
    for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache"), (kv_scale, "kv_scale"), (block_table, "block_table")):
        _check_input(t, n)
        _same_device(k_cache, t, "k_cache", n)
    _chk(k_cache.dtype in _CODES, "k_cache must be int8 or float8_e4m3fn")
    _chk(v_cache.dtype == k_cache.dtype, "v_cache must have the dtype of k_cache")
    _check_dim(k_cache, 4, "k_cache")
    _chk(k_cache.shape == v_cache.shape, "k_cache and v_cache must have the same shape")
    pages, heads, page, dim = k_cache.shape
    _chk(page == PAGE_BLOCK_SIZE, "k_cache block size mismatch")
    _chk(dim in SUPPORTED_D, f"head dimension {dim} is not built (64, 128, 256)")
    _chk(kv_scale.dtype == torch.float32 and tuple(kv_scale.shape) == (pages, heads, 2), "kv_scale must be float32 [pages, H_KV, 2]")
    _chk(block_table.dtype == torch.int32 and block_table.dim() == 2, "block_table must be a 2D int32 tensor")
    _chk(block_table.size(0) >= batch, "block_table batch size must match")
    max_num_blocks = int(max_num_blocks)
    _chk(0 < max_num_blocks <= _INT, "max_num_blocks must be positive and below 2^31")
    used = min(max_num_blocks, block_table.size(1))
    _chk(used > 0 and (batch - 1) * max_num_blocks + used <= block_table.numel(), "max_num_blocks (row stride) is larger than block_table allows")
    return _lib.Kv8Cache(k=_ptr(k_cache), v=_ptr(v_cache), scale=_ptr(kv_scale), pages=pages, heads=heads, dim=dim, codes=_CODES[k_cache.dtype],
                         table=_ptr(block_table), width=max_num_blocks, max_pages=used)


def _ints(t, name, n, like):
    _check_input(t, name)
    _chk(t.dtype == torch.int32 and t.dim() == 1 and t.numel() == n, f"{name} must be int32 [{n}]")
    _same_device(like, t, "k_cache", name)


def _token_rows(t, name, tokens, heads, dim):
    """Elements from token to token of [tokens, heads, dim] whose heads are contiguous: a part of a fused projection's rows is one too."""
    _chk(t.stride(-1) == 1 and (heads == 1 or t.stride(1) == dim), f"{name}: the heads of a token must be contiguous")
    stride = t.stride(0) if tokens > 1 else heads * dim
    _chk(stride >= heads * dim and stride % 8 == 0 and t.data_ptr() % 16 == 0, f"{name}: rows of a token must start at multiples of 16 bytes and not overlap")
    return stride


def append_paged_kv8(k, v, k_cache, v_cache, kv_scale, block_table, positions, max_num_blocks, cu_seqlens=None):
    """New keys and values into the pages of an 8-bit cache, in place.

    Decode step (cu_seqlens is None): k, v [B,H_KV,1,D]; positions [B] int32 = slot of the new token.  Packed prompts: k, v [total,H_KV,D],
    cu_seqlens [B+1] int32; token j of sequence s is stored at slot positions[s] + j (positions None = 0).  A sequence
    with a negative position is left out (padded batches; attention takes a seq_len of 0 for it).  The tokens of k and v may be any
    multiple of 8 elements apart (slices of a fused projection).  Per page, head and kind: the scale is the largest magnitude of its rows / 127
    (e4m3: 448), at least 2^-100.  Where a page goes on being filled its scale only grows, and the codes it has are then rounded again.  NaN and
    infinities make a page's scale infinite, and what attends to it NaN.  Two sequences of a call must not write to the same page."""
    if _native("kv8_append", k, v, k_cache, v_cache, kv_scale, block_table, positions, max_num_blocks, cu_seqlens):
        return
    _chk(isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor), "k and v must be tensors")
    _chk(k.is_cuda and v.is_cuda, "k and v must be CUDA tensors")
    _chk(k.dtype in _ROWS, "k must be float16 or bfloat16")
    _chk(v.dtype == k.dtype and v.shape == k.shape, "v must have the dtype and shape of k")
    _same_device(k, k_cache, "k", "k_cache"); _same_device(k, v, "k", "v")
    if cu_seqlens is None:
        _check_dim(k, 4, "k")
        _chk(k.size(2) == 1, "k sequence length must be 1 for a decode step")
        _chk(positions is not None, "positions is required for a decode step")
        tokens, heads, _, dim = k.shape
        batch = tokens
    else:
        _check_dim(k, 3, "k")
        tokens, heads, dim = k.shape
        _check_input(cu_seqlens, "cu_seqlens")
        _chk(cu_seqlens.dim() == 1 and cu_seqlens.numel() > 0, "cu_seqlens must be a 1D int32 tensor")
        batch = cu_seqlens.numel() - 1
        _ints(cu_seqlens, "cu_seqlens", batch + 1, k_cache)
    if positions is not None:
        _ints(positions, "positions", batch, k_cache)
    c = _cache(k_cache, v_cache, kv_scale, block_table, batch, max_num_blocks)
    _chk((heads, dim) == (c.heads, c.dim), "k must match k_cache in heads and head dimension")
    if tokens == 0 or batch == 0:
        return
    ks, vs = _token_rows(k, "k", tokens, heads, dim), _token_rows(v, "v", tokens, heads, dim)
    with _on(k.device):
        _rc(_kv8().fak_append_paged(ctypes.byref(c), _ptr(k), _ptr(v), ks, vs, _ROWS[k.dtype], None if positions is None else _ptr(positions),
                                    None if cu_seqlens is None else _ptr(cu_seqlens), batch, tokens, _stream_ptr(k.device)))


def _check_mass(mass, mass_index, batch, c, like):
    _check_input(mass, "mass")
    _same_device(like, mass, "k_cache", "mass")
    _chk(mass.dtype == torch.float32 and mass.dim() == 3 and mass.size(1) == c.heads, "mass must be float32 [rows, H_KV, tokens]")
    _chk(max(mass.size(0), mass.size(2)) <= _INT, "mass must have fewer than 2^31 rows and tokens")
    _chk(mass.size(2) >= c.max_pages * PAGE_BLOCK_SIZE, "mass must have room for every token of a block_table row")
    if mass_index is None:
        _chk(mass.size(0) >= batch, "mass must have a row for each sequence")
    else:
        _ints(mass_index, "mass_index", batch, like)
        _chk(mass.size(0) > 0, "mass must have a row for each sequence")


def forward_paged_decode_gqa_kv8(q, k_cache, v_cache, kv_scale, block_table, seq_lens, max_num_blocks, softcap=0.0, mass=None, mass_index=None):
    """Attention of the newest T tokens of each sequence on a paged 8-bit cache.

    q [B,H_Q,T,D], seq_lens [B] int32 (the T tokens counted in) -> new [B,H_Q,T,D].  Token t sees the keys before seq_len - T + t + 1 and is what those
    make it, whatever the scales of pages behind them; one that sees none gets zeros.  With softcap > 0 a score x becomes softcap * tanh(x / softcap).  `mass` [rows,H_KV,tokens] fp32: what every key
    is given by the softmax, summed over the query heads of its KV head and the T tokens, is added in place to row mass_index[b] (None: b); the
    rows of a call must be different ones.  It takes 4 bytes of scratch for every query row and token that a block_table row has room for."""
    done = _native("kv8_decode", q, k_cache, v_cache, kv_scale, block_table, seq_lens, max_num_blocks, softcap, mass, mass_index)
    if done is not None:
        return done
    _check_input(q, "q")
    _check_dim(q, 4, "q")
    _chk(q.dtype in _ROWS, "q must be float16 or bfloat16")
    batch, H_Q, T, D = q.shape
    c = _cache(k_cache, v_cache, kv_scale, block_table, batch, max_num_blocks)
    _same_device(q, k_cache, "q", "k_cache")
    _check_gqa_heads(H_Q, c.heads)
    _chk(D == c.dim, "k_cache head dimension must match q")
    _chk(T > 0, "q must have at least one token")
    _ints(seq_lens, "seq_lens", batch, k_cache)
    softcap = float(softcap)
    _chk(softcap == 0.0 or 1e-30 <= softcap <= 1e30, "softcap must be 0 or from 1e-30 to 1e30")
    if mass is not None:
        _check_mass(mass, mass_index, batch, c, k_cache)
    else:
        _chk(mass_index is None, "mass_index goes with mass")
    lib = _kv8()
    with _on(q.device):
        out = torch.empty_like(q)
        if batch == 0:
            return out
        ws = torch.empty(lib.fak_decode_workspace(ctypes.byref(c), batch, H_Q, T, mass is not None), dtype=torch.uint8, device=q.device)
        _rc(lib.fak_decode_paged(ctypes.byref(c), _ptr(q), _ptr(out), _ptr(seq_lens), batch, H_Q, T, _ROWS[q.dtype], softcap,
                                 None if mass is None else _ptr(mass), None if mass_index is None else _ptr(mass_index),
                                 0 if mass is None else mass.size(0), 0 if mass is None else mass.size(2), _ptr(ws), ws.numel(), _stream_ptr(q.device)))
    return out


def evict_paged_kv8(mass, k_cache, v_cache, kv_scale, block_table, seq_lens, max_num_blocks, new_block_table, budget, sink=0, recent=0, mass_index=None):
    """The tokens of each sequence that matter most, head by head, into new pages.

    Of a sequence with more than `budget` tokens every KV head keeps the first `sink`, the last `recent`, and of the rest those with the largest
    mass (NaN above all, ties to the lowest index); a shorter one keeps all.  They go in order to the pages of new_block_table [B, >= budget / 16]
    int32, which must be none of the pages that block_table's rows hold: those are left as they were.  A new page's scale is the largest of its tokens', and
    codes from a smaller one are rounded again.  mass as in `forward_paged_decode_gqa_kv8`.  Returns (indices kept [B,H_KV,budget] int32, -1 behind
    the last; new seq_lens [B] int32; their mass [B,H_KV,budget] fp32, 0 behind the last)."""
    done = _native("kv8_evict", mass, k_cache, v_cache, kv_scale, block_table, seq_lens, max_num_blocks, new_block_table, budget, sink, recent, mass_index)
    if done is not None:
        return done
    _chk(isinstance(seq_lens, torch.Tensor) and seq_lens.dim() == 1, "seq_lens must be a 1D tensor")
    batch = seq_lens.numel()
    c = _cache(k_cache, v_cache, kv_scale, block_table, batch, max_num_blocks)
    _ints(seq_lens, "seq_lens", batch, k_cache)
    _check_mass(mass, mass_index, batch, c, k_cache)
    _check_input(new_block_table, "new_block_table")
    _same_device(k_cache, new_block_table, "k_cache", "new_block_table")
    budget, sink, recent = int(budget), int(sink), int(recent)
    _chk(budget > 0 and sink >= 0 and recent >= 0 and sink + recent <= budget, "budget must be positive and hold sink and recent")
    _chk(new_block_table.dtype == torch.int32 and new_block_table.dim() == 2 and new_block_table.size(0) >= batch, "new_block_table must be int32 [B, *]")
    _chk(max(budget, new_block_table.size(1)) <= _INT, "budget and the rows of new_block_table must be below 2^31")
    _chk(new_block_table.size(1) * PAGE_BLOCK_SIZE >= budget, "new_block_table must have room for budget tokens")
    with _on(k_cache.device):
        kept = torch.empty((batch, c.heads, budget), dtype=torch.int32, device=k_cache.device)
        new_mass = torch.empty((batch, c.heads, budget), dtype=torch.float32, device=k_cache.device)
        new_lens = torch.empty_like(seq_lens)
        if batch == 0:
            return kept, new_lens, new_mass
        _rc(_kv8().fak_evict_paged(ctypes.byref(c), _ptr(mass), None if mass_index is None else _ptr(mass_index), mass.size(0), mass.size(2),
                                   _ptr(seq_lens), batch, _ptr(new_block_table), new_block_table.size(1), budget, sink, recent, _ptr(kept),
                                   _ptr(new_lens), _ptr(new_mass), _stream_ptr(k_cache.device)))
    return kept, new_lens, new_mass


def check_errors(device=None) -> None:
    """Synchronise and raise RuntimeError if an operator on an 8-bit cache has met a page outside it since the last check."""
    if "kv8" not in _lib._libs:
        return
    used = _kv8().fak_devices()
    for dev in range(used.bit_length()):
        if not used >> dev & 1 or device is not None and torch.device(device).index not in (None, dev):
            continue
        with torch.cuda.device(dev):
            st = ctypes.c_int(0)
            torch.cuda.synchronize(dev)
            _rc(_kv8().fak_status(torch.cuda.current_stream(dev).cuda_stream, ctypes.byref(st), 1))
