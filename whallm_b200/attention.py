"""Attention over a paged key-value cache and over packed prompts.

A paged cache tensor is a pool ``[n_pages, Hkv, page_size, D]`` of rows in one
of the formats

* ``"bf16"``         bf16 rows, no scales;
* ``"fp8_f32_b64"``  e4m3 bytes (uint8), float32 scales ``[n_pages, Hkv, page_size, D/64]``;
* ``"mxfp8"``        e4m3 bytes (uint8), E8M0 scales (uint8) ``[n_pages, Hkv, page_size, D/32]``,

the latter two with the bytes of ``kv_quantize``.  Entry ``e`` of sequence ``b``
is slot ``e % page_size`` of page ``page_table[b, e // page_size]``; ``lengths``
counts a sequence's entries.  Tables, lengths and counts are int32 tensors on
the device that the kernels read, so a captured call follows their contents.
``kvcache.PagedKVCache`` keeps all of them together.

Activations are bf16; D is 64, 128 or 256; the page size a multiple of 16.
Every function runs on the current stream of its tensors' device.
"""
from __future__ import annotations

import math

import torch

from . import _lib as L

PAGED_FORMATS = {"bf16": L.WKV_BF16, "fp8_f32_b64": L.WKV_FP8_F32_B64, "mxfp8": L.WKV_MXFP8_B32}
_INT = torch.int32


def _call(name, t, *args):
    """Call an entry point on t's device and its current stream."""
    if t.device.index == torch.cuda.current_device():
        L.call(name, *args, L.stream_of(t))
    else:
        with torch.cuda.device(t.device):
            L.call(name, *args, L.stream_of(t))


def _same_device(first, *tensors):
    for t in tensors:
        if t is not None and t.device != first.device:
            raise ValueError("all tensors of a call must be on one device")


def _ints(name, t, shape):
    if t.dtype != _INT or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be int32 {list(shape)}")


def _tokens(name, t, heads=None):
    """bf16 [T, heads, D] whose heads are dense -> (T, heads, D, values between tokens)."""
    if t.dtype != torch.bfloat16 or t.dim() != 3:
        raise ValueError(f"{name} must be bf16 [tokens, heads, D]")
    n, h, d = t.shape
    if heads is not None and h != heads:
        raise ValueError(f"{name} has {h} heads, expected {heads}")
    if not t.is_cuda:
        raise ValueError("whallm_b200 ops take CUDA tensors (no CPU fallback)")
    if (d > 1 and t.stride(2) != 1) or (h > 1 and t.stride(1) != d):
        raise ValueError(f"the heads of a token of {name} must be contiguous")
    return n, h, d, (t.stride(0) if n > 1 else h * d)


def _pool(k_cache, v_cache, k_scales, v_scales, page_table, fmt):
    """Check a paged cache's tensors -> (format id, n_pages, Hkv, page_size, D, B, max_pages)."""
    if fmt not in PAGED_FORMATS:
        raise ValueError(f"paged cache format must be one of {sorted(PAGED_FORMATS)}, got {fmt!r}")
    f = PAGED_FORMATS[fmt]
    dt = torch.bfloat16 if f == L.WKV_BF16 else torch.uint8
    if k_cache.dim() != 4 or k_cache.dtype != dt or v_cache.dtype != dt or v_cache.shape != k_cache.shape:
        raise ValueError(f"caches must be {dt} [n_pages, heads, page_size, D] of one shape")
    pages, heads, size, d = k_cache.shape
    if f == L.WKV_BF16:
        if k_scales is not None or v_scales is not None:
            raise ValueError("bf16 caches take no scales")
    else:
        sdt, blk = (torch.float32, 64) if f == L.WKV_FP8_F32_B64 else (torch.uint8, 32)
        for s in (k_scales, v_scales):
            if s is None or s.dtype != sdt or tuple(s.shape) != (pages, heads, size, d // blk):
                raise ValueError(f"{fmt} caches need {sdt} scales [n_pages, heads, page_size, D/{blk}]")
    if page_table.dim() != 2 or page_table.dtype != _INT:
        raise ValueError("page_table must be int32 [sequences, max_pages]")
    L.require_cuda(k_cache, v_cache, k_scales, v_scales, page_table)
    _same_device(k_cache, v_cache, k_scales, v_scales, page_table)
    return f, pages, heads, size, d, page_table.shape[0], page_table.shape[1]


def _per_entry(name, t, dtype, shape):
    if t is not None and (t.dtype != dtype or tuple(t.shape) != shape):
        raise ValueError(f"{name} must be {dtype} {list(shape)}")


def _scale(scale, d):
    if scale is None:
        return 1.0 / math.sqrt(d)
    if not (0.0 < scale < math.inf):
        raise ValueError("scale must be positive and finite")
    return float(scale)


def paged_append(k, v, cu_seqlens, k_cache, v_cache, page_table, lengths, fmt="bf16", k_scales=None, v_scales=None,
                 mass=None, positions=None, seen=None):
    """Write new tokens into the cache.

    k, v bf16 [T, Hkv, D] are packed by sequence (``cu_seqlens`` int32 [B+1]) and
    become the last entries of their sequences: ``lengths`` int32 [B] counts them
    already.  Their ``mass`` (float32 [B, Hkv, capacity]) becomes 0 and their
    ``positions`` (int32, same shape) the token's position, ``seen`` int32 [B]
    counting every token of the sequence up to and including these."""
    f, pages, heads, size, d, B, width = _pool(k_cache, v_cache, k_scales, v_scales, page_table, fmt)
    T, _, dk, ks = _tokens("k", k, heads)
    Tv, _, dv, vs = _tokens("v", v, heads)
    if dk != d or dv != d or Tv != T:
        raise ValueError("k and v must have one shape and the cache's head dimension")
    _ints("cu_seqlens", cu_seqlens, (B + 1,))
    _ints("lengths", lengths, (B,))
    shape = (B, heads, width * size)
    _per_entry("mass", mass, torch.float32, shape)
    _per_entry("positions", positions, _INT, shape)
    if positions is not None and seen is None:
        raise ValueError("positions need the sequences' token counts (seen)")
    if seen is not None:
        _ints("seen", seen, (B,))
    L.require_cuda(cu_seqlens, lengths, mass, positions, seen)
    _same_device(k_cache, k, v, cu_seqlens, lengths, mass, positions, seen)
    p = L.ptr
    _call("wkv_paged_append", k, p(k), p(v), ks, vs, p(cu_seqlens), T, B, heads, d, p(k_cache), p(v_cache), p(k_scales),
          p(v_scales), f, pages, size, p(page_table), width, p(lengths), p(mass), p(positions), p(seen))


def paged_evict(k_cache, v_cache, page_table, lengths, mass, positions, seen, budget, recent=0, sinks=0, fmt="bf16",
                k_scales=None, v_scales=None, out=None):
    """Reduce every sequence longer than ``budget`` to ``budget`` entries per head:
    those at positions >= seen - recent or < sinks stay, then those of the largest
    mass (ties to the lower entry).  Kept entries behind the budget move into the
    freed ones before it; the others stay where they are.

    Without ``out``, mass and positions are updated in place; else ``out`` is
    ``(mass, positions, lengths)`` to write, which may share the input's mass and
    positions but not its lengths.  Returns (mass, positions, lengths)."""
    f, pages, heads, size, d, B, width = _pool(k_cache, v_cache, k_scales, v_scales, page_table, fmt)
    shape = (B, heads, width * size)
    new_mass, new_pos, new_len = out if out is not None else (mass, positions, torch.empty_like(lengths))
    _ints("lengths", lengths, (B,))
    _ints("new lengths", new_len, (B,))
    _ints("seen", seen, (B,))
    for m, q in ((mass, positions), (new_mass, new_pos)):
        _per_entry("mass", m, torch.float32, shape)
        _per_entry("positions", q, _INT, shape)
    budget, recent, sinks = int(budget), int(recent), int(sinks)
    if budget <= 0 or recent < 0 or sinks < 0 or recent + sinks > budget:
        raise ValueError("the budget must be positive and hold the recent and the first positions")
    L.require_cuda(lengths, mass, positions, seen, new_mass, new_pos, new_len)
    _same_device(k_cache, lengths, mass, positions, seen, new_mass, new_pos, new_len)
    budget = min(budget, 2**31 - 1)
    nbytes = L.lib().wkv_evict_workspace_size(B, heads, min(budget, max(width * size, 1)))
    ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=k_cache.device)
    p = L.ptr
    _call("wkv_paged_evict", k_cache, B, heads, d, p(k_cache), p(v_cache), p(k_scales), p(v_scales), f, pages, size,
          p(page_table), width, p(lengths), p(seen), p(mass), p(positions), budget, recent, sinks, p(new_mass), p(new_pos),
          p(new_len), p(ws), ws.numel())
    return new_mass, new_pos, new_len


def decode_attention(q, k_cache, v_cache, page_table, lengths, fmt="bf16", k_scales=None, v_scales=None, scale=None,
                     mass=None, return_lse=False, out=None):
    """Attention of one new token per sequence over the paged cache.

    q bf16 [B, Hq, D] with Hq a multiple of the cache's heads -> bf16 [B, Hq, D];
    with ``return_lse`` also the scores' log-sum-exp, float32 [B, Hq].  ``mass``
    (float32 [B, Hkv, capacity]) collects every entry's attention weight, summed
    over the query heads of its key-value head.  ``scale`` defaults to D^-1/2.  A
    sequence without entries gets zeros (lse -inf); one whose length or pages are
    out of range gets NaN."""
    f, pages, heads, size, d, B, width = _pool(k_cache, v_cache, k_scales, v_scales, page_table, fmt)
    Bq, Hq, dq, qs = _tokens("q", q)
    if Bq != B or dq != d or Hq % heads:
        raise ValueError("q must be [sequences, a multiple of the cache's heads, D]")
    _ints("lengths", lengths, (B,))
    _per_entry("mass", mass, torch.float32, (B, heads, width * size))
    scale = _scale(scale, d)
    if out is None:
        out = torch.empty((B, Hq, d), dtype=torch.bfloat16, device=q.device)
    elif out.dtype != torch.bfloat16 or tuple(out.shape) != (B, Hq, d):
        raise ValueError("out must be bf16 [sequences, heads, D]")
    L.require_cuda(lengths, mass, out)
    _same_device(k_cache, q, lengths, mass, out)
    lse = torch.empty((B, Hq), dtype=torch.float32, device=q.device) if return_lse else None
    nbytes = L.lib().wattn_decode_workspace_size(B, Hq, heads, d, f, size, width, mass is not None)
    ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=q.device)
    p = L.ptr
    _call("wattn_decode", q, p(q), qs, B, Hq, heads, d, p(k_cache), p(v_cache), p(k_scales), p(v_scales), f, pages, size,
          p(page_table), width, p(lengths), scale, p(out), p(lse), p(mass), p(ws), ws.numel())
    return (out, lse) if return_lse else out


def prompt_attention(q, k, v, cu_seqlens, cu_seqlens_k=None, scale=None, causal=True, return_lse=False, out=None):
    """Attention of packed prompts: q bf16 [Tq, Hq, D], k, v bf16 [Tk, Hkv, D] ->
    bf16 [Tq, Hq, D]; with ``return_lse`` also float32 [Tq, Hq].

    Sequence b has the rows ``cu_seqlens[b]:cu_seqlens[b+1]`` and, where
    ``cu_seqlens_k`` is given, keys of their own; causal row i of nq then sees the
    keys up to i + nk - nq (a prompt that continues a history).  Tokens may be
    strided (slices of one projection).  A row that sees no key gets zeros (lse
    -inf); rows outside every sequence are not written."""
    Tq, Hq, d, qs = _tokens("q", q)
    Tk, Hkv, dk, ks = _tokens("k", k)
    Tv, _, dv, vs = _tokens("v", v, Hkv)
    if dk != d or dv != d or Tv != Tk or Hkv == 0 or Hq % Hkv:
        raise ValueError("k and v must have one shape, q's head dimension and a divisor of q's heads")
    if cu_seqlens_k is None:
        if Tk != Tq:
            raise ValueError("keys of another count than the rows need cu_seqlens_k")
        cu_seqlens_k = cu_seqlens
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError("cu_seqlens must be int32 [sequences + 1]")
    B = cu_seqlens.numel() - 1
    _ints("cu_seqlens", cu_seqlens, (B + 1,))
    _ints("cu_seqlens_k", cu_seqlens_k, (B + 1,))
    scale = _scale(scale, d)
    if out is None:
        out = torch.empty((Tq, Hq, d), dtype=torch.bfloat16, device=q.device)
    elif out.dtype != torch.bfloat16 or tuple(out.shape) != (Tq, Hq, d):
        raise ValueError("out must be bf16 [tokens, heads, D]")
    L.require_cuda(cu_seqlens, cu_seqlens_k, out)
    _same_device(q, k, v, cu_seqlens, cu_seqlens_k, out)
    lse = torch.empty((Tq, Hq), dtype=torch.float32, device=q.device) if return_lse else None
    p = L.ptr
    _call("wattn_prompt", q, p(q), p(k), p(v), qs, ks, vs, p(cu_seqlens), p(cu_seqlens_k), B, Tq, Tk, Hq, Hkv, d, scale,
          int(bool(causal)), p(out), p(lse))
    return (out, lse) if return_lse else out
