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

import functools
import math

import torch

from . import _lib as L

PAGED_FORMATS = {"bf16": L.WKV_BF16, "fp8_f32_b64": L.WKV_FP8_F32_B64, "mxfp8": L.WKV_MXFP8_B32}
_BF16, _F32, _INT, _U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8
_NO_CPU = "whallm_b200 ops take CUDA tensors (no CPU fallback)"
_raw_stream = torch._C._cuda_getCurrentRawStream

# The checks below run on every call of a decode step, where for small batches the host's time is what counts:
# each function tests everything that a good call meets in one expression and looks for the reason only when it
# fails, and addresses go to the library as plain integers.


def _call(name, dev, *args):
    """Call an entry point on device number ``dev`` and its current stream."""
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return _call(name, dev, *args)
    rc = getattr(L._lib or L.lib(), name)(*args, _raw_stream(dev))
    if rc:
        L.fail(name, rc)


@functools.lru_cache(maxsize=512)
def _bytes(name, dev, *shape):
    """Workspace of a call on device number ``dev``: the plan behind it follows that device's SMs."""
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return getattr(L.lib(), name)(*shape)
    return getattr(L.lib(), name)(*shape)


def _at(name, t, dtype, shape, dev):
    """Address of a contiguous tensor of a given type, shape and device (None: 0)."""
    if t is None:
        return None
    if t.dtype is dtype and t.shape == shape and t.get_device() == dev and t.is_contiguous():
        return t.data_ptr()
    if t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{name} must be {dtype} {list(shape)}")
    if not t.is_cuda:
        raise ValueError(_NO_CPU)
    if not t.is_contiguous():
        raise ValueError("whallm_b200 ops take contiguous tensors")
    raise ValueError("all tensors of a call must be on one device")


def _tokens(name, t, heads, d, dev):
    """bf16 [T, heads, D] whose heads are dense (heads, d, dev: what it must match, or None) -> (T, heads, D,
    values between tokens)."""
    shape = t.shape
    if len(shape) == 3 and t.dtype is _BF16:
        n, h, e = shape
        s0, s1, s2 = t.stride()
        at = t.get_device()
        if ((heads is None or h == heads) and (d is None or e == d) and (at == dev or dev is None) and at >= 0
                and (s2 == 1 or e == 1) and (s1 == e or h == 1)):
            return n, h, e, (s0 if n > 1 else h * e)
    if t.dtype != _BF16 or t.dim() != 3:
        raise ValueError(f"{name} must be bf16 [tokens, heads, D]")
    if heads is not None and shape[1] != heads:
        raise ValueError(f"{name} has {shape[1]} heads, expected {heads}")
    if d is not None and shape[2] != d:
        raise ValueError(f"{name} has head dimension {shape[2]}, expected {d}")
    if not t.is_cuda:
        raise ValueError(_NO_CPU)
    if dev is not None and t.get_device() != dev:
        raise ValueError("all tensors of a call must be on one device")
    raise ValueError(f"the heads of a token of {name} must be contiguous")


def _pool(k_cache, v_cache, k_scales, v_scales, page_table, fmt):
    """Check a paged cache's tensors -> (format id, n_pages, Hkv, page_size, D, B, max_pages, device, and the
    addresses of caches, scales and table)."""
    f = PAGED_FORMATS.get(fmt)
    if f is None:
        raise ValueError(f"paged cache format must be one of {sorted(PAGED_FORMATS)}, got {fmt!r}")
    shape, tshape, dev = k_cache.shape, page_table.shape, k_cache.get_device()
    dt = _BF16 if f == L.WKV_BF16 else _U8
    if not (len(shape) == 4 and len(tshape) == 2 and k_cache.dtype is dt and page_table.dtype is _INT):
        if len(shape) != 4 or k_cache.dtype != dt:
            raise ValueError(f"caches must be {dt} [n_pages, heads, page_size, D] of one shape")
        raise ValueError("page_table must be int32 [sequences, max_pages]")
    pages, heads, size, d = shape
    if f == L.WKV_BF16:
        if k_scales is not None or v_scales is not None:
            raise ValueError("bf16 caches take no scales")
        ks = vs = None
    else:
        sdt, blk = (_F32, 64) if f == L.WKV_FP8_F32_B64 else (_U8, 32)
        sshape = (pages, heads, size, d // blk)
        if k_scales is None or v_scales is None:
            raise ValueError(f"{fmt} caches need {sdt} scales [n_pages, heads, page_size, D/{blk}]")
        ks, vs = _at("k_scales", k_scales, sdt, sshape, dev), _at("v_scales", v_scales, sdt, sshape, dev)
    v = _at("v_cache", v_cache, dt, shape, dev)
    t = _at("page_table", page_table, _INT, tshape, dev)
    if dev < 0 or not heads or not k_cache.is_contiguous():
        if not heads:
            raise ValueError("a paged cache needs heads")
        raise ValueError(_NO_CPU if dev < 0 else "whallm_b200 ops take contiguous tensors")
    return f, pages, heads, size, d, tshape[0], tshape[1], dev, k_cache.data_ptr(), v, ks, vs, t


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
    f, pages, heads, size, d, B, width, dev, kc, vc, ksc, vsc, table = _pool(k_cache, v_cache, k_scales, v_scales,
                                                                             page_table, fmt)
    T, _, _, ks = _tokens("k", k, heads, d, dev)
    Tv, _, _, vs = _tokens("v", v, heads, d, dev)
    if Tv != T:
        raise ValueError("k and v must have as many tokens")
    if positions is not None and seen is None:
        raise ValueError("positions need the sequences' token counts (seen)")
    shape = (B, heads, width * size)
    _call("wkv_paged_append", dev, k.data_ptr(), v.data_ptr(), ks, vs, _at("cu_seqlens", cu_seqlens, _INT, (B + 1,), dev),
          T, B, heads, d, kc, vc, ksc, vsc, f, pages, size, table, width, _at("lengths", lengths, _INT, (B,), dev),
          _at("mass", mass, _F32, shape, dev), _at("positions", positions, _INT, shape, dev),
          _at("seen", seen, _INT, (B,), dev))


def paged_evict(k_cache, v_cache, page_table, lengths, mass, positions, seen, budget, recent=0, sinks=0, fmt="bf16",
                k_scales=None, v_scales=None, out=None):
    """Reduce every sequence longer than ``budget`` to ``budget`` entries per head:
    those at positions >= seen - recent or < sinks stay, then those of the largest
    mass (ties to the lower entry).  Kept entries behind the budget move into the
    freed ones before it; the others stay where they are.

    Without ``out``, mass and positions are updated in place; else ``out`` is
    ``(mass, positions, lengths)`` to write, which may share the input's mass and
    positions but not its lengths.  Returns (mass, positions, lengths)."""
    f, pages, heads, size, d, B, width, dev, kc, vc, ksc, vsc, table = _pool(k_cache, v_cache, k_scales, v_scales,
                                                                             page_table, fmt)
    cap = width * size
    shape = (B, heads, cap)
    new_mass, new_pos, new_len = out if out is not None else (mass, positions, torch.empty_like(lengths))
    budget, recent, sinks = int(budget), int(recent), int(sinks)
    if budget <= 0 or recent < 0 or sinks < 0 or recent + sinks > budget:
        raise ValueError("the budget must be positive and hold the recent and the first positions")
    budget = min(budget, 2**31 - 1)
    ws = mass.new_empty((B * heads * (6 * max(1, min(budget, cap)) + 1),))
    _call("wkv_paged_evict", dev, B, heads, d, kc, vc, ksc, vsc, f, pages, size, table, width,
          _at("lengths", lengths, _INT, (B,), dev), _at("seen", seen, _INT, (B,), dev), _at("mass", mass, _F32, shape, dev),
          _at("positions", positions, _INT, shape, dev), budget, recent, sinks, _at("new mass", new_mass, _F32, shape, dev),
          _at("new positions", new_pos, _INT, shape, dev), _at("new lengths", new_len, _INT, (B,), dev), ws.data_ptr(),
          4 * ws.numel())
    return new_mass, new_pos, new_len


def decode_attention(q, k_cache, v_cache, page_table, lengths, fmt="bf16", k_scales=None, v_scales=None, scale=None,
                     mass=None, return_lse=False, out=None):
    """Attention of one new token per sequence over the paged cache.

    q bf16 [B, Hq, D] with Hq a multiple of the cache's heads -> bf16 [B, Hq, D];
    with ``return_lse`` also the scores' log-sum-exp, float32 [B, Hq].  ``mass``
    (float32 [B, Hkv, capacity]) collects every entry's attention weight, summed
    over the query heads of its key-value head.  ``scale`` defaults to D^-1/2.  A
    sequence without entries gets zeros (lse -inf); one whose length or pages are
    out of range gets NaN.  A key whose score is -inf weighs nothing.  With ``mass``
    time and workspace grow with the capacity (the table's width), so keep that near
    the longest sequence."""
    f, pages, heads, size, d, B, width, dev, kc, vc, ksc, vsc, table = _pool(k_cache, v_cache, k_scales, v_scales,
                                                                             page_table, fmt)
    Bq, Hq, _, qs = _tokens("q", q, None, d, dev)
    if Bq != B or Hq % heads:
        raise ValueError("q must be [sequences, a multiple of the cache's heads, D]")
    scale = _scale(scale, d)
    if out is None:
        out = q.new_empty((B, Hq, d))
    lse = q.new_empty((B, Hq), dtype=_F32) if return_lse else None
    nbytes = _bytes("wattn_decode_workspace_size", dev, B, Hq, heads, d, f, size, width, mass is not None)
    ws = q.new_empty((nbytes,), dtype=_U8) if nbytes else None     # short caches need none
    _call("wattn_decode", dev, q.data_ptr(), qs, B, Hq, heads, d, kc, vc, ksc, vsc, f, pages, size, table, width,
          _at("lengths", lengths, _INT, (B,), dev), scale, _at("out", out, _BF16, (B, Hq, d), dev),
          lse.data_ptr() if return_lse else None, _at("mass", mass, _F32, (B, heads, width * size), dev),
          ws.data_ptr() if nbytes else None, nbytes)
    return (out, lse) if return_lse else out


def prompt_attention(q, k, v, cu_seqlens, cu_seqlens_k=None, scale=None, causal=True, return_lse=False, out=None):
    """Attention of packed prompts: q bf16 [Tq, Hq, D], k, v bf16 [Tk, Hkv, D] ->
    bf16 [Tq, Hq, D]; with ``return_lse`` also float32 [Tq, Hq].

    Sequence b has the rows ``cu_seqlens[b]:cu_seqlens[b+1]`` and, where
    ``cu_seqlens_k`` is given, keys of their own; causal row i of nq then sees the
    keys up to i + nk - nq (a prompt that continues a history).  Tokens may be
    strided (slices of one projection).  A row that sees no key gets zeros (lse
    -inf); rows outside every sequence are not written.  Equal calls give equal
    bits; how a sequence's keys are summed may depend on the batch around it."""
    dev = q.get_device()
    Tq, Hq, d, qs = _tokens("q", q, None, None, None)
    Tk, Hkv, _, ks = _tokens("k", k, None, d, dev)
    Tv, _, _, vs = _tokens("v", v, Hkv, d, dev)
    if Tv != Tk or Hkv == 0 or Hq % Hkv:
        raise ValueError("k and v must have one shape and a divisor of q's heads")
    if cu_seqlens_k is None:
        if Tk != Tq:
            raise ValueError("keys of another count than the rows need cu_seqlens_k")
        cu_seqlens_k = cu_seqlens
    B = cu_seqlens.numel() - 1
    if B < 0:
        raise ValueError("cu_seqlens must be int32 [sequences + 1]")
    scale = _scale(scale, d)
    if out is None:
        out = q.new_empty((Tq, Hq, d))
    lse = q.new_empty((Tq, Hq), dtype=_F32) if return_lse else None
    nbytes = _bytes("wattn_prompt_workspace_size", dev, B, Tq, Tk, Hq, Hkv, d)
    ws = q.new_empty((nbytes,), dtype=_U8) if nbytes else None     # only few rows on many keys need one
    _call("wattn_prompt", dev, q.data_ptr(), k.data_ptr(), v.data_ptr(), qs, ks, vs,
          _at("cu_seqlens", cu_seqlens, _INT, (B + 1,), dev), _at("cu_seqlens_k", cu_seqlens_k, _INT, (B + 1,), dev), B, Tq,
          Tk, Hq, Hkv, d, scale, 1 if causal else 0, _at("out", out, _BF16, (Tq, Hq, d), dev),
          lse.data_ptr() if return_lse else None, ws.data_ptr() if nbytes else None, nbytes)
    return (out, lse) if return_lse else out
