"""Cases for the attention operators and the paged key-value cache they read.

Four operators, each with a plain form in elementary torch operations:

* ``append``  new keys and values of several sequences into a paged cache
  (bf16 rows, or e4m3 rows with block scales quantized on the way in);
* ``decode``  attention of one new token per sequence over the paged cache,
  optionally adding each cached entry's attention weight to a running mass;
* ``prompt``  causal attention over packed sequences with grouped heads, on
  their own keys or on a longer history that they continue;
* ``evict``   reduction of a cache to a budget of entries per key-value head
  by accumulated weight, with the first and the latest positions kept.

``own`` selects the framework's kernels; otherwise the plain form runs.
"""
import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
NEG = float("-inf")


# ------------------------------------------------------------------- cases --

def listed():
    return [
        # one decode step of a serving batch: 64 sequences write one token each
        dict(name="append a step", op="append", B=64, new_min=1, new_max=1, old_max=110, mix=1, Hkv=8, D=128, page=16,
             fmt="bf16", track=False),
        # prompts of several users stored as e4m3 with float32 scales (the 2 x 256 heads of the QSA caches)
        dict(name="append prompts", op="append", B=8, new_min=300, new_max=4099, old_max=500, mix=2, Hkv=2, D=256,
             page=64, fmt="fp8_f32_b64", track=True),
        # one user at a middling context: latency counts
        dict(name="decode one", op="decode", B=1, len_min=4095, len_max=4095, mix=3, Hq=32, Hkv=8, D=128, page=64,
             fmt="bf16", track=False),
        # a full serving batch with contexts of very different lengths
        dict(name="decode batch", op="decode", B=64, len_min=90, len_max=8190, mix=4, Hq=32, Hkv=8, D=128, page=64,
             fmt="bf16", track=False),
        # two long documents in an e4m3 cache
        dict(name="decode long", op="decode", B=2, len_min=120001, len_max=131071, mix=5, Hq=16, Hkv=2, D=256,
             page=128, fmt="fp8_f32_b64", track=False),
        # eight sequences near 32768 positions whose entries collect their weights for eviction
        dict(name="decode tracked", op="decode", B=8, len_min=30001, len_max=32768, mix=6, Hq=16, Hkv=2, D=256,
             page=64, fmt="mxfp8", track=True),
        # a few short questions
        dict(name="prompt short", op="prompt", B=4, q_min=17, q_max=201, old_min=0, old_max=0, mix=7, Hq=32, Hkv=8,
             D=64),
        # a prefill batch of ragged prompts
        dict(name="prompt packed", op="prompt", B=8, q_min=333, q_max=4096, old_min=0, old_max=0, mix=8, Hq=32, Hkv=8,
             D=128),
        # one long document at the Qwen-class head shape
        dict(name="prompt long", op="prompt", B=1, q_min=16383, q_max=16383, old_min=0, old_max=0, mix=9, Hq=16,
             Hkv=2, D=256),
        # the next chunk of four prompts whose beginnings are already there
        dict(name="prompt continued", op="prompt", B=4, q_min=400, q_max=515, old_min=3000, old_max=8000, mix=10,
             Hq=32, Hkv=8, D=128),
        # a cache at its budget makes room for the token just written
        dict(name="evict a step", op="evict", B=8, len_min=2049, len_max=2049, mix=11, Hkv=8, D=128, page=64,
             fmt="bf16", budget=2048, recent=128, sinks=4),
        # long prompts cut down to a working set
        dict(name="evict prompts", op="evict", B=4, len_min=20000, len_max=32768, mix=12, Hkv=2, D=256, page=64,
             fmt="fp8_f32_b64", budget=4096, recent=512, sinks=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limits = {}
    for c in listed():
        limits[c["op"]] = max(limits.get(c["op"], 0.0), _cost(c))
    while True:
        op = rng.choice(["append", "decode", "decode", "prompt", "prompt", "evict"])
        mix = rng.randrange(1 << 30)
        D = rng.choice([64, 128, 256])
        Hkv = rng.choice([1, 2, 4, 8])
        G = rng.choice([1, 2, 4, 5, 8, 16])
        page = rng.choice([16, 32, 64, 128])
        fmt = rng.choice(["bf16", "fp8_f32_b64", "mxfp8"])
        if op == "append":
            top = _log(rng, 1, 4096)
            c = dict(op=op, B=_log(rng, 1, 128), new_min=max(1, top // 8), new_max=top, old_max=_log(rng, 1, 512), mix=mix, Hkv=Hkv,
                     D=D, page=page, fmt=fmt, track=rng.random() < 0.5)
        elif op == "decode":
            top = _log(rng, 1, 131071)
            c = dict(op=op, B=_log(rng, 1, 96), len_min=max(1, int(top * rng.random())), len_max=top, mix=mix,
                     Hq=Hkv * G, Hkv=Hkv, D=D, page=page, fmt=fmt, track=rng.random() < 0.4)
        elif op == "prompt":
            top = _log(rng, 1, 16384)
            old = rng.choice([0, 0, _log(rng, 1, 8192)])
            c = dict(op=op, B=_log(rng, 1, 24), q_min=max(1, top // rng.choice([1, 2, 8])), q_max=top,
                     old_min=old // 3, old_max=old, mix=mix, Hq=Hkv * G, Hkv=Hkv, D=D)
        else:
            top = _log(rng, 128, 32768)
            budget = max(64, int(top * rng.uniform(0.1, 1.0)))
            c = dict(op=op, B=_log(rng, 1, 32), len_min=max(1, int(top * rng.random())), len_max=top, mix=mix, Hkv=Hkv,
                     D=D, page=page, fmt=fmt, budget=budget, recent=_log(rng, 1, budget // 4), sinks=rng.choice([0, 1, 4]))
        if _cost(c) <= limits[op]:
            return c


def _spread(case, lo, hi, salt):
    """One length per sequence between lo and hi, the last one at hi; the same for every seed."""
    r = random.Random(case["mix"] * 7 + salt)
    return [r.randint(lo, hi) for _ in range(case["B"] - 1)] + [hi]


def _q_lens(c):
    new = _spread(c, c["q_min"], c["q_max"], 1)
    old = _spread(c, c["old_min"], c["old_max"], 2)
    return new, [n + o for n, o in zip(new, old)]


def _append_lens(c):
    new = _spread(c, c["new_min"], c["new_max"], 1)
    old = _spread(c, 0, c["old_max"], 2)
    return new, [n + o for n, o in zip(new, old)]


def _row_bytes(c):
    """Bytes of one cached row of one tensor with its scales."""
    D = c["D"]
    return {"bf16": 2 * D, "fp8_f32_b64": D + 4 * (D // 64), "mxfp8": D + D // 32}[c["fmt"]]


def _padded(c):
    """float32 values of the largest padded intermediate of the plain form."""
    if c["op"] == "prompt":
        new, total = _q_lens(c)
        return c["B"] * c["Hq"] * max(new) * max(total)
    if c["op"] == "append":
        return sum(_append_lens(c)[0]) * c["Hkv"] * c["D"]
    return c["B"] * c["Hkv"] * c["len_max"] * c["D"]


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50, _padded(c) / 4)


def work(case):
    c = case
    if c["op"] == "append":
        new, _ = _append_lens(c)
        n = sum(new) * c["Hkv"]
        return dict(bytes=2 * n * (2 * c["D"] + _row_bytes(c)) + (8 * n if c["track"] else 0), flops=0)
    if c["op"] == "decode":
        n = sum(_spread(c, c["len_min"], c["len_max"], 1))
        qo = 4 * c["B"] * c["Hq"] * c["D"] + 4 * c["B"] * c["Hq"]
        return dict(bytes=2 * n * c["Hkv"] * _row_bytes(c) + qo + (8 * n * c["Hkv"] if c["track"] else 0),
                    flops=4 * n * c["Hq"] * c["D"])
    if c["op"] == "prompt":
        new, total = _q_lens(c)
        pairs = sum(q * (t - q) + q * (q + 1) // 2 for q, t in zip(new, total))
        return dict(bytes=4 * sum(new) * c["Hq"] * c["D"] + 4 * sum(new) * c["Hq"] + 4 * sum(total) * c["Hkv"] * c["D"],
                    flops=4 * pairs * c["Hq"] * c["D"])
    # every weight and position is read, a kept entry's are written, and a row moves at least for every
    # kept entry that lies behind the budget (for evenly spread weights a share of (length - budget) / length)
    lens = _spread(c, c["len_min"], c["len_max"], 1)
    read = sum(8 * n for n in lens) * c["Hkv"]
    kept = sum(8 * min(n, c["budget"]) for n in lens) * c["Hkv"]
    moved = sum(min(n, c["budget"]) * max(0, n - c["budget"]) / n for n in lens) * c["Hkv"]
    return dict(bytes=read + kept + moved * 4 * _row_bytes(c), flops=0)


# ------------------------------------------------------------------ inputs --

def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(g, shape, dtype=torch.bfloat16):
    """Standard normal values, made in pieces of the type asked for."""
    out = torch.empty(shape, dtype=dtype, device=DEVICE)
    return out.normal_(generator=g)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEVICE)


def _cu(lens):
    return _ints([0] + np.cumsum(lens).tolist())


def _quantize(x, fmt):
    """Rows in the cache's format: (payload, scales)."""
    if fmt == "bf16":
        return x, None
    blk = 64 if fmt == "fp8_f32_b64" else 32
    f = x.float().unflatten(-1, (-1, blk))
    amax = f.abs().amax(-1)
    if fmt == "fp8_f32_b64":
        scales = amax / torch.full_like(amax, 448.0)            # a true quotient: dividing by a plain number is not
        div = torch.where(scales > 0, scales, torch.inf)       # a block of zeros: scale 0, codes 0
    else:
        e = torch.where(amax > 0, torch.frexp(amax)[1] - 1 - 8, torch.full_like(amax, -127, dtype=torch.int32))
        e = e.clamp(-127, 127)
        scales, div = (e + 127).to(torch.uint8), torch.ldexp(torch.ones_like(amax), e)
    code = (f / div.unsqueeze(-1)).clamp(-448.0, 448.0).flatten(-2).to(torch.float8_e4m3fn)
    return code.view(torch.uint8), scales


def _pool(g, c, need):
    """A page pool with rows in every page, and a table that spreads each sequence's pages over it."""
    per = [-(-n // c["page"]) for n in need]
    width, total = max(per), sum(per) + 3
    order = torch.randperm(total, generator=g, device=DEVICE, dtype=torch.int64).to(torch.int32)
    table = torch.full((c["B"], width), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, p in enumerate(per):
        table[b, :p] = order[at:at + p]
        at += p
    shape = (total, c["Hkv"], c["page"], c["D"])
    k, ks = _quantize(_normal(g, shape), c["fmt"])
    v, vs = _quantize(_normal(g, shape), c["fmt"])
    return dict(k_cache=k, v_cache=v, k_scales=ks, v_scales=vs, table=table, cap=width * c["page"])


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    s = dict(c)
    if c["op"] == "append":
        new, total = _append_lens(c)
        s.update(_pool(g, c, total))
        T = sum(new)
        qkv = _normal(g, (T, 2 * c["Hkv"], c["D"]))     # keys and values side by side, as a projection leaves them
        s.update(k=qkv[:, :c["Hkv"]], v=qkv[:, c["Hkv"]:], cu=_cu(new), lengths=_ints(total), seen=_ints(total), T=T)
        if c["track"]:
            s["mass"] = torch.rand((c["B"], c["Hkv"], s["cap"]), generator=g, device=DEVICE)
            s["positions"] = torch.zeros((c["B"], c["Hkv"], s["cap"]), dtype=torch.int32, device=DEVICE)
    elif c["op"] == "decode":
        lens = _spread(c, c["len_min"], c["len_max"], 1)
        s.update(_pool(g, c, lens))
        s.update(q=_normal(g, (c["B"], c["Hq"], c["D"])) * 2, lengths=_ints(lens))   # scores of deviation 2
        if c["track"]:
            s["mass"] = torch.zeros((c["B"], c["Hkv"], s["cap"]), device=DEVICE)
    elif c["op"] == "prompt":
        new, total = _q_lens(c)
        qkv = None
        if new == total:                                # one projection's output: strided views of it
            qkv = _normal(g, (sum(new), c["Hq"] + 2 * c["Hkv"], c["D"]))
            qkv[:, :c["Hq"]] *= 2
            q, k, v = qkv.split([c["Hq"], c["Hkv"], c["Hkv"]], dim=1)
        else:
            q = _normal(g, (sum(new), c["Hq"], c["D"])) * 2
            k, v = (_normal(g, (sum(total), c["Hkv"], c["D"])) for _ in range(2))
        s.update(q=q, k=k, v=v, cu_q=_cu(new), cu_k=_cu(total), max_q=max(new), max_k=max(total))
    else:
        lens = _spread(c, c["len_min"], c["len_max"], 1)
        s.update(_pool(g, c, lens))
        shape = (c["B"], c["Hkv"], s["cap"])
        # sums of softmax weights: most entries get little, a few get most of it
        s["mass"] = torch.empty(shape, device=DEVICE).normal_(generator=g).mul_(2).exp_()
        s["positions"] = torch.arange(s["cap"], dtype=torch.int32, device=DEVICE).expand(shape).contiguous()
        s.update(lengths=_ints(lens), seen=_ints(lens), new_mass=torch.zeros_like(s["mass"]),
                 new_positions=torch.zeros_like(s["positions"]), new_lengths=torch.zeros_like(_ints(lens)))
    return s


# ------------------------------------------------------------- plain forms --

def _values(cache, scales, fmt):
    """Cached rows as float32 values."""
    if fmt == "bf16":
        return cache.float()
    blk = 64 if fmt == "fp8_f32_b64" else 32
    s = scales if fmt == "fp8_f32_b64" else torch.ldexp(torch.ones((), device=DEVICE), scales.int() - 127)
    return (cache.view(torch.float8_e4m3fn).float().unflatten(-1, (-1, blk)) * s.unsqueeze(-1)).flatten(-2)


def _pages(cache, table):
    """[B, Hkv, capacity, ...] of a pool through a table (pages that are not there read page 0)."""
    return cache[table.clamp(min=0).long()].transpose(1, 2).flatten(2, 3)


def _as_values(payload):
    return payload.view(torch.float8_e4m3fn) if payload.dtype == torch.uint8 else payload


def _cache_out(s):
    d = dict(k=_as_values(s["k_cache"]), v=_as_values(s["v_cache"]))
    if s["k_scales"] is not None:
        d.update(ks=s["k_scales"], vs=s["v_scales"])
    return d


def _append_plain(s):
    t = torch.arange(s["T"], device=DEVICE)
    b = torch.searchsorted(s["cu"][1:].long(), t, right=True)
    n_new = (s["cu"][1:] - s["cu"][:-1]).long()
    back = s["cu"][1:].long()[b] - t                       # tokens from here to the sequence's end, this one too
    at = s["lengths"].long()[b] - back
    page = s["table"][b, at // s["page"]].long()
    slot = at % s["page"]
    for name in ("k", "v"):
        p, sc = _quantize(s[name].contiguous(), s["fmt"])
        s[name + "_cache"][page, :, slot] = p
        if sc is not None:
            s[name + "_scales"][page, :, slot] = sc
    if s["track"]:
        s["mass"][b, :, at] = 0.0
        s["positions"][b, :, at] = (s["seen"].long()[b] - back).int()[:, None].expand(-1, s["Hkv"])
    return n_new


def _decode_plain(s):
    B, Hq, Hkv, D = s["B"], s["Hq"], s["Hkv"], s["D"]
    k = _values(_pages(s["k_cache"], s["table"]),
                None if s["k_scales"] is None else _pages(s["k_scales"], s["table"]), s["fmt"])
    q = s["q"].float().view(B, Hkv, Hq // Hkv, D)
    x = q @ k.transpose(-1, -2) / math.sqrt(D)
    del k
    x.masked_fill_(torch.arange(s["cap"], device=DEVICE) >= s["lengths"][:, None, None, None], NEG)
    m = x.amax(-1, keepdim=True)
    p = x.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    v = _values(_pages(s["v_cache"], s["table"]),
                None if s["v_scales"] is None else _pages(s["v_scales"], s["table"]), s["fmt"])
    out = (p @ v) / l
    if s["track"]:
        s["mass"] += (p / l).sum(2)
    return out.view(B, Hq, D).to(torch.bfloat16), (m + l.log()).view(B, Hq)


def _prompt_plain(s):
    Hq, Hkv, D, G = s["Hq"], s["Hkv"], s["D"], s["Hq"] // s["Hkv"]
    T = s["q"].shape[0]
    iq, ik = torch.arange(s["max_q"], device=DEVICE), torch.arange(s["max_k"], device=DEVICE)
    nq, nk = (s["cu_q"][1:] - s["cu_q"][:-1]).long(), (s["cu_k"][1:] - s["cu_k"][:-1]).long()
    at_q = torch.where(iq < nq[:, None], s["cu_q"][:-1, None].long() + iq, T)          # row T: a row to throw away
    at_k = (s["cu_k"][:-1, None].long() + ik).clamp(max=s["k"].shape[0] - 1)
    q = s["q"][at_q.clamp(max=T - 1)].float().transpose(1, 2).unflatten(1, (Hkv, G))   # [B, Hkv, G, q, D]
    k, v = (s[n][at_k].float().transpose(1, 2).unsqueeze(2) for n in ("k", "v"))       # [B, Hkv, 1, k, D]
    x = q.flatten(2, 3).mul_(1.0 / math.sqrt(D)) @ k[:, :, 0].transpose(-1, -2)
    x = x.unflatten(2, (G, -1))
    hidden = ik > (iq[:, None] + (nk - nq)[:, None, None])                             # [B, q, k]
    x.masked_fill_(hidden[:, None, None], NEG)
    m = x.amax(-1, keepdim=True)
    x.sub_(m).exp_()
    l = x.sum(-1, keepdim=True)
    o = (x.flatten(2, 3) @ v[:, :, 0]).unflatten(2, (G, -1)) / l
    out = torch.zeros((T + 1, Hq, D), dtype=torch.bfloat16, device=DEVICE)
    lse = torch.zeros((T + 1, Hq), device=DEVICE)
    out[at_q] = o.flatten(1, 2).transpose(1, 2).to(torch.bfloat16)
    lse[at_q] = (m + l.log()).flatten(1, 2).squeeze(-1).transpose(1, 2)
    return out[:T], lse[:T]


def _evict_plain(s):
    B, Hkv, page, cap = s["B"], s["Hkv"], s["page"], s["cap"]
    n = min(s["budget"], cap)
    idx = torch.arange(cap, device=DEVICE).expand(B, Hkv, cap)
    live = idx < s["lengths"][:, None, None]
    keep_pos = (s["positions"] >= (s["seen"] - s["recent"])[:, None, None]) | (s["positions"] < s["sinks"])
    key = torch.where(keep_pos, torch.inf, s["mass"]).masked_fill(~live, -1.0)
    first = torch.sort(key, dim=-1, descending=True, stable=True)[1][..., :n]
    kept = torch.zeros_like(live).scatter_(-1, first, True) & live
    hole = ~kept & (idx < n) & live
    tail = kept & (idx >= n)
    # the r-th hole takes the r-th kept entry behind the budget; any other entry stays
    rank = torch.where(tail, tail.cumsum(-1) - 1, cap)
    tails = torch.zeros((B, Hkv, cap + 1), dtype=torch.long, device=DEVICE).scatter_(-1, rank, idx)
    src = torch.where(hole[..., :n], tails.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0)[..., :n]), idx[..., :n])
    ok = live[..., :n]
    src = torch.where(ok, src, 0)                            # entries behind the end: entry 0 onto itself
    dst = torch.where(ok, idx[..., :n], 0)
    src = torch.where(ok, src, src[..., :1])                 # ... with what that one takes
    bb = torch.arange(B, device=DEVICE)[:, None, None]
    hh = torch.arange(Hkv, device=DEVICE)[None, :, None]
    sp, dp = s["table"][bb, src // page].long(), s["table"][bb, dst // page].long()
    for name in ("k_cache", "v_cache", "k_scales", "v_scales"):
        if s[name] is not None:
            s[name][dp, hh, dst % page] = s[name][sp, hh, src % page]
    for name in ("mass", "positions"):
        new = s["new_" + name]
        new[..., :n] = torch.where(ok, s[name].gather(-1, src), new[..., :n])
    s["new_lengths"].copy_(s["lengths"].clamp(max=n))


# --------------------------------------------------------------------- run --

def run(state):
    s = state
    if own:
        import whallm_b200 as W
        if s["op"] == "append":
            W.paged_append(s["k"], s["v"], s["cu"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], fmt=s["fmt"],
                           k_scales=s["k_scales"], v_scales=s["v_scales"], mass=s.get("mass"),
                           positions=s.get("positions"), seen=s["seen"])
        elif s["op"] == "decode":
            out, lse = W.decode_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], fmt=s["fmt"],
                                          k_scales=s["k_scales"], v_scales=s["v_scales"], mass=s.get("mass"),
                                          return_lse=True)
        elif s["op"] == "prompt":
            out, lse = W.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], return_lse=True)
        else:
            W.paged_evict(s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["mass"], s["positions"], s["seen"],
                          s["budget"], recent=s["recent"], sinks=s["sinks"], fmt=s["fmt"], k_scales=s["k_scales"],
                          v_scales=s["v_scales"], out=(s["new_mass"], s["new_positions"], s["new_lengths"]))
    elif s["op"] == "append":
        _append_plain(s)
    elif s["op"] == "decode":
        out, lse = _decode_plain(s)
    elif s["op"] == "prompt":
        out, lse = _prompt_plain(s)
    else:
        _evict_plain(s)
    if s["op"] == "append":
        return dict(_cache_out(s), **{n: s[n] for n in ("mass", "positions") if n in s})
    if s["op"] == "evict":
        return dict(_cache_out(s), mass=s["new_mass"], positions=s["new_positions"], lengths=s["new_lengths"])
    return dict(out=out, lse=lse, **({"mass": s["mass"]} if "mass" in s else {}))


# ------------------------------------------------------------- 64-bit forms --

_E4M3 = None


def _e4m3_table():
    """The 256 e4m3 values from the format's definition: sign, 4 exponent bits of bias 7, 3 mantissa bits."""
    global _E4M3
    if _E4M3 is None:
        v = []
        for code in range(256):
            e, m = (code >> 3) & 15, code & 7
            x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
            v.append(math.nan if (e, m) == (15, 7) else (-x if code & 128 else x))
        _E4M3 = torch.tensor(v, dtype=torch.float64, device=DEVICE)
    return _E4M3


def _rows64(s, name, b, h, n):
    """The first n cached rows of sequence b, head h in 64 bits."""
    pages = s["table"][b, :-(-n // s["page"])].long()
    x = s[name + "_cache"][pages, h].reshape(-1, s["D"])[:n]
    if s["fmt"] == "bf16":
        return x.double()
    sc = s[name + "_scales"][pages, h].reshape(x.shape[0] + (-n) % s["page"], -1)[:n]
    f = sc.double() if s["fmt"] == "fp8_f32_b64" else torch.exp2(sc.double() - 127)
    return _e4m3_table()[x.long()] * f.repeat_interleave(s["D"] // f.shape[1], dim=1)


def _exact_append(s, case):
    """Row by row: token i of a sequence of n new ones goes to entry length - n + i."""
    new, total = _append_lens(case)
    at = 0
    for b, (n, t) in enumerate(zip(new, total)):
        e = torch.arange(t - n, t, device=DEVICE)
        page, slot = s["table"][b][e // s["page"]].long(), e % s["page"]
        for name in ("k", "v"):
            x = s[name][at:at + n].double()
            if s["fmt"] == "bf16":
                s[name + "_cache"][page, :, slot] = x.to(torch.bfloat16)
                continue
            blk = 64 if s["fmt"] == "fp8_f32_b64" else 32
            x = x.reshape(n, s["Hkv"], -1, blk)
            top = x.abs().amax(-1)
            if blk == 64:
                kept = (top / 448.0).float()           # the stored scale is a float32
                f = torch.where(kept > 0, kept.double(), torch.inf)
            else:
                ex = torch.floor(torch.log2(top.clamp(min=2.0 ** -140))) - 8
                ex = torch.where(top > 0, ex.clamp(-127, 127), torch.full_like(ex, -127.0))
                f, kept = torch.exp2(ex), (ex + 127).to(torch.uint8)
            # nearest value of the format, ties to the even code, from the sorted list of its values
            vals = _e4m3_table()[:127]
            y = (x / f.unsqueeze(-1)).float().double()  # the quotient is a float32
            a = y.abs().clamp(max=448.0)
            hi = torch.searchsorted(vals, a.contiguous()).clamp(max=126)
            lo = (hi - 1).clamp(min=0)
            dl, dh = a - vals[lo], vals[hi] - a
            code = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
            code = code + torch.where(torch.signbit(y), 128, 0)
            s[name + "_cache"][page, :, slot] = code.to(torch.uint8).reshape(n, s["Hkv"], -1)
            s[name + "_scales"][page, :, slot] = kept
        if s["track"]:
            s["mass"][b][:, e] = 0.0
            s["positions"][b][:, e] = e.int()
        at += n
    return dict(_cache_out(s), **{n: s[n] for n in ("mass", "positions") if n in s})


def _exact_decode(s, case):
    B, Hq, Hkv, D = s["B"], s["Hq"], s["Hkv"], s["D"]
    G = Hq // Hkv
    out = torch.zeros((B, Hq, D), dtype=torch.float64, device=DEVICE)
    lse = torch.full((B, Hq), NEG, dtype=torch.float64, device=DEVICE)
    mass = torch.zeros((B, Hkv, s["cap"]), dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(_spread(case, case["len_min"], case["len_max"], 1)):
        for h in range(Hkv):
            x = torch.einsum("gd,ld->gl", s["q"][b, h * G:(h + 1) * G].double(), _rows64(s, "k", b, h, n)) * D ** -0.5
            z = torch.logsumexp(x, 1)
            p = torch.exp(x - z[:, None])
            out[b, h * G:(h + 1) * G] = torch.einsum("gl,ld->gd", p, _rows64(s, "v", b, h, n))
            lse[b, h * G:(h + 1) * G] = z
            mass[b, h, :n] = p.sum(0)
    return dict(out=out, lse=lse, **({"mass": mass} if "mass" in s else {}))


def _exact_prompt(s, case):
    new, total = _q_lens(case)
    Hq, G, D = s["Hq"], s["Hq"] // s["Hkv"], s["D"]
    out = torch.zeros((sum(new), Hq, D), dtype=torch.float64, device=DEVICE)
    lse = torch.zeros((sum(new), Hq), dtype=torch.float64, device=DEVICE)
    cq, ck = np.cumsum([0] + new).tolist(), np.cumsum([0] + total).tolist()
    for b, (n, t) in enumerate(zip(new, total)):
        last = torch.arange(t - n, t, device=DEVICE)             # each row's last visible key
        for h in range(Hq):
            k, v = (s[x][ck[b]:ck[b + 1], h // G].double() for x in ("k", "v"))
            for a in range(0, n, 4096):
                z = min(n, a + 4096)
                x = s["q"][cq[b] + a:cq[b] + z, h].double() @ k.T * D ** -0.5
                x = torch.where(torch.arange(t, device=DEVICE) <= last[a:z, None], x, NEG)
                w = torch.logsumexp(x, 1)
                out[cq[b] + a:cq[b] + z, h] = torch.exp(x - w[:, None]) @ v
                lse[cq[b] + a:cq[b] + z, h] = w
    return dict(out=out, lse=lse)


def _exact_evict(s, case):
    page, budget = s["page"], s["budget"]
    mass, pos = s["mass"].cpu().numpy(), s["positions"].cpu().numpy()
    nm, npos, nlen = s["new_mass"].cpu().numpy(), s["new_positions"].cpu().numpy(), []
    for b, n in enumerate(_spread(case, case["len_min"], case["len_max"], 1)):
        m = min(n, budget)
        nlen.append(m)
        table = s["table"][b].long()
        for h in range(s["Hkv"]):
            w, p = mass[b, h, :n].astype(np.float64), pos[b, h, :n]
            w = np.where((p >= n - s["recent"]) | (p < s["sinks"]), np.inf, w)
            kept = np.sort(np.lexsort((np.arange(n), -w))[:m])   # heaviest first, ties to the lower entry
            holes, tails = np.setdiff1d(np.arange(m), kept), kept[kept >= m]
            nm[b, h, :m], npos[b, h, :m] = mass[b, h, :m], pos[b, h, :m]
            nm[b, h, holes], npos[b, h, holes] = mass[b, h, tails], pos[b, h, tails]
            d, t = (torch.from_numpy(a).to(DEVICE) for a in (holes, tails))
            for name in ("k_cache", "v_cache", "k_scales", "v_scales"):
                if s[name] is not None:
                    s[name][table[d // page], h, d % page] = s[name][table[t // page], h, t % page]
    return dict(_cache_out(s), mass=torch.from_numpy(nm), positions=torch.from_numpy(npos), lengths=_ints(nlen))


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "prompt": _exact_prompt,
            "evict": _exact_evict}[case["op"]](s, case)
