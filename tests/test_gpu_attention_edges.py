"""Attention over scores, sums and scales at the ends of their ranges, vs 64-bit results.

The bounds are those of test_gpu_attention.  A key whose score is minus infinity
weighs nothing, so its reference is the same call without that key.
"""
import numpy as np
import pytest
import torch

import whallm_b200 as W
from oracle import attention as A
from tests.test_gpu_attention import Cache, check_lse, check_mass, check_out, f64, gen, rnd, run_prompt

pytestmark = pytest.mark.gpu


def forbid(c, b, keys):
    """Give keys of sequence b a first block of dimensions whose score with a negative query is minus infinity in 32
    bits: an infinite component in bf16 rows, the largest e4m3 values under the largest scale in the others."""
    dev = c.k.device
    e = torch.tensor(keys)
    at, slot = c.table.cpu()[b][e // c.page].long().to(dev), (e % c.page).to(dev)
    if c.fmt == "bf16":
        c.k[at, :, slot, 5] = float("inf")
    else:
        c.k[at, :, slot, :32] = 0x7e                                     # 448
        c.ks[at, :, slot, 0] = 254 if c.fmt == "mxfp8" else 3e38         # 448 x 32 x 2^127 is behind 2^128


@pytest.mark.parametrize("fmt", ["bf16", "fp8_f32_b64", "mxfp8"])
@pytest.mark.parametrize("D,G", [(64, 2), (128, 4), (256, 12), (128, 17)])
@pytest.mark.parametrize("max_pages,mass", [(None, False), (200, False), (None, True)])
def test_decode_keys_of_minus_infinity(dev, fmt, D, G, max_pages, mass):
    # single keys at a tile's start and end, a tile's only key, whole tiles and units, all but the last key; over a
    # cluster and over the line
    lens = [17, 33, 2, 200, 1000, 130, 65, 64]
    dead = [[16], [32], [0], range(16), [*range(0, 400), 999], [*range(0, 64), *range(80, 96), 128, 129], range(64),
            [*range(16, 32), 63]]
    Hkv = 2
    c = Cache(dev, lens, Hkv, D, 64, fmt, seed=D + G, max_pages=max_pages)
    for b, keys in enumerate(dead):
        forbid(c, b, list(keys))
    q = rnd(gen(7, dev), len(lens), G * Hkv, D, std=2.0, dev=dev)
    q[:, :, :64] = -q[:, :, :64].abs() - 0.25
    m = torch.rand((len(lens), Hkv, c.width * 64), generator=gen(8, dev), device=dev) if mass else None
    before = m.clone() if mass else None
    out, lse = W.decode_attention(q, *c.args, mass=m, return_lse=True)
    for b, n in enumerate(lens):
        live = [j for j in range(n) if j not in set(dead[b])]
        ref = A.attend(f64(q[b:b + 1]), *(x[live] for x in c.rows[b]), D ** -0.5)
        check_out(out[b:b + 1], ref, D)
        check_lse(lse[b:b + 1], ref, D)
        if mass:
            check_mass(f64(m[b, :, live]), ref, D, f64(before[b, :, live]))
            gone = list(dead[b])
            assert torch.equal(m[b, :, gone], before[b, :, gone])


@pytest.mark.parametrize("D,G", [(64, 3), (128, 4), (256, 12)])
@pytest.mark.parametrize("max_pages", [None, 300])
def test_decode_values_that_are_not_finite(dev, D, G, max_pages):
    # a live value shows in its dimension and its kv head's rows, a NaN key in its kv head's; nowhere else
    Hkv, lens = 2, [40, 500, 17]
    c = Cache(dev, lens, Hkv, D, 64, "bf16", seed=D, max_pages=max_pages)
    q = rnd(gen(10, dev), len(lens), G * Hkv, D, dev=dev)
    want, lse = W.decode_attention(q, *c.args, return_lse=True)
    for bad in (float("inf"), float("-inf"), float("nan")):
        v = c.v.clone()
        v[c.table[1, 3], 1, 9, D - 2] = bad
        got, l2 = W.decode_attention(q, c.k, v, *c.args[2:], return_lse=True)
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[1, G:, D - 2] = True
        assert torch.equal(got[~hit], want[~hit]) and torch.equal(l2, lse)
        assert (torch.isnan(got[hit]) if bad != bad else got[hit] == bad).all()
    k = c.k.clone()
    k[c.table[1, 3], 1, 9, 0] = float("nan")
    got, l2 = W.decode_attention(q, k, c.v, *c.args[2:], return_lse=True)
    hit = torch.zeros_like(lse, dtype=torch.bool)
    hit[1, G:] = True
    assert torch.equal(got[~hit], want[~hit]) and torch.equal(l2[~hit], lse[~hit])
    assert torch.isnan(got[hit]).all() and torch.isnan(l2[hit]).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nq,nk,Hq,Hkv", [
    ([4], [256], 8, 2), ([4, 3], [257, 390], 4, 1),                      # blocks of one tile
    ([300], [256], 4, 4), ([300, 140], [256, 384], 8, 4),                # blocks of two
    ([4], [4096], 4, 2), ([300], [5000], 2, 2),                          # keys in parts
])
@pytest.mark.parametrize("tile", [0, 1])
def test_prompt_tile_of_nan_keys(dev, D, nq, nk, Hq, Hkv, tile):
    """128 keys of NaN, before or behind finite ones: the rows that see them are NaN, their lse too."""
    g = gen(60 + D, dev)
    q, k, v = rnd(g, sum(nq), Hq, D, dev=dev), rnd(g, sum(nk), Hkv, D, dev=dev), rnd(g, sum(nk), Hkv, D, dev=dev)
    at = 0
    for n in nk:
        k[at + 128 * tile:at + 128 * (tile + 1), 0] = float("nan")
        at += n
    cu = lambda n: torch.tensor(np.cumsum([0] + n), dtype=torch.int32, device=dev)  # noqa: E731
    out, lse = W.prompt_attention(q, k, v, cu(nq), cu(nk), causal=False, return_lse=True)
    G = Hq // Hkv
    assert torch.isnan(out[:, :G]).all() and torch.isnan(lse[:, :G]).all()
    assert torch.isfinite(out[:, G:]).all() and torch.isfinite(lse[:, G:]).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nq,nk,Hq,Hkv", [
    ([1, 2, 1, 0, 1] * 8, [0, 1, 0, 3, 0] * 8, 8, 8),                    # one-tile blocks, most of them without keys
    ([1] * 60, [0] * 60, 64, 8),
    ([300, 5, 260] * 12, [0, 5, 0] * 12, 8, 8),                          # two-tile blocks
    ([900, 700], [100, 650], 32, 8),                                     # rows in front of a sequence's keys
])
def test_prompt_blocks_without_keys_in_a_row(dev, D, nq, nk, Hq, Hkv):
    # more blocks than SMs, so that a CTA gets several without a key, one after the other; each call once more while
    # the caches are warm
    q, k, v, out, lse = run_prompt(dev, nq, nk, Hq, Hkv, D, seed=70)
    cu = lambda n: torch.tensor(np.cumsum([0] + n), dtype=torch.int32, device=dev)  # noqa: E731
    cq, ck = cu(nq), cu(nk)
    for _ in range(300):
        again, lse2 = W.prompt_attention(q, k, v, cq, ck, return_lse=True)
        torch.cuda.synchronize()
        assert torch.equal(lse2, lse) and torch.equal(again, out)


@pytest.mark.parametrize("fmt,D", [("fp8_f32_b64", 128), ("fp8_f32_b64", 256), ("mxfp8", 64), ("mxfp8", 128), ("mxfp8", 256)])
@pytest.mark.parametrize("G,max_pages,mass", [(4, None, False), (9, None, False), (4, 300, False), (16, 300, True)])
def test_decode_blocks_of_far_apart_scales(dev, fmt, D, G, max_pages, mass):
    # every block of value dimensions in a range of its own, up to 2^100 apart: each is as exact as alone
    lens = [1, 16, 17, 100, 700]
    Hkv = 2
    c = Cache(dev, lens, Hkv, D, 64, fmt, seed=D + G, max_pages=max_pages)
    blocks = c.vs.shape[-1]
    e = np.random.RandomState(D + G).randint(-60, 41, (len(lens), Hkv, blocks))
    e[:, :, 0], e[:, :, 1] = 40, -60
    for b, n in enumerate(lens):
        f = torch.tensor(e[b], device=dev)
        for p in c.table[b, :-(-n // 64)].tolist():
            if fmt == "mxfp8":
                c.vs[p] = (c.vs[p].int() + f[:, None, :]).clamp(0, 254).to(torch.uint8)
            else:
                c.vs[p] *= torch.exp2(f.double()).float()[:, None, :]
        c.rows[b][1] = (c.rows[b][1].reshape(n, Hkv, blocks, -1) * 2.0 ** e[b][None, :, :, None]).reshape(n, Hkv, D)
    q = rnd(gen(9, dev), len(lens), G * Hkv, D, std=2.0, dev=dev)
    m = torch.zeros((len(lens), Hkv, c.width * 64), device=dev) if mass else None
    out, lse = W.decode_attention(q, *c.args, mass=m, return_lse=True)
    for b in range(len(lens)):
        ref = A.attend(f64(q[b:b + 1]), *c.rows[b], D ** -0.5)
        check_out(out[b:b + 1], ref, D)
        check_lse(lse[b:b + 1], ref, D)


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
def test_captured_steps_go_on_with_the_class(dev, fmt):
    """reserve, captured steps, refresh, reserve, more of them over page borders, evict, append: the same cache as one
    that only the class's own calls filled."""
    B, Hkv, Hq, D, page = 3, 2, 8, 64, 16
    g = gen(71, dev)
    a, b = (W.PagedKVCache(B, Hkv, D, n_pages=20, page_size=page, max_pages=8, fmt=fmt, track=True) for _ in range(2))
    start = [rnd(g, 34, Hkv, D, dev=dev) for _ in range(2)]
    for c in (a, b):
        c.append(*start, [16, 15, 3])
    cu = torch.arange(B + 1, dtype=torch.int32, device=dev)
    q, k, v = (torch.zeros((B, h, D), dtype=torch.bfloat16, device=dev) for h in (Hq, Hkv, Hkv))

    def step(c):
        c.lengths.add_(1)
        c.seen.add_(1)
        W.paged_append(k, v, cu, c.keys, c.values, c.page_table, c.lengths, c.fmt, c.key_scales, c.value_scales, c.mass,
                       c.positions, c.seen)
        return W.decode_attention(q, c.keys, c.values, c.page_table, c.lengths, c.fmt, c.key_scales, c.value_scales,
                                  mass=c.mass)

    spare = W.PagedKVCache(B, Hkv, D, n_pages=3, page_size=page, max_pages=8, fmt=fmt, track=True)
    spare.reserve([1] * B)
    step(spare)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = step(b)

    def feed():
        for t in (q, k, v):
            t.copy_(rnd(g, *t.shape, dev=dev))

    for _ in range(3):                               # 3 x 8 steps: each run of them ends in new pages
        b.reserve([8] * B)
        for _ in range(8):
            feed()
            a.append(k, v)
            want = a.attend(q)
            gr.replay()
            assert torch.equal(out, want) and torch.isfinite(out).all()
        b.refresh()
        assert a.offsets == b.offsets == a.lengths.tolist()
    for c in (a, b):
        c.evict(24, recent=4, sinks=1)
    assert a.offsets == b.offsets == [24, 24, 24] == b.lengths.tolist() and a.free_pages == b.free_pages
    feed()
    outs = []
    for c in (a, b):
        c.append(k, v)
        outs.append(c.attend(q))
    assert torch.equal(*outs) and torch.isfinite(outs[0]).all()
    for x in range(B):
        assert torch.equal(a.mass[x, :, :25], b.mass[x, :, :25]) and torch.equal(a.positions[x, :, :25], b.positions[x, :, :25])
