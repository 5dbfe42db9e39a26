"""Paged-cache and prompt attention, cache append and eviction vs 64-bit results.

Error bounds (fixed before the first run; u = half a step):
* a weight p is rounded to bf16 once (u = 2^-8) before it meets v: at most
  2^-8 * spread, spread = sum_j w_j |v_j|; the output is rounded once: 2^-8 |out|;
* a score is a 32-bit sum of D exact products: at most (D + 2) 2^-23 mag,
  mag = scale sum |q||k|, and moves a weight relatively by e^(2 err) - 1 (its own
  score and the normaliser's).  2^-23 rather than 2^-24 allows for sums that are
  cut instead of rounded; exp2 and log2 add at most 2^-20 in all.
Rows that only move (append, evict) must be equal.
"""
import numpy as np
import pytest
import torch

import whallm_b200 as W
from oracle import attention as A

pytestmark = pytest.mark.gpu

FMTS = ["bf16", "fp8_f32_b64", "mxfp8"]


def rnd(g, *shape, std=1.0, dev="cuda"):
    return (torch.randn(shape, generator=g, device=dev) * std).to(torch.bfloat16)


def gen(seed, dev="cuda"):
    return torch.Generator(device=dev).manual_seed(seed)


def f64(t):
    return t.double().cpu().numpy()


def score_err(ref, D):
    return (D + 2) * 2.0 ** -23 * ref["mag"]


def check_out(out, ref, D):
    weight_err = np.expm1(2 * score_err(ref, D)) + 2.0 ** -20
    tol = 2.0 ** -8 * (np.abs(ref["out"]) + ref["spread"]) * (1 + 2.0 ** -7) + weight_err[..., None] * ref["spread"]
    err = np.abs(f64(out) - ref["out"])
    assert np.all(np.isfinite(f64(out))), "not finite"
    assert np.all(err <= tol), float((err - tol).max())


def check_lse(lse, ref, D):
    got = f64(lse)
    assert np.array_equal(np.isneginf(got), np.isneginf(ref["lse"]))
    fin = np.isfinite(ref["lse"])
    tol = score_err(ref, D) + 2.0 ** -20 * (1 + np.abs(ref["lse"]))
    assert np.all(np.abs(got[fin] - ref["lse"][fin]) <= tol[fin])


def check_mass(mass, ref, D, before=0.0):
    e = np.expm1(2 * score_err(ref, D).max()) + 2.0 ** -18
    assert np.all(np.abs(mass - before - ref["weight"]) <= e * ref["weight"] + 2.0 ** -23 * np.abs(before) + 1e-30)


class Cache:
    """A page pool full of NaN with the rows of a batch spread over it, and the rows' values in 64 bits."""

    def __init__(self, dev, lens, Hkv, D, page, fmt, seed=0, spare=3, std=1.0, max_pages=None):
        g = gen(seed, dev)
        self.lens, self.page, self.fmt, self.D, self.Hkv = lens, page, fmt, D, Hkv
        per = [-(-n // page) for n in lens]
        self.width = max_pages or max(max(per), 1)
        total = sum(per) + spare
        order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        shape = (total, Hkv, page, D)
        if fmt == "bf16":
            self.k, self.v = (torch.full(shape, float("nan"), dtype=torch.bfloat16, device=dev) for _ in range(2))
            self.ks = self.vs = None
        else:
            blk = 64 if fmt == "fp8_f32_b64" else 32
            self.k, self.v = (torch.full(shape, 0x7f, dtype=torch.uint8, device=dev) for _ in range(2))
            fill = (torch.float32, float("nan")) if blk == 64 else (torch.uint8, 255)
            self.ks, self.vs = (torch.full((*shape[:3], D // blk), fill[1], dtype=fill[0], device=dev) for _ in range(2))
        self.rows = []
        for b, n in enumerate(lens):
            pages = [order.pop() for _ in range(per[b])]
            table[b, :per[b]] = torch.tensor(pages, dtype=torch.int32)
            pair = []
            for cache, scales in ((self.k, self.ks), (self.v, self.vs)):
                x = rnd(g, n, Hkv, D, std=std, dev=dev)
                e = torch.arange(n)
                at, slot = table[b][e // page].long().to(dev), (e % page).to(dev)
                if fmt == "bf16":
                    cache[at, :, slot] = x
                    pair.append(f64(x))
                else:
                    p, s = W.kv_quantize(x, fmt)
                    cache[at, :, slot] = p
                    scales[at, :, slot] = s
                    val = p.view(torch.float8_e4m3fn).double().reshape(n, Hkv, D // blk, blk)
                    f = s.double() if blk == 64 else torch.exp2(s.double() - 127)
                    pair.append((val * f.unsqueeze(-1)).reshape(n, Hkv, D).cpu().numpy())
            self.rows.append(pair)
        self.table = table.to(dev)
        self.lengths = torch.tensor(lens, dtype=torch.int32, device=dev)

    @property
    def args(self):
        return (self.k, self.v, self.table, self.lengths, self.fmt, self.ks, self.vs)


def run_decode(dev, lens, Hq, Hkv, D, page, fmt, seed=0, mass=False, scale=None, std=1.0, max_pages=None):
    c = Cache(dev, lens, Hkv, D, page, fmt, seed, std=std, max_pages=max_pages)
    q = rnd(gen(seed + 1, dev), len(lens), Hq, D, std=2.0, dev=dev)
    m = torch.rand((len(lens), Hkv, c.width * page), generator=gen(seed + 2, dev), device=dev) if mass else None
    before = m.clone() if mass else None
    out, lse = W.decode_attention(q, *c.args, scale=scale, mass=m, return_lse=True)
    for b, n in enumerate(lens):
        ref = A.attend(f64(q[b:b + 1]), *c.rows[b], scale or D ** -0.5)
        check_out(out[b:b + 1], ref, D)
        check_lse(lse[b:b + 1], ref, D)
        if mass:
            check_mass(f64(m[b, :, :n]), ref, D, f64(before[b, :, :n]))
            assert torch.equal(m[b, :, n:], before[b, :, n:])
    return c, q, out, lse


RAGGED = [1, 0, 15, 16, 17, 63, 64, 65, 130, 997]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(8, 8), (32, 4), (16, 1)])
def test_decode_vs_64_bits(dev, fmt, D, Hq, Hkv):
    run_decode(dev, RAGGED, Hq, Hkv, D, 64, fmt, seed=D + Hq)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(6, 2), (16, 1)])
def test_decode_long_capacity(dev, fmt, D, Hq, Hkv):
    # a capacity that is split over the GPU whatever the lengths: few and many parts per pair
    run_decode(dev, [9000, 0, 3, 64, 65, 2000], Hq, Hkv, D, 64, fmt, seed=D + Hq + 1)
    run_decode(dev, [4100], Hq, Hkv, D, 128, fmt, seed=D + Hq + 2, max_pages=100)


def test_decode_long_capacity_batch(dev):
    r = np.random.RandomState(5)
    run_decode(dev, [int(x) for x in r.randint(0, 900, 90)], 8, 4, 64, 64, "mxfp8", seed=6, max_pages=200)
    run_decode(dev, [0, 0, 0], 8, 4, 64, 64, "bf16", seed=7, max_pages=200)


@pytest.mark.parametrize("G", [1, 3, 5, 7, 9, 12, 17, 40])
def test_decode_group_sizes(dev, G):
    run_decode(dev, [33, 700], 2 * G, 2, 128, 32, "bf16", seed=G, mass=True)


@pytest.mark.parametrize("page", [16, 48, 128, 1024])
@pytest.mark.parametrize("fmt", FMTS)
def test_decode_page_sizes(dev, page, fmt):
    run_decode(dev, [page - 1, page, page + 1, 3 * page + 5], 8, 2, 64, page, fmt, seed=page)


@pytest.mark.parametrize("fmt,D,G", [("bf16", 128, 4), ("fp8_f32_b64", 256, 8), ("mxfp8", 64, 16), ("bf16", 256, 20)])
def test_decode_collects_weights(dev, fmt, D, G):
    run_decode(dev, [0, 1, 47, 2048, 2049, 5000], 2 * G, 2, D, 64, fmt, seed=9, mass=True)


def test_decode_many_sequences(dev):
    # more sequences than a warp has lanes, and more pairs than CTAs
    r = np.random.RandomState(3)
    run_decode(dev, [int(x) for x in r.randint(0, 150, 300)], 8, 4, 64, 16, "bf16", seed=4, mass=True)


@pytest.mark.parametrize("n", [20011, 70001])
def test_decode_long(dev, n):
    run_decode(dev, [n], 8, 1, 128, 64, "fp8_f32_b64", seed=5, mass=True)


@pytest.mark.parametrize("B", [1, 2, 9, 20, 40, 80, 160])
def test_decode_short_caches(dev, B):
    # clusters of 8, 4, 2 and 1 CTAs per (sequence, head), lengths from nothing to a few units per CTA
    r = np.random.RandomState(B)
    run_decode(dev, [int(x) for x in r.randint(0, 1025, B - 1)] + [0 if B == 1 else 1024], 4, 2, 64, 64, FMTS[B % 3], seed=B)


@pytest.mark.parametrize("cap", [8192, 8256])
@pytest.mark.parametrize("fmt,D,G", [("bf16", 128, 4), ("mxfp8", 256, 12)])
def test_decode_at_the_cluster_limit(dev, cap, fmt, D, G):
    # the longest capacity that one cluster joins, and the next page
    run_decode(dev, [5, cap - 3], 2 * G, 2, D, 64, fmt, seed=cap)


@pytest.mark.parametrize("fmt,D,Hq,Hkv,mass", [("bf16", 128, 8, 2, False), ("mxfp8", 64, 4, 1, True), ("fp8_f32_b64", 256, 8, 4, False)])
def test_decode_in_rounds(dev, fmt, D, Hq, Hkv, mass):
    # enough units for three rounds of CTAs: their borders fall inside pairs, and some pairs inside one CTA
    r = np.random.RandomState(8)
    want = 64 * 592 * 64 // Hkv                                  # keys for the largest number of CTAs in a round
    lens = [int(x) for x in r.randint(1, 2 * want // 40, 44)] + [0, 1, 70, 0]
    c = Cache(dev, lens, Hkv, D, 64, fmt, seed=12)
    q = rnd(gen(13, dev), len(lens), Hq, D, std=2.0, dev=dev)
    m = torch.zeros((len(lens), Hkv, c.width * 64), device=dev) if mass else None
    out, lse = W.decode_attention(q, *c.args, mass=m, return_lse=True)
    for b in (0, 7, 20, 33, 43, 44, 45, 46, 47):
        ref = A.attend(f64(q[b:b + 1]), *c.rows[b], D ** -0.5)
        check_out(out[b:b + 1], ref, D)
        check_lse(lse[b:b + 1], ref, D)
        if mass:
            check_mass(f64(m[b, :, :lens[b]]), ref, D)
    for b in range(len(lens)):                                   # and every sequence as when it is alone
        one = W.decode_attention(q[b:b + 1], c.k, c.v, c.table[b:b + 1], c.lengths[b:b + 1], fmt, c.ks, c.vs)
        assert (one.float() - out[b:b + 1].float()).abs().max() <= 2.0 ** -6 * out[b].float().abs().max() + 1e-6


@pytest.mark.parametrize("mass", [False, True])
def test_decode_more_parts_than_join_threads(dev, mass):
    # one pair over every CTA: 592 parts, more than the join holds factors for at once
    run_decode(dev, [90001], 1, 1, 64, 64, "mxfp8", seed=11, mass=mass)


def test_decode_large_scores(dev):
    # scores of deviation ~60: nearly one-hot weights, running maxima that grow late
    run_decode(dev, [300, 5], 8, 2, 128, 16, "bf16", seed=6, scale=2.0, std=1.5)


def test_decode_offsets_past_32_bits(dev):
    # a pool of more than 2^32 bytes, the sequence's pages at both of its ends
    D, Hkv, page, n = 256, 8, 64, 200
    pages = (1 << 32) // (page * Hkv * D * 2) + 64
    k, v = (torch.zeros((pages, Hkv, page, D), dtype=torch.bfloat16, device=dev) for _ in range(2))
    g = gen(8, dev)
    x, y = rnd(g, n, Hkv, D, dev=dev), rnd(g, n, Hkv, D, dev=dev)
    table = torch.tensor([[pages - 1, 0, pages - 2, pages // 2]], dtype=torch.int32, device=dev)
    ln = torch.tensor([n], dtype=torch.int32, device=dev)
    W.paged_append(x, y, torch.tensor([0, n], dtype=torch.int32, device=dev), k, v, table, ln)
    assert torch.equal(k[pages - 1].transpose(0, 1), x[:page]) and torch.equal(v[pages // 2, :, :8].transpose(0, 1), y[192:])
    q = rnd(g, 1, Hkv, D, dev=dev)
    ref = A.attend(f64(q), f64(x), f64(y), D ** -0.5)
    check_out(W.decode_attention(q, k, v, table, ln), ref, D)


def test_decode_repeats_and_strides(dev):
    c, q, out, lse = run_decode(dev, RAGGED, 16, 2, 128, 64, "mxfp8", seed=12)
    again, lse2 = W.decode_attention(q, *c.args, return_lse=True)
    assert torch.equal(again, out) and torch.equal(lse2, lse)
    wide = torch.zeros((len(RAGGED), 20, 128), dtype=torch.bfloat16, device=dev)
    wide[:, :16] = q                                      # the queries of a joint projection
    buf = torch.empty_like(out)
    assert W.decode_attention(wide[:, :16], *c.args, out=buf) is buf and torch.equal(buf, out)


def test_decode_bad_lengths_and_pages(dev):
    # reported as NaN by the kernel's own range checks; nothing is read through them
    c = Cache(dev, [100, 100, 100, 100, 100], 2, 64, 16, "bf16", seed=13)
    q = rnd(gen(14, dev), 5, 4, 64, dev=dev)
    good = W.decode_attention(q, *c.args)
    c.lengths[0] = -1
    c.lengths[1] = c.width * c.page + 1
    c.table[2, 3] = c.k.shape[0]
    c.table[3, 6] = -7
    mass = torch.zeros((5, 2, c.width * c.page), device=dev)
    out, lse = W.decode_attention(q, *c.args, mass=mass, return_lse=True)
    assert torch.isnan(out[:4]).all() and torch.isnan(lse[:4]).all()
    assert torch.equal(out[4], good[4]) and torch.isfinite(mass[4]).all()


@pytest.mark.parametrize("max_pages", [None, 300])
def test_decode_captured_follows_lengths(dev, max_pages):
    """Two graphs, one pool: each follows the lengths and tables as they are at its replay."""
    c = Cache(dev, [500, 60, 0], 2, 128, 32, "bf16", seed=15, max_pages=max_pages)
    q = rnd(gen(16, dev), 3, 8, 128, dev=dev)
    W.decode_attention(q, *c.args)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = W.decode_attention(q, *c.args)
        graphs.append((gr, out))
    for lens in ([500, 60, 0], [1, 0, 0], [450, 17, 0]):
        c.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        want = W.decode_attention(q, *c.args)
        for gr, out in graphs:
            out.fill_(7.0)
            gr.replay()
        for _, out in graphs:
            assert torch.equal(out, want)


@pytest.mark.parametrize("max_pages", [None, 600])
def test_decode_on_two_streams(dev, max_pages):
    """Calls on two streams at once: each has its own workspace."""
    cs = [Cache(dev, [300 + 50 * i, 17], 2, 64, 16, "bf16", seed=17 + i, max_pages=max_pages) for i in range(2)]
    qs = [rnd(gen(18 + i, dev), 2, 4, 64, dev=dev) for i in range(2)]
    want = [W.decode_attention(q, *c.args) for q, c in zip(qs, cs)]
    sides = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(30):
        for i, s in enumerate(sides):
            with torch.cuda.stream(s):
                outs[i].append(W.decode_attention(qs[i], *cs[i].args))
    for s in sides:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i])


@pytest.mark.parametrize("fmt,max_pages", [("bf16", 8), ("mxfp8", 300)])
def test_captured_step(dev, fmt, max_pages):
    """A whole decode step in a graph -- lengths, append, attention with weights -- replayed over new inputs, gives
    the eager steps' results; the eviction after it likewise."""
    B, Hkv, Hq, D, page = 3, 2, 8, 128, 16
    g = gen(61, dev)

    def cache():
        c = W.PagedKVCache(B, Hkv, D, n_pages=30, page_size=page, max_pages=max_pages, fmt=fmt, track=True)
        c.reserve([100, 40, 9])
        return c

    a, b = cache(), cache()
    b.page_table.copy_(a.page_table)
    start = [rnd(gen(62 + i, dev), 90, Hkv, D, dev=dev) for i in range(2)]
    for c in (a, b):
        c.append(*start, [60, 30, 0])
    cu = torch.arange(B + 1, dtype=torch.int32, device=dev)
    qkv = torch.zeros((B, Hq + 2 * Hkv, D), dtype=torch.bfloat16, device=dev)

    def step(c):
        q, k, v = qkv.split([Hq, Hkv, Hkv], dim=1)
        c.lengths.add_(1)
        c.seen.add_(1)
        W.paged_append(k, v, cu, c.keys, c.values, c.page_table, c.lengths, c.fmt, c.key_scales, c.value_scales, c.mass,
                       c.positions, c.seen)
        return W.decode_attention(q, c.keys, c.values, c.page_table, c.lengths, c.fmt, c.key_scales, c.value_scales,
                                  mass=c.mass)

    warm = cache()
    step(warm)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = step(b)
    for _ in range(9):
        qkv.copy_(rnd(g, B, Hq + 2 * Hkv, D, dev=dev))
        want = step(a)
        gr.replay()
        assert torch.equal(out, want)
    live = [69, 39, 9]
    assert a.lengths.tolist() == live == b.lengths.tolist()
    outs = []
    for c in (a, b):
        new = torch.zeros_like(c.lengths)
        args = (c.keys, c.values, c.page_table, c.lengths, c.mass, c.positions, c.seen, 32, 8, 2, c.fmt, c.key_scales,
                c.value_scales, (c.mass, c.positions, new))
        if c is b:
            ev = torch.cuda.CUDAGraph()
            with torch.cuda.graph(ev):
                W.paged_evict(*args)
            ev.replay()
        else:
            W.paged_evict(*args)
        c.lengths.copy_(new)
        outs.append(W.decode_attention(qkv[:, :Hq], c.keys, c.values, c.page_table, c.lengths, c.fmt, c.key_scales,
                                       c.value_scales))
    assert a.lengths.tolist() == [32, 32, 9] == b.lengths.tolist()
    assert torch.equal(outs[0], outs[1])
    for x, n in enumerate([32, 32, 9]):
        assert torch.equal(a.mass[x, :, :n], b.mass[x, :, :n]) and torch.equal(a.positions[x, :, :n], b.positions[x, :, :n])


# ------------------------------------------------------------------ prompts --

def run_prompt(dev, nq, nk, Hq, Hkv, D, causal=True, seed=0, joint=False, std=1.0, scale=None):
    g = gen(seed, dev)
    Tq, Tk = sum(nq), sum(nk)
    if joint:
        x = rnd(g, Tq, Hq + 2 * Hkv, D, std=std, dev=dev)
        q, k, v = x.split([Hq, Hkv, Hkv], dim=1)
    else:
        q, k, v = rnd(g, Tq, Hq, D, std=2 * std, dev=dev), rnd(g, Tk, Hkv, D, std=std, dev=dev), rnd(g, Tk, Hkv, D, std=std, dev=dev)
    cu = lambda n: torch.tensor(np.cumsum([0] + list(n)), dtype=torch.int32, device=dev)  # noqa: E731
    out, lse = W.prompt_attention(q, k, v, cu(nq), None if joint else cu(nk), causal=causal, scale=scale, return_lse=True)
    a = b = 0
    for x, y in zip(nq, nk):
        ref = A.attend(f64(q[a:a + x]), f64(k[b:b + y]), f64(v[b:b + y]), scale or D ** -0.5, causal)
        if x:
            check_out(out[a:a + x], ref, D)
            check_lse(lse[a:a + x], ref, D)
        a, b = a + x, b + y
    return q, k, v, out, lse


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (8, 1)])
def test_prompt_packed(dev, D, Hq, Hkv):
    n = [1, 2, 127, 0, 128, 129, 300, 31]
    run_prompt(dev, n, n, Hq, Hkv, D, seed=D + Hq, joint=True)


@pytest.mark.parametrize("G", [3, 5, 6, 16, 40])
def test_prompt_group_sizes(dev, G):
    n = [50, 140]
    run_prompt(dev, n, n, 2 * G, 2, 64, seed=G)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_continues_a_history(dev, D):
    run_prompt(dev, [1, 40, 130, 0, 3], [600, 41, 130, 50, 1030], 8, 2, D, seed=21)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_rows_without_keys(dev, D):
    # more rows than keys: the first rows see nothing; a sequence without keys sees nothing at all
    run_prompt(dev, [200, 5, 70], [60, 0, 69], 4, 2, D, seed=22)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_full(dev, D):
    run_prompt(dev, [5, 129, 260], [300, 1, 257], 4, 1, D, causal=False, seed=23)


@pytest.mark.parametrize("D,n", [(64, 1500), (128, 1111), (256, 900)])
def test_prompt_long(dev, D, n):
    run_prompt(dev, [n], [n], 2, 1, D, seed=24)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_many_sequences(dev, D):
    # more sequences than a warp has lanes and more blocks than SMs, with and without keys
    r = np.random.RandomState(D)
    nq = [int(x) for x in r.randint(0, 40, 75)]
    nk = [max(0, n + int(d)) for n, d in zip(nq, r.randint(-20, 60, 75))]
    run_prompt(dev, nq, nk, 8, 4, D, seed=29)


@pytest.mark.parametrize("D,Hkv", [(64, 8), (128, 8), (256, 4)])
def test_prompt_blocks_handed_on(dev, D, Hkv):
    # several blocks per SM, long and short ones in turn: the same rows as when each sequence is alone
    n = [700, 3, 400, 1, 129, 900]
    g = gen(30, dev)
    q, k, v = (rnd(g, sum(n), h, D, dev=dev) for h in (2 * Hkv, Hkv, Hkv))
    cu = torch.tensor(np.cumsum([0] + n), dtype=torch.int32, device=dev)
    out = W.prompt_attention(q, k, v, cu)
    at = 0
    for x in n:
        one = torch.tensor([0, x], dtype=torch.int32, device=dev)
        assert torch.equal(W.prompt_attention(q[at:at + x], k[at:at + x], v[at:at + x], one), out[at:at + x])
        at += x


def test_prompt_malformed_sequence_bounds(dev):
    """Bounds outside the tensors are cut to them; bounds that run backwards are empty sequences."""
    g = gen(31, dev)
    q, k, v = (rnd(g, 100, h, 64, dev=dev) for h in (4, 2, 2))
    good = torch.tensor([0, 40, 100], dtype=torch.int32, device=dev)
    want = W.prompt_attention(q, k, v, good)
    cut = torch.tensor([-5, 40, 5000], dtype=torch.int32, device=dev)
    assert torch.equal(W.prompt_attention(q, k, v, cut), want)
    out = torch.full_like(q, 7.0)
    W.prompt_attention(q, k, v, torch.tensor([0, 40, 20, 20], dtype=torch.int32, device=dev), out=out)
    assert torch.equal(out[:40], want[:40]) and (out[40:] == 7.0).all()


def test_prompt_large_scores(dev):
    run_prompt(dev, [400], [400], 4, 2, 128, seed=25, std=2.0, scale=1.0)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_padding_and_neighbours(dev, D):
    """Rows outside every sequence stay as they were, and what stands behind a sequence's keys does not reach it."""
    g = gen(26, dev)
    q, k, v = (rnd(g, 300, h, D, dev=dev) for h in (4, 2, 2))
    cu = torch.tensor([0, 70, 201], dtype=torch.int32, device=dev)
    want = W.prompt_attention(q, k, v, cu)
    out = torch.full_like(q, 7.0)
    k2, v2, q2 = k.clone(), v.clone(), q.clone()
    for t in (k2, v2, q2):
        t[201:] = float("nan")
    assert W.prompt_attention(q2, k2, v2, cu, out=out) is out
    assert torch.equal(out[:201], want[:201]) and (out[201:] == 7.0).all()
    k2[70:201], v2[70:201] = float("inf"), float("nan")
    assert torch.equal(W.prompt_attention(q2, k2, v2, cu)[:70], want[:70])
    cu2 = torch.tensor([70, 201], dtype=torch.int32, device=dev)       # a first sequence that does not begin at 0
    out = torch.full_like(q, 7.0)
    W.prompt_attention(q, k, v, cu2, out=out)
    assert torch.equal(out[70:201], want[70:201]) and (out[:70] == 7.0).all()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_later_rows_do_not_reach_earlier_ones(dev, D):
    """A key or value that is not finite shows in the rows that see it and in no other."""
    g = gen(27, dev)
    q, k, v = (rnd(g, 400, h, D, dev=dev) for h in (4, 2, 2))
    cu = torch.tensor([0, 400], dtype=torch.int32, device=dev)
    want = W.prompt_attention(q, k, v, cu)
    for bad in (float("nan"), float("inf"), float("-inf")):
        k2, v2 = k.clone(), v.clone()
        v2[150, 1, D - 1] = bad
        v2[301, 0, 3] = bad
        got = W.prompt_attention(q, k2, v2, cu)
        assert torch.equal(got[:150], want[:150]) and torch.equal(got[150:301, :2], want[150:301, :2])
        assert torch.equal(got[150:, 2:, :D - 1], want[150:, 2:, :D - 1])
        if bad == bad:
            assert (got[150:, 2:, D - 1] == bad).all() and (got[301:, :2, 3] == bad).all()
        else:
            assert torch.isnan(got[150:, 2:, D - 1]).all() and torch.isnan(got[301:, :2, 3]).all()
        k2[201, 1, 5] = float("nan")
        got = W.prompt_attention(q, k2, v, cu)
        assert torch.equal(got[:201], want[:201]) and torch.equal(got[:, :2], want[:, :2])
        assert torch.isnan(got[201:, 2:]).all()


def test_prompt_repeats_and_captures(dev):
    n = [300, 77, 513]
    q, k, v, out, _ = run_prompt(dev, n, n, 8, 2, 128, seed=28)
    cu = torch.tensor(np.cumsum([0] + n), dtype=torch.int32, device=dev)
    assert torch.equal(W.prompt_attention(q, k, v, cu), out)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = W.prompt_attention(q, k, v, cu)
    for lens in ([300, 77, 513], [10, 800, 80]):
        cu.copy_(torch.tensor(np.cumsum([0] + lens), dtype=torch.int32))
        want = W.prompt_attention(q, k, v, cu)
        got.fill_(7.0)
        gr.replay()
        assert torch.equal(got, want)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nq,nk,Hq,Hkv", [
    ([64], [9000], 8, 2), ([1], [30011], 4, 1),                          # one block a head, many parts
    ([1, 40, 0, 130, 5, 3], [5000, 41, 30, 130, 9001, 0], 6, 2),         # ragged; q not by TMA; sequences without rows or keys
    ([300, 70], [4200, 60], 4, 4),                                       # rows without keys beside split ones
    ([1000], [5000], 16, 1), ([4500], [4500], 2, 2),                     # blocks of very different lengths
])
def test_prompt_few_rows_on_many_keys(dev, D, nq, nk, Hq, Hkv):
    run_prompt(dev, nq, nk, Hq, Hkv, D, seed=40 + D)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nq,nk,Hq,Hkv", [
    ([32] * 20, [700 + 3 * i for i in range(20)], 8, 2),                 # one full tile each, several keys' tiles
    ([1] * 30 + [400], [300] * 30 + [900], 12, 3),                       # a long one among single rows: several blocks
    ([5, 0, 1, 33, 2], [5, 9, 0, 33, 128], 7, 1),                        # q not by TMA; no rows, no keys
    ([100] * 150, [129] * 150, 1, 1),                                    # more blocks than SMs
])
def test_prompt_one_tile_blocks(dev, D, nq, nk, Hq, Hkv):
    run_prompt(dev, nq, nk, Hq, Hkv, D, seed=50 + D)
    run_prompt(dev, nq, nk, Hq, Hkv, D, causal=False, seed=51 + D)


def test_prompt_split_full_and_many_sequences(dev):
    run_prompt(dev, [5, 129], [6000, 4097], 4, 1, 128, causal=False, seed=41)
    nq = [3] * 40                                                        # more sequences than a warp's lanes
    run_prompt(dev, nq, [10 + 60 * i for i in range(40)], 4, 2, 64, seed=42)
    run_prompt(dev, [70], [8192], 4, 2, 128, seed=43, scale=1.0)         # scores far apart


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_split_values_that_are_not_finite(dev, D):
    g = gen(44, dev)
    nk = 9000
    q, k, v = rnd(g, 40, 4, D, dev=dev), rnd(g, nk, 2, D, dev=dev), rnd(g, nk, 2, D, dev=dev)
    cq, ck = (torch.tensor([0, n], dtype=torch.int32, device=dev) for n in (40, nk))
    want, lse = W.prompt_attention(q, k, v, cq, ck, return_lse=True)
    for bad in (float("nan"), float("inf")):
        k2, v2 = k.clone(), v.clone()
        v2[nk - 11, 1, D - 1] = bad                                      # rows from 29 on see it
        v2[100, 0, 2] = bad                                              # every row sees it
        got = W.prompt_attention(q, k, v2, cq, ck)
        assert torch.equal(got[:29, 2:], want[:29, 2:]) and torch.equal(got[:, 2:, :D - 1], want[:, 2:, :D - 1])
        late, all_ = got[29:, 2:, D - 1], got[:, :2, 2]
        assert (torch.isnan(late) if bad != bad else late == bad).all() and not torch.isfinite(all_).any()
        assert torch.equal(got[:, :2, 3:], want[:, :2, 3:])
        k2[nk - 21, 0, 5] = float("nan")
        got, l2 = W.prompt_attention(q, k2, v, cq, ck, return_lse=True)
        assert torch.equal(got[:19], want[:19]) and torch.equal(got[:, 2:], want[:, 2:]) and torch.equal(l2[:19], lse[:19])
        assert torch.isnan(got[19:, :2]).all() and torch.isnan(l2[19:, :2]).all()


def test_prompt_split_captured_streams_and_bounds(dev):
    """A captured call follows the device's bounds; two captured calls keep their own sums; rows outside stay."""
    g = gen(45, dev)
    q, k, v = rnd(g, 200, 8, 128, dev=dev), rnd(g, 12000, 2, 128, dev=dev), rnd(g, 12000, 2, 128, dev=dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)      # noqa: E731
    cq, ck, k2 = i32(0, 64, 200), i32(0, 12000, 12000), k.flip(0).contiguous()
    graphs, outs = [], []
    for kk in (k, k2):
        W.prompt_attention(q, kk, v, cq, ck)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(W.prompt_attention(q, kk, v, cq, ck))
        graphs.append(gr)
    for a, b in (((0, 64, 200), (0, 12000, 12000)), ((0, 1, 150), (0, 3, 11900)), ((10, 60, 200), (50, 6000, 12000))):
        cq.copy_(i32(*a))
        ck.copy_(i32(*b))
        want = []
        for kk in (k, k2):
            out = torch.full_like(q, 7.0)
            want.append(W.prompt_attention(q, kk, v, cq, ck, out=out))
            assert (out[:a[0]] == 7.0).all() and (out[a[2]:] == 7.0).all()
        s = torch.cuda.Stream(dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        for o in outs:
            o.fill_(7.0)
        graphs[0].replay()
        graphs[1].replay()
        with torch.cuda.stream(s):
            side = W.prompt_attention(q, k, v, cq, ck, out=torch.full_like(q, 7.0))
        torch.cuda.synchronize(dev)
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(side, want[0])
    # bounds that overlap or run backwards: every access stays inside, rows of one owner are right
    W.prompt_attention(q, k, v, i32(0, 200, 0, 200, 0, 200), i32(0, 12000, 0, 12000, 0, 12000))
    good = W.prompt_attention(q, k, v, i32(0, 200, 0, 0), i32(0, 12000, 0, 0))
    ref = A.attend(f64(q), f64(k), f64(v), 128 ** -0.5, True)
    check_out(good, ref, 128)


# ------------------------------------------------------------ append, evict --

@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_append_rows_are_the_formats_rows(dev, fmt, D):
    Hkv, page, new, old = 3, 16, [5, 0, 1, 33], [0, 40, 15, 30]
    total = [a + b for a, b in zip(new, old)]
    c = Cache(dev, total, Hkv, D, page, fmt, seed=31)
    g = gen(32, dev)
    T = sum(new)
    both = rnd(g, T + 2, 2 * Hkv, D, dev=dev)             # two rows behind the last sequence are no tokens
    both[0, 0, :64] = 0.0
    k, v = both[:, :Hkv], both[:, Hkv:]
    cu = torch.tensor(np.cumsum([0] + new), dtype=torch.int32, device=dev)
    seen = torch.tensor([n + 100 for n in total], dtype=torch.int32, device=dev)
    mass = torch.ones((4, Hkv, c.width * page), device=dev)
    pos = torch.full((4, Hkv, c.width * page), -5, dtype=torch.int32, device=dev)
    before = [None if t is None else t.clone() for t in (c.k, c.v, c.ks, c.vs)]
    W.paged_append(k, v, cu, c.k, c.v, c.table, c.lengths, fmt, c.ks, c.vs, mass, pos, seen)
    want = before
    at = 0
    for b, n in enumerate(new):
        e = torch.arange(total[b] - n, total[b], device=dev)
        pg, sl = c.table[b][e // page].long(), e % page
        for i, x in enumerate((k, v)):
            x = x[at:at + n].contiguous()
            if fmt == "bf16":
                want[i][pg, :, sl] = x
            elif n:
                p, s = W.kv_quantize(x, fmt)
                want[i][pg, :, sl], want[i + 2][pg, :, sl] = p, s
        assert (mass[b][:, e] == 0).all() and (pos[b][:, e] == (e + 100).int()).all()
        at += n
    assert int((mass == 0).sum()) == T * Hkv and int((pos != -5).sum()) == T * Hkv
    for got, w in zip((c.k, c.v, c.ks, c.vs), want):
        if w is not None:
            assert torch.equal(got.view(torch.uint8), w.view(torch.uint8))


@pytest.mark.parametrize("fmt", FMTS)
def test_append_a_long_prompt(dev, fmt):
    # several pieces per thread, the last ones partly past the end
    Hkv, D, page, n = 5, 128, 64, 4001
    c = Cache(dev, [n], Hkv, D, page, fmt, seed=35)
    k, v = (rnd(gen(36 + i, dev), n, Hkv, D, dev=dev) for i in range(2))
    W.paged_append(k, v, torch.tensor([0, n], dtype=torch.int32, device=dev), c.k, c.v, c.table, c.lengths, fmt, c.ks, c.vs)
    e = torch.arange(n, device=dev)
    pg, sl = c.table[0][e // page].long(), e % page
    for x, cache, scales in ((k, c.k, c.ks), (v, c.v, c.vs)):
        if fmt == "bf16":
            assert torch.equal(cache[pg, :, sl], x)
        else:
            p, s = W.kv_quantize(x, fmt)
            assert torch.equal(cache[pg, :, sl], p) and torch.equal(scales[pg, :, sl], s)


def test_append_skips_what_is_out_of_range(dev):
    c = Cache(dev, [20, 20, 20], 2, 64, 16, "bf16", seed=33)
    k = rnd(gen(34, dev), 3, 2, 64, dev=dev)
    c.lengths.copy_(torch.tensor([0, c.width * 16 + 1, 20], dtype=torch.int32))
    c.table[2, 1] = c.k.shape[0] + 5
    before = c.k.view(torch.int16).clone()
    W.paged_append(k, k, torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=dev), c.k, c.v, c.table, c.lengths)
    assert torch.equal(c.k.view(torch.int16), before)


def check_evict(dev, lens, Hkv, D, page, fmt, budget, recent, sinks, mass_fn, seed=0, in_place=False, max_pages=None):
    c = Cache(dev, lens, Hkv, D, page, fmt, seed, max_pages=max_pages)
    cap = c.width * page
    mass = mass_fn(torch.rand((len(lens), Hkv, cap), generator=gen(seed + 1, dev), device=dev))
    pos = torch.stack([torch.stack([torch.randperm(cap, generator=torch.Generator().manual_seed(seed + 7 * b + h))
                                    for h in range(Hkv)]) for b in range(len(lens))]).to(torch.int32).to(dev)
    seen = torch.tensor([max(1, n + 3) for n in lens], dtype=torch.int32, device=dev)
    want = [None if t is None else t.clone() for t in (c.k, c.v, c.ks, c.vs)]
    wm, wp = mass.clone(), pos.clone()
    mn, pn, tn = mass.cpu().numpy(), pos.cpu().numpy(), c.table.cpu()
    moved = 0
    for b, n in enumerate(lens):
        for h in range(Hkv):
            holes, tails = A.evict(mn[b, h], pn[b, h], n, n + 3, budget, recent, sinks)
            assert len(holes) == len(tails)
            if not holes:
                continue
            moved += len(holes)
            d, t = torch.tensor(holes), torch.tensor(tails)
            dp, tp = tn[b][d // page].long(), tn[b][t // page].long()
            for x in want:
                if x is not None:
                    x[dp.to(dev), h, (d % page).to(dev)] = x[tp.to(dev), h, (t % page).to(dev)]
            wm[b, h, d.to(dev)], wp[b, h, d.to(dev)] = mass[b, h, t.to(dev)], pos[b, h, t.to(dev)]
    if in_place:
        m2, p2, l2 = W.paged_evict(c.k, c.v, c.table, c.lengths, mass, pos, seen, budget, recent, sinks, fmt, c.ks, c.vs)
        assert m2 is mass and p2 is pos
        assert torch.equal(m2.view(torch.int32), wm.view(torch.int32)) and torch.equal(p2, wp)
    else:
        out = (torch.full_like(mass, -1.0), torch.full_like(pos, -1), torch.zeros_like(c.lengths))
        m2, p2, l2 = W.paged_evict(c.k, c.v, c.table, c.lengths, mass, pos, seen, budget, recent, sinks, fmt, c.ks, c.vs,
                                   out=out)
        for b, n in enumerate(lens):
            m = min(n, budget)
            assert torch.equal(m2[b, :, :m].view(torch.int32), wm[b, :, :m].view(torch.int32))
            assert torch.equal(p2[b, :, :m], wp[b, :, :m])
            assert (m2[b, :, m:] == -1.0).all() and (p2[b, :, m:] == -1).all()
    assert l2.tolist() == [min(n, budget) for n in lens]
    for got, w in zip((c.k, c.v, c.ks, c.vs), want):
        if w is not None:
            assert torch.equal(got.view(torch.uint8), w.view(torch.uint8))
    return moved


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_vs_oracle(dev, fmt, in_place):
    moved = check_evict(dev, [0, 1, 99, 100, 101, 517], 3, 64, 16, fmt, 100, 20, 4, lambda m: m, 41, in_place)
    assert moved > 0


@pytest.mark.parametrize("fmt,D", [("bf16", 256), ("fp8_f32_b64", 128), ("mxfp8", 256)])
def test_evict_row_widths(dev, fmt, D):
    check_evict(dev, [300, 70], 2, D, 48, fmt, 64, 0, 0, lambda m: m, 42)


@pytest.mark.parametrize("name,fn", [
    ("all equal", lambda m: torch.full_like(m, 0.25)), ("zeros of both signs", lambda m: torch.where(m < 0.5, 0.0, -0.0)),
    ("few values", lambda m: (m * 5).floor()), ("infinite", lambda m: torch.where(m < 0.3, torch.inf, m)),
    ("tiny", lambda m: m * 1e-42), ("one bit apart", lambda m: (m * 3).int().add(0x3f800000).view(torch.float32))])
def test_evict_ties_and_extremes(dev, name, fn):
    check_evict(dev, [700, 1500], 2, 64, 64, "bf16", 333, 10, 2, fn, 43)


@pytest.mark.parametrize("n,budget", [(9000, 1000), (20000, 19999), (33000, 4096)])
def test_evict_over_a_cluster(dev, n, budget):
    check_evict(dev, [n, n // 2], 2, 64, 64, "bf16", budget, 100, 4, lambda m: (m * 1000).floor(), 44, in_place=True)


def test_evict_budget_behind_the_capacity_and_bad_rows(dev):
    check_evict(dev, [90, 20], 2, 64, 16, "bf16", 10 ** 6, 5, 5, lambda m: m, 45)
    c = Cache(dev, [200, 200, 200], 1, 64, 16, "bf16", 46)
    cap = c.width * 16
    mass = torch.rand((3, 1, cap), device=dev)
    pos = torch.arange(cap, dtype=torch.int32, device=dev).expand(3, 1, cap).contiguous()
    c.lengths[0] = cap + 9
    c.table[1, 2] = -3
    k, m0 = c.k.view(torch.int16).clone(), mass.clone()
    _, _, ln = W.paged_evict(c.k, c.v, c.table, c.lengths, mass, pos, c.lengths.clone(), 50)
    assert ln.tolist() == [cap + 9, 200, 50] and torch.equal(mass[:2], m0[:2])
    same = (c.k.view(torch.int16) == k).all(-1).all(-1).all(-1)
    third = set(c.table[2].tolist())
    assert all(bool(same[p]) for p in range(c.k.shape[0]) if p not in third)


def test_evict_longer_than_shared_memory_holds(dev):
    # 8 CTAs x 40960 keys: longer slices are read again in every pass
    n, budget = 400000, 300000
    k, v = (torch.zeros((n // 64, 1, 64, 64), dtype=torch.bfloat16, device=dev) for _ in range(2))
    k[:] = torch.arange(n, device=dev).reshape(n // 64, 1, 64, 1).remainder(251)
    table = torch.arange(n // 64, dtype=torch.int32, device=dev)[None]
    mass = torch.rand((1, 1, n), generator=gen(47, dev), device=dev)
    pos = torch.arange(n, dtype=torch.int32, device=dev)[None, None].contiguous()
    ln = torch.tensor([n], dtype=torch.int32, device=dev)
    order = torch.sort(mass[0, 0], descending=True, stable=True)[1][:budget]
    kept = torch.sort(order)[0]
    W.paged_evict(k, v, table, ln, mass, pos, ln, budget)
    assert torch.equal(torch.sort(pos[0, 0, :budget])[0].long(), kept)
    assert torch.equal(k.reshape(n, 64)[:budget, 0].long(), pos[0, 0, :budget].long() % 251)


# ------------------------------------------------------------- all together --

@pytest.mark.parametrize("fmt,D", [("bf16", 128), ("fp8_f32_b64", 256), ("mxfp8", 64)])
def test_serving_run(dev, fmt, D):
    """Prompts, their cache, decode steps that collect weights, eviction, more steps, a sequence that
    ends and another in its place -- against the same run on 64-bit rows."""
    Hq, Hkv, B = 8, 2, 3
    g = gen(51, dev)
    cache = W.PagedKVCache(B, Hkv, D, n_pages=24, page_size=16, max_pages=12, fmt=fmt, track=True)

    def values(x):
        if fmt == "bf16":
            return f64(x)
        p, s = W.kv_quantize(x.contiguous(), fmt)
        blk = 64 if fmt == "fp8_f32_b64" else 32
        f = s.double() if blk == 64 else torch.exp2(s.double() - 127)
        return (p.view(torch.float8_e4m3fn).double().reshape(*x.shape[:-1], D // blk, blk) * f.unsqueeze(-1)).reshape(x.shape).cpu().numpy()

    # per sequence and head: list of (position, key, value, mass) as the cache orders them
    state = [[[] for _ in range(Hkv)] for _ in range(B)]
    seen = [0] * B

    def push(b, ks, vs):
        for i in range(ks.shape[0]):
            for h in range(Hkv):
                state[b][h].append([seen[b] + i, ks[i, h], vs[i, h], 0.0])
        seen[b] += ks.shape[0]

    def add(counts):
        T = sum(counts)
        x = rnd(g, T, Hq + 2 * Hkv, D, dev=dev)
        q, k, v = x.split([Hq, Hkv, Hkv], dim=1)
        cache.append(k, v, counts)
        kv, vv = values(k), values(v)
        at = 0
        for b, n in enumerate(counts):
            push(b, kv[at:at + n], vv[at:at + n])
            at += n
        return q, k, v

    def step():
        q, _, _ = add([1] * B)
        out, lse = cache.attend(q, return_lse=True)
        for b in range(B):
            for h in range(Hkv):
                e = state[b][h]
                G = Hq // Hkv
                ref = A.attend(f64(q[b:b + 1, h * G:(h + 1) * G]), np.stack([r[1] for r in e])[:, None],
                               np.stack([r[2] for r in e])[:, None], D ** -0.5)
                check_out(out[b:b + 1, h * G:(h + 1) * G], ref, D)
                check_lse(lse[b:b + 1, h * G:(h + 1) * G], ref, D)
                for r, w in zip(e, ref["weight"][0]):
                    r[3] += w
                got = cache.mass[b, h, :len(e)].double().cpu().numpy()
                assert np.allclose(got, [r[3] for r in e], rtol=1e-3, atol=1e-9)
                assert cache.positions[b, h, :len(e)].tolist() == [r[0] for r in e]

    counts = [100, 37, 3]
    q, k, v = add(counts)
    cu = torch.tensor(np.cumsum([0] + counts), dtype=torch.int32, device=dev)
    out = W.prompt_attention(q, k, v, cu)
    at = 0
    for n in counts:
        sl = slice(at, at + n)
        check_out(out[sl], A.attend(f64(q[sl]), f64(k[sl]), f64(v[sl]), D ** -0.5, True), D)
        at += n
    for _ in range(3):
        step()
    free = cache.free_pages
    masses = cache.mass.clone()
    cache.evict(48, recent=8, sinks=2)
    assert cache.offsets == [48, 40, 6] and cache.lengths.tolist() == [48, 40, 6] and cache.free_pages == free + 4
    for h in range(Hkv):
        e = state[0][h]
        holes, tails = A.evict(masses[0, h].tolist(), [r[0] for r in e], len(e), seen[0], 48, 8, 2)
        for d, t in zip(holes, tails):
            e[d] = e[t]
        del e[48:]
    for _ in range(2):
        step()
    cache.clear(1)
    state[1], seen[1] = [[] for _ in range(Hkv)], 0
    add([0, 20, 0])
    step()
