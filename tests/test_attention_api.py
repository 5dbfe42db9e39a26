"""Argument checks of the attention and paged-cache calls, and the paged cache's
host side, without a GPU: every refusal comes before any CUDA call."""
import ctypes
import os
import subprocess

import pytest
import torch

import whallm_b200 as W
from whallm_b200 import _lib as L
from whallm_b200 import build

P = ctypes.c_void_p(1 << 20)          # an aligned address that no refused call touches
ODD = ctypes.c_void_p((1 << 20) + 2)


def expect(name, args, msg, code=L.WM_ERR_INVALID):
    rc = getattr(L.lib(), name)(*args)
    assert rc == code, (name, rc, L.last_error())
    if msg:
        assert msg in L.last_error(), L.last_error()


def append_args(**c):
    d = dict(k=P, v=P, ks=512, vs=512, cu=P, T=4, B=2, Hkv=4, D=128, kc=P, vc=P, ksc=None, vsc=None, fmt=L.WKV_BF16, n=8, page=16,
             table=P, width=4, lengths=P, mass=None, pos=None, seen=None, stream=None)
    return tuple({**d, **c}.values())


def evict_args(**c):
    d = dict(B=2, Hkv=4, D=128, kc=P, vc=P, ksc=None, vsc=None, fmt=L.WKV_BF16, n=8, page=16, table=P, width=4, lengths=P, seen=P,
             mass=P, pos=P, budget=32, recent=4, sinks=4, mo=P, po=P, lo=ctypes.c_void_p(1 << 21), ws=P, bytes=1 << 20, stream=None)
    return tuple({**d, **c}.values())


def decode_args(**c):
    d = dict(q=P, qs=1024, B=2, Hq=8, Hkv=4, D=128, kc=P, vc=P, ksc=None, vsc=None, fmt=L.WKV_BF16, n=8, page=16, table=P, width=4,
             lengths=P, scale=0.1, out=P, lse=None, mass=None, ws=P, bytes=1 << 30, stream=None)
    return tuple({**d, **c}.values())


def prompt_args(**c):
    d = dict(q=P, k=P, v=P, qs=1024, ks=512, vs=512, cq=P, ck=P, B=2, Tq=8, Tk=8, Hq=8, Hkv=4, D=128, scale=0.1, causal=1, out=P,
             lse=None, ws=None, ws_bytes=0, stream=None)
    return tuple({**d, **c}.values())


@pytest.mark.parametrize("name,make", [("wkv_paged_append", append_args), ("wkv_paged_evict", evict_args),
                                       ("wattn_decode", decode_args)])
def test_pool_refusals(name, make):
    expect(name, make(fmt=L.WKV_FP8_UE8M0_B32), "paged cache rows are")
    expect(name, make(fmt=L.WKV_MXFP4_B32), "paged cache rows are")
    expect(name, make(D=96), "head dimension 64, 128 or 256")
    expect(name, make(page=24), "multiple of 16")
    expect(name, make(page=0), "multiple of 16")
    expect(name, make(B=-1), "negative or empty shape")
    expect(name, make(Hkv=0), "negative or empty shape")
    expect(name, make(page=1 << 20, width=1 << 12), "at most 2^31 - 1 entries")
    expect(name, make(kc=None), "missing cache or page table")
    expect(name, make(table=None), "missing cache or page table")
    expect(name, make(ksc=P), "bf16 rows take none")
    expect(name, make(fmt=L.WKV_MXFP8_B32, ksc=P), "quantized rows need scales")
    expect(name, make(vc=ODD), "16-byte aligned")


def test_append_refusals():
    f = "wkv_paged_append"
    expect(f, append_args(T=-1), "negative token count")
    expect(f, append_args(k=None), "missing input")
    expect(f, append_args(ks=511), "16-byte aligned and hold")
    expect(f, append_args(vs=504), "16-byte aligned and hold")
    expect(f, append_args(v=ODD), "16-byte aligned and hold")
    expect(f, append_args(pos=P), "token counts")
    expect(f, append_args(Hkv=5000, ks=5000 * 128, vs=5000 * 128), "at most 4096 heads")
    expect(f, append_args(Hkv=4096, ks=4096 * 128, vs=4096 * 128, T=1 << 20), "too many values")
    expect(f, append_args(T=0), None, L.WM_OK)
    expect(f, append_args(B=0), None, L.WM_OK)


def test_evict_refusals():
    f = "wkv_paged_evict"
    expect(f, evict_args(budget=0), "budget")
    expect(f, evict_args(budget=8, recent=6, sinks=3), "budget")
    expect(f, evict_args(recent=-1), "budget")
    expect(f, evict_args(mass=None), "missing array")
    expect(f, evict_args(lo=P), "array of their own")
    expect(f, evict_args(mo=ctypes.c_void_p(1 << 21)), "both in place")
    expect(f, evict_args(bytes=8), "workspace too small", L.WM_ERR_WORKSPACE)
    expect(f, evict_args(B=0), None, L.WM_OK)
    assert L.lib().wkv_evict_workspace_size(2, 4, 32) == 2 * 4 * (2 * 32 * 12 + 4)
    assert L.lib().wkv_evict_workspace_size(0, 4, 32) == 0


def test_decode_refusals():
    f = "wattn_decode"
    expect(f, decode_args(Hq=6), "multiple of the key-value heads")
    expect(f, decode_args(Hq=0), "multiple of the key-value heads")
    for s in (0.0, -1.0, float("nan"), float("inf")):
        expect(f, decode_args(scale=s), "positive and finite")
    expect(f, decode_args(q=None), "missing input or output")
    expect(f, decode_args(qs=1000), "4-byte aligned")
    expect(f, decode_args(width=1024, bytes=16), "workspace too small", L.WM_ERR_WORKSPACE)
    expect(f, decode_args(width=1024, ws=ODD), "256-byte aligned")
    expect(f, decode_args(mass=P, bytes=16), "workspace too small", L.WM_ERR_WORKSPACE)
    expect(f, decode_args(mass=P, page=1 << 20, width=100, bytes=1 << 60), "batch or capacity too large")
    expect(f, decode_args(out=ctypes.c_void_p((1 << 20) + 4)), "8-byte aligned")
    expect(f, decode_args(B=0), None, L.WM_OK)
    size = L.lib().wattn_decode_workspace_size
    assert size(2, 6, 4, 128, L.WKV_BF16, 16, 4, 0) == 0 and size(2, 8, 4, 100, L.WKV_BF16, 16, 4, 0) == 0
# one cluster per pair joins short caches without a workspace; collecting weights needs the scores
    assert size(2, 8, 4, 128, L.WKV_BF16, 16, 4, 0) == 0 and size(2, 8, 4, 128, L.WKV_BF16, 16, 4, 1) > 2 * 4 * 64 * 2 * 4
    assert size(2, 8, 4, 128, L.WKV_BF16, 16, 1024, 1) - size(2, 8, 4, 128, L.WKV_BF16, 16, 1024, 0) == 2 * 4 * 16384 * 2 * 4


def test_prompt_refusals():
    f = "wattn_prompt"
    expect(f, prompt_args(Hq=6), "multiple of the key-value heads")
    expect(f, prompt_args(Tq=-1), "multiple of the key-value heads")
    expect(f, prompt_args(D=80), "head dimension")
    expect(f, prompt_args(scale=0.0), "positive and finite")
    expect(f, prompt_args(out=None), "missing input or output")
    expect(f, prompt_args(ck=None), "missing input or output")
    expect(f, prompt_args(ks=500), "16-byte aligned and hold")
    expect(f, prompt_args(qs=1028), "16-byte aligned and hold")
    expect(f, prompt_args(k=ODD), "16-byte aligned and hold")
    expect(f, prompt_args(out=ctypes.c_void_p((1 << 20) + 16)), "32-byte aligned")
    expect(f, prompt_args(Tq=1 << 30, Hq=16, qs=2048), "too many rows")
    expect(f, prompt_args(Tq=0), None, L.WM_OK)
    # few rows on many keys are split over the GPU, which takes a workspace: at most one slot of 256 rows per SM
    size = L.lib().wattn_prompt_workspace_size
    some = size(2, 8, 8192, 8, 4, 128)
    assert some > 0 and some % (256 * 130 * 4) == 0 and size(2, 8, 8192, 8, 4, 256) % (128 * 258 * 4) == 0
    assert size(2, 8, 100, 8, 4, 128) == 0 and size(2, 32768, 32768, 8, 4, 128) == 0 and size(0, 8, 8192, 8, 4, 128) == 0
    assert size(2, 8, 8192, 6, 4, 128) == 0 and size(2, 8, 8192, 8, 4, 96) == 0
    expect(f, prompt_args(Tk=8192, ws=P, ws_bytes=some - 1), "workspace too small", L.WM_ERR_WORKSPACE)
    expect(f, prompt_args(Tk=8192, ws_bytes=some), "256-byte aligned")
    expect(f, prompt_args(Tk=8192, ws=ctypes.c_void_p((1 << 20) + 64), ws_bytes=some), "256-byte aligned")


def test_python_refusals():
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)    # noqa: E731
    pool = (bf(4, 2, 16, 64), bf(4, 2, 16, 64), i32(3, 2), i32(3))
    with pytest.raises(ValueError, match="format"):
        W.decode_attention(bf(3, 4, 64), *pool, fmt="fp8_ue8m0")
    with pytest.raises(ValueError, match="CUDA tensors"):
        W.decode_attention(bf(3, 4, 64), *pool)
    with pytest.raises(ValueError, match="scales"):
        W.decode_attention(bf(3, 4, 64), pool[0].to(torch.uint8), pool[1].to(torch.uint8), *pool[2:], fmt="mxfp8")
    with pytest.raises(ValueError, match="of one shape"):
        W.decode_attention(bf(3, 4, 64), pool[0].float(), *pool[1:])
    with pytest.raises(ValueError, match="page_table"):
        W.decode_attention(bf(3, 4, 64), pool[0], pool[1], pool[2].long(), pool[3])
    with pytest.raises(ValueError, match="take no scales"):
        W.paged_evict(pool[0], pool[1], pool[2], pool[3], None, None, pool[3], 4, k_scales=bf(1))
    with pytest.raises(ValueError, match=r"bf16 \[tokens, heads, D\]"):
        W.prompt_attention(bf(3, 4, 64).float(), bf(3, 2, 64), bf(3, 2, 64), i32(2))
    with pytest.raises(ValueError, match="CUDA tensors"):
        W.prompt_attention(bf(3, 4, 64), bf(3, 2, 64), bf(3, 2, 64), i32(2))


def test_paged_cache_hands_out_pages():
    c = W.PagedKVCache(3, 2, 64, n_pages=10, page_size=16, max_pages=5, device="cpu")
    assert c.mass is None and c.page_table.tolist() == [[-1] * 5] * 3
    c.reserve([17, 0, 1])
    assert c.free_pages == 7 and (c.page_table[0, :2] >= 0).all() and (c.page_table[0, 2:] == -1).all()
    assert (c.page_table[1] == -1).all()
    used = [p for p in c.page_table.flatten().tolist() if p >= 0]
    assert len(set(used)) == 3 and all(0 <= p < 10 for p in used)
    before = c.page_table.clone()
    c.reserve([32, 0, 16])                       # already there
    assert torch.equal(c.page_table, before) and c.free_pages == 7
    with pytest.raises(ValueError, match="page table"):
        c.reserve([81, 0, 0])
    with pytest.raises(ValueError, match="out of pages"):
        c.reserve([80, 80, 80])
    with pytest.raises(ValueError, match="counts"):
        c.reserve([1, 1])
    with pytest.raises(ValueError, match="counts"):
        c.reserve([1, -1, 0])
    assert torch.equal(c.page_table, before) and c.free_pages == 7   # a refused call changes nothing
    c.clear(0)
    assert c.free_pages == 9 and (c.page_table[0] == -1).all()
    c.reserve([80, 64, 0])
    assert c.free_pages == 0


def test_paged_cache_refusals():
    for bad in (dict(dimension=96), dict(page_size=24), dict(fmt="mxfp4"), dict(batch=0), dict(n_pages=0), dict(max_pages=0)):
        with pytest.raises(ValueError):
            W.PagedKVCache(**{**dict(batch=1, heads=2, dimension=64, n_pages=2, device="cpu"), **bad})
    c = W.PagedKVCache(2, 2, 64, n_pages=2, device="cpu", fmt="fp8_f32_b64")
    assert c.key_scales.shape == (2, 2, 64, 1) and c.keys.dtype == torch.uint8
    with pytest.raises(ValueError, match="track"):
        c.evict(8)
    x = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="sum of counts"):
        c.append(x, x, [1, 2])
    with pytest.raises(ValueError, match="CUDA tensors"):
        c.append(x, x)
    assert c.offsets == [0, 0]                   # the refused call added no entry
    assert c.lengths.tolist() == [0, 0] and c.seen.tolist() == [0, 0]


def test_evict_refuses_what_32_bits_cannot_count():
    """The eviction kernel's indexes run past the last entry by up to a round of loads or a page, in 32 bits."""
    f, big = "wkv_paged_evict", dict(bytes=1 << 60)
    expect(f, evict_args(page=16, width=(1 << 27) - 1, **big), "below 2^31")        # 2^31 - 16 entries
    expect(f, evict_args(page=16, width=(1 << 27) - 512, **big), "below 2^31")
    expect(f, evict_args(page=(1 << 30) + 16, width=1, **big), "below 2^31")        # length + page - 1 behind 2^31
    expect(f, evict_args(page=16, width=(1 << 27) - 514, mass=None, **big), "missing array")     # the most that is taken
    expect(f, evict_args(page=1 << 29, width=2, mass=None, **big), "missing array")


def test_a_wait_that_ran_out_leaves_nan(tmp_path):
    """What the prompt kernel does when a bounded wait runs out, compiled for the host: every element of the output, the
    log-sum-exp and the parts' sums is NaN, none beyond them is touched, and absent arrays are left alone."""
    src = tmp_path / "giveup.cu"
    src.write_text('#include "wm_giveup.cuh"\n'
                   'extern "C" void poison(void *o, long n, void *l, long nl, void *p, long np, int first, int step) {\n'
                   '  wm_giveup::poison((uint16_t *)o, n, (float *)l, nl, (float2 *)p, np, first, step);\n}\n')
    lib = tmp_path / "giveup.so"
    subprocess.run([build.NVCC, "-I", build.CSRC, "-Xcompiler", "-fPIC", "-shared", "-o", str(lib), str(src)], check=True)
    poison = ctypes.CDLL(str(lib)).poison
    out, lse, parts = torch.zeros(103, dtype=torch.bfloat16), torch.zeros(17), torch.zeros((9, 2))
    at = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    n = ctypes.c_long
    for t in range(4):
        poison(at(out), n(100), None, n(16), None, n(8), t, 4)
    assert torch.isnan(out[:100]).all() and (out[100:] == 0).all() and (lse == 0).all() and (parts == 0).all()
    for t in range(4):
        poison(at(out), n(0), at(lse), n(16), at(parts), n(8), t, 4)
    assert torch.isnan(lse[:16]).all() and lse[16] == 0
    assert torch.isnan(parts[:8, 1]).all() and (parts[:8, 0] == 0).all() and (parts[8] == 0).all()
    # and the prompt kernel hands it all three
    text = open(os.path.join(build.CSRC, "attn_prompt.cu")).read()
    assert "poison(a.out, heads * D, a.lse, heads, SP ? a.part_ml : nullptr" in text


def test_paged_cache_follows_steps_on_the_device():
    """Steps that advance ``lengths`` on the device, as a captured one does: after ``refresh`` the host hands out pages
    from the new counts, and refuses counts that its pages do not hold."""
    c = W.PagedKVCache(2, 2, 64, n_pages=8, page_size=16, max_pages=5, device="cpu")
    c.reserve([16, 3])
    c.lengths += torch.tensor([16, 3], dtype=torch.int32)
    c.refresh()
    assert c.offsets == [16, 3] and c.free_pages == 6
    c.reserve([16, 16])
    assert c.free_pages == 4 and (c.page_table[:, :2] >= 0).all()
    c.lengths.fill_(0)                               # shortened on the device: its pages stay handed out
    c.refresh()
    c.reserve([32, 32])
    assert c.offsets == [0, 0] and c.free_pages == 4
    for bad in ([33, 0], [0, -1]):
        c.lengths.copy_(torch.tensor(bad, dtype=torch.int32))
        with pytest.raises(ValueError, match="reserve before"):
            c.refresh()
        assert c.offsets == [0, 0]
    c.clear(0)
    assert c.free_pages == 6 and c.offsets == [0, 0]


def test_workspaces_are_planned_on_the_tensors_device(monkeypatch):
    """Two devices of different sizes, stood in for on the host: each call's workspace is the one that its own device
    asks for, whichever is current and whichever came first."""
    from whallm_b200 import attention as A

    class Tensor:
        def __init__(self, dev, dtype, *shape):
            self.dev, self.dtype, self.shape, self.is_cuda = dev, dtype, torch.Size(shape), True

        def stride(self):
            return torch.empty(self.shape, device="meta").stride()

        def new_empty(self, shape, dtype=None):
            return Tensor(self.dev, dtype or self.dtype, *shape)

        get_device, is_contiguous, data_ptr = lambda s: s.dev, lambda s: True, lambda s: 1 << 20
        numel = lambda s: s.shape.numel()  # noqa: E731

    current, calls = [0], []

    class Device:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            self.before, current[0] = current[0], self.dev

        def __exit__(self, *_):
            current[0] = self.before

    class Lib:
        def __getattr__(self, name):
            if name.endswith("_size"):
                return lambda *shape: 1000 * (current[0] + 1)
            return lambda *args: calls.append((name, current[0], args[-2])) or 0

    monkeypatch.setattr(L, "_lib", Lib())
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(A, "_raw_stream", lambda dev: dev)
    bf, i32 = torch.bfloat16, torch.int32
    for dev in (1, 0, 2, 1):
        t = lambda dtype, *shape: Tensor(dev, dtype, *shape)  # noqa: E731, B023
        W.decode_attention(t(bf, 7, 8, 64), t(bf, 4, 2, 16, 64), t(bf, 4, 2, 16, 64), t(i32, 7, 300), t(i32, 7))
        W.prompt_attention(t(bf, 7, 8, 64), t(bf, 9001, 2, 64), t(bf, 9001, 2, 64), t(i32, 2), t(i32, 2))
        assert calls[-2:] == [("wattn_decode", dev, 1000 * (dev + 1)), ("wattn_prompt", dev, 1000 * (dev + 1))]
