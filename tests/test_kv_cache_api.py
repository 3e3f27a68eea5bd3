"""Host-side checks of the block-scaled KV cache (CPU only): refused arguments of the
Python entry points and of the C ABI, and the 64-bit restatements themselves."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import _kv_reference as ref
from switchattentionkernels_b200 import (SwitchKVCache, _native, make_switch_kv_cache, switch_gqa_decode_cached,
                                         switch_kv_cache_append, switch_kv_cache_evict)
from test_host_api import dev

E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def _cache(B=2, S=50, H=2, dtype=E4M3, block=16, weights=True):
    c = make_switch_kv_cache(B, S, H, device="cpu", dtype=dtype, block_size=block, track_weights=weights)
    return SwitchKVCache(*(None if t is None else dev(t) for t in (c.k, c.v, c.k_scale, c.v_scale, c.seq_lens, c.key_weights)),
                         c.block_size)


def _rows(*shape):
    return dev(torch.zeros(*shape, dtype=torch.bfloat16))


def test_make_cache():
    c = make_switch_kv_cache(2, 33, 3, device="cpu", dtype=INT8, block_size=32, track_weights=True)
    assert c.k.shape == c.v.shape == (2, 3, 33, 128) and c.k.dtype == INT8
    assert c.k_scale.shape == c.v_scale.shape == (2, 3, 2) and c.key_weights.shape == (2, 3, 33)
    assert not c.seq_lens.any() and c.seq_lens.dtype == torch.int32
    assert make_switch_kv_cache(1, 1, 1, device="cpu").key_weights is None
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, -1)):
        with pytest.raises(ValueError, match="positive"):
            make_switch_kv_cache(*bad, device="cpu")
    with pytest.raises(TypeError, match="dtype"):
        make_switch_kv_cache(1, 1, 1, device="cpu", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="block_size"):
        make_switch_kv_cache(1, 1, 1, device="cpu", block_size=48)


@pytest.mark.parametrize("field,value,error", [
    ("k", torch.zeros(2, 2, 50, 128), TypeError), ("v", torch.zeros(2, 2, 50, 128, dtype=torch.int8), TypeError),
    ("k_scale", torch.zeros(2, 2, 3), ValueError), ("v_scale", torch.zeros(2, 2, 4, dtype=torch.float64), ValueError),
    ("seq_lens", torch.zeros(2, dtype=torch.int64), ValueError), ("seq_lens", torch.zeros(3, dtype=torch.int32), ValueError),
    ("key_weights", torch.zeros(2, 2, 49), ValueError), ("k_scale", torch.zeros(2, 4, 2).transpose(1, 2), ValueError),
    ("k_scale", None, ValueError), ("k", None, TypeError),
])
def test_malformed_caches_are_refused(field, value, error):
    c = _cache()
    setattr(c, field, None if value is None else dev(value))
    q, route = _rows(2, 4, 128), dev(torch.zeros(2, dtype=torch.bool))
    for call in (lambda: switch_kv_cache_append(c, _rows(2, 2, 128), _rows(2, 2, 128)),
                 lambda: switch_gqa_decode_cached(q, c, route), lambda: switch_kv_cache_evict(c, keep=3)):
        with pytest.raises(error):
            call()
    with pytest.raises(TypeError):
        switch_kv_cache_evict({"k": 1}, keep=3)
    c = _cache()
    c.block_size = 17
    with pytest.raises(ValueError, match="block_size"):
        switch_kv_cache_evict(c, keep=3)


def test_append_refusals():
    c = _cache()
    ok = _rows(2, 5, 2, 128)
    for k, v, error in ((dev(torch.zeros(2, 5, 2, 128)), ok, TypeError), (ok, _rows(2, 4, 2, 128), ValueError),
                        (_rows(2, 5, 1, 128), ok, ValueError), (_rows(1, 5, 2, 128), ok, ValueError),
                        (_rows(2, 5, 2, 64), ok, ValueError), (_rows(2, 128), ok, ValueError), (None, ok, ValueError),
                        (ok, _rows(2, 2, 128), ValueError), (ok, _rows(2, 5, 128, 2).transpose(2, 3), ValueError),
                        (dev(torch.zeros(2, 5, 2, 129, dtype=torch.bfloat16)[..., :128]), ok, ValueError),
                        (dev(torch.zeros(2 * 5 * 2 * 128 + 1, dtype=torch.bfloat16)[1:].view(2, 5, 2, 128)), ok, ValueError)):
        with pytest.raises(error):
            switch_kv_cache_append(c, k, v)
    for name in ("new_lens", "start"):
        for bad in (torch.zeros(2), torch.zeros(3, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32), [1, 2]):
            with pytest.raises(ValueError, match=name):
                switch_kv_cache_append(c, ok, ok, **{name: dev(bad) if isinstance(bad, torch.Tensor) else bad})
    # the stride of a single entry does not matter, only its address
    from switchattentionkernels_b200 import kv_cache
    one = dev(torch.zeros(4096, dtype=torch.bfloat16).as_strided((1, 3, 1, 128), (37, 256, 5, 1)))
    assert kv_cache._check_rows(one, "x", (1, 3, 1, 128), one.device) == (0, 256, 0, 1)
    with pytest.raises(ValueError, match="multiples of 8"):
        kv_cache._check_rows(dev(torch.zeros(4096, dtype=torch.bfloat16).as_strided((1, 3, 2, 128), (37, 256, 5, 1))), "x",
                             (1, 3, 2, 128), one.device)
    empty = _rows(2, 0, 2, 128)
    switch_kv_cache_append(c, empty, empty)  # nothing to do: no launch


def test_decode_refusals():
    c = _cache()
    q, route = _rows(2, 4, 128), dev(torch.zeros(2, dtype=torch.bool))
    with pytest.raises(TypeError):
        switch_gqa_decode_cached(dev(torch.zeros(2, 4, 128)), c, route)
    for bad in (_rows(3, 4, 128), _rows(2, 3, 128), _rows(2, 4, 64), _rows(2, 2, 4, 128), _rows(2, 128), _rows(2, 0, 128)):
        with pytest.raises(ValueError):
            switch_gqa_decode_cached(bad, c, route)
    for bad in (torch.zeros(2, dtype=torch.uint8), torch.zeros(3, dtype=torch.bool)):
        with pytest.raises(ValueError, match="route_full"):
            switch_gqa_decode_cached(q, c, dev(bad))
    with pytest.raises(ValueError, match="window_size"):
        switch_gqa_decode_cached(q, c, route, window_size=0)
    with pytest.raises(ValueError, match="sm_scale"):
        switch_gqa_decode_cached(q, c, route, sm_scale=-1.0)
    with pytest.raises(ValueError, match="status_out"):
        switch_gqa_decode_cached(q, c, route, status_out=dev(torch.zeros(1)))


def test_evict_refusals():
    c = _cache()
    for kw in (dict(keep=0), dict(keep=-1), dict(keep=5, sink=-1), dict(keep=5, recent=-1), dict(keep=5, sink=3, recent=3)):
        with pytest.raises(ValueError, match="keep"):
            switch_kv_cache_evict(c, **kw)
    with pytest.raises(ValueError, match="key_weights"):
        switch_kv_cache_evict(_cache(weights=False), keep=5)
    with pytest.raises(ValueError, match="key_weights"):
        switch_kv_cache_evict(c, keep=5, out=_cache(weights=False))
    for out in (_cache(B=3), _cache(H=3), _cache(dtype=INT8), _cache(block=32)):
        with pytest.raises(ValueError, match="batch, heads"):
            switch_kv_cache_evict(c, keep=5, out=out)
    with pytest.raises(ValueError, match="fewer rows"):
        switch_kv_cache_evict(c, keep=20, out=_cache(S=19))
    shared = _cache()
    shared.v = c.v
    with pytest.raises(ValueError, match="share memory"):
        switch_kv_cache_evict(c, keep=5, out=shared)


def test_c_abi_refusals():
    # refused before any device call: the library needs no GPU for these
    lib = _native.load()
    one, two, three, four = (ctypes.c_void_p(x) for x in (256, 512, 768, 1024))
    none = None

    def append(k=one, v=one, ks=128, B=1, T=1, H=1, S=16, D=128, block=16, dtype=1, start=one, new=none, vc=two, vs=four, lens=one):
        return lib.swa_kv_append(k, v, 256, 256, ks, 256, 256, 128, start, new, one, vc, three, vs, none, lens, B, T, H, S, D, block, dtype, none)

    def decode(q=one, sb=128, B=1, S=16, Hq=2, H=1, D=128, block=16, window=4, scale=1.0, dtype=1, ws=one, nbytes=0):
        return lib.swa_kv_decode(q, sb, 128, one, one, one, one, one, one, one, one, none, B, S, Hq, H, D, block, window, scale,
                                 dtype, ws, nbytes, none)

    def evict(k=one, ko=one, vo=two, vs=four, B=1, H=1, S=16, So=16, D=128, block=16, keep=4, sink=0, recent=0, dtype=1):
        return lib.swa_kv_evict(k, two, three, four, one, one, ko, vo, three, vs, one, one, one, B, H, S, So, D, block, keep, sink,
                                recent, dtype, none)

    invalid, unsupported = -1, -3
    for rc in (append(k=none), append(start=none), append(lens=none), append(k=ctypes.c_void_p(8)), append(ks=4), append(ks=-4),
               append(B=0), append(T=0), append(H=-1), append(S=0), append(block=48), append(dtype=0), decode(q=none),
               decode(q=ctypes.c_void_p(4)), decode(sb=4), decode(B=0), decode(Hq=3, H=2), decode(Hq=0), decode(window=0),
               decode(scale=0.0), decode(scale=math.nan), decode(block=8), decode(dtype=3), decode(ws=none), evict(k=none),
               evict(keep=0), evict(sink=-1), evict(keep=4, sink=3, recent=2), evict(S=0), evict(dtype=9),
               evict(ko=ctypes.c_void_p(2048)), evict(So=3), evict(So=17), append(vc=one), append(vs=three), evict(vo=one),
               evict(vs=three), append(B=4, start=ctypes.c_void_p(260)), append(B=4, new=ctypes.c_void_p(252))):
        assert rc == invalid
    for rc in (append(D=64), decode(D=256), evict(D=1), append(B=70000, T=2), append(H=40000, T=2), append(S=(1 << 30) + 1)):
        assert rc == unsupported
    for bad in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 3, 2), (1, 1, 0, 1)):
        assert lib.swa_kv_decode_workspace_bytes(*bad, 0) == 0


def test_reference_rounding_is_nearest_even():
    # every e4m3 value is kept, halfway points go to the even neighbour, the rest to the nearer one
    grid = torch.arange(0, 0x7F, dtype=torch.uint8).view(E4M3).double()
    assert torch.equal(ref.values(ref.round8(grid, E4M3)), grid)
    mid = (grid[1:] + grid[:-1]) / 2
    even = torch.where(torch.arange(0, 0x7E) % 2 == 0, grid[:-1], grid[1:])
    assert torch.equal(ref.values(ref.round8(mid, E4M3)), even)
    assert torch.equal(ref.values(ref.round8(-mid * (1 + 2.0 ** -40), E4M3)), -grid[1:])
    assert torch.equal(ref.values(ref.round8(torch.tensor([1e9, -math.inf], dtype=torch.float64), E4M3)),
                       torch.tensor([448.0, -448.0], dtype=torch.float64))
    assert ref.round8(torch.tensor([0.5, 1.5, -2.5, 200.0, math.nan, -math.inf], dtype=torch.float64), INT8).tolist() == [0, 2, -2, 127, 0, -127]


def test_reference_append_and_decode():
    # dequantised rows are within half a step of what was appended, and the decode of an int8 cache of
    # small integers is the plain softmax over them
    g = torch.Generator().manual_seed(1)
    for dtype, step in ((E4M3, 2.0 ** -4), (INT8, None)):
        c = ref.clone(make_switch_kv_cache(1, 40, 1, device="cpu", dtype=dtype, block_size=16, track_weights=True))
        x = torch.randn(1, 40, 1, 128, generator=g).bfloat16()
        ref.append(c, x[:, :30], x[:, :30])
        ref.append(c, x[:, 30:], x[:, 30:])
        s = ref.values(c["k_scale"])[0, 0].repeat_interleave(16)[:40, None]
        err = (ref.values(c["k"])[0, 0] * s - ref.values(x)[0, :, 0]).abs()
        # a row of the second block may have been rounded twice (its scale grew): twice half a step
        assert bool((err <= (2 * ref.values(x)[0, :, 0].abs() * 2.0 ** -4 + s * 2.0 ** -9 if dtype == E4M3 else s)).all())
    c["k"].copy_(torch.randint(-3, 4, c["k"].shape, generator=g))
    c["k_scale"].fill_(1.0)
    q = torch.randn(1, 2, 128, generator=g).bfloat16()
    O, L, w, _ = ref.decode(c, q, torch.tensor([False]), 7)
    s = q[0].double() @ c["k"][0, 0, 33:].double().T / math.sqrt(128)
    assert torch.allclose(L[0] / ref.LOG2E, torch.logsumexp(s, 1)) and torch.allclose(w[0, 0, 33:], torch.softmax(s, 1).sum(0))
    assert not w[0, 0, :33].any()


def test_reference_evict():
    c = ref.clone(make_switch_kv_cache(1, 10, 1, device="cpu", block_size=16, track_weights=True))
    c["seq_lens"][0] = 10
    c["key_weights"][0, 0] = torch.tensor([0, 5, 1, math.nan, 5, 2, 2, 9, 0, 0])
    assert ref.evict(c, 6, 1, 2)[1].tolist() == [[[0, 1, 4, 7, 8, 9]]]
    assert ref.evict(c, 7, 1, 2)[1].tolist() == [[[0, 1, 4, 5, 7, 8, 9]]]
    assert ref.evict(c, 10, 1, 2)[1].tolist() == [[list(range(10))]]
