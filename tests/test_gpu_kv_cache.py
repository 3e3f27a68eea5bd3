"""Block-scaled 8-bit KV cache on the GPU (append, decode attention, eviction) against
plain restatements in 64 bits.  Appended and evicted bytes, scales and rows are equal;
the decode step is held to the error that its number formats allow."""
from __future__ import annotations

import math

import pytest
import torch

import _kv_reference as ref
from switchattentionkernels_b200 import (SwitchKVCache, make_switch_kv_cache, switch_gqa_decode_cached,
                                         switch_kv_cache_append, switch_kv_cache_evict)

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BOTH = pytest.mark.parametrize("dtype", [E4M3, INT8], ids=["e4m3", "int8"])


def _rows(g, *shape, spread=1.0):
    """BF16 rows whose channels and tokens differ in size."""
    x = torch.randn(*shape, generator=g)
    x = x * torch.exp(spread * torch.randn(shape[-1], generator=g)) * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=g))
    return x.bfloat16()


def _filled(g, dev, B, Smax, Hkv, lens, *, dtype, block, weights=True):
    """A cache that holds rows of several sizes; rows past the lengths hold NaN bytes (e4m3) or the
    largest value (int8), under the largest scales."""
    c = make_switch_kv_cache(B, Smax, Hkv, device=dev, dtype=dtype, block_size=block, track_weights=weights)
    c.k.view(torch.uint8).fill_(0x7F)
    c.v.view(torch.uint8).fill_(0x7F)
    c.k_scale.fill_(3.0e38)
    c.v_scale.fill_(3.0e38)
    lens = torch.as_tensor(lens, dtype=torch.int32)
    T = max(1, int(lens.max()))
    k, v = _rows(g, B, T, Hkv, 128), _rows(g, B, T, Hkv, 128)
    switch_kv_cache_append(c, k.to(dev), v.to(dev), new_lens=lens.to(dev))
    if weights:
        c.key_weights.copy_(torch.rand(B, Hkv, Smax, generator=g) ** 4)
    return c


def _equal(got: SwitchKVCache, want: dict, rows=None):
    """Bytes, scales, lengths and weights of the rows below the lengths (all rows without ``rows``)."""
    B, Hkv = got.k.shape[:2]
    assert torch.equal(got.seq_lens.cpu(), want["seq_lens"])
    for b in range(B):
        n = got.k.shape[2] if rows is None else int(rows[b])
        nb = -(-n // got.block_size)
        for name in ("k", "v"):
            assert ref.same_bytes(getattr(got, name)[b, :, :n].cpu(), want[name][b, :, :n]), (name, b)
            sc = name + "_scale"
            assert torch.equal(getattr(got, sc)[b, :, :nb].cpu(), want[sc][b, :, :nb]), (sc, b)
        if got.key_weights is not None:
            assert torch.equal(got.key_weights[b, :, :n].cpu(), want["key_weights"][b, :, :n]), b


# --------------------------------------------------------------------------- append
@BOTH
@pytest.mark.parametrize("B,T,Hkv,Smax,block", [
    (1, 1, 1, 1, 16), (3, 1, 2, 40, 16), (2, 2, 3, 33, 32), (5, 17, 2, 100, 16), (2, 200, 4, 333, 64),
    (3, 129, 1, 300, 128), (1, 1000, 2, 1003, 128), (2, 64, 20, 130, 64),
])
def test_append_matches_reference(cuda_device, dtype, B, T, Hkv, Smax, block):
    dev = cuda_device
    g = torch.Generator().manual_seed(B * 1000 + T + block)
    c = make_switch_kv_cache(B, Smax, Hkv, device=dev, dtype=dtype, block_size=block, track_weights=True)
    c.key_weights.fill_(7.0)
    want = ref.clone(c)
    lens = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
    lens[0] = T
    # three calls: fresh, behind ragged rows (inside blocks, scales growing and not), past the end
    for step, size in enumerate((1.0, 0.3, 40.0)):
        k, v = (_rows(g, B, T, Hkv, 128) * size for _ in range(2))
        nl = None if step == 2 else lens
        switch_kv_cache_append(c, k.to(dev), v.to(dev), new_lens=None if nl is None else nl.to(dev))
        ref.append(want, k, v, nl)
        torch.cuda.synchronize()
        _equal(c, want)


@pytest.mark.parametrize("Smax", [1, 100, 300])
@pytest.mark.parametrize("T", [301, 2 ** 31 - 1, 2 ** 32 + 1])
def test_append_more_rows_than_the_cache_has(cuda_device, T, Smax):
    # one row expanded: behind the cached ones it fills the cache, whatever T and new_lens say
    dev = cuda_device
    g = torch.Generator().manual_seed(T % 1000 + Smax)
    c = make_switch_kv_cache(2, Smax, 2, device=dev, block_size=16)
    want = ref.clone(c)
    first = _rows(g, 2, Smax, 2, 128)
    lens = torch.tensor([0, Smax - 1], dtype=torch.int32)
    switch_kv_cache_append(c, first.to(dev), first.to(dev), new_lens=lens.to(dev))
    ref.append(want, first, first, lens)
    k, v = _rows(g, 2, 1, 2, 128), _rows(g, 2, 1, 2, 128)
    many = torch.full((2,), 2 ** 31 - 1, dtype=torch.int32, device=dev)
    switch_kv_cache_append(c, k.to(dev).expand(2, T, 2, 128), v.to(dev).expand(2, T, 2, 128), new_lens=many)
    ref.append(want, k.expand(2, Smax, 2, 128), v.expand(2, Smax, 2, 128), None)
    torch.cuda.synchronize()
    _equal(c, want)


@BOTH
def test_append_tokens_grow_a_block(cuda_device, dtype):
    # token by token, each larger than the last: the block's rows are rounded again at each doubling
    dev = cuda_device
    g = torch.Generator().manual_seed(5)
    c = make_switch_kv_cache(2, 70, 3, device=dev, dtype=dtype, block_size=32)
    want = ref.clone(c)
    for t in range(40):
        k, v = (_rows(g, 2, 3, 128, spread=0.3) * 1.3 ** (t % 23) for _ in range(2))
        switch_kv_cache_append(c, k.to(dev), v.to(dev))
        ref.append(want, k.unsqueeze(1), v.unsqueeze(1))
    torch.cuda.synchronize()
    _equal(c, want)


@BOTH
@pytest.mark.parametrize("T", [1, 30])
def test_append_special_values_and_edges(cuda_device, dtype, T):
    dev = cuda_device
    g = torch.Generator().manual_seed(11 + T)
    k, v = _rows(g, 6, T, 2, 128), _rows(g, 6, T, 2, 128)
    k[0, 0, 0, :5] = torch.tensor([math.inf, -math.inf, math.nan, 0.0, -0.0]).bfloat16()
    k[1] = 0.0                                            # a block of zeros: scale 0
    k[2] = 1e-40                                          # BF16 subnormals: the smallest scale
    k[3, 0, 1, 7] = 3.3e38                                # the largest values
    v[4] = math.inf                                       # no finite value at all
    v[5] = math.nan
    c = make_switch_kv_cache(6, 64, 2, device=dev, dtype=dtype, block_size=16)
    for start in ([0, 0, 0, 0, 0, 0], [0, 3, 16, 63, 64, 60], [70, -5, 15, 17, 1, 31]):
        start = torch.tensor(start, dtype=torch.int32)
        want = ref.clone(c)
        switch_kv_cache_append(c, k.to(dev), v.to(dev), start=start.to(dev))
        ref.append(want, k, v, start=start)
        torch.cuda.synchronize()
        _equal(c, want)


def test_append_takes_strided_rows_and_foreign_scales(cuda_device):
    # K and V as slices of a fused projection; earlier rows under scales that are no powers of two
    dev = cuda_device
    g = torch.Generator().manual_seed(3)
    B, T, Hq, Hkv = 3, 21, 4, 2
    for dtype in (E4M3, INT8):
        qkv = _rows(g, B, T, Hq + 2 * Hkv, 128).to(dev)
        k, v = qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]
        c = _filled(g, dev, B, 100, Hkv, [5, 0, 40], dtype=dtype, block=32)
        c.k_scale[:, :, 0] = 0.013
        want = ref.clone(c)
        switch_kv_cache_append(c, k, v)
        ref.append(want, k.cpu(), v.cpu())
        torch.cuda.synchronize()
        # 0.013 / s is rounded to FP32 before it meets a byte, which moves no product across a rounding
        # border unless the product lies within 2^-22 of one; these do not
        _equal(c, want, rows=want["seq_lens"])
        one = qkv[:, 3]
        switch_kv_cache_append(c, one[:, Hq:Hq + Hkv], one[:, Hq + Hkv:])
        ref.append(want, one[:, None, Hq:Hq + Hkv].cpu(), one[:, None, Hq + Hkv:].cpu())
        torch.cuda.synchronize()
        _equal(c, want, rows=want["seq_lens"])


# --------------------------------------------------------------------------- decode
def _worst(off, tol, want):
    ratio = torch.where(tol > 0, off / tol, torch.zeros_like(off)).flatten()
    i = int(ratio.argmax())
    at = tuple(int(x) for x in torch.unravel_index(torch.tensor(i), off.shape))
    return f"off by {off.flatten()[i]:.3e} of {want.flatten()[i]:.3e} at {at}, {ratio[i]:.2f} times what is allowed; {int((ratio > 1).sum())} such"


def _check_decode(c, q, route, W, *, sm_scale=None, label="", accumulate=True):
    dev = c.k.device
    before = ref.clone(c)
    O, L = switch_gqa_decode_cached(q.to(dev), c, route.to(dev), window_size=W, sm_scale=sm_scale, accumulate=accumulate)
    torch.cuda.synchronize()
    want, lse, w, (eO, eL, eW) = ref.decode(before, q, route, W, sm_scale)
    O, L = O.cpu().double(), L.cpu().double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(O), nan), label
    off = torch.where(nan, 0.0, (O - want).abs())
    assert bool((off[~nan] <= eO[~nan]).all()), f"{label}: O {_worst(off, eO, want)}"
    none = torch.isneginf(lse)
    assert torch.equal(torch.isneginf(L), none), label
    off = torch.where(none, 0.0, (L - lse).abs())
    assert bool((off[~none] <= eL[~none]).all()), f"{label}: LSE {_worst(off, eL, lse)}"
    if c.key_weights is not None:
        got = c.key_weights.cpu().double()
        old = before["key_weights"].double()
        if not accumulate:
            w, eW = torch.zeros_like(w), torch.zeros_like(eW)
        tol = eW + (old + w) * 2.0 ** -24 * 2
        off = (got - old - w).abs()
        assert bool((off <= tol).all()), f"{label}: weights {_worst(off, tol, w)}"
        assert torch.equal(got[w == 0.0], old[w == 0.0]), label
    return O, L


@BOTH
@pytest.mark.parametrize("B,Smax,Hq,Hkv,W,block", [
    (1, 1, 1, 1, 1, 16), (3, 100, 8, 2, 1, 16), (5, 1000, 32, 8, 200, 64), (4, 5000, 64, 8, 4096, 128),
    (2, 3001, 32, 1, 512, 32), (7, 777, 6, 2, 64, 16), (3, 2049, 40, 8, 1000, 64), (33, 700, 8, 2, 128, 32),
    (2, 20000, 32, 4, 2048, 128), (2, 260, 12, 1, 129, 16), (300, 40, 2, 1, 7, 16),
])
def test_decode_matches_reference(cuda_device, dtype, B, Smax, Hq, Hkv, W, block):
    g = torch.Generator().manual_seed(B * 7919 + Smax + W)
    lens = torch.randint(1, Smax + 1, (B,), generator=g)
    lens[0] = Smax
    if B > 1:
        lens[1] = 1
    if B > 2:
        lens[2] = 0
    if B > 3:
        lens[-1] = 0
    c = _filled(g, cuda_device, B, Smax, Hkv, lens, dtype=dtype, block=block)
    q = _rows(g, B, Hq, 128, spread=0.5)
    route = torch.rand(B, generator=g) < 0.5
    route[0] = True
    _check_decode(c, q, route, W, label=f"B={B} Smax={Smax} Hq={Hq} Hkv={Hkv} W={W}")
    _check_decode(c, q, ~route, W, label="routes swapped, not accumulated", accumulate=False, sm_scale=0.02)


@BOTH
def test_decode_window_edges(cuda_device, dtype):
    # windows around tile and block borders at every alignment of the sequence's end
    g = torch.Generator().manual_seed(29)
    lens = torch.arange(120, 140)
    c = _filled(g, cuda_device, 20, 140, 1, lens, dtype=dtype, block=16)
    q = _rows(g, 20, 4, 128, spread=0.5)
    route = torch.zeros(20, dtype=torch.bool)
    for W in (1, 2, 15, 16, 17, 127, 128, 129, 139, 140, 10 ** 12):
        _check_decode(c, q, route, W, label=f"W={W}")


@BOTH
def test_decode_ignores_what_is_masked(cuda_device, dtype):
    # NaN and infinite rows before the window, NaN bytes behind the length
    dev = cuda_device
    g = torch.Generator().manual_seed(31)
    B, S, Hkv, W = 3, 600, 2, 100
    k, v = _rows(g, B, S, Hkv, 128), _rows(g, B, S, Hkv, 128)
    k[:, :300] = math.nan
    v[:, :300:2] = math.nan
    v[:, 1:300:2] = math.inf
    c = make_switch_kv_cache(B, 700, Hkv, device=dev, dtype=dtype, block_size=64, track_weights=True)
    c.k.view(torch.uint8).fill_(0xFF)
    c.v.view(torch.uint8).fill_(0xFF)
    switch_kv_cache_append(c, k.to(dev), v.to(dev))
    q = _rows(g, B, 8, 128, spread=0.3)
    O, L = _check_decode(c, q, torch.zeros(B, dtype=torch.bool), W, label="window behind NaN rows")
    assert torch.isfinite(O).all() and torch.isfinite(L).all()


def test_decode_carries_nan_through(cuda_device):
    # a query with NaN or infinity; a NaN value that is attended to (e4m3 holds it)
    dev = cuda_device
    g = torch.Generator().manual_seed(37)
    for dtype in (E4M3, INT8):
        c = _filled(g, dev, 3, 300, 2, [300, 200, 150], dtype=dtype, block=32)
        q = _rows(g, 3, 8, 128, spread=0.3)
        q[0, 1, 5] = math.nan
        q[1, 6, 0] = -math.inf
        before = ref.clone(c)
        O, L = switch_gqa_decode_cached(q.to(dev), c, torch.ones(3, dtype=torch.bool, device=dev))
        torch.cuda.synchronize()
        bad = torch.zeros(3, 8, dtype=torch.bool)
        bad[0, 1] = bad[1, 6] = True
        assert torch.equal(torch.isnan(O.cpu()).all(-1), bad) and torch.equal(torch.isnan(O.cpu()).any(-1), bad)
        assert torch.equal(torch.isnan(L.cpu()), bad)
        clean = torch.where(torch.isfinite(q), q, torch.zeros_like(q))
        want, _, _, (eO, _, _) = ref.decode(before, clean, torch.ones(3, dtype=torch.bool), 1024)
        assert bool(((O.cpu().double() - want).abs() <= eO)[~bad].all())
    c = _filled(g, dev, 1, 300, 1, [300], dtype=E4M3, block=32)
    v = c.v.view(torch.uint8)
    v[0, 0, 100, 7] = 0x7F
    O, L = switch_gqa_decode_cached(q[2:, :4].to(dev), c, torch.ones(1, dtype=torch.bool, device=dev))
    O = O.cpu()
    assert torch.isnan(O[0, :, 7]).all() and torch.isfinite(O[0, :, :7]).all() and torch.isfinite(O[0, :, 8:]).all()
    assert torch.isfinite(L.cpu()).all()


@BOTH
@pytest.mark.parametrize("size", [1e-30, 1e-3, 1e4, 1e30])
def test_decode_values_of_any_size(cuda_device, dtype, size):
    # V far from 1 (its scales are taken out tile by tile), K and Q far from 1 with a moderate product
    dev = cuda_device
    g = torch.Generator().manual_seed(41)
    c = make_switch_kv_cache(2, 500, 2, device=dev, dtype=dtype, block_size=64, track_weights=True)
    k = _rows(g, 2, 500, 2, 128, spread=0.3).float() * size
    v = _rows(g, 2, 500, 2, 128).float() * size
    switch_kv_cache_append(c, k.bfloat16().to(dev), v.bfloat16().to(dev))
    q = (_rows(g, 2, 8, 128, spread=0.3).float() / size).bfloat16()
    _check_decode(c, q, torch.tensor([True, False]), 200, label=f"size {size}")


@BOTH
def test_decode_zero_scales_and_peaked_scores(cuda_device, dtype):
    # all-zero K (uniform weights), all-zero V, and one key that takes nearly everything
    dev = cuda_device
    g = torch.Generator().manual_seed(43)
    c = make_switch_kv_cache(3, 400, 1, device=dev, dtype=dtype, block_size=16, track_weights=True)
    k, v = _rows(g, 3, 400, 1, 128), _rows(g, 3, 400, 1, 128)
    k[0] = 0.0
    v[1] = 0.0
    q = _rows(g, 3, 5, 128, spread=0.2)
    k[2, 17, 0] = (q[2, 0].float() * 8).bfloat16()
    switch_kv_cache_append(c, k.to(dev), v.to(dev))
    O, _ = _check_decode(c, q, torch.ones(3, dtype=torch.bool), 64)
    assert torch.equal(O[1], torch.zeros_like(O[1]))


def test_decode_strided_query_four_dims_and_status(cuda_device):
    dev = cuda_device
    g = torch.Generator().manual_seed(47)
    c = _filled(g, dev, 2, 300, 2, [300, 77], dtype=E4M3, block=64, weights=False)
    fused = _rows(g, 2, 12, 128, spread=0.4).to(dev)
    q = fused[:, :8]
    route = torch.tensor([True, False], device=dev)
    st = torch.full((1,), 9, dtype=torch.int32, device=dev)
    O, L = switch_gqa_decode_cached(q, c, route, window_size=50, status_out=st)
    O2, L2 = switch_gqa_decode_cached(q.contiguous().unsqueeze(1), c, route, window_size=50)
    assert O2.shape == (2, 1, 8, 128) and L2.shape == (2, 1, 8)
    assert torch.equal(O, O2[:, 0]) and torch.equal(L, L2[:, 0]) and int(st) == 0


def test_decode_repeats_bit_for_bit(cuda_device):
    dev = cuda_device
    g = torch.Generator().manual_seed(53)
    c = _filled(g, dev, 2, 9000, 2, [9000, 4000], dtype=E4M3, block=64)
    q = _rows(g, 2, 32, 128, spread=0.5).to(dev)
    route = torch.ones(2, dtype=torch.bool, device=dev)
    w0 = c.key_weights.clone()
    first = None
    for _ in range(5):
        c.key_weights.copy_(w0)
        O, L = switch_gqa_decode_cached(q, c, route)
        got = (O, L, c.key_weights.clone())
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


@BOTH
@pytest.mark.parametrize("B,Smax,Hq,Hkv,W", [(40, 6000, 16, 4, 300), (3, 40000, 48, 4, 2000), (5, 700, 72, 3, 129), (6, 9000, 64, 2, 1), (2500, 130, 8, 2, 64)])
def test_decode_many_tiles_per_cta(cuda_device, dtype, B, Smax, Hq, Hkv, W):
    # several tiles a CTA: shares with steps for starting a unit, short and long units mixed, units that span
    # CTAs, several head blocks; and more sequences than threads
    g = torch.Generator().manual_seed(Smax)
    lens = torch.randint(0, Smax + 1, (B,), generator=g)
    lens[:2] = Smax
    c = _filled(g, cuda_device, B, Smax, Hkv, lens, dtype=dtype, block=128)
    q = _rows(g, B, Hq, 128, spread=0.5)
    route = torch.rand(B, generator=g) < 0.4
    route[0] = True
    _check_decode(c, q, route, W, label=f"B={B} Smax={Smax} Hq={Hq} Hkv={Hkv} W={W}")


def test_decode_wait_that_runs_out_reports_timeout(cuda_device):
    # a withheld tile: the bounded wait gives up, the call reports it and the next one is right
    from switchattentionkernels_b200 import _native
    lib = _native.load()
    g = torch.Generator().manual_seed(59)
    c = _filled(g, cuda_device, 64, 2000, 8, [2000] * 64, dtype=E4M3, block=64, weights=False)
    q = _rows(g, 64, 32, 128, spread=0.5).to(cuda_device)
    route = torch.ones(64, dtype=torch.bool, device=cuda_device)
    O, L = switch_gqa_decode_cached(q, c, route)
    lib.swa_test_withhold_kv_load(1)
    try:
        with pytest.raises(RuntimeError, match="timed out"):
            switch_gqa_decode_cached(q, c, route)
    finally:
        lib.swa_test_withhold_kv_load(0)
    torch.cuda.synchronize()
    again = switch_gqa_decode_cached(q, c, route)
    assert torch.equal(again[0], O) and torch.equal(again[1], L)


# --------------------------------------------------------------------------- evict
@BOTH
@pytest.mark.parametrize("B,Smax,Hkv,block,keep,sink,recent", [
    (1, 64, 1, 16, 1, 0, 0), (3, 100, 2, 16, 40, 4, 10), (2, 1000, 3, 64, 300, 0, 0), (4, 777, 2, 32, 500, 0, 500),
    (2, 5000, 2, 128, 1111, 7, 300), (3, 300, 1, 64, 300, 5, 5), (2, 300, 1, 64, 10 ** 12, 5, 5), (2, 9000, 1, 64, 4097, 1, 33),
    (1, 40000, 1, 16, 9000, 3, 1000), (2, 600, 2, 128, 130, 130, 0), (40, 50, 2, 16, 20, 2, 3),
    (10, 2000, 2, 64, 1500, 4, 64),
])
def test_evict_matches_reference(cuda_device, dtype, B, Smax, Hkv, block, keep, sink, recent):
    dev = cuda_device
    g = torch.Generator().manual_seed(Smax + keep % 1000)
    lens = torch.randint(1, Smax + 1, (B,), generator=g)
    lens[0] = Smax
    if B > 1:
        lens[1] = min(keep, Smax)
    if B > 2:
        lens[2] = 0
    c = _filled(g, dev, B, Smax, Hkv, lens, dtype=dtype, block=block)
    c.key_weights[torch.rand(c.key_weights.shape, generator=g).to(dev) < 0.4] = 0.0  # ties
    before = ref.clone(c)
    want, slots = ref.evict(before, min(keep, Smax), sink if keep < Smax else 0, recent if keep < Smax else 0)
    n = min(keep, Smax)
    out = make_switch_kv_cache(B, n + 3, Hkv, device=dev, dtype=dtype, block_size=block, track_weights=True)
    got = switch_kv_cache_evict(c, keep=keep, sink=sink, recent=recent, out=out)
    torch.cuda.synchronize()
    assert torch.equal(got.cpu(), slots)
    _equal(out, want, rows=want["seq_lens"])
    # rows behind the kept ones, and the source, stay as they were
    for b in range(B):
        assert not out.k[b, :, int(want["seq_lens"][b]):].view(torch.uint8).any()
        assert not out.key_weights[b, :, int(want["seq_lens"][b]):].any()
    _equal(c, before)
    # in place: the same rows; everything behind them untouched
    got = switch_kv_cache_evict(c, keep=keep, sink=sink, recent=recent)
    torch.cuda.synchronize()
    assert torch.equal(got.cpu(), slots)
    _equal(c, want, rows=want["seq_lens"])
    for b in range(B):
        m = int(want["seq_lens"][b])
        assert torch.equal(c.k[b, :, m:].cpu().view(torch.uint8), before["k"][b, :, m:].view(torch.uint8))
        assert torch.equal(c.v[b, :, m:].cpu().view(torch.uint8), before["v"][b, :, m:].view(torch.uint8))
        assert torch.equal(c.key_weights[b, :, m:].cpu(), before["key_weights"][b, :, m:])


@pytest.mark.parametrize("Smax,keep", [(65536, 30000), (65537, 65536), (120000, 777), (131073, 100000), (300001, 5001)])
def test_evict_long_sequences(cuda_device, Smax, keep):
    # weights held by 1 to 8 CTAs, 8 or 16 a thread, and read again at every pass past 131072 rows
    dev = cuda_device
    g = torch.Generator().manual_seed(Smax)
    c = make_switch_kv_cache(2, Smax, 1, device=dev, dtype=INT8, block_size=128, track_weights=True)
    c.seq_lens.copy_(torch.tensor([Smax, Smax - 1000]))
    w = torch.rand(2, 1, Smax, generator=g) ** 8
    w[torch.rand(w.shape, generator=g) < 0.3] = 0.0
    c.key_weights.copy_(w)
    c.k.copy_(torch.randint(-127, 128, (1, 1, Smax, 128), generator=g, dtype=torch.int8).expand(2, -1, -1, -1))
    c.v.copy_(c.k.flip(-1))
    c.k_scale.fill_(1.0)
    c.v_scale.fill_(0.5)
    k, v = c.k.clone(), c.v.clone()
    slots = switch_kv_cache_evict(c, keep=keep, sink=3, recent=100)
    torch.cuda.synchronize()
    for b, L in ((0, Smax), (1, Smax - 1000)):
        mid = torch.argsort(w[b, 0, 3:L - 100], descending=True, stable=True)[:keep - 103] + 3
        rows = torch.cat([torch.arange(3), mid.sort().values, torch.arange(L - 100, L)]) if L > keep else torch.arange(L)
        n = rows.numel()
        assert torch.equal(slots[b, 0, :n].cpu(), rows.to(torch.int32)) and bool((slots[b, 0, n:] == -1).all())
        at = rows.to(dev)
        assert torch.equal(c.k[b, 0, :n], k[b, 0, at]) and torch.equal(c.v[b, 0, :n], v[b, 0, at])
        assert torch.equal(c.key_weights[b, 0, :n].cpu(), w[b, 0, rows]) and int(c.seq_lens[b]) == n


@pytest.mark.parametrize("kind", ["equal", "nan", "signed", "infinite", "near"])
def test_evict_orders_any_weights(cuda_device, kind):
    dev = cuda_device
    g = torch.Generator().manual_seed(61)
    c = _filled(g, dev, 2, 700, 2, [700, 650], dtype=E4M3, block=32)
    w = torch.randn(2, 2, 700, generator=g)
    if kind == "equal":
        w[:] = 0.25
    elif kind == "nan":
        w[torch.rand(w.shape, generator=g) < 0.9] = math.nan
    elif kind == "infinite":
        w[:, :, ::3] = math.inf
        w[:, :, 1::3] = -math.inf
        w[:, :, 5::7] = math.nan
    elif kind == "near":  # one unit in the last place apart, zeros of both signs
        w = (torch.randint(0, 40, w.shape, generator=g, dtype=torch.int32) + 0x3F000000).view(torch.float32)
        w[:, :, ::5] = 0.0
        w[:, :, 1::5] = -0.0
    c.key_weights.copy_(w)
    want, slots = ref.evict(ref.clone(c), 300, 5, 17)
    got = switch_kv_cache_evict(c, keep=300, sink=5, recent=17)
    torch.cuda.synchronize()
    assert torch.equal(got.cpu(), slots)


# --------------------------------------------------------------------------- together
@BOTH
def test_serving_loop(cuda_device, dtype):
    # prompt, then tokens: append, decode with weights, cut to the budget when it is exceeded; a captured
    # graph of the step is replayed beside eager steps
    dev = cuda_device
    g = torch.Generator().manual_seed(71)
    B, Hq, Hkv, W, keep = 3, 8, 2, 24, 96
    c = make_switch_kv_cache(B, 128, Hkv, device=dev, dtype=dtype, block_size=16, track_weights=True)
    k, v = _rows(g, B, 90, Hkv, 128, spread=0.4), _rows(g, B, 90, Hkv, 128, spread=0.4)
    lens = torch.tensor([90, 33, 1], dtype=torch.int32)
    switch_kv_cache_append(c, k.to(dev), v.to(dev), new_lens=lens.to(dev))
    want = ref.clone(c)
    route = torch.tensor([True, False, True])
    kt, vt = torch.zeros(B, Hkv, 128, dtype=torch.bfloat16, device=dev), torch.zeros(B, Hkv, 128, dtype=torch.bfloat16, device=dev)
    qt, rt = torch.zeros(B, Hq, 128, dtype=torch.bfloat16, device=dev), route.to(dev)

    def step():
        switch_kv_cache_append(c, kt, vt)
        return switch_gqa_decode_cached(qt, c, rt, window_size=W)

    def cut():
        switch_kv_cache_evict(c, keep=keep, sink=4, recent=32)

    graph, gcut, outs = None, None, None
    for t in range(60):
        k1, v1, q1 = (_rows(g, B, h, 128, spread=0.4) for h in (Hkv, Hkv, Hq))
        kt.copy_(k1)
        vt.copy_(v1)
        qt.copy_(q1)
        if t == 30:
            torch.cuda.synchronize()
            state = {n: getattr(c, n).clone() for n in ("k", "v", "k_scale", "v_scale", "seq_lens", "key_weights")}
            graph, gcut = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
            from switchattentionkernels_b200 import _core
            check, _core.CHECK_DEVICE_STATUS = _core.CHECK_DEVICE_STATUS, False  # reads back: not in a capture
            try:
                with torch.cuda.graph(graph):
                    outs = step()
                with torch.cuda.graph(gcut):
                    cut()
            finally:
                _core.CHECK_DEVICE_STATUS = check
            assert all(torch.equal(getattr(c, n).view(torch.uint8), s.view(torch.uint8)) for n, s in state.items())
        if graph is not None and t % 2 == 0:
            graph.replay()
            O, L = outs
        else:
            O, L = step()
        ref.append(want, k1.unsqueeze(1), v1.unsqueeze(1))
        _equal(c, dict(want, key_weights=c.key_weights.cpu()), rows=want["seq_lens"])
        ro, rl, rw, (eO, eL, eW) = ref.decode(want, q1, route, W)
        assert bool(((O.cpu().double() - ro).abs() <= eO).all()) and bool(((L.cpu().double() - rl).abs() <= eL).all())
        old = want["key_weights"].double()
        for b in range(B):
            n = int(want["seq_lens"][b])
            got = c.key_weights[b, :, :n].cpu().double()
            assert bool(((got - old[b, :, :n] - rw[b, :, :n]).abs() <= eW[b, :, :n] + (old[b, :, :n] + rw[b, :, :n]) * 2.0 ** -23).all())
        want["key_weights"] = c.key_weights.cpu().clone()
        if t % 5 == 4:
            if graph is not None and t % 2 == 0:
                gcut.replay()
            else:
                cut()
            torch.cuda.synchronize()
            kept, _ = ref.evict(want, keep, 4, 32)
            for b in range(B):
                n = int(kept["seq_lens"][b])
                for name in ("k", "v", "key_weights"):
                    want[name][b, :, :n] = kept[name][b, :, :n]
                for name in ("k_scale", "v_scale"):
                    want[name][b, :, :-(-n // 16)] = kept[name][b, :, :-(-n // 16)]
            want["seq_lens"] = kept["seq_lens"]
            _equal(c, want, rows=want["seq_lens"])
    assert int(want["seq_lens"].max()) <= keep + 5


def test_two_streams_at_once(cuda_device):
    # two caches, each driven on a stream of its own, neither the default one
    dev = cuda_device
    g = torch.Generator().manual_seed(73)
    jobs = []
    for i, dtype in enumerate((E4M3, INT8)):
        c = _filled(g, dev, 2, 5000, 2, [4000, 2500], dtype=dtype, block=64)
        k, v, q = _rows(g, 2, 900, 2, 128).to(dev), _rows(g, 2, 900, 2, 128).to(dev), _rows(g, 2, 8, 128, spread=0.4).to(dev)
        jobs.append((c, k, v, q, torch.cuda.Stream()))
    route = torch.ones(2, dtype=torch.bool, device=dev)

    def work(c, k, v, q):
        switch_kv_cache_append(c, k, v)
        O, L = switch_gqa_decode_cached(q, c, route)
        return O, L, switch_kv_cache_evict(c, keep=1500, sink=4, recent=100)

    def copy(c):
        return SwitchKVCache(c.k.clone(), c.v.clone(), c.k_scale.clone(), c.v_scale.clone(), c.seq_lens.clone(),
                             c.key_weights.clone(), c.block_size)

    alone = []
    for c, k, v, q, _ in jobs:
        mine = copy(c)
        alone.append((*work(mine, k, v, q), mine))
    torch.cuda.synchronize()
    got = [None, None]
    for i, (c, k, v, q, s) in enumerate(jobs):
        with torch.cuda.stream(s):
            got[i] = work(c, k, v, q)
    torch.cuda.synchronize()
    for i, (c, *_rest) in enumerate(jobs):
        O, L, slots, mine = alone[i]
        assert torch.equal(got[i][0], O) and torch.equal(got[i][1], L) and torch.equal(got[i][2], slots)
        for n in ("k", "v", "k_scale", "v_scale", "seq_lens", "key_weights"):
            assert torch.equal(getattr(c, n).view(torch.uint8), getattr(mine, n).view(torch.uint8)), n


def test_captured_behind_a_memset_and_a_join(cuda_device):
    # the dependent launches in a graph whose nodes before them are a memset, a copy and another stream's
    # work, replayed several times; and two graphs over the same caches replayed one after the other
    from switchattentionkernels_b200 import _core
    dev = cuda_device
    g = torch.Generator().manual_seed(83)
    c = _filled(g, dev, 2, 3000, 2, [2900, 1700], dtype=E4M3, block=64)
    k, v, q = (_rows(g, 2, h, 128, spread=0.4).to(dev) for h in (2, 2, 8))
    route = torch.tensor([True, False], device=dev)
    out = make_switch_kv_cache(2, 1000, 2, device=dev, block_size=64, track_weights=True)
    lens0, w0 = c.seq_lens.clone(), c.key_weights.clone()
    side = torch.cuda.Stream()

    def step():
        out.k.view(torch.uint8).zero_()
        c.seq_lens.copy_(lens0)
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            c.key_weights.copy_(w0)
            kk = k * 2
        main.wait_stream(side)
        switch_kv_cache_append(c, kk, v)
        O, L = switch_gqa_decode_cached(q, c, route, window_size=500)
        return O, L, switch_kv_cache_evict(c, keep=900, sink=4, recent=100, out=out), c.key_weights.clone(), out.v.view(torch.uint8).clone()

    check, _core.CHECK_DEVICE_STATUS = _core.CHECK_DEVICE_STATUS, False
    try:
        want = step()
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = step()
            graphs.append((graph, got))
    finally:
        _core.CHECK_DEVICE_STATUS = check
    for _ in range(3):
        for graph, got in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rows_past_four_gigabytes(cuda_device):
    # each head's rows take more than 2^31 bytes, the two together more than 2^32
    dev = cuda_device
    g = torch.Generator().manual_seed(79)
    S = 18_000_000
    c = make_switch_kv_cache(1, S, 2, device=dev, dtype=INT8, block_size=128, track_weights=True)
    n = 700
    c.seq_lens.fill_(S - n - 1)
    k, v = _rows(g, 1, n, 2, 128, spread=0.3), _rows(g, 1, n, 2, 128, spread=0.3)
    switch_kv_cache_append(c, k.to(dev), v.to(dev))
    k1, v1 = _rows(g, 1, 2, 128, spread=0.3), _rows(g, 1, 2, 128, spread=0.3)
    switch_kv_cache_append(c, k1.to(dev), v1.to(dev))
    assert int(c.seq_lens) == S
    # the same rows at the same places of their blocks
    off = (S - n - 1) % 128
    small = make_switch_kv_cache(1, n + 1 + off, 2, device=dev, dtype=INT8, block_size=128, track_weights=True)
    small.seq_lens.fill_(off)
    switch_kv_cache_append(small, k.to(dev), v.to(dev))
    switch_kv_cache_append(small, k1.to(dev), v1.to(dev))
    assert torch.equal(c.k[:, :, -(n + 1):], small.k[:, :, off:]) and torch.equal(c.v[:, :, -(n + 1):], small.v[:, :, off:])
    q = _rows(g, 1, 8, 128, spread=0.3).to(dev)
    route = torch.zeros(1, dtype=torch.bool, device=dev)
    O, L = switch_gqa_decode_cached(q, c, route, window_size=n)
    O2, L2 = switch_gqa_decode_cached(q, small, route, window_size=n)
    assert torch.allclose(L, L2, rtol=0, atol=2.0 ** -15) and torch.allclose(O.float(), O2.float(), rtol=2.0 ** -7, atol=2.0 ** -10)
    # the step's weights, then only the window's rows are kept
    slots = switch_kv_cache_evict(c, keep=n, recent=10)
    torch.cuda.synchronize()
    assert int(slots.min()) == S - n and int(slots.max()) == S - 1 and int(c.seq_lens) == n
    switch_kv_cache_evict(small, keep=n, recent=10)
    assert torch.equal(c.k[:, :, :n], small.k[:, :, :n]) and torch.equal(c.v[:, :, :n], small.v[:, :, :n])
    assert torch.equal(c.v_scale[:, :, :6], small.v_scale[:, :, :6])
