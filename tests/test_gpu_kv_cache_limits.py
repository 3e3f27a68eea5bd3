"""Block-scaled 8-bit KV cache on the GPU, at the limits of its formats and calls:
blocks without a finite value, empty batches, V scales far apart, a step that failed."""
from __future__ import annotations

import math

import pytest
import torch

import _kv_reference as ref
from switchattentionkernels_b200 import make_switch_kv_cache, switch_gqa_decode_cached, switch_kv_cache_append

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BOTH = pytest.mark.parametrize("dtype", [E4M3, INT8], ids=["e4m3", "int8"])


# --------------------------------------------------------------------------- append
@BOTH
@pytest.mark.parametrize("T", [1, 30])
def test_infinities_of_a_block_without_finite_values_are_zero(cuda_device, dtype, T):
    # infinities saturate at 448 / 127 times a scale that they do not count for: 0 where nothing else raises
    # it; NaN stays NaN (e4m3) or becomes 0 (int8).  Later rows that raise the scale leave both as they are.
    dev = cuda_device
    x = torch.zeros(4, T, 2, 128, dtype=torch.bfloat16)
    x[0] = math.inf
    x[1, :, :, ::2] = -math.inf
    x[2] = math.inf
    x[2, 0, 1, 5] = math.nan
    x[3, 0, 0, 3], x[3, 0, 0, 4] = math.inf, 1.0  # (a finite value next to it: it saturates)
    c = make_switch_kv_cache(4, 64, 2, device=dev, dtype=dtype, block_size=32)
    switch_kv_cache_append(c, x.to(dev), (-x).to(dev))
    value = {n: (t.float() * s.repeat_interleave(32, 2)[..., None]).cpu() for n, t, s in (("k", c.k, c.k_scale), ("v", c.v, c.v_scale))}
    for n, sign in (("k", 1.0), ("v", -1.0)):
        assert not value[n][:2].any()
        nan = torch.zeros(2, 64, 128, dtype=torch.bool)
        nan[1, 0, 5] = dtype == E4M3
        assert torch.equal(torch.isnan(value[n][2]), nan) and not value[n][2][~nan].any()
        one, top = (2.0 ** -8, 448.0) if dtype == E4M3 else (2.0 ** -6, 127.0)
        assert value[n][3, 0, 0, 3] == sign * top * one and value[n][3, 0, 0, 4] == sign
    ones = torch.ones(4, 2, 2, 128, dtype=torch.bfloat16, device=dev)
    switch_kv_cache_append(c, ones, ones)
    for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
        v = (t.float() * s.repeat_interleave(32, 2)[..., None]).cpu()
        assert not v[:2, :, :T].any() and bool((v[:2, :, T:T + 2] == 1.0).all())
        assert torch.equal(torch.isnan(v[2]), nan)


@BOTH
def test_empty_batch_with_start_drops_the_rows_from_there_on(cuda_device, dtype):
    # no new row (T = 0) is what new_lens = 0 is: the sequence ends at `start`
    dev = cuda_device
    g = torch.Generator().manual_seed(7)
    x = torch.randn(3, 20, 2, 128, generator=g).bfloat16().to(dev)
    start = torch.tensor([5, -3, 70], dtype=torch.int32, device=dev)
    none = torch.zeros(3, dtype=torch.int32, device=dev)
    got = []
    for rows, lens in ((x[:, :0], None), (x[:, :0], none), (x, none), (x[:, :1], none)):
        c = make_switch_kv_cache(3, 40, 2, device=dev, dtype=dtype, block_size=16, track_weights=True)
        switch_kv_cache_append(c, x, x)
        before = ref.clone(c)
        switch_kv_cache_append(c, rows, rows, new_lens=lens, start=start)
        got.append(c.seq_lens.tolist())
        assert torch.equal(c.k.cpu().view(torch.uint8), before["k"].view(torch.uint8)) and torch.equal(c.k_scale.cpu(), before["k_scale"])
    assert got == [[5, 0, 40]] * 4
    switch_kv_cache_append(c, x[:, :0], x[:, :0])  # behind the cached rows: nothing changes
    assert c.seq_lens.tolist() == [5, 0, 40]


# --------------------------------------------------------------------------- decode
def _within_its_own_size(c, q, route, W, label):
    """Decode against 64 bits, the error counted against what each head's keys contribute."""
    dev = c.k.device
    before = ref.clone(c)
    O, L = switch_gqa_decode_cached(q.to(dev), c, route.to(dev), window_size=W)
    torch.cuda.synchronize()
    want, lse, _, (_, eL, _) = ref.decode(before, q, route, W)
    B, Hq, _ = q.shape
    Hkv, bs = c.k.shape[1], c.block_size
    r = Hq // Hkv
    for b in range(B):
        n = int(before["seq_lens"][b])
        at = torch.arange(0 if bool(route[b]) else max(0, n - W), n)
        for h in range(Hq):
            g = h // r
            k = ref.values(before["k"][b, g, at]) * ref.values(before["k_scale"][b, g])[at // bs][:, None]
            vs = ref.values(before["v_scale"][b, g])[at // bs]
            v8 = ref.values(before["v"][b, g, at]).abs()
            qq = ref.values(q[b, h])
            w = torch.exp2((k @ qq) * (ref.LOG2E / math.sqrt(128.0)) - lse[b, h])
            # a weight: its score and the LSE, each a sum of 3 x 128 FP32 products times FP32 factors (off by at
            # most (384 + 8) 2^-23 of the sum of magnitudes), exp2 and sums 2^-18; P rounded to FP16: 2^-11;
            # the FP32 sums of 3 x 128 products again
            ds = (k.abs() @ qq.abs()) * (ref.LOG2E / math.sqrt(128.0)) * (392 * 2.0 ** -23)
            rel = math.log(2.0) * 1.01 * (ds + ds.max()) + 2.0 ** -18 + 2.0 ** -11 + 392 * 2.0 ** -23
            # P's last step: 2^-24 (int8; e4m3 2^-26) of a reference that lies less than 2^4 above the
            # largest w vs of its tile
            last = 2.0 ** -20 * float((w * vs).max())
            tol = (w * vs * rel) @ v8 + last * v8.sum(0)
            tol = tol + (want[b, h].abs() + tol) * 2.0 ** -8  # and O to BF16
            off = (O[b, h].cpu().double() - want[b, h]).abs()
            i = int((off / tol.clamp(min=1e-300)).argmax())
            assert bool((off <= tol).all()), f"{label}: head {h}, off by {off[i]:.3e} of {want[b, h, i]:.3e}, allowed {tol[i]:.3e}"
    assert bool(((L.cpu().double() - lse).abs() <= eL).all()), label


@BOTH
@pytest.mark.parametrize("light,heavy", [(2.0 ** -20, 1.0), (2.0 ** -30, 1.0), (1.0, 2.0 ** 30), (3e-5, 7.0), (2.0 ** -60, 2.0 ** 60),
                                         (2.0 ** -100, 2.0 ** -60), (0.25, 1.0), (1.0, 0.0)])
@pytest.mark.parametrize("Hq,Hkv,block", [(2, 1, 16), (8, 1, 32), (12, 1, 64), (8, 2, 128)])
def test_decode_v_scales_far_apart(cuda_device, dtype, light, heavy, Hq, Hkv, block):
    # keys that take all of the weight lie under a V scale far below another block's of the same tile, whose
    # keys take next to none, as much of the sum as the others, or all of it
    dev = cuda_device
    g = torch.Generator().manual_seed(Hq * 100 + block)
    S, lens = 700, [700, 333, 130]
    nb = -(-S // block)
    is_heavy = torch.rand(3, Hkv, nb, generator=g) < 0.4
    is_heavy[:, :, 0] = False
    is_heavy[:, :, 1] = True
    gap = math.log2(heavy / light) if heavy > 0 else 0.0
    for below in (gap + 30.0, gap, 0.0):  # log2 of a light key's weight over a heavy one's
        c = make_switch_kv_cache(3, S, Hkv, device=dev, dtype=dtype, block_size=block)
        k = torch.randint(-2, 3, (3, Hkv, S, 128), generator=g).float()
        # the first dim sets the score: 16 * d * 2^-3 log2(e) / sqrt(128) in log2 units
        d = below / (16.0 * 2.0 ** -3 * ref.LOG2E / math.sqrt(128.0))
        top = torch.where(is_heavy, -0.5 * d, 0.5 * d).clamp(-120.0, 120.0).round()
        k[..., 0] = top.repeat_interleave(block, 2)[:, :, :S]
        c.k.copy_(k.to(dtype).to(dev))
        c.k_scale.fill_(2.0 ** -3)
        c.v.copy_(torch.randint(-100, 101, (3, Hkv, S, 128), generator=g).float().to(dtype).to(dev))
        c.v_scale.copy_(torch.where(is_heavy, torch.tensor(heavy), torch.tensor(light)).to(dev))
        c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        q = torch.randn(3, Hq, 128, generator=g).bfloat16()
        q[..., 0] = 16.0
        _within_its_own_size(c, q, torch.tensor([True, False, True]), 200, f"{light} {heavy} {below}")


@BOTH
@pytest.mark.parametrize("B,S,Hq,Hkv,block", [(24, 4000, 8, 4, 32), (6, 9000, 40, 2, 16)])
def test_decode_v_scales_far_apart_in_some_tiles(cuda_device, dtype, B, S, Hq, Hkv, block):
    # many tiles a CTA, every third stretch of 400 rows with scales of any size
    dev = cuda_device
    g = torch.Generator().manual_seed(S)
    c = make_switch_kv_cache(B, S, Hkv, device=dev, dtype=dtype, block_size=block)
    shape = (B, Hkv, c.k_scale.shape[2])
    c.k.copy_(torch.randint(-100, 101, c.k.shape, generator=g).float().to(dtype).to(dev))
    c.v.copy_(torch.randint(-100, 101, c.k.shape, generator=g).float().to(dtype).to(dev))
    c.k_scale.copy_(2.0 ** torch.randint(-10, -5, shape, generator=g).float())
    wild = torch.arange(shape[2]) * block // 400 % 3 == 1
    c.v_scale.copy_(torch.where(wild, 2.0 ** torch.randint(-30, 1, shape, generator=g).float(), torch.tensor(2.0 ** -14)))
    c.seq_lens.copy_(torch.randint(S // 2, S + 1, (B,), generator=g, dtype=torch.int32))
    q = torch.randn(B, Hq, 128, generator=g).bfloat16()
    _within_its_own_size(c, q, torch.rand(B, generator=g) < 0.5, 1000, f"B={B} S={S}")


@BOTH
@pytest.mark.parametrize("Hq", [1, 8])
def test_decode_v_scales_far_apart_under_scores_of_any_size(cuda_device, dtype, Hq):
    # scores so large that a unit in their last place is not small, V scales whose ratio is no power of two: the
    # keys with all the weight share one V row, which is O whatever the scores' rounding is
    dev = cuda_device
    g = torch.Generator().manual_seed(Hq)
    row = torch.randint(-100, 101, (128,), generator=g).float().to(dtype)
    for size in (1.0, 10.0, 90.0, 100.0, 117.0, 131.0, 150.0, 176.0, 200.0, 255.0, 1000.0):
        for light, heavy in ((3e-5, 7.0), (0.001, 0.9), (2.0 ** -20, 1.0)):
            c = make_switch_kv_cache(1, 300, 1, device=dev, dtype=dtype, block_size=16)
            k = torch.full((300, 128), 100.0)
            k[16:48], k[130:150] = -100.0, -100.0
            c.k.copy_(k.to(dtype)[None, None].to(dev))
            c.v.copy_(row.expand(1, 1, 300, 128).to(dev))
            c.k_scale.fill_(1.0)
            c.v_scale.fill_(light)
            c.v_scale[:, :, 1:3] = heavy
            c.v[0, 0, 130:150] = 0  # (these under the light scale)
            c.seq_lens.fill_(300)
            q = torch.full((1, Hq, 128), size, dtype=torch.bfloat16, device=dev)
            O, _ = switch_gqa_decode_cached(q, c, torch.ones(1, dtype=torch.bool, device=dev))
            want = ref.values(row) * float(torch.tensor(light))
            # equal scores give equal weights, 1 / n each: P's FP16 and last steps, sums, and O to BF16
            tol = want.abs() * (2.0 ** -8 + 2.0 ** -10) + 1e-12
            off = (O[0].cpu().double() - want).abs()
            assert bool((off <= tol).all()), (size, light, heavy, float((off / tol).max()))


@BOTH
@pytest.mark.parametrize("size", [1.0, 2.0 ** 8, 2.0 ** 14])
def test_decode_query_with_a_far_larger_entry(cuda_device, dtype, size):
    # a large entry that meets no key: the others are held to within 2^-23.9 of it, 2^-25 in e4m3 parts
    dev = cuda_device
    g = torch.Generator().manual_seed(41)
    c = make_switch_kv_cache(2, 900, 2, device=dev, dtype=dtype, block_size=64)
    k, v = torch.randn(2, 900, 2, 128, generator=g).bfloat16(), torch.randn(2, 900, 2, 128, generator=g).bfloat16()
    k[..., 0] = 0.0
    switch_kv_cache_append(c, k.to(dev), v.to(dev))
    before = ref.clone(c)
    q = torch.randn(2, 8, 128, generator=g).bfloat16()
    q[..., 0] = size
    route = torch.ones(2, dtype=torch.bool)
    O, L = switch_gqa_decode_cached(q.to(dev), c, route.to(dev))
    torch.cuda.synchronize()
    want, lse, _, (eO, eL, _) = ref.decode(before, q, route, 1024)
    kk = ref.values(before["k"]) * ref.values(before["k_scale"]).repeat_interleave(64, 2)[:, :, :900, None]
    top = ref.values(q).abs().amax(-1)
    for b in range(2):
        for h in range(8):
            ds = 2.0 ** (-23.9 if dtype == INT8 else -25) * float(top[b, h] * kk[b, h // 4].abs().sum(-1).max()) * ref.LOG2E / math.sqrt(128.0)
            # a score off by ds moves the LSE by at most that, and every weight by at most twice that in log2
            assert abs(float(L[b, h]) - float(lse[b, h])) <= float(eL[b, h]) + ds
            v8 = (ref.values(before["v"][b, h // 4]).abs() * ref.values(before["v_scale"][b, h // 4]).repeat_interleave(64)[:900, None]).amax(0)
            off = (O[b, h].cpu().double() - want[b, h]).abs()
            assert bool((off <= eO[b, h] + (2.0 ** (2.0 * ds) - 1.0) * v8 * (1.0 + 2.0 ** -8)).all())


def test_decode_that_timed_out_leaves_the_weights(cuda_device):
    # a withheld tile: the call reports it, key_weights are what they were, and the step can be taken again
    from switchattentionkernels_b200 import _native
    lib = _native.load()
    dev = cuda_device
    g = torch.Generator().manual_seed(61)
    c = make_switch_kv_cache(64, 2000, 8, device=dev, block_size=64, track_weights=True)
    x = torch.randn(64, 2000, 8, 128, generator=g).bfloat16().to(dev)
    switch_kv_cache_append(c, x, x.flip(-1).contiguous())
    c.key_weights.copy_(torch.rand(64, 8, 2000, generator=g))
    before = c.key_weights.clone()
    q = torch.randn(64, 32, 128, generator=g).bfloat16().to(dev)
    route = torch.ones(64, dtype=torch.bool, device=dev)
    O, L = switch_gqa_decode_cached(q, c, route)
    after = c.key_weights.clone()
    assert not torch.equal(after, before)
    c.key_weights.copy_(before)
    lib.swa_test_withhold_kv_load(1)
    try:
        with pytest.raises(RuntimeError, match="timed out"):
            switch_gqa_decode_cached(q, c, route)
    finally:
        lib.swa_test_withhold_kv_load(0)
    torch.cuda.synchronize()
    assert torch.equal(c.key_weights, before)
    again = switch_gqa_decode_cached(q, c, route)
    assert torch.equal(again[0], O) and torch.equal(again[1], L) and torch.equal(c.key_weights, after)


def test_decode_that_times_out_takes_one_limit(cuda_device):
    # the loads in flight are waited for before the CTA ends, the one that was never issued is not
    from switchattentionkernels_b200 import _native
    lib = _native.load()
    c = make_switch_kv_cache(1, 300000, 1, device=cuda_device)
    c.seq_lens.fill_(300000)
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16, device=cuda_device)
    route = torch.ones(1, dtype=torch.bool, device=cuda_device)
    switch_gqa_decode_cached(q, c, route)
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    lib.swa_test_withhold_kv_load(1)
    try:
        a.record()
        with pytest.raises(RuntimeError, match="timed out"):
            switch_gqa_decode_cached(q, c, route)
        b.record()
    finally:
        lib.swa_test_withhold_kv_load(0)
    torch.cuda.synchronize()
    assert 900 < a.elapsed_time(b) < 1800  # ms; a limit is 1 s


def test_first_calls_from_several_threads(cuda_device):
    # every thread with its own cache and stream; the results are those of the calls one by one
    import threading
    dev = cuda_device
    g = torch.Generator().manual_seed(67)
    jobs = []
    for i in range(6):
        c = make_switch_kv_cache(2, 3000, 2, device=dev, dtype=(E4M3, INT8)[i % 2], block_size=64, track_weights=i % 3 == 0)
        x = torch.randn(2, 2500, 2, 128, generator=g).bfloat16().to(dev)
        q = torch.randn(2, (8, 16)[i // 3], 128, generator=g).bfloat16().to(dev)
        jobs.append((c, x, q, torch.cuda.Stream()))
    route = torch.tensor([True, False], device=dev)
    torch.cuda.synchronize()
    got, errors = [None] * 6, []

    def work(i):
        c, x, q, stream = jobs[i]
        try:
            with torch.cuda.stream(stream):
                switch_kv_cache_append(c, x, x)
                got[i] = [switch_gqa_decode_cached(q, c, route, accumulate=False) for _ in range(5)]
                stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors
    for i, (c, _, q, _) in enumerate(jobs):
        O, L = switch_gqa_decode_cached(q, c, route, accumulate=False)
        assert c.seq_lens.tolist() == [2500, 2500]
        for o, lse in got[i]:
            assert torch.equal(o, O) and torch.equal(lse, L)
