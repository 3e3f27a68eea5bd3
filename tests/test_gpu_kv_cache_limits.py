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
