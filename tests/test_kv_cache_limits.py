"""Block-scaled 8-bit KV cache at the limits of its formats and calls (CPU only)."""
from __future__ import annotations

import math

import pytest
import torch

import _kv_reference as ref
from switchattentionkernels_b200 import SwitchKVCache, make_switch_kv_cache, switch_kv_cache_append
from test_host_api import dev

E4M3, INT8 = torch.float8_e4m3fn, torch.int8


@pytest.mark.parametrize("dtype", [E4M3, INT8], ids=["e4m3", "int8"])
def test_reference_infinities_saturate_at_the_scale(dtype):
    # +-qmax times the block's scale, which is 0 in a block that holds nothing else but zeros; NaN stays NaN
    # (e4m3) or becomes 0 (int8)
    x = torch.zeros(1, 32, 1, 128, dtype=torch.bfloat16)
    x[0, 0, 0, :3] = torch.tensor([math.inf, -math.inf, math.nan]).bfloat16()
    x[0, 16, 0, :3] = torch.tensor([math.inf, -math.inf, 1.0]).bfloat16()
    c = ref.clone(make_switch_kv_cache(1, 32, 1, device="cpu", dtype=dtype, block_size=16))
    ref.append(c, x, x)
    s = c["k_scale"][0, 0]
    v = ref.values(c["k"])[0, 0] * s.double().repeat_interleave(16)[:, None]
    assert s.tolist() == [0.0, 2.0 ** -8 if dtype == E4M3 else 2.0 ** -6]
    assert v[0, :2].tolist() == [0.0, 0.0] and not v[1:16].any() and not v[0, 3:].any()
    assert math.isnan(v[0, 2]) if dtype == E4M3 else v[0, 2] == 0.0
    top = ref.QMAX[dtype]
    assert v[16, :3].tolist() == [top * float(s[1]), -top * float(s[1]), 1.0]


def test_empty_batch_ends_the_sequences_at_start():
    c = make_switch_kv_cache(3, 40, 2, device="cpu", block_size=16)
    c = SwitchKVCache(*(dev(t) for t in (c.k, c.v, c.k_scale, c.v_scale, c.seq_lens)), block_size=16)
    c.seq_lens.fill_(20)
    empty = dev(torch.zeros(3, 0, 2, 128, dtype=torch.bfloat16))
    switch_kv_cache_append(c, empty, empty)
    assert c.seq_lens.tolist() == [20, 20, 20]
    lens = c.seq_lens
    switch_kv_cache_append(c, empty, empty, start=dev(torch.tensor([5, -3, 70], dtype=torch.int32)))
    assert lens.tolist() == [5, 0, 40] and c.seq_lens is lens
    with pytest.raises(ValueError, match="start"):
        switch_kv_cache_append(c, empty, empty, start=dev(torch.tensor([5, -3], dtype=torch.int32)))
