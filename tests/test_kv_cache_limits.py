"""Block-scaled 8-bit KV cache at the limits of its formats and calls (CPU only)."""
from __future__ import annotations

import math

import pytest
import torch

import _kv_reference as ref
from switchattentionkernels_b200 import make_switch_kv_cache

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
    v = ref.values(c["k"])[0, 0]
    assert s.tolist() == [0.0, 2.0 ** -8 if dtype == E4M3 else 2.0 ** -6]
    assert v[0, :2].tolist() == [0.0, 0.0] and not v[1:16].any() and not v[0, 3:].any()
    assert math.isnan(v[0, 2]) if dtype == E4M3 else v[0, 2] == 0.0
    top = ref.QMAX[dtype]
    assert v[16, :3].tolist() == [top, -top, 1.0 / float(s[1])]
