"""Plain restatements, in 64 bits on the CPU, of the block-scaled KV cache operators."""
from __future__ import annotations

import math

import torch

D = 128
LOG2E = 1.0 / math.log(2.0)
QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def pow2_at_least(a: float) -> float:
    """Smallest power of two >= a (at least 2^-126); 0 for 0."""
    if a == 0.0:
        return 0.0
    m, e = math.frexp(a)  # a = m 2^e, 1/2 <= m < 1
    return math.ldexp(1.0, max(e - 1 if m == 0.5 else e, -126))


def round8(y: torch.Tensor, dtype) -> torch.Tensor:
    """float64 values -> 8-bit, to nearest even, saturating; NaN kept (e4m3) or 0 (int8)."""
    if dtype == torch.int8:
        return torch.nan_to_num(y, nan=0.0, posinf=127.0, neginf=-127.0).clamp(-127, 127).round().to(torch.int8)
    c = y.clamp(-448.0, 448.0)
    mag = c.abs().clamp(min=2.0 ** -6)
    _, e = torch.frexp(mag)
    step = torch.ldexp(torch.ones_like(c), e - 4)  # 8 steps in each binade, from 2^-6 on
    r = (c / step).round() * step
    return torch.where(torch.isnan(y), y, r).float().to(torch.float8_e4m3fn)  # (already on the e4m3 grid)


def values(t: torch.Tensor) -> torch.Tensor:
    return t.float().double()


def clone(cache):
    """The cache's tensors on the CPU."""
    return {n: (None if getattr(cache, n) is None else getattr(cache, n).detach().cpu().clone())
            for n in ("k", "v", "k_scale", "v_scale", "seq_lens", "key_weights")} | {"block": cache.block_size}


def append(c: dict, k_new, v_new, new_lens=None, start=None) -> None:
    """Append to the cloned cache ``c`` in place."""
    bs = c["block"]
    B, Hkv, Smax, _ = c["k"].shape
    T = k_new.shape[1]
    start = c["seq_lens"].clone() if start is None else start
    for b in range(B):
        s0 = min(max(int(start[b]), 0), Smax)
        n = T if new_lens is None else min(max(int(new_lens[b]), 0), T)
        e0 = min(s0 + n, Smax)
        c["seq_lens"][b] = e0
        for x, cache, scale in ((k_new, c["k"], c["k_scale"]), (v_new, c["v"], c["v_scale"])):
            dtype = cache.dtype
            for g in range(Hkv):
                for blk in range(s0 // bs, -(-e0 // bs)):
                    lo, hi = max(s0, blk * bs), min(e0, (blk + 1) * bs)
                    if lo >= hi:
                        continue
                    rows = values(x[b, lo - s0:hi - s0, g])
                    fin = rows[torch.isfinite(rows)].abs()
                    need = pow2_at_least(float(fin.max()) / QMAX[dtype]) if fin.numel() and float(fin.max()) > 0 else 0.0
                    old = float(scale[b, g, blk])
                    new = max(need, pow2_at_least(old) if lo > blk * bs else 0.0)
                    if lo > blk * bs and new != old:
                        past = values(cache[b, g, blk * bs:lo])
                        cache[b, g, blk * bs:lo] = round8(past * (old / new), dtype)
                    cache[b, g, lo:hi] = round8(rows / new if new > 0 else rows * (dtype != torch.int8), dtype)
                    scale[b, g, blk] = new
        if c["key_weights"] is not None:
            c["key_weights"][b, :, s0:e0] = 0.0


def decode(c: dict, q, route, window: int, sm_scale=None):
    """``(O, LSE, weights, err)``: float64 O, LSE (log2) and each key's weight of the step, and
    the error bounds ``err = (O, LSE, weights)`` that the kernel's number formats allow."""
    bs = c["block"]
    B, Hkv, Smax, _ = c["k"].shape
    Hq = q.shape[1]
    r = Hq // Hkv
    sl2 = (sm_scale if sm_scale is not None else D ** -0.5) * LOG2E
    O = torch.full((B, Hq, D), math.nan, dtype=torch.float64)
    LSE = torch.full((B, Hq), -math.inf, dtype=torch.float64)
    W = torch.zeros((B, Hkv, Smax), dtype=torch.float64)
    eO, eL, eW = torch.zeros_like(O), torch.zeros_like(LSE), torch.zeros_like(W)
    for b in range(B):
        L = min(max(int(c["seq_lens"][b]), 0), Smax)
        lo = 0 if bool(route[b]) else max(0, L - window)
        if L <= lo:
            continue
        blk = torch.arange(lo, L) // bs
        for g in range(Hkv):
            k = values(c["k"][b, g, lo:L]) * values(c["k_scale"][b, g])[blk][:, None]
            v = values(c["v"][b, g, lo:L]) * values(c["v_scale"][b, g])[blk][:, None]
            qq = values(q[b, g * r:(g + 1) * r])
            s = (qq @ k.T) * sl2
            m = s.amax(1, keepdim=True)
            p = torch.exp2(s - m)
            lse = m[:, 0] + torch.log2(p.sum(1))
            w = torch.exp2(s - lse[:, None])
            O[b, g * r:(g + 1) * r] = w @ v
            LSE[b, g * r:(g + 1) * r] = lse
            W[b, g, lo:L] = w.sum(0)
            # a score is a sum of 3 x 128 products in FP32 (each addition off by at most 2^-23 of the
            # sum of magnitudes, truncation included), times FP32 factors: off by at most
            # (384 + 8) 2^-23 of that sum; the rest of q that three parts leave is far below it
            ds = (qq.abs() @ k.abs().T) * sl2 * (392 * 2.0 ** -23)
            dmax = ds.amax(1, keepdim=True)
            rel = math.log(2.0) * (ds + dmax) * 1.01 + 2.0 ** -18  # of a weight: its score and the LSE; exp2 and sums
            eL[b, g * r:(g + 1) * r] = dmax[:, 0] + 2.0 ** -18 + lse.abs() * 2.0 ** -22
            eW[b, g, lo:L] = (w * rel).sum(0)
            # O: P to FP16 (2^-11) and FP32 sums of 3 x 128 products (2^-14), on top of the weights'.
            # Then P's last step.  What is cut into three parts is x = 2^(s - m) vs / vref, m the largest
            # score and vref the largest V scale of a tile: for int8 in steps of 1 / (127 * 65536), so x is off
            # by at most 1 / 16646144 < 2^-23.9 and the key's share of O by that times 2^(m - lse) vref
            # |v8| <= 2^-23.9 max(vs) |v8|; for e4m3 (steps of 2^-17 of 1 / 256, FP16's 2^-24 of it) by less.
            v8 = values(c["v"][b, g, lo:L]).abs()
            last = 2.0 ** -23.9 * values(c["v_scale"][b, g])[blk].max() * v8.sum(0)[None, :]
            eo = (w * (rel + 2.0 ** -11 + 392 * 2.0 ** -23)) @ v.abs() + last
            # and O to BF16 (2^-8)
            eO[b, g * r:(g + 1) * r] = eo + (O[b, g * r:(g + 1) * r].abs() + eo) * 2.0 ** -8
    return O, LSE, W, (eO, eL, eW)


def evict(c: dict, keep: int, sink: int, recent: int):
    """``(kept, slots)``: the cut cache (rows past the kept ones zero) and the former rows."""
    bs = c["block"]
    B, Hkv, Smax, _ = c["k"].shape
    n = min(keep, Smax)
    dtype = c["k"].dtype
    zero8 = lambda: torch.zeros((B, Hkv, n, D), dtype=torch.int8).view(dtype)  # noqa: E731
    nb = -(-n // bs)
    out = {"k": zero8(), "v": zero8(), "k_scale": torch.zeros(B, Hkv, nb), "v_scale": torch.zeros(B, Hkv, nb),
           "seq_lens": torch.zeros(B, dtype=torch.int32), "key_weights": torch.zeros(B, Hkv, n), "block": bs}
    slots = torch.full((B, Hkv, n), -1, dtype=torch.int32)
    for b in range(B):
        L = min(max(int(c["seq_lens"][b]), 0), Smax)
        out["seq_lens"][b] = min(L, keep)
        for g in range(Hkv):
            if L <= keep:
                rows = list(range(L))
            else:
                w = c["key_weights"][b, g].tolist()
                mid = sorted(range(sink, L - recent), key=lambda i: (-w[i] if w[i] == w[i] else math.inf, i))
                rows = sorted(list(range(sink)) + mid[:keep - sink - recent] + list(range(L - recent, L)))
            at = torch.tensor(rows, dtype=torch.long)
            m = at.numel()
            slots[b, g, :m] = at.to(torch.int32)
            out["key_weights"][b, g, :m] = c["key_weights"][b, g, at]
            for name in ("k", "v"):
                src = values(c[name + "_scale"][b, g])[at // bs]
                for blk in range(-(-m // bs)):
                    sl = slice(blk * bs, min(m, (blk + 1) * bs))
                    top = float(src[sl].max())
                    out[name + "_scale"][b, g, blk] = top
                    x = c[name][b, g, at[sl]]
                    ratio = torch.where(src[sl] == top, torch.ones_like(src[sl]), src[sl] / top if top > 0 else src[sl])
                    same = (ratio == 1.0)[:, None]
                    moved = round8(values(x) * ratio[:, None], dtype)
                    out[name][b, g, sl] = torch.where(same, x.view(torch.int8), moved.view(torch.int8)).view(dtype)
    return out, slots


def same_bytes(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Equal 8-bit values; a NaN's sign does not count."""
    if a.dtype == torch.int8:
        return torch.equal(a, b)
    x, y = a.view(torch.uint8), b.view(torch.uint8)
    nan = ((x & 0x7F) == 0x7F) & ((y & 0x7F) == 0x7F)
    return bool(((x == y) | nan).all())
