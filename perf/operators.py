"""Cases and plain forms of the operators of the block-scaled 8-bit KV cache.

Three operators of one serving loop, over a cache ``k`` / ``v`` ``[B, Hkv, Smax, 128]``
(e4m3 or int8) with one FP32 scale per (block of ``block`` rows, KV head):

* ``append``: new BF16 K/V rows into the cache.  The scale of a block is a power of
  two that only grows; rows that the block held before are rounded again when it does.
* ``decode``: one query token per sequence attends to its cached keys (all of them, or
  the last ``window``); optionally every key's attention weight, summed over the
  query heads of its group, is added to ``key_weights``.
* ``evict``: of every (sequence, KV head) keep the first ``sink`` rows, the last
  ``recent`` and the heaviest of the rest, ``keep`` rows in all, moved together in order.

``own`` selects the framework's kernels; otherwise the plain torch forms run.
"""
import math

import torch

own = False

QMAX = {"e4m3": 448.0, "int8": 127.0}
DTYPE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
D = 128


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of every running sequence of a serving batch: pure latency
        {"name": "append_token_b64", "op": "append", "dtype": "e4m3", "B": 64, "Hkv": 8, "T": 1, "Smax": 1024, "block": 64, "fill": 1023, "ragged": True},
        # ragged prompts of a packed batch written into fresh sequences
        {"name": "append_prompts_ragged16", "op": "append", "dtype": "e4m3", "B": 16, "Hkv": 8, "T": 8192, "Smax": 8192, "block": 64, "fill": 0, "ragged": True},
        # a long chunk of two long sequences, starting inside a block
        {"name": "append_chunk_32k_int8", "op": "append", "dtype": "int8", "B": 2, "Hkv": 4, "T": 32768, "Smax": 34000, "block": 128, "fill": 1000, "ragged": False},
        # a single short sequence: latency of the whole step
        {"name": "decode_b1_1k", "op": "decode", "dtype": "e4m3", "B": 1, "Hq": 8, "Hkv": 2, "Smax": 1024, "block": 64, "window": 256, "p_full": 1.0, "weights": False, "idle": False},
        # the serving batch: 64 sequences of 16K-32K keys, one in eight routed full
        {"name": "decode_b64_32k", "op": "decode", "dtype": "e4m3", "B": 64, "Hq": 32, "Hkv": 8, "Smax": 32768, "block": 64, "window": 1024, "p_full": 0.125, "weights": False, "idle": False},
        # ragged batch with an idle slot, int8 cache, attention weights accumulated for eviction
        {"name": "decode_ragged16_int8_weights", "op": "decode", "dtype": "int8", "B": 16, "Hq": 64, "Hkv": 8, "Smax": 8192, "block": 32, "window": 4096, "p_full": 0.3, "weights": True, "idle": True},
        # two 131K-token sequences, every key read, weights accumulated
        {"name": "decode_b2_131k_weights", "op": "decode", "dtype": "e4m3", "B": 2, "Hq": 32, "Hkv": 4, "Smax": 131072, "block": 128, "window": 2048, "p_full": 1.0, "weights": True, "idle": False},
        # a few short sequences cut to a quarter
        {"name": "evict_b8_1k", "op": "evict", "dtype": "e4m3", "B": 8, "Hkv": 2, "Smax": 1024, "block": 16, "keep": 256, "sink": 4, "recent": 64},
        # ragged batch: some sequences are under the budget and stay whole
        {"name": "evict_ragged16_int8", "op": "evict", "dtype": "int8", "B": 16, "Hkv": 8, "Smax": 8192, "block": 64, "keep": 2000, "sink": 4, "recent": 1024},
        # long sequences cut to 8K rows around their window
        {"name": "evict_b4_32k", "op": "evict", "dtype": "e4m3", "B": 4, "Hkv": 8, "Smax": 32768, "block": 64, "keep": 8192, "sink": 16, "recent": 1024},
    ]


def _log_int(rng, lo, hi):
    """A whole number in [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "evict"])
    dtype = rng.choice(["e4m3", "int8"])
    Hkv = rng.choice([1, 2, 3, 4, 8])
    block = rng.choice([16, 32, 64, 128])
    B = _log_int(rng, 1, 64)
    if op == "append":
        T = 1 if rng.random() < 0.4 else _log_int(rng, 2, 16384)
        T = max(1, min(T, 65536 // B))
        fill = _log_int(rng, 1, 1500) - 1
        return {"op": op, "dtype": dtype, "B": B, "Hkv": Hkv, "T": T, "Smax": T + fill + rng.randint(0, 100), "block": block, "fill": fill,
                "ragged": rng.random() < 0.5}
    Smax = _log_int(rng, 1 if op == "decode" else 64, 131072)
    Smax = max(16, min(Smax, 1048576 // (B * Hkv)))
    if op == "decode":
        return {"op": op, "dtype": dtype, "B": B, "Hq": Hkv * rng.choice([1, 2, 4, 4, 5, 8, 8, 16]), "Hkv": Hkv, "Smax": Smax, "block": block,
                "window": _log_int(rng, 1, 4096), "p_full": rng.choice([0.0, 0.125, 0.5, 1.0]), "weights": rng.random() < 0.5,
                "idle": rng.random() < 0.2}
    keep = max(2, int(Smax * rng.uniform(0.1, 0.9)))
    sink = rng.randint(0, min(16, keep // 2))
    return {"op": op, "dtype": dtype, "B": B, "Hkv": Hkv, "Smax": Smax, "block": block, "keep": keep, "sink": sink,
            "recent": rng.randint(0, keep - sink)}


def _lens(case):
    """``(start, new)`` of an append case, or ``(lens, route)``: the case's own, whatever the seed of its data."""
    g = torch.Generator().manual_seed(case["B"] * 1000003 + case["Smax"])
    B = case["B"]
    if case["op"] == "append":
        if not case["ragged"]:
            return torch.full((B,), case["fill"]), torch.full((B,), case["T"])
        start = torch.randint(0, case["fill"] + 1, (B,), generator=g)
        return start, torch.randint((case["T"] + 15) // 16, case["T"] + 1, (B,), generator=g)
    lens = torch.randint((case["Smax"] + 1) // 2, case["Smax"] + 1, (B,), generator=g)
    if case["op"] == "decode":
        if B == 16:  # ragged serving batch: down to a sixteenth of the longest
            lens = torch.randint((case["Smax"] + 15) // 16, case["Smax"] + 1, (B,), generator=g)
        if case["idle"]:
            lens[0] = 0
        return lens, torch.rand(B, generator=g) < case["p_full"]
    if B == 16:
        lens = torch.randint((case["Smax"] + 15) // 16, case["Smax"] + 1, (B,), generator=g)
    return lens, None


# --------------------------------------------------------------------------- inputs
def _pow2_at_least(a, qmax):
    """Smallest power of two ``s`` (at least 2^-126) with ``s * qmax >= a``; 0 where ``a`` is 0.  FP32, exact."""
    m, e = torch.frexp(a)
    mq, eq = math.frexp(qmax)
    e = torch.where(m <= mq, e - eq, e - eq + 1).clamp(min=-126)
    return torch.where(a > 0, ((e + 127) << 23).view(torch.float32), torch.zeros_like(a))  # 2^e from its bits: exact


def _round8(x, dtype):
    """FP32 -> 8-bit values, to nearest even, saturating; NaN stays NaN (e4m3) or becomes 0 (int8)."""
    if dtype == "e4m3":
        return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return torch.nan_to_num(x, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127).to(torch.int8)


def _rows(g, dev, shape, mean_scale):
    """BF16 rows as a model's projections give them: channels of unequal size, a few of them large."""
    chan = torch.exp(0.7 * torch.randn(shape[-1], generator=g, device=dev))
    chan[::37] *= 6.0
    return (torch.randn(shape, generator=g, device=dev) * (chan * mean_scale)).bfloat16()


def _cache(g, dev, case):
    """A cache whose every row holds values (those past a sequence's length are an earlier request's)."""
    B, Hkv, S, bs = case["B"], case["Hkv"], case["Smax"], case["block"]
    nb = (S + bs - 1) // bs
    out = []
    for mean_scale in (0.6, 0.25):
        x = torch.zeros((B, Hkv, nb * bs, D), dtype=torch.bfloat16, device=dev)
        x[:, :, :S] = _rows(g, dev, (B, Hkv, S, D), mean_scale)
        s = _pow2_at_least(x.reshape(B, Hkv, nb, bs * D).abs().amax(-1).float(), QMAX[case["dtype"]])
        x = _round8(x.reshape(B, Hkv, nb, bs, D) / s[..., None, None], case["dtype"])
        out += [x.reshape(B, Hkv, nb * bs, D)[:, :, :S].contiguous(), s]
    return out[0], out[2], out[1], out[3]


def _zero_cache(dev, dtype, B, Hkv, S, bs):
    nb = (S + bs - 1) // bs
    z8 = lambda: torch.zeros((B, Hkv, S, D), dtype=torch.int8, device=dev).view(DTYPE[dtype])  # noqa: E731
    return z8(), z8(), torch.zeros((B, Hkv, nb), device=dev), torch.zeros((B, Hkv, nb), device=dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    B, Hkv, bs = case["B"], case["Hkv"], case["block"]
    a, b = _lens(case)
    lens = a.to(dev, torch.int32)
    st = {"case": dict(case)}
    if case["op"] == "append":
        if case["fill"]:
            k, v, ks, vs = _cache(g, dev, case)
        else:
            k, v, ks, vs = _zero_cache(dev, case["dtype"], B, Hkv, case["Smax"], bs)
        st.update(k=k, v=v, ks=ks, vs=vs, start=lens, seq_lens=lens.clone(), new=b.to(dev, torch.int32),
                  k_new=_rows(g, dev, (B, case["T"], Hkv, D), 0.7), v_new=_rows(g, dev, (B, case["T"], Hkv, D), 0.3))
        return st
    k, v, ks, vs = _cache(g, dev, case)
    st.update(k=k, v=v, ks=ks, vs=vs, seq_lens=lens)
    if case["op"] == "decode":
        st["q"] = _rows(g, dev, (B, case["Hq"], D), 0.8)
        st["route"] = b.to(dev)
        if case["weights"]:
            st["w0"] = torch.rand((B, Hkv, case["Smax"]), generator=g, device=dev)
            st["w"] = st["w0"].clone()
        return st
    # accumulated weights: heavy-tailed, with exact ties (keys that no head looked at)
    w = torch.exp(3.0 * torch.randn((B, Hkv, case["Smax"]), generator=g, device=dev) - 6.0)
    st["w"] = torch.where(torch.rand(w.shape, generator=g, device=dev) < 0.2, torch.zeros_like(w), w)
    n = min(case["keep"], case["Smax"])
    st["out"] = _zero_cache(dev, case["dtype"], B, Hkv, n, bs) + (
        torch.zeros((B, Hkv, n), device=dev), torch.zeros((B,), dtype=torch.int32, device=dev))
    return st


# --------------------------------------------------------------------------- plain forms
def _expand(scale, bs, S):
    return scale.repeat_interleave(bs, dim=2)[:, :, :S]


def _plain_append_one(cache, scale, x, start, end, bs, dtype):
    """New rows ``x`` [B, T, Hkv, D] at [start, end) of one 8-bit tensor and its scales; both rewritten in place."""
    B, Hkv, S, _ = cache.shape
    nb = scale.shape[2]
    pos = torch.arange(nb * bs, device=cache.device)
    is_new = (pos >= start[:, None]) & (pos < end[:, None])                                  # [B, nb * bs]
    idx = (pos[None, :] - start[:, None]).clamp(0, x.shape[1] - 1).long()
    rows = x.gather(1, idx[:, :, None, None].expand(-1, -1, Hkv, D)).permute(0, 2, 1, 3).float()
    finite = is_new[:, None, :, None] & torch.isfinite(rows)
    amax = torch.where(finite, rows.abs(), torch.zeros_like(rows)).reshape(B, Hkv, nb, bs * D).amax(-1)
    need = _pow2_at_least(amax, QMAX[dtype])
    holds = (torch.arange(nb, device=cache.device) * bs)[None, :] < start[:, None]             # rows from before
    touched = is_new.reshape(B, nb, bs).any(-1)[:, None, :]
    old = torch.where(holds[:, None, :], _pow2_at_least(scale, 1.0), torch.zeros_like(scale))
    new = torch.maximum(old, need)
    new_row, old_row = _expand(new, bs, S)[..., None], _expand(scale, bs, S)[..., None]
    fresh = torch.where(new_row > 0, rows[:, :, :S] / new_row, torch.zeros_like(rows[:, :, :S]))
    again = torch.where(new_row != old_row, cache.float() * (old_row / new_row), cache.float())
    put = is_new[:, None, :S, None]
    redo = (_expand(touched.expand_as(scale), bs, S) & (pos[None, :S] < start[:, None])[:, None, :])[..., None]
    as_bytes = cache.view(torch.int8)
    as_bytes.copy_(torch.where(put, _round8(fresh, dtype).view(torch.int8),
                               torch.where(redo, _round8(again, dtype).view(torch.int8), as_bytes)))
    scale.copy_(torch.where(touched, new, scale))


def _plain_append(st, case):
    S = case["Smax"]
    start = st["start"].clamp(0, S)
    end = (start + st["new"].clamp(0, case["T"])).clamp(max=S)
    _plain_append_one(st["k"], st["ks"], st["k_new"], start, end, case["block"], case["dtype"])
    _plain_append_one(st["v"], st["vs"], st["v_new"], start, end, case["block"], case["dtype"])
    st["seq_lens"].copy_(end)


def _plain_decode(st, case):
    B, Hq, Hkv, S, bs = case["B"], case["Hq"], case["Hkv"], case["Smax"], case["block"]
    q = st["q"].float().reshape(B, Hkv, Hq // Hkv, D)
    L = st["seq_lens"].clamp(0, S)
    lo = torch.where(st["route"], torch.zeros_like(L), (L - case["window"]).clamp(min=0))
    pos = torch.arange(S, device=q.device)
    legal = ((pos >= lo[:, None]) & (pos < L[:, None]))[:, None, None, :]                      # [B, 1, 1, S]
    s = torch.matmul(q, st["k"].float().transpose(2, 3)) * (_expand(st["ks"], bs, S)[:, :, None, :] * (D ** -0.5))
    s = torch.where(legal, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    p = torch.where(legal, torch.exp(s - m), torch.zeros_like(s))
    total = p.sum(-1, keepdim=True)
    v = torch.where(legal.reshape(B, 1, S, 1), st["v"].float() * _expand(st["vs"], bs, S)[..., None], torch.zeros((), device=q.device))
    w = p / total
    out = torch.matmul(w, v).reshape(B, Hq, D).bfloat16()
    lse = ((m + torch.log(total)) * (1.0 / math.log(2.0))).reshape(B, Hq)
    lse = torch.where((L > 0)[:, None], lse, torch.full_like(lse, -math.inf))
    if case["weights"]:
        st["w"].copy_(st["w0"] + torch.where(legal[:, :, 0], w.sum(2), torch.zeros((), device=q.device)))
        return {"out": out, "lse": lse, "weights": st["w"]}
    return {"out": out, "lse": lse}


def _kept(weights, lens, keep, sink, recent):
    """``(slots [B, Hkv, n], counts [B])``: the kept rows of each head in order, -1 past the count."""
    B, Hkv, S = weights.shape
    n = min(keep, S)
    pos = torch.arange(S, device=weights.device)
    L = lens[:, None, None]
    rank = torch.where(torch.isnan(weights), torch.full_like(weights, -math.inf), weights)
    safe = (pos < sink) | (pos >= L - recent) | (L <= keep)
    rank = torch.where(safe, torch.full_like(rank, math.inf), rank)
    rank = torch.where(pos < L, rank, torch.full_like(rank, -math.inf))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :n]
    count = lens.clamp(max=n)[:, None, None]
    order = torch.where(torch.arange(n, device=order.device) < count, order, torch.full_like(order, S))
    slots = torch.sort(order, dim=-1).values
    return torch.where(slots < S, slots, torch.full_like(slots, -1)).to(torch.int32), lens.clamp(max=n)


def _plain_move(cache, scale, out, out_scale, slots, bs, dtype):
    B, Hkv, n = slots.shape
    nb = out_scale.shape[2]
    have = slots >= 0
    src = slots.clamp(min=0).long()
    s_src = torch.where(have, scale.gather(2, src // bs), torch.zeros((), device=scale.device))
    pad = torch.zeros((B, Hkv, nb * bs), device=scale.device)
    pad[:, :, :n] = s_src
    s_dst = pad.reshape(B, Hkv, nb, bs).amax(-1)
    row = _expand(s_dst, bs, n)
    ratio = torch.where(s_src == row, torch.ones_like(row), s_src / row)
    x = cache.float().gather(2, src[..., None].expand(-1, -1, -1, D)) * ratio[..., None]
    as_bytes = out.view(torch.int8)
    as_bytes.copy_(torch.where(have[..., None], _round8(x, dtype).view(torch.int8), as_bytes))
    some = torch.zeros((B, Hkv, nb * bs), dtype=torch.bool, device=scale.device)
    some[:, :, :n] = have
    out_scale.copy_(torch.where(some.reshape(B, Hkv, nb, bs).any(-1), s_dst, out_scale))


def _plain_evict(st, case):
    lens = st["seq_lens"].clamp(0, case["Smax"])
    slots, counts = _kept(st["w"], lens, case["keep"], case["sink"], case["recent"])
    k, v, ks, vs, w, n = st["out"]
    _plain_move(st["k"], st["ks"], k, ks, slots, case["block"], case["dtype"])
    _plain_move(st["v"], st["vs"], v, vs, slots, case["block"], case["dtype"])
    w.copy_(torch.where(slots >= 0, st["w"].gather(2, slots.clamp(min=0).long()), w))
    n.copy_(counts)
    return slots


# --------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        import switchattentionkernels_b200 as sw
        cache = sw.SwitchKVCache(k=state["k"], v=state["v"], k_scale=state["ks"], v_scale=state["vs"], seq_lens=state["seq_lens"],
                                 key_weights=state.get("w"), block_size=case["block"])
    if op == "append":
        if own:
            sw.switch_kv_cache_append(cache, state["k_new"], state["v_new"], new_lens=state["new"], start=state["start"])
        else:
            _plain_append(state, case)
        return {"k": state["k"], "v": state["v"], "k_scale": state["ks"], "v_scale": state["vs"], "seq_lens": state["seq_lens"]}
    if op == "decode":
        if not own:
            return _plain_decode(state, case)
        if case["weights"]:
            state["w"].copy_(state["w0"])  # a pass adds to the same weights each time
        out, lse = sw.switch_gqa_decode_cached(state["q"], cache, state["route"], window_size=case["window"])
        return {"out": out, "lse": lse, "weights": state["w"]} if case["weights"] else {"out": out, "lse": lse}
    k, v, ks, vs, w, n = state["out"]
    if own:
        kept = sw.SwitchKVCache(k=k, v=v, k_scale=ks, v_scale=vs, seq_lens=n, key_weights=w, block_size=case["block"])
        slots = sw.switch_kv_cache_evict(cache, keep=case["keep"], sink=case["sink"], recent=case["recent"], out=kept)
    else:
        slots = _plain_evict(state, case)
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "weights": w, "seq_lens": n, "slots": slots}


def work(case):
    a, b = _lens(case)
    Hkv, bs, S = case["Hkv"], case["block"], case["Smax"]
    if case["op"] == "append":
        rows = int((torch.minimum(a + b, torch.tensor(S)) - a).sum())
        # two bytes read and one written of each value of K and V, and a scale for each block
        return {"bytes": rows * Hkv * (2 * D * 3 + 8 / bs), "flops": rows * Hkv * 2 * D * 3}
    if case["op"] == "decode":
        keys = int(torch.where(b, a, a.clamp(max=case["window"])).sum())
        r = case["Hq"] // Hkv
        bytes_ = keys * Hkv * (2 * D + 8 / bs + (8 if case["weights"] else 0)) + case["B"] * case["Hq"] * (4 * D + 4)
        return {"bytes": bytes_, "flops": keys * Hkv * r * 4 * D}
    kept, seen = int(a.clamp(max=case["keep"]).sum()), int(a.sum())
    # every weight once; a kept row is read and written, with its weight, its slot and its share of the scales
    return {"bytes": seen * Hkv * 4 + kept * Hkv * (4 * D + 8 + 16 / bs), "flops": seen * Hkv * 4}


# --------------------------------------------------------------------------- definition in 64 bits
def _grid(y, dtype):
    """``y`` (64 bits) on the 8-bit grid: nearest, ties to even, saturating."""
    if dtype == "int8":
        return torch.nan_to_num(y, nan=0.0).clamp(-127, 127).round()
    e = torch.floor(torch.log2(y.abs().clamp(min=1e-300))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return ((y / step).round() * step).clamp(-448, 448)


def _ceil_pow2(a):
    e = torch.ceil(torch.log2(a.clamp(min=1e-300)))
    e = torch.where(torch.exp2(e - 1) >= a, e - 1, e)
    e = torch.where(torch.exp2(e) < a, e + 1, e)
    return torch.where(a > 0, torch.exp2(e.clamp(min=-126)), torch.zeros_like(a))


def _exact_append(st, case):
    dtype, bs, S = case["dtype"], case["block"], case["Smax"]
    res = {}
    for name, sname, new in (("k", "ks", "k_new"), ("v", "vs", "v_new")):
        val, scale = st[name].double(), st[sname].double()
        for b in range(case["B"]):
            s0 = int(st["start"][b])
            e0 = min(S, s0 + int(st["new"][b]))
            if e0 <= s0:
                continue
            first, last = s0 // bs, (e0 + bs - 1) // bs
            rows = torch.zeros((case["Hkv"], (last - first) * bs, D), dtype=torch.float64, device=val.device)
            rows[:, s0 - first * bs:e0 - first * bs] = st[new][b, :e0 - s0].double().transpose(0, 1)
            need = _ceil_pow2(rows.abs().reshape(case["Hkv"], last - first, bs * D).amax(-1) / QMAX[dtype])
            before = scale[b, :, first:last].clone()
            if s0 > first * bs:  # rows from before share the first block
                need[:, 0] = torch.maximum(need[:, 0], _ceil_pow2(before[:, 0]))
                old = val[b, :, first * bs:s0]
                val[b, :, first * bs:s0] = _grid(old * (before[:, 0] / need[:, 0].clamp(min=1e-300))[:, None, None], dtype)
            div = need.repeat_interleave(bs, dim=1)[..., None]
            y = torch.where(div > 0, rows / div.clamp(min=1e-300), torch.zeros_like(rows))
            val[b, :, s0:e0] = _grid(y, dtype)[:, s0 - first * bs:e0 - first * bs]
            scale[b, :, first:last] = need
        res[name], res[name + "_scale"] = val, scale
    lens = (st["start"] + st["new"]).clamp(max=S)
    return {**res, "seq_lens": lens}


def _exact_decode(st, case):
    B, Hq, Hkv, bs = case["B"], case["Hq"], case["Hkv"], case["block"]
    r = Hq // Hkv
    out = torch.full((B, Hq, D), math.nan, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device="cuda")
    w = st["w0"].double() if case["weights"] else None
    lens, route = st["seq_lens"].tolist(), st["route"].tolist()
    for b in range(B):
        lo, hi = (0 if route[b] else max(0, lens[b] - case["window"])), lens[b]
        if hi <= lo:
            continue
        at = torch.arange(lo, hi, device="cuda") // bs
        for g in range(Hkv):
            k = st["k"][b, g, lo:hi].double() * st["ks"][b, g].double()[at][:, None]
            v = st["v"][b, g, lo:hi].double() * st["vs"][b, g].double()[at][:, None]
            s = (st["q"][b, g * r:(g + 1) * r].double() @ k.T) / math.sqrt(D)
            z = torch.logsumexp(s, dim=1)
            p = torch.exp(s - z[:, None])
            out[b, g * r:(g + 1) * r] = p @ v
            lse[b, g * r:(g + 1) * r] = z / math.log(2.0)
            if w is not None:
                w[b, g, lo:hi] += p.sum(0)
    return {"out": out, "lse": lse, "weights": w} if case["weights"] else {"out": out, "lse": lse}


def _exact_evict(st, case):
    B, Hkv, bs, dtype = case["B"], case["Hkv"], case["block"], case["dtype"]
    n, keep, sink, recent = min(case["keep"], case["Smax"]), case["keep"], case["sink"], case["recent"]
    res = {x: y.double() for x, y in zip(("k", "v", "k_scale", "v_scale", "weights"), st["out"][:5])}
    slots = torch.full((B, Hkv, n), -1, dtype=torch.int32, device="cuda")
    lens = st["seq_lens"].tolist()
    for b in range(B):
        L = lens[b]
        for g in range(Hkv):
            mid = torch.arange(sink, L - recent, device="cuda")
            if L <= keep:
                rows = torch.arange(L, device="cuda")
            else:
                w = st["w"][b, g, sink:L - recent].double()
                take = torch.argsort(-w, stable=True)[:keep - sink - recent]
                rows = torch.cat([torch.arange(sink, device="cuda"), mid[take].sort().values, torch.arange(L - recent, L, device="cuda")])
            c = rows.numel()
            slots[b, g, :c] = rows.to(torch.int32)
            res["weights"][b, g, :c] = st["w"][b, g, rows].double()
            blk = torch.arange(c, device="cuda") // bs
            for name, sname in (("k", "ks"), ("v", "vs")):
                src = st[sname][b, g].double()[rows // bs]
                top = torch.zeros((c + bs - 1) // bs, dtype=torch.float64, device="cuda").scatter_reduce(0, blk, src, "amax")
                x = st[name][b, g, rows].double() * (src / top[blk].clamp(min=1e-300))[:, None]
                res[name][b, g, :c] = _grid(x, dtype)
                res[name + "_scale"][b, g, :top.numel()] = top
    return {**res, "seq_lens": st["seq_lens"].clamp(max=n), "slots": slots}


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "evict": _exact_evict}[case["op"]](st, case)
