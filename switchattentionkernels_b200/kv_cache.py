"""Block-scaled 8-bit KV cache: append, decode attention, eviction.

Not part of the reference (its kernels are prefill only).  ``switch_gqa_decode_forward``
reads an e4m3 cache with one scale per (sequence, KV head), which has to be known
before the first token is cached; here every block of 16 to 128 rows of a KV head has
its own scale, made as the rows arrive.  The three operators of a serving loop:

* ``switch_kv_cache_append``: BF16 K/V rows (a prompt, a chunk, one token) into the cache;
* ``switch_gqa_decode_cached``: the decode step over it, routed full or window per
  sequence as ``switch_gqa_decode_forward`` is, which can also accumulate the attention
  weight that every cached key received;
* ``switch_kv_cache_evict``: cuts every sequence to a budget of rows, keeping the first
  and last ones and, of the rest, those with the largest accumulated weight.

All three run on the current stream of the cache's device, read lengths on the device,
never synchronise and can be captured into a CUDA graph.
"""
from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache

import torch

from . import _core, _native
from ._core import LOG2E

HEAD_DIM = 128
BLOCK_SIZES = (16, 32, 64, 128)
_DTYPES = {torch.float8_e4m3fn: _native.KV_E4M3, torch.int8: _native.KV_INT8}


@dataclass
class SwitchKVCache:
    """A batch's cache.  The rows of one KV head lie together; value = byte * scale.

    Row ``s`` of (sequence ``b``, KV head ``g``) belongs to block ``s // block_size`` of it.
    Rows from ``seq_lens[b]`` on hold nothing.  Scales are FP32 and non-negative
    (``switch_kv_cache_append`` makes powers of two; the other operators take any).
    """
    k: torch.Tensor                           # float8_e4m3fn or int8 [B, Hkv, Smax, 128]
    v: torch.Tensor
    k_scale: torch.Tensor                     # float32 [B, Hkv, ceil(Smax / block_size)]
    v_scale: torch.Tensor
    seq_lens: torch.Tensor                    # int32 [B] cached rows of each sequence
    key_weights: torch.Tensor | None = None   # float32 [B, Hkv, Smax] accumulated attention weight
    block_size: int = 64


def make_switch_kv_cache(batch: int, max_len: int, kv_heads: int, *, device, dtype: torch.dtype = torch.float8_e4m3fn,
                         block_size: int = 64, track_weights: bool = False) -> SwitchKVCache:
    """An empty cache of ``max_len`` rows per sequence; ``track_weights`` adds ``key_weights``."""
    if batch <= 0 or max_len <= 0 or kv_heads <= 0:
        raise ValueError("batch, max_len and kv_heads must be positive")
    if dtype not in _DTYPES:
        raise TypeError("dtype must be float8_e4m3fn or int8")
    if block_size not in BLOCK_SIZES:
        raise ValueError("block_size must be 16, 32, 64 or 128")
    blocks = -(-max_len // block_size)
    rows = lambda: torch.zeros((batch, kv_heads, max_len, HEAD_DIM), dtype=torch.int8, device=device).view(dtype)  # noqa: E731
    scales = lambda: torch.zeros((batch, kv_heads, blocks), dtype=torch.float32, device=device)  # noqa: E731
    weights = torch.zeros((batch, kv_heads, max_len), dtype=torch.float32, device=device) if track_weights else None
    return SwitchKVCache(rows(), rows(), scales(), scales(), torch.zeros(batch, dtype=torch.int32, device=device),
                         weights, block_size)


def _bad(name: str, field: str, dtype, shape) -> ValueError:
    return ValueError(f"{name}.{field} must be a contiguous {dtype} {list(shape)} tensor on the device of {name}.k")


def _check_cache(cache: SwitchKVCache, name: str = "cache") -> tuple[int, int, int, torch.device]:
    """``(B, Hkv, Smax, device)`` of a well-formed cache."""
    if not isinstance(cache, SwitchKVCache):
        raise TypeError(f"{name} must be a SwitchKVCache")
    k, v = cache.k, cache.v
    if not isinstance(k, torch.Tensor) or k.dtype not in _DTYPES or not k.is_cuda:
        raise TypeError(f"{name}.k must be a device-resident float8_e4m3fn or int8 tensor")
    if not isinstance(v, torch.Tensor) or v.dtype != k.dtype or not v.is_cuda:
        raise TypeError(f"{name}.v must be a device-resident tensor of {name}.k's dtype")
    shape = k.shape
    if len(shape) != 4 or v.shape != shape:
        raise ValueError(f"{name}.k and {name}.v must be [B, Hkv, Smax, 128]")
    B, Hkv, Smax, D = shape
    if D != HEAD_DIM:
        raise ValueError("head_dim must be 128")
    if B == 0 or Hkv == 0 or Smax == 0:
        raise ValueError(f"{name} is empty")
    if cache.block_size not in BLOCK_SIZES:
        raise ValueError("block_size must be 16, 32, 64 or 128")
    dev = k.device
    if not k.is_contiguous():
        raise _bad(name, "k", k.dtype, shape)
    if not v.is_contiguous() or v.device != dev:
        raise _bad(name, "v", k.dtype, shape)
    scales = (B, Hkv, -(-Smax // cache.block_size))
    for field, t in (("k_scale", cache.k_scale), ("v_scale", cache.v_scale)):
        if (not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.shape != scales or t.device != dev
                or not t.is_contiguous()):
            raise _bad(name, field, torch.float32, scales)
    t = cache.seq_lens
    if (not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.shape != (B,) or t.device != dev
            or not t.is_contiguous()):
        raise _bad(name, "seq_lens", torch.int32, (B,))
    t = cache.key_weights
    if t is not None and (not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.shape != (B, Hkv, Smax)
                          or t.device != dev or not t.is_contiguous()):
        raise _bad(name, "key_weights", torch.float32, (B, Hkv, Smax))
    return B, Hkv, Smax, dev


def _check_rows(t, name: str, shape: tuple, dev) -> tuple:
    """The strides of BF16 rows of ``shape``."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16 or not t.is_cuda:
        raise TypeError(f"{name} must be a device-resident bfloat16 tensor")
    if t.device != dev:
        raise ValueError(f"{name} must be on the device of the cache")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {list(shape)}")
    # a slice of a fused projection is fine: only the 128 values of a row have to lie together
    st = t.stride()
    bits = t.data_ptr() >> 1
    for s in st[:-1]:
        bits |= s
    if st[-1] != 1 or bits & 7:
        st = tuple(s if n > 1 else 0 for s, n in zip(st[:-1], shape)) + st[-1:]  # a single entry's stride is never used
        if st[-1] != 1 or t.data_ptr() % 16 or any(s % 8 for s in st[:-1]):
            raise ValueError(f"{name} needs contiguous, 16-byte aligned rows (other strides multiples of 8 elements)")
    return st


def _check_lens(t, name: str, B: int, dev) -> int:
    if (not isinstance(t, torch.Tensor) or t.device != dev or t.dtype != torch.int32 or t.shape != (B,)
            or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous int32 [B] tensor on the device of the cache")
    return t.data_ptr()


def _call(what: str, fn, dev: torch.device, *args) -> None:
    """``fn(*args, stream)`` with ``dev`` current and its current stream.

    The raw handles are read without the device guard and the Stream object of
    ``torch.cuda``: together some 3 us of a call that takes 14 to 25 on the host.
    """
    index = dev.index
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _native.check(rc, what)


@lru_cache(maxsize=256)
def _decode_workspace_bytes(B: int, Smax: int, Hq: int, Hkv: int, weights: bool, device_index: int) -> int:
    """The decode step's workspace on a device: a function of the shapes."""
    lib = _native.load()
    with torch.cuda.device(device_index):
        nbytes = int(lib.swa_kv_decode_workspace_bytes(B, Smax, Hq, Hkv, int(weights)))
    if nbytes <= 0:
        raise RuntimeError("decode workspace size query failed: " + lib.swa_last_error_string().decode(errors="replace"))
    return nbytes


def switch_kv_cache_append(cache: SwitchKVCache, k_new: torch.Tensor, v_new: torch.Tensor, *,
                           new_lens: torch.Tensor | None = None, start: torch.Tensor | None = None) -> None:
    """Write new K/V rows behind each sequence's cached ones; ``cache.seq_lens`` is advanced.

    ``k_new`` / ``v_new``: BF16 ``[B, T, Hkv, 128]``, or ``[B, Hkv, 128]`` for one token per
    sequence; views with contiguous rows (slices of a fused projection) are taken as
    they are.  ``new_lens``: int32 ``[B]``, the rows of a padded batch that count (default:
    all ``T``).  ``start``: int32 ``[B]``, the row at which each sequence's new rows begin
    (default ``cache.seq_lens``; earlier: the rows from there on are dropped and replaced, e.g.
    after rejected draft tokens, also by no row at all; later: the rows between count as
    cached and hold whatever lies there).  Neither may overlap ``cache.seq_lens`` unless it is that tensor.
    Rows that do not fit (``>= Smax``) are dropped.

    A block's scale is the smallest power of two that its rows need, and only grows:
    when it does, the block's earlier rows are rounded again.  Rounding is to nearest
    even; infinities saturate and do not count for the scale (0 in a block without another
    value but zeros), NaN stays NaN in an e4m3 cache and becomes 0 in an int8 one.
    Appended rows start with ``key_weights`` 0.
    """
    B, Hkv, Smax, dev = _check_cache(cache)
    if not isinstance(k_new, torch.Tensor) or k_new.ndim not in (3, 4):
        raise ValueError("k_new must have shape [B, T, Hkv, 128] or [B, Hkv, 128]")
    token = k_new.ndim == 3
    T = 1 if token else int(k_new.shape[1])
    shape = (B, Hkv, HEAD_DIM) if token else (B, T, Hkv, HEAD_DIM)
    ks, vs = _check_rows(k_new, "k_new", shape, dev), _check_rows(v_new, "v_new", shape, dev)
    lens_ptr = None if new_lens is None else _check_lens(new_lens, "new_lens", B, dev)
    seq_ptr = cache.seq_lens.data_ptr()
    start_ptr = seq_ptr if start is None else _check_lens(start, "start", B, dev)
    if T == 0:  # no new row: the sequences end at `start`
        if start is not None:
            torch.clamp(start, 0, Smax, out=cache.seq_lens)
        return
    T = min(T, Smax)  # rows past Smax are dropped; an expanded view may have more than an int counts
    weights = cache.key_weights
    _call("switch_kv_cache_append", _native.load().swa_kv_append, dev, k_new.data_ptr(), v_new.data_ptr(),
          ks[0], 0 if token else ks[1], ks[-2], vs[0], 0 if token else vs[1], vs[-2], start_ptr, lens_ptr,
          cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(),
          None if weights is None else weights.data_ptr(), seq_ptr, B, T, Hkv, Smax, HEAD_DIM, cache.block_size,
          _DTYPES[cache.k.dtype])


def switch_gqa_decode_cached(q: torch.Tensor, cache: SwitchKVCache, route_full: torch.Tensor, *,
                             window_size: int = 1024, sm_scale: float | None = None, accumulate: bool = True,
                             status_out: torch.Tensor | None = None):
    """Attention of each sequence's new token over its cached rows (the new one's included).

    ``q``: BF16 ``[B, Hq, 128]`` or ``[B, 1, Hq, 128]`` (views with contiguous rows are
    taken as they are), ``Hq`` a multiple of the cache's KV heads; ``route_full``: bool
    ``[B]``, True = all cached rows, False = the last ``window_size`` of them.  Returns
    ``(O, LSE)``: BF16 ``[B, Hq, 128]`` and FP32 ``[B, Hq]`` (log2 units), shaped like ``q``;
    a sequence without rows gets O = NaN, LSE = -inf.  A query with an infinity or NaN
    gets NaN in both.

    The products take the cached bytes as they are.  Attention weights enter the sum over
    V rounded to 11 bits (e4m3 cache, as FP16) or in steps of 2^-19 or less of the largest
    contribution (int8), query entries to within 2^-23.9 of their head's largest one;
    scores, their maxima and sums, LSE and ``key_weights`` are FP32.

    With ``accumulate`` and a cache that has ``key_weights``, the softmax weight of every
    row that was attended to, summed over the query heads of its KV head, is added to
    them.  ``status_out``: as in ``switch_gqa_decode_forward``; with a non-zero word
    ``key_weights`` is unchanged.
    """
    B, Hkv, Smax, dev = _check_cache(cache)
    squeeze = isinstance(q, torch.Tensor) and q.ndim == 4
    if squeeze:
        if q.shape[1] != 1:
            raise ValueError("decode takes one query token per sequence")
        q = q[:, 0]
    if not isinstance(q, torch.Tensor) or q.ndim != 3:
        raise ValueError("q must have shape [B, Hq, 128] or [B, 1, Hq, 128]")
    Hq = int(q.shape[1])
    st = _check_rows(q, "q", (B, Hq, HEAD_DIM), dev)
    if Hq == 0 or Hq % Hkv != 0:
        raise ValueError("query heads must be divisible by KV heads")
    if window_size <= 0:
        raise ValueError("window_size must be positive")
    if (not isinstance(route_full, torch.Tensor) or route_full.device != dev or route_full.dtype != torch.bool
            or route_full.shape != (B,)):
        raise ValueError("route_full must be a bool [B] tensor on the device of the cache")
    scale = (sm_scale if sm_scale is not None else (1.0 / HEAD_DIM) ** 0.5) * LOG2E
    if not scale > 0:
        raise ValueError("sm_scale must be positive")
    _core._check_status_out(status_out, dev)
    weights = cache.key_weights if accumulate else None
    out = q.new_empty((B, Hq, HEAD_DIM))
    lse = cache.k_scale.new_empty((B, Hq))
    nbytes = _decode_workspace_bytes(B, Smax, Hq, Hkv, weights is not None, dev.index)
    ws = cache.seq_lens.new_empty((nbytes + 15) // 16 * 4)
    route = route_full if route_full.is_contiguous() else route_full.contiguous()
    _call("switch_gqa_decode_cached", _native.load().swa_kv_decode, dev, q.data_ptr(), st[0], st[1], cache.k.data_ptr(),
          cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), cache.seq_lens.data_ptr(),
          route.data_ptr(), out.data_ptr(), lse.data_ptr(), None if weights is None else weights.data_ptr(), B, Smax,
          Hq, Hkv, HEAD_DIM, cache.block_size, min(int(window_size), Smax), float(scale), _DTYPES[cache.k.dtype],
          ws.data_ptr(), nbytes)
    if status_out is not None or _core.CHECK_DEVICE_STATUS:
        _core.publish_status(ws[0:1], status_out)
    if squeeze:
        return out.unsqueeze(1), lse.unsqueeze(1)
    return out, lse


def switch_kv_cache_evict(cache: SwitchKVCache, *, keep: int, sink: int = 0, recent: int = 0,
                          out: SwitchKVCache | None = None) -> torch.Tensor:
    """Cut every sequence longer than ``keep`` rows to ``keep`` of them; needs ``key_weights``.

    Each KV head keeps its first ``sink`` rows, its last ``recent`` rows and, of those
    between, the ones with the largest ``key_weights`` (ties: the lowest row; NaN: last),
    moved together in their order with their weights.  Shorter sequences keep all rows.
    A sequence's sliding window keeps its meaning while ``recent >= window_size``: window
    rows are the last cached ones.  A block's new scale is the largest of its rows'
    scales; rows of a smaller one are rounded again.

    In place by default.  ``out``: another cache of the same batch, heads, dtype and block
    size, sharing no memory with ``cache`` and with at least ``min(keep, Smax)`` rows,
    that takes the result; ``cache`` is then left as it is.  Returns int32
    ``[B, Hkv, min(keep, Smax)]``: the former row of each kept row, -1 past the last one.
    """
    B, Hkv, Smax, dev = _check_cache(cache)
    if cache.key_weights is None:
        raise ValueError("eviction needs a cache with key_weights")
    keep, sink, recent = int(keep), int(sink), int(recent)
    if keep <= 0 or sink < 0 or recent < 0 or sink + recent > keep:
        raise ValueError("keep must be positive and at least sink + recent, both non-negative")
    if keep >= Smax:  # no sequence is longer
        keep, sink, recent = Smax, 0, 0
    src = _pointers(cache)
    dst, So = src, Smax  # in place
    if out is not None and out is not cache:
        Bo, Ho, So, dev_out = _check_cache(out, "out")
        if (Bo, Ho) != (B, Hkv) or out.k.dtype != cache.k.dtype or out.block_size != cache.block_size:
            raise ValueError("out must have the batch, heads, dtype and block size of the cache")
        if dev_out != dev:
            raise ValueError("out must be on the device of the cache")
        if out.key_weights is None:
            raise ValueError("out must have key_weights")
        if So < keep:
            raise ValueError("out holds fewer rows than are kept")
        dst = _pointers(out)
        ends = [0, 0]  # of the cache's and of out's memory up to here, by address
        for first, end, owner in sorted(_spans(src, B, Hkv, Smax, cache.block_size, 0) +
                                        _spans(dst, B, Hkv, So, cache.block_size, 1)):
            if first < ends[1 - owner]:
                raise ValueError("out must not share memory with the cache")
            ends[owner] = max(ends[owner], end)
    slots = cache.seq_lens.new_empty((B, Hkv, keep))
    _call("switch_kv_cache_evict", _native.load().swa_kv_evict, dev, *src, *dst, slots.data_ptr(), B, Hkv, Smax, So,
          HEAD_DIM, cache.block_size, keep, sink, recent, _DTYPES[cache.k.dtype])
    return slots


def _pointers(c: SwitchKVCache) -> tuple:
    return (c.k.data_ptr(), c.v.data_ptr(), c.k_scale.data_ptr(), c.v_scale.data_ptr(), c.key_weights.data_ptr(),
            c.seq_lens.data_ptr())


def _spans(ptrs: tuple, B: int, Hkv: int, Smax: int, block: int, owner: int) -> list:
    """``(first byte, end, owner)`` of a cache's tensors."""
    k, v, ks, vs, w, n = ptrs
    weights = 4 * B * Hkv * Smax
    rows, scales = HEAD_DIM // 4 * weights, 4 * B * Hkv * -(-Smax // block)
    return [(k, k + rows, owner), (v, v + rows, owner), (ks, ks + scales, owner), (vs, vs + scales, owner),
            (w, w + weights, owner), (n, n + 4 * B, owner)]
