"""A paged KV cache held in 8 bits: the append that rotates, quantizes and writes a step's keys and values, and the
attention that reads the cache (no counterpart in the reference, whose checks read caches that others write).

A cache is what KVLedger and the attention check read, (pages, kv heads, slots, 2 head size) with the keys, then the
values, in the last dimension, here of float8_e4m3fn or int8 codes; scales is (pages, kv heads, 2) fp32: a key is its
code times scales[page, head, 0], a value its code times scales[page, head, 1].  A step is described as the serving
stack does it: qsl (query_start_loc), seq_lens (lengths with this step's tokens) and bt (block table), int32 on the
device.  Request r's query tokens qsl[r] .. qsl[r + 1] - 1 are the last positions of its seq_lens[r]; position p is in
page bt[r, p // slots], slot p % slots.  Tokens past qsl[-1] are a captured step's padding.

One launch appends (csrc/kv_append.hip) and one to three attend (csrc/kv_attend.hip), on the current stream, without
waiting and without a read of the device on the host, so both can be captured in a graph (attention after one call
with the same sizes, which makes its workspace).  There is no CPU implementation.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .rope import check_positions, check_turns

CACHE_E4M3, CACHE_I8, CACHE_16 = 0, 1, 2
_CODES = {torch.float8_e4m3fn: CACHE_E4M3, torch.int8: CACHE_I8}
MAX_HEAD = 256                                       # head size attention takes


def make_cache(pages: int, kv_heads: int, slots: int, head_size: int, dtype: torch.dtype = torch.float8_e4m3fn,
               device="cuda"):
    """(kv, scales) of an empty cache, zeroed; scales is None for a 16-bit dtype."""
    kv = torch.zeros(pages, kv_heads, slots, 2 * head_size, dtype=torch.uint8 if dtype in _CODES else dtype,
                     device=device)
    if dtype not in _CODES:
        _lib.dtype_code(dtype)
        return kv, None
    return kv.view(dtype), torch.zeros(pages, kv_heads, 2, device=device)


def _step(qsl, seq_lens, bt, dev):
    for t, n in ((qsl, "qsl"), (seq_lens, "seq_lens"), (bt, "bt")):
        if t.dtype not in (torch.int32, torch.int64) or t.device != dev:
            raise ValueError(f"{n} must be an integer tensor on the tensors' device")
    R = seq_lens.shape[0] if seq_lens.dim() == 1 else -1
    if R < 0 or qsl.shape != (R + 1,) or bt.dim() != 2 or bt.shape[0] < R:
        raise ValueError("a step is qsl (requests + 1), seq_lens (requests) and bt (at least requests, pages)")
    qsl, seq_lens, bt = (t if t.dtype == torch.int32 else t.to(torch.int32) for t in (qsl, seq_lens, bt))
    if bt.stride(1) != 1:
        bt = bt.contiguous()
    return qsl.contiguous(), seq_lens.contiguous(), bt


def _cache(kv, scales, dtype, head_size, dev):
    if kv.dim() != 4 or kv.shape[3] != 2 * head_size or kv.stride(3) != 1 or kv.shape[0] < 1 or kv.device != dev:
        raise ValueError("a cache is (pages, kv heads, slots, 2 * head size) with the last dimension contiguous")
    code = _CODES.get(kv.dtype, CACHE_16 if kv.dtype == dtype else None)
    if code is None:
        raise ValueError(f"a cache of {kv.dtype}: float8_e4m3fn, int8, or the keys' own 16 bits")
    if code != CACHE_16 and (scales is None or scales.shape != (kv.shape[0], kv.shape[1], 2) or
                             scales.dtype != torch.float32 or scales.device != dev or scales.stride(2) != 1):
        raise ValueError("scales must be (pages, kv heads, 2) fp32 with the last dimension contiguous")
    return code


def kv_append(key: torch.Tensor, value: torch.Tensor, kv: torch.Tensor, scales: Optional[torch.Tensor],
              qsl: torch.Tensor, seq_lens: torch.Tensor, bt: torch.Tensor, *, turns: Optional[torch.Tensor] = None,
              positions: Optional[torch.Tensor] = None, interleaved: bool = False, mscale: float = 1.0,
              query: Optional[torch.Tensor] = None, query_out: Optional[torch.Tensor] = None):
    """Write key and value (tokens, kv heads, head size; bf16 or fp16, any strides) to the step's slots of the cache.

    With `turns` (rope.frequencies) the keys, and the queries if given, are rotated first, by `positions` (one per token)
    or else by the tokens' positions in their requests.  Returns the rotated queries (query_out, which may be query
    itself, or a new tensor; the padding's rows are zeros), or None without queries.

    An 8-bit page's scale is the smallest power of two that holds the largest finite magnitude appended since its
    slot 0 was last written; where a call makes it grow, the codes already in the page are brought to it.  Writing slot 0
    starts a page anew.  e4m3 keeps infinities and NaN as NaN; int8 makes the page's scale NaN.  A 16-bit cache
    (of the keys' type, scales None) takes the rotated keys rounded once.  A token whose page lies outside the table or
    the cache is not written.  Requests of one step must not share the pages they write to."""
    _lib.require_gpu(key, value, kv, scales, qsl, seq_lens, bt, turns, positions, query, query_out)
    if key.dim() != 3 or value.shape != key.shape or value.dtype != key.dtype:
        raise ValueError("key and value must be (tokens, kv heads, head size) of one type")
    T, Hkv, D = key.shape
    dev, dt = key.device, _lib.dtype_code(key.dtype)
    if value.device != dev or kv.shape[1:2] != (Hkv,):
        raise ValueError("key, value and cache must have the same kv heads, on one device")
    code = _cache(kv, scales, key.dtype, D, dev)
    rot = 0 if turns is None else check_turns(turns, D, dev)
    qsl, seq_lens, bt = _step(qsl, seq_lens, bt, dev)
    if positions is not None:
        positions = check_positions(positions, T, dev)
    Hq = 0
    if query is None:
        if query_out is not None:
            raise ValueError("query_out without query")
    else:
        if query.dim() != 3 or query.shape[0] != T or query.shape[2] != D or query.dtype != key.dtype or \
                query.device != dev:
            raise ValueError("query must be (tokens, heads, head size) of the keys' type")
        Hq = query.shape[1]
        if query_out is None:
            query_out = torch.empty(query.shape, dtype=query.dtype, device=dev)
        elif query_out.shape != query.shape or query_out.dtype != query.dtype or query_out.device != dev:
            raise ValueError("query_out must have query's shape, type and device")
    q, qo = query, query_out
    with torch.cuda.device(dev):
        rc = _lib.lib().sdc_kv_append(
            dt, code, key.data_ptr(), *key.stride(), value.data_ptr(), *value.stride(), T, Hkv, D, kv.data_ptr(),
            *kv.stride()[:3], kv.shape[0], kv.shape[2], _lib.ptr(scales) if code != CACHE_16 else 0,
            *(scales.stride()[:2] if code != CACHE_16 else (0, 0)), qsl.data_ptr(), seq_lens.data_ptr(),
            seq_lens.shape[0], bt.data_ptr(), bt.stride(0), bt.shape[1], _lib.ptr(positions),
            0 if positions is None else positions.element_size(), _lib.ptr(turns), rot, int(interleaved),
            float(mscale), _lib.ptr(q), *(q.stride() if q is not None else (0, 0, 0)), _lib.ptr(qo),
            *(qo.stride() if q is not None else (0, 0, 0)), Hq, _lib.stream_of(key))
        _lib.check(rc, "sdc_kv_append")
    return query_out


def kv_attend(q: torch.Tensor, kv: torch.Tensor, scales: torch.Tensor, qsl: torch.Tensor, seq_lens: torch.Tensor,
              bt: torch.Tensor, *, scale: Optional[float] = None, window: int = 0, max_seq_len: Optional[int] = None,
              out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Causal attention of q (tokens, heads, head size; bf16 or fp16) over an 8-bit cache, kv heads shared by equal
    groups of query heads: out, or (out, lse) with lse (tokens, heads) fp32, the natural logarithm of the sum of
    exp(scale q . k).

    scale: head size ** -0.5 unless given.  window > 0: a query sees the last `window` keys, its own included.
    max_seq_len: a bound on seq_lens that the host knows (default: what the table holds); keys past it are not read.
    A query that sees no key, and the padding's, get zeros and -inf.  A page of a query's keys that lies outside the
    cache makes its output NaN."""
    _lib.require_gpu(q, kv, scales, qsl, seq_lens, bt, out)
    if q.dim() != 3:
        raise ValueError("q must be (tokens, heads, head size)")
    T, Hq, D = q.shape
    dev, dt = q.device, _lib.dtype_code(q.dtype)
    code = _cache(kv, scales, None, D, dev)
    Hkv, N = kv.shape[1], kv.shape[2]
    if Hkv < 1 or Hq < 1 or Hq % Hkv or D > MAX_HEAD:
        raise ValueError(f"{Hq} heads of {D} over {Hkv} kv heads: a multiple of them, and head sizes up to {MAX_HEAD}")
    if window < 0:
        raise ValueError("window must not be negative (0: none)")
    qsl, seq_lens, bt = _step(qsl, seq_lens, bt, dev)
    if out is None:
        out = torch.empty(T, Hq, D, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev:
        raise ValueError("out must have q's shape, type and device")
    lse = torch.empty(T, Hq, dtype=torch.float32, device=dev) if return_lse else None
    R, W = seq_lens.shape[0], bt.shape[1]
    most = W * N if max_seq_len is None else min(W * N, int(max_seq_len))
    if most < 0:
        raise ValueError("max_seq_len must not be negative")
    L = _lib.lib()
    with torch.cuda.device(dev):
        need = L.sdc_kv_attend_workspace(T, R, Hq, Hkv, D, N, most, int(window))
        ws = _lib.workspace(dev, need) if need else None
        rc = L.sdc_kv_attend(
            dt, code, q.data_ptr(), *q.stride(), out.data_ptr(), *out.stride(), _lib.ptr(lse), Hq, T, Hq, D,
            kv.data_ptr(), *kv.stride()[:3], kv.shape[0], Hkv, N, scales.data_ptr(), *scales.stride()[:2],
            qsl.data_ptr(), seq_lens.data_ptr(), R, bt.data_ptr(), bt.stride(0), W,
            D ** -0.5 if scale is None else float(scale), int(window), most, _lib.ptr(ws),
            0 if ws is None else ws.numel(), _lib.stream_of(q))
        _lib.check(rc, "sdc_kv_attend")
    return (out, lse) if return_lse else out
