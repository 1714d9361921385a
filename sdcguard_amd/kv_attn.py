"""A paged KV cache held in 8 bits: the append that rotates, quantizes and writes a step's keys and values, and the
attention that reads the cache (no counterpart in the reference, whose checks read caches that others write).

A cache has the layout of a KVLedger's and the attention check's, (pages, kv heads, slots, 2 head size) with the keys, then
the values, in the last dimension, here of float8_e4m3fn or int8 codes (the ledger takes these, and the scales; the check
recomputes from 16-bit caches of the queries' type, which kv_append writes too); scales is (pages, kv heads, 2) fp32: a key is its
code times scales[page, head, 0], a value its code times scales[page, head, 1].  A step is described as the serving
stack does it: qsl (query_start_loc), seq_lens (lengths with this step's tokens) and bt (block table), int32 on the
device.  Request r's query tokens qsl[r] .. qsl[r + 1] - 1 are the last positions of its seq_lens[r]; position p is in
page bt[r, p // slots], slot p % slots.  Tokens past qsl[-1] are a captured step's padding.

One launch appends (csrc/kv_append.hip) and one to three attend (csrc/kv_attend.hip), on the current stream, without
waiting and without a read of the device on the host, so both can be captured in a graph.  Arguments are checked in
csrc/bind.cpp.  Neither has a gradient: with grad mode on, tensors that require one are refused.  There is no CPU
implementation.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

_CODES = (torch.float8_e4m3fn, torch.int8)


def make_cache(pages: int, kv_heads: int, slots: int, head_size: int, dtype: torch.dtype = torch.float8_e4m3fn,
               device="cuda"):
    """(kv, scales) of an empty cache, zeroed; scales is None for a 16-bit dtype."""
    kv = torch.zeros(pages, kv_heads, slots, 2 * head_size, dtype=torch.uint8 if dtype in _CODES else dtype,
                     device=device)
    if dtype not in _CODES:
        _lib.dtype_code(dtype)
        return kv, None
    return kv.view(dtype), torch.zeros(pages, kv_heads, 2, device=device)


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
    return _lib.bound().append(key, value, kv, scales, qsl, seq_lens, bt, turns, positions, interleaved, mscale, query,
                               query_out)


def kv_attend(q: torch.Tensor, kv: torch.Tensor, scales: torch.Tensor, qsl: torch.Tensor, seq_lens: torch.Tensor,
              bt: torch.Tensor, *, scale: Optional[float] = None, window: int = 0, max_seq_len: Optional[int] = None,
              out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Causal attention of q (tokens, heads, head size; bf16 or fp16) over an 8-bit cache, kv heads shared by equal
    groups of query heads: out, or (out, lse) with lse (tokens, heads) fp32, the natural logarithm of the sum of
    exp(scale q . k).

    scale: head size ** -0.5 unless given.  window > 0: a query sees the last `window` keys, its own included.
    max_seq_len: a bound on seq_lens that the host knows (default: what the table holds); keys past it are not read, and
    the call plans its workspace and kernels for it, so a bound near the lengths is faster.
    A query that sees no key, and the padding's, get zeros and -inf.  A page of a query's keys that lies outside the
    cache makes its output NaN."""
    return _lib.bound().attend(q, kv, scales, qsl, seq_lens, bt, scale, window, max_seq_len, out, return_lse)
