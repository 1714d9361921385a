// What the append to a paged cache and the attention over it share: the step's metadata, and which request a query
// token or a work item belongs to.
#pragma once
#include "common.h"

// Element kinds of a cache.
enum SdcCache { SDC_CACHE_E4M3 = 0, SDC_CACHE_I8 = 1, SDC_CACHE_16 = 2 };

struct PagedStep {
  const int32_t* qsl;          // (R + 1): where each request's query tokens start, non-decreasing
  const int32_t* lens;         // (R): tokens of the request, this step's included
  const int32_t* bt;           // (R, W): the page of each run of N positions
  int64_t sbt, W, NB, T;
  int R, N;
};

// One request: its query tokens q0 .. q1 - 1 are its last positions, up to len - 1 (position of token t:
// t - q1 + len; a length shorter than the query leaves the first tokens without one).
struct Request {
  int r;
  int64_t q0, q1, len;
};

__device__ __forceinline__ Request sdc_request(const PagedStep& s, int r) {
  Request q;
  q.r = r;
  q.q0 = min(max((int64_t)s.qsl[r], (int64_t)0), s.T);
  if (r >= s.R) {
    q.q1 = s.T;
    q.len = 0;
    return q;
  }
  q.q1 = min(max((int64_t)s.qsl[r + 1], q.q0), s.T);
  q.len = max(s.lens[r], 0);
  return q;
}

// The last r in 0 .. R with qsl[r] / B + C r <= j, by the whole wave (all lanes active, j uniform), and -1 if there is
// none; R stands for the tokens past the last request (the padding of a captured step).  Work items of up to B tokens each
// are numbered so that no scan over the requests is needed: request r's items start at qsl[r] / B + C r.  With C = 1 that
// leaves room for items of B tokens from the request's first on, with C = 2 for items that begin at positions divisible by
// B.  Every lane reads two requests' starts and lengths at once, so that up to 127 requests cost one trip to memory.
// first: the number of the request's first item.
__device__ __forceinline__ int sdc_find_request(const PagedStep& s, int64_t j, int B, int C, Request& q, int64_t& first) {
  const int lane = threadIdx.x & 63;
  int n = 0, c = 0;
  int32_t start[2] = {0, 0}, len[2] = {0, 0};
  for (int b = 0; b <= s.R; b += 128) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = min(b + 64 * u + lane, s.R);
      start[u] = s.qsl[i];
      len[u] = s.R ? s.lens[min(i, s.R - 1)] : 0;
    }
    c = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = b + 64 * u + lane;
      c += __popcll(__ballot(i <= s.R && (int64_t)((uint32_t)start[u] / (uint32_t)B) + (int64_t)C * i <= j));
    }
    n += c;
    if (c < 128) break;
  }
  const int r = n - 1;
  if (r < 0) return r;
  if (c > 0 && c < 128) {
    // the request, and the one after it, are among those just read
    const int32_t at = __builtin_amdgcn_readlane(c > 64 ? start[1] : start[0], (c - 1) & 63);
    const int32_t to = __builtin_amdgcn_readlane(c > 63 ? start[1] : start[0], c & 63);
    q.r = r;
    q.q0 = min(max((int64_t)at, (int64_t)0), s.T);
    q.q1 = r >= s.R ? s.T : min(max((int64_t)to, q.q0), s.T);
    q.len = r >= s.R ? 0 : max(__builtin_amdgcn_readlane(c > 64 ? len[1] : len[0], (c - 1) & 63), 0);
    first = (int64_t)((uint32_t)at / (uint32_t)B) + (int64_t)C * r;
  } else {
    q = sdc_request(s, r);
    first = (int64_t)((uint32_t)s.qsl[r] / (uint32_t)B) + (int64_t)C * r;
  }
  return r;
}
