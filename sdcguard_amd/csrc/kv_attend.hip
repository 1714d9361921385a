// Attention of a step's queries over a paged cache of 8-bit codes, a scale for the keys and one for the values of each
// (page, kv head): o = sum_j p_j v_j / sum_j p_j over the keys j a query sees (its own position and those before it, the
// last `window` of them), p_j = exp(s_j - max s), s_j = scale q . k_j, k_j = ks[page] kcode_j, v_j = vs[page] vcode_j;
// lse = max s + log sum p.  A query that sees no key gets zeros and lse = -inf; a key in a page outside the cache
// counts as NaN.
//
// kv_attend_rows: tiles of 16 query rows, for decode steps and small chunks (HBM bound, or by latency).  kv_attend_tiles:
// tiles of 256 query rows, for chunks of a prompt (bound by the matrix cores and the softmax between them).  kv_attend_any:
// any head size and alignment, a row a wave; parts whose value scales are far from 1 are left to the same (plain_row).
// A part of a tile's keys is one workgroup's; kv_attend_join joins the parts in their order.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.h"
#include "paged.h"
#include "profile.h"
#include "rope.h"

namespace {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr float NEG_INF = -__builtin_inff();

struct AttendArgs {
  PagedStep st;
  const uint16_t* q; uint16_t* o; float* lse;
  int64_t sqt, sqh, sqd, sot, soh, sod, slt;   // lse (T, Hq): token stride slt, heads contiguous
  const uint8_t* kv;
  int64_t cb, ch, cn;                          // page, head and slot strides of the cache, in bytes
  const float* scales;
  int64_t sb, sh;
  float scale;                                 // on q . k, times log2(e)
  int64_t window, maxlen;                      // keys a query sees at most; keys of a sequence that are read
  int Hq, Hkv, G, D, fp16;
};

// The work of a tiled kernel: tiles of TB query tokens x GB heads of one kv head (at most `rows` query rows), whose keys
// are cut into at most S parts, one part a workgroup.  A call with chunks runs both kernels: requests of up to `few`
// tokens go to kv_attend_rows, the others, and the padding, to kv_attend_tiles.
// part: (tile, part) records: `rows` heads (the exponent of the row's sums of values, that of its sum of probabilities, which is
// the maximum, and that sum, 0), then rows x D sums.
struct Split {
  int64_t tiles;
  int TB, GB, NHB, S, rows;
  int C;                                       // keys of a part at least (a multiple of 128)
  int slots;                                   // tiles numbered by request, so many each (0: by their tokens)
  int few;                                     // requests of up to so many tokens are left out (0: none)
  uint32_t div;                                // ceil(2^32 / N), to divide by N
  float* part;
};

template <int CT>
__device__ __forceinline__ float value_of(uint32_t c) {
  if constexpr (CT == SDC_CACHE_E4M3) return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
  else return (float)(int8_t)c;
}

constexpr int ANY_D = 256;                     // largest head size

// A value scale's exponent field: v < 2^(field - 126).  0 of zero, infinity and NaN.
__device__ __forceinline__ uint32_t scale_field(float v) {
  const uint32_t e = (__float_as_uint(v) >> 23) & 0xFFu;
  return e == 0xFFu ? 0u : max(e, (uint32_t)(v != 0.f));
}

// A query into `row` (of the wave), after a power of two that brings its largest element under 1, so that no product with codes
// passes fp32; and the factor on its scores.
__device__ __forceinline__ float plain_query(const AttendArgs& a, int64_t t, int h, float* row) {
  const uint16_t* q = a.q + t * a.sqt + h * a.sqh;
  float x[ANY_D / 64], amax = 0.f;
#pragma unroll
  for (int i = 0; i < ANY_D / 64; ++i) {
    const int d = (threadIdx.x & 63) + 64 * i;
    x[i] = d >= a.D ? 0.f : a.fp16 ? half_to_f32<SDC_FP16>(q[d * a.sqd]) : half_to_f32<SDC_BF16>(q[d * a.sqd]);
    if (fabsf(x[i]) < __builtin_inff()) amax = fmaxf(amax, fabsf(x[i]));
  }
  int e = 0;
  (void)frexpf(wave_max_f32_dpp(amax), &e);
  sdc_wave_lds_fence();                        // (another row's may be read still)
#pragma unroll
  for (int i = 0; i < ANY_D / 64; ++i) row[(threadIdx.x & 63) + 64 * i] = ldexpf(x[i], -e);
  sdc_wave_lds_fence();
  return ldexpf(a.scale, e);
}
// One query row over keys lo .. hi of request r, by a wave, all in fp32: a lane has a key's score, then elements lane + 64 e of
// the output, in units of 2^u where values would pass fp32 in their sum.
struct PlainRow {
  float m, l, o[ANY_D / 64];
  int u;
};
template <int CT>
__device__ __forceinline__ PlainRow plain_row(const AttendArgs& a, const float* q, float scale, int r, int hk, int64_t lo, int64_t hi) {
  const int lane = threadIdx.x & 63, D = a.D;
  PlainRow s{NEG_INF, 0.f, {}, 0};
  for (int64_t b = lo; b < hi; b += 64) {
    const int64_t j = b + lane;
    float x = NEG_INF, vs = 0.f;
    int64_t row = 0;
    if (j < hi) {
      const int64_t wp = j / a.st.N, page = a.st.bt[r * a.st.sbt + wp];
      const bool in = page >= 0 && page < a.st.NB;
      row = (in ? page : 0) * a.cb + hk * a.ch + (j - wp * a.st.N) * a.cn;
      const float* sc = a.scales + (in ? page : 0) * a.sb + hk * a.sh;
      const float ks = in ? sc[0] : __builtin_nanf("");
      vs = in ? sc[1] : __builtin_nanf("");
      float dot = 0.f;
      for (int d = 0; d < D; ++d) dot = fmaf(q[d], value_of<CT>(a.kv[row + d]), dot);
      x = dot * (ks * scale);
    }
    const float mn = fmaxf(s.m, wave_max_f32_dpp(x)), ms = mn == NEG_INF ? 0.f : mn;
    const int u = max(s.u, (int)wave_max_u32_dpp(scale_field(vs)) - 126 - 80);
    const float p = j < hi ? exp2f(x - ms) : 0.f, f = exp2f(s.m - ms);
    s.l = s.l * f + wave_sum_f32_dpp(p);
#pragma unroll
    for (int e = 0; e < ANY_D / 64; ++e) s.o[e] = ldexpf(s.o[e] * f, s.u - u);
    const float pv = p * ldexpf(vs, -u);
    for (int i = 0; i < 64 && b + i < hi; ++i) {
      const float pi = __shfl(pv, i);
      const int64_t ri = (int64_t)__shfl((long long)row, i) + D;
#pragma unroll
      for (int e = 0; e < ANY_D / 64; ++e)
        if (lane + 64 * e < D) s.o[e] = fmaf(pi, value_of<CT>(a.kv[ri + lane + 64 * e]), s.o[e]);
    }
    s.m = mn;
    s.u = u;
  }
  return s;
}
// Its results; `any`: it has keys.
__device__ __forceinline__ void write_plain(const AttendArgs& a, int64_t t, int h, const PlainRow& s, bool any) {
  const int lane = threadIdx.x & 63;
  // (a query whose keys all score -inf: 0 / 0)
  const float inv = any ? 1.f / s.l : 0.f;
#pragma unroll
  for (int e = 0; e < ANY_D / 64; ++e) {
    const int d = lane + 64 * e;
    const float x = any ? ldexpf(s.o[e] * inv, s.u) : 0.f;
    if (d < a.D) a.o[t * a.sot + h * a.soh + d * a.sod] = a.fp16 ? sdc_to_half<SDC_FP16>(x) : sdc_to_half<SDC_BF16>(x);
  }
  if (a.lse && lane == 0) a.lse[t * a.slt + h] = any ? (s.m + log2f(s.l)) * LN2 : NEG_INF;
}

template <int CT>
__global__ __launch_bounds__(256) void kv_attend_any(AttendArgs a) {
  __shared__ float qs[4][ANY_D];
  const int w = threadIdx.x >> 6;
  const int64_t id = (int64_t)blockIdx.x * 4 + w;
  if (id >= a.st.T * a.Hq) return;
  const int64_t t = id / a.Hq;
  const int h = (int)(id - t * a.Hq);
  const float scale = plain_query(a, t, h, qs[w]);
  Request rq;
  int64_t first;
  const int r = sdc_find_request(a.st, t, 1, 0, rq, first);
  int64_t lo = 0, hi = 0;
  if (r >= 0 && r < a.st.R) {
    hi = min(t - rq.q1 + rq.len + 1, a.maxlen);
    lo = max(t - rq.q1 + rq.len + 1 - a.window, (int64_t)0);
  }
  write_plain(a, t, h, plain_row<CT>(a, qs[w], scale, r, h / a.G, lo, hi), hi > lo);
}

// ------------------------------------------------------------------------------------------------ few query rows
constexpr int ROWS = 16;                       // query rows (tokens x heads of one kv head) of a tile
constexpr int MAXP = 1024;                     // page-table entries a workgroup holds
constexpr float M0 = -3.0e38f;                 // a maximum before the first key
constexpr float BIAS = 13.f;                   // the largest probability is 2^BIAS .. 2^(BIAS + 2): fp16 has room under it
constexpr int HEAD = 4;                        // numbers of a row at the start of a part's record

// Four codes as two pairs of fp16, exactly.
template <int CT>
__device__ __forceinline__ u32x2 widen(uint32_t x) {
  u32x2 o;
  if constexpr (CT == SDC_CACHE_E4M3) {
    o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, false));
    o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, true));
  } else {
    // bytes u = code + 128 as the mantissas of 1024 + u, less 1152
    x ^= 0x80808080u;
    const f16x2 bias = {(_Float16)-1152.f, (_Float16)-1152.f};
    o.x = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) + bias);
    o.y = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) + bias);
  }
  return o;
}
template <int CT>
__device__ __forceinline__ f16x8 widen8(uint32_t a, uint32_t b) {
  const u32x2 x = widen<CT>(a), y = widen<CT>(b);
  return __builtin_bit_cast(f16x8, u32x4{x.x, x.y, y.x, y.y});
}

// 4 x 4 bytes transposed: y[b] = byte b of x[0], x[1], x[2], x[3]
__device__ __forceinline__ void transpose4(const uint32_t* x, uint32_t* y) {
  const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), b = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);
  const uint32_t c = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u), d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
  y[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  y[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  y[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  y[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// which of the four codes are NaN (0x7F or 0xFF), as 0x80 bits
__device__ __forceinline__ uint32_t nan_codes(uint32_t x) { return ((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

// The largest field of a part's value scales, and of 255 - field without the smallest scale, which pages of zeros have.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2 larger(u16x2 x, uint32_t y) { return __builtin_elementwise_max(x, __builtin_bit_cast(u16x2, y)); }
__device__ __forceinline__ u16x2 scale_ends(u16x2 x, float v) {
  const uint32_t f = scale_field(v);
  return larger(x, f | (f > 1 ? 255u - f : 0u) << 16);
}
__device__ __forceinline__ u16x2 wave_larger(u16x2 v) {
  v = larger(v, dpp_u32<0xB1>(__builtin_bit_cast(uint32_t, v)));
  v = larger(v, dpp_u32<0x4E>(__builtin_bit_cast(uint32_t, v)));
  v = larger(v, dpp_u32<0x141>(__builtin_bit_cast(uint32_t, v)));
  v = larger(v, dpp_u32<0x140>(__builtin_bit_cast(uint32_t, v)));
  const int x = __builtin_bit_cast(int, v);
#pragma unroll
  for (int l = 0; l < 64; l += 16) v = larger(v, (uint32_t)__builtin_amdgcn_readlane(x, l));
  return v;
}
// How a page's value scale enters the products: as 2^b times a factor in [1/2, 1).  2^(x + b), x a score, is what a probability's
// product with its scale is rounded in, so it is that exponent whose maximum is followed; the sum of probabilities takes 2^-b of
// it.  With b from LOW_B to HIGH_B neither loses keys to fp32's ends.  A part with scales outside that (values of 1e15 and more,
// or under 4e-16) takes them all relative to a 2^ve; zero, and the scale 2^-126 of a page of zeros, count as LOW_B then too.
constexpr int LOW_B = -60, HIGH_B = 40;
__device__ __forceinline__ int scale_exponent(float v, int ve) {
  const int f = (int)scale_field(v);
  return f ? max(f - 126 - ve, LOW_B) : v == 0.f ? LOW_B : 0;
}
__device__ __forceinline__ float scale_factor(float v, int b) { return ldexpf(v, -b); }
// From the ends of a part's scales: whether no ve is right (values as 1e15 beside 1e-15), and it is left to plain_row; and ve, 0
// but for such parts as above.
__device__ __forceinline__ bool scales_apart(u16x2 ends) {
  const int top = __builtin_amdgcn_readfirstlane(ends.x), low = __builtin_amdgcn_readfirstlane(ends.y);
  return low && top - (255 - low) > HIGH_B - LOW_B;
}
__device__ __forceinline__ int scale_unit(u16x2 ends) {
  const int top = __builtin_amdgcn_readfirstlane(ends.x), low = __builtin_amdgcn_readfirstlane(ends.y);
  return top <= 126 + HIGH_B && top != 1 && (!low || 255 - low >= 126 + LOW_B) ? 0 : top - 126 - HIGH_B;
}

// Over the lanes l, l + 16, l + 32, l + 48: rows of 16 swapped by VALU moves (a trip through LDS takes ten times as long:
// 7 % of 24 sequences with a chunk of 500).
template <class F>
__device__ __forceinline__ float over_groups(float v, F join) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = join(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return join(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float over_groups_max(float v) {
  return over_groups(v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float over_groups_sum(float v) {
  return over_groups(v, [](float x, float y) { return x + y; });
}
// The largest of a row of 16 lanes, in all of them.
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, __uint_as_float(dpp_u32<0xB1>(__float_as_uint(v))));
  v = fmaxf(v, __uint_as_float(dpp_u32<0x4E>(__float_as_uint(v))));
  v = fmaxf(v, __uint_as_float(dpp_u32<0x141>(__float_as_uint(v))));
  return fmaxf(v, __uint_as_float(dpp_u32<0x140>(__float_as_uint(v))));
}

// A tile's place in the step.
struct Tile {
  int r, hk, hb, ntok;                         // request (R: padding), kv head, block of GB heads, tokens
  int64_t tok0, p0;                            // first token and its position
  int64_t klo, khi, c0;                        // keys that some row sees, and where the parts are counted from
  int nsp, C;                                  // parts with keys, and their keys
};
// the keys of a tile whose first token is given
__device__ __forceinline__ void find_keys(const AttendArgs& a, const Split& sp, const Request& rq, Tile& t) {
  t.ntok = (int)min((int64_t)sp.TB, rq.q1 - t.tok0);
  t.p0 = t.r < a.st.R ? t.tok0 - rq.q1 + rq.len : -(int64_t)sp.TB;
  t.khi = min(t.p0 + t.ntok, a.maxlen);
  t.klo = max(t.p0 - a.window + 1, (int64_t)0);
  t.c0 = t.klo & ~(int64_t)31;
  // as many parts as there is room for, from the keys there are
  const int nk = t.khi > t.klo ? (int)(t.khi - t.c0) : 0;
  t.C = max(sp.C, ((nk + sp.S - 1) / sp.S + 127) & ~127);
  t.nsp = (nk + t.C - 1) / t.C;
}
__device__ __forceinline__ bool find_tile(const AttendArgs& a, const Split& sp, int id, Tile& t) {
  t.hb = id % sp.NHB;
  id /= sp.NHB;
  t.hk = id % a.Hkv;
  id /= a.Hkv;
  Request rq;
  if (sp.slots) {
    t.r = id / sp.slots;
    if (t.r >= a.st.R) return false;
    rq = sdc_request(a.st, t.r);
    if (rq.q1 - rq.q0 > (int64_t)sp.slots * sp.TB) return false;
    t.tok0 = rq.q0 + (int64_t)(id - t.r * sp.slots) * sp.TB;
  } else {
    int64_t first;
    t.r = sdc_find_request(a.st, id, sp.TB, 1, rq, first);
    if (t.r < 0) return false;
    if (t.r < a.st.R && rq.q1 - rq.q0 <= sp.few) return false;
    t.tok0 = rq.q0 + (id - first) * sp.TB;
  }
  if (t.tok0 < rq.q0 || t.tok0 >= rq.q1) return false;
  find_keys(a, sp, rq, t);
  return true;
}

// Four results of a row at element d (a multiple of 4), scaled.
__device__ __forceinline__ void write_four(const AttendArgs& a, int64_t tok, int h, int d, f32x4 x, float f) {
  uint16_t* o = a.o + tok * a.sot + h * a.soh;
  x *= f;
  uint32_t v[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    v[i] = a.fp16 ? sdc_to_half<SDC_FP16>(x[2 * i]) | (uint32_t)sdc_to_half<SDC_FP16>(x[2 * i + 1]) << 16
                  : sdc_to_half<SDC_BF16>(x[2 * i]) | (uint32_t)sdc_to_half<SDC_BF16>(x[2 * i + 1]) << 16;
  if (a.sod == 1 && ((uintptr_t)a.o % 8 | (uint64_t)(a.sot | a.soh) % 4) == 0) *reinterpret_cast<u32x2*>(o + d) = u32x2{v[0], v[1]};
  else
    for (int i = 0; i < 4; ++i) o[(d + i) * a.sod] = (uint16_t)(v[i / 2] >> (16 * (i % 2)));
}

// What a row's sums come to: x (elements d .. d + 3) in units of 2^(m + up), l in units of 2^(m - bias), x too.
__device__ __forceinline__ void write_row(const AttendArgs& a, const Tile& t, int tok, int64_t token, int head, int d, float m, float up,
                                          float l, f32x4 x, float bias) {
  // (a row with keys whose scores are all -inf: 0 / 0)
  const int64_t p = t.p0 + tok;
  const bool any = min(p + 1, a.maxlen) > max(p - a.window + 1, (int64_t)0);
  const float half = up == 0.f ? 1.f : __builtin_amdgcn_exp2f(0.5f * up);       // (2^up itself may be no fp32 number)
  write_four(a, token, head, d, x * (any ? half / l : 0.f), half);
  if (a.lse && d == 0) a.lse[token * a.slt + head] = any ? (m + log2f(l) - bias) * LN2 : NEG_INF;
}

// One row's results: x[0 .. n) at elements d.., scaled.
__device__ __forceinline__ void write_out(const AttendArgs& a, int64_t tok, int h, int d, const float* x, int n, float f) {
  uint16_t* o = a.o + tok * a.sot + h * a.soh;
  for (int i = 0; i < n && d + i < a.D; ++i)
    o[(d + i) * a.sod] = a.fp16 ? sdc_to_half<SDC_FP16>(x[i] * f) : sdc_to_half<SDC_BF16>(x[i] * f);
}

// The workgroup's part by plain_row, a wave a row; q: ANY_D floats of LDS a wave.  The kernel's arguments are read again, and the
// tile is found again: kept for this they would cost the callers their registers.
template <int CT>
__device__ __forceinline__ void plain_part(float* q, int waves) {
  auto args = (const __attribute__((address_space(4))) char*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  const AttendArgs& a = *(const AttendArgs*)args;
  const Split& sp = *(const Split*)(args + sizeof(AttendArgs));
  static_assert(sizeof(AttendArgs) % alignof(Split) == 0, "the second argument follows the first");
  const int lane = threadIdx.x & 63, D = a.D, w = threadIdx.x >> 6;
  const int s = blockIdx.x % sp.S, tile = sp.rows == ROWS ? blockIdx.x / sp.S : (int)(sp.tiles - 1 - blockIdx.x / sp.S);
  Tile t;
  if (!find_tile(a, sp, tile, t)) return;
  const int64_t a0 = t.c0 + (int64_t)s * t.C, a1 = min(t.khi, a0 + t.C);
  q += w * ANY_D;
  for (int row = w; row < sp.GB * sp.TB; row += waves) {
    const int tok = row / sp.GB, hd = t.hb * sp.GB + row % sp.GB;
    if (tok >= t.ntok || hd >= a.G) continue;
    const int64_t p = t.p0 + tok, token = t.tok0 + tok, lo = max(p - a.window + 1, a0), hi = min(min(p + 1, a.maxlen), a1);
    const int head = t.hk * a.G + hd;
    const float scale = plain_query(a, token, head, q);
    const PlainRow r = plain_row<CT>(a, q, scale, t.r, t.hk, lo, hi);
    if (t.nsp == 1) {
      write_plain(a, token, head, r, hi > lo);
      continue;
    }
    float* rec = sp.part + ((int64_t)tile * sp.S + s) * sp.rows * (D + HEAD);
    const float m = fmaxf(r.m, M0);
    if (lane == 0) *reinterpret_cast<f32x4*>(rec + HEAD * row) = f32x4{m + (float)r.u, m, r.l, 0.f};
#pragma unroll
    for (int e = 0; e < ANY_D / 64; ++e)
      if (lane + 64 * e < D) rec[HEAD * sp.rows + row * D + lane + 64 * e] = r.o[e];
  }
}

// Tiles of up to 16 query rows over a part of their keys: HBM bound, so a wave streams 32 keys at a time straight into
// registers and everything else stays there.  S^T = K Q^T on v_mfma_f32_16x16x32_f16 (lane l: key l % 16, a quarter of
// the depth; the depth's order is free, so a lane reads DP / 4 adjacent codes); the accumulator's layout (key 4 (l / 16)
// + i, row l % 16) is then the B operand of O^T = V^T P^T with the keys in that order, so the probabilities move to no
// other lane; V^T's fragments are 4 x 4 byte transposes of rows that a lane reads DP / 16 codes of.  Codes are exact in
// fp16; queries are scaled to it by a power of two per row (a bf16 element 2^-27 of its row's largest keeps all bits).
// The key scales multiply the scores, the value scales the probabilities, in fp32.  Probabilities are rounded to fp16's
// 11 bits, in units that put their largest product with a value scale at 2^12 .. 2^15 (scale_exponent).
// With fp16 outputs that leaves 1.4 times the error of fp32 probabilities against 64 bits; under bf16's own rounding it is gone.
// Four sequences of 100-131k tokens, 8 heads of 128: 172 us, 5.6 TB/s; 64 of 512-2048 tokens 37 us; one of 500 11 us.
// Registers for four workgroups a CU where heads are of 64 (24 sequences with a chunk of 500 24.3 us, with three 25.0; 64 decoding
// 25.5 and 25.1).
template <int CT, int DP, int PN>
__global__ __launch_bounds__(256, DP > 128 ? 1 : DP > 64 || PN == 1 ? 2 : 4) void kv_attend_rows(AttendArgs a, Split sp) {
  constexpr int NW = 4, KEYS = 32 * NW;                     // keys that the workgroup's waves take at a time
  constexpr int KW = DP / 64;                  // 16-byte reads of a key per lane; dwords of a value per lane
  constexpr int NS = DP / 32, ND = DP / 16;    // depth steps of a score, row blocks of the output
  constexpr int QS = DP + 8, OS = DP + 4;      // row pitches in LDS
  struct Head {
    float2 ks[MAXP], vs[MAXP];                 // of each page: ks and b; 2^-b and the factor on 2^b (in [1/2, 1) mostly)
    int32_t pg[MAXP];
    _Float16 q[ROWS][QS];
  };
  __shared__ union {
    Head h;
    float o[NW][ROWS][OS];
    float plain[NW][ANY_D];
  } sh;
  __shared__ float rowf[ROWS], ml[NW][ROWS][2];
  __shared__ u16x2 wends[NW];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int D = a.D, N = a.st.N;
  const int s = blockIdx.x % sp.S, tile = blockIdx.x / sp.S;
  Tile t;
  if (!find_tile(a, sp, tile, t)) return;
  if (s >= max(t.nsp, 1)) return;
  const int orow = (tid >> 4) & 15, od = (tid & 15) * ND;               // the output that a thread of the first 256 writes
  const int otok = orow / sp.GB, oh = t.hb * sp.GB + orow % sp.GB;
  const bool olive = tid < 256 && orow < sp.GB * sp.TB && otok < t.ntok && oh < a.G;
  const int64_t otoken = t.tok0 + otok;
  const int ohead = t.hk * a.G + oh;
  if (t.nsp == 0) {                            // no row sees a key
    const float zero[ND] = {};
    if (olive) {
      write_out(a, otoken, ohead, od, zero, ND, 0.f);
      if (a.lse && (tid & 15) == 0) a.lse[otoken * a.slt + ohead] = NEG_INF;
    }
    return;
  }
  const int64_t a0 = t.c0 + (int64_t)s * t.C, a1 = min(t.khi, a0 + t.C);
  const int64_t fp = (uint32_t)a0 / (uint32_t)N;
  const int np = (int)((uint32_t)(a1 - 1) / (uint32_t)N - fp) + 1, base0 = (int)(a0 - fp * N);

  // the part's pages; a page outside the cache is page 0, marked by its sign
  for (int i = tid; i < np; i += 64 * NW) {
    const int32_t page = a.st.bt[t.r * a.st.sbt + fp + i];
    sh.h.pg[i] = page >= 0 && page < a.st.NB ? page : (int32_t)0x80000000;
  }
  // the queries, a row per 16 threads
  uint32_t qr[ND / 2];
  {
    const uint16_t* qp = a.q + (olive ? otoken * a.sqt + ohead * a.sqh : 0);
    const bool vec = a.sqd == 1 && ((uintptr_t)a.q % 16 | (uint64_t)(a.sqt | a.sqh) % 8) == 0;
#pragma unroll
    for (int i = 0; i < ND / 2; ++i) qr[i] = 0u;
    if (olive && od < D) {
      if (vec) {                               // (D is a multiple of 16, and ND 4, 8 or 16)
        constexpr int C = ND / 2 < 4 ? 2 : 4;
        typedef uint32_t vt __attribute__((ext_vector_type(C)));
#pragma unroll
        for (int i = 0; i < ND / 2; i += C) {
          const vt x = *reinterpret_cast<const vt*>(qp + od + 2 * i);
#pragma unroll
          for (int j = 0; j < C; ++j) qr[i + j] = x[j];
        }
      } else {
#pragma unroll
        for (int i = 0; i < ND / 2; ++i)
          qr[i] = (uint32_t)qp[(od + 2 * i) * a.sqd] | (uint32_t)qp[(od + 2 * i + 1) * a.sqd] << 16;
      }
    }
  }
  __syncthreads();
  const int nk = (int)(a1 - a0);
  const uint8_t* base = a.kv + t.hk * a.ch;
  // page entry and slot of a key counted from a0
  auto place = [&](int key, int& slot) {
    const uint32_t loc = (uint32_t)(base0 + key);
    const int i = PN == 1 && N == 1 ? (int)loc : (int)__umulhi(loc, sp.div);
    slot = (int)loc - i * N;
    return min(i, np - 1);
  };
  struct Buf {
    u32x4 k[2][KW];
    uint32_t v[8][KW];
    int e[8];                                  // the keys' page entries
  };
  // where a lane's codes lie in its rows; columns past the head's are read from its last ones (keys': then taken as zeros)
  const uint32_t cn = (uint32_t)a.cn;          // (N cn is below 2^31)
  uint32_t kcol[KW];
#pragma unroll
  for (int j = 0; j < KW; ++j) kcol[j] = min(g * (DP / 4) + 16 * j, D - 16);
  const uint32_t vcol = D + min(c * (DP / 16), D - DP / 16);
  const uint32_t krow = c * cn, vrow = 4 * g * cn + vcol;
  typedef uint32_t vt __attribute__((ext_vector_type(KW)));
  auto load = [&](int k0, Buf& b) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      int slot;
      if constexpr (PN == 16) {                // the 16 keys lie in one page
        const int e = place(__builtin_amdgcn_readfirstlane(k0 + 16 * u), slot);
        const uint8_t* row = base + (int64_t)(__builtin_amdgcn_readfirstlane(sh.h.pg[e]) & 0x7FFFFFFF) * a.cb + (uint32_t)slot * cn;
#pragma unroll
        for (int j = 0; j < KW; ++j) b.k[u][j] = *reinterpret_cast<const u32x4*>(row + (krow + kcol[j]));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          vt x;
          if constexpr (KW == 1) x[0] = *reinterpret_cast<const uint32_t*>(row + i * cn + vrow);
          else x = *reinterpret_cast<const vt*>(row + i * cn + vrow);
          b.e[4 * u + i] = e;
#pragma unroll
          for (int j = 0; j < KW; ++j) b.v[4 * u + i][j] = x[j];
        }
      } else {
        int e = place(k0 + 16 * u + c, slot);
        const uint8_t* row = base + (int64_t)(sh.h.pg[e] & 0x7FFFFFFF) * a.cb + (uint32_t)slot * cn;
#pragma unroll
        for (int j = 0; j < KW; ++j) b.k[u][j] = *reinterpret_cast<const u32x4*>(row + kcol[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e = place(k0 + 16 * u + 4 * g + i, slot);
          b.e[4 * u + i] = e;
          const uint8_t* vr = base + (int64_t)(sh.h.pg[e] & 0x7FFFFFFF) * a.cb + (uint32_t)slot * cn + vcol;
#pragma unroll
          for (int j = 0; j < KW; ++j) b.v[4 * u + i][j] = *reinterpret_cast<const uint32_t*>(vr + 4 * j);
        }
      }
    }
  };

  // the pages' scales, then the first codes: a wait for the former leaves the latter on their way
  u16x2 ends = {0, 0};
  Buf b0, b1;
  int k = 32 * w;
  float2 sc0 = {0.f, 0.f};
  if (tid < np) {
    const float* scp = a.scales + (int64_t)(sh.h.pg[tid] & 0x7FFFFFFF) * a.sb + t.hk * a.sh;
    sc0 = {scp[0], scp[1]};
  }
  if (k < nk) load(k, b0);
  if (k + KEYS < nk) load(k + KEYS, b1);
  for (int i = tid; i < np; i += 64 * NW) {
    const int32_t page = sh.h.pg[i];
    const float* scp = a.scales + (int64_t)(page & 0x7FFFFFFF) * a.sb + t.hk * a.sh;
    float2 sc = sc0;
    if (i != tid) sc = {scp[0], scp[1]};
    if (page < 0) sc = {__builtin_nanf(""), __builtin_nanf("")};
    const int b = scale_exponent(sc.y, 0);
    sh.h.ks[i] = {sc.x, (float)b};
    sh.h.vs[i] = {ldexpf(1.f, -b), scale_factor(sc.y, b)};
    ends = scale_ends(ends, sc.y);
  }
  ends = wave_larger(ends);
  if (lane == 0) wends[w] = ends;
  {
    float x[ND], amax = 0.f;
    if (a.fp16) {
#pragma unroll
      for (int i = 0; i < ND / 2; ++i) {
        x[2 * i] = f16_lo(qr[i]);
        x[2 * i + 1] = f16_hi(qr[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < ND / 2; ++i) {
        x[2 * i] = bf16_lo(qr[i]);
        x[2 * i + 1] = bf16_hi(qr[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const float f = fabsf(x[i]);
      if (f < __builtin_inff()) amax = fmaxf(amax, f);
    }
    amax = row_max(amax);
    int e = 0;
    (void)frexpf(amax, &e);
    e = max(e, -100);
    const float f = ldexpf(1.f, 13 - e);
#pragma unroll
    for (int i = 0; i < ND; ++i)
      if (tid < 256) sh.h.q[orow][od + i] = (_Float16)(x[i] * f);
    if (tid < 256 && (tid & 15) == 0) rowf[orow] = ldexpf(a.scale, e - 13);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NW; ++i) ends = __builtin_elementwise_max(ends, wends[i]);
  if (scales_apart(ends)) {
    __syncthreads();                           // (the tables' place is the plain rows')
    plain_part<CT>(&sh.plain[0][0], NW);
    __builtin_amdgcn_endpgm();                 // (after a return in its place the rest spills 60 scalar registers)
  }
  const int ve = scale_unit(ends);
  if (ve != 0) {
    for (int i = tid; i < np; i += 64 * NW) {
      const float v = ldexpf(sh.h.vs[i].y, (int)sh.h.ks[i].y);
      const int b = scale_exponent(v, ve);
      sh.h.ks[i].y = (float)b;
      sh.h.vs[i] = {ldexpf(1.f, -b), scale_factor(v, b + ve)};
    }
    __syncthreads();
  }
  f16x8 qf[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) qf[i] = *reinterpret_cast<const f16x8*>(&sh.h.q[c][g * (DP / 4) + 8 * i]);
  const float rf = rowf[c];
  // the keys that the lane's row sees, counted from a0
  const int64_t prow = t.p0 + c / sp.GB;
  const int rhi = (int)(min(min(prow + 1, a.maxlen), a1) - a0);
  const int rlo = (int)max(min(prow - a.window + 1 - a0, (int64_t)1 << 30), -((int64_t)1 << 30));
  // those that every row of the tile sees
  const int fhi = (int)(min(min(t.p0 + 1, a.maxlen), a1) - a0);
  const int flo = (int)max(min(t.p0 + t.ntok - a.window - a0, (int64_t)1 << 30), -((int64_t)1 << 30));

  f32x4 o[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = M0, l = 0.f;
  auto compute = [&](int k0, Buf& b) {
    if (D < DP) {
      asm volatile("");                        // (a branch)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < KW; ++j)
          if (g * (DP / 4) + 16 * j >= D) b.k[u][j] = u32x4{0, 0, 0, 0};
    }
    f32x4 sc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      sc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NS; ++i)
        sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen8<CT>(b.k[u][i / 2][2 * (i % 2)], b.k[u][i / 2][2 * (i % 2) + 1]),
                                                       qf[i], sc[u], 0, 0, 0);
    }
    // With b the exponent of the page's value scale, p v is 2^(x + b) times a factor of at most 1: it is that exponent whose
    // maximum m is, and the sum of probabilities takes 2^-b of it.
    float x[8], top = M0;
    float2 ps[8];                              // the keys' scales
#pragma unroll
    for (int j = 0; j < 8; ++j) ps[j] = sh.h.ks[b.e[j]];
    const bool edge = k0 < flo || k0 + 32 > fhi;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = fmaf(sc[j / 4][j % 4], ps[j].x * rf, ps[j].y);
    bool seen[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) seen[j] = true;
    if (edge) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = k0 + 16 * (j / 4) + 4 * g + j % 4;
        seen[j] = key >= rlo && key < rhi;
        x[j] = seen[j] ? x[j] : NEG_INF;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, x[j]);
    // the maximum follows only when it is passed by 2 (a factor of 4, which fp16 has room for)
    if (__any(top > m + 2.f)) {
      const float mn = fmaxf(m, over_groups_max(top));
      const float f = exp2f(m - mn);
      l *= f;
#pragma unroll
      for (int n = 0; n < ND; ++n) o[n] *= f;
      m = mn;
    }
    const float down = BIAS - m;
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) ps[j] = sh.h.vs[b.e[j]];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = __builtin_amdgcn_exp2f(x[j] + down);
      l = fmaf(p[j], ps[j].x, l);
      p[j] *= ps[j].y;
    }
    if (edge) {
      // what no row sees may hold anything: as if it were zero
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = k0 + 16 * (j / 4) + 4 * g + j % 4;
        const bool any = key + a0 >= t.klo && key < nk;
        p[j] = seen[j] ? p[j] : 0.f;
#pragma unroll
        for (int i = 0; i < KW; ++i) b.v[j][i] = any ? b.v[j][i] : 0u;
      }
    }
    f16x8 pf;
#pragma unroll
    for (int j = 0; j < 8; ++j) pf[j] = (_Float16)p[j];
    if constexpr (CT == SDC_CACHE_E4M3) {
      if (edge) {
        // a value of NaN reaches only the rows that see its key (0 times NaN would reach the others): counted by a product
        // of its own, and taken out of the values
        uint32_t bad = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 0; i < KW; ++i) bad |= nan_codes(b.v[j][i]);
        if (__any(bad != 0)) {
          f16x8 sf;
#pragma unroll
          for (int j = 0; j < 8; ++j) sf[j] = (_Float16)(seen[j] ? 1.f : 0.f);
#pragma unroll
          for (int n = 0; n < ND; ++n) {
            f16x8 nf;
#pragma unroll
            for (int j = 0; j < 8; ++j) nf[j] = (_Float16)(((b.v[j][n / 4] >> (8 * (n % 4))) & 0x7F) == 0x7F ? 1.f : 0.f);
            const f32x4 cnt = __builtin_amdgcn_mfma_f32_16x16x32_f16(nf, sf, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][i] = cnt[i] > 0.f ? __builtin_nanf("") : o[n][i];
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < KW; ++i) {
              const uint32_t z = nan_codes(b.v[j][i]);
              b.v[j][i] &= ~((z >> 7) * 0xFFu);
            }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < KW; ++i) {
      uint32_t lo[4], hi[4];
      const uint32_t xl[4] = {b.v[0][i], b.v[1][i], b.v[2][i], b.v[3][i]};
      const uint32_t xh[4] = {b.v[4][i], b.v[5][i], b.v[6][i], b.v[7][i]};
      transpose4(xl, lo);
      transpose4(xh, hi);
#pragma unroll
      for (int n = 0; n < 4; ++n)
        o[4 * i + n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen8<CT>(lo[n], hi[n]), pf, o[4 * i + n], 0, 0, 0);
    }
  };

  while (k < nk) {                             // the next keys in flight
    compute(k, b0);
    if (k + 2 * KEYS < nk) load(k + 2 * KEYS, b0);
    k += KEYS;
    if (k >= nk) break;
    compute(k, b1);
    if (k + 2 * KEYS < nk) load(k + 2 * KEYS, b1);
    k += KEYS;
  }

  // the waves' sums joined: a lane holds DP / 4 adjacent outputs of its row
  l = over_groups_sum(l);
  __syncthreads();
  if (g == 0) {
    ml[w][c][0] = m;
    ml[w][c][1] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < ND; n += 4)
      *reinterpret_cast<f32x4*>(&sh.o[w][c][(4 * g + i) * ND + n]) = f32x4{o[n][i], o[n + 1][i], o[n + 2][i], o[n + 3][i]};
  __syncthreads();
  constexpr int Q = DP / 4;                    // threads of a row, four elements each
  for (int i = tid; i < ROWS * Q; i += 64 * NW) {
    const int row = i / Q, d = 4 * (i - row * Q), tok = row / sp.GB, hd = t.hb * sp.GB + row % sp.GB;
    if (row >= sp.GB * sp.TB || tok >= t.ntok || hd >= a.G || d >= D) continue;
    const int64_t token = t.tok0 + tok;
    const int head = t.hk * a.G + hd;
    float mt = M0, lt = 0.f;
#pragma unroll
    for (int u = 0; u < NW; ++u) mt = fmaxf(mt, ml[u][row][0]);
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < NW; ++u) {
      const float f = __builtin_amdgcn_exp2f(ml[u][row][0] - mt);
      lt = fmaf(f, ml[u][row][1], lt);
      x += f * *reinterpret_cast<const f32x4*>(&sh.o[u][row][d]);
    }
    if (t.nsp == 1) {
      write_row(a, t, tok, token, head, d, mt, (float)ve, lt, x, BIAS);
    } else {
      float* rec = sp.part + (int64_t)blockIdx.x * ROWS * (D + HEAD);
      constexpr float unit = 0x1p-13f;         // 2^-BIAS
      if (d == 0) *reinterpret_cast<f32x4*>(rec + HEAD * row) = f32x4{mt + (float)ve, mt, lt * unit, 0.f};
      *reinterpret_cast<f32x4*>(rec + HEAD * ROWS + row * D + d) = x * unit;
    }
  }
}

// ---------------------------------------------------------------------------------------------- many query rows
// Waves of a workgroup, 32 query rows each: a head of 256 needs all 512 registers of a lane.
constexpr int tall_waves(int64_t D) { return D > 128 ? 4 : 8; }

// The largest of both lanes (l, l + 32) that share a query row, and their sum.
__device__ __forceinline__ float over_halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float over_halves_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Tiles of up to 256 query rows over a part of their keys, KT keys at a time.  The workgroup widens a tile of codes to
// fp16 (exact) once, into LDS, keys row by row and values transposed; each wave then reads them as A fragments of
// v_mfma_f32_32x32x16_f16.  S^T = K Q^T leaves a lane with one query row (l % 32) and keys 8 j + 4 (l / 32) + i; that is
// the B operand of O^T = V^T P^T if a value row's 16 keys are stored in the order 0-3, 8-11, 4-7, 12-15, so the
// probabilities never leave their lane.  A tile's codes are loaded a step before they are widened, into the other of two
// buffers: one barrier a tile.
//
// The softmax takes as long as the products (a score is 4 D / 1024 cycles of the matrix cores and each VALU instruction a
// 16th), so it is short: keys of a group (16, or 4 where a page holds no multiple of 16, or 1) share their scales, and with
// y = x + log2 vs the product p vs is 2^(y - m): one fused multiply-add and one exponential a score, while the next tile's
// scores are computed.  m follows the largest y, and the sum takes the group's sum over vs.  Scales without a logarithm are
// factors on the widened values; keys that a row does not see score -inf; values of NaN under a tile that some row sees only
// in part are left out and put in at the end.  Rounding of the probabilities, and scales far from 1: as kv_attend_rows.
//
// Two chunks of 2048 tokens behind up to 3000 keys, 32 heads of 128: 293 us, 864 TFLOP/s; the matrix cores are busy 38 % of
// it.  Waves of 32 rows: 64 would need all 512 registers, 16 twice the fragments.
template <int CT, int DP, int PN>
__global__ __launch_bounds__(64 * tall_waves(DP), tall_waves(DP) / 4) void kv_attend_tiles(AttendArgs a, Split sp) {
  constexpr int KT = DP > 128 ? 32 : 64, KB = KT / 32;                  // keys of a tile, blocks of 32
  // depth steps of a score; the values' rows, by which of a dword's four codes they are, and blocks of 32 of them (a head of
  // 96 in quarters of 32, 8 of them unused: a lane then has adjacent outputs)
  constexpr int NS = DP / 16, VR = DP == 96 ? 32 : DP / 4, ND = 4 * VR / 32;
  constexpr int KP = 2 * DP + 16, VP = 2 * KT + 16;                     // row pitches in bytes
  constexpr int NW = tall_waves(DP), TALL = 32 * NW, HT = 32 * NW;      // half of the threads load keys, half values
  // reads of a key and of a thread, 16 codes each; columns of 4 codes of a value, units (8 keys x 4 codes) of a thread
  // (sized so that what a wave reads lies in one page where a page holds multiples of 16 keys)
  constexpr int KC = DP == 96 ? 8 : DP / 16, KU = (KT * KC + HT - 1) / HT;
  constexpr int VC = DP <= 96 ? 32 : DP / 4, VUN = KT / 8 * VC, VU = (VUN + HT - 1) / HT;
  constexpr int NX = 4 * KU > 8 * VU ? 4 * KU : 8 * VU;
  struct Stage {
    uint8_t k[KT * KP];
    uint8_t v[4 * VR * VP];
    float4 sc[KT];                             // of each key, as of its page
  };
  struct WaveScales {
    u16x2 ends;
    bool flip, mul;
  };
  __shared__ Stage st[2];
  __shared__ WaveScales wscales[NW];
  __shared__ int32_t pg[MAXP];
  __shared__ float4 ps[MAXP];                  // of each page (page_scales)
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int D = a.D, N = a.st.N;
  const int s = blockIdx.x % sp.S, tile = (int)(sp.tiles - 1 - blockIdx.x / sp.S);  // late tokens, with the most keys, first
  Tile t;
  if (!find_tile(a, sp, tile, t)) return;
  if (s >= max(t.nsp, 1)) return;
  // the lane's row (found again at the end, rather than kept)
  struct Row {
    int row, tok, head;
    int64_t token;
    bool live;
  };
  auto row_of = [&]() {
    int id = threadIdx.x;
    asm volatile("" : "+v"(id));
    Row r;
    r.row = 32 * (id >> 6) + (id & 31);
    r.tok = r.row / sp.GB;
    const int hd = t.hb * sp.GB + r.row % sp.GB;
    r.live = r.row < sp.GB * sp.TB && r.tok < t.ntok && hd < a.G;
    r.token = t.tok0 + (r.live ? r.tok : 0);
    r.head = t.hk * a.G + (r.live ? hd : 0);
    return r;
  };
  if (t.nsp == 0) {                            // no row sees a key
    const Row r = row_of();
    if (r.live) {
      for (int d = 4 * h; d < D; d += 8) write_four(a, r.token, r.head, d, f32x4{0.f, 0.f, 0.f, 0.f}, 0.f);
      if (a.lse && h == 0) a.lse[r.token * a.slt + r.head] = NEG_INF;
    }
    return;
  }
  const int64_t a0 = t.c0 + (int64_t)s * t.C, a1 = min(t.khi, a0 + t.C);
  const int64_t fp = (uint32_t)a0 / (uint32_t)N;
  const int np = (int)((uint32_t)(a1 - 1) / (uint32_t)N - fp) + 1, base0 = (int)(a0 - fp * N);
  // |ks|; log2 of |vs| / 2^ve, at least LOW_B; the power of two that goes back; the factor on the stored values
  auto page_scales = [](float ks, float vs, int ve) -> float4 {
    const int f = (int)scale_field(vs);
    const float v = ldexpf(fabsf(vs), -ve);
    const bool log = f && f - 126 - ve >= LOW_B, small = !log && (f || vs == 0.f);
    const float inv = log ? 1.f / v : small ? ldexpf(1.f, -LOW_B) : 1.f;
    if (ks != ks) return {0.f, 0.f, ks, ks};
    return {fabsf(ks), log ? log2f(v) : small ? (float)LOW_B : 0.f, inv, log ? (vs < 0.f ? -1.f : 1.f) : ldexpf(vs, -ve) * inv};
  };
  // the queries: fragments of the lane's row, in fp16 after a power of two
  f16x8 qf[NS];
  float rf;
  bool flip = false, mul = false;
  u16x2 ends = {0, 0};
  int64_t prow;                                // the lane's position
  {
    const Row r = row_of();
    const bool live = r.live;
    prow = t.p0 + min(r.tok, t.ntok - 1);
    const uint16_t* qp = a.q + r.token * a.sqt + r.head * a.sqh;
    const bool vec = a.sqd == 1 && ((uintptr_t)a.q % 16 | (uint64_t)(a.sqt | a.sqh) % 8) == 0;
    u32x4 raw[NS];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      raw[i] = u32x4{0, 0, 0, 0};
      const int run = 2 * i + h, d = 16 * (run % NS) + 8 * (run / NS);  // (the order in which the keys' codes are stored)
      if (live && d < D) {
        if (vec) raw[i] = *reinterpret_cast<const u32x4*>(qp + d);
        else
          for (int e = 0; e < 4; ++e)
            raw[i][e] = (uint32_t)qp[(d + 2 * e) * a.sqd] | (uint32_t)qp[(d + 2 * e + 1) * a.sqd] << 16;
      }
    }
    int e = 0;
    // The part's pages and their scales.  A page outside the cache is page 0 with scales of NaN.  Value scales that have no
    // logarithm (infinity, NaN) become factors on the widened values, and so do signs and what scales under 2^LOW_B are less
    // than that; a key scale of NaN makes the page's share of the sum and its values NaN.
    for (int i = tid; i < np; i += 2 * HT) {
      const int32_t p = a.st.bt[t.r * a.st.sbt + fp + i];
      const bool in = p >= 0 && p < a.st.NB;
      const float* scp = a.scales + (in ? (int64_t)p : 0) * a.sb + t.hk * a.sh;
      const float ks = in ? scp[0] : __builtin_nanf(""), vs = in ? scp[1] : __builtin_nanf("");
      ps[i] = page_scales(ks, vs, 0);
      pg[i] = (in ? p : 0) | (ks < 0.f ? (int32_t)0x80000000 : 0);        // the sign of ks, which the keys take
      ends = scale_ends(ends, vs);
      flip |= ks < 0.f;
      mul |= ps[i].w != 1.f;
    }
    auto narrow = [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = fabsf(lo_of<DT>(raw[i][j])), y = fabsf(hi_of<DT>(raw[i][j]));
          amax = fmaxf(amax, fmaxf(x < __builtin_inff() ? x : 0.f, y < __builtin_inff() ? y : 0.f));
        }
      amax = over_halves_max(amax);
      (void)frexpf(amax, &e);
      e = max(e, -100);
      const float f = ldexpf(a.scale < 0.f ? -1.f : 1.f, 13 - e);
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          qf[i][2 * j] = (_Float16)(lo_of<DT>(raw[i][j]) * f);
          qf[i][2 * j + 1] = (_Float16)(hi_of<DT>(raw[i][j]) * f);
        }
    };
    if (a.fp16) narrow(std::integral_constant<int, SDC_FP16>{});
    else narrow(std::integral_constant<int, SDC_BF16>{});
    rf = ldexpf(fabsf(a.scale), e - 13);       // (scores times key scales that are not negative keep their order)
  }
  ends = wave_larger(ends);
  const bool wave_flip = __any(flip), wave_mul = __any(mul);
  if (lane == 0) wscales[w] = {ends, wave_flip, wave_mul};
  __syncthreads();
  flip = mul = false;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const WaveScales x = wscales[i];
    ends = __builtin_elementwise_max(ends, x.ends);
    flip |= x.flip;
    mul |= x.mul;
  }
  const bool flips = __builtin_amdgcn_readfirstlane(flip), muls = __builtin_amdgcn_readfirstlane(mul);
  if (scales_apart(ends)) {
    plain_part<CT>(reinterpret_cast<float*>(st), NW);
    __builtin_amdgcn_endpgm();
  }
  const int ve = scale_unit(ends);
  if (ve != 0) {
    for (int i = tid; i < np; i += 2 * HT)
      if (ps[i].z == ps[i].z) {                // (pages outside the cache, and whose key scale is NaN, are as they were)
        const float* scp = a.scales + (int64_t)(pg[i] & 0x7FFFFFFF) * a.sb + t.hk * a.sh;
        ps[i] = page_scales(scp[0], scp[1], ve);
      }
    __syncthreads();
  }
  // keys, counted from a0: those of the tile; those that the lane's row sees; those that a row of the wave, and every row of
  // the wave sees; those that every row of the tile sees
  auto clip = [](int64_t x) { return (int)max(min(x, (int64_t)1 << 30), -((int64_t)1 << 30)); };
  const int nk = (int)(a1 - a0), lo0 = clip(t.klo - a0);
  const int tok_a = 32 * w / sp.GB, tok_b = min((32 * w + 31) / sp.GB, t.ntok - 1);
  const int rhi = (int)(min(min(prow + 1, a.maxlen), a1) - a0), rlo = clip(prow - a.window + 1 - a0);
  const uint32_t span = (uint32_t)max(rhi - rlo, 0);
  const bool busy = tok_a < t.ntok;            // the wave has rows
  const int whi = busy ? (int)(min(min(t.p0 + tok_b + 1, a.maxlen), a1) - a0) : 0, wlo = clip(t.p0 + tok_a - a.window + 1 - a0);
  const int fhi = (int)(min(min(t.p0 + tok_a + 1, a.maxlen), a1) - a0), flo = clip(t.p0 + tok_b - a.window + 1 - a0);
  const int ahi = (int)(min(min(t.p0 + 1, a.maxlen), a1) - a0), alo = clip(t.p0 + t.ntok - a.window - a0);
  const uint8_t* base = a.kv + t.hk * a.ch;

  const uint32_t cn = (uint32_t)a.cn;          // (N cn is below 2^31)
  auto place = [&](int key, int& slot) {       // page entry and slot of a key counted from a0
    const uint32_t loc = (uint32_t)(base0 + key);
    const int i = PN == 1 && N == 1 ? (int)loc : (int)__umulhi(loc, sp.div);
    slot = (int)loc - i * N;
    return min(i, np - 1);
  };
  // The first half of the waves loads and widens the keys, the second the values.  Keys outside the tile's, and codes past
  // the head's, are read from where there is something to read and taken as zeros.
  const int half = tid & (HT - 1);
  const bool vals = w >= NW / 2;
  bool bad = false;
  const uint32_t in0 = (uint32_t)(nk - lo0);
  struct Next {
    uint32_t x[NX];
  };
  // a thread's codes: column and first key (of values: keys key0 + (0..3, 8..11)), where they lie in memory and in LDS
  const int col = vals ? 4 * (half % VC) : 16 * (half % KC), cg0 = half / VC;
  const int key0 = vals ? 16 * (cg0 >> 1) + 4 * (cg0 & 1) : half / KC;
  const uint32_t code = vals ? D + min(col, D - 4) : min(col, D - 16);
  const uint32_t at = (uint32_t)(vals ? 4 * (cg0 & 1) : key0 % 16) * cn + code;
  const int lds = vals ? col / 4 * VP + 16 * cg0 : key0 * KP + col;
  const bool pad = col >= D;
  auto row_at = [&](int key) {
    int slot;
    const int e = place(key, slot);
    return base + (int64_t)(pg[e] & 0x7FFFFFFF) * a.cb + (uint32_t)slot * cn;
  };
  // Where a wave's keys are in one page its entry is read a step before it is needed (its 16 keys are the same for all lanes).
  constexpr int KSTEP = HT / KC, VSTEP = 8 * (HT / VC);                 // keys between a thread's reads
  int entry[KU > VU ? KU : VU];
  auto group = [&](int k0, int u) { return __builtin_amdgcn_readfirstlane((k0 + key0 + (vals ? VSTEP : KSTEP) * u) & ~15); };
  auto find = [&](int k0) {
#pragma unroll
    for (int u = 0; u < (KU > VU ? KU : VU); ++u) {
      int slot;
      if (PN == 16) entry[u] = pg[place(group(k0, u), slot)];
    }
  };
  auto group_at = [&](int k0, int u) {
    int slot;
    (void)place(group(k0, u), slot);
    return base + (int64_t)(__builtin_amdgcn_readfirstlane(entry[u]) & 0x7FFFFFFF) * a.cb + (uint32_t)slot * cn;
  };
  auto load = [&](int k0, Next& n) {
    if (!vals) {
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        u32x4 x;
        if constexpr (PN == 16) x = *reinterpret_cast<const u32x4*>(group_at(k0, u) + (KSTEP * u % 16) * cn + at);
        else x = *reinterpret_cast<const u32x4*>(row_at(k0 + key0 + KSTEP * u) + code);
#pragma unroll
        for (int i = 0; i < 4; ++i) n.x[4 * u + i] = x[i];
      }
      return;
    }
#pragma unroll
    for (int u = 0; u < VU; ++u) {
      const int key = k0 + key0 + VSTEP * u;
      if (VUN < HT && half >= VUN) continue;
      if constexpr (PN == 16) {
        const uint8_t* p = group_at(k0, u);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          n.x[8 * u + i] = *reinterpret_cast<const uint32_t*>(p + (i % 4 + 8 * (i / 4)) * cn + at);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          n.x[8 * u + i] = *reinterpret_cast<const uint32_t*>(row_at(key + i % 4 + 8 * (i / 4)) + code);
      }
    }
  };
  auto store = [&](int k0, Next n, Stage& d) {
    const bool whole = k0 >= lo0 && k0 + KT <= nk;
    if (!vals) {
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        const int key = k0 + key0 + HT / KC * u;
        if (DP == 96 && col >= DP) continue;
        if (!whole || D < DP) {
          asm volatile("");                    // (a branch: it is the same for all lanes and hardly ever taken)
          if ((uint32_t)(key - lo0) >= in0 || pad) n.x[4 * u] = n.x[4 * u + 1] = n.x[4 * u + 2] = n.x[4 * u + 3] = 0u;
        }
        f16x8 p0 = widen8<CT>(n.x[4 * u], n.x[4 * u + 1]), p1 = widen8<CT>(n.x[4 * u + 2], n.x[4 * u + 3]);
        if (flips) {
          asm volatile("");
          int slot;
          const _Float16 f = pg[place(key, slot)] < 0 ? (_Float16)-1.f : (_Float16)1.f;
          p0 *= f;
          p1 *= f;
        }
        uint8_t* p = d.k + lds + HT / KC * u * KP;            // (two runs of 8 codes, half a row apart)
        *reinterpret_cast<f16x8*>(p) = p0;
        *reinterpret_cast<f16x8*>(p + DP) = p1;
      }
      return;
    }
    const bool part = k0 < alo || k0 + KT > ahi;
#pragma unroll
    for (int u = 0; u < VU; ++u) {
      const int vkey = k0 + key0 + 8 * (HT / VC) * u;
      if ((VUN < HT && half >= VUN) || (4 * VC > DP && col >= DP)) continue;
      if (!whole || D < DP) {
        asm volatile("");
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if ((uint32_t)(vkey + i % 4 + 8 * (i / 4) - lo0) >= in0 || pad) n.x[8 * u + i] = 0u;
      }
      // values that are NaN, where some row may not see them (0 times NaN would reach it): left to the end
      if (CT == SDC_CACHE_E4M3 && part) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t z = nan_codes(n.x[8 * u + i]);
          n.x[8 * u + i] &= ~((z >> 7) * 0xFFu);
          bad |= z != 0;
        }
      }
      uint32_t lo[4], hi[4];
      transpose4(n.x + 8 * u, lo);
      transpose4(n.x + 8 * u + 4, hi);
      f16x8 v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = widen8<CT>(lo[e], hi[e]);
      if (muls) {
        asm volatile("");
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = vkey + i % 4 + 8 * (i / 4);
          int slot;
          const int e = place(key, slot);
          float x = (uint32_t)(key - lo0) < in0 ? ps[e].w : 1.f;
          if (part && !(fabsf(x) <= 1.f)) {
            x = 0.f;
            bad = true;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j][i] *= (_Float16)x;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<f16x8*>(d.v + lds + e * VR * VP + 16 * (HT / VC) * u) = v[e];
    }
    if (half < KT) {
      int slot;
      const int e = place(k0 + half, slot);
      d.sc[half] = ps[e];
    }
  };

  f32x16 o[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[n][i] = 0.f;
  float m = M0, l = 0.f;

  const int klane = c * KP + 16 * h, vlane = c * VP + 16 * h;           // row c of a block, the half's run of 8
  auto products = [&](const uint8_t* k, f32x16* x) {                    // the scores of a tile's keys
#pragma unroll
    for (int b = 0; b < KB; ++b) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[b][i] = 0.f;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const f16x8 kf = *reinterpret_cast<const f16x8*>(k + klane + 32 * b * KP + 32 * i);
        x[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[i], x[b], 0, 0, 0);
      }
    }
  };
  // the softmax and the values' products of a tile whose scores are x; between its exponentials, the next tile's scores
  auto finish = [&](int k0, const Stage& d, f32x16* x, const uint8_t* next, f32x16* y) {
    // Fragments are read AHEAD products before they are used (left to itself the compiler reads one at a time and waits for
    // it: two prompt chunks of 2048 tokens 323 us, 297 so), first the keys', then the values', neighbours into different accumulators.
    constexpr int MK = KB * NS, MV = ND * KT / 16, AHEAD = 4;
    f16x8 fr[AHEAD];
    auto fragment = [&](int q) {
      return *reinterpret_cast<const f16x8*>(q < MK ? next + klane + 32 * (q % KB) * KP + 32 * (q / KB)
                                                    : d.v + vlane + 32 * ((q - MK) % ND) * VP + 32 * ((q - MK) / ND));
    };
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) fr[q] = fragment(q);
    __builtin_amdgcn_sched_barrier(0x6);
    if (k0 < flo || k0 + KT > fhi) {           // some rows see some of the keys
      const uint32_t from = (uint32_t)(k0 + 4 * h - rlo);
#pragma unroll
      for (int j = 0; j < 16 * KB; ++j) {
        const bool in = from + (uint32_t)(32 * (j / 16) + 8 * (j % 16 / 4) + j % 4) < span;
        x[j / 16][j % 16] = in ? x[j / 16][j % 16] : NEG_INF;
      }
    }
    constexpr int GE = PN == 16 ? 8 : PN, NG = 16 * KB / GE;            // a lane's scores of a group, groups
    const float4* scp = d.sc + (PN == 16 ? 0 : 4 * h);
    auto scales = [&](int j0) { return scp[PN == 16 ? 2 * j0 : 32 * (j0 / 16) + 8 * (j0 % 16 / 4) + j0 % 4]; };
    auto factor = [&](float ks) { return fmaxf(ks * rf, 0x1p-126f); };  // (not 0: -inf stays)
    float top = NEG_INF;
    auto largest = [&](int j0) {
      float z = x[j0 / 16][j0 % 16];
#pragma unroll
      for (int i = 1; i < GE; ++i) z = fmaxf(z, x[(j0 + i) / 16][(j0 + i) % 16]);
      return z;
    };
    if (muls) {                                // (a key scale of NaN, however little its keys would weigh)
      asm volatile("");
#pragma unroll
      for (int g = 0; g < NG; ++g) l = scales(g * GE).z != scales(g * GE).z && largest(g * GE) > NEG_INF ? __builtin_nanf("") : l;
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int j0 = g * GE;
      const float4 sc = scales(j0);
      const float z = largest(j0);
      top = fmaxf(top, fmaf(z, factor(sc.x), sc.y));
    }
    // the maximum follows the scores when they pass it by 2 (fp16 has room for that)
    if (__any(top > m + 2.f)) {
      const float mn = fmaxf(m, over_halves_max(top));
      const float f = __builtin_amdgcn_exp2f(m - mn);
      l *= f;
#pragma unroll
      for (int n = 0; n < ND; ++n) o[n] *= f;
      m = mn;
    }
    f16x8 pf[KT / 16];
    // (keys that share no page: their scales are read where they are used, 128 registers would not hold them)
    constexpr bool EACH = GE == 1;
    float cs[NG], b0[NG], inv[NG], sum[NG];
#pragma unroll
    for (int g = 0; g < (EACH ? 0 : NG); ++g) {
      const float4 sc = scales(g * GE);
      cs[g] = factor(sc.x);
      b0[g] = sc.y - m + BIAS;
      inv[g] = sc.z;
      sum[g] = 0.f;
    }
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) y[b][i] = 0.f;
#pragma unroll
    for (int q = 0; q < MK + MV; ++q) {
      if (q < MK) y[q % KB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[q % AHEAD], qf[q / KB], y[q % KB], 0, 0, 0);
      else o[(q - MK) % ND] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[q % AHEAD], pf[(q - MK) / ND], o[(q - MK) % ND], 0, 0, 0);
      if (q + AHEAD < MK + MV) fr[q % AHEAD] = fragment(q + AHEAD);
      if (q < MK) {
#pragma unroll
        for (int j = q * 16 * KB / MK; j < (q + 1) * 16 * KB / MK; ++j) {
          const int g = j / GE;
          float p;
          if constexpr (EACH) {
            const float4 sc = scales(j);
            p = __builtin_amdgcn_exp2f(fmaf(x[j / 16][j % 16], factor(sc.x), sc.y - m + BIAS));
            l = p == 0.f ? l : fmaf(p, sc.z, l);
          } else {
            p = __builtin_amdgcn_exp2f(fmaf(x[j / 16][j % 16], cs[g], b0[g]));
            sum[g] += p;
          }
          pf[j / 8][j % 8] = (_Float16)p;
        }
      }
      __builtin_amdgcn_sched_barrier(0x6);
    }
#pragma unroll
    for (int g = 0; g < (EACH ? 0 : NG); ++g) l = sum[g] == 0.f ? l : fmaf(sum[g], inv[g], l);
  };

  // In the step of tile t the waves take the values of t and the keys of t + 1.  At its start the values of t + 1 and the keys of
  // t + 2, loaded during the step before, are put where the values of t - 1 and the keys of t were.
  Next n;
  {
    Next first;
    find(0);
    load(0, first);
    if (KT < nk) {
      find(KT);
      load(KT, n);
    }
    store(0, first, st[0]);
  }
  if (!vals && KT < nk) {
    store(KT, n, st[1]);
    if (2 * KT < nk) {
      find(2 * KT);
      load(2 * KT, n);
    }
  }
  const int ahead = vals ? KT : 2 * KT;
  find(ahead + KT);
  __syncthreads();
  f32x16 xa[KB], xb[KB];
  products(st[0].k, xa);
  __syncthreads();
  auto step = [&](int k, Stage& d, Stage& e, f32x16* x, f32x16* y) {
    if (k + ahead < nk) store(k + ahead, n, vals ? e : d);
    if (k + ahead + KT < nk) load(k + ahead + KT, n);
    if (k < whi && k + KT > wlo) finish(k, d, x, e.k, y);
    else if (k + KT < whi && k + 2 * KT > wlo) products(e.k, y);
    find(k + ahead + 2 * KT);
    __syncthreads();
  };
  for (int k = 0; k < nk; k += 2 * KT) {
    step(k, st[0], st[1], xa, xb);
    if (k + KT < nk) step(k + KT, st[1], st[0], xb, xa);
  }

  // o[q][i] of a lane is element 4 (p % VR) + p / VR, p = 32 q + 8 (i / 4) + 4 h + i % 4: the values' rows lie in that order
  auto element = [&](int q, int i) {
    const int p = 32 * q + 8 * (i / 4) + 4 * h + i % 4;
    return 4 * (p % VR) + p / VR;
  };
  auto each = [&](auto use) {                  // four adjacent elements at a time
    constexpr int B = VR > 32 ? VR / 32 : 1, E = VR < 32 ? 8 : 16;      // blocks and registers of a quarter's rows
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int i = 0; i < E; ++i) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = VR < 32 ? o[e / 2][i + 8 * (e % 2)] : o[b + B * e][i];
        if (element(b, i) < D) use(element(b, i), x);
      }
  };
  if (__syncthreads_or(bad)) {                 // values that were left out: NaN for the rows that see them
    for (int key = max(lo0, rlo); key < rhi; ++key) {
      const int k0 = key / KT * KT;
      if (!(k0 < alo || k0 + KT > ahi)) continue;
      int slot;
      const int e = place(key, slot);
      const uint8_t* vp = base + (int64_t)(pg[e] & 0x7FFFFFFF) * a.cb + (uint32_t)slot * cn + D;
      const bool all = !(fabsf(ps[e].w) <= 1.f);
#pragma unroll
      for (int q = 0; q < ND; ++q)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          uint32_t z = all;
          if constexpr (CT == SDC_CACHE_E4M3) z |= (uint32_t)((vp[min(element(q, i), D - 1)] & 0x7F) == 0x7F);
          o[q][i] = z ? __builtin_nanf("") : o[q][i];
        }
    }
  }
  l = over_halves_sum(l);
  const Row r = row_of();
  if (!r.live) return;
  if (t.nsp == 1) {
    // (a row with keys whose scores are all -inf: 0 / 0)
    const int64_t p = t.p0 + r.tok;
    const bool any = min(p + 1, a.maxlen) > max(p - a.window + 1, (int64_t)0);
    const float half = ve == 0 ? 1.f : __builtin_amdgcn_exp2f(0.5f * (float)ve), f = any ? half / l : 0.f;
    each([&](int d, f32x4 x) { write_four(a, r.token, r.head, d, x * f, half); });
    if (a.lse && h == 0) a.lse[r.token * a.slt + r.head] = any ? (m + log2f(l) - BIAS) * LN2 : NEG_INF;
  } else {
    float* rec = sp.part + ((int64_t)tile * sp.S + s) * TALL * (D + HEAD);
    if (h == 0) *reinterpret_cast<f32x4*>(rec + HEAD * r.row) = f32x4{m + (float)ve, m, l * 0x1p-13f, 0.f};
    each([&](int d, f32x4 x) { *reinterpret_cast<f32x4*>(rec + HEAD * TALL + r.row * D + d) = x * 0x1p-13f; });
  }
}

// Lanes that join a row: 4 elements each, a power of two.
__host__ __device__ constexpr int join_lanes(int D) { return D <= 64 ? 16 : D <= 128 ? 32 : 64; }

// The parts joined, in their order: a wave for some heads of a token.  `all`: every token of the call; else those of the
// requests that kv_attend_rows takes beside chunks.
__global__ __launch_bounds__(256) void kv_attend_join(AttendArgs a, Split rows, Split tiles, int all) {
  const int lane = threadIdx.x & 63, D = a.D, LG = join_lanes(D), per = 64 / LG, waves = (a.Hq + per - 1) / per;
  const int64_t id = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), k = id / waves;
  const int head = (int)(id - k * waves) * per + lane / LG, hd = head % a.G, d = 4 * (lane % LG);
  Tile t;
  Request rq;
  int64_t token = k, first;
  if (all) {
    if (token >= a.st.T) return;
    t.r = sdc_find_request(a.st, token, 1, 0, rq, first);
    if (t.r < 0 || t.r >= a.st.R) return;
    if (token >= rq.q1) return;
  } else {
    t.r = (int)(k / tiles.few);
    if (t.r >= a.st.R) return;
    rq = sdc_request(a.st, t.r);
    token = rq.q0 + (k - (int64_t)t.r * tiles.few);
    if (rq.q1 - rq.q0 > tiles.few || token >= rq.q1) return;
  }
  const Split& sp = tiles.few && rq.q1 - rq.q0 > tiles.few ? tiles : rows;
  const int tt = (int)(token - rq.q0) / sp.TB, tok = (int)(token - rq.q0) - tt * sp.TB;
  t.hk = head / a.G;
  t.hb = hd / sp.GB;
  t.tok0 = rq.q0 + (int64_t)tt * sp.TB;
  find_keys(a, sp, rq, t);
  if (t.nsp < 2) return;
  const int row = tok * sp.GB + hd - t.hb * sp.GB;
  first = sp.slots ? (int64_t)t.r * sp.slots : (int64_t)((uint32_t)a.st.qsl[t.r] / (uint32_t)sp.TB) + t.r;
  const int64_t tile = ((first + tt) * a.Hkv + t.hk) * sp.NHB + t.hb, size = (int64_t)sp.rows * (D + HEAD);
  const float* rec = sp.part + tile * sp.S * size;
  if (head >= a.Hq || d >= D) return;
  const float* begin = rec + HEAD * row;
  const float* v = rec + HEAD * sp.rows + row * D + d;
  float m = M0, ml = M0, l = 0.f;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;                         // parts whose loads are on their way at once
  for (int b = 0; b < t.nsp; b += U) {
    f32x4 w[U], y[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t at = min(b + i, t.nsp - 1) * size;
      w[i] = *reinterpret_cast<const f32x4*>(begin + at);
      y[i] = *reinterpret_cast<const f32x4*>(v + at);
    }
    float mn = m, mln = ml;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      mn = fmaxf(mn, w[i][0]);
      mln = fmaxf(mln, w[i][1]);
    }
    x *= __builtin_amdgcn_exp2f(m - mn);
    l *= __builtin_amdgcn_exp2f(ml - mln);
    m = mn;
    ml = mln;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (b + i < t.nsp) {
        x += __builtin_amdgcn_exp2f(w[i][0] - m) * y[i];
        l = fmaf(__builtin_amdgcn_exp2f(w[i][1] - ml), w[i][2], l);
      }
  }
  write_row(a, t, tok, token, head, d, ml, m - ml, l, x, 0.f);
}

// The tiles and parts of a call, from its sizes alone.
struct Plan {
  Split rows, tiles;
  bool tall;                                   // kv_attend_tiles takes the requests of more than tiles.few tokens
};
constexpr int64_t CROSS = 640000000;           // small tiles x their keys x head size from which large ones are faster
// Beside chunks, kv_attend_rows takes requests of up to so many of its tiles: with 1 / 2 / 4, 32 sequences of 6 tokens behind
// 16k keys 518 / 270 / 272 us, 64 of 16 tokens behind 8k 460 / 460 / 424, 32 decoding beside a chunk of 2048 205 / 215 / 261.
constexpr int FEW = 2;
Split split_of(int rows, int64_t G, int64_t N) {
  Split sp{};
  sp.rows = rows;
  sp.GB = (int)std::min<int64_t>(G, rows);
  sp.NHB = (int)sdc_cdiv(G, rows);
  sp.TB = std::max(1, rows / sp.GB);
  sp.div = N == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + N - 1) / N);
  return sp;
}
// Parts of at least `least` keys, as many as bring `busy` tiles to `want` workgroups; no part has more pages than a
// workgroup's table.
void cut(Split& sp, int64_t busy, int64_t want, int64_t least, int64_t keys, int64_t N) {
  const int64_t most = std::min<int64_t>(16384, std::max<int64_t>(128, (MAXP - 2) * N / 128 * 128));
  sp.C = (int)std::min(least, most);
  keys += 31;
  const int64_t s = std::min(want / std::max<int64_t>(1, busy), keys / sp.C);
  // (a tile's keys over S parts, rounded up to 128, must stay within `most`)
  sp.S = (int)std::max<int64_t>({1, s, sdc_cdiv(keys, most)});
}
// The keys a query sees at most: without a window, or with one so wide that sums with it could pass 64 bits, more than any
// length.
int64_t seen(int64_t window) {
  constexpr int64_t all = (int64_t)1 << 40;
  return window > 0 ? std::min(window, all) : all;
}
Plan plan(int64_t T, int64_t R, int64_t Hkv, int64_t G, int64_t D, int64_t N, int64_t max_len, int64_t window) {
  Plan p{};
  // keys a tile's rows can see together
  auto keys = [&](const Split& sp) { return std::min(max_len, seen(window) + sp.TB); };
  p.rows = split_of(ROWS, G, N);
  p.tiles = split_of(32 * tall_waves(D), G, N);
  // One round of the workgroups that a lane's registers leave room for, two a CU: 64 sequences of 512-2048 tokens 39 us,
  // four of 100-131k 181 us, 32 of 1000-4000 with their append 51 us (three rounds: 48, 192 and 56).  Parts of fewer than 512
  // keys cost more to join than they save.
  constexpr int64_t resident = 512;
  // More tokens than requests: some have a chunk.  The tiles of 16 rows read every key anew, those of 256 cost two more
  // launches and fill the chip later: a chunk behind 4096 keys, 32 heads, 127 / 505 / 1009 / 2017 tokens in small and in large
  // tiles, heads of 128: 38 and 50 / 108 and 102 / 219 and 145 / 469 and 242 us, heads of 64: 27 and 38 / 56 and 74 / 108 and
  // 106 / 224 and 180 us.
  const int64_t small = (T / p.rows.TB + R) * Hkv * p.rows.NHB;
  p.tall = T > R && T > FEW * p.rows.TB && small * keys(p.rows) >= CROSS / D;
  if (p.tall) {
    p.tiles.few = p.rows.TB * FEW;
    p.rows.slots = FEW;
    p.tiles.tiles = (T / p.tiles.TB + R + 1) * Hkv * p.tiles.NHB;
    cut(p.tiles, (T / p.tiles.TB + 1) * Hkv * p.tiles.NHB, 512, 512, keys(p.tiles), N);
    p.rows.tiles = R * FEW * Hkv * p.rows.NHB;
    cut(p.rows, R * Hkv * p.rows.NHB, resident, 512, keys(p.rows), N);
  } else {
    p.rows.tiles = (T / p.rows.TB + R + 1) * Hkv * p.rows.NHB;
    cut(p.rows, std::min(T, T / p.rows.TB + R) * Hkv * p.rows.NHB, resident, 512, keys(p.rows), N);
  }
  return p;
}
int64_t part_bytes(const Split& sp, int64_t D) { return sp.S <= 1 ? 0 : sp.tiles * sp.S * sp.rows * (D + HEAD) * 4; }

int launch_join(const AttendArgs& a, const Plan& p, hipStream_t stream) {
  if (p.rows.S == 1 && p.tiles.S <= 1) return SDC_OK;
  const bool all = !p.tall || p.tiles.S > 1;
  const int64_t waves = sdc_cdiv(a.Hq, 64 / join_lanes(a.D));
  const int64_t blocks = sdc_cdiv((all ? a.st.T : (int64_t)a.st.R * p.tiles.few) * waves, 4);
  if (blocks > 0x7FFFFFFF) return SDC_EUNSUPPORTED;
  if (blocks == 0) return SDC_OK;
  SdcProf prof("kv_attend_join", stream);
  hipLaunchKernelGGL(kv_attend_join, dim3((unsigned)blocks), dim3(256), 0, stream, a, p.rows, p.tiles, (int)all);
  SDC_LAUNCH_CHECK();
  return SDC_OK;
}
template <int CT, int DP>
int launch_rows(const AttendArgs& a, const Split& sp, hipStream_t stream) {
  const int64_t blocks = sp.tiles * sp.S;
  if (blocks > 0x7FFFFFFF) return SDC_EUNSUPPORTED;
  if (blocks == 0) return SDC_OK;
  SdcProf prof("kv_attend", stream);
  const dim3 grid((unsigned)blocks), threads(256);
  if (a.st.N % 16 == 0) hipLaunchKernelGGL((kv_attend_rows<CT, DP, 16>), grid, threads, 0, stream, a, sp);
  else hipLaunchKernelGGL((kv_attend_rows<CT, DP, 1>), grid, threads, 0, stream, a, sp);
  SDC_LAUNCH_CHECK();
  return SDC_OK;
}
template <int CT>
int run_rows(const AttendArgs& a, const Split& sp, hipStream_t stream) {
  if (a.D <= 64) return launch_rows<CT, 64>(a, sp, stream);
  return a.D <= 128 ? launch_rows<CT, 128>(a, sp, stream) : launch_rows<CT, 256>(a, sp, stream);
}
template <int CT, int DP>
int launch_tiles(const AttendArgs& a, const Split& sp, hipStream_t stream) {
  const int64_t blocks = sp.tiles * sp.S;
  if (blocks > 0x7FFFFFFF) return SDC_EUNSUPPORTED;
  SdcProf prof("kv_attend_tiles", stream);
  const dim3 grid((unsigned)blocks), threads(64 * tall_waves(DP));
  if (a.st.N % 16 == 0) hipLaunchKernelGGL((kv_attend_tiles<CT, DP, 16>), grid, threads, 0, stream, a, sp);
  else if (a.st.N % 4 == 0) hipLaunchKernelGGL((kv_attend_tiles<CT, DP, 4>), grid, threads, 0, stream, a, sp);
  else hipLaunchKernelGGL((kv_attend_tiles<CT, DP, 1>), grid, threads, 0, stream, a, sp);
  SDC_LAUNCH_CHECK();
  return SDC_OK;
}
template <int CT>
int run_tiles(const AttendArgs& a, const Split& sp, hipStream_t stream) {
  if (a.D <= 64) return launch_tiles<CT, 64>(a, sp, stream);
  if (a.D <= 96) return launch_tiles<CT, 96>(a, sp, stream);
  return a.D <= 128 ? launch_tiles<CT, 128>(a, sp, stream) : launch_tiles<CT, 256>(a, sp, stream);
}

int run(int cache, const AttendArgs& a, hipStream_t stream) {
  const int64_t blocks = sdc_cdiv(a.st.T * a.Hq, 4);
  if (blocks > 0x7FFFFFFF) return SDC_EUNSUPPORTED;
  SdcProf prof("kv_attend", stream);
  if (cache == SDC_CACHE_E4M3) hipLaunchKernelGGL((kv_attend_any<SDC_CACHE_E4M3>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((kv_attend_any<SDC_CACHE_I8>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  SDC_LAUNCH_CHECK();
  return SDC_OK;
}

}  // namespace

extern "C" int64_t sdc_kv_attend_workspace(int64_t T, int64_t R, int64_t Hq, int64_t Hkv, int64_t D, int64_t N,
                                           int64_t max_len, int64_t window) {
  if (T < 1 || R < 0 || Hkv < 1 || Hq < Hkv || D < 1 || N < 1 || max_len < 0 || T > 0x3FFFFFFF || R > 0x0FFFFFFF) return 0;
  const Plan p = plan(T, R, Hkv, Hq / Hkv, D, N, max_len, window);
  return part_bytes(p.rows, D) + part_bytes(p.tiles, D);
}

extern "C" int sdc_kv_attend(int dtype, int cache, const void* q, int64_t sqt, int64_t sqh, int64_t sqd, void* o,
                             int64_t sot, int64_t soh, int64_t sod, float* lse, int64_t slt, int64_t T, int64_t Hq,
                             int64_t D, const void* kv, int64_t cb, int64_t ch, int64_t cn, int64_t NB, int64_t Hkv,
                             int64_t N, const float* scales, int64_t sb, int64_t sh, const int32_t* qsl,
                             const int32_t* seq_lens, int64_t R, const int32_t* bt, int64_t sbt, int64_t W, float scale,
                             int64_t window, int64_t max_len, void* workspace, int64_t workspace_bytes,
                             hipStream_t stream) {
  SDC_CLEAR_ERRORS();
  if ((dtype != SDC_BF16 && dtype != SDC_FP16) || (cache != SDC_CACHE_E4M3 && cache != SDC_CACHE_I8) || T < 0 ||
      Hq < 1 || Hkv < 1 || Hq % Hkv || D < 1 || D > ANY_D || NB < 1 || N < 1 || N > 65536 || R < 0 || W < 0 || window < 0 ||
      max_len < 0 || max_len > W * N || !std::isfinite(scale))
    return SDC_EINVAL;
  if (T == 0) return SDC_OK;
  if (!q || !o || !kv || !scales || !qsl || (R && !seq_lens) || (R && W && !bt)) return SDC_EINVAL;
  if (T > 0x3FFFFFFF || R > 0x0FFFFFFF || Hq > 65536 || W * N > 0x7FFFFFFF || max_len > 0x3FFFFFFF)
    return SDC_EUNSUPPORTED;                    // (numbers of keys are added up in 32 bits)
  AttendArgs a{};
  a.st = PagedStep{qsl, seq_lens, bt, sbt, W, NB, T, (int)R, (int)N};
  a.q = (const uint16_t*)q; a.o = (uint16_t*)o; a.lse = lse;
  a.sqt = sqt; a.sqh = sqh; a.sqd = sqd; a.sot = sot; a.soh = soh; a.sod = sod; a.slt = slt;
  a.kv = (const uint8_t*)kv; a.cb = cb; a.ch = ch; a.cn = cn;
  a.scales = scales; a.sb = sb; a.sh = sh;
  a.scale = scale * LOG2E;
  a.maxlen = max_len;
  a.window = seen(window);
  a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.G = (int)(Hq / Hkv); a.D = (int)D; a.fp16 = dtype == SDC_FP16;
  // the tiled kernels read 16 codes at a time, and divide by N by a product (exact up to this many slots)
  if (D % 16 == 0 && N <= 4096 && cn >= 0 && cn < (1 << 19) && ((uintptr_t)kv | (uintptr_t)(cb | ch | cn)) % 16 == 0) {
    Plan p = plan(T, R, Hkv, a.G, D, N, max_len, window);
    const int64_t first = part_bytes(p.rows, D), need = first + part_bytes(p.tiles, D);
    if (workspace_bytes < need || (need && !workspace)) return SDC_EWORKSPACE;
    p.rows.part = (float*)workspace;
    p.tiles.part = (float*)((uint8_t*)workspace + first);
    int rc = SDC_OK;
    if (p.tall)
      rc = cache == SDC_CACHE_E4M3 ? run_tiles<SDC_CACHE_E4M3>(a, p.tiles, stream) : run_tiles<SDC_CACHE_I8>(a, p.tiles, stream);
    if (rc == SDC_OK)
      rc = cache == SDC_CACHE_E4M3 ? run_rows<SDC_CACHE_E4M3>(a, p.rows, stream) : run_rows<SDC_CACHE_I8>(a, p.rows, stream);
    return rc == SDC_OK ? launch_join(a, p, stream) : rc;
  }
  return run(cache, a, stream);
}
