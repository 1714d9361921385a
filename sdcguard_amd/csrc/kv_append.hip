// Appending a step's keys and values to a paged cache, the keys rotated by position and both quantized on the way (and
// the queries rotated beside them): one launch.
//
// A cache of 8-bit codes has one scale S for the keys and one for the values of each (page, kv head).  The scale is
// the smallest power of two with max |x| <= Q S (Q = 448 for e4m3, 127 for int8) over what was appended since the page's
// first slot was last written; powers of two, because when later tokens need a larger scale the codes already in the
// page are rescaled, and then e4m3 codes only change where they become subnormal (a page of 16 tokens would otherwise
// be rounded up to 16 times).  A workgroup takes one page that the step writes to and four kv heads, a wave each: the
// largest magnitudes (of the page's new tokens, rotated), the scales, the rescaled old codes where the scale grew, the
// new codes.  Nobody else writes to that (page, head), so there are no atomics and no order to depend on.
//
// A page that the step starts anew (its slot 0 is among the new tokens) ignores the old scale and codes.  Values that
// are not finite take no part in the scale; e4m3 keeps them as NaN, int8, which has no such code, makes the scale NaN.
#include <float.h>

#include <algorithm>

#include "common.h"
#include "paged.h"
#include "profile.h"
#include "rope.h"

namespace {

constexpr int TAB = 1024, WIDE = 4096;         // (cos, sin) pairs a workgroup holds; of large pages
constexpr int QTOK = 4;                        // tokens a workgroup of the queries' rotation takes

struct AppendArgs {
  PagedStep st;
  const void* k; const void* v; const void* q; void* qo;
  int64_t skt, skh, skd, svt, svh, svd, sqt, sqh, sqd, sot, soh, sod;
  uint8_t* kv;                                 // bytes
  int64_t cb, ch, cn;                          // page, head and slot strides of the cache, in bytes
  float* scales;
  int64_t sb, sh;                              // page and head strides of the scales (keys, then values)
  const void* pos;                             // (T) positions to rotate by; null: the tokens' own
  const double* turns;
  double m;
  int Hkv, Hq, D, rot, inter, pos32, items, hgroups;
  int qheads;                                  // query heads of a workgroup
};

__device__ __forceinline__ double position_of(const AppendArgs& a, int64_t t, int64_t own) {
  if (!a.pos) return (double)own;
  return a.pos32 ? (double)((const int32_t*)a.pos)[t] : (double)((const int64_t*)a.pos)[t];
}

// the smallest power of two whose product with the largest code holds amax (at most 2^120 for e4m3 and 2^122 for int8, of
// values next to 2^128: reciprocals are normal numbers), 2^-126 at least
template <int CT>
__device__ __forceinline__ float scale_for(float amax) {
  if (amax == 0.f) return 0x1p-126f;
  int e;
  const float f = frexpf(amax, &e);                                     // f in [0.5, 1)
  constexpr float top = CT == SDC_CACHE_E4M3 ? 0.875f : 127.f / 128.f;  // 448 / 2^9, 127 / 2^7
  e += (f > top) - (CT == SDC_CACHE_E4M3 ? 9 : 7);
  return ldexpf(1.f, max(e, -126));
}

// x / S: a power of two's reciprocal is exact (S may be another quantizer's, of any value)
struct Divide {
  float s, inv;
  bool pow2;
  __device__ explicit Divide(float v) : s(v), inv(1.f / v), pow2((__float_as_uint(v) & 0x007FFFFFu) == 0) {}
  __device__ __forceinline__ float operator()(float x) const { return pow2 ? x * inv : x / s; }
};

template <int CT>
__device__ __forceinline__ uint32_t code_of(float x) {                  // |x| <= the largest code, or not finite
  if constexpr (CT == SDC_CACHE_E4M3) {
    const uint32_t c = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, 0.f, 0, false) & 0xFFu;
    return fabsf(x) <= 448.f ? c : ((__float_as_uint(x) >> 24) & 0x80u) | 0x7Fu;
  } else {
    return (uint32_t)(int)fminf(fmaxf(rintf(x), -127.f), 127.f) & 0xFFu;
  }
}
template <int CT>
__device__ __forceinline__ float value_of(uint32_t c) {
  if constexpr (CT == SDC_CACHE_E4M3) return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
  else return (float)(int8_t)c;
}

// Four codes of values that are finite and lie within the codes' range.
template <int CT>
__device__ __forceinline__ uint32_t codes4(const float* x, float inv) {
  if constexpr (CT == SDC_CACHE_E4M3) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, lo, true);
  } else {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = (uint32_t)(int)rintf(x[i] * inv);
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[3], c[2], 0x0C0C0400u), __builtin_amdgcn_perm(c[1], c[0], 0x0C0C0400u),
                                 0x05040100u);
  }
}

// n (8 or 1) codes at p; plain: the values are finite, and so large at most that the scale, a power of two, holds them
template <int CT, int UP>
__device__ __forceinline__ void store_codes(uint8_t* p, const float* x, const Divide& d, bool plain) {
  if constexpr (UP == 8) {
    if (plain) {
      *reinterpret_cast<u32x2*>(p) = u32x2{codes4<CT>(x, d.inv), codes4<CT>(x + 4, d.inv)};
      return;
    }
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      w[i] = code_of<CT>(d(x[4 * i])) | code_of<CT>(d(x[4 * i + 1])) << 8 | code_of<CT>(d(x[4 * i + 2])) << 16 |
             code_of<CT>(d(x[4 * i + 3])) << 24;
    *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
  } else {
    *p = (uint8_t)code_of<CT>(d(x[0]));
  }
}

// the codes of one row (n of them at p) from scale `from` to scale d.s
template <int CT, int UP>
__device__ __forceinline__ void rescale(uint8_t* p, float ratio) {
  if constexpr (UP == 8) {
    u32x2 w = *reinterpret_cast<u32x2*>(p);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t o = 0;
#pragma unroll
      for (int b = 0; b < 32; b += 8) o |= code_of<CT>(value_of<CT>((w[i] >> b) & 0xFFu) * ratio) << b;
      w[i] = o;
    }
    *reinterpret_cast<u32x2*>(p) = w;
  } else {
    *p = (uint8_t)code_of<CT>(value_of<CT>(*p) * ratio);
  }
}

__device__ __forceinline__ void finite_max(float x, float& amax, bool& bad) {
  const float f = fabsf(x);
  if (f <= FLT_MAX) amax = fmaxf(amax, f);
  else bad = true;
}

// Two results of each wave joined over the waves that share a head (by all threads of the workgroup).
template <class T, class F>
__device__ __forceinline__ void over_waves(T& x, T& y, F join) {
  __shared__ T all[4][2];
  __syncthreads();
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    all[w][0] = x;
    all[w][1] = y;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x = join(x, all[i][0]);
    y = join(y, all[i][1]);
  }
}
__device__ __forceinline__ void finish_maxima(float& mk, float& mv, bool& bk, bool& bv) {
  over_waves(mk, mv, [](float x, float y) { return fmaxf(x, y); });
  int ik = bk, iv = bv;
  over_waves(ik, iv, [](int x, int y) { return x | y; });
  bk = ik != 0;
  bv = iv != 0;
}

// A unit of a key and of its value into the slot's row.
template <int DT, int CT, int UP>
__device__ __forceinline__ void put(uint8_t* row, RopeUnit rk, RopeUnit rv, int D, const float* x, const float* y,
                                    const Divide& dk, const Divide& dv, bool plain) {
  if constexpr (CT == SDC_CACHE_16) {
    typedef typename RopeElem<DT>::T E;
    sdc_store_unit<DT, UP>((E*)row, 1, rk, D, x);
    sdc_store_unit<DT, UP>((E*)row + D, 1, rv, D, y);
  } else {
    store_codes<CT, UP>(row + rk.c0, x, dk, plain);
    if (UP == 8 || rk.c1 < D) store_codes<CT, UP>(row + rk.c1, x + UP, dk, plain);
    store_codes<CT, UP>(row + D + rv.c0, y, dv, plain);
    if (UP == 8 || rv.c1 < D) store_codes<CT, UP>(row + D + rv.c1, y + UP, dv, plain);
  }
}

// A page's largest magnitudes, scales and old codes: from the largest finite magnitudes of the new keys and values (of the
// whole wave) and whether any is not finite, the scales to write with.  ok, ov: the page's scales before.
// `first`, `step`: the caller's share of the old codes.
template <int CT, int UP>
__device__ __forceinline__ void settle(const AppendArgs& a, int first, int step, uint8_t* base, float* sc, int s0, int n, float mk, float mv, bool bk,
                                       bool bv, float ok, float ov, float& sk, float& sv) {
  const int N = a.st.N, D = a.D;
  sk = scale_for<CT>(mk);
  sv = scale_for<CT>(mv);
  if (CT == SDC_CACHE_I8 && bk) sk = __builtin_nanf("");
  if (CT == SDC_CACHE_I8 && bv) sv = __builtin_nanf("");
  if (s0 > 0) {
    sk = sk > ok ? sk : (sk == sk ? ok : sk);                           // (a scale that is NaN stays)
    sv = sv > ov ? sv : (sv == sv ? ov : sv);
    const float rk = ok / sk, rv = ov / sv;
    const bool gk = ok < sk, gv = ov < sv;
    if (gk || gv) {
      constexpr int C = UP == 8 ? 8 : 1;
      const int nc = D / C;
      for (int i = first; i < (N - n) * nc; i += step) {
        int s = i / nc;
        const int c = (i - s * nc) * C;
        if (s >= s0) s += n;
        uint8_t* p = base + (int64_t)s * a.cn + c;
        if (gk) rescale<CT, UP>(p, rk);
        if (gv) rescale<CT, UP>(p + D, rv);
      }
    }
  }
  if (first == 0) {
    sc[0] = sk;
    sc[1] = sv;
  }
}

// SHARE waves of the workgroup (1, or all 4) on one head.
template <int DT, int CT, int UP, int SHARE>
__device__ __forceinline__ void append_page(const AppendArgs& a, int item, int hg, float2* tab) {
  typedef typename RopeElem<DT>::T E;
  constexpr int HOLD = SHARE > 1 ? WIDE : TAB;
  const PagedStep& st = a.st;
  const int N = st.N, D = a.D, tid = threadIdx.x, lane = tid & 63;
  const int P = a.rot / 2, nu = sdc_units(D, UP);
  const double turn = P ? a.turns[tid % P] : 0.0;                       // (on its way while the request is found)
  Request rq;
  int64_t first;
  const int r = sdc_find_request(st, item, N, 2, rq, first);
  if (r < 0 || r >= st.R) return;
  const int64_t pos0 = max(rq.len - (rq.q1 - rq.q0), (int64_t)0);
  const int64_t w = pos0 / N + (item - first);
  const int64_t lo = max(pos0, w * N), hi = min(rq.len, (w + 1) * N);
  if (lo >= hi || w >= st.W) return;
  const int32_t page = st.bt[r * st.sbt + w];
  const int n = (int)(hi - lo), s0 = (int)(lo - w * N);
  const int64_t t0 = rq.q1 - rq.len + lo;
  const int h = SHARE == 4 ? hg : hg * 4 + (tid >> 6);
  const bool live = h < a.Hkv;
  const int mine = SHARE == 4 ? tid : lane, step = 64 * SHARE;          // the wave's part of the head's units
  const E* kp = (const E*)a.k + (live ? h : 0) * a.skh;
  const E* vp = (const E*)a.v + (live ? h : 0) * a.svh;
  const int units = n * nu;

  // Up to HELD units a lane stay in registers, all loads of keys and values on their way at once (a token of 64 sequences each:
  // 6.4 us, 12 with the two passes below, which larger pages take).
  constexpr int HELD = 2;
  if (SHARE == 1 || (units <= step * HELD && n * P <= HOLD)) {           // (a wave alone: always, by launch()'s choice)
    float x[HELD][2 * UP], y[HELD][2 * UP];
    RopeUnit ru[HELD], rv[HELD];
    int tok[HELD];
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      const int i = mine + step * j;
      const bool on = live && i < units;
      tok[j] = on ? i / nu : -1;
      const int t = on ? tok[j] : 0, u = on ? i - t * nu : 0;
      ru[j] = sdc_unit<UP>(u, a.rot, a.inter);
      rv[j] = sdc_unit<UP>(u, 0, 0);
      if (on) {
        sdc_load_unit<DT, UP>(kp + (t0 + t) * a.skt, a.skd, ru[j], D, x[j]);
        sdc_load_unit<DT, UP>(vp + (t0 + t) * a.svt, a.svd, rv[j], D, y[j]);
      } else {
#pragma unroll
        for (int e = 0; e < 2 * UP; ++e) x[j][e] = y[j][e] = 0.f;
      }
    }
    if (page < 0 || page >= st.NB) return;
    uint8_t* base = a.kv + (int64_t)page * a.cb + (live ? h : 0) * a.ch;
    float* sc = a.scales + (int64_t)page * a.sb + (live ? h : 0) * a.sh;
    float ok = 0.f, ov = 0.f;
    if (CT != SDC_CACHE_16 && s0 > 0) {
      ok = sc[0];
      ov = sc[1];
    }
    for (int i = tid; i < n * P; i += 256) {
      const int t = i / P;
      tab[i] = sdc_turn(position_of(a, t0 + t, lo + t), i < 256 || 256 % P == 0 ? turn : a.turns[i - t * P], a.m);
    }
    __syncthreads();
    // the largest magnitudes as bits, of which those of infinities and NaN are the largest
    uint32_t uk = 0, uv = 0;
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      if (tok[j] >= 0) sdc_rotate_unit<UP>(x[j], ru[j], a.inter, tab + tok[j] * P);
#pragma unroll
      for (int e = 0; e < 2 * UP; ++e) {
        uk = max(uk, __float_as_uint(x[j][e]) & 0x7FFFFFFFu);
        uv = max(uv, __float_as_uint(y[j][e]) & 0x7FFFFFFFu);
      }
    }
    float sk = 1.f, sv = 1.f;
    bool plain = false;
    if constexpr (CT != SDC_CACHE_16) {
      uk = wave_max_u32_dpp(uk);
      uv = wave_max_u32_dpp(uv);
      if constexpr (SHARE > 1) over_waves(uk, uv, [](uint32_t x, uint32_t y) { return max(x, y); });
      float mk = __uint_as_float(uk), mv = __uint_as_float(uv);
      bool bk = false, bv = false;
      plain = max(uk, uv) < 0x7F800000u;
      if (!plain) {
        mk = mv = 0.f;
#pragma unroll 1
        for (int j = 0; j < HELD; ++j)
#pragma unroll
          for (int e = 0; e < 2 * UP; ++e) {
            finite_max(j ? x[1][e] : x[0][e], mk, bk);
            finite_max(j ? y[1][e] : y[0][e], mv, bv);
          }
        mk = wave_max_f32_dpp(mk);
        mv = wave_max_f32_dpp(mv);
        bk = __any(bk);
        bv = __any(bv);
        if constexpr (SHARE > 1) finish_maxima(mk, mv, bk, bv);
      }
      if (!live) return;
      settle<CT, UP>(a, mine, step, base, sc, s0, n, mk, mv, bk, bv, ok, ov, sk, sv);
    }
    const Divide dk(sk), dv(sv);
    plain = plain && dk.pow2 && dv.pow2;
#pragma unroll
    for (int j = 0; j < HELD; ++j)
      if (tok[j] >= 0) put<DT, CT, UP>(base + (int64_t)(s0 + tok[j]) * a.cn, ru[j], rv[j], D, x[j], y[j], dk, dv, plain);
    return;
  }

  if (page < 0 || page >= st.NB) return;
  const int rows = P ? min(n, HOLD / P) : n;                             // tokens whose angles are held at once
  uint8_t* base = a.kv + (int64_t)page * a.cb + (live ? h : 0) * a.ch;
  auto angles = [&](int first) {                                        // by the whole workgroup
    const int m = min(rows, n - first);
    __syncthreads();
    for (int i = tid; i < m * P; i += 256) {
      const int t = i / P;
      tab[i] = sdc_turn(position_of(a, t0 + first + t, lo + first + t), a.turns[i - t * P], a.m);
    }
    __syncthreads();
    return m;
  };
  auto key = [&](int first, int t, int u, float* x) {
    const RopeUnit ru = sdc_unit<UP>(u, a.rot, a.inter);
    sdc_load_unit<DT, UP>(kp + (t0 + first + t) * a.skt, a.skd, ru, D, x);
    sdc_rotate_unit<UP>(x, ru, a.inter, tab + t * P);
    return ru;
  };
  auto value = [&](int first, int t, int u, float* x) {
    const RopeUnit ru = sdc_unit<UP>(u, 0, 0);
    sdc_load_unit<DT, UP>(vp + (t0 + first + t) * a.svt, a.svd, ru, D, x);
    return ru;
  };

  float sk = 1.f, sv = 1.f;
  if constexpr (CT != SDC_CACHE_16) {
    // (read before the barriers behind which one of the head's waves writes them)
    float* sc = a.scales + (int64_t)page * a.sb + (live ? h : 0) * a.sh;
    const float ok = s0 > 0 ? sc[0] : 0.f, ov = s0 > 0 ? sc[1] : 0.f;
    float mk = 0.f, mv = 0.f;
    bool bk = false, bv = false;
    for (int first = 0; first < n; first += rows) {
      const int m = angles(first);
      for (int i = mine; live && i < m * nu; i += step) {
        const int t = i / nu, u = i - t * nu;
        float x[2 * UP], y[2 * UP];
        key(first, t, u, x);
        value(first, t, u, y);
#pragma unroll
        for (int e = 0; e < 2 * UP; ++e) {
          finite_max(x[e], mk, bk);
          finite_max(y[e], mv, bv);
        }
      }
    }
    mk = wave_max_f32_dpp(mk);
    mv = wave_max_f32_dpp(mv);
    bk = __any(bk);
    bv = __any(bv);
    if constexpr (SHARE > 1) finish_maxima(mk, mv, bk, bv);
    if (live) {
      settle<CT, UP>(a, mine, step, base, sc, s0, n, mk, mv, bk, bv, ok, ov, sk, sv);
    }
  }
  const Divide dk(sk), dv(sv);
  for (int first = 0; first < n; first += rows) {
    const int m = (CT != SDC_CACHE_16 && rows >= n) ? n : angles(first);
    for (int i = mine; live && i < m * nu; i += step) {
      const int t = i / nu, u = i - t * nu;
      float x[2 * UP], y[2 * UP];
      const RopeUnit rk = key(first, t, u, x), rv = value(first, t, u, y);
      put<DT, CT, UP>(base + (int64_t)(s0 + first + t) * a.cn, rk, rv, D, x, y, dk, dv, false);
    }
  }
}

// The queries of QTOK tokens, rotated; those past the last request are written as zeros.  A thread's first unit is on its
// way while the tokens' requests are found.
template <int DT, int UP>
__device__ __forceinline__ void rotate_queries(const AppendArgs& a, int64_t block, int h0, float2* tab) {
  typedef typename RopeElem<DT>::T E;
  constexpr int HELD = 1;
  const int tid = threadIdx.x, P = a.rot / 2, nu = sdc_units(a.D, UP);
  const int TB = P ? min(QTOK, TAB / P) : QTOK;
  __shared__ int64_t own[QTOK];                                         // the tokens' positions in their requests
  for (int64_t t0 = block * QTOK, te = min(t0 + QTOK, a.st.T); t0 < te; t0 += TB) {
    const int nt = (int)min((int64_t)TB, te - t0), nh = min(a.qheads, a.Hq - h0), all = nt * nh * nu;
    struct Unit {
      int t, h;
      RopeUnit ru;
      float x[2 * UP];
    };
    auto load = [&](int i, Unit& u) {
      const int th = i / nu;
      u.t = th / nh;
      u.h = h0 + th - u.t * nh;
      u.ru = sdc_unit<UP>(i - th * nu, a.rot, a.inter);
      sdc_load_unit<DT, UP>((const E*)a.q + (t0 + u.t) * a.sqt + u.h * a.sqh, a.sqd, u.ru, a.D, u.x);
    };
    auto store = [&](Unit& u) {
      sdc_rotate_unit<UP>(u.x, u.ru, a.inter, tab + u.t * P);
      if (own[u.t] < 0) {
#pragma unroll
        for (int e = 0; e < 2 * UP; ++e) u.x[e] = 0.f;
      }
      sdc_store_unit<DT, UP>((E*)a.qo + (t0 + u.t) * a.sot + u.h * a.soh, a.sod, u.ru, a.D, u.x);
    };
    const double turn = P && tid < nt * P ? a.turns[tid % P] : 0.0;
    Unit held[HELD];
#pragma unroll
    for (int j = 0; j < HELD; ++j)
      if (tid + 256 * j < all) load(tid + 256 * j, held[j]);
    __syncthreads();
    for (int t = tid >> 6; t < nt; t += 4) {                            // a wave per token: its request, its position
      Request rq;
      int64_t first, p = -1;
      const int r = sdc_find_request(a.st, t0 + t, 1, 0, rq, first);
      if (r >= 0 && r < a.st.R) p = max(t0 + t - rq.q1 + rq.len, (int64_t)0);
      if ((tid & 63) == 0) own[t] = p;
    }
    __syncthreads();
    for (int i = tid; i < nt * P; i += 256) {
      const int t = i / P;
      tab[i] = sdc_turn(position_of(a, t0 + t, own[t]), i < 256 || 256 % P == 0 ? turn : a.turns[i - t * P], a.m);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < HELD; ++j)
      if (tid + 256 * j < all) store(held[j]);
    for (int i = tid + 256 * HELD; i < all; i += 256) {
      Unit u;
      load(i, u);
      store(u);
    }
  }
}

template <int DT, int CT, int UP, int SHARE>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
  __shared__ float2 tab[SHARE > 1 ? WIDE : TAB];
  const int64_t b = blockIdx.x, pages = (int64_t)a.items * a.hgroups;
  if (b < pages) append_page<DT, CT, UP, SHARE>(a, (int)(b / a.hgroups), (int)(b % a.hgroups), tab);
  else {
    const int groups = (a.Hq + a.qheads - 1) / a.qheads;
    rotate_queries<DT, UP>(a, (b - pages) / groups, (int)((b - pages) % groups) * a.qheads, tab);
  }
}
template <int DT, int CT, int UP>
int launch(AppendArgs a, hipStream_t stream) {
  // four waves share a head where a page holds more units than one keeps in registers (chunks of 50 tokens into pages of 64
  // slots of 128: 10 us, 33 with a wave a head); a workgroup takes up to 1024 units of queries
  const int nu = sdc_units(a.D, UP);
  const bool share = a.st.N * nu > 128;
  a.hgroups = share ? a.Hkv : (int)sdc_cdiv(a.Hkv, 4);
  a.qheads = std::min(std::max(a.Hq, 1), std::max(1, 1024 / (QTOK * nu)));
  const int64_t blocks = (int64_t)a.items * a.hgroups + (a.q ? sdc_cdiv(a.st.T, QTOK) * sdc_cdiv(a.Hq, a.qheads) : 0);
  if (blocks > 0x7FFFFFFF) return SDC_EUNSUPPORTED;
  SdcProf prof("kv_append", stream);
  if (share) hipLaunchKernelGGL((kv_append_kernel<DT, CT, UP, 4>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((kv_append_kernel<DT, CT, UP, 1>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  SDC_LAUNCH_CHECK();
  return SDC_OK;
}

template <int DT, int CT>
int pick(const AppendArgs& a, hipStream_t stream) {
  constexpr int es = CT == SDC_CACHE_16 ? 2 : 1;
  // 16-byte runs of keys, values and queries; 8-element runs of the cache
  uintptr_t in = (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)(2 * (a.skt | a.skh | a.svt | a.svh));
  bool unit = a.skd == 1 && a.svd == 1;
  if (a.q) {
    in |= (uintptr_t)a.q | (uintptr_t)a.qo | (uintptr_t)(2 * (a.sqt | a.sqh | a.sot | a.soh));
    unit = unit && a.sqd == 1 && a.sod == 1;
  }
  const uintptr_t cache = (uintptr_t)a.kv | (uintptr_t)(a.cb | a.ch | a.cn);
  const bool vec = unit && a.D % 16 == 0 && a.rot % 16 == 0 && in % 16 == 0 && cache % (8 * es) == 0;
  return vec ? launch<DT, CT, 8>(a, stream) : launch<DT, CT, 1>(a, stream);
}

template <int DT>
int pick_cache(int cache, const AppendArgs& a, hipStream_t stream) {
  switch (cache) {
    case SDC_CACHE_E4M3: return pick<DT, SDC_CACHE_E4M3>(a, stream);
    case SDC_CACHE_I8: return pick<DT, SDC_CACHE_I8>(a, stream);
    default: return pick<DT, SDC_CACHE_16>(a, stream);
  }
}

}  // namespace

extern "C" int sdc_kv_append(int dtype, int cache, const void* key, int64_t skt, int64_t skh, int64_t skd,
                             const void* val, int64_t svt, int64_t svh, int64_t svd, int64_t T, int64_t Hkv, int64_t D,
                             void* kv, int64_t cb, int64_t ch, int64_t cn, int64_t NB, int64_t N, float* scales,
                             int64_t sb, int64_t sh, const int32_t* qsl, const int32_t* seq_lens, int64_t R,
                             const int32_t* bt, int64_t sbt, int64_t W, const void* positions, int pos_bytes,
                             const double* turns, int64_t rot, int interleaved, double mscale, const void* q,
                             int64_t sqt, int64_t sqh, int64_t sqd, void* q_out, int64_t sot, int64_t soh, int64_t sod,
                             int64_t Hq, hipStream_t stream) {
  SDC_CLEAR_ERRORS();
  if ((dtype != SDC_BF16 && dtype != SDC_FP16) || cache < SDC_CACHE_E4M3 || cache > SDC_CACHE_16 || T < 0 || Hkv < 1 ||
      D < 1 || D > 1024 || NB < 1 || N < 1 || N > 65536 || R < 0 || W < 0 || rot < 0 || rot % 2 || rot > D ||
      (positions && pos_bytes != 4 && pos_bytes != 8) || (q && (Hq < 1 || !q_out)))
    return SDC_EINVAL;
  if (T == 0) return SDC_OK;
  if (!key || !val || !kv || !qsl || (R && !seq_lens) || (R && W && !bt) || (rot && !turns) || (cache != SDC_CACHE_16 && !scales))
    return SDC_EINVAL;
  if (T > 0x3FFFFFFF || R > 0x0FFFFFFF || Hkv * D > 1 << 24 || (q && Hq * D > 1 << 24)) return SDC_EUNSUPPORTED;
  const int64_t es = cache == SDC_CACHE_16 ? 2 : 1;
  AppendArgs a{};
  a.st = PagedStep{qsl, seq_lens, bt, sbt, W, NB, T, (int)R, (int)N};
  a.k = key; a.v = val; a.q = q; a.qo = q_out;
  a.skt = skt; a.skh = skh; a.skd = skd; a.svt = svt; a.svh = svh; a.svd = svd;
  a.sqt = sqt; a.sqh = sqh; a.sqd = sqd; a.sot = sot; a.soh = soh; a.sod = sod;
  a.kv = (uint8_t*)kv; a.cb = cb * es; a.ch = ch * es; a.cn = cn * es;
  a.scales = scales; a.sb = sb; a.sh = sh;
  a.pos = positions; a.pos32 = pos_bytes == 4; a.turns = turns; a.m = mscale;
  a.Hkv = (int)Hkv; a.Hq = (int)Hq; a.D = (int)D; a.rot = (int)rot; a.inter = interleaved != 0;
  // a request of q tokens touches at most q / N + 2 pages (paged.h)
  const int64_t items = T / N + 2 * R;
  if (items > 0x3FFFFFFF) return SDC_EUNSUPPORTED;
  a.items = (int)items;
  return dtype == SDC_BF16 ? pick_cache<SDC_BF16>(cache, a, stream) : pick_cache<SDC_FP16>(cache, a, stream);
}
