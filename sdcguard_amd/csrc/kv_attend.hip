// Attention of a step's queries over a paged cache of 8-bit codes, a scale for the keys and one for the values of each
// (page, kv head): o = sum_j p_j v_j / sum_j p_j over the keys j a query sees (its own position and those before it, the
// last `window` of them), p_j = exp(s_j - max s), s_j = scale q . k_j, k_j = ks[page] kcode_j, v_j = vs[page] vcode_j;
// lse = max s + log sum p.  A query that sees no key gets zeros and lse = -inf; a key in a page outside the cache
// counts as NaN.
//
// The path for any head size and alignment: a wave per (query token, head), a key per lane for the products, then the
// head's elements over the lanes for the sum of the values.
#include <algorithm>

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

// The work of the tiled kernels: tiles of TB query tokens x GB heads of one kv head, whose keys are cut into at most S
// parts of C keys, one part a workgroup.  part: (tile, part) records of ROWS (maximum, sum) pairs and ROWS x D sums.
struct Split {
  int64_t tiles;
  int TB, GB, NHB, C, S;
  uint32_t div;                                // ceil(2^32 / N), to divide by N
  float* part;
};

template <int CT>
__device__ __forceinline__ float value_of(uint32_t c) {
  if constexpr (CT == SDC_CACHE_E4M3) return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
  else return (float)(int8_t)c;
}

constexpr int ANY_D = 256;                     // largest head size

template <int DT, int CT>
__global__ __launch_bounds__(256) void kv_attend_any(AttendArgs a) {
  __shared__ float qs[4][ANY_D];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t id = (int64_t)blockIdx.x * 4 + w;
  const bool live = id < a.st.T * a.Hq;
  const int64_t t = live ? id / a.Hq : 0;
  const int h = live ? (int)(id - t * a.Hq) : 0, hk = h / a.G;
  const int D = a.D;
  for (int d = lane; d < D; d += 64) qs[w][d] = half_to_f32<DT>(a.q[t * a.sqt + h * a.sqh + d * a.sqd]);
  sdc_wave_lds_fence();
  if (!live) return;
  const int r = sdc_request_of(a.st, t, 1, 0);
  int64_t lo = 0, hi = 0;
  if (r >= 0 && r < a.st.R) {
    const Request rq = sdc_request(a.st, r);
    hi = min(t - rq.q1 + rq.len + 1, a.maxlen);
    lo = max(t - rq.q1 + rq.len + 1 - a.window, (int64_t)0);
  }
  float m = NEG_INF, l = 0.f, o[ANY_D / 64] = {};
  for (int64_t b = lo; b < hi; b += 64) {
    const int64_t j = b + lane;
    float s = NEG_INF, vs = 0.f;
    int64_t row = 0;
    if (j < hi) {
      const int64_t wp = j / a.st.N, page = a.st.bt[r * a.st.sbt + wp];
      const bool in = page >= 0 && page < a.st.NB;
      row = (in ? page : 0) * a.cb + hk * a.ch + (j - wp * a.st.N) * a.cn;
      const float* sc = a.scales + (in ? page : 0) * a.sb + hk * a.sh;
      const float ks = in ? sc[0] : __builtin_nanf("");
      vs = in ? sc[1] : __builtin_nanf("");
      float dot = 0.f;
      for (int d = 0; d < D; ++d) dot = fmaf(qs[w][d], value_of<CT>(a.kv[row + d]), dot);
      s = dot * ks * a.scale;
    }
    const float mn = fmaxf(m, wave_max_f32_dpp(s)), ms = mn == NEG_INF ? 0.f : mn;
    const float p = j < hi ? exp2f(s - ms) : 0.f, f = exp2f(m - ms);
    l = l * f + wave_sum_f32_dpp(p);
#pragma unroll
    for (int e = 0; e < ANY_D / 64; ++e) o[e] *= f;
    const float pv = p * vs;
    for (int i = 0; i < 64 && b + i < hi; ++i) {
      const float pi = __shfl(pv, i);
      const int64_t ri = (int64_t)__shfl((long long)row, i) + D;
#pragma unroll
      for (int e = 0; e < ANY_D / 64; ++e)
        if (lane + 64 * e < D) o[e] = fmaf(pi, value_of<CT>(a.kv[ri + lane + 64 * e]), o[e]);
    }
    m = mn;
  }
  // (a query whose keys all score -inf: 0 / 0)
  const float inv = hi > lo ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < ANY_D / 64; ++e)
    if (lane + 64 * e < D) a.o[t * a.sot + h * a.soh + (lane + 64 * e) * a.sod] = sdc_to_half<DT>(hi > lo ? o[e] * inv : 0.f);
  if (a.lse && lane == 0) a.lse[t * a.slt + h] = hi > lo ? (m + log2f(l)) * LN2 : NEG_INF;
}

// ------------------------------------------------------------------------------------------------ few query rows
constexpr int ROWS = 16;                       // query rows (tokens x heads of one kv head) of a tile
constexpr int MAXP = 1024;                     // page-table entries a workgroup holds
constexpr float M0 = -3.0e38f;                 // a maximum before the first key

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

__device__ __forceinline__ float over_groups_max(float v) {             // lanes l, l + 16, l + 32, l + 48
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float over_groups_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// A tile's place in the step.
struct Tile {
  int r, hk, hb, ntok;                         // request (R: padding), kv head, block of GB heads, tokens
  int64_t tok0, p0;                            // first token and its position
  int64_t klo, khi, c0;                        // keys that some row sees, and where the parts are counted from
  int nsp;                                     // parts with keys
};
__device__ __forceinline__ bool find_tile(const AttendArgs& a, const Split& sp, int id, Tile& t) {
  t.hb = id % sp.NHB;
  id /= sp.NHB;
  t.hk = id % a.Hkv;
  id /= a.Hkv;
  t.r = sdc_request_of(a.st, id, sp.TB, 1);
  if (t.r < 0) return false;
  const Request rq = sdc_request(a.st, t.r);
  t.tok0 = rq.q0 + (id - ((int64_t)((uint32_t)a.st.qsl[t.r] / (uint32_t)sp.TB) + t.r)) * sp.TB;
  if (t.tok0 < rq.q0 || t.tok0 >= rq.q1) return false;
  t.ntok = (int)min((int64_t)sp.TB, rq.q1 - t.tok0);
  t.p0 = t.r < a.st.R ? t.tok0 - rq.q1 + rq.len : -(int64_t)sp.TB;
  t.khi = min(t.p0 + t.ntok, a.maxlen);
  t.klo = max(t.p0 - a.window + 1, (int64_t)0);
  t.c0 = t.klo & ~(int64_t)31;
  t.nsp = t.khi > t.klo ? (int)sdc_cdiv(t.khi - t.c0, sp.C) : 0;
  return true;
}

// One row's results: x[0 .. n) at elements d.., scaled.
__device__ __forceinline__ void write_out(const AttendArgs& a, int64_t tok, int h, int d, const float* x, int n, float f) {
  uint16_t* o = a.o + tok * a.sot + h * a.soh;
  for (int i = 0; i < n && d + i < a.D; ++i)
    o[(d + i) * a.sod] = a.fp16 ? sdc_to_half<SDC_FP16>(x[i] * f) : sdc_to_half<SDC_BF16>(x[i] * f);
}

// Tiles of up to 16 query rows over a part of their keys: HBM bound, so a wave streams 32 keys at a time straight into
// registers and everything else stays there.  S^T = K Q^T on v_mfma_f32_16x16x32_f16 (lane l: key l % 16, a quarter of
// the depth; the depth's order is free, so a lane reads DP / 4 adjacent codes); the accumulator's layout (key 4 (l / 16)
// + i, row l % 16) is then the B operand of O^T = V^T P^T with the keys in that order, so the probabilities move to no
// other lane; V^T's fragments are 4 x 4 byte transposes of rows that a lane reads DP / 16 codes of.  Codes are exact in
// fp16; queries are scaled to it by a power of two per row (a bf16 element 2^-27 of its row's largest keeps all bits).
// The key scales multiply the scores, the value scales the probabilities, in fp32.  Probabilities are rounded to fp16's
// 11 bits, in units that put their largest product with a value scale at 2^13 .. 2^15.
template <int CT, int DP, int PN>
__global__ __launch_bounds__(256) void kv_attend_rows(AttendArgs a, Split sp) {
  constexpr int KW = DP / 64;                  // 16-byte reads of a key per lane; dwords of a value per lane
  constexpr int NS = DP / 32, ND = DP / 16;    // depth steps of a score, row blocks of the output
  constexpr int QS = DP + 8, OS = DP + 4;      // row pitches in LDS
  struct Head {
    float2 sc[MAXP];
    int32_t pg[MAXP];
    _Float16 q[ROWS][QS];
  };
  __shared__ union {
    Head h;
    float o[4][ROWS][OS];
  } sh;
  __shared__ float rowf[ROWS], wmax[4], ml[4][ROWS][2];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, c = lane & 15, g = lane >> 4;
  const int D = a.D, N = a.st.N;
  const int s = blockIdx.x % sp.S, tile = blockIdx.x / sp.S;
  Tile t;
  if (!find_tile(a, sp, tile, t)) return;
  if (s >= max(t.nsp, 1)) return;
  const int orow = tid >> 4, od = (tid & 15) * ND;                      // the output a thread writes: row, elements
  const int otok = orow / sp.GB, oh = t.hb * sp.GB + orow % sp.GB;
  const bool olive = orow < sp.GB * sp.TB && otok < t.ntok && oh < a.G;
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
  const int64_t a0 = t.c0 + (int64_t)s * sp.C, a1 = min(t.khi, a0 + sp.C);
  const int64_t fp = (uint32_t)a0 / (uint32_t)N;
  const int np = (int)((uint32_t)(a1 - 1) / (uint32_t)N - fp) + 1, base0 = (int)(a0 - fp * N);

  // the part's pages and their scales; a page outside the cache is page 0 with scales of NaN
  float vmax = 0.f;
  for (int i = tid; i < np; i += 256) {
    const int32_t page = a.st.bt[t.r * a.st.sbt + fp + i];
    const bool in = page >= 0 && page < a.st.NB;
    const float* scp = a.scales + (in ? (int64_t)page : 0) * a.sb + t.hk * a.sh;
    float2 sc = {scp[0], scp[1]};
    if (!in) sc = {__builtin_nanf(""), __builtin_nanf("")};
    sh.h.pg[i] = in ? page : 0;
    sh.h.sc[i] = sc;
    const float v = fabsf(sc.y);
    if (v <= 3.0e38f) vmax = fmaxf(vmax, v);
  }
  // the queries, a row per 16 threads
  {
    float x[ND], amax = 0.f;
    const uint16_t* qp = a.q + (olive ? otoken * a.sqt + ohead * a.sqh : 0);
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const uint16_t v = olive && od + i < D ? qp[(od + i) * a.sqd] : (uint16_t)0;
      x[i] = a.fp16 ? half_to_f32<SDC_FP16>(v) : half_to_f32<SDC_BF16>(v);
      const float f = fabsf(x[i]);
      if (f <= 3.3e38f) amax = fmaxf(amax, f);
    }
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) amax = fmaxf(amax, __shfl_xor(amax, m));
    int e = 0;
    (void)frexpf(amax, &e);
    e = max(e, -100);
    const float f = ldexpf(1.f, 13 - e);
#pragma unroll
    for (int i = 0; i < ND; ++i) sh.h.q[orow][od + i] = (_Float16)(x[i] * f);
    if ((tid & 15) == 0) rowf[orow] = ldexpf(a.scale, e - 13);
  }
  vmax = wave_max_f32_dpp(vmax);
  if (lane == 0) wmax[w] = vmax;
  __syncthreads();
  vmax = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
  int ve;
  (void)frexpf(vmax, &ve);
  const int bias = 13 - min(max(ve, -100), 100);                        // probabilities in units of 2^-bias
  const float fbias = (float)bias, unit = ldexpf(1.f, -bias);
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
  const int nk = (int)(a1 - a0);

  f32x4 o[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = M0, l = 0.f;
  const uint8_t* base = a.kv + t.hk * a.ch;

  // page entry and slot of a key counted from a0
  auto place = [&](int key, int& slot) {
    const uint32_t loc = (uint32_t)(base0 + key);
    const int i = N == 1 ? (int)loc : (int)__umulhi(loc, sp.div);
    slot = (int)loc - i * N;
    return min(i, np - 1);
  };
  struct Buf {
    u32x4 k[2][KW];
    uint32_t v[8][KW];
    float2 sc[8];
  };
  auto load = [&](int k0, Buf& b) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      int slot, e;
      const uint8_t* row;
      if constexpr (PN == 16) {                // the 16 keys lie in one page
        e = __builtin_amdgcn_readfirstlane(place(k0 + 16 * u, slot));
        slot = __builtin_amdgcn_readfirstlane(slot);
        const float2 sc = sh.h.sc[e];
        row = base + (int64_t)__builtin_amdgcn_readfirstlane(sh.h.pg[e]) * a.cb + (int64_t)slot * a.cn;
        const uint8_t* kr = row + c * a.cn + g * (DP / 4);
#pragma unroll
        for (int j = 0; j < KW; ++j)
          b.k[u][j] = g * (DP / 4) + 16 * j < D ? *reinterpret_cast<const u32x4*>(kr + 16 * j) : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t* vr = row + (4 * g + i) * a.cn + D + c * (DP / 16);
          b.sc[4 * u + i] = sc;
          typedef uint32_t vt __attribute__((ext_vector_type(KW)));
          if constexpr (KW == 1) b.v[4 * u + i][0] = c * (DP / 16) < D ? *reinterpret_cast<const uint32_t*>(vr) : 0u;
          else {
            vt x = {};
            if (c * (DP / 16) < D) x = *reinterpret_cast<const vt*>(vr);
#pragma unroll
            for (int j = 0; j < KW; ++j) b.v[4 * u + i][j] = x[j];
          }
        }
      } else {
        e = place(k0 + 16 * u + c, slot);
        row = base + (int64_t)sh.h.pg[e] * a.cb + (int64_t)slot * a.cn;
#pragma unroll
        for (int j = 0; j < KW; ++j)
          b.k[u][j] = g * (DP / 4) + 16 * j < D ? *reinterpret_cast<const u32x4*>(row + g * (DP / 4) + 16 * j) : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e = place(k0 + 16 * u + 4 * g + i, slot);
          b.sc[4 * u + i] = sh.h.sc[e];
          const uint8_t* vr = base + (int64_t)sh.h.pg[e] * a.cb + (int64_t)slot * a.cn + D + c * (DP / 16);
#pragma unroll
          for (int j = 0; j < KW; ++j)
            b.v[4 * u + i][j] = c * (DP / 16) < D ? *reinterpret_cast<const uint32_t*>(vr + 4 * j) : 0u;
        }
      }
    }
  };

  auto compute = [&](int k0, Buf& b) {
    f32x4 sc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      sc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NS; ++i)
        sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen8<CT>(b.k[u][i / 2][2 * (i % 2)], b.k[u][i / 2][2 * (i % 2) + 1]),
                                                       qf[i], sc[u], 0, 0, 0);
    }
    float x[8], top = M0;
    const bool edge = k0 < flo || k0 + 32 > fhi;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = sc[j / 4][j % 4] * (b.sc[j].x * rf);
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
    // the maximum follows the scores only when they pass it by 2 (a factor of 4, which fp16 has room for)
    if (__any(top > m + 2.f)) {
      const float mn = fmaxf(m, over_groups_max(top));
      const float f = exp2f(m - mn);
      l *= f;
#pragma unroll
      for (int n = 0; n < ND; ++n) o[n] *= f;
      m = mn;
    }
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = __builtin_amdgcn_exp2f(x[j] - m + fbias);
      l += p[j];
      p[j] *= b.sc[j].y;
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

  Buf b0, b1;
  int k = 32 * w;
  if (k < nk) load(k, b0);
  while (k < nk) {                             // 128 keys of the workgroup's four waves at a time, the next ones in flight
    if (k + 128 < nk) load(k + 128, b1);
    compute(k, b0);
    k += 128;
    if (k >= nk) break;
    if (k + 128 < nk) load(k + 128, b0);
    compute(k, b1);
    k += 128;
  }

  // the four waves' sums joined: a lane holds DP / 4 adjacent outputs of its row
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
  float mt = M0, lt = 0.f, f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) mt = fmaxf(mt, ml[i][orow][0]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = exp2f(ml[i][orow][0] - mt);
    lt += f[i] * ml[i][orow][1];
  }
  float x[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) {
    x[n] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[n] += f[i] * sh.o[i][orow][od + n];
  }
  if (!olive) return;
  if (t.nsp == 1) {
    // (a row with keys whose scores are all -inf: 0 / 0)
    const int64_t p = t.p0 + otok;
    const bool any = min(p + 1, a.maxlen) > max(p - a.window + 1, (int64_t)0);
    write_out(a, otoken, ohead, od, x, ND, any ? 1.f / lt : 0.f);
    if (a.lse && (tid & 15) == 0) a.lse[otoken * a.slt + ohead] = any ? (mt + log2f(lt) - fbias) * LN2 : NEG_INF;
  } else {
    float* rec = sp.part + (int64_t)blockIdx.x * ROWS * (D + 2);
    if ((tid & 15) == 0) {
      rec[2 * orow] = mt;
      rec[2 * orow + 1] = lt * unit;
    }
    for (int n = 0; n < ND && od + n < D; ++n) rec[2 * ROWS + orow * D + od + n] = x[n] * unit;
  }
}

// The parts of a tile joined, in their order.
__global__ __launch_bounds__(256) void kv_attend_join(AttendArgs a, Split sp) {
  const int tid = threadIdx.x, orow = tid >> 4, D = a.D;
  Tile t;
  if (!find_tile(a, sp, blockIdx.x, t) || t.nsp < 2) return;
  const int otok = orow / sp.GB, oh = t.hb * sp.GB + orow % sp.GB;
  if (orow >= sp.GB * sp.TB || otok >= t.ntok || oh >= a.G) return;
  const int64_t token = t.tok0 + otok, size = (int64_t)ROWS * (D + 2);
  const int head = t.hk * a.G + oh;
  const float* rec = sp.part + (int64_t)blockIdx.x * sp.S * size;
  float m = M0, l = 0.f;
  for (int s = 0; s < t.nsp; ++s) m = fmaxf(m, rec[s * size + 2 * orow]);
  for (int s = 0; s < t.nsp; ++s) l += exp2f(rec[s * size + 2 * orow] - m) * rec[s * size + 2 * orow + 1];
  const int64_t p = t.p0 + otok;
  const bool any = min(p + 1, a.maxlen) > max(p - a.window + 1, (int64_t)0);
  for (int d = tid & 15; d < D; d += 16) {
    float x = 0.f;
    for (int s = 0; s < t.nsp; ++s) x += exp2f(rec[s * size + 2 * orow] - m) * rec[s * size + 2 * ROWS + orow * D + d];
    write_out(a, token, head, d, &x, 1, any ? 1.f / l : 0.f);
  }
  if (a.lse && (tid & 15) == 0) a.lse[token * a.slt + head] = any ? (m + log2f(l)) * LN2 : NEG_INF;
}

// The tiles and parts of a call, from its sizes alone.
Split plan(int64_t T, int64_t R, int64_t Hkv, int64_t G, int64_t N, int64_t most) {
  Split sp{};
  sp.GB = (int)std::min<int64_t>(G, ROWS);
  sp.NHB = (int)sdc_cdiv(G, ROWS);
  sp.TB = std::max(1, ROWS / sp.GB);
  sp.tiles = (T / sp.TB + R + 1) * Hkv * sp.NHB;
  const int64_t busy = std::max<int64_t>(1, std::min(T, T / sp.TB + R) * Hkv * sp.NHB);
  // parts of at least 256 keys, as many as fill the chip about three times
  const int64_t want = std::max<int64_t>(1, 1024 / busy);
  int64_t C = std::max<int64_t>(256, sdc_cdiv(sdc_cdiv(most + 31, want), 128) * 128);
  C = std::min(C, std::max<int64_t>(128, (MAXP - 2) * N / 128 * 128));
  C = std::min<int64_t>(C, 16384);
  sp.C = (int)C;
  sp.S = (int)std::max<int64_t>(1, sdc_cdiv(most + 31, C));
  sp.div = N == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + N - 1) / N);
  return sp;
}
int64_t part_bytes(const Split& sp, int64_t D) {
  return sp.S == 1 ? 0 : sp.tiles * sp.S * ROWS * (D + 2) * 4;
}
// keys a tile's rows can see together
int64_t most_keys(int64_t max_len, int64_t window) { return window > 0 ? std::min(max_len, window + ROWS) : max_len; }

template <int CT, int DP>
int launch_rows(const AttendArgs& a, const Split& sp, hipStream_t stream) {
  const int64_t blocks = sp.tiles * sp.S;
  if (blocks > 0x7FFFFFFF) return SDC_EUNSUPPORTED;
  {
    SdcProf prof("kv_attend", stream);
    if (a.st.N % 16 == 0)
      hipLaunchKernelGGL((kv_attend_rows<CT, DP, 16>), dim3((unsigned)blocks), dim3(256), 0, stream, a, sp);
    else
      hipLaunchKernelGGL((kv_attend_rows<CT, DP, 1>), dim3((unsigned)blocks), dim3(256), 0, stream, a, sp);
    SDC_LAUNCH_CHECK();
  }
  if (sp.S > 1) {
    SdcProf prof("kv_attend_join", stream);
    hipLaunchKernelGGL(kv_attend_join, dim3((unsigned)sp.tiles), dim3(256), 0, stream, a, sp);
    SDC_LAUNCH_CHECK();
  }
  return SDC_OK;
}
template <int CT>
int run_rows(const AttendArgs& a, const Split& sp, hipStream_t stream) {
  if (a.D <= 64) return launch_rows<CT, 64>(a, sp, stream);
  return a.D <= 128 ? launch_rows<CT, 128>(a, sp, stream) : launch_rows<CT, 256>(a, sp, stream);
}

template <int DT>
int run(int cache, const AttendArgs& a, hipStream_t stream) {
  const int64_t blocks = sdc_cdiv(a.st.T * a.Hq, 4);
  if (blocks > 0x7FFFFFFF) return SDC_EUNSUPPORTED;
  SdcProf prof("kv_attend", stream);
  if (cache == SDC_CACHE_E4M3)
    hipLaunchKernelGGL((kv_attend_any<DT, SDC_CACHE_E4M3>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((kv_attend_any<DT, SDC_CACHE_I8>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  SDC_LAUNCH_CHECK();
  return SDC_OK;
}

}  // namespace

extern "C" int64_t sdc_kv_attend_workspace(int64_t T, int64_t R, int64_t Hq, int64_t Hkv, int64_t D, int64_t N,
                                           int64_t max_len, int64_t window) {
  if (T < 1 || R < 0 || Hkv < 1 || Hq < Hkv || D < 1 || N < 1 || max_len < 0 || T > 0x3FFFFFFF || R > 0x0FFFFFFF) return 0;
  return part_bytes(plan(T, R, Hkv, Hq / Hkv, N, most_keys(max_len, window)), D);
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
      max_len < 0 || max_len > W * N)
    return SDC_EINVAL;
  if (T == 0) return SDC_OK;
  if (!q || !o || !kv || !scales || !qsl || !seq_lens || !bt) return SDC_EINVAL;
  if (T > 0x3FFFFFFF || R > 0x0FFFFFFF || Hq > 65536 || W * N > 0x7FFFFFFF) return SDC_EUNSUPPORTED;
  AttendArgs a{};
  a.st = PagedStep{qsl, seq_lens, bt, sbt, W, NB, T, (int)R, (int)N};
  a.q = (const uint16_t*)q; a.o = (uint16_t*)o; a.lse = lse;
  a.sqt = sqt; a.sqh = sqh; a.sqd = sqd; a.sot = sot; a.soh = soh; a.sod = sod; a.slt = slt;
  a.kv = (const uint8_t*)kv; a.cb = cb; a.ch = ch; a.cn = cn;
  a.scales = scales; a.sb = sb; a.sh = sh;
  a.scale = scale * LOG2E;
  a.maxlen = max_len;
  a.window = window > 0 ? window : (int64_t)1 << 40;
  a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.G = (int)(Hq / Hkv); a.D = (int)D; a.fp16 = dtype == SDC_FP16;
  // the tiled kernels read 16 codes at a time, and divide by N by a product (exact up to this many slots)
  if (D % 16 == 0 && N <= 4096 && ((uintptr_t)kv | (uintptr_t)(cb | ch | cn)) % 16 == 0) {
    Split sp = plan(T, R, Hkv, a.G, N, most_keys(max_len, window));
    sp.part = (float*)workspace;
    if (workspace_bytes < part_bytes(sp, D) || (sp.S > 1 && !workspace)) return SDC_EWORKSPACE;
    return cache == SDC_CACHE_E4M3 ? run_rows<SDC_CACHE_E4M3>(a, sp, stream) : run_rows<SDC_CACHE_I8>(a, sp, stream);
  }
  return dtype == SDC_BF16 ? run<SDC_BF16>(cache, a, stream) : run<SDC_FP16>(cache, a, stream);
}
