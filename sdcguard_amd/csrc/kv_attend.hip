// Attention of a step's queries over a paged cache of 8-bit codes, a scale for the keys and one for the values of each
// (page, kv head): o = sum_j p_j v_j / sum_j p_j over the keys j a query sees (its own position and those before it, the
// last `window` of them), p_j = exp(s_j - max s), s_j = scale q . k_j, k_j = ks[page] kcode_j, v_j = vs[page] vcode_j;
// lse = max s + log sum p.  A query that sees no key gets zeros and lse = -inf; a key in a page outside the cache
// counts as NaN.
//
// The path for any head size and alignment: a wave per (query token, head), a key per lane for the products, then the
// head's elements over the lanes for the sum of the values.
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
  int Hq, Hkv, G, D;
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

extern "C" int64_t sdc_kv_attend_workspace(int64_t T, int64_t R, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_len) {
  (void)T; (void)R; (void)Hq; (void)Hkv; (void)D; (void)max_len;
  return 0;
}

extern "C" int sdc_kv_attend(int dtype, int cache, const void* q, int64_t sqt, int64_t sqh, int64_t sqd, void* o,
                             int64_t sot, int64_t soh, int64_t sod, float* lse, int64_t slt, int64_t T, int64_t Hq,
                             int64_t D, const void* kv, int64_t cb, int64_t ch, int64_t cn, int64_t NB, int64_t Hkv,
                             int64_t N, const float* scales, int64_t sb, int64_t sh, const int32_t* qsl,
                             const int32_t* seq_lens, int64_t R, const int32_t* bt, int64_t sbt, int64_t W, float scale,
                             int64_t window, int64_t max_len, void* workspace, int64_t workspace_bytes,
                             hipStream_t stream) {
  SDC_CLEAR_ERRORS();
  (void)workspace; (void)workspace_bytes;
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
  a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.G = (int)(Hq / Hkv); a.D = (int)D;
  return dtype == SDC_BF16 ? run<SDC_BF16>(cache, a, stream) : run<SDC_FP16>(cache, a, stream);
}
