// Rotary positions of (tokens, heads, head size) tensors: the first `rot` elements of each head rotated by the token's
// position, the rest copied; `inverse` rotates back (times the same factor), which is the gradient of the forward call.
//
// HBM bound: each element is read and written once (8192 tokens of 32 heads of 128: 26 us, 5.1 TB/s).  A workgroup takes TB tokens of HB heads: its threads compute
// the tokens' cosines and sines once into LDS (64-bit angles, rope.h) and then rotate units of 16 elements (two
// 16-byte runs: the two halves of a pair range, or 16 adjacent elements), so a pair never crosses threads.
#include <algorithm>

#include "common.h"
#include "profile.h"
#include "rope.h"

namespace {

constexpr int TAB = 1024;                      // (cos, sin) pairs a workgroup holds

struct RopeArgs {
  const void* x; void* y; const void* pos; const double* turns;
  int64_t T, sxt, sxh, sxd, syt, syh, syd;
  double m;                                    // factor on the result
  int H, D, rot, inter, inverse, pos32, TB, HB;
};

template <int DT, int UP>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
  typedef typename RopeElem<DT>::T E;
  __shared__ float2 tab[TAB];
  const int tid = threadIdx.x, P = a.rot / 2;
  const int64_t t0 = (int64_t)blockIdx.x * a.TB;
  const int nt = (int)min((int64_t)a.TB, a.T - t0);
  const int h0 = blockIdx.y * a.HB, nh = min(a.HB, a.H - h0);
  for (int i = tid; i < nt * P; i += 256) {
    const int t = i / P, f = i - t * P;
    const double p = a.pos32 ? (double)((const int32_t*)a.pos)[t0 + t] : (double)((const int64_t*)a.pos)[t0 + t];
    float2 cs = sdc_turn(p, a.turns[f], a.m);
    if (a.inverse) cs.y = -cs.y;
    tab[i] = cs;
  }
  __syncthreads();
  const int nu = sdc_units(a.D, UP);
  for (int i = tid; i < nt * nh * nu; i += 256) {
    const int th = i / nu, u = i - th * nu, t = th / nh, h = h0 + th - t * nh;
    const RopeUnit r = sdc_unit<UP>(u, a.rot, a.inter);
    float v[2 * UP];
    sdc_load_unit<DT, UP>((const E*)a.x + (t0 + t) * a.sxt + h * a.sxh, a.sxd, r, a.D, v);
    sdc_rotate_unit<UP>(v, r, a.inter, tab + t * P);
    sdc_store_unit<DT, UP>((E*)a.y + (t0 + t) * a.syt + h * a.syh, a.syd, r, a.D, v);
  }
}

template <int DT, int UP>
int launch(RopeArgs a, hipStream_t stream) {
  const int P = a.rot / 2;
  // A unit a thread: a token of 32 heads of 128 a workgroup 3.1 us at 16 tokens, 5.3 at 1024, 22.8 at 8192, four tokens 5.8,
  // 7.1 and 23.0; four tokens of 12 heads of 80 5.7 us at 4099, one token 7.0; 300 tokens of 128 heads 7.8 us in one piece,
  // 6.1 in four.
  const int nu = sdc_units(a.D, UP), units = a.H * nu;
  a.TB = std::max(1, 256 / units);
  while (a.TB > 1 && a.TB * P > TAB) a.TB /= 2;
  a.HB = units > 512 ? std::max({1, 256 / nu, (int)sdc_cdiv(a.H, 65535)}) : a.H;
  SdcProf prof("rope", stream);
  const dim3 grid((unsigned)sdc_cdiv(a.T, a.TB), (unsigned)sdc_cdiv(a.H, a.HB));
  hipLaunchKernelGGL((rope_kernel<DT, UP>), grid, dim3(256), 0, stream, a);
  SDC_LAUNCH_CHECK();
  return SDC_OK;
}

template <int DT>
int pick(const RopeArgs& a, hipStream_t stream) {
  constexpr int es = DT == SDC_F32 ? 4 : 2, UP = 16 / es;
  // 16-byte runs: rows, heads and both runs of every unit on 16-byte boundaries
  const bool vec = a.sxd == 1 && a.syd == 1 && a.D % (2 * UP) == 0 && a.rot % (2 * UP) == 0 &&
                   ((uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)(a.sxt * es) | (uintptr_t)(a.sxh * es) |
                    (uintptr_t)(a.syt * es) | (uintptr_t)(a.syh * es)) % 16 == 0;
  return vec ? launch<DT, UP>(a, stream) : launch<DT, 1>(a, stream);
}

}  // namespace

extern "C" int sdc_rope(int dtype, const void* x, int64_t sxt, int64_t sxh, int64_t sxd, void* y, int64_t syt,
                        int64_t syh, int64_t syd, int64_t T, int64_t H, int64_t D, const void* positions,
                        int pos_bytes, const double* turns, int64_t rot, int interleaved, double mscale, int inverse,
                        hipStream_t stream) {
  SDC_CLEAR_ERRORS();
  if (T < 0 || H < 0 || D < 1 || D > 65536 || H > (1 << 24) || rot < 0 || rot % 2 || rot > D || rot / 2 > TAB ||
      (pos_bytes != 4 && pos_bytes != 8))
    return SDC_EINVAL;
  if (T == 0 || H == 0) return SDC_OK;
  if (!x || !y || !positions || (rot && !turns)) return SDC_EINVAL;
  if (T > (int64_t)1 << 31 || H * D > (int64_t)1 << 26) return SDC_EUNSUPPORTED;    // (32-bit unit numbers and grid)
  RopeArgs a{x, y, positions, turns, T, sxt, sxh, sxd, syt, syh, syd, mscale, (int)H, (int)D, (int)rot,
             interleaved != 0, inverse != 0, pos_bytes == 4, 1, 1};
  switch (dtype) {
    case SDC_BF16: return pick<SDC_BF16>(a, stream);
    case SDC_FP16: return pick<SDC_FP16>(a, stream);
    case SDC_F32: return pick<SDC_F32>(a, stream);
    default: return SDC_EINVAL;
  }
}
