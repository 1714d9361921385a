// Rotation by position: pair (a, b) of frequency i at position p becomes (a c - b s, b c + a s) with c = m cos(2 pi t),
// s = m sin(2 pi t), t = p turns_i.  Used by the rotation itself (rope.hip) and by the append to a paged cache
// (kv_append.hip).
#pragma once
#include "common.h"

// Element kinds of the rotated tensors: SDC_BF16, SDC_FP16, and fp32.
constexpr int SDC_F32 = 4;

// A value as it is rounded to its type: the compiler fuses no multiply-add across it.
template <class T>
__device__ __forceinline__ T sdc_rounded(T x) {
  asm("" : "+v"(x));
  return x;
}

// The angle is taken in 64 bits (at position 2^20 a 32-bit angle is off by 0.06), as turns: t - rint(t) is exact, and so
// is the quarter turn taken off next; the two series run to a^15 and a^16, which at pi/4 leaves under 1e-16.  The
// results are then the 64-bit ones rounded to 32 bits once, whatever the position.  Fp64 FMAs run at the rate of fp32
// ones here, so a table of cosines (a read per token and frequency) would only cost bandwidth.
__device__ __forceinline__ float2 sdc_turn(double pos, double turns, double m) {
  const double t = sdc_rounded(pos * turns);
  const double r = t - rint(t);
  const double k = rint(r * 4.0);
  const double a = fma(k, -0.25, r) * 6.283185307179586476925;
  const double z = a * a;
  double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;
  s = fma(s, z, 1.0 / 6227020800.0);
  c = fma(c, z, -1.0 / 87178291200.0);
  s = fma(s, z, -1.0 / 39916800.0);
  c = fma(c, z, 1.0 / 479001600.0);
  s = fma(s, z, 1.0 / 362880.0);
  c = fma(c, z, -1.0 / 3628800.0);
  s = fma(s, z, -1.0 / 5040.0);
  c = fma(c, z, 1.0 / 40320.0);
  s = fma(s, z, 1.0 / 120.0);
  c = fma(c, z, -1.0 / 720.0);
  s = fma(s, z, -1.0 / 6.0);
  c = fma(c, z, 1.0 / 24.0);
  c = fma(c, z, -0.5);
  s = fma(s * z, a, a);
  c = fma(c, z, 1.0);
  const int q = (int)k & 3;                           // quarter turns: (c, s) -> (-s, c) for each
  const double cc = (q & 1) ? s : c, ss = (q & 1) ? c : s;
  const double cq = (q == 1 || q == 2) ? -cc : cc, sq = (q >= 2) ? -ss : ss;
  return make_float2((float)(cq * m), (float)(sq * m));
}

// One pair.  Products and sum are rounded one by one (no fused multiply-add): the same bits as the same three
// operations anywhere else, so that a quantized key does not depend on who computed it.
__device__ __forceinline__ void sdc_rotate(float& a, float& b, float2 cs) {
  const float p = sdc_rounded(a * cs.x), q = sdc_rounded(b * cs.y), u = sdc_rounded(b * cs.x), v = sdc_rounded(a * cs.y);
  a = p - q;
  b = u + v;
}

template <int DT>
struct RopeElem { typedef uint16_t T; };
template <>
struct RopeElem<SDC_F32> { typedef float T; };

// Where unit u of a head's row lies: UP pairs as two runs of UP elements, at c0 and c1; `freq` is its first
// frequency, or -1 where the elements are not rotated (past `rot`).  Layout 0: pairs (i, i + rot / 2), layout 1:
// adjacent pairs, whose elements alternate over the two runs taken together.
struct RopeUnit { int c0, c1, freq; };
template <int UP>
__device__ __forceinline__ RopeUnit sdc_unit(int u, int rot, int inter) {
  const int p = rot / 2, nr = p / UP;
  RopeUnit r;
  if (u < nr) {
    r.freq = u * UP;
    r.c0 = inter ? 2 * UP * u : UP * u;
    r.c1 = inter ? r.c0 + UP : p + UP * u;
  } else {
    r.freq = -1;
    r.c0 = rot + 2 * UP * (u - nr);
    r.c1 = r.c0 + UP;
  }
  return r;
}

// The unit's 2 UP values as floats: UP = 8 (4 for fp32) reads 16 bytes a run, UP = 1 any stride and alignment (a run
// past the row's end reads 0).
template <int DT, int UP>
__device__ __forceinline__ void sdc_load_unit(const typename RopeElem<DT>::T* row, int64_t sd, RopeUnit r, int D, float* v) {
  if constexpr (UP == 1) {
    if constexpr (DT == SDC_F32) {
      v[0] = row[r.c0 * sd];
      v[1] = r.c1 < D ? row[r.c1 * sd] : 0.f;
    } else {
      v[0] = half_to_f32<DT>(row[r.c0 * sd]);
      v[1] = r.c1 < D ? half_to_f32<DT>(row[r.c1 * sd]) : 0.f;
    }
  } else {
    const u32x4 a = *reinterpret_cast<const u32x4*>(row + r.c0), b = *reinterpret_cast<const u32x4*>(row + r.c1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == SDC_F32) {
        v[i] = __uint_as_float(a[i]);
        v[UP + i] = __uint_as_float(b[i]);
      } else {
        v[2 * i] = lo_of<DT>(a[i]);
        v[2 * i + 1] = hi_of<DT>(a[i]);
        v[UP + 2 * i] = lo_of<DT>(b[i]);
        v[UP + 2 * i + 1] = hi_of<DT>(b[i]);
      }
    }
  }
}

// fp32 -> 16 bits, to nearest, ties to even
template <int DT>
__device__ __forceinline__ uint16_t sdc_to_half(float f) {
  if constexpr (DT == SDC_BF16) return __builtin_bit_cast(uint16_t, (__bf16)f);
  else return __builtin_bit_cast(uint16_t, (_Float16)f);
}

template <int DT, int UP>
__device__ __forceinline__ void sdc_store_unit(typename RopeElem<DT>::T* row, int64_t sd, RopeUnit r, int D, const float* v) {
  if constexpr (UP == 1) {
    if constexpr (DT == SDC_F32) {
      row[r.c0 * sd] = v[0];
      if (r.c1 < D) row[r.c1 * sd] = v[1];
    } else {
      row[r.c0 * sd] = sdc_to_half<DT>(v[0]);
      if (r.c1 < D) row[r.c1 * sd] = sdc_to_half<DT>(v[1]);
    }
  } else {
    u32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == SDC_F32) {
        a[i] = __float_as_uint(v[i]);
        b[i] = __float_as_uint(v[UP + i]);
      } else {
        a[i] = (uint32_t)sdc_to_half<DT>(v[2 * i]) | ((uint32_t)sdc_to_half<DT>(v[2 * i + 1]) << 16);
        b[i] = (uint32_t)sdc_to_half<DT>(v[UP + 2 * i]) | ((uint32_t)sdc_to_half<DT>(v[UP + 2 * i + 1]) << 16);
      }
    }
    *reinterpret_cast<u32x4*>(row + r.c0) = a;
    *reinterpret_cast<u32x4*>(row + r.c1) = b;
  }
}

// tab: the token's (cos, sin) by frequency
template <int UP>
__device__ __forceinline__ void sdc_rotate_unit(float* v, RopeUnit r, int inter, const float2* tab) {
  if (r.freq < 0) return;
#pragma unroll
  for (int j = 0; j < UP; ++j) {
    const float2 cs = tab[r.freq + j];
    if (inter) sdc_rotate(v[2 * j], v[2 * j + 1], cs);
    else sdc_rotate(v[j], v[UP + j], cs);
  }
}

// units of a row: every element lies in one
__host__ __device__ static inline int sdc_units(int D, int up) { return (D + 2 * up - 1) / (2 * up); }
