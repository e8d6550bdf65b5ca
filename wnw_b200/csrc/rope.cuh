// Rotary positions: angles in 64 bits, shared by the rotary kernel and the
// 8-bit cache's append.
#pragma once

#include "common.cuh"

namespace wnw {

// Cosine and sine of x in 64 bits, within 2^-49 for |x| up to 2^31 and more.
// x is brought to [-pi/4, pi/4] by the nearest multiple n of pi/2, held in two
// doubles (the reduction of Cody and Waite; both products are fused, so only
// the remainder is rounded), where the Taylor series, the sine's to r^15 / 15!
// and the cosine's to r^14 / 14!, leave out less than 2^-53 and 2^-49.8; the
// operations' own roundings add some 2^-52.  Some 20 double operations and no conversion but the two
// results': integers and doubles meet through sums with 1.5 x 2^52, whose low
// bits are the integer.
constexpr double kIntMagic = 6755399441055744.0;  // 1.5 x 2^52: |integers| below 2^51
__device__ __forceinline__ double int_to_double(long long i) {
  return __longlong_as_double(i + 0x4338000000000000ll) - kIntMagic;
}
// (the quadrant n mod 4 is left to the caller, who may turn rounded values)
__device__ __forceinline__ int cos_sin(double x, double& c, double& s) {
  const double t = fma(x, 0.63661977236758134308, kIntMagic);  // 2 / pi, rounded to an integer
  const double n = t - kIntMagic;
  double r = fma(-n, 1.57079632679489655800e+00, x);           // pi / 2 rounded
  r = fma(-n, 6.12323399573676603587e-17, r);                  // and what the rounding left
  const double z = r * r;
  double ps = -1.0 / 1307674368000.0, pc = -1.0 / 87178291200.0;  // -1/15!, -1/14!
  ps = fma(ps, z, 1.0 / 6227020800.0);
  pc = fma(pc, z, 1.0 / 479001600.0);
  ps = fma(ps, z, -1.0 / 39916800.0);
  pc = fma(pc, z, -1.0 / 3628800.0);
  ps = fma(ps, z, 1.0 / 362880.0);
  pc = fma(pc, z, 1.0 / 40320.0);
  ps = fma(ps, z, -1.0 / 5040.0);
  pc = fma(pc, z, -1.0 / 720.0);
  ps = fma(ps, z, 1.0 / 120.0);
  pc = fma(pc, z, 1.0 / 24.0);
  ps = fma(ps, z, -1.0 / 6.0);
  pc = fma(pc, z, -0.5);
  s = fma(ps * z, r, r);
  c = fma(pc, z, 1.0);
  return __double2loint(t) & 3;
}

// A pair's axis and frequency, a token's position on an axis, and the cosine
// and sine of their product, scaled and rounded once to fp32.  A position of a
// long context times a frequency near 1 leaves fp32 with an angle off by 2^-24
// of the position (0.007 rad at 120k tokens), so the angle and its reduction
// are in 64 bits.
struct RopePair {
  int axis;
  double freq;
};
__device__ __forceinline__ RopePair rope_pair(const wnw_rope& r, int i, int32_t* err) {
  int ax = __ldg(r.axis + i);
  if (ax < 0 || ax >= r.num_axes) {
    atomicOr(err, WNW_DEVERR_BAD_INDEX);
    ax = 0;
  }
  return RopePair{ax, __ldg(r.inv_freq + i)};
}
__device__ __forceinline__ double rope_pos(const wnw_rope& r, int axis, int64_t b, int64_t n) {
  const int64_t at = axis * r.pos_stride_a + b * r.pos_stride_b + n * r.pos_stride_n;
  return int_to_double(r.pos_is64 ? __ldg(static_cast<const long long*>(r.pos) + at)
                                  : static_cast<long long>(__ldg(static_cast<const int32_t*>(r.pos) + at)));
}
__device__ __forceinline__ float2 rope_turn_of(const wnw_rope& r, double angle) {
  double s, c;
  const int q = cos_sin(angle, c, s);
  // by quadrants the two swap and change sign, after the rounding as well as before
  const uint32_t fc = __float_as_uint(static_cast<float>(c * r.scaling));
  const uint32_t fs = __float_as_uint(static_cast<float>(s * r.scaling));
  return make_float2(__uint_as_float((q & 1 ? fs : fc) ^ uint32_t(q + 1 & 2) << 30),
                     __uint_as_float((q & 1 ? fc : fs) ^ uint32_t(q & 2) << 30));
}

// one pair of dimensions; every product and sum rounded (no contraction), so
// that a value does not depend on which kernel rotates it
__device__ inline void rope_turn(float a, float b, float2 cs, float& ya, float& yb) {
  ya = __fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y));
  yb = __fadd_rn(__fmul_rn(b, cs.x), __fmul_rn(a, cs.y));
}

inline wnw_status check_rope(const wnw_rope& r, int head_dim) {
  WNW_CHECK_ARG(r.rot >= 0 && r.rot % 16 == 0 && r.rot <= head_dim,
                "rotated dimensions %d: a multiple of 16 up to head_dim %d", r.rot, head_dim);
  if (r.rot == 0) return WNW_OK;
  WNW_CHECK_ARG(r.num_axes >= 1 && r.num_axes <= 4, "num_axes %d (1..4)", r.num_axes);
  WNW_CHECK_ARG(r.inv_freq && r.axis && r.pos, "rotation without frequencies, axes or positions");
  return WNW_OK;
}

}  // namespace wnw
