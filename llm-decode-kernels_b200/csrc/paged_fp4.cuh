// A paged cache held in 4 bits: what its kernels share.
//
// A value is code * scale * power: a 4-bit E2M1 code (a sign and 0, 0.5, 1, 1.5, 2, 3, 4 or 6), an E4M3 scale for each 16 dims of
// a position, and a power of two for the whole pool. The significands have 2 and 4 bits, so code * scale is exact in fp16 (a
// multiple of 2^-10 up to 2688) and in bf16, and nothing is lost between the cache and the products.
// A pool is [n_pages, n_kv, page_size, 9/16 head_dim] bytes; the block of a (page, kv head) holds the codes first,
// head_dim / 2 bytes a position (dim 2 i in the low half of byte i), then the scales, head_dim / 16 bytes a position.
#pragma once

#include <cmath>

#include "paged.cuh"

namespace dk {
namespace paged {

template <int kHd>
struct Fp4 {
  static constexpr int kCodes = kHd / 2, kScales = kHd / 16, kRow = kCodes + kScales;  // bytes of a position
};

// The values of four bytes' codes: d[i] has byte i's, its low half first. (w: four bytes loaded as such. Given a loaded byte widened to 32 bits,
// nvcc 12.9 produced code that gave zeros.)
__device__ __forceinline__ void fp4_codes(uint32_t w, uint32_t (&d)[4]) {
  asm("{\n.reg .b8 a, b, c, e;\nmov.b32 {a, b, c, e}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, a;\ncvt.rn.f16x2.e2m1x2 %1, b;\ncvt.rn.f16x2.e2m1x2 %2, c;\ncvt.rn.f16x2.e2m1x2 %3, e;\n}"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(w));
}

// Two scales (the low 16 bits of w) as fp16.
__device__ __forceinline__ uint32_t fp4_scales(uint32_t w) {
  uint32_t d;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(static_cast<uint16_t>(w)));
  return d;
}

__device__ __forceinline__ float fp4_scale(uint8_t w) {
  const uint32_t d = fp4_scales(w);
  return __low2float(*reinterpret_cast<const __half2*>(&d));
}

// max and min that keep a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Quantises the 8 values of this lane, whose 16-dim group the lane's neighbour (lane ^ 1) has the other half of: the codes as 4
// bytes, and the group's scale. The values come from a 16-bit type; inv_power is a power of two.
//   scale = E4M3(max |x| / 6),  code = E2M1(x / scale), both to nearest, ties to even; infinities saturate, a NaN makes the scale NaN
// Both divisions are products with a reciprocal, off by less than 2^-21 of the ratio, which is then rounded to a grid that has the
// borders between the results on it and is far finer than the distance of any other ratio from a border:
// * max / 6 to 16 bits (t 257 - (t 257 - t)). A border between two scales has 5 bits and 6 times it 7, the maximum 11: where they
//   differ, it is by the maximum's last place, 2^-11 of it, or more;
// * x / scale to multiples of 2^-16 (adding and taking away 192, whose neighbours are 2^-16 apart). A border has at most 3 bits and
//   border * scale 7, x 11: where they differ, the ratio is 2^-13 away from the border or more, the smallest border being 1/4.
__device__ __forceinline__ uint32_t fp4_quantise8(const float (&x)[8], float inv_power, int lane, uint8_t& scale) {
  float m = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(x[i]));
  m = max_nan(m, __shfl_xor_sync(3u << (lane & 30), m, 1));  // (the two lanes of a group are always in the same branch)
  const float t = min_nan(m * inv_power * (1.f / 6.f), 512.f), c = __fmul_rn(t, 257.f);
  uint16_t bits;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(bits) : "f"(0.f), "f"(__fsub_rn(c, __fsub_rn(c, t))));
  scale = static_cast<uint8_t>(bits);
  const float s = fp4_scale(scale);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  r = s == 0.f ? 0.f : r * inv_power;
  float a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = copysignf(__fsub_rn(__fadd_rn(fabsf(x[i] * r), 192.f), 192.f), x[i]);
  uint32_t code;
  asm("{\n.reg .b8 a, b, c, e;\n"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 e, %8, %7;\nmov.b32 %0, {a, b, c, e};\n}"
      : "=r"(code)
      : "f"(a[0]), "f"(a[1]), "f"(a[2]), "f"(a[3]), "f"(a[4]), "f"(a[5]), "f"(a[6]), "f"(a[7]));
  return code;
}

// A pool's power of two that the kernels take.
inline bool fp4_power(double x) {
  int e;
  return x > 0. && std::frexp(x, &e) == 0.5 && e >= -63 && e <= 65;  // (x = 0.5 * 2^e; an infinity or a NaN is not 0.5)
}

}  // namespace paged
}  // namespace dk
