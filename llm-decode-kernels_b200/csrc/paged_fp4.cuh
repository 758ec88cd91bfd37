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

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Quantises the 8 values of this lane, whose 16-dim group the lane's neighbour (lane ^ 1) has the other half of: the codes as 4
// bytes, and the group's scale. The values come from a 16-bit type; inv_power is a power of two.
//   scale = E4M3(max |x| / 6),  code = E2M1(x / scale), both to nearest, ties to even; infinities saturate, a NaN makes the scale NaN
// The division by the scale is a product with its reciprocal, off by 2^-23 of the ratio. A ratio either is a border between two
// codes, which has at most 3 bits, or is 2^-13 away from it at least: x has 11 bits, border * scale 7, so their difference is
// a unit of x's last place or more, and the smallest border is 1/4. So the ratio is first rounded to a multiple of 2^-16
// (adding and taking away 192, whose neighbours are 2^-16 apart), which puts exact borders back in their places.
__device__ __forceinline__ uint32_t fp4_quantise8(const float (&x)[8], float inv_power, int lane, uint8_t& scale) {
  float y[8], m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = x[i] * inv_power;
    m = max_nan(m, fabsf(y[i]));
  }
  m = max_nan(m, __shfl_xor_sync(3u << (lane & 30), m, 1));  // (the two lanes of a group are always in the same branch)
  uint16_t bits;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(bits) : "f"(0.f), "f"(__fdiv_rn(m, 6.f)));
  scale = static_cast<uint8_t>(bits);
  const float s = fp4_scale(scale), r = s == 0.f ? 0.f : __frcp_rn(s);
  uint32_t code = 0;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float a[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float t = fabsf(y[i + j]) * r;
      a[j] = copysignf(__fsub_rn(__fadd_rn(t, 192.f), 192.f), x[i + j]);
    }
    uint32_t byte;
    asm("{\n.reg .b8 a, z;\nmov.b16 {z, _}, 0;\ncvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\nmov.b32 %0, {a, z, z, z};\n}"
        : "=r"(byte)
        : "f"(a[0]), "f"(a[1]));
    code |= byte << (4 * i);
  }
  return code;
}

// A pool's power of two that the kernels take.
inline bool fp4_power(double x) {
  int e;
  return x > 0. && std::frexp(x, &e) == 0.5 && e >= -63 && e <= 65;  // (x = 0.5 * 2^e; an infinity or a NaN is not 0.5)
}

}  // namespace paged
}  // namespace dk
