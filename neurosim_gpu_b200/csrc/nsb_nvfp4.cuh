// nsb_nvfp4.cuh -- the dense NVFP4 format on the device: 16 consecutive values of a row to
// codes and a block scale, and where a block's scale lies.
//
//   scale       g = max(amax / 2688, FLT_MIN)          (2688 = 6 * 448; amax of the row or matrix)
//   block scale s = e4m3(min(block_amax / (6 g), 448))
//   code          E2M1 level nearest to |x| / (g s), a tie to the even code; sign in bit 3
//   value         level * (s g)
// the same steps as the sparse weights' encoder (encode.cu), with every quotient an IEEE one.  A
// row (or matrix) that holds an infinity or a NaN gets g = NaN and zero codes: what is read back
// or multiplied from it is NaN everywhere, so the fault stays visible.
#pragma once

#include "nsb_device.cuh"
#include "nsb_values.cuh"

namespace nsb {

constexpr float kScaleLeast = 1.17549435082228750797e-38f;  // FLT_MIN

// Block scales lie as the tensor core reads them: a 512-byte tile holds 128 rows x 4 blocks.
__device__ __forceinline__ int64_t block_scale_at(int64_t row, int64_t block, int64_t tiles) {
  return ((row >> 7) * tiles + (block >> 2)) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4 + (block & 3);
}
// 512-byte tiles per 128 rows: columns are padded to 256.
__host__ __device__ __forceinline__ int64_t block_scale_tiles(int64_t cols) { return (cols + 255) / 256 * 4; }

__device__ __forceinline__ uint32_t e4m3_round(float x) {
  unsigned short pair;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(pair) : "f"(0.0f), "f"(x));
  return pair & 0xffu;
}

__device__ __forceinline__ float scale_of_amax(unsigned int bits) {
  if (bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return fmaxf(__fdiv_rn(__uint_as_float(bits), 2688.0f), kScaleLeast);
}

__device__ __forceinline__ uint32_t e2m1_round(float x) {
  return static_cast<uint32_t>(x > 0.25f) + static_cast<uint32_t>(x >= 0.75f) +
         static_cast<uint32_t>(x > 1.25f) + static_cast<uint32_t>(x >= 1.75f) +
         static_cast<uint32_t>(x > 2.5f) + static_cast<uint32_t>(x >= 3.5f) +
         static_cast<uint32_t>(x > 5.0f);
}

struct Block4 {
  unsigned long long codes;  // code k in bits [4k, 4k + 4)
  uint32_t scale;            // E4M3
};

__device__ __forceinline__ Block4 encode_block(const float (&v)[16], float g) {
  if (!(g < __uint_as_float(0x7f800000u))) return {0ull, 0u};  // NaN: see above
  float amax = 0.0f;
#pragma unroll
  for (int k = 0; k < 16; ++k) amax = fmaxf(amax, fabsf(v[k]));
  Block4 r;
  r.scale = e4m3_round(fminf(__fdiv_rn(amax, __fmul_rn(6.0f, g)), 448.0f));
  const float step = __fmul_rn(g, e4m3_value(r.scale));
  const float divisor = step > 0.0f ? step : 1.0f;
  r.codes = 0ull;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const unsigned long long code = e2m1_round(__fdiv_rn(fabsf(v[k]), divisor)) |
                                    ((__float_as_uint(v[k]) >> 31) << 3);
    r.codes |= code << (4 * k);
  }
  return r;
}

}  // namespace nsb
