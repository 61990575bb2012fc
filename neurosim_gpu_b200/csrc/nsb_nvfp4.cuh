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

// Two float32 values in one register pair, for the packed float32 instructions.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair_of(float low, float high) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(low), "f"(high));
  return p;
}
__device__ __forceinline__ void split(Pair p, float* low, float* high) { asm("mov.b64 {%0, %1}, %2;" : "=f"(*low), "=f"(*high) : "l"(p)); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// E2M1 codes of eight numbers (nearest, ties to even, saturated, sign kept), the first in the low nibble.
__device__ __forceinline__ uint32_t e2m1_round8(const Pair* x) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) split(x[i], &v[2 * i], &v[2 * i + 1]);
  uint32_t codes;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(codes)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return codes;
}

// The exact value of an E4M3 byte that is not NaN, by way of float16, which holds them all.
__device__ __forceinline__ float e4m3_exact(uint32_t code) {
  uint32_t halves;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(halves) : "h"(static_cast<unsigned short>(code)));
  return __half2float(__ushort_as_half(static_cast<unsigned short>(halves & 0xffffu)));
}

// The levels of eight codes, the first in the low nibble.
__device__ __forceinline__ void e2m1_levels8(uint32_t codes, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = x.x;
    v[2 * i + 1] = x.y;
  }
}

struct Block4 {
  unsigned long long codes;  // code k in bits [4k, 4k + 4)
  uint32_t scale;            // E4M3
};

static __device__ __noinline__ uint32_t e2m1_divided(float x, float divisor) {
  return e2m1_round(__fdiv_rn(fabsf(x), divisor)) | (__float_as_uint(x) >> 31) << 3;
}

// v: the block's 16 values; amax: the bits of the largest size among them.
// The codes go by the float32 quotients q = x / (g s).  One correctly rounded reciprocal y serves the
// block: x y is within two units of q, and a step q + y (x - q d), the difference exact by FMA, taken
// twice gives the quotient that division gives (Markstein's theorem asks for q within one unit before
// the last step).  Held negated, it keeps the sign of a zero.  Two values per instruction: 40 for the
// block, where 16 divisions take about 200.
__device__ __forceinline__ Block4 encode_block(const Pair (&v)[8], unsigned int amax, float g) {
  if (!(g < __uint_as_float(0x7f800000u))) return {0ull, 0u};  // NaN: see above
  Block4 r;
  r.scale = e4m3_round(fminf(__fdiv_rn(__uint_as_float(amax), __fmul_rn(6.0f, g)), 448.0f));
  const float step = __fmul_rn(g, e4m3_exact(r.scale));
  const float divisor = step > 0.0f ? step : 1.0f;
  if (divisor < 1e-28f) {  // the differences would not be exact any more
    r.codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float low, high;
      split(v[i], &low, &high);
      r.codes |= static_cast<unsigned long long>(e2m1_divided(low, divisor) | e2m1_divided(high, divisor) << 4) << (8 * i);
    }
    return r;
  }
  const float inverse = __frcp_rn(divisor);
  const Pair d = pair_of(divisor, divisor), minus_y = pair_of(-inverse, -inverse);
  Pair q[8];  // minus the quotients
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    q[i] = mul2(v[i], minus_y);
    q[i] = fma2(minus_y, fma2(d, q[i], v[i]), q[i]);
    q[i] = fma2(minus_y, fma2(d, q[i], v[i]), q[i]);
  }
  r.codes = (static_cast<unsigned long long>(e2m1_round8(q + 4)) << 32 | e2m1_round8(q)) ^ 0x8888888888888888ull;
  return r;
}

}  // namespace nsb
