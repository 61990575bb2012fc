// microscale_product.cu -- the product of two dense NVFP4 matrices (the format: nsb_nvfp4.cuh):
//
//   out[m, n] = round( (sum_k level_a sa level_b sb) * ga[m] * gb[n] + bias[n] )
//
// with the sum in float32.  One CTA computes a 64 x 64 tile, one block of 16 columns at a time,
// decoded to shared memory (levels times E4M3 scales are exact in float32).
#include "nsb_nvfp4.cuh"
#include "nsb_tokens.h"

namespace nsb {
namespace {

constexpr int kSide = 64;

template <typename O>
__global__ void __launch_bounds__(256)
product_kernel(Nvfp4 a, Nvfp4 b, const float* bias, Dense out, int64_t n_tiles) {
  __shared__ float as[16][kSide + 1], bs[16][kSide + 1];
  const int64_t m0 = blockIdx.x / n_tiles * kSide, n0 = (blockIdx.x % n_tiles) * kSide;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t blocks = (a.cols + 15) / 16, tiles = block_scale_tiles(a.cols);
  float acc[4][4] = {};
  for (int64_t k = 0; k < blocks; ++k) {
    for (int i = threadIdx.x; i < 2 * kSide * 2; i += 256) {
      const int half = i & 1, r = (i >> 1) & (kSide - 1);
      const bool second = i >= 2 * kSide;
      const Nvfp4& x = second ? b : a;
      const int64_t row = (second ? n0 : m0) + r;
      uint32_t codes = 0;
      float s = 0.0f;
      if (row < x.rows) {
        codes = *reinterpret_cast<const uint32_t*>(x.codes + row * x.pitch + k * 8 + half * 4);
        s = e4m3_value(x.block_scales[block_scale_at(row, k, tiles)]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) (second ? bs : as)[half * 8 + j][r] = e2m1_value((codes >> (4 * j)) & 15u) * s;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = as[j][ty * 4 + i];
        y[i] = bs[j][tx * 4 + i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int l = 0; l < 4; ++l) acc[i][l] = fmaf(x[i], y[l], acc[i][l]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int l = 0; l < 4; ++l) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + l;
      if (m < out.rows && n < out.cols) {
        const float y = acc[i][l] * a.scale[a.per_row ? m : 0] * b.scale[b.per_row ? n : 0];
        static_cast<O*>(out.data)[m * out.stride + n] = Values<O>::down(bias ? y + bias[n] : y);
      }
    }
}

}  // namespace

cudaError_t launch_nvfp4_product(const Nvfp4& a, const Nvfp4& b, const float* bias, const Dense& out,
                                 int* status, cudaStream_t stream) {
  (void)status;
  return with_type(out.type, [&](auto zero) {
    using O = decltype(zero);
    const int64_t m_tiles = (out.rows + kSide - 1) / kSide, n_tiles = (out.cols + kSide - 1) / kSide;
    if (m_tiles * n_tiles > 0x7fffffff) return cudaErrorInvalidConfiguration;
    product_kernel<O><<<static_cast<unsigned>(m_tiles * n_tiles), 256, 0, stream>>>(a, b, bias, out, n_tiles);
    return cudaGetLastError();
  });
}

}  // namespace nsb
