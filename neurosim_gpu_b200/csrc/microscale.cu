// microscale.cu -- dense matrices into NVFP4 and back (the format: nsb_nvfp4.cuh), and column sums.
//
// Quantising is bound by memory: each value is read once, 0.5625 bytes per value are written.
//   quantize_rows_kernel    one CTA per row: the row's amax, then its blocks (the second read hits L2);
//   quantize_columns_kernel the transpose: a CTA stages 64 rows x 128 columns in shared memory and
//                           encodes runs of 16 down the columns; its 512 block-scale bytes are one
//                           tile of the format.  The scales come from an amax pass before it.
#include <algorithm>

#include "nsb_nvfp4.cuh"
#include "nsb_tokens.h"

namespace nsb {
namespace {

constexpr int kRowThreads = 512;
constexpr int kTileRows = 64;   // of the input: 4 blocks of a transposed row
constexpr int kTileCols = 128;  // of the input: rows of the result
constexpr int kTileThreads = 256;
constexpr int kAmaxThreads = 256;

__device__ __forceinline__ unsigned int amax_bits(float v) { return __float_as_uint(fabsf(v)); }

// 16 consecutive values from column c of a row, zeros beyond `cols`.
template <typename T, bool kVec>
__device__ __forceinline__ void load_block(const T* row, int64_t c, int64_t cols, float (&v)[16]) {
  constexpr int P = 16 / static_cast<int>(sizeof(T));
  if (kVec && c + 16 <= cols) {
#pragma unroll
    for (int q = 0; q < 16 / P; ++q) {
      const Pack<T, P> x = load_pack<T, P>(row + c + q * P);
#pragma unroll
      for (int i = 0; i < P; ++i) v[q * P + i] = Values<T>::up(x.v[i]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = c + k < cols ? Values<T>::up(row[c + k]) : 0.0f;
  }
}

__device__ __forceinline__ unsigned int warp_max(unsigned int best) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, off));
  return best;
}

// amax: the matrix's, or null for the row's own.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kRowThreads)
quantize_rows_kernel(Dense x, Nvfp4 out, const unsigned int* amax) {
  __shared__ unsigned int best_of[kRowThreads / 32];
  const int64_t r = blockIdx.x;
  const int64_t tiles = block_scale_tiles(x.cols), blocks = tiles * 4;
  if (r >= x.rows) {  // rows that pad the last tile: their scales only
    for (int64_t b = threadIdx.x; b < blocks; b += kRowThreads) out.block_scales[block_scale_at(r, b, tiles)] = 0;
    return;
  }
  const T* row = static_cast<const T*>(x.data) + r * x.stride;
  unsigned int best = 0;
  if (amax) {
    best = *amax;
  } else {
    for (int64_t b = threadIdx.x; b * 16 < x.cols; b += kRowThreads) {
      float v[16];
      load_block<T, kVec>(row, b * 16, x.cols, v);
#pragma unroll
      for (int k = 0; k < 16; ++k) best = max(best, amax_bits(v[k]));
    }
    best = warp_max(best);
    if ((threadIdx.x & 31) == 0) best_of[threadIdx.x >> 5] = best;
    __syncthreads();
    best = warp_max(best_of[threadIdx.x & (kRowThreads / 32 - 1)]);
  }
  const float g = scale_of_amax(best);
  if (threadIdx.x == 0 && (out.per_row || r == 0)) out.scale[out.per_row ? r : 0] = g;
  for (int64_t b = threadIdx.x; b < blocks; b += kRowThreads) {
    Block4 e{0ull, 0u};
    if (b * 16 < x.cols) {
      float v[16];
      load_block<T, kVec>(row, b * 16, x.cols, v);
      e = encode_block(v, g);
    }
    out.block_scales[block_scale_at(r, b, tiles)] = static_cast<uint8_t>(e.scale);
    if (b * 8 < out.pitch) *reinterpret_cast<unsigned long long*>(out.codes + r * out.pitch + b * 8) = e.codes;
  }
}

// amax: one word, or one per column (out.per_row).
template <typename T, bool kVec>
__global__ void __launch_bounds__(kTileThreads)
quantize_columns_kernel(Dense x, Nvfp4 out, const unsigned int* amax) {
  constexpr int P = kVec ? 16 / static_cast<int>(sizeof(T)) : 1;
  __shared__ Pack<T, P> tile[kTileRows][kTileCols / P + 1];
  const int64_t across = (x.cols + kTileCols - 1) / kTileCols;
  const int64_t c0 = blockIdx.x % across * kTileCols, r0 = blockIdx.x / across * kTileRows;
  const T* data = static_cast<const T*>(x.data);
  for (int i = threadIdx.x; i < kTileRows * (kTileCols / P); i += kTileThreads) {
    const int tr = i / (kTileCols / P), tc = i - tr * (kTileCols / P);
    const int64_t r = r0 + tr, c = c0 + tc * P;
    Pack<T, P> v;
    if (r < x.rows && c + P <= x.cols) {
      v = load_pack<T, P>(data + r * x.stride + c);
    } else {
#pragma unroll
      for (int k = 0; k < P; ++k)
        v.v[k] = r < x.rows && c + k < x.cols ? data[r * x.stride + c + k] : Values<T>::down(0.0f);
    }
    tile[tr][tc] = v;
  }
  __syncthreads();
  const int64_t tiles = block_scale_tiles(x.rows);
  for (int i = threadIdx.x; i < kTileCols * 4; i += kTileThreads) {
    const int tc = i & (kTileCols - 1), b = i / kTileCols;
    const int64_t row = c0 + tc, block = r0 / 16 + b;
    Block4 e{0ull, 0u};
    if (row < x.cols) {
      const float g = scale_of_amax(amax[out.per_row ? row : 0]);
      float v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = Values<T>::up(tile[b * 16 + k][tc / P].v[tc % P]);
      e = encode_block(v, g);
      if (block == 0 && (out.per_row || row == 0)) out.scale[out.per_row ? row : 0] = g;
      if (block * 8 < out.pitch) *reinterpret_cast<unsigned long long*>(out.codes + row * out.pitch + block * 8) = e.codes;
    }
    out.block_scales[block_scale_at(row, block, tiles)] = static_cast<uint8_t>(e.scale);
  }
}

// Largest |x| of the matrix into amax[0], or of each column into amax[column]; amax starts at zero.
template <typename T>
__global__ void __launch_bounds__(kAmaxThreads)
amax_kernel(Dense x, unsigned int* amax, bool columns) {
  const T* data = static_cast<const T*>(x.data);
  if (columns) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kAmaxThreads + threadIdx.x;
    if (c >= x.cols) return;
    unsigned int best = 0;
#pragma unroll 4
    for (int64_t r = blockIdx.y; r < x.rows; r += gridDim.y) best = max(best, amax_bits(Values<T>::up(data[r * x.stride + c])));
    if (best) atomicMax(amax + c, best);
    return;
  }
  unsigned int best = 0;
  for (int64_t r = blockIdx.y; r < x.rows; r += gridDim.y)
    for (int64_t c = static_cast<int64_t>(blockIdx.x) * kAmaxThreads + threadIdx.x; c < x.cols; c += static_cast<int64_t>(gridDim.x) * kAmaxThreads)
      best = max(best, amax_bits(Values<T>::up(data[r * x.stride + c])));
  best = warp_max(best);
  if ((threadIdx.x & 31) == 0 && best) atomicMax(amax, best);
}

template <typename O>
__global__ void __launch_bounds__(kRowThreads)
dequantize_kernel(Nvfp4 in, Dense out) {
  const int64_t per_row = (in.cols + 15) / 16, tiles = block_scale_tiles(in.cols);
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x;
  const int64_t r = i / per_row, b = i - r * per_row;
  if (r >= in.rows) return;
  const unsigned long long codes = *reinterpret_cast<const unsigned long long*>(in.codes + r * in.pitch + b * 8);
  const float step = __fmul_rn(e4m3_value(in.block_scales[block_scale_at(r, b, tiles)]), in.scale[in.per_row ? r : 0]);
  O* to = static_cast<O*>(out.data) + r * out.stride + b * 16;
#pragma unroll
  for (int k = 0; k < 16; ++k)
    if (b * 16 + k < in.cols) to[k] = Values<O>::down(__fmul_rn(e2m1_value((codes >> (4 * k)) & 15u), step));
}

// Sums of the columns over rows [blockIdx.y * span, + span), in ascending rows, to row blockIdx.y of `sums`.
template <typename T>
__global__ void __launch_bounds__(kAmaxThreads)
column_sums_kernel(Dense x, int64_t span, float* sums) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kAmaxThreads + threadIdx.x;
  if (c >= x.cols) return;
  const int64_t last = min(x.rows, (blockIdx.y + 1) * span);
  float sum = 0.0f;
#pragma unroll 8
  for (int64_t r = blockIdx.y * span; r < last; ++r) sum += Values<T>::up(static_cast<const T*>(x.data)[r * x.stride + c]);
  sums[blockIdx.y * x.cols + c] = sum;
}

__global__ void __launch_bounds__(kAmaxThreads)
join_sums_kernel(const float* sums, int64_t parts, int64_t cols, float* out) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kAmaxThreads + threadIdx.x;
  if (c >= cols) return;
  float sum = 0.0f;
#pragma unroll 8
  for (int64_t p = 0; p < parts; ++p) sum += sums[p * cols + c];
  out[c] = sum;
}

// Rows per partial sum: short enough to fill the GPU, and at most 1,024 parts.
int64_t sum_span(int64_t rows) { return std::max<int64_t>(64, (rows + 1023) / 1024); }

unsigned ceil_div(int64_t a, int64_t b) { return static_cast<unsigned>((a + b - 1) / b); }

}  // namespace

size_t nvfp4_quantize_workspace_bytes(const Nvfp4& out, bool transpose) {
  if (out.per_row) return transpose ? static_cast<size_t>(out.rows) * 4 : 0;
  return 4;
}

cudaError_t launch_nvfp4_quantize(const Dense& value, bool transpose, const Nvfp4& out,
                                  void* workspace, cudaStream_t stream) {
  return with_type(value.type, [&](auto zero) {
    using T = decltype(zero);
    auto* amax = static_cast<unsigned int*>(workspace);
    cudaError_t err = cudaSuccess;
    const size_t bytes = nvfp4_quantize_workspace_bytes(out, transpose);
    if (bytes > 0) {
      err = cudaMemsetAsync(amax, 0, bytes, stream);
      if (err != cudaSuccess) return err;
      const bool columns = out.per_row;
      const dim3 grid(std::min(ceil_div(value.cols, kAmaxThreads), 0x7fffffffu), static_cast<unsigned>(std::min<int64_t>(value.rows, 256)));
      amax_kernel<T><<<grid, kAmaxThreads, 0, stream>>>(value, amax, columns);
      err = cudaGetLastError();
      if (err != cudaSuccess) return err;
    }
    const bool vec = rows_aligned(value, sizeof(T), 16);
    if (transpose) {
      const unsigned grid = ceil_div(value.cols, kTileCols) * static_cast<unsigned>(block_scale_tiles(value.rows));
      if (vec)
        quantize_columns_kernel<T, true><<<grid, kTileThreads, 0, stream>>>(value, out, amax);
      else
        quantize_columns_kernel<T, false><<<grid, kTileThreads, 0, stream>>>(value, out, amax);
    } else {
      const unsigned grid = ceil_div(value.rows, 128) * 128;
      const unsigned int* given = bytes > 0 ? amax : nullptr;
      if (vec)
        quantize_rows_kernel<T, true><<<grid, kRowThreads, 0, stream>>>(value, out, given);
      else
        quantize_rows_kernel<T, false><<<grid, kRowThreads, 0, stream>>>(value, out, given);
    }
    return cudaGetLastError();
  });
}

cudaError_t launch_nvfp4_dequantize(const Nvfp4& in, const Dense& out, cudaStream_t stream) {
  return with_type(out.type, [&](auto zero) {
    using T = decltype(zero);
    const int64_t blocks = (in.cols + 15) / 16 * in.rows;
    dequantize_kernel<T><<<ceil_div(blocks, kRowThreads), kRowThreads, 0, stream>>>(in, out);
    return cudaGetLastError();
  });
}

size_t column_sums_workspace_bytes(int64_t rows, int64_t cols) {
  return static_cast<size_t>((rows + sum_span(rows) - 1) / sum_span(rows) * cols) * 4;
}

cudaError_t launch_column_sums(const Dense& value, float* out, void* workspace, cudaStream_t stream) {
  return with_type(value.type, [&](auto zero) {
    using T = decltype(zero);
    auto* sums = static_cast<float*>(workspace);
    const int64_t span = sum_span(value.rows), parts = (value.rows + span - 1) / span;
    const dim3 grid(ceil_div(value.cols, kAmaxThreads), static_cast<unsigned>(parts));
    if (parts > 0) {  // no rows: the sums are zero
      column_sums_kernel<T><<<grid, kAmaxThreads, 0, stream>>>(value, span, sums);
      const cudaError_t err = cudaGetLastError();
      if (err != cudaSuccess) return err;
    }
    join_sums_kernel<<<grid.x, kAmaxThreads, 0, stream>>>(sums, parts, value.cols, out);
    return cudaGetLastError();
  });
}

}  // namespace nsb
