// microscale.cu -- dense matrices into NVFP4 and back (the format: nsb_nvfp4.cuh), and column sums.
//
// Quantising is bound by memory: each value is read once, 0.5625 bytes per value are written.
//   quantize_rows_kernel    a row's blocks stay in registers between its amax and the codes: 16 ...
//                           256 threads per row, or a cluster of CTAs for long rows, whose amaxes
//                           are joined over distributed shared memory;
//   quantize_columns_kernel the transpose: a CTA stages 128 rows x 64 columns in shared memory,
//                           encodes runs of 16 down the columns, and collects a column's codes
//                           there, so that they leave as 64 consecutive bytes.
// One scale for the whole matrix, and the scales of a transpose, need an amax pass before.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "nsb_nvfp4.cuh"
#include "nsb_tokens.h"

namespace cg = cooperative_groups;

namespace nsb {
namespace {

constexpr int kRowThreads = 256;
constexpr int kTileRows = 128;  // of the input: 8 blocks of a transposed row
constexpr int kTileCols = 64;   // of the input: rows of the result
constexpr int kTileThreads = 256;
constexpr int kAmaxThreads = 256;

__device__ __forceinline__ unsigned int amax_bits(float v) { return __float_as_uint(fabsf(v)); }

// Two 16-bit values of a word as float32.
template <typename T>
__device__ __forceinline__ Pair widen(uint32_t word) {
  if constexpr (Values<T>::kType == NSB_VALUE_BF16) return pair_of(__uint_as_float(word << 16), __uint_as_float(word & 0xffff0000u));
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&word));
  return pair_of(v.x, v.y);
}

// 16 consecutive values as 32-bit words.
template <typename T>
struct Words {
  static constexpr int kCount = 4 * static_cast<int>(sizeof(T));
  uint32_t w[kCount];
  __device__ __forceinline__ void pairs(Pair (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 4) v[i] = pair_of(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
      else v[i] = widen<T>(w[i]);
    }
  }
  // The bits, as a float32, of the largest size: of 16-bit types two sizes at a time, ordered like their bits.
  __device__ __forceinline__ unsigned int amax() const {
    unsigned int best = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < kCount; ++i) best = max(best, w[i] & 0x7fffffffu);
      return best;
    } else {
#pragma unroll
      for (int i = 0; i < kCount; ++i) best = __vmaxu2(best, w[i] & 0x7fff7fffu);
      best = max(best & 0xffffu, best >> 16);
      return __float_as_uint(Values<T>::up(*reinterpret_cast<const T*>(&best)));
    }
  }
};

// The values from column c of a row, zeros beyond `cols`.  kVec: rows start on that many bytes, 32 or 16
// (a lane's 64 bytes of float32 in two loads instead of four halve the work of L1).  Where it is 0 a row
// starts `lead` values after a multiple of 16 bytes: the words are cut out of the aligned vectors
// around them, as long as these lie within the matrix, [first, last).
template <typename T, int kVec>
__device__ __forceinline__ Words<T> load_block(const T* row, int64_t c, int64_t cols, int lead, const T* first, const T* last) {
  constexpr int P = 16 / static_cast<int>(sizeof(T)), kVectors = 16 / P;
  Words<T> r;
  if (kVec == 32 && c + 16 <= cols) {
#pragma unroll
    for (int q = 0; q < kVectors / 2; ++q)
      asm("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
          : "=r"(r.w[8 * q]), "=r"(r.w[8 * q + 1]), "=r"(r.w[8 * q + 2]), "=r"(r.w[8 * q + 3]), "=r"(r.w[8 * q + 4]),
            "=r"(r.w[8 * q + 5]), "=r"(r.w[8 * q + 6]), "=r"(r.w[8 * q + 7])
          : "l"(row + c + 2 * q * P));
    return r;
  }
  if (kVec == 16 && c + 16 <= cols) {
#pragma unroll
    for (int q = 0; q < kVectors; ++q) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(row + c) + q);
      r.w[4 * q] = x.x, r.w[4 * q + 1] = x.y, r.w[4 * q + 2] = x.z, r.w[4 * q + 3] = x.w;
    }
    return r;
  }
  if (c >= cols) {
#pragma unroll
    for (int i = 0; i < Words<T>::kCount; ++i) r.w[i] = 0;
    return r;
  }
  const T* from = row + c - lead;
  if (!kVec && c + 16 <= cols && from >= first && from + 16 + P <= last) {
    uint32_t all[4 * kVectors + 4];
#pragma unroll
    for (int q = 0; q <= kVectors; ++q) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(from) + q);
      all[4 * q] = x.x, all[4 * q + 1] = x.y, all[4 * q + 2] = x.z, all[4 * q + 3] = x.w;
    }
    const int words = lead * static_cast<int>(sizeof(T)) / 4, bits = lead * static_cast<int>(sizeof(T)) % 4 * 8;
    auto cut = [&](auto skip) {
#pragma unroll
      for (int i = 0; i < Words<T>::kCount; ++i) {
        constexpr int kSkip = decltype(skip)::value;
        if constexpr (sizeof(T) == 4) r.w[i] = all[i + kSkip];
        else r.w[i] = __funnelshift_r(all[i + kSkip], all[i + kSkip + 1], bits);
      }
    };
    if (words == 0) cut(std::integral_constant<int, 0>{});
    else if (words == 1) cut(std::integral_constant<int, 1>{});
    else if (words == 2) cut(std::integral_constant<int, 2>{});
    else cut(std::integral_constant<int, 3>{});
    return r;
  }
  T v[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) v[k] = c + k < cols ? row[c + k] : Values<T>::down(0.0f);
#pragma unroll
  for (int i = 0; i < Words<T>::kCount; ++i) {
    if constexpr (sizeof(T) == 4) r.w[i] = __float_as_uint(v[i]);
    else r.w[i] = *reinterpret_cast<const uint16_t*>(&v[2 * i]) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&v[2 * i + 1])) << 16;
  }
  return r;
}

__device__ __forceinline__ unsigned int warp_max(unsigned int best) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, off));
  return best;
}

template <typename T>
__device__ __forceinline__ void write_block(const Nvfp4& out, int64_t r, int64_t b, int64_t tiles, int64_t blocks,
                                            const Words<T>& v, unsigned int amax, float g) {
  Pair x[8];
  v.pairs(x);
  const Block4 e = encode_block(x, amax, g);
  // Four neighbouring lanes hold four neighbouring blocks of the row: one word of scales.
  uint32_t scales = e.scale | __shfl_down_sync(0xffffffffu, e.scale, 1) << 8;
  scales |= __shfl_down_sync(0xffffffffu, scales, 2) << 16;
  if (r >= out.rows) return;
  if (b < blocks && (b & 3) == 0) *reinterpret_cast<uint32_t*>(out.block_scales + block_scale_at(r, b, tiles)) = scales;
  if (b * 8 < out.pitch) *reinterpret_cast<unsigned long long*>(out.codes + r * out.pitch + b * 8) = e.codes;
}

// 2^per_row threads (16 ... 256) take a row, the CTA's 256 several rows; or a cluster of 2^cluster CTAs
// takes one.  B blocks per thread stay in registers, further ones are read twice.  `given`: the matrix's amax (its bits), or null
// for each row's own; `most`: receives the matrix's amax (zero before), or null.
// Bound by the encoding's instructions (17 per value, 65 % of the issue slots): 8,192 x 4,096 bf16 24 us, 3.6 TB/s.
template <typename T, int kVec, int B>
__global__ void __launch_bounds__(kRowThreads)
quantize_rows_kernel(Dense x, Nvfp4 out, const unsigned int* given, unsigned int* most, int per_row, int cluster, unsigned work) {
  __shared__ unsigned int best_of[kRowThreads / 32];
  __shared__ unsigned int cta_best;
  asm volatile("griddepcontrol.launch_dependents;");  // a product after it may start (and wait)
  if (blockIdx.x >= work) {  // zero scales for the rows that fill up the last 128
    const int64_t tiles = block_scale_tiles(x.cols);
    const int word = threadIdx.x & 127, row = (word & 3) * 32 + (word >> 2);
    auto* scales = reinterpret_cast<uint32_t*>(out.block_scales) + (x.rows >> 7) * tiles * 128 + word;
    if (row >= (x.rows & 127))
      for (int64_t t = (blockIdx.x - work) * 2 + (threadIdx.x >> 7); t < tiles; t += (gridDim.x - work) * 2) scales[t * 128] = 0;
    return;
  }
  const int part = blockIdx.x & ((1 << cluster) - 1);
  const int64_t r = cluster > 0 ? blockIdx.x >> cluster : (static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x) >> per_row;
  const int64_t tiles = block_scale_tiles(x.cols), blocks = tiles * 4;
  const int step = 1 << (per_row + cluster);
  const int64_t first = (part << per_row) + (threadIdx.x & ((1 << per_row) - 1));
  const int lane = threadIdx.x & 31 & ((1 << per_row) - 1);  // of the warp's threads on this row
  const int64_t cols = r < x.rows ? x.cols : 0;
  const T* row = static_cast<const T*>(x.data) + (r < x.rows ? r : 0) * x.stride;
  const T* data = static_cast<const T*>(x.data);
  const T* end = data + (x.rows - 1) * x.stride + x.cols;
  const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
  auto load = [&](int64_t b) { return load_block<T, kVec>(row, b * 16, cols, lead, data, end); };
  Words<T> v[B];
  unsigned int amax[B];
  unsigned int best = 0;
#pragma unroll
  for (int i = 0; i < B; ++i) v[i] = load(first + i * step);
#pragma unroll
  for (int i = 0; i < B; ++i) best = max(best, amax[i] = v[i].amax());
  if (given) {
    best = __ldg(given);
  } else {
    for (int64_t b = first + B * step; b * 16 < cols; b += step) best = max(best, load(b).amax());
    if (per_row > 4) best = __reduce_max_sync(0xffffffffu, best);
    else best = __reduce_max_sync(0xffffu << (threadIdx.x & 16), best);
    if (per_row > 5) {
      if ((threadIdx.x & 31) == 0) best_of[threadIdx.x >> 5] = best;
      __syncthreads();
      const int warps = 1 << (per_row - 5), own = threadIdx.x >> per_row << (per_row - 5);
      best = __reduce_max_sync(0xffffffffu, best_of[own + (threadIdx.x & (warps - 1))]);
    }
    if (cluster > 0) {
      cg::cluster_group group = cg::this_cluster();
      if (threadIdx.x == 0) cta_best = best;
      group.sync();
      best = 0;
      for (int c = 0; c < 1 << cluster; ++c) best = max(best, *group.map_shared_rank(&cta_best, c));
      group.sync();  // no CTA leaves while its word is read
    }
  }
  const float g = scale_of_amax(best);
  if (first == 0 && r < x.rows) {
    if (out.per_row || r == 0) out.scale[out.per_row ? r : 0] = g;
    if (most) atomicMax(most, best);
  }
#pragma unroll
  for (int i = 0; i < B; ++i)
    if (first - lane + i * step < blocks) write_block(out, r, first + i * step, tiles, blocks, v[i], amax[i], g);  // whole warps
  for (int64_t b = first + B * step; b - lane < blocks; b += step) {
    const Words<T> w = load(b);
    write_block(out, r, b, tiles, blocks, w, w.amax(), g);
  }
}

// amax: one word, or one per column (out.per_row).  As the rows' kernel, and the tile's way through shared memory:
// 8,190 x 4,104 bf16 37 us.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kTileThreads)
quantize_columns_kernel(Dense x, Nvfp4 out, const unsigned int* amax) {
  constexpr int P = kVec ? 16 / static_cast<int>(sizeof(T)) : 1;
  constexpr int kAcross = kTileCols / P, kLoads = kTileRows * kAcross / kTileThreads;
  constexpr int kRowBytes = kTileCols * static_cast<int>(sizeof(T)) + 16;  // odd multiples of 16: fewer bank conflicts
  __shared__ alignas(16) uint8_t tile[kTileRows * kRowBytes];
  auto place = [&](int at) -> Pack<T, P>& { return *reinterpret_cast<Pack<T, P>*>(tile + at / kAcross * kRowBytes + at % kAcross * sizeof(Pack<T, P>)); };
  __shared__ unsigned long long codes[kTileCols][kTileRows / 16 + 1];
  __shared__ uint8_t scales[kTileCols][kTileRows / 16 + 4];
  const unsigned across = static_cast<unsigned>((x.cols + 127) / 128 * 2);  // the result's rows are padded to 128 for their scales
  const unsigned down = blockIdx.x / across;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x - down * across) * kTileCols, r0 = static_cast<int64_t>(down) * kTileRows;
  const T* data = static_cast<const T*>(x.data);
  Pack<T, P> v[kVec ? kLoads : 1];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int at = threadIdx.x + i * kTileThreads, tr = at / kAcross, tc = at % kAcross;
    const int64_t r = r0 + tr, c = c0 + tc * P;
    Pack<T, P>& to = v[kVec ? i : 0];
    if (r < x.rows && c + P <= x.cols) {
      to = load_pack<T, P>(data + r * x.stride + c);
    } else {
#pragma unroll
      for (int k = 0; k < P; ++k)
        to.v[k] = r < x.rows && c + k < x.cols ? data[r * x.stride + c + k] : Values<T>::down(0.0f);
    }
    if (!kVec) place(at) = to;
  }
  if (kVec) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = threadIdx.x + i * kTileThreads;
      place(at) = v[i];
    }
  }
  auto scale_at = [&](int64_t row) { return scale_of_amax(row < x.cols ? __ldg(amax + (out.per_row ? row : 0)) : 0u); };
  if (r0 == 0 && threadIdx.x < kTileCols) {
    const int64_t row = c0 + threadIdx.x;
    if (row < x.cols && (out.per_row || row == 0)) out.scale[out.per_row ? row : 0] = scale_at(row);
  }
  __syncthreads();
  {  // a warp takes one block of all 64 columns, two neighbouring columns to a lane
    const int b = threadIdx.x >> 5, c = 2 * (threadIdx.x & 31);
    const uint8_t* from = reinterpret_cast<const uint8_t*>(tile) + b * 16 * kRowBytes + c * sizeof(T);
    Pair even[8], odd[8];
    unsigned int most[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 16; k += 2) {
      float v[2][2];  // [row][column]
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const Pack<T, 2> x = *reinterpret_cast<const Pack<T, 2>*>(from + (k + i) * kRowBytes);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          v[i][j] = Values<T>::up(x.v[j]);
          most[j] = max(most[j], amax_bits(v[i][j]));
        }
      }
      even[k / 2] = pair_of(v[0][0], v[1][0]);
      odd[k / 2] = pair_of(v[0][1], v[1][1]);
    }
    const float g[2] = {scale_at(c0 + c), scale_at(c0 + c + 1)};
    const Block4 e = encode_block(even, most[0], g[0]), o = encode_block(odd, most[1], g[1]);
    codes[c][b] = e.codes;
    codes[c + 1][b] = o.codes;
    scales[c][b] = static_cast<uint8_t>(e.scale);
    scales[c + 1][b] = static_cast<uint8_t>(o.scale);
  }
  __syncthreads();
  {  // four threads write a row's 64 bytes of codes
    const int to = threadIdx.x / 4, pair = threadIdx.x % 4;
    const int64_t byte = r0 / 2 + pair * 16;  // the pitch is a multiple of 16
    if (c0 + to < x.cols && byte < out.pitch)
      *reinterpret_cast<ulonglong2*>(out.codes + (c0 + to) * out.pitch + byte) = make_ulonglong2(codes[to][2 * pair], codes[to][2 * pair + 1]);
  }
  if (threadIdx.x < 2 * kTileCols) {
    const int to = threadIdx.x % kTileCols, half = threadIdx.x / kTileCols;
    *reinterpret_cast<uint32_t*>(out.block_scales + block_scale_at(c0 + to, r0 / 16 + 4 * half, block_scale_tiles(x.rows))) =
        *reinterpret_cast<const uint32_t*>(&scales[to][4 * half]);
  }
}

// Largest |x| of the matrix into *amax (its bits; zero before).  Contiguous matrices come as one row.
// 8,190 x 4,104 bf16: 17.5 us, 3.8 TB/s.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kAmaxThreads)
amax_kernel(Dense x, unsigned int* amax) {
  constexpr int P = kVec ? 16 / static_cast<int>(sizeof(T)) : 1;
  constexpr int U = 4;
  __shared__ unsigned int best_of[kAmaxThreads / 32];
  const T* data = static_cast<const T*>(x.data);
  unsigned int best = 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kAmaxThreads;
  const int64_t vectors = x.cols / P;
  for (int64_t r = blockIdx.y; r < x.rows; r += gridDim.y) {
    const T* row = data + r * x.stride;
    int64_t i = static_cast<int64_t>(blockIdx.x) * kAmaxThreads + threadIdx.x;
    for (; i + (U - 1) * step < vectors; i += U * step) {
      Pack<T, P> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = load_pack<T, P>(row + (i + u * step) * P);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < P; ++k) best = max(best, amax_bits(Values<T>::up(v[u].v[k])));
    }
    for (; i < vectors; i += step) {
      const Pack<T, P> v = load_pack<T, P>(row + i * P);
#pragma unroll
      for (int k = 0; k < P; ++k) best = max(best, amax_bits(Values<T>::up(v.v[k])));
    }
    if (blockIdx.x == 0 && vectors * P + threadIdx.x < x.cols) best = max(best, amax_bits(Values<T>::up(row[vectors * P + threadIdx.x])));
  }
  best = warp_max(best);
  if ((threadIdx.x & 31) == 0) best_of[threadIdx.x >> 5] = best;
  __syncthreads();
  if (threadIdx.x < 32) {
    best = warp_max(best_of[threadIdx.x & (kAmaxThreads / 32 - 1)]);
    if (threadIdx.x == 0 && best) atomicMax(amax, best);
  }
}

// ... of each column into amax[column].  A CTA takes 32 * P columns; its 8 warps share the rows.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kAmaxThreads)
column_amax_kernel(Dense x, unsigned int* amax) {
  constexpr int P = kVec ? 16 / static_cast<int>(sizeof(T)) : 1;
  constexpr int kWarps = kAmaxThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * 32 + lane) * P;
  unsigned int best[P] = {};
  if (c + P <= x.cols) {
#pragma unroll 8
    for (int64_t r = static_cast<int64_t>(blockIdx.y) * kWarps + warp; r < x.rows; r += static_cast<int64_t>(gridDim.y) * kWarps) {
      const Pack<T, P> v = load_pack<T, P>(static_cast<const T*>(x.data) + r * x.stride + c);
#pragma unroll
      for (int k = 0; k < P; ++k) best[k] = max(best[k], amax_bits(Values<T>::up(v.v[k])));
    }
  } else {
    for (int64_t r = static_cast<int64_t>(blockIdx.y) * kWarps + warp; r < x.rows; r += static_cast<int64_t>(gridDim.y) * kWarps)
      for (int k = 0; k < P; ++k)
        if (c + k < x.cols) best[k] = max(best[k], amax_bits(Values<T>::up(static_cast<const T*>(x.data)[r * x.stride + c + k])));
  }
  __shared__ unsigned int all[kWarps][32 * P];
#pragma unroll
  for (int k = 0; k < P; ++k) all[warp][lane * P + k] = best[k];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * P; i += kAmaxThreads) {
    unsigned int most = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) most = max(most, all[w][i]);
    const int64_t to = static_cast<int64_t>(blockIdx.x) * 32 * P + i;
    if (to < x.cols && most) atomicMax(amax + to, most);
  }
}

// A thread decodes half a block.  kVec: it writes its 8 values; else the rows do not start on 16 bytes,
// and the warp's lanes, which hold 256 values of one row, pass codes and scales around so that they write
// P neighbouring values each, 32 * P together (4,104 x 8,190 bf16: 30 us, 82 % of the issue slots).  On 16 bytes
// bound by its writes: 8,192 x 4,096 bf16 20 us, 4.3 TB/s.  blockDim = (half blocks of a row, rows).
template <typename O, bool kVec, int P>
__global__ void __launch_bounds__(kRowThreads)
dequantize_kernel(Nvfp4 in, Dense out, unsigned chunks) {
  const unsigned group = blockIdx.x / chunks;
  const int64_t r = static_cast<int64_t>(group) * blockDim.y + threadIdx.y;
  const unsigned i = (blockIdx.x - group * chunks) * blockDim.x + threadIdx.x;  // columns are below 2^31
  const int64_t c = static_cast<int64_t>(i) * 8;
  const bool valid = r < in.rows && c < in.cols;
  uint32_t codes = 0;
  float step = 0.0f;
  if (valid) {
    codes = __ldg(reinterpret_cast<const uint32_t*>(in.codes + r * in.pitch) + i);
    step = __fmul_rn(e4m3_exact(__ldg(in.block_scales + block_scale_at(r, i >> 1, block_scale_tiles(in.cols)))),
                     __ldg(in.scale + (in.per_row ? r : 0)));
  }
  if constexpr (kVec) {
    if (!valid) return;
    float level[8];
    e2m1_levels8(codes, level);
#pragma unroll
    for (int k = 0; k < 8; ++k) level[k] = __fmul_rn(level[k], step);
    const Pack<O, 8> v = round_pack<O, 8>(level);
    O* to = static_cast<O*>(out.data) + r * out.stride + c;
    if (c + 8 <= in.cols) {
#pragma unroll
      for (int q = 0; q < 8 / P; ++q) {
        Pack<O, P> x;
#pragma unroll
        for (int k = 0; k < P; ++k) x.v[k] = v.v[q * P + k];
        store_pack<O, P>(to + q * P, x);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c + k < in.cols) to[k] = v.v[k];
    }
  } else {  // blockDim.x is a multiple of 32: a warp holds one row
    if (r >= in.rows) return;
    const int lane = threadIdx.x & 31;
    const int64_t c0 = c - 8 * lane;
    O* to = static_cast<O*>(out.data) + r * out.stride;
#pragma unroll
    for (int j = 0; j < 8 / P; ++j) {
      const int e = (j * 32 + lane) * P;  // of the warp's 256
      const uint32_t word = __shfl_sync(0xffffffffu, codes, e / 8);
      const float s = __shfl_sync(0xffffffffu, step, e / 8);
      Pack<O, P> x;
      float level[8];
      e2m1_levels8(word >> (4 * (e % 8)), level);
#pragma unroll
      for (int k = 0; k < P; ++k) x.v[k] = Values<O>::down(__fmul_rn(level[k], s));
      if (c0 + e + P <= in.cols) {
        store_pack<O, P>(to + c0 + e, x);
      } else {
#pragma unroll
        for (int k = 0; k < P; ++k)
          if (c0 + e + k < in.cols) to[c0 + e + k] = x.v[k];
      }
    }
  }
}

// Sums of the columns over rows [blockIdx.y * span, + span) to row blockIdx.y of `sums`.  A CTA takes 32 * P
// columns; its 8 warps take every 8th row, and are added in order.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kAmaxThreads)
column_sums_kernel(Dense x, int64_t span, float* sums) {
  constexpr int P = kVec ? 16 / static_cast<int>(sizeof(T)) : 1;
  constexpr int kWarps = kAmaxThreads / 32;
  __shared__ float all[kWarps][32 * P];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * 32 + lane) * P;
  const int64_t last = min(x.rows, (blockIdx.y + 1) * span);
  const T* data = static_cast<const T*>(x.data);
  float sum[P] = {};
  if (c + P <= x.cols) {
#pragma unroll 8
    for (int64_t r = blockIdx.y * span + warp; r < last; r += kWarps) {
      const Pack<T, P> v = load_pack<T, P>(data + r * x.stride + c);
#pragma unroll
      for (int k = 0; k < P; ++k) sum[k] += Values<T>::up(v.v[k]);
    }
  } else {
    for (int64_t r = blockIdx.y * span + warp; r < last; r += kWarps)
      for (int k = 0; k < P; ++k)
        if (c + k < x.cols) sum[k] += Values<T>::up(data[r * x.stride + c + k]);
  }
#pragma unroll
  for (int k = 0; k < P; ++k) all[warp][lane * P + k] = sum[k];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * P; i += kAmaxThreads) {
    const int64_t to = static_cast<int64_t>(blockIdx.x) * 32 * P + i;
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) total += all[w][i];
    if (to < x.cols) sums[blockIdx.y * x.cols + to] = total;
  }
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

// Rows per partial sum: short enough to fill the GPU, and at most 64 parts, which one thread a column adds up.  At least
// 64 rows: 256 x 50,000 f32 12.4 us, with 16 18.6, with 256 12.5 (488 x 25 f32: 3.5, 5.7 and 4.5).  64 parts:
// 65,536 x 64 f32 14 us, 16 parts 39; 8,192 x 8,192 bf16 28 us, 16 parts 25, 256 parts 34.
int64_t sum_span(int64_t rows) { return std::max<int64_t>(64, (rows + 63) / 64); }

unsigned ceil_div(int64_t a, int64_t b) { return static_cast<unsigned>((a + b - 1) / b); }

}  // namespace

namespace {

template <typename T, bool kVec>
cudaError_t amax_pass(Dense x, bool columns, unsigned int* amax, cudaStream_t stream) {
  constexpr int P = kVec ? 16 / static_cast<int>(sizeof(T)) : 1;
  cudaError_t err = cudaMemsetAsync(amax, 0, columns ? static_cast<size_t>(x.cols) * 4 : 4, stream);
  if (err != cudaSuccess) return err;
  DeviceInfo info;
  if ((err = device_info(&info)) != cudaSuccess) return err;
  if (columns) {
    const unsigned across = ceil_div(x.cols, 32 * P);
    // Eight CTAs an SM, each with 64 rows at least.  8,190 x 4,104 bf16, codes included: 57 us, with four 56.5, sixteen
    // 54; 32,768 x 256 f32 22.8, rows of 16 24.6; 100 x 50,000 bf16 19.3, rows of 256 20.3.
    const int64_t down = std::max<int64_t>(1, std::min<int64_t>((x.rows + 63) / 64, info.sm_count * 8 / across));
    column_amax_kernel<T, kVec><<<dim3(across, static_cast<unsigned>(down)), kAmaxThreads, 0, stream>>>(x, amax);
    return cudaGetLastError();
  }
  if (x.stride == x.cols) x = {x.data, 1, x.rows * x.cols, x.rows * x.cols, x.type};
  // Four vectors a thread, 32 CTAs an SM at most.  8,192 x 8,192 f32 in strided rows, codes included: 102 us, with one
  // vector 121, eight CTAs 107; 8,190 x 4,104 bf16 45.5 us, 16 vectors 47.9, eight CTAs 47.3.
  const unsigned across = ceil_div(std::max<int64_t>(x.cols / P, 1), kAmaxThreads * 4);
  const unsigned most = static_cast<unsigned>(info.sm_count) * 32;
  const dim3 grid(std::min(across, most), static_cast<unsigned>(std::min<int64_t>(x.rows, std::max(1u, most / across))));
  amax_kernel<T, kVec><<<grid, kAmaxThreads, 0, stream>>>(x, amax);
  return cudaGetLastError();
}

template <typename T, int kVec>
cudaError_t quantize_rows(const Dense& x, const Nvfp4& out, const unsigned int* given, unsigned int* most, cudaStream_t stream) {
  DeviceInfo info;
  cudaError_t err = device_info(&info);
  if (err != cudaSuccess) return err;
  const int64_t blocks = block_scale_tiles(x.cols) * 4;
  // Two blocks to a thread, and up to a quarter more read twice (four in registers leave half the warps;
  // off the boundaries, where each takes more registers yet, two: 1,453 x 46,171 float16 101 us against 127;
  // 8,192 x 4,104 f32 43 us, four in registers 56; 1 x 166,000 f32 7.2, two 8.1; 1,000 x 60,000 bf16 62, two 66);
  // a long row is shared by a cluster while there are SMs for it (8 x 50,000 f32: 4.4 us, without 5.3), then by up
  // to eight CTAs where four blocks do not hold it (1 x 166,000 f32: one CTA 40), then read twice.  Up to three
  // blocks to a thread before a row gets more threads: 8,192 x 4,104 f32 with two 55, with five 101 (300 rows: 5.1,
  // 4.3 and 6.5).
  int per_row = 4, cluster = 0;
  while (1 << per_row < kRowThreads && blocks > int64_t{3} << per_row) ++per_row;
  while (cluster < 3 && blocks > int64_t{2} << (per_row + cluster) && x.rows << (cluster + 1) <= info.sm_count) ++cluster;
  while (cluster < 3 && blocks > int64_t{4} << (per_row + cluster)) ++cluster;
  if (cluster > 0) per_row = 8;  // a cluster's CTAs are whole
  const int held = blocks <= int64_t{1} << (per_row + cluster) ? 1 : blocks * 2 <= int64_t{5} << (per_row + cluster) || !kVec ? 2 : 4;
  const int64_t grid = cluster > 0 ? x.rows << cluster : ((x.rows << per_row) + kRowThreads - 1) / kRowThreads;
  const int64_t fill = x.rows % 128 ? ((blocks + 63) / 64 + (1 << cluster) - 1) >> cluster << cluster : 0;
  if (grid + fill > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(grid + fill));
  config.blockDim = dim3(kRowThreads);
  config.stream = stream;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim = {1u << cluster, 1, 1};
  config.attrs = &attribute;
  config.numAttrs = 1;
  auto* kernel = held == 1 ? quantize_rows_kernel<T, kVec, 1> : held == 2 ? quantize_rows_kernel<T, kVec, 2> : quantize_rows_kernel<T, kVec, 4>;
  return cudaLaunchKernelEx(&config, kernel, x, out, given, most, per_row, cluster, static_cast<unsigned>(grid));
}

}  // namespace

size_t nvfp4_quantize_workspace_bytes(const Nvfp4& out, bool transpose) {
  if (out.per_row) return transpose ? static_cast<size_t>(out.rows) * 4 : 0;
  return 4;
}

cudaError_t launch_nvfp4_quantize(const Dense& value, bool transpose, const Nvfp4& out, unsigned int* amax,
                                  bool amax_given, void* workspace, cudaStream_t stream) {
  return with_type(value.type, [&](auto zero) {
    using T = decltype(zero);
    auto call = [&](auto flag) {
      constexpr bool kVec = decltype(flag)::value;
      cudaError_t err = cudaSuccess;
      const bool by_row = out.per_row && !transpose;
      // The words that the scales come from: one per column of a transpose, or the matrix's.
      unsigned int* words = out.per_row && transpose ? static_cast<unsigned int*>(workspace) : amax ? amax : static_cast<unsigned int*>(workspace);
      // Rows on 32 bytes, on 16 or off them: 8,192 x 4,104 f32 42.7, 46.1 and 69.1 us, 8,192 x 4,096 bf16 25.7, 25.8 and 35.3.
      const bool wide = rows_aligned(value, sizeof(T), 32);
      auto* rows = !kVec ? quantize_rows<T, 0> : wide ? quantize_rows<T, 32> : quantize_rows<T, 16>;
      if (by_row) {
        if (amax && (err = cudaMemsetAsync(amax, 0, 4, stream)) != cudaSuccess) return err;
        return rows(value, out, nullptr, amax, stream);
      }
      if (out.per_row || !amax_given)
        if ((err = amax_pass<T, kVec>(value, out.per_row, words, stream)) != cudaSuccess) return err;
      if (!transpose) return rows(value, out, words, nullptr, stream);
      const int64_t grid = (value.cols + 127) / 128 * 2 * (block_scale_tiles(value.rows) / 2);
      if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
      quantize_columns_kernel<T, kVec><<<static_cast<unsigned>(grid), kTileThreads, 0, stream>>>(value, out, words);
      return cudaGetLastError();
    };
    // Vectors where rows start on 16 bytes: 8,190 x 4,104 bf16 transposed, a scale per row 57 us, value by value 116.
    return rows_aligned(value, sizeof(T), 16) ? call(std::true_type{}) : call(std::false_type{});
  });
}

cudaError_t launch_nvfp4_dequantize(const Nvfp4& in, const Dense& out, cudaStream_t stream) {
  return with_type(out.type, [&](auto zero) {
    using T = decltype(zero);
    const int64_t halves = (in.cols + 7) / 8;
    int x = 32;
    while (x < kRowThreads && x < halves) x *= 2;
    const dim3 block(x, kRowThreads / x);
    const int64_t chunks = (halves + x - 1) / x, groups = (in.rows + block.y - 1) / block.y;
    if (chunks * groups > 0x7fffffff) return cudaErrorInvalidConfiguration;
    // 8,192 x 4,096 on 16 bytes, and the lanes' exchange for the same: bf16 20.5 and 28.2 us, f32 35.5 and 32.1.
    constexpr int kWide = 16 / static_cast<int>(sizeof(T)), kWord = 4 / static_cast<int>(sizeof(T));
    auto* kernel = rows_aligned(out, sizeof(T), 16) ? dequantize_kernel<T, true, kWide>
                   : rows_aligned(out, sizeof(T), 4) ? dequantize_kernel<T, false, kWord>
                                                     : dequantize_kernel<T, false, 1>;
    kernel<<<static_cast<unsigned>(chunks * groups), block, 0, stream>>>(in, out, static_cast<unsigned>(chunks));
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
    if (parts > 0) {  // no rows: the sums are zero
      const bool vec = rows_aligned(value, sizeof(T), 16);  // (8,192 x 8,192 bf16: 28 us, value by value 48)
      const dim3 grid(ceil_div(value.cols, vec ? 512 / sizeof(T) : 32), static_cast<unsigned>(parts));
      auto* kernel = vec ? column_sums_kernel<T, true> : column_sums_kernel<T, false>;
      kernel<<<grid, kAmaxThreads, 0, stream>>>(value, span, sums);
      const cudaError_t err = cudaGetLastError();
      if (err != cudaSuccess) return err;
    }
    join_sums_kernel<<<ceil_div(value.cols, kAmaxThreads), kAmaxThreads, 0, stream>>>(sums, parts, value.cols, out);
    return cudaGetLastError();
  });
}

}  // namespace nsb
