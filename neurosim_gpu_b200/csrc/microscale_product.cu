// microscale_product.cu -- the product of two dense NVFP4 matrices (the format: nsb_nvfp4.cuh):
//
//   out[m, n] = round( (sum_k level_a sa level_b sb) * ga[m] * gb[n] + bias[n] )
//
// on the fifth-generation tensor cores (tcgen05.mma, kind mxf4nvf4): the levels and the E4M3 block
// scales go in as stored, the sums are float32 in tensor memory, and the two float32 scales and the
// bias are applied on the way out.
//
// One operand lies along the 128 lanes of tensor memory, the other along its columns.  The columns
// take the operand with fewer rows (the states of a few networks, say), so that the larger one,
// usually the weights, is read once and fills the lanes.
//
// A CTA has six warps: one thread loads K tiles of 256 (128 bytes of codes per row by TMA, the block
// scales by bulk copies) into a ring of stages; one thread copies a stage's scales to tensor memory
// and issues its four products of K = 64; four warps read the finished tile (each its own 32 lanes)
// and write it.  The scales of a stage have tensor memory of their own, reused only after the stage's
// products are complete.  Where two accumulators fit, the next tile starts while one is written.
//
// Where there are too few tiles for the GPU, a cluster of 2, 4 or 8 CTAs shares a tile along K: each
// leaves its float32 partial sums in its shared memory, and each adds a part of the columns of all
// of them in rank order (deterministic) over distributed shared memory.
#include <cuda.h>

#include <algorithm>

#include "nsb_nvfp4.cuh"
#include "nsb_tcgen05.cuh"
#include "nsb_tokens.h"

namespace nsb {
namespace {

constexpr int kThreads = 192;
constexpr int kLanes = 128;
constexpr int kTileBytes = 128;    // of codes: 256 columns of the operands
constexpr int kScaleBytes = 2048;  // block scales of 128 rows and 256 columns
constexpr int kTmemColumns = 512;
constexpr int kMostStages = 8;
constexpr int kMostShared = 232448;   // dynamic shared memory of a CTA
constexpr int kLeastShared = 120000;  // more than half an SM's: one CTA per SM, so tensor memory is free
constexpr int kHeader = 4096;         // barriers, column scales; the stages follow, 1,024-byte aligned

// The operand along the lanes (`rows` of it) and the one along the columns.
struct Side {
  const uint8_t* block_scales;
  const float* scale;
  const float* bias;  // along this side, or null
  int64_t stride;     // of the output
  int32_t rows;
  bool per_row;
};

struct ProductArgs {
  Side lane, column;
  void* out;
  int64_t scale_tiles;  // 512-byte tiles per 128 rows
  int32_t k_tiles;
  int32_t column_tile;  // 16 ... 256; box rows of the column operand
  int32_t stages, accumulators, split;
  int32_t lane_tiles, column_tiles;
  int* status;
};

struct Header {
  uint64_t full[kMostStages], empty[kMostStages];
  uint64_t sum_full[2], sum_empty[2], drained;
  uint32_t tmem;
  int aborted;
  float scale[2][256], bias[256];  // of the tile's columns
};
static_assert(sizeof(Header) <= kHeader, "header");

__device__ int g_product_status;  // where no status word is given

__device__ __forceinline__ void give_up(const ProductArgs& a, volatile int* aborted, int code) {
  *aborted = 1;
  atomicExch(a.status ? a.status : &g_product_status, code);
}

// Lane tiles in groups of 8 that walk all column tiles: the tiles in flight share both operands in L2.
__device__ __forceinline__ void place(const ProductArgs& a, int tile, int* lane_tile, int* column_tile) {
  const int group = tile / (8 * a.column_tiles), first = 8 * group;
  const int tall = min(8, a.lane_tiles - first), at = tile - first * a.column_tiles;
  *lane_tile = first + at % tall;
  *column_tile = at / tall;
}

template <typename O>
__device__ __forceinline__ void put(const ProductArgs& a, int64_t lane, int64_t column, float sum, float lane_scale,
                                    float column_scale, float bias) {
  const float y = __fadd_rn(__fmul_rn(__fmul_rn(sum, lane_scale), column_scale), bias);
  static_cast<O*>(a.out)[lane * a.lane.stride + column * a.column.stride] = Values<O>::down(y);
}

template <typename O>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap lane_map, const __grid_constant__ CUtensorMap column_map,
               const __grid_constant__ ProductArgs a) {
  extern __shared__ __align__(1024) uint8_t shared[];
  Header& h = *reinterpret_cast<Header*>(shared);
  uint8_t* stages = shared + kHeader;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* aborted = &h.aborted;
  const int column_blocks = (a.column_tile + 127) / 128;
  const int lane_bytes = kLanes * kTileBytes, column_bytes = a.column_tile * kTileBytes;
  const int stage_bytes = lane_bytes + column_bytes + kScaleBytes * (1 + column_blocks);
  const int slot_columns = 16 * (1 + column_blocks);  // tensor memory of a stage's scales
  int rank = 0;
  if (a.split > 1) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int tiles = a.lane_tiles * a.column_tiles;
  const int first = blockIdx.x / a.split, step = gridDim.x / a.split;
  const int k0 = static_cast<int>(static_cast<int64_t>(a.k_tiles) * rank / a.split);
  const int k1 = static_cast<int>(static_cast<int64_t>(a.k_tiles) * (rank + 1) / a.split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      barrier_init(&h.full[s], 1);
      barrier_init(&h.empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      barrier_init(&h.sum_full[s], 1);
      barrier_init(&h.sum_empty[s], 4);
    }
    barrier_init(&h.drained, 1);
    h.aborted = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&h.tmem, kTmemColumns);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = h.tmem;
  const uint32_t slots = tmem + a.accumulators * a.column_tile;

  if (threadIdx.x == 0) {  // loads
    int n = 0;
    bool ok = true;
    for (int tile = first; ok && tile < tiles; tile += step) {
      int lt, ct;
      place(a, tile, &lt, &ct);
      for (int k = k0; k < k1; ++k, ++n) {
        const int s = n % a.stages;
        if (n >= a.stages && !barrier_wait(&h.empty[s], (n / a.stages - 1) & 1, aborted)) {
          give_up(a, aborted, 1);
          ok = false;
          break;
        }
        uint8_t* to = stages + s * stage_bytes;
        barrier_arrive_expect(&h.full[s], stage_bytes);
        load_box(to, &lane_map, k * kTileBytes, lt * kLanes, &h.full[s]);
        load_box(to + lane_bytes, &column_map, k * kTileBytes, ct * a.column_tile, &h.full[s]);
        to += lane_bytes + column_bytes;
        load_bytes(to, a.lane.block_scales + (lt * a.scale_tiles + k * 4) * 512, kScaleBytes, &h.full[s]);
        for (int c = 0; c < column_blocks; ++c) {
          // A tile that ends before its second block of 128 rows loads the first one again.
          const int64_t block = static_cast<int64_t>(ct) * column_blocks + c;
          const int64_t in = block * 128 < a.column.rows ? block : 0;
          load_bytes(to + kScaleBytes * (1 + c), a.column.block_scales + (in * a.scale_tiles + k * 4) * 512, kScaleBytes,
                     &h.full[s]);
        }
      }
    }
    if (*aborted)  // nothing may land in shared memory after the CTA has gone
      for (int u = max(0, n - a.stages); u < n; ++u)
        for (int i = 0; i < kBarrierPolls && !barrier_try(&h.full[u % a.stages], (u / a.stages) & 1); ++i) {
        }
  } else if (threadIdx.x == 32) {  // products
    int n = 0, t = 0;
    bool ok = true;
    for (int tile = first; ok && tile < tiles; tile += step, ++t) {
      int lt, ct;
      place(a, tile, &lt, &ct);
      const int b = t % a.accumulators, use = t / a.accumulators;
      if (use > 0 && !barrier_wait(&h.sum_empty[b], (use - 1) & 1, aborted)) {
        give_up(a, aborted, 2);
        break;
      }
      tcgen05_fence_after();
      const int columns = min(a.column_tile, (a.column.rows - ct * a.column_tile + 15) / 16 * 16);
      const uint32_t instruction = nvfp4_instruction(columns);
      const uint32_t sum = tmem + b * a.column_tile;
      for (int k = k0; k < k1; ++k, ++n) {
        const int s = n % a.stages;
        if (!barrier_wait(&h.full[s], (n / a.stages) & 1, aborted)) {
          give_up(a, aborted, 3);
          ok = false;
          break;
        }
        tcgen05_fence_after();
        const uint32_t at = shared_addr(stages + s * stage_bytes);
        const uint32_t scales = at + lane_bytes + column_bytes;
        const uint32_t lane_scales = slots + s * slot_columns, column_scales = lane_scales + 16;
        // Tensor memory: four columns per product for the lanes, four per product and 128 columns.
        for (int q = 0; q < 4; ++q) copy_scales(lane_scales + 4 * q, plain_descriptor(scales + 512 * q));
        for (int q = 0; q < 4; ++q)
          for (int c = 0; c < column_blocks; ++c)
            copy_scales(column_scales + 4 * (q * column_blocks + c), plain_descriptor(scales + kScaleBytes * (1 + c) + 512 * q));
        const uint64_t x = swizzled_descriptor(at), y = swizzled_descriptor(at + lane_bytes);
        for (int q = 0; q < 4; ++q)  // 64 elements are 32 bytes: 2 units of 16
          nvfp4_mma(sum, x + 2 * q, y + 2 * q, instruction, lane_scales + 4 * q, column_scales + 4 * q * column_blocks,
                    k > k0 || q > 0);
        mma_commit(&h.empty[s]);
      }
      if (ok) mma_commit(&h.sum_full[b]);
    }
    if (*aborted) {
      mma_commit(&h.drained);
      for (int i = 0; i < kBarrierPolls && !barrier_try(&h.drained, 0); ++i) {
      }
    }
  } else if (warp >= 2) {  // results: warp w reads lanes 32 (w % 4) ...
    const int quarter = warp & 3, slot = threadIdx.x - 64;
    int t = 0;
    bool ok = true;  // once a wait has given up, the tiles are walked for their barriers alone
    for (int tile = first; tile < tiles; tile += step, ++t) {
      int lt, ct;
      place(a, tile, &lt, &ct);
      const int b = t % a.accumulators, use = t / a.accumulators;
      const int64_t column0 = static_cast<int64_t>(ct) * a.column_tile;
      const int columns = static_cast<int>(min(static_cast<int64_t>(a.column_tile), a.column.rows - column0));
      if (a.split == 1) {
        asm volatile("bar.sync 1, 128;" ::: "memory");  // the last tile's scales are no longer read
        for (int c = slot; c < columns; c += 128) {
          h.scale[0][c] = __ldg(a.column.scale + (a.column.per_row ? column0 + c : 0));
          h.bias[c] = a.column.bias ? __ldg(a.column.bias + column0 + c) : 0.0f;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
      const int64_t row = static_cast<int64_t>(lt) * kLanes + quarter * 32 + lane;
      const bool in = row < a.lane.rows;
      const float row_scale = in ? __ldg(a.lane.scale + (a.lane.per_row ? row : 0)) : 0.0f;
      const float row_bias = in && a.lane.bias ? __ldg(a.lane.bias + row) : 0.0f;
      if (ok && lane == 0 && !barrier_wait(&h.sum_full[b], use & 1, aborted)) {
        give_up(a, aborted, 4);
        ok = false;
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) continue;
      tcgen05_fence_after();
      const uint32_t from = tmem + b * a.column_tile + (static_cast<uint32_t>(quarter * 32) << 16);
      float* partial = reinterpret_cast<float*>(stages) + quarter * 32 + lane;  // [column][lane], split only
      for (int c = 0; c < columns; c += 16) {
        uint32_t v[16];
        tmem_load16(from + c, v);
        tmem_wait(v);
        if (a.split > 1) {
#pragma unroll
          for (int i = 0; i < 16; ++i) partial[(c + i) * kLanes] = __uint_as_float(v[i]);
        } else if (in) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (c + i < columns)
              put<O>(a, row, column0 + c + i, __uint_as_float(v[i]), row_scale, h.scale[0][c + i],
                     a.column.bias ? h.bias[c + i] : row_bias);
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) barrier_arrive(&h.sum_empty[b]);
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (a.split > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    int lt, ct;
    place(a, first, &lt, &ct);
    const int64_t column0 = static_cast<int64_t>(ct) * a.column_tile;
    const int columns = static_cast<int>(min(static_cast<int64_t>(a.column_tile), a.column.rows - column0));
    const int64_t row = static_cast<int64_t>(lt) * kLanes + threadIdx.x;
    if (threadIdx.x < kLanes && row < a.lane.rows && !*aborted) {
      const float row_scale = __ldg(a.lane.scale + (a.lane.per_row ? row : 0));
      const float row_bias = a.lane.bias ? __ldg(a.lane.bias + row) : 0.0f;
      for (int c = rank; c < columns; c += a.split) {
        float sum = 0.0f;
        for (int r = 0; r < a.split; ++r) {
          uint32_t remote;
          float x;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                       : "=r"(remote)
                       : "r"(shared_addr(stages) + (c * kLanes + threadIdx.x) * 4), "r"(r));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(remote) : "memory");
          sum += x;
        }
        put<O>(a, row, column0 + c, sum, row_scale, __ldg(a.column.scale + (a.column.per_row ? column0 + c : 0)),
               a.column.bias ? __ldg(a.column.bias + column0 + c) : row_bias);
      }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  if (warp == 1) tmem_free(tmem, kTmemColumns);
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's tensor-map encoder (host code only; the library does not link the driver).
EncodeTiled encoder() {
  static EncodeTiled function = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return function;
}

// Boxes of 128 bytes x `rows` of a matrix's codes, in the 128-byte swizzle; zeros beyond it.
bool map_codes(const Nvfp4& m, int rows, CUtensorMap* map) {
  const cuuint64_t size[2] = {static_cast<cuuint64_t>(m.pitch), static_cast<cuuint64_t>(m.rows)};
  const cuuint64_t stride[1] = {static_cast<cuuint64_t>(m.pitch)};
  const cuuint32_t box[2] = {kTileBytes, static_cast<cuuint32_t>(rows)}, one[2] = {1, 1};
  return encoder() && encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, m.codes, size, stride, box, one,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename O>
cudaError_t launch(const Nvfp4& lane, const Nvfp4& column, ProductArgs a, cudaStream_t stream) {
  DeviceInfo info;
  cudaError_t err = device_info(&info);
  if (err != cudaSuccess) return err;
  a.lane_tiles = (a.lane.rows + kLanes - 1) / kLanes;
  a.column_tile = std::min(256, (a.column.rows + 15) / 16 * 16);
  if (a.column_tile > 128) a.column_tile = 256;  // tiles start on the block scales' 128-row tiles
  a.column_tiles = (a.column.rows + a.column_tile - 1) / a.column_tile;
  const int64_t tiles = static_cast<int64_t>(a.lane_tiles) * a.column_tiles;
  if (tiles > 0x3fffffff) return cudaErrorInvalidConfiguration;
  const int blocks = (a.column_tile + 127) / 128, slot = 16 * (1 + blocks);
  const int stage = kTileBytes * (kLanes + a.column_tile) + kScaleBytes * (1 + blocks);
  a.accumulators = a.column_tile <= 128 ? 2 : 1;
  a.stages = std::min({kMostStages, (kMostShared - kHeader) / stage, (kTmemColumns - a.accumulators * a.column_tile) / slot});
  a.split = 1;
  while (a.split < 8 && tiles * a.split * 2 <= info.sm_count && a.k_tiles >= a.split * 2) a.split *= 2;
  if (a.split > 1) a.accumulators = 1;
  const int shared = std::max({kLeastShared, kHeader + a.stages * stage, a.split > 1 ? kHeader + a.column_tile * kLanes * 4 : 0});
  CUtensorMap lane_map, column_map;
  if (!map_codes(lane, kLanes, &lane_map) || !map_codes(column, a.column_tile, &column_map)) return cudaErrorInvalidValue;
  err = cudaFuncSetAttribute(product_kernel<O>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(a.split > 1 ? tiles * a.split : std::min<int64_t>(tiles, info.sm_count)));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim = {static_cast<unsigned>(a.split), 1, 1};
  config.attrs = &cluster;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, product_kernel<O>, lane_map, column_map, a);
}

}  // namespace

cudaError_t launch_nvfp4_product(const Nvfp4& a, const Nvfp4& b, const float* bias, const Dense& out,
                                 int* status, cudaStream_t stream) {
  return with_type(out.type, [&](auto zero) {
    using O = decltype(zero);
    const Side rows{a.block_scales, a.scale, nullptr, out.stride, static_cast<int32_t>(a.rows), a.per_row};
    const Side cols{b.block_scales, b.scale, bias, 1, static_cast<int32_t>(b.rows), b.per_row};
    ProductArgs args{};
    args.out = out.data;
    args.scale_tiles = block_scale_tiles(a.cols);
    args.k_tiles = static_cast<int32_t>((a.cols + 255) / 256);
    args.status = status;
    // Few rows of b (a narrow readout of many states) go along the columns; else b along the lanes,
    // where neighbouring lanes write neighbouring outputs.
    const bool narrow = b.rows <= 128 && b.rows < a.rows;
    args.lane = narrow ? rows : cols;
    args.column = narrow ? cols : rows;
    return narrow ? launch<O>(a, b, args, stream) : launch<O>(b, a, args, stream);
  });
}

}  // namespace nsb
