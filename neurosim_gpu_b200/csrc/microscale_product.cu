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
// Warp 0 loads K tiles of 256 (128 bytes of codes per row by TMA, the block scales by bulk copies)
// into a ring of stages; warp 1 copies a stage's scales to tensor memory and issues its four products
// of K = 64; four or eight warps take the finished tile to registers, which frees its tensor memory
// for the next tile, and write it.  The scales of a stage have tensor memory of their own, reused
// only after the stage's products are complete.
//
// Large products run on pairs of CTAs (tcgen05 cta_group::2): a tile of 256 lanes x 256 columns, of which
// each CTA holds 128 lanes' sums and loads its 128 lanes' codes and half of the columns'.  A CTA of its
// own takes 54 KB from L2 per K tile, at 64 bytes a cycle longer than its products do (860 cycles against
// 512 of the tensor core); one of a pair takes 38 KB.  The first CTA issues for both: the loads of both,
// which are tensor copies throughout, complete on its barriers.
//
// Few rows are bound by reading the weights: 1 x 32,000 x 4,096 15.3 us, 4.8 TB/s.  Many are bound by the tensor
// cores, 77 % of the time active: 8,192 x 8,192 x 4,096 104-107 us, 5.2 PFLOP/s; x 32,768 770 us, 5.7 PFLOP/s.
//
// Where there are too few tiles for the GPU, a cluster of 2, 4 or 8 CTAs shares a tile along K: each
// leaves its float32 partial sums in its shared memory, and each adds a part of the columns of all
// of them over distributed shared memory, every column in the same order.
#include <cuda.h>

#include <algorithm>
#include <atomic>

#include "nsb_nvfp4.cuh"
#include "nsb_tcgen05.cuh"
#include "nsb_tokens.h"

namespace nsb {
namespace {

constexpr int kLanes = 128;
constexpr int kTileBytes = 128;    // of codes: 256 columns of the operands
constexpr int kScaleBytes = 2048;  // block scales of 128 rows and 256 columns
constexpr int kLaneBytes = kLanes * kTileBytes;
constexpr int kTmemColumns = 512;
constexpr int kMostShared = 232448;   // dynamic shared memory of a CTA
constexpr int kLeastShared = 120000;  // more than half an SM's: one CTA per SM, so tensor memory is free
constexpr int kHeader = 4096;         // barriers, column scales; the stages follow, 1,024-byte aligned

// What a tile of 128 lanes (of a pair 2 x 128) x kColumns columns takes of a CTA.
template <int kColumns, bool kPair>
struct Shape {
  static constexpr int kBlocks = (kColumns + 127) / 128;  // of 128 rows of block scales
  static constexpr int kColumnRows = kPair ? kColumns / 2 : kColumns;  // of the column operand's codes
  static constexpr int kColumnBytes = kColumnRows * kTileBytes;
  static constexpr int kStageBytes = kLaneBytes + kColumnBytes + kScaleBytes * (1 + kBlocks);
  static constexpr int kSlot = 16 * (1 + kBlocks);        // tensor memory columns of a stage's scales
  static constexpr int kSums = kColumns <= 128 ? 2 : 1;   // accumulators
  static constexpr int kStages = std::min({8, (kMostShared - kHeader) / kStageBytes, (kTmemColumns - kSums * kColumns) / kSlot});
  static constexpr int kShared = std::max(kLeastShared, kHeader + kStages * kStageBytes);
  static constexpr int kOutWarps = kColumns >= 64 ? 8 : 4;  // each reads 32 lanes of a half, or all, of the columns
  static constexpr int kOutColumns = kColumns / (kOutWarps / 4);
  static constexpr int kThreads = 64 + 32 * kOutWarps;
  static_assert(kStages * kStageBytes >= kColumns * kLanes * 4, "the partial sums of a split tile lie in the stages");
};

// The operand along the lanes (`rows` of it) or the one along the columns.
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
  int32_t k_tiles, split;
  int32_t lane_tiles, column_tiles;  // lane tiles of 128, of pairs 256
  int polls;  // of a bounded wait; below kBarrierPolls no product is issued, and the waits for them run out
  bool lane_ready;  // the operand along the lanes was complete before the kernel ahead of this one started
  int* status;
};

struct Header {
  uint64_t full[8], empty[8];
  uint64_t sum_full[2], sum_empty[2], drained;
  uint32_t tmem;
  int aborted;
  int peer_aborted, peer_loads;  // of a pair: what the other CTA leaves as its roles end
  alignas(16) float scale[256];  // of the tile's columns
  alignas(16) float bias[256];
};
static_assert(sizeof(Header) <= kHeader, "header");

__device__ int g_product_status;  // where no status word is given
std::atomic<int> g_polls{kBarrierPolls};

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

__device__ __forceinline__ float scaled(float sum, float lane_scale, float column_scale, float bias) {
  return __fadd_rn(__fmul_rn(__fmul_rn(sum, lane_scale), column_scale), bias);
}

// Boxes of both operands' codes; of a pair also rows of 2,048 bytes of their block scales.
template <bool kPair>
struct Maps {
  CUtensorMap lane, column;
};
template <>
struct Maps<true> {
  CUtensorMap lane, column, lane_scales, column_scales;
};

// A position in the ring of stages and the parity of its round.
template <int kStages>
struct Ring {
  int stage = 0;
  uint32_t round = 0;
  __device__ __forceinline__ void next() {
    if (++stage == kStages) {
      stage = 0;
      ++round;
    }
  }
};

template <typename O, int kColumns, bool kPair>
__global__ void __launch_bounds__(Shape<kColumns, kPair>::kThreads, 1)
product_kernel(const __grid_constant__ Maps<kPair> maps, const __grid_constant__ ProductArgs a) {
  using S = Shape<kColumns, kPair>;
  extern __shared__ __align__(1024) uint8_t shared[];
  Header& h = *reinterpret_cast<Header*>(shared);
  uint8_t* stages = shared + kHeader;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int* aborted = &h.aborted;
  int rank = 0;
  if (kPair || a.split > 1) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int tiles = a.lane_tiles * a.column_tiles;
  const int group = kPair ? 2 : a.split;  // CTAs that share a tile: a pair its lanes, others its K tiles
  const int first = blockIdx.x / group, step = gridDim.x / group;
  const int k0 = kPair ? 0 : static_cast<int>(static_cast<int64_t>(a.k_tiles) * rank / group);
  const int k1 = kPair ? a.k_tiles : static_cast<int>(static_cast<int64_t>(a.k_tiles) * (rank + 1) / group);
  // A pair's second 128 lanes may lie beyond the operand: any scales do for them.
  auto lane_scale_block = [&](int lane_tile) -> int64_t {
    const int64_t block = kPair ? 2 * lane_tile + rank : lane_tile;
    return block * kLanes < a.lane.rows ? block : 0;
  };
  const bool issues = !kPair || rank == 0;
  auto lane_block = [&](int lane_tile) { return kPair ? 2 * lane_tile + rank : lane_tile; };  // of 128 lanes

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      barrier_init(&h.full[s], 1);
      barrier_init(&h.empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      barrier_init(&h.sum_full[s], 1);
      barrier_init(&h.sum_empty[s], S::kOutWarps * (kPair ? 2 : 1));
    }
    barrier_init(&h.drained, 1);
    h.aborted = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc<kPair>(&h.tmem, kTmemColumns);
  tcgen05_fence_before();
  __syncthreads();
  if (kPair) cluster_barrier();  // the other CTA's barriers are ready
  tcgen05_fence_after();
  const uint32_t tmem = h.tmem;

  int loads = 0;         // K tiles that warp 0 has asked for
  bool drained = false;  // warp 1 has waited for its products
  if (warp == 0) {  // loads
    Ring<S::kStages> ring;
    // One thread: the lanes' share of a stage, which its barrier then expects whole (a pair's both halves).
    auto load_lanes = [&](int stage, int lane_tile, int k) {
      uint8_t* to = stages + stage * S::kStageBytes;
      uint64_t* full = &h.full[stage];
      if (issues) barrier_arrive_expect(full, (kPair ? 2 : 1) * S::kStageBytes);
      if constexpr (kPair) {
        const uint32_t bar = remote_address(shared_addr(full), 0);
        load_box_pair(to, &maps.lane, k * kTileBytes, lane_block(lane_tile) * kLanes, bar);
        load_row_pair(to + kLaneBytes + S::kColumnBytes, &maps.lane_scales, k, static_cast<int>(lane_scale_block(lane_tile)), bar);
      } else {
        load_box(to, &maps.lane, k * kTileBytes, lane_block(lane_tile) * kLanes, full);
        load_bytes(to + kLaneBytes + S::kColumnBytes, a.lane.block_scales + (lane_scale_block(lane_tile) * a.scale_tiles + static_cast<int64_t>(k) * 4) * 512,
                   kScaleBytes, full);
      }
    };
    auto load_columns = [&](int stage, int column_tile, int k) {
      uint8_t* to = stages + stage * S::kStageBytes + kLaneBytes;
      uint64_t* full = &h.full[stage];
      const uint32_t bar = kPair ? remote_address(shared_addr(full), 0) : 0;
      if constexpr (kPair) load_box_pair(to, &maps.column, k * kTileBytes, column_tile * kColumns + rank * S::kColumnRows, bar);
      else load_box(to, &maps.column, k * kTileBytes, column_tile * kColumns, full);
      to += S::kColumnBytes;
#pragma unroll
      for (int c = 0; c < S::kBlocks; ++c) {
        // A tile that ends before its second block of 128 rows loads the first one again.
        const int64_t ahead_of = static_cast<int64_t>(column_tile) * S::kBlocks + c, block = ahead_of * 128 < a.column.rows ? ahead_of : 0;
        if constexpr (kPair) load_row_pair(to + kScaleBytes * (1 + c), &maps.column_scales, k, static_cast<int>(block), bar);
        else load_bytes(to + kScaleBytes * (1 + c), a.column.block_scales + (block * a.scale_tiles + static_cast<int64_t>(k) * 4) * 512, kScaleBytes, full);
      }
    };
    int ahead = 0;
    bool ok = true;
    if (a.lane_ready && first < tiles) {  // its first stages' share while the kernel ahead still runs
      int lt, ct;
      place(a, first, &lt, &ct);
      ahead = min(S::kStages, k1 - k0);
      if (elect_one())
        for (int s = 0; s < ahead; ++s) load_lanes(s, lt, k0 + s);
      __syncwarp();
    }
    grid_wait();
    for (int tile = first; ok && tile < tiles; tile += step) {
      int lt, ct;
      place(a, tile, &lt, &ct);
      for (int k = k0; k < k1; ++k, ++loads, ring.next()) {
        if (ring.round > 0 && !barrier_wait(&h.empty[ring.stage], (ring.round - 1) & 1, aborted, a.polls)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          if (loads >= ahead) load_lanes(ring.stage, lt, k);
          load_columns(ring.stage, ct, k);
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) give_up(a, aborted, 1);
  } else if (warp == 1 && issues) {  // products
    Ring<S::kStages> ring;
    int t = 0;
    bool ok = a.polls == kBarrierPolls;
    const uint64_t lane_codes = swizzled_descriptor(shared_addr(stages));
    const uint64_t column_codes = swizzled_descriptor(shared_addr(stages + kLaneBytes));
    const uint64_t scales = plain_descriptor(shared_addr(stages + kLaneBytes + S::kColumnBytes));
    for (int tile = first; ok && tile < tiles; tile += step, ++t) {
      int lt, ct;
      place(a, tile, &lt, &ct);
      const int b = t % S::kSums, use = t / S::kSums;
      if (use > 0 && !barrier_wait(&h.sum_empty[b], (use - 1) & 1, aborted, a.polls)) {
        if (lane == 0) give_up(a, aborted, 2);
        break;
      }
      tcgen05_fence_after();
      // A pair's halves of B are always whole.
      const uint32_t instruction = nvfp4_instruction(kPair ? 2 * kLanes : kLanes, kPair ? kColumns : min(kColumns, (a.column.rows - ct * kColumns + 15) / 16 * 16));
      const uint32_t sum = tmem + b * kColumns;
      for (int k = k0; k < k1; ++k, ring.next()) {
        if (!barrier_wait(&h.full[ring.stage], ring.round & 1, aborted, a.polls)) {
          if (lane == 0) give_up(a, aborted, 3);
          ok = false;
          break;
        }
        tcgen05_fence_after();
        if (elect_one()) {
          const uint64_t offset = ring.stage * (S::kStageBytes >> 4);
          const uint32_t lane_scales = tmem + S::kSums * kColumns + ring.stage * S::kSlot, column_scales = lane_scales + 16;
          // In tensor memory four columns per product for the lanes, then four per product and 128 columns.
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            copy_scales<kPair>(lane_scales + 4 * q, scales + offset + 32 * q);
#pragma unroll
            for (int c = 0; c < S::kBlocks; ++c)
              copy_scales<kPair>(column_scales + 4 * (q * S::kBlocks + c), scales + offset + (kScaleBytes >> 4) * (1 + c) + 32 * q);
          }
#pragma unroll
          for (int q = 0; q < 4; ++q)  // 64 elements are 32 bytes: 2 units of 16
            nvfp4_mma<kPair>(sum, lane_codes + offset + 2 * q, column_codes + offset + 2 * q, instruction, lane_scales + 4 * q,
                      column_scales + 4 * q * S::kBlocks, k > k0 || q > 0);
          mma_commit<kPair>(&h.empty[ring.stage]);
          if (k == k1 - 1) mma_commit<kPair>(&h.sum_full[b]);
        }
        __syncwarp();
      }
    }
    if (*aborted) {
      if (elect_one()) mma_commit<kPair>(&h.drained);
      barrier_drain(&h.drained, 0);
      drained = true;
    }
  } else if (warp > 1) {  // results: a warp reads lanes 32 (warp % 4) ... of its columns
    grid_wait();  // the scales may be the kernel's ahead, and what it reads may lie where this one writes
    const int quarter = warp & 3, slot = threadIdx.x - 64;
    const int part = (warp - 2) / 4 * S::kOutColumns;  // first column
    int t = 0;
    bool ok = true;  // once a wait has given up, the tiles are walked for their barriers alone
    for (int tile = first; tile < tiles; tile += step, ++t) {
      int lt, ct;
      place(a, tile, &lt, &ct);
      const int b = t % S::kSums, use = t / S::kSums;
      const int64_t column0 = static_cast<int64_t>(ct) * kColumns;
      const int columns = static_cast<int>(min(static_cast<int64_t>(kColumns), a.column.rows - column0));
      if (a.split == 1) {
        asm volatile("bar.sync 1, %0;" ::"n"(32 * S::kOutWarps) : "memory");  // the last tile's scales are no longer read
        if (slot < kColumns) {
          h.scale[slot] = slot < columns ? __ldg(a.column.scale + (a.column.per_row ? column0 + slot : 0)) : 0.0f;
          h.bias[slot] = a.column.bias && slot < columns ? __ldg(a.column.bias + column0 + slot) : 0.0f;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * S::kOutWarps) : "memory");
      }
      const int64_t row = static_cast<int64_t>(lane_block(lt)) * kLanes + quarter * 32 + lane;
      const bool in = row < a.lane.rows;
      const float row_scale = in ? __ldg(a.lane.scale + (a.lane.per_row ? row : 0)) : 0.0f;
      const float row_bias = in && a.lane.bias ? __ldg(a.lane.bias + row) : 0.0f;
      if (ok && !barrier_wait(&h.sum_full[b], use & 1, aborted, a.polls)) {
        if (lane == 0) give_up(a, aborted, 4);
        ok = false;
      }
      if (!ok) continue;
      __syncwarp();
      tcgen05_fence_after();
      // All of the warp's sums to registers, so that the tile's tensor memory is free at once.
      uint32_t v[S::kOutColumns / 16][16];
      const uint32_t from = tmem + b * kColumns + part + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll
      for (int c = 0; c < S::kOutColumns / 16; ++c) tmem_load16(from + 16 * c, v[c]);
      tmem_wait();
#pragma unroll
      for (int c = 0; c < S::kOutColumns / 16; ++c) tmem_loaded(v[c]);
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (kPair) barrier_arrive_at(&h.sum_empty[b], 0);
        else barrier_arrive(&h.sum_empty[b]);
      }
      if (a.split > 1) {
        float* partial = reinterpret_cast<float*>(stages) + part * kLanes + quarter * 32 + lane;  // [column][lane]
#pragma unroll
        for (int c = 0; c < S::kOutColumns; ++c) partial[c * kLanes] = __uint_as_float(v[c / 16][c % 16]);
      } else if (in) {
        O* to = static_cast<O*>(a.out) + row * a.lane.stride + (column0 + part) * a.column.stride;
        if (columns == kColumns && !a.column.bias) {
#pragma unroll
          for (int c = 0; c < S::kOutColumns; ++c, to += a.column.stride)
            *to = Values<O>::down(scaled(__uint_as_float(v[c / 16][c % 16]), row_scale, h.scale[part + c], row_bias));
        } else {
#pragma unroll
          for (int c = 0; c < S::kOutColumns; ++c, to += a.column.stride)
            if (part + c < columns)
              *to = Values<O>::down(scaled(__uint_as_float(v[c / 16][c % 16]), row_scale, h.scale[part + c],
                                           a.column.bias ? h.bias[part + c] : row_bias));
        }
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (*aborted) {  // by any role: no copy may land and no product run after the CTA has gone
    if (warp == 1 && issues && !drained) {
      if (elect_one()) mma_commit<kPair>(&h.drained);
      barrier_drain(&h.drained, 0);
    }
    if (!kPair && warp == 0)
      for (int u = max(0, loads - S::kStages); u < loads; ++u) barrier_drain(&h.full[u % S::kStages], (u / S::kStages) & 1);
    __syncthreads();
  }
  if (kPair) {
    if (threadIdx.x == 0) {
      remote_store(&h.peer_aborted, rank ^ 1, *aborted);
      remote_store(&h.peer_loads, rank ^ 1, loads);
    }
    __syncwarp();
    cluster_barrier();  // neither CTA goes while the other may still arrive on its barriers or use its memory
    if (*aborted || h.peer_aborted) {
      if (warp == 0 && issues) {  // the copies of both: a K tile that one of them has not asked for lacks its share
        const int other = h.peer_loads, most = max(loads, other);
        for (int u = max(0, most - S::kStages); u < most; ++u) {
          uint64_t* full = &h.full[u % S::kStages];
          if (elect_one()) {
            if (u >= loads) barrier_arrive_expect(full, S::kStageBytes);
            else if (u >= other) barrier_forgo(full, S::kStageBytes);
          }
          __syncwarp();
          barrier_drain(full, (u / S::kStages) & 1);
        }
      }
      cluster_barrier();
    }
  } else if (a.split > 1) {
    cluster_barrier();
    int lt, ct;
    place(a, first, &lt, &ct);
    const int64_t column0 = static_cast<int64_t>(ct) * kColumns;
    const int columns = static_cast<int>(min(static_cast<int64_t>(kColumns), a.column.rows - column0));
    // A thread adds up L neighbouring lanes of two columns at a time: four of a wide tile, where the other
    // CTAs' shared memory is read at its rate (512 x 2,048 x 4,096: 10.5 us, single lanes 13.9), one of a narrow
    // one, where there are threads enough (60 x 1,001 x 4,096: 6.7 us, four lanes 7.4).
    constexpr int L = kColumns >= 128 ? 4 : 1, kTeams = S::kThreads * L / kLanes;
    const int team = threadIdx.x * L / kLanes, at = threadIdx.x * L % kLanes;
    const int64_t row = static_cast<int64_t>(lt) * kLanes + at;
    const int rows = static_cast<int>(max(int64_t{0}, min(static_cast<int64_t>(L), a.lane.rows - row)));
    if (team < kTeams && rows > 0 && !*aborted) {
      float row_scale[L], row_bias[L];
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const int64_t r = row + min(i, rows - 1);
        row_scale[i] = __ldg(a.lane.scale + (a.lane.per_row ? r : 0));
        row_bias[i] = a.lane.bias ? __ldg(a.lane.bias + r) : 0.0f;
      }
      const int step = kTeams * a.split;
      for (int c0 = rank + team * a.split; c0 < columns; c0 += 2 * step) {
        Pack<float, L> part[2][8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int c = min(c0 + u * step, kColumns - 1);
#pragma unroll
          for (int r = 0; r < 8; ++r)  // its own first, so that the CTAs do not all read the same one
            if (r < a.split) remote_load(shared_addr(stages) + (c * kLanes + at) * 4, (rank + r) & (a.split - 1), part[u][r].v);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int c = c0 + u * step;
          if (c >= columns) break;
          const float scale = __ldg(a.column.scale + (a.column.per_row ? column0 + c : 0));
          O* to = static_cast<O*>(a.out) + row * a.lane.stride + (column0 + c) * a.column.stride;
#pragma unroll
          for (int i = 0; i < L; ++i) {
            // Opposite CTAs first: whichever rank a column falls to, the same pairs and the same sums of pairs,
            // so that equal rows of the operands give equal results.
            if (a.split == 8) {
#pragma unroll
              for (int r = 0; r < 4; ++r) part[u][r].v[i] += part[u][r + 4].v[i];
            }
            if (a.split >= 4) {
#pragma unroll
              for (int r = 0; r < 2; ++r) part[u][r].v[i] += part[u][r + 2].v[i];
            }
            const float sum = part[u][0].v[i] + part[u][1].v[i];
            if (i < rows)
              to[i * a.lane.stride] = Values<O>::down(scaled(sum, row_scale[i], scale, a.column.bias ? __ldg(a.column.bias + column0 + c) : row_bias[i]));
          }
        }
      }
    }
    cluster_barrier();
  }
  if (warp == 1) tmem_free<kPair>(tmem, kTmemColumns);
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

// Rows of 2,048 bytes, the block scales of 128 rows and 256 columns: [ceil(rows / 128), ceil(cols / 256), 256 words of 8 bytes].
bool map_scales(const Nvfp4& m, CUtensorMap* map) {
  const auto across = static_cast<cuuint64_t>(block_scale_tiles(m.cols) / 4);
  const cuuint64_t size[3] = {kScaleBytes / 8, across, static_cast<cuuint64_t>((m.rows + 127) / 128)};
  const cuuint64_t stride[2] = {kScaleBytes, kScaleBytes * across};
  const cuuint32_t box[3] = {kScaleBytes / 8, 1, 1}, one[3] = {1, 1, 1};
  return encoder() && encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT64, 3, m.block_scales, size, stride, box, one,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename O, int kColumns, bool kPair = false>
cudaError_t launch(const Nvfp4& lane, const Nvfp4& column, ProductArgs a, int sm_count, cudaStream_t stream) {
  using S = Shape<kColumns, kPair>;
  const int lanes = kPair ? 2 * kLanes : kLanes;
  a.lane_tiles = (a.lane.rows + lanes - 1) / lanes;
  a.column_tiles = (a.column.rows + kColumns - 1) / kColumns;
  const int64_t tiles = static_cast<int64_t>(a.lane_tiles) * a.column_tiles;
  if (tiles > 0x3fffffff) return cudaErrorInvalidConfiguration;
  Maps<kPair> maps;
  if (!map_codes(lane, kLanes, &maps.lane) || !map_codes(column, S::kColumnRows, &maps.column)) return cudaErrorInvalidValue;
  if constexpr (kPair) {
    if (!map_scales(lane, &maps.lane_scales) || !map_scales(column, &maps.column_scales)) return cudaErrorInvalidValue;
  }
  static SharedLimit limit;
  cudaError_t err = limit.raise(product_kernel<O, kColumns, kPair>, S::kShared);
  if (err != cudaSuccess) return err;
  // As many CTAs to a tile as leave every cluster a place at once: 74 clusters of 2, 33 of 4, 15 of 8 (8 x
  // 1,001 x 50,000: 10.9 us with eight, 46 with one; 16 tiles of 64 x 2,000 x 4,096: 7.7 with four, 12.6 with
  // eight, one of whose clusters has to wait).
  static ClusterLimit clusters[3];
  a.split = 1;
  for (int i = 0; !kPair && i < 3 && a.k_tiles >= 4 << i; ++i) {
    int most = 0;
    if ((err = clusters[i].most(product_kernel<O, kColumns, kPair>, 2 << i, S::kThreads, S::kShared, &most)) != cudaSuccess) return err;
    if (tiles > most) break;
    a.split = 2 << i;
  }
  const int group = kPair ? 2 : a.split;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(a.split > 1 ? tiles * a.split : std::min<int64_t>(tiles, sm_count / group) * group));
  config.blockDim = dim3(S::kThreads);
  config.dynamicSmemBytes = S::kShared;
  config.stream = stream;
  // The kernel may start while the one ahead of it in the stream ends; it waits before it reads (grid_wait).
  cudaLaunchAttribute attributes[2]{};
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim = {static_cast<unsigned>(group), 1, 1};
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attributes;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, product_kernel<O, kColumns, kPair>, maps, a);
}

}  // namespace

void set_product_polls(int polls) { g_polls.store(polls < 0 ? kBarrierPolls : std::min(polls, kBarrierPolls - 1), std::memory_order_relaxed); }

cudaError_t take_product_status(int* code, cudaStream_t stream) {
  void* word = nullptr;
  cudaError_t err = cudaGetSymbolAddress(&word, g_product_status);
  if (err == cudaSuccess) err = cudaMemcpyAsync(code, word, sizeof(int), cudaMemcpyDeviceToHost, stream);
  if (err == cudaSuccess) err = cudaStreamSynchronize(stream);
  if (err == cudaSuccess && *code != 0) err = cudaMemsetAsync(word, 0, sizeof(int), stream);
  return err;
}

cudaError_t launch_nvfp4_product(const Nvfp4& a, const Nvfp4& b, const float* bias, const Dense& out,
                                 bool b_ready, int* status, cudaStream_t stream) {
  return with_type(out.type, [&](auto zero) {
    using O = decltype(zero);
    const Side rows{a.block_scales, a.scale, nullptr, out.stride, static_cast<int32_t>(a.rows), a.per_row};
    const Side cols{b.block_scales, b.scale, bias, 1, static_cast<int32_t>(b.rows), b.per_row};
    ProductArgs args{};
    args.out = out.data;
    args.scale_tiles = block_scale_tiles(a.cols);
    args.k_tiles = static_cast<int32_t>((a.cols + 255) / 256);
    args.status = status;
    args.polls = g_polls.load(std::memory_order_relaxed);
    // Few rows of b (a narrow readout of many states) go along the columns (8,192 x 25 x 4,096: 10.3 us against
    // 20.1 along the lanes; 300 x 25 x 4,096: 6.1 against 10.8); else b along the lanes, where neighbouring
    // lanes write neighbouring outputs.
    const bool narrow = b.rows <= 128 && b.rows < a.rows;
    args.lane = narrow ? rows : cols;
    args.column = narrow ? cols : rows;
    args.lane_ready = b_ready && !narrow;
    const Nvfp4 &x = narrow ? a : b, &y = narrow ? b : a;
    DeviceInfo info;
    const cudaError_t err = device_info(&info);
    if (err != cudaSuccess) return err;
    // The least tile that holds all columns (1 x 32,000 x 4,096: 15.3 us with 16 columns, 21.9 with 128;
    // 60 x 16,000 x 4,096: 10.7 with 64, 14.2 with 128).  Beyond 128 (a tile has to start on a 128-row tile
    // of block scales) pairs' tiles of 256 lanes x 256 columns, unless all tiles of 128 x 128 run at once
    // (1,024 x 2,048 x 4,096: 7.9 us, pairs 10.5; 256 x 2,048 x 16,384: 13.4 on four CTAs a tile, pairs 24.4;
    // 2,048 x 2,048 x 4,096: pairs 11.1, 128 x 128 12.3; 8,192 x 8,192 x 4,096: pairs 109, 128 x 128 143).
    if (y.rows <= 16) return launch<O, 16>(x, y, args, info.sm_count, stream);
    if (y.rows <= 32) return launch<O, 32>(x, y, args, info.sm_count, stream);
    if (y.rows <= 64) return launch<O, 64>(x, y, args, info.sm_count, stream);
    if ((x.rows + 127) / 128 * ((y.rows + 127) / 128) <= info.sm_count || y.rows <= 128) return launch<O, 128>(x, y, args, info.sm_count, stream);
    return launch<O, 256, true>(x, y, args, info.sm_count, stream);
  });
}

}  // namespace nsb
