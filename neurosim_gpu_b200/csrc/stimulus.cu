// stimulus.cu -- token ids to drive rows, and the gradient of the stimulus table.
//
//   drive:    out[t, :]   = round(scale * table[token[t], :])
//   gradient: dtable[v,:] = round(scale * sum over {t : token[t] = v} of dout[t, :])
//
// A token outside [0, rows) is "no stimulus": a zero row, and no gradient.  Both are
// bound by memory: the drive reads each used row once and writes T rows; the gradient
// reads T rows and writes the whole table.
//
// The gradient is deterministic: the sum of a row runs over its occurrences in
// ascending t, in float32, cut at fixed tiles of the sorted order and joined in
// ascending tile order.  Three launches:
//   1. sort_fill_kernel: one cluster sorts (token, t) stably, byte by byte (radix
//      sort; the keys stay in L2), while all other clusters write the table's zeros.
//      The sort is all latency, the zeros are all bandwidth: neither waits.
//   2. segment_kernel: one CTA per (tile of the sorted order, slice of the columns)
//      sums runs of equal tokens; a run inside the tile is written to its row, one
//      that crosses the tile's edge goes to the workspace as a float32 partial.
//   3. join_kernel: the tile where such a run starts adds its partials.
// A token that makes up most of a batch is thereby spread over all SMs, like any other.
#include <cooperative_groups.h>

#include <algorithm>

#include "nsb_tokens.h"

namespace cg = cooperative_groups;

namespace nsb {
namespace {

constexpr int kDriveThreads = 256;
constexpr int kSortCtas = 8;       // one portable cluster
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kDigits = 256;
constexpr int kSegmentThreads = 128;
constexpr int kJoinGroups = 16;

__device__ __forceinline__ int64_t token_at(const void* tokens, int bytes, int64_t t) {
  return bytes == 8 ? __ldg(static_cast<const long long*>(tokens) + t)
                    : static_cast<int64_t>(__ldg(static_cast<const int*>(tokens) + t));
}

// ---------------------------------------------------------------------------
// Drive
// ---------------------------------------------------------------------------

// blockDim = (vectors of a row, rows of the block); the grid runs over row groups x column chunks.
template <typename In, typename O, int V>
__global__ void __launch_bounds__(kDriveThreads)
drive_kernel(const void* tokens, int token_bytes, int64_t n, Dense table, float scale, Dense out,
             int64_t chunks) {
  const int64_t group = blockIdx.x / chunks;
  const int64_t t = group * blockDim.y + threadIdx.y;
  const int64_t c = ((blockIdx.x - group * chunks) * blockDim.x + threadIdx.x) * V;
  if (t >= n || c >= out.cols) return;
  const int64_t token = token_at(tokens, token_bytes, t);
  O* to = static_cast<O*>(out.data) + t * out.stride + c;
  Pack<O, V> r;
  if (token >= 0 && token < table.rows) {
    const Pack<In, V> x = load_pack<In, V>(static_cast<const In*>(table.data) + token * table.stride + c);
    float y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = __fmul_rn(Values<In>::up(x.v[i]), scale);
    r = round_pack<O, V>(y);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = Values<O>::down(0.0f);
  }
  store_pack<O, V>(to, r);
}

// ---------------------------------------------------------------------------
// Gradient
// ---------------------------------------------------------------------------

// Workspace: keys and positions, two buffers each, then the partial rows.
struct Sorted {
  uint32_t* key[2];
  uint32_t* pos[2];
};

// Stable least-significant-byte radix sort of the keys min(token, limit) by one cluster.
// Warp g of the cluster's 256 owns elements [g * span, (g + 1) * span).  Per pass: each warp
// counts its digits; a scan over (digit, CTA, warp) gives each warp the first slot of each of
// its digits; the warp walks its elements again in order and places them.
__device__ void sort_tokens(cg::cluster_group& cluster, const void* tokens, int token_bytes,
                            int64_t n, int64_t limit, const Sorted& s, int passes,
                            uint32_t (*hist)[kDigits], uint32_t* totals, uint32_t* scan) {
  const int rank = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t span = ((n + kSortCtas * kSortWarps - 1) / (kSortCtas * kSortWarps) + 31) / 32 * 32;
  const int64_t first = (rank * kSortWarps + warp) * span;
  const int64_t last = min(n, first + span);
  const uint32_t below = (1u << lane) - 1u;
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = 8 * pass;
    // L1 is not coherent between SMs: the other CTAs' keys of the last pass are read from L2.
    auto key_of = [&](int64_t i) -> uint32_t {
      if (pass > 0) return __ldcg(s.key[(pass - 1) & 1] + i);
      const int64_t token = token_at(tokens, token_bytes, i);
      return static_cast<uint32_t>(token < 0 || token >= limit ? limit : token);
    };
    for (int d = lane; d < kDigits; d += 32) hist[warp][d] = 0;
    __syncwarp();
    for (int64_t i = first; i < last; i += 32) {
      const bool in = i + lane < last;
      const uint32_t digit = in ? (key_of(i + lane) >> shift) & (kDigits - 1) : ~0u;
      const uint32_t same = __match_any_sync(0xffffffffu, digit);
      if (in && (same & below) == 0) hist[warp][digit] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
      uint32_t sum = 0;
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = hist[w][threadIdx.x];
        hist[w][threadIdx.x] = sum;
        sum += c;
      }
      totals[threadIdx.x] = sum;
    }
    cluster.sync();
    uint32_t before = 0, all = 0;
    if (threadIdx.x < kDigits) {
      for (int c = 0; c < kSortCtas; ++c) {
        const uint32_t x = *cluster.map_shared_rank(totals + threadIdx.x, c);
        before += c < rank ? x : 0;
        all += x;
      }
      // Exclusive scan over the digits: within the warp, then over the 8 warps that hold them.
      uint32_t sum = all;
      for (int off = 1; off < 32; off <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += up;
      }
      if (lane == 31) scan[warp] = sum;
      all = sum - all;
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
      uint32_t base = before + all;
      for (int w = 0; w < warp; ++w) base += scan[w];
      for (int w = 0; w < kSortWarps; ++w) hist[w][threadIdx.x] += base;
    }
    __syncthreads();
    uint32_t* key_out = s.key[pass & 1];
    uint32_t* pos_out = s.pos[pass & 1];
    for (int64_t i = first; i < last; i += 32) {
      const bool in = i + lane < last;
      const uint32_t key = in ? key_of(i + lane) : 0;
      const uint32_t pos = !in ? 0 : pass > 0 ? __ldcg(s.pos[(pass - 1) & 1] + i + lane)
                                              : static_cast<uint32_t>(i + lane);
      const uint32_t digit = in ? (key >> shift) & (kDigits - 1) : ~0u;
      const uint32_t same = __match_any_sync(0xffffffffu, digit);
      uint32_t slot = 0;
      if (in) slot = hist[warp][digit] + __popc(same & below);
      __syncwarp();
      if (in && (same & below) == 0) hist[warp][digit] += __popc(same);
      __syncwarp();
      if (in) {
        key_out[slot] = key;
        pos_out[slot] = pos;
      }
    }
    cluster.sync();  // also orders this pass's keys in global memory before the next pass reads them
  }
}

template <typename O, int V>
__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(kSortThreads)
sort_fill_kernel(const void* tokens, int token_bytes, int64_t n, Sorted s, int passes, Dense out) {
  __shared__ uint32_t hist[kSortWarps][kDigits];
  __shared__ uint32_t totals[kDigits];
  __shared__ uint32_t scan[kDigits / 32];
  cg::cluster_group cluster = cg::this_cluster();
  if (blockIdx.x < kSortCtas) {
    sort_tokens(cluster, tokens, token_bytes, n, out.rows, s, passes, hist, totals, scan);
    return;
  }
  const int64_t vectors = out.cols / V;  // V divides the columns
  const int64_t all = out.rows * vectors;
  const int64_t stride = static_cast<int64_t>(gridDim.x - kSortCtas) * kSortThreads;
  Pack<O, V> zero;
#pragma unroll
  for (int i = 0; i < V; ++i) zero.v[i] = Values<O>::down(0.0f);
  int64_t i = static_cast<int64_t>(blockIdx.x - kSortCtas) * kSortThreads + threadIdx.x;
  if (out.stride == out.cols) {
    for (; i < all; i += stride) store_pack<O, V>(static_cast<O*>(out.data) + i * V, zero);
  } else {
    for (; i < all; i += stride) {
      const int64_t row = i / vectors;
      store_pack<O, V>(static_cast<O*>(out.data) + row * out.stride + (i - row * vectors) * V, zero);
    }
  }
}

// Partial row (tile, slot): slot 0 continues a run of the tile before, slot 1 starts one that goes on.
struct Partials {
  float* data;
  int64_t pitch;  // floats, a multiple of 8
  __device__ __forceinline__ float* row(int64_t tile, int slot) const {
    return data + (2 * tile + slot) * pitch;
  }
};

template <typename In, typename O, int V>
__global__ void __launch_bounds__(kSegmentThreads)
segment_kernel(const uint32_t* __restrict__ key, const uint32_t* __restrict__ pos, int64_t n,
               int tile, Dense grad, float scale, Dense out, Partials partials, int slices) {
  constexpr int U = 8;  // rows in flight per thread
  const int64_t j = blockIdx.x / slices;
  const int64_t c = (static_cast<int64_t>(blockIdx.x - j * slices) * kSegmentThreads + threadIdx.x) * V;
  if (c >= grad.cols) return;
  const int64_t i0 = j * tile, i1 = min(n, i0 + tile);
  const uint32_t limit = static_cast<uint32_t>(out.rows);
  uint32_t run = __ldg(key + i0);
  bool head = i0 > 0 && __ldg(key + i0 - 1) == run;
  float acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.0f;
  auto flush = [&](bool tail) {
    if (run >= limit) return;
    if (!head && !tail) {
      float r[V];
#pragma unroll
      for (int v = 0; v < V; ++v) r[v] = __fmul_rn(acc[v], scale);
      store_pack<O, V>(static_cast<O*>(out.data) + run * out.stride + c, round_pack<O, V>(r));
    } else {
      float* to = partials.row(j, head ? 0 : 1) + c;
#pragma unroll
      for (int v = 0; v < V; ++v) to[v] = acc[v];
    }
  };
  for (int64_t i = i0; i < i1; i += U) {
    uint32_t k[U];
    Pack<In, V> g[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      k[u] = i + u < i1 ? __ldg(key + i + u) : limit;
      const uint32_t p = i + u < i1 ? __ldg(pos + i + u) : 0;
      if (k[u] < limit) {
        g[u] = load_pack<In, V>(static_cast<const In*>(grad.data) + p * grad.stride + c);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) g[u].v[v] = Values<In>::down(0.0f);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u < i1) {
        if (k[u] != run) {
          flush(false);
          head = false;
          run = k[u];
#pragma unroll
          for (int v = 0; v < V; ++v) acc[v] = 0.0f;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] += Values<In>::up(g[u].v[v]);
      }
    }
  }
  flush(i1 < n && __ldg(key + i1) == run);
}

// Tile j joins the run that starts in it and goes on into later tiles.  16 groups of 32 lanes
// take every 16th tile of the run; their sums are added in group order.
template <typename O>
__global__ void __launch_bounds__(32 * kJoinGroups)
join_kernel(const uint32_t* __restrict__ key, int64_t n, int tile, float scale, Dense out,
            Partials partials) {
  __shared__ float4 sums[kJoinGroups][32];
  const int64_t j = blockIdx.x, i1 = (j + 1) * tile;
  if (i1 >= n) return;
  const uint32_t run = __ldg(key + i1 - 1);
  if (run >= static_cast<uint32_t>(out.rows) || __ldg(key + i1) != run) return;
  if (j > 0 && __ldg(key + j * tile - 1) == run) return;  // the run started earlier
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
  // The last tile that the run reaches: 32 tiles' first keys at a time.
  int64_t last = j;
  for (;;) {
    const int64_t first = (last + 1 + lane) * tile;
    const uint32_t stop = __ballot_sync(0xffffffffu, first >= n || __ldg(key + min(first, n - 1)) != run);
    last += stop ? __ffs(stop) - 1 : 32;
    if (stop) break;
  }
  for (int64_t c0 = static_cast<int64_t>(blockIdx.y) * 128; c0 < out.cols; c0 += gridDim.y * 128) {
    const int64_t c = c0 + 4 * lane;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (c < out.cols) {  // the pitch is a multiple of 8: a float4 stays inside the row
#pragma unroll 4
      for (int64_t t = j + group; t <= last; t += kJoinGroups) {
        const float4 x = *reinterpret_cast<const float4*>(partials.row(t, t == j ? 1 : 0) + c);
        sum.x += x.x;
        sum.y += x.y;
        sum.z += x.z;
        sum.w += x.w;
      }
    }
    sums[group][lane] = sum;
    __syncthreads();
    if (group == 0) {
      for (int g = 1; g < kJoinGroups; ++g) {
        const float4 x = sums[g][lane];
        sum.x += x.x;
        sum.y += x.y;
        sum.z += x.z;
        sum.w += x.w;
      }
      const float r[4] = {sum.x, sum.y, sum.z, sum.w};
      for (int v = 0; v < 4; ++v)
        if (c + v < out.cols)
          static_cast<O*>(out.data)[run * out.stride + c + v] = Values<O>::down(__fmul_rn(r[v], scale));
    }
    __syncthreads();
  }
}

int64_t partial_pitch(int64_t cols) { return (cols + 7) / 8 * 8; }

// Long tiles leave fewer partials; short ones fill the GPU: about eight CTAs on each of 148 SMs.
int64_t tile_of(int64_t n, int64_t slices) {
  return std::max<int64_t>(8, std::min<int64_t>(64, n * slices / (148 * 8)));
}

template <typename In, typename O, int V>
cudaError_t drive(const void* tokens, int token_bytes, int64_t n, const Dense& table, float scale,
                  const Dense& out, cudaStream_t stream) {
  const int64_t vectors = (out.cols + V - 1) / V;
  int x = 32;
  while (x < kDriveThreads && x < vectors) x *= 2;
  const dim3 block(x, kDriveThreads / x);
  const int64_t chunks = (vectors + x - 1) / x;
  const int64_t groups = (n + block.y - 1) / block.y;
  if (chunks * groups > 0x7fffffff) return cudaErrorInvalidConfiguration;
  drive_kernel<In, O, V><<<static_cast<unsigned>(chunks * groups), block, 0, stream>>>(
      tokens, token_bytes, n, table, scale, out, chunks);
  return cudaGetLastError();
}

template <typename In, typename O, int V>
cudaError_t gradient(const void* tokens, int token_bytes, const Dense& grad, float scale,
                     const Dense& out, void* workspace, cudaStream_t stream) {
  DeviceInfo info;
  cudaError_t err = device_info(&info);
  if (err != cudaSuccess) return err;
  const int64_t n = grad.rows;
  const int64_t padded = (n + 3) / 4 * 4;
  auto* words = static_cast<uint32_t*>(workspace);
  const Sorted s{{words, words + padded}, {words + 2 * padded, words + 3 * padded}};
  const Partials partials{reinterpret_cast<float*>(words + 4 * padded), partial_pitch(out.cols)};
  int passes = 1;
  while (passes < 4 && (out.rows >> (8 * passes)) > 0) ++passes;
  const int64_t fill = (out.rows * (out.cols / V) + kSortThreads - 1) / kSortThreads;
  const int64_t clusters = 1 + std::min<int64_t>((fill + kSortCtas - 1) / kSortCtas, info.sm_count / kSortCtas * 2);
  sort_fill_kernel<O, V><<<static_cast<unsigned>(clusters * kSortCtas), kSortThreads, 0, stream>>>(
      tokens, token_bytes, n, s, n > 0 ? passes : 0, out);
  if ((err = cudaGetLastError()) != cudaSuccess || n == 0) return err;
  const uint32_t* key = s.key[(passes - 1) & 1];
  const uint32_t* pos = s.pos[(passes - 1) & 1];
  const int64_t slices = (out.cols / V + kSegmentThreads - 1) / kSegmentThreads;
  const int tile = static_cast<int>(tile_of(n, slices));
  const int64_t tiles = (n + tile - 1) / tile;
  if (tiles * slices > 0x7fffffff) return cudaErrorInvalidConfiguration;
  segment_kernel<In, O, V><<<static_cast<unsigned>(tiles * slices), kSegmentThreads, 0, stream>>>(
      key, pos, n, tile, grad, scale, out, partials, static_cast<int>(slices));
  if ((err = cudaGetLastError()) != cudaSuccess || tiles == 1) return err;
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(std::min<int64_t>(8, (out.cols + 127) / 128)));
  join_kernel<O><<<grid, 32 * kJoinGroups, 0, stream>>>(key, n, tile, scale, out, partials);
  return cudaGetLastError();
}

// The widest vector, up to 16 bytes of `In`, that divides the columns and fits both matrices' rows.
template <typename In, typename O>
int vector_of(const Dense& in, const Dense& out) {
  for (int v = 16 / static_cast<int>(sizeof(In)); v > 1; v /= 2)
    if (out.cols % v == 0 && rows_aligned(in, sizeof(In), v * sizeof(In)) &&
        rows_aligned(out, sizeof(O), v * sizeof(O)))
      return v;
  return 1;
}

}  // namespace

cudaError_t launch_stimulus_drive(const void* tokens, int token_bytes, int64_t n, const Dense& table,
                                  float scale, const Dense& out, cudaStream_t stream) {
  return with_type(table.type, [&](auto in) {
    using In = decltype(in);
    auto call = [&](auto o) {
      using O = decltype(o);
      const int v = vector_of<In, O>(table, out);
      if (sizeof(In) == 2 && v == 8) return drive<In, O, sizeof(In) == 2 ? 8 : 4>(tokens, token_bytes, n, table, scale, out, stream);
      if (v >= 4) return drive<In, O, 4>(tokens, token_bytes, n, table, scale, out, stream);
      if (v == 2) return drive<In, O, 2>(tokens, token_bytes, n, table, scale, out, stream);
      return drive<In, O, 1>(tokens, token_bytes, n, table, scale, out, stream);
    };
    return out.type == NSB_VALUE_F32 ? call(float{}) : call(in);
  });
}

size_t stimulus_gradient_workspace_bytes(int64_t n, int64_t cols) {
  // The fewest slices (eight values per thread) give the shortest tiles, so the most partials.
  const int64_t tile = tile_of(n, (cols + 8 * kSegmentThreads - 1) / (8 * kSegmentThreads));
  const int64_t padded = (n + 3) / 4 * 4, tiles = (n + tile - 1) / tile;
  return static_cast<size_t>(16 * padded + 8 * tiles * partial_pitch(cols));
}

cudaError_t launch_stimulus_gradient(const void* tokens, int token_bytes, const Dense& grad,
                                     float scale, const Dense& out, void* workspace,
                                     cudaStream_t stream) {
  return with_type(grad.type, [&](auto in) {
    using In = decltype(in);
    auto call = [&](auto o) {
      using O = decltype(o);
      const int v = vector_of<In, O>(grad, out);
      if (sizeof(In) == 2 && v == 8) return gradient<In, O, sizeof(In) == 2 ? 8 : 4>(tokens, token_bytes, grad, scale, out, workspace, stream);
      if (v >= 4) return gradient<In, O, 4>(tokens, token_bytes, grad, scale, out, workspace, stream);
      if (v == 2) return gradient<In, O, 2>(tokens, token_bytes, grad, scale, out, workspace, stream);
      return gradient<In, O, 1>(tokens, token_bytes, grad, scale, out, workspace, stream);
    };
    if constexpr (sizeof(In) == 4) return with_type(out.type, call);  // a wide drive of a narrow table
    return out.type == NSB_VALUE_F32 ? call(float{}) : call(in);
  });
}

}  // namespace nsb
