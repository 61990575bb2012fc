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
//      sort; the pairs stay in L2), while all other clusters write the table's zeros.
//      The sort is all latency, the zeros are all bandwidth: neither waits.
//   2. segment_kernel: one CTA per (tile of the sorted order, slice of the columns)
//      sums runs of equal tokens; a run inside the tile is written to its row, one
//      that crosses the tile's edge goes to the workspace as a float32 partial.
//   3. join_kernel: the tile where such a run starts adds its partials.
// A token that makes up most of a batch is thereby spread over all SMs, like any other.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "nsb_tokens.h"

namespace cg = cooperative_groups;

namespace nsb {
namespace {

constexpr int kDriveThreads = 256;
constexpr int kSortCtas = 8;       // one portable cluster
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kDigits = 256;
constexpr int kHeld = 8;           // of a warp's rounds in registers: 65,536 tokens in all
constexpr int kSegmentThreads = 128;
constexpr int kTileMost = 64;
constexpr int kJoinWarps = 8;

__device__ __forceinline__ int64_t token_at(const void* tokens, int bytes, int64_t t) {
  return bytes == 8 ? __ldg(static_cast<const long long*>(tokens) + t)
                    : static_cast<int64_t>(__ldg(static_cast<const int*>(tokens) + t));
}

// ---------------------------------------------------------------------------
// Drive
// ---------------------------------------------------------------------------

// 16 bytes of values from any place p.  Off a 16-byte boundary they are cut out of the two aligned
// vectors around them, as long as these lie within [first, last); p + 16 bytes does.
template <typename T>
__device__ __forceinline__ Pack<T, 16 / sizeof(T)> load_anywhere(const T* p, const T* first, const T* last) {
  constexpr int P = 16 / static_cast<int>(sizeof(T));
  const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
  if (lead == 0) return load_pack<T, P>(p);
  Pack<T, P> r;
  const T* from = p - lead;
  if (from >= first && from + 2 * P <= last) {
    const uint4 a = *reinterpret_cast<const uint4*>(from), b = *(reinterpret_cast<const uint4*>(from) + 1);
    const uint32_t all[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    const int words = lead * static_cast<int>(sizeof(T)) / 4, bits = lead * static_cast<int>(sizeof(T)) % 4 * 8;
    auto* to = reinterpret_cast<uint32_t*>(&r);
    auto cut = [&](auto skip) {
      constexpr int kSkip = decltype(skip)::value;
#pragma unroll
      for (int i = 0; i < 4; ++i) to[i] = __funnelshift_r(all[i + kSkip], all[(i + kSkip + 1) % 8], bits);
    };
    if (words == 0) cut(std::integral_constant<int, 0>{});
    else if (words == 1) cut(std::integral_constant<int, 1>{});
    else if (words == 2) cut(std::integral_constant<int, 2>{});
    else cut(std::integral_constant<int, 3>{});
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) r.v[i] = p[i];
  }
  return r;
}

// blockDim = (vectors of a row, rows of the block); the grid runs over row groups x column chunks.  A
// vector is 16 bytes of the table's type.  kAligned: rows of both matrices start on vectors; else a row
// is cut where its output reaches a vector's boundary, and the table's values are shifted into place
// (4,000 x 4,001 bf16: 14.4 us; single columns a warp's width apart 20.0; on vectors 6 would do).
// Bound by HBM: 160 ids x 166,000 bf16 to f32 23.8 us, 6.7 TB/s with the table's rows counted once.
template <typename In, typename O, bool kAligned>
__global__ void __launch_bounds__(kDriveThreads)
drive_kernel(const void* tokens, int token_bytes, int64_t n, Dense table, float scale, Dense out,
             unsigned chunks) {
  constexpr int V = 16 / static_cast<int>(sizeof(In));
  const unsigned group = blockIdx.x / chunks;
  const int64_t t = static_cast<int64_t>(group) * blockDim.y + threadIdx.y;
  if (t >= n) return;
  O* row = static_cast<O*>(out.data) + t * out.stride;
  const int shift = kAligned ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(row) % (V * sizeof(O)) / sizeof(O));
  const int64_t c = static_cast<int64_t>((blockIdx.x - group * chunks) * blockDim.x + threadIdx.x) * V - shift;
  if (c >= out.cols) return;
  const int64_t token = token_at(tokens, token_bytes, t);
  const bool valid = token >= 0 && token < table.rows;
  const In* first = static_cast<const In*>(table.data);
  const In* from = first + (valid ? token : 0) * table.stride;
  if (c >= 0 && c + V <= out.cols) {
    float y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = 0.0f;
    if (valid) {
      Pack<In, V> x;
      if constexpr (kAligned) x = load_pack<In, V>(from + c);
      else x = load_anywhere<In>(from + c, first, first + (table.rows - 1) * table.stride + table.cols);
#pragma unroll
      for (int i = 0; i < V; ++i) y[i] = __fmul_rn(Values<In>::up(x.v[i]), scale);
    }
    store_pack<O, V>(row + c, round_pack<O, V>(y));
  } else {
    for (int i = 0; i < V; ++i)
      if (c + i >= 0 && c + i < out.cols)
        row[c + i] = Values<O>::down(valid ? __fmul_rn(Values<In>::up(from[c + i]), scale) : 0.0f);
  }
}

// ---------------------------------------------------------------------------
// Gradient
// ---------------------------------------------------------------------------

// Workspace: keys and positions, two buffers each, then the partial rows.
struct Sorted {
  uint2* pair[2];  // key and position
};

// Elements of a warp.
__host__ __device__ inline int64_t sort_span(int64_t n) {
  return ((n + kSortCtas * kSortWarps - 1) / (kSortCtas * kSortWarps) + 31) / 32 * 32;
}

// Stable least-significant-byte radix sort of the keys min(token, limit) by one cluster.
// Warp g of the cluster's 256 owns elements [g * span, (g + 1) * span).  Per pass: each warp
// counts its digits; a scan over (digit, CTA, warp) gives each warp the first slot of each of
// its digits; the warp walks its elements again in order and places them: in the CTA's shared memory
// first, from where each digit's elements leave side by side (single words scattered over global memory:
// 22.2 us, this way 19.0 for 32,768 ids in two passes), or at once where a warp has too many to hold.
// All latency; more than one cluster would have to meet in global memory between the passes.
__device__ void sort_tokens(cg::cluster_group& cluster, const void* tokens, int token_bytes,
                            int64_t n, int64_t limit, const Sorted& s, int passes,
                            uint32_t (*hist)[kDigits], uint32_t* totals, uint2* scan, uint2* first_of, uint2* local) {
  const int rank = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t span = sort_span(n);
  const bool staged = span <= 32 * kHeld;
  const int64_t first = (rank * kSortWarps + warp) * span;
  const int64_t last = min(n, first + span);
  const uint32_t below = (1u << lane) - 1u;
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = 8 * pass;
    // L1 is not coherent between SMs: the other CTAs' keys of the last pass are read from L2.
    auto pair_of = [&](int64_t i) -> uint2 {
      if (pass > 0) return __ldcg(s.pair[(pass - 1) & 1] + i);
      const int64_t token = token_at(tokens, token_bytes, i);
      return make_uint2(static_cast<uint32_t>(token < 0 || token >= limit ? limit : token), static_cast<uint32_t>(i));
    };
    // The first kHeld rounds of 32 elements stay in registers for both walks.
    uint2 held[kHeld];
#pragma unroll
    for (int r = 0; r < kHeld; ++r) {
      const int64_t i = first + 32 * r + lane;
      held[r] = i < last ? pair_of(i) : make_uint2(0, 0);
    }
    for (int d = lane; d < kDigits; d += 32) hist[warp][d] = 0;
    __syncwarp();
    // The lanes that hold the same digit, of those that hold one.
    auto equals = [&](bool in, uint32_t key) {
      uint32_t same = __ballot_sync(0xffffffffu, in);
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const bool bit = key >> (shift + b) & 1;
        const uint32_t set = __ballot_sync(0xffffffffu, bit);
        same &= bit ? set : ~set;
      }
      return same;
    };
    auto count = [&](bool in, uint32_t key, uint32_t same) {
      if (in && (same & below) == 0) hist[warp][(key >> shift) & (kDigits - 1)] += __popc(same);
      __syncwarp();
    };
    uint32_t held_same[kHeld];
#pragma unroll
    for (int r = 0; r < kHeld; ++r) {
      const bool in = first + 32 * r + lane < last;
      if (first + 32 * r < last) count(in, held[r].x, held_same[r] = equals(in, held[r].x));
    }
    for (int64_t i = first + 32 * kHeld; i < last; i += 32) {
      const bool in = i + lane < last;
      const uint32_t key = in ? pair_of(i + lane).x : 0;
      count(in, key, equals(in, key));
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
      uint32_t c[kSortWarps], sum = 0;
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) c[w] = hist[w][threadIdx.x];
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        hist[w][threadIdx.x] = sum;
        sum += c[w];
      }
      totals[threadIdx.x] = sum;
    }
    cluster.sync();
    uint32_t before = 0, all = 0, here = 0;
    if (threadIdx.x < kDigits) {
      uint32_t x[kSortCtas];
#pragma unroll
      for (int c = 0; c < kSortCtas; ++c) x[c] = *cluster.map_shared_rank(totals + threadIdx.x, c);
#pragma unroll
      for (int c = 0; c < kSortCtas; ++c) {
        before += c < rank ? x[c] : 0;
        all += x[c];
      }
      // Exclusive scans over the digits, of the cluster and of the CTA: within the warp, then over the 8
      // warps that hold them.
      here = totals[threadIdx.x];
      uint32_t sum = all, own = here;
      for (int off = 1; off < 32; off <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, sum, off), up_own = __shfl_up_sync(0xffffffffu, own, off);
        if (lane >= off) {
          sum += up;
          own += up_own;
        }
      }
      if (lane == 31) scan[warp] = make_uint2(sum, own);
      all = sum - all;
      here = own - here;
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
      uint32_t base = before + all;
      for (int w = 0; w < warp; ++w) {
        base += scan[w].x;
        here += scan[w].y;
      }
      first_of[threadIdx.x] = make_uint2(base, here);
    }
    __syncthreads();
    uint2* pair_out = s.pair[pass & 1];
    auto place = [&](bool in, uint2 pair, uint32_t same) {
      const uint32_t digit = (pair.x >> shift) & (kDigits - 1);
      uint32_t slot = 0;
      if (in) slot = (staged ? first_of[digit].y : first_of[digit].x) + hist[warp][digit] + __popc(same & below);
      __syncwarp();
      if (in && (same & below) == 0) hist[warp][digit] += __popc(same);
      __syncwarp();
      if (in) (staged ? local : pair_out)[slot] = pair;
    };
#pragma unroll
    for (int r = 0; r < kHeld; ++r)
      if (first + 32 * r < last) place(first + 32 * r + lane < last, held[r], held_same[r]);
    for (int64_t i = first + 32 * kHeld; i < last; i += 32) {
      const bool in = i + lane < last;
      const uint2 pair = in ? pair_of(i + lane) : make_uint2(0, 0);
      place(in, pair, equals(in, pair.x));
    }
    if (staged) {  // sorted within the CTA first, so that a digit's elements leave side by side
      __syncthreads();
      const int64_t start = rank * kSortWarps * span;
      const int elements = static_cast<int>(max(int64_t{0}, min(n - start, kSortWarps * span)));
      for (int i = threadIdx.x; i < elements; i += kSortThreads) {
        const uint2 pair = local[i];
        const uint2 first_one = first_of[(pair.x >> shift) & (kDigits - 1)];
        pair_out[first_one.x + static_cast<uint32_t>(i) - first_one.y] = pair;
      }
    }
    cluster.sync();  // also orders this pass's keys in global memory before the next pass reads them
  }
}

__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(kSortThreads)
sort_fill_kernel(const void* tokens, int token_bytes, int64_t n, Sorted s, int passes, Dense out, int bytes_each) {
  __shared__ uint32_t hist[kSortWarps][kDigits];
  __shared__ uint32_t totals[kDigits];
  __shared__ uint2 scan[kDigits / 32];
  __shared__ uint2 first_of[kDigits];  // of the cluster and of the CTA
  extern __shared__ uint2 local[];     // the CTA's elements, where a warp holds its own
  cg::cluster_group cluster = cg::this_cluster();
  if (blockIdx.x < kSortCtas) {
    sort_tokens(cluster, tokens, token_bytes, n, out.rows, s, passes, hist, totals, scan, first_of, local);
    return;
  }
  // Zero is all bits clear in every type.  The CTAs share the 16-byte vectors of contiguous rows, or take
  // a row each.
  const bool whole = out.stride == out.cols;
  const int64_t ctas = gridDim.x - kSortCtas, cta = blockIdx.x - kSortCtas;
  const int64_t bytes = (whole ? out.rows : 1) * out.cols * bytes_each;
  const int64_t stride = (whole ? ctas : 1) * kSortThreads, own = (whole ? cta : 0) * kSortThreads + threadIdx.x;
  for (int64_t r = whole ? 0 : cta; r < (whole ? 1 : out.rows); r += ctas) {
    uint8_t* row = static_cast<uint8_t*>(out.data) + r * out.stride * bytes_each;
    const int64_t head = min(bytes, static_cast<int64_t>((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16));
    const int64_t vectors = (bytes - head) / 16;
    for (int64_t i = own; i < vectors; i += stride) __stcs(reinterpret_cast<uint4*>(row + head) + i, make_uint4(0, 0, 0, 0));
    if (own < head) row[own] = 0;
    if (own < bytes - head - vectors * 16) row[head + vectors * 16 + own] = 0;
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

// A thread sums 16 bytes' worth of columns: a vector (kAligned: rows of both matrices start on vectors),
// or single columns kSegmentThreads apart (60,000 tokens x 1,001 bf16: 40 us; cutting vectors out of
// aligned loads 95: too many selects in front of the sums).  Bound by HBM where tokens do not repeat much:
// 32,768 x 2,048 bf16 31.7 us, 4.2 TB/s.
template <typename In, typename O, bool kAligned>
__global__ void __launch_bounds__(kSegmentThreads, kAligned ? 8 : 6)
segment_kernel(const uint2* __restrict__ sorted, int64_t n,
               int tile, Dense grad, float scale, Dense out, Partials partials, int slices) {
  constexpr int U = kAligned ? 8 : 4;  // rows in flight per thread
  constexpr int V = 16 / static_cast<int>(sizeof(In));
  __shared__ uint32_t keys[kTileMost + 2], places[kTileMost];  // keys: with the neighbours of the tile
  const int64_t j = blockIdx.x / slices;
  constexpr int kStep = kAligned ? 1 : kSegmentThreads;  // between a thread's columns
  const int64_t c = static_cast<int64_t>(blockIdx.x - j * slices) * kSegmentThreads * V + (kAligned ? threadIdx.x * V : threadIdx.x);
  const int64_t i0 = j * tile;
  const int count = static_cast<int>(min(n - i0, static_cast<int64_t>(tile)));
  if (threadIdx.x < count + 2) {
    const int64_t i = i0 + threadIdx.x - 1;
    const uint2 pair = i >= 0 && i < n ? __ldg(sorted + i) : make_uint2(~0u, 0);  // beyond the ends: no token's key
    keys[threadIdx.x] = pair.x;
    if (threadIdx.x >= 1 && threadIdx.x <= count) places[threadIdx.x - 1] = pair.y;
  }
  __syncthreads();
  if (c >= grad.cols) return;
  const uint32_t limit = static_cast<uint32_t>(out.rows);
  uint32_t run = keys[1];
  bool head = keys[0] == run;
  float acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.0f;
  auto flush = [&](bool tail) {
    if (run >= limit) return;
    if (!head && !tail) {
      float r[V];
#pragma unroll
      for (int v = 0; v < V; ++v) r[v] = __fmul_rn(acc[v], scale);
      O* to = static_cast<O*>(out.data) + run * out.stride + c;
      if constexpr (kAligned) {
        store_pack<O, V>(to, round_pack<O, V>(r));
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (c + v * kStep < out.cols) to[v * kStep] = Values<O>::down(r[v]);
      }
    } else {
      float* to = partials.row(j, head ? 0 : 1) + c;
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (kAligned || c + v * kStep < out.cols) to[v * kStep] = acc[v];
    }
  };
  for (int i = 0; i < count; i += U) {
    Pack<In, V> g[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // a row again where the tile ends
      const In* from = static_cast<const In*>(grad.data) + places[min(i + u, count - 1)] * grad.stride + c;
      if constexpr (kAligned) {
        g[u] = load_pack<In, V>(from);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) g[u].v[v] = c + v * kStep < grad.cols ? from[v * kStep] : Values<In>::down(0.0f);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= count) break;
      const uint32_t k = keys[1 + i + u];
      if (k != run) {
        flush(false);
        head = false;
        run = k;
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
      }
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += Values<In>::up(g[u].v[v]);
    }
  }
  flush(keys[1 + count] == run);
}

// Tile j joins the run that starts in it and goes on into later tiles.  A short run: each of the CTA's
// warps takes 128 columns; a long one: the warps share its tiles, and their sums are added in warp order.
// A chain of dependent loads (keys, then partials): 9.0 us for 32,768 x 2,048.
template <typename O>
__global__ void __launch_bounds__(32 * kJoinWarps)
join_kernel(const uint2* __restrict__ sorted, int64_t n, int tile, float scale, Dense out,
            Partials partials) {
  __shared__ float4 sums[kJoinWarps][32];
  const int64_t j = blockIdx.x, i1 = (j + 1) * tile;
  if (i1 >= n) return;
  auto key = [&](int64_t i) { return __ldg(&sorted[i].x); };
  const uint32_t run = key(i1 - 1), after = key(i1), ahead = j > 0 ? key(j * tile - 1) : ~0u;
  if (run >= static_cast<uint32_t>(out.rows) || after != run || ahead == run) return;  // ahead: it started earlier
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // The last tile that the run reaches: 32 tiles' first keys at a time.
  int64_t last = j;
  for (;;) {
    const int64_t first = (last + 1 + lane) * tile;
    const uint32_t stop = __ballot_sync(0xffffffffu, first >= n || key(min(first, n - 1)) != run);
    last += stop ? __ffs(stop) - 1 : 32;
    if (stop) break;
  }
  const bool shared = last - j >= 128;  // (32,768 x 2,048 bf16, 7 in 10 tokens alike: 85 us, from 32 on 85, from 512 on 94)
  auto sum_of = [&](int64_t c, int64_t first, int step) {
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 16
    for (int64_t t = first; t <= last; t += step) {
      const float4 x = *reinterpret_cast<const float4*>(partials.row(t, t == j ? 1 : 0) + c);  // the pitch is a multiple of 8
      sum.x += x.x;
      sum.y += x.y;
      sum.z += x.z;
      sum.w += x.w;
    }
    return sum;
  };
  auto write = [&](int64_t c, const float4& sum) {
    const float r[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (c + v < out.cols)
        static_cast<O*>(out.data)[run * out.stride + c + v] = Values<O>::down(__fmul_rn(r[v], scale));
  };
  if (!shared) {
    for (int64_t c0 = (static_cast<int64_t>(blockIdx.y) * kJoinWarps + warp) * 128; c0 < out.cols; c0 += gridDim.y * kJoinWarps * 128) {
      const int64_t c = c0 + 4 * lane;
      if (c < out.cols) write(c, sum_of(c, j, 1));
    }
    return;
  }
  for (int64_t c0 = static_cast<int64_t>(blockIdx.y) * 128; c0 < out.cols; c0 += gridDim.y * 128) {
    const int64_t c = c0 + 4 * lane;
    sums[warp][lane] = c < out.cols ? sum_of(c, j + warp, kJoinWarps) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    __syncthreads();
    if (warp == 0 && c < out.cols) {
      float4 sum = sums[0][lane];
#pragma unroll
      for (int w = 1; w < kJoinWarps; ++w) {
        const float4 x = sums[w][lane];
        sum.x += x.x;
        sum.y += x.y;
        sum.z += x.z;
        sum.w += x.w;
      }
      write(c, sum);
    }
    __syncthreads();
  }
}

int64_t partial_pitch(int64_t cols) { return (cols + 7) / 8 * 8; }

// Long tiles leave fewer partials; short ones fill the GPU: up to eight CTAs on each of a B200's 148 SMs (the size of
// the workspace is asked for without a device).  32,768 x 2,048 bf16, 7 in 10 tokens alike: 85 us, with four CTAs an SM
// 87, sixteen 137, tiles of 32 at most 129; 65,536 x 1,024, all alike: 90, 84, 144 and 128.  At least 8 tokens:
// 1,999 x 1,024 f32 28.6 us, at least 4 or 16 29.3.
int64_t tile_of(int64_t n, int64_t slices) {
  return std::max<int64_t>(8, std::min<int64_t>(kTileMost, (n * slices + 148 * 8 - 1) / (148 * 8)));
}

// Whether the rows of both matrices are whole vectors of 16 bytes of `In`.
template <typename In, typename O>
bool vectors_fit(const Dense& in, const Dense& out) {
  constexpr int V = 16 / static_cast<int>(sizeof(In));
  return out.cols % V == 0 && rows_aligned(in, sizeof(In), 16) && rows_aligned(out, sizeof(O), V * sizeof(O));
}

template <typename In, typename O>
cudaError_t drive(const void* tokens, int token_bytes, int64_t n, const Dense& table, float scale,
                  const Dense& out, cudaStream_t stream) {
  constexpr int V = 16 / static_cast<int>(sizeof(In));
  const bool aligned = vectors_fit<In, O>(table, out);
  const int64_t vectors = (out.cols + V - 1) / V + (aligned ? 0 : 1);
  int x = 32;
  while (x < kDriveThreads && x < vectors) x *= 2;
  const dim3 block(x, kDriveThreads / x);
  const int64_t chunks = (vectors + x - 1) / x;
  const int64_t groups = (n + block.y - 1) / block.y;
  if (chunks * groups > 0x7fffffff) return cudaErrorInvalidConfiguration;
  auto* kernel = aligned ? drive_kernel<In, O, true> : drive_kernel<In, O, false>;
  kernel<<<static_cast<unsigned>(chunks * groups), block, 0, stream>>>(tokens, token_bytes, n, table, scale, out,
                                                                       static_cast<unsigned>(chunks));
  return cudaGetLastError();
}

template <typename In, typename O>
cudaError_t gradient(const void* tokens, int token_bytes, const Dense& grad, float scale,
                     const Dense& out, void* workspace, cudaStream_t stream) {
  constexpr int V = 16 / static_cast<int>(sizeof(In));
  DeviceInfo info;
  cudaError_t err = device_info(&info);
  if (err != cudaSuccess) return err;
  const int64_t n = grad.rows;
  const int64_t padded = (n + 3) / 4 * 4;
  auto* words = static_cast<uint32_t*>(workspace);
  const Sorted s{{reinterpret_cast<uint2*>(words), reinterpret_cast<uint2*>(words) + padded}};
  const Partials partials{reinterpret_cast<float*>(words + 4 * padded), partial_pitch(out.cols)};
  int passes = 1;
  while (passes < 4 && (out.rows >> (8 * passes)) > 0) ++passes;
  const int64_t fill = (out.rows * out.cols * static_cast<int64_t>(sizeof(O)) / 16 + kSortThreads - 1) / kSortThreads;
  const int shared = sort_span(n) <= 32 * kHeld ? static_cast<int>(sort_span(n)) * kSortWarps * 8 : 0;
  static SharedLimit limit;
  constexpr int kMost = 32 * kHeld * kSortWarps * 8;
  if ((err = limit.raise(sort_fill_kernel, kMost)) != cudaSuccess) return err;
  // As many clusters as run at once, 30 (32,000 x 1,024 f32: 30.5 us; with 34, of which some wait, 35.6).
  static ClusterLimit at_once;
  int most = 0;
  if ((err = at_once.most(sort_fill_kernel, kSortCtas, kSortThreads, kMost, &most)) != cudaSuccess) return err;
  const int64_t clusters = 1 + std::min<int64_t>((fill + kSortCtas - 1) / kSortCtas + 1, std::max(1, most - 1));
  sort_fill_kernel<<<static_cast<unsigned>(clusters * kSortCtas), kSortThreads, shared, stream>>>(
      tokens, token_bytes, n, s, n > 0 ? passes : 0, out, static_cast<int>(sizeof(O)));
  if ((err = cudaGetLastError()) != cudaSuccess || n == 0) return err;
  const uint2* sorted = s.pair[(passes - 1) & 1];
  const int64_t slices = (out.cols + V * kSegmentThreads - 1) / (V * kSegmentThreads);
  const int tile = static_cast<int>(tile_of(n, slices));
  const int64_t tiles = (n + tile - 1) / tile;
  if (tiles * slices > 0x7fffffff) return cudaErrorInvalidConfiguration;
  auto* kernel = vectors_fit<In, O>(grad, out) ? segment_kernel<In, O, true> : segment_kernel<In, O, false>;
  kernel<<<static_cast<unsigned>(tiles * slices), kSegmentThreads, 0, stream>>>(sorted, n, tile, grad, scale, out, partials,
                                                                                static_cast<int>(slices));
  if ((err = cudaGetLastError()) != cudaSuccess || tiles == 1) return err;
  // A CTA per 1,024 columns, and four at least: 32,768 x 2,048 bf16 58.6 us, 85 where 7 in 10 tokens are alike.  One per
  // 128 columns 67.9 and 72.6: more CTAs that find nothing to join; one per 1,024 throughout 57.7 and 111.
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(std::min<int64_t>(16, std::max((out.cols + 1023) / 1024, std::min<int64_t>(4, (out.cols + 255) / 256)))));
  join_kernel<O><<<grid, 32 * kJoinWarps, 0, stream>>>(sorted, n, tile, scale, out, partials);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_stimulus_drive(const void* tokens, int token_bytes, int64_t n, const Dense& table,
                                  float scale, const Dense& out, cudaStream_t stream) {
  return with_type(table.type, [&](auto in) {
    using In = decltype(in);
    auto call = [&](auto o) {
      using O = decltype(o);
      return drive<In, O>(tokens, token_bytes, n, table, scale, out, stream);
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
      return gradient<In, O>(tokens, token_bytes, grad, scale, out, workspace, stream);
    };
    if constexpr (sizeof(In) == 4) return with_type(out.type, call);  // a wide drive of a narrow table
    return out.type == NSB_VALUE_F32 ? call(float{}) : call(in);
  });
}

}  // namespace nsb
