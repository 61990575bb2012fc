// logits.cu -- penalties for repeated tokens, biases and masks on logits, and the greedy choice
// (the formula: nsb_adjust_logits in neurosim_b200.h).
//
// Bound by memory: each logit is read and written once, beside a mask bit and the histories.
// A cluster of 8 CTAs works on one row, each on its part of the vocabulary.  A CTA counts the
// history's tokens that fall into its part in shared memory (a 32-bit word per token: occurrences
// in the generated part, and bit 31 for "seen at all"), up to kPart tokens at a time, and applies
// the counts as it streams its logits: no table of rows x vocabulary counts exists anywhere.  The
// history is read by all 8 CTAs, from L2.  The largest value and its lowest index are joined over
// distributed shared memory.
//
// Vectors are cut at 16-byte boundaries of the row's logits, which for an odd vocabulary fall at
// another index in each row; the indexes of bias and mask follow.
#include <cooperative_groups.h>

#include <algorithm>

#include "nsb_tokens.h"

namespace cg = cooperative_groups;

namespace nsb {
namespace {

constexpr int kLogitsCtas = 8;
constexpr int kLogitsThreads = 512;
constexpr int kPart = 8192;  // tokens counted at a time: 32 KB
constexpr uint32_t kSeen = 0x80000000u;

struct Best {
  float value;
  int64_t index;
};

// The larger value; of equal ones the lower index.
__device__ __forceinline__ Best better(Best a, Best b) {
  return b.value > a.value || (b.value == a.value && b.index < a.index) ? b : a;
}

__device__ __forceinline__ Best warp_best(Best b) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    b = better(b, Best{__shfl_xor_sync(0xffffffffu, b.value, off), __shfl_xor_sync(0xffffffffu, b.index, off)});
  return b;
}

__device__ __forceinline__ float row_value(const nsb_row_values& r, int64_t b) {
  return r.data ? __ldg(r.data + b * r.stride) : r.scalar;
}

struct Penalties {
  float repetition, presence, frequency;
};

__device__ __forceinline__ float adjust(float x, uint32_t count, const Penalties& p) {
  if (count) {
    x = x > 0.0f ? __fdiv_rn(x, p.repetition) : __fmul_rn(x, p.repetition);
    const uint32_t c = count & ~kSeen;
    if (c) x = __fsub_rn(__fsub_rn(x, __fmul_rn(p.frequency, static_cast<float>(c))), p.presence);
  }
  return x;
}

template <typename T, bool kVec>
__global__ void __cluster_dims__(kLogitsCtas, 1, 1) __launch_bounds__(kLogitsThreads)
logits_kernel(LogitsArgs a) {
  constexpr int P = kVec ? 16 / static_cast<int>(sizeof(T)) : 1;
  __shared__ alignas(16) uint32_t counts[kPart];
  __shared__ Best best_of[kLogitsThreads / 32];
  __shared__ Best cta_best;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int64_t b = blockIdx.x / kLogitsCtas, vocabulary = a.logits.cols;
  const T* in = static_cast<const T*>(a.logits.data) + b * a.logits.stride;
  T* out = static_cast<T*>(a.out.data) + b * a.out.stride;
  const float* bias = a.bias ? a.bias + b * a.bias_stride : nullptr;
  const int32_t* mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
  const int32_t* history = a.history + b * a.history_stride;
  const int64_t length = a.history_length == 0 ? 0 : a.lengths ? max(int64_t{0}, min(a.history_length, static_cast<int64_t>(__ldg(a.lengths + b)))) : a.history_length;
  const int64_t prompt = a.prompt_lengths ? __ldg(a.prompt_lengths + b) : 0;
  const Penalties p{row_value(a.repetition, b), row_value(a.presence, b), row_value(a.frequency, b)};

  // Vector i of the row covers tokens [i * P - shift, + P): vectors start on 16-byte boundaries.
  const int64_t shift = kVec ? static_cast<int64_t>(reinterpret_cast<uintptr_t>(in) / sizeof(T) % P) : 0;
  const int64_t vectors = (vocabulary + shift + P - 1) / P;
  const int64_t share = (vectors + kLogitsCtas - 1) / kLogitsCtas;
  const int64_t last = min(vectors, (rank + 1) * share);
  Best best{-__int_as_float(0x7f800000), vocabulary};
  for (int64_t i0 = rank * share; i0 < last; i0 += kPart / P) {
    const int64_t i1 = min(last, i0 + kPart / P);
    const int64_t v0 = i0 * P - shift;  // the token of counts[0]; may be below 0
    if (length > 0) {
      for (int i = threadIdx.x; i < kPart; i += kLogitsThreads) counts[i] = 0;
      __syncthreads();
      const int64_t v_last = min(vocabulary, i1 * P - shift);
      for (int64_t h = threadIdx.x; h < length; h += kLogitsThreads) {
        const int64_t v = __ldg(history + h);
        if (v >= max(v0, int64_t{0}) && v < v_last) {
          if (h >= prompt)
            atomicAdd(counts + (v - v0), 1u);
          else
            atomicOr(counts + (v - v0), kSeen);
        }
      }
      __syncthreads();
    }
    for (int64_t i = i0 + threadIdx.x; i < i1; i += kLogitsThreads) {
      const int64_t v = i * P - shift;
      Pack<T, P> x;
      const bool whole = v >= 0 && v + P <= vocabulary;
      if (whole) {
        x = load_pack<T, P>(in + v);
      } else {
#pragma unroll
        for (int k = 0; k < P; ++k) x.v[k] = v + k >= 0 && v + k < vocabulary ? in[v + k] : Values<T>::down(0.0f);
      }
#pragma unroll
      for (int k = 0; k < P; ++k) {
        const int64_t t = v + k;
        if (!whole && (t < 0 || t >= vocabulary)) continue;
        float y = Values<T>::up(x.v[k]);
        if (length > 0) y = adjust(y, counts[t - v0], p);
        if (bias) y = __fadd_rn(y, __ldg(bias + t));
        if (mask && !((__ldg(mask + (t >> 5)) >> (t & 31)) & 1)) y = -__int_as_float(0x7f800000);
        x.v[k] = Values<T>::down(y);
        const float rounded = Values<T>::up(x.v[k]);
        if (rounded > best.value) best = Best{rounded, t};  // tokens ascend: the first of equals stays
      }
      if (whole) {
        store_pack<T, P>(out + v, x);
      } else {
#pragma unroll
        for (int k = 0; k < P; ++k)
          if (v + k >= 0 && v + k < vocabulary) out[v + k] = x.v[k];
      }
    }
    if (length > 0) __syncthreads();  // the counts are reused
  }
  if (!a.choice) return;
  best = warp_best(best);
  if ((threadIdx.x & 31) == 0) best_of[threadIdx.x >> 5] = best;
  __syncthreads();
  if (threadIdx.x < 32) {
    best = warp_best(best_of[threadIdx.x & (kLogitsThreads / 32 - 1)]);
    if (threadIdx.x == 0) cta_best = best;
  }
  cluster.sync();
  if (rank == 0 && threadIdx.x == 0) {
    for (int c = 1; c < kLogitsCtas; ++c) best = better(best, *cluster.map_shared_rank(&cta_best, c));
    a.choice[b] = best.index < vocabulary ? best.index : -1;
  }
  cluster.sync();  // no CTA leaves while its shared memory is read
}

}  // namespace

cudaError_t launch_adjust_logits(const LogitsArgs& a, cudaStream_t stream) {
  return with_type(a.logits.type, [&](auto zero) {
    using T = decltype(zero);
    if (a.logits.rows > 0x7fffffff / kLogitsCtas) return cudaErrorInvalidConfiguration;
    const auto grid = static_cast<unsigned>(a.logits.rows * kLogitsCtas);
    // Vectors need each row of the result at the same place within 16 bytes as the row of the logits.
    const bool vec = reinterpret_cast<uintptr_t>(a.logits.data) % 16 == reinterpret_cast<uintptr_t>(a.out.data) % 16 &&
                     (a.logits.rows == 1 || (a.logits.stride - a.out.stride) * static_cast<int64_t>(sizeof(T)) % 16 == 0);
    if (vec)
      logits_kernel<T, true><<<grid, kLogitsThreads, 0, stream>>>(a);
    else
      logits_kernel<T, false><<<grid, kLogitsThreads, 0, stream>>>(a);
    return cudaGetLastError();
  });
}

}  // namespace nsb
