// logits.cu -- penalties for repeated tokens, biases and masks on logits, and the greedy choice
// (the formula: nsb_adjust_logits in neurosim_b200.h).
//
// The stream is bound by memory: each logit is read and written once, beside a mask bit.  The histories are all
// latency.  256 x 131,071 bf16 with a shared bias and mask: 34 us (4.2 TB/s); with 4,096 tokens of history 60.
// A cluster of 1 to 8 CTAs works on one row, each on its part of the vocabulary, kPart tokens at a
// time.  Few of them occur in a history, so the streaming pass treats the others alone: a bit per
// token says which (8 KB of shared memory), and prefix sums of the bits' words number the set bits,
// which gives each such token a counter without a table over the vocabulary.  The history is read
// twice: once to set the bits, once to count.  A short history is read by every CTA of the cluster; of
// a long one each CTA reads a share, and works on the token's CTA over distributed shared memory.  The
// counted tokens are adjusted and written after the streaming pass, a thread to a token, with their
// logits read again from L2 (before the pass, at random from memory, that costs as much as the pass);
// where the result is written over the logits, the pass leaves them in shared memory as it meets them.
//
// While streaming, a thread keeps its largest value and the vector that has it; the place within the
// CTA's best vector is looked up at the end.
//
// Vectors are cut at 16-byte boundaries of the row's logits, which for an odd vocabulary fall at
// another index in each row; the bias, whose boundaries lie elsewhere, is cut out of aligned vectors,
// and the mask's bits are shifted into place.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "nsb_tokens.h"

namespace cg = cooperative_groups;

namespace nsb {
namespace {

constexpr int kMostCtas = 8;
constexpr int kPart = 65536 + 512;  // tokens of a CTA at a time: half of a 2^17 vocabulary, however its vectors fall
constexpr int kListed = 16384;    // ... and where the history is longer than this: so many may occur
// Tokens of a history that every CTA reads: one that may fill the counters is walked again for each part, and
// shared (16 rows x 262,143 f32: 16,000 tokens 35 us against 41 shared; 64 x 131,072 bf16: 20,000 tokens 130
// shared against 176).
constexpr int kShort = kListed;

struct Best {
  float value;
  int index;
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

// A logit whose token occurs, `count` times in the generated part.
__device__ __forceinline__ float penalised(float x, uint32_t count, const Penalties& p) {
  x = x > 0.0f ? __fdiv_rn(x, p.repetition) : __fmul_rn(x, p.repetition);
  return count ? __fsub_rn(__fsub_rn(x, __fmul_rn(p.frequency, static_cast<float>(count))), p.presence) : x;
}

__device__ __forceinline__ float minus_infinity() { return -__int_as_float(0x7f800000); }

// Shared memory of a CTA of the cluster.  A pointer that may be either a remote or the CTA's own would
// make every access a generic one, and the atomics several times slower: own words go by their names.
__device__ __forceinline__ uint32_t remote_address(const void* own, int rank) {
  uint32_t address;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(address) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(own))), "r"(rank));
  return address;
}
__device__ __forceinline__ uint32_t remote_load(uint32_t address) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(address) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t remote_load16(uint32_t address) {
  unsigned short v;
  asm volatile("ld.shared::cluster.u16 %0, [%1];" : "=h"(v) : "r"(address) : "memory");
  return v;
}
__device__ __forceinline__ void remote_or(uint32_t address, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(address), "r"(v) : "memory");
}
__device__ __forceinline__ void remote_add(uint32_t address, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(address), "r"(v) : "memory");
}

// The largest of the P values of a pack, a NaN passed over.
template <typename T, int P>
__device__ __forceinline__ float largest(const Pack<T, P>& r) {
  if constexpr (sizeof(T) == 2 && P == 8) {
    const auto* w = reinterpret_cast<const typename Values<T>::Two*>(&r);
    const auto m = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
    return fmaxf(Values<T>::up(m.x), Values<T>::up(m.y));
  } else {
    float most = minus_infinity();
#pragma unroll
    for (int k = 0; k < P; ++k) most = fmaxf(most, Values<T>::up(r.v[k]));
    return most;
  }
}

// Value k of a vector, k not known to the compiler: shifts instead of an index.
template <typename T, int P>
__device__ __forceinline__ T at_place(const Pack<T, P>& x, int k) {
  if constexpr (sizeof(T) == 4) {
    return k < 2 ? (k == 0 ? x.v[0] : x.v[1 % P]) : (k == 2 ? x.v[2 % P] : x.v[3 % P]);
  } else if constexpr (P == 8) {
    const auto* w = reinterpret_cast<const uint32_t*>(&x);
    const uint32_t word = k < 4 ? (k < 2 ? w[0] : w[1]) : (k < 6 ? w[2] : w[3]);
    const auto half = static_cast<uint16_t>(word >> (16 * (k & 1)));
    return *reinterpret_cast<const T*>(&half);
  } else {
    return x.v[0];
  }
}

// P consecutive floats that start `phase` after a 16-byte boundary: the aligned vectors around them, and
// their sum with y.
template <int P>
struct Floats {
  float all[P + 4];
  __device__ __forceinline__ void load(const float* p, int phase) {
    const float4* from = reinterpret_cast<const float4*>(p - phase);
#pragma unroll
    for (int q = 0; q < P / 4 + 1; ++q) {
      if (q == P / 4 && phase == 0) break;
      const float4 x = __ldg(from + q);
      all[4 * q] = x.x, all[4 * q + 1] = x.y, all[4 * q + 2] = x.z, all[4 * q + 3] = x.w;
    }
  }
  __device__ __forceinline__ void add_to(float (&y)[P], int phase) const {
    auto add = [&](auto skip) {
#pragma unroll
      for (int k = 0; k < P; ++k) y[k] = __fadd_rn(y[k], all[k + decltype(skip)::value]);
    };
    if (phase == 0) add(std::integral_constant<int, 0>{});
    else if (phase == 1) add(std::integral_constant<int, 1>{});
    else if (phase == 2) add(std::integral_constant<int, 2>{});
    else add(std::integral_constant<int, 3>{});
  }
};

template <typename T, bool kVec, bool kHistory, int threads>
__global__ void __launch_bounds__(threads, threads == 256 ? 4 : 1)
logits_kernel(LogitsArgs a, int ctas, int room) {
  constexpr int P = kVec ? 16 / static_cast<int>(sizeof(T)) : 1;
  constexpr int U = 2;       // vectors in flight per thread
  constexpr int kBatch = 4;  // tokens of the history in flight per thread
  constexpr int kOwn = (kPart + 32 * threads - 1) / (32 * threads) | 1;  // words of bits per thread; odd: no bank conflicts
  constexpr int kWords = kOwn * threads;
  const int part_vectors = (room < kListed ? kPart : kListed) / P;
  __shared__ uint32_t bits[kHistory ? kWords : 1];    // of the part's tokens: it occurs in the history
  __shared__ uint16_t before[kHistory ? kWords : 1];  // set bits in the words before: at most kListed
  extern __shared__ uint32_t counts[];                // per set bit
  // Which 16-bit values of a vector a byte of bits drops, as masks of them.
  constexpr bool kTable = kVec && sizeof(T) == 2;
  __shared__ uint4 masks[kTable ? 256 : 1];
  auto* listed = reinterpret_cast<uint16_t*>(counts + room);          // its token, less v0, the low 16 bits
  T* met = reinterpret_cast<T*>(listed + (room + 1) / 2 * 2);         // its logit, where the result is written over it
  __shared__ uint32_t scan[32];
  __shared__ Best best_of[32], stream_of[32];
  __shared__ Best cta_best;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = ctas > 1 ? static_cast<int>(cluster.block_rank()) : 0;
  const int64_t b = blockIdx.x / ctas;
  const int vocabulary = static_cast<int>(a.logits.cols);
  const T* in = static_cast<const T*>(a.logits.data) + b * a.logits.stride;
  T* out = static_cast<T*>(a.out.data) + b * a.out.stride;
  const bool in_place = a.logits.data == a.out.data;
  const float* bias = a.bias ? a.bias + b * a.bias_stride : nullptr;
  const int32_t* mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
  const int32_t* history = a.history + b * a.history_stride;
  uint32_t length = 0;
  if (kHistory) length = static_cast<uint32_t>(a.lengths ? max(int64_t{0}, min(a.history_length, static_cast<int64_t>(__ldg(a.lengths + b)))) : a.history_length);
  const uint32_t prompt = a.prompt_lengths ? max(0, __ldg(a.prompt_lengths + b)) : 0;
  if (kTable && threadIdx.x < 256) {
    auto word = [](uint32_t two) { return (two & 1 ? 0xffffu : 0u) | (two & 2 ? 0xffff0000u : 0u); };
    const uint32_t byte = threadIdx.x;
    masks[byte] = make_uint4(word(byte), word(byte >> 2), word(byte >> 4), word(byte >> 6));
  }
  if (kTable && !kHistory) __syncthreads();  // a history has barriers of its own
  const Penalties p{row_value(a.repetition, b), row_value(a.presence, b), row_value(a.frequency, b)};

  // Vector i of the row covers tokens [i * P - shift, + P): vectors start on 16-byte boundaries.
  const int shift = kVec ? static_cast<int>(reinterpret_cast<uintptr_t>(in) / sizeof(T) % P) : 0;
  const int vectors = static_cast<int>((static_cast<int64_t>(vocabulary) + shift + P - 1) / P);
  const int share = (vectors + ctas - 1) / ctas;
  const int own = (min(share, part_vectors) * P + 32 * threads - 1) / (32 * threads) | 1;  // words of bits per thread here
  const uint32_t share_inverse = 0xffffffffu / static_cast<uint32_t>(share);
  const bool together = ctas > 1 && length > kShort;  // the CTAs share the history
  auto sync = [&] { if (together) cluster.sync(); else __syncthreads(); };
  const int phase = bias ? static_cast<int>((reinterpret_cast<uintptr_t>(bias) / 4 - shift) & 3) : 0;  // of every vector's bias
  Best best{minus_infinity(), vocabulary};
  Best stream{minus_infinity(), vocabulary};  // among the whole vectors: the token where the vector starts

  auto finish = [&](T x, int t, float add, uint32_t allowed, auto penalty) {
    float y = penalty(Values<T>::up(x));
    if (bias) y = __fadd_rn(y, add);
    return Values<T>::down(allowed >> (t & 31) & 1 ? y : minus_infinity());
  };
  auto offer = [&](T r, int t) { best = better(best, Values<T>::up(r) > minus_infinity() ? Best{Values<T>::up(r), t} : best); };

  for (int part = 0; part * part_vectors < share; ++part) {
    const int i0 = rank * share + part * part_vectors;
    const int i1 = min(min(vectors, (rank + 1) * share), i0 + part_vectors);  // i1 <= i0: nothing left for this CTA
    const int v0 = i0 * P - shift;  // the token of bit 0; may be below 0
    // A batch of the history's tokens: where the bit of each lies, bit | owner << 20, or -1 for one that is
    // not in this part.
    // Places in the history are unsigned: a walk ends up to a batch beyond a length just below 2^31.
    const uint32_t step = together ? ctas * threads : threads, h_first = (together ? rank * threads : 0) + threadIdx.x;
    auto read = [&](uint32_t h0, int (&token)[kBatch]) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) token[j] = h0 + j * step < length ? __ldg(history + h0 + j * step) : -1;
    };
    auto locate = [&](const int (&token)[kBatch], int (&place)[kBatch]) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int t = token[j];
        place[j] = -1;
        if (t < 0 || t >= vocabulary) continue;
        const uint32_t i = static_cast<uint32_t>(t + shift) / P;
        uint32_t owner = __umulhi(i, share_inverse);  // i / share, or one less
        if (i - owner * share >= static_cast<uint32_t>(share)) ++owner;
        const int at = static_cast<int>(i - owner * share) - part * part_vectors;
        if ((together || owner == rank) && at >= 0 && at < part_vectors)
          place[j] = at * P + static_cast<int>(static_cast<uint32_t>(t + shift) % P) | static_cast<int>(owner << 20);
      }
    };
    // The vectors whose bias vectors lie in the row, [low, high); the tokens beside them go one by one.
    const int low = max(i0, (phase + shift + P - 1) / P), high = min(i1, vocabulary >= P + 4 ? (vocabulary - P - 4 + shift) / P + 1 : 0);
    uint32_t found = 0;
    if (kHistory) {
      for (int w = threadIdx.x; w < own * threads; w += threads) bits[w] = 0;
      sync();
      int place[kBatch], token[kBatch];
      read(h_first, token);
      for (uint32_t h0 = h_first; h0 < length; h0 += kBatch * step) {
        locate(token, place);
        read(h0 + kBatch * step, token);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          if (place[j] < 0) continue;
          const int w = (place[j] & 0xfffff) >> 5, owner = place[j] >> 20;
          const uint32_t bit = 1u << (place[j] & 31);
          if (together) {
            const uint32_t at = remote_address(bits + w, owner);
            if (!(remote_load(at) & bit)) remote_or(at, bit);
          } else if (!(bits[w] & bit)) {  // frequent tokens are there already
            atomicOr(bits + w, bit);
          }
        }
      }
      sync();
      // Exclusive prefix sums over the words: consecutive ones to a thread, then over the threads.
      uint32_t sum = 0;
      for (int i = 0; i < own; ++i) {
        const int w = threadIdx.x * own + i;
        before[w] = static_cast<uint16_t>(sum);
        sum += __popc(bits[w]);
      }
      uint32_t upto = sum;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= off) upto += x;
      }
      if (lane == 31) scan[warp] = upto;
      __syncthreads();
      const uint32_t one = lane < threads / 32 ? scan[lane] : 0;
      found = __reduce_add_sync(0xffffffffu, one);
      const uint32_t start = upto - sum + __reduce_add_sync(0xffffffffu, lane < warp ? one : 0);
      for (int i = 0; i < own; ++i) before[threadIdx.x * own + i] += static_cast<uint16_t>(start);
      __syncthreads();
      for (int w = threadIdx.x; w < own * threads; w += threads) {
        uint32_t n = before[w];
        for (uint32_t left = bits[w]; left; left &= left - 1, ++n) {
          counts[n] = 0;
          listed[n] = static_cast<uint16_t>(w * 32 + __ffs(left) - 1);
        }
      }
      sync();
      read(h_first, token);
      for (uint32_t h0 = h_first; h0 < length; h0 += kBatch * step) {
        locate(token, place);
        read(h0 + kBatch * step, token);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          if (place[j] < 0 || h0 + j * step < prompt) continue;
          const int w = (place[j] & 0xfffff) >> 5, owner = place[j] >> 20;
          const uint32_t lower = (1u << (place[j] & 31)) - 1u;
          if (together) {
            const uint32_t n = remote_load16(remote_address(before + w, owner)) + __popc(remote_load(remote_address(bits + w, owner)) & lower);
            remote_add(remote_address(counts + n, owner), 1u);
          } else {
            atomicAdd(counts + before[w] + __popc(bits[w] & lower), 1u);
          }
        }
      }
      sync();
    }
    auto single = [&](int t) {
      if (kHistory) {
        const uint32_t word = bits[(t - v0) >> 5], bit = 1u << ((t - v0) & 31);
        if (word & bit) {
          if (in_place) met[before[(t - v0) >> 5] + __popc(word & (bit - 1u))] = in[t];
          return;
        }
      }
      const T r = finish(in[t], t, bias ? __ldg(bias + t) : 0.0f, mask ? __ldg(mask + (t >> 5)) : ~0u, [](float x) { return x; });
      out[t] = r;
      offer(r, t);
    };
    if constexpr (!kVec) {
      for (int t = i0 + threadIdx.x; t < i1; t += threads) single(t);
    } else {
      for (int i = low + threadIdx.x; i < high; i += U * threads) {
        Pack<T, P> x[U];
        uint32_t allowed[U][2];
        Floats<P> add[2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int v = min(i + u * threads, high - 1) * P - shift;
          x[u] = load_pack<T, P>(in + v);
          allowed[u][0] = allowed[u][1] = ~0u;
          if (mask) {
            allowed[u][0] = __ldg(mask + (v >> 5));
            allowed[u][1] = __ldg(mask + ((v + P - 1) >> 5));
          }
          if (u == 0 && bias) add[0].load(bias + v, phase);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (u + 1 < U && bias) add[(u + 1) % 2].load(bias + min(i + (u + 1) * threads, high - 1) * P - shift, phase);
          const int at = i + u * threads, v = at * P - shift;
          if (at >= high) break;
          uint32_t drop = ~__funnelshift_r(allowed[u][0], allowed[u][1], v & 31);  // masked, or written later
          if (kHistory) {
            const int place = (at - i0) * P;
            const uint32_t word = bits[place >> 5];
            uint32_t left = word >> (place & 31) & ((1u << P) - 1u);
            drop |= left;
            if (in_place && left) {
              uint32_t n = before[place >> 5] + __popc(word & ((1u << (place & 31)) - 1u));
              for (; left; left &= left - 1, ++n) met[n] = at_place<T, P>(x[u], __ffs(left) - 1);
            }
          }
          float y[P];
#pragma unroll
          for (int k = 0; k < P; ++k) y[k] = Values<T>::up(x[u].v[k]);
          if (bias) add[u % 2].add_to(y, phase);
          if constexpr (!kTable) {
#pragma unroll
            for (int k = 0; k < P; ++k) y[k] = drop >> k & 1 ? minus_infinity() : y[k];
          }
          Pack<T, P> r = round_pack<T, P>(y);
          if constexpr (kTable) {
            constexpr uint32_t kInfinity = Values<T>::kType == NSB_VALUE_BF16 ? 0xff80ff80u : 0xfc00fc00u;  // minus, twice
            const uint4 m = masks[drop & 255];
            auto* w = reinterpret_cast<uint32_t*>(&r);
            w[0] = (w[0] & ~m.x) | (m.x & kInfinity);
            w[1] = (w[1] & ~m.y) | (m.y & kInfinity);
            w[2] = (w[2] & ~m.z) | (m.z & kInfinity);
            w[3] = (w[3] & ~m.w) | (m.w & kInfinity);
          }
          store_pack<T, P>(out + v, r);
          const float most = largest<T, P>(r);
          if (most > stream.value) stream = Best{most, v};  // vectors ascend: the first of equals stays
        }
      }
      for (int t = max(0, v0) + threadIdx.x; t < min(vocabulary, min(i1, max(low, i0)) * P - shift); t += threads) single(t);
      for (int t = max(0, max(low, max(high, i0)) * P - shift) + threadIdx.x; t < min(vocabulary, i1 * P - shift); t += threads) single(t);
    }
    if (kHistory) {
      __syncthreads();
      const uint32_t wrap = own * threads > 2048 ? before[2048] : found;  // the list is in order: from here on places are past 2^16
      for (uint32_t n0 = threadIdx.x; n0 < found; n0 += 4 * threads) {
        T x[4];
        float add[4];
        uint32_t allowed[4];
        int t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t n = min(n0 + j * threads, found - 1);
          t[j] = v0 + static_cast<int>(listed[n]) + (n < wrap ? 0 : 65536);
          x[j] = in_place ? met[n] : in[t[j]];
          add[j] = bias ? __ldg(bias + t[j]) : 0.0f;
          allowed[j] = mask ? __ldg(mask + (t[j] >> 5)) : ~0u;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t n = n0 + j * threads;
          if (n >= found) break;
          const T r = finish(x[j], t[j], add[j], allowed[j], [&](float y) { return penalised(y, counts[n], p); });
          out[t[j]] = r;
          offer(r, t[j]);
        }
      }
      sync();  // the bits may be set again
    }
  }
  if (!a.choice) return;
  best = warp_best(best);
  stream = warp_best(stream);
  if (lane == 0) {
    best_of[warp] = best;
    stream_of[warp] = stream;
  }
  __syncthreads();
  if (warp == 0) {
    best = warp_best(lane < threads / 32 ? best_of[lane] : Best{minus_infinity(), vocabulary});
    stream = warp_best(lane < threads / 32 ? stream_of[lane] : Best{minus_infinity(), vocabulary});
    if (stream.index < vocabulary && lane < P && Values<T>::up(out[stream.index + lane]) == stream.value)
      best = better(best, Best{stream.value, stream.index + lane});
    best = warp_best(best);
    if (lane == 0) cta_best = best;
  }
  if (ctas == 1) {
    if (threadIdx.x == 0) a.choice[b] = best.index < vocabulary ? best.index : -1;
    return;
  }
  cluster.sync();
  if (rank == 0 && threadIdx.x == 0) {
    for (int c = 1; c < ctas; ++c) best = better(best, *cluster.map_shared_rank(&cta_best, c));
    a.choice[b] = best.index < vocabulary ? best.index : -1;
  }
  cluster.sync();  // no CTA leaves while its shared memory is read
}

template <typename T, bool kVec, bool kHistory>
cudaError_t adjust_rows(const LogitsArgs& a, cudaStream_t stream) {
  DeviceInfo info;
  cudaError_t err = device_info(&info);
  if (err != cudaSuccess) return err;
  // Few CTAs to a row count its history less often; more fill the GPU: three or four of 256 threads per SM,
  // as long as they have 2,048 tokens each (256 x 131,071 bf16: 60 us with two to a row, 77 with one).
  // Where even eight to a row leave SMs idle, they get 1,024 threads (1 x 131,072 f32, 4,096 tokens of
  // history: 13.3 us against 16.0 with 256).
  unsigned ctas = 1, threads = 256;
  while (ctas < kMostCtas && a.logits.cols >= 4096 * int64_t{ctas} && a.logits.rows * ctas < info.sm_count * 3) ctas *= 2;
  if (a.logits.rows * ctas <= info.sm_count && a.logits.cols >= 4096 * int64_t{ctas}) threads = 1024;
  auto* kernel = threads == 256 ? logits_kernel<T, kVec, kHistory, 256> : logits_kernel<T, kVec, kHistory, 1024>;
  const int room = kHistory ? static_cast<int>(std::min<int64_t>(a.history_length, kListed)) : 0;
  // A counter and a place for each token that may occur, and its logit where the result is written over it
  // (less shared memory leaves more of it to L1, which the shifted vectors of the bias need).
  constexpr int kMost = kListed * (6 + static_cast<int>(sizeof(T)));
  const int shared = (room + 1) / 2 * 2 * (6 + (a.logits.data == a.out.data ? static_cast<int>(sizeof(T)) : 0));
  static SharedLimit limits[2];
  if (kHistory && (err = limits[threads == 256 ? 0 : 1].raise(kernel, kMost)) != cudaSuccess) return err;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(a.logits.rows * ctas));
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim = {ctas, 1, 1};
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, a, static_cast<int>(ctas), room);
}

}  // namespace

cudaError_t launch_adjust_logits(const LogitsArgs& a, cudaStream_t stream) {
  return with_type(a.logits.type, [&](auto zero) {
    using T = decltype(zero);
    if (a.logits.rows > 0x7fffffff / kMostCtas) return cudaErrorInvalidConfiguration;
    // Vectors need each row of the result at the same place within 16 bytes as the row of the logits (256 x 131,072
    // bf16 with bias and mask: 31 us, token by token 158; 64 x 50,000 f32 8.8 and 11.5).
    const bool vec = reinterpret_cast<uintptr_t>(a.logits.data) % 16 == reinterpret_cast<uintptr_t>(a.out.data) % 16 &&
                     (a.logits.rows == 1 || (a.logits.stride - a.out.stride) * static_cast<int64_t>(sizeof(T)) % 16 == 0);
    const bool history = a.history_length > 0;
    if (vec) return history ? adjust_rows<T, true, true>(a, stream) : adjust_rows<T, true, false>(a, stream);
    return history ? adjust_rows<T, false, true>(a, stream) : adjust_rows<T, false, false>(a, stream);
  });
}

}  // namespace nsb
