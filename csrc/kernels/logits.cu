// Penalties for repeated tokens, biases and allowed-token masks on rows of logits, with each row's
// first maximum, in one pass over the logits.
//
// Of token t with logit x, n occurrences in the row's output list and the row's lists:
//   listed (prompt or output):  x = x > 0 ? x / repetition : x * repetition
//   n > 0:                      x = x - frequency * n, then x - presence
//   biased:                     x = x + bias (a token named twice: its last bias)
//   not allowed:                x = -inf
// in FP32, each step rounded as written (no contraction), so the result does not depend on the
// kernel's layout.
//
// A CTA takes 8192 tokens of a row, with a 32-bit word a token in shared memory: bit 31 "in the
// prompt", below it 1 + the place of the token's last bias, below that its count; where the call's
// lists are so long that the two might not fit, places get a second word. Every CTA reads the row's
// lists and counts the tokens of its slice: integer maxima, then adds, so their order does not matter.
// A second kernel takes the first of a row's maxima.
//
// Bound by HBM: every logit is read once (none where a mask leaves nothing and no output is
// written), mask words once, lists once a slice (from L2). What costs beside that is the way to the
// logits: the lists' bounds, then the lists, then a barrier. So a thread's vectors, all of its slice,
// are loaded before the table is built, and five or more CTAs share an SM, some building while others
// stream. Measured on 64 rows of 128256 FP32 logits with all features, and on 256 rows of 151936 BF16
// logits, in and out: 29 and 76 us. With a cluster of CTAs a row (no second kernel, a part of the
// lists each, added through distributed shared memory): 45 and 228 us for sixteen CTAs, of whose
// clusters the GPU holds 14, 35 and 112 us for eight without the remote adds.

#include <climits>

#include "decode_ops.cuh"
#include "launch.cuh"
#include "sm100.cuh"

namespace foa {
namespace {

constexpr int kSlice = 8192;   // tokens of a CTA
constexpr int kThreads = 256;
constexpr uint32_t kPrompt = 0x80000000u;

__device__ __forceinline__ void better(float& bv, int& bi, float v, int i) {
  if (v > bv || (v == bv && i < bi)) {
    bv = v;
    bi = i;
  }
}

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ void store(float* p, const float (&x)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[8]) {
    x[0] = bf16_lo(v.x), x[1] = bf16_hi(v.x), x[2] = bf16_lo(v.y), x[3] = bf16_hi(v.y);
    x[4] = bf16_lo(v.z), x[5] = bf16_hi(v.z), x[6] = bf16_lo(v.w), x[7] = bf16_hi(v.w);
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&x)[8]) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
};

// The penalties and the bias of a token; out of line, since few tokens have any.
__device__ __noinline__ float adjusted(float v, uint32_t word, const float* bias, float rep, float freq, float pres) {
  if (word != 0u) {
    v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
    const uint32_t n = word & ~kPrompt;
    if (n != 0u) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)n)), pres);
  }
  return bias != nullptr ? __fadd_rn(v, *bias) : v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4)
    process_logits_kernel(const LogitsArgs p, int slices, int count_bits) {
  extern __shared__ __align__(16) uint32_t table[];
  using V = Vec<T>;
  constexpr int kBatch = kSlice / (kThreads * V::kN);  // vectors of a thread
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.x / slices, part = blockIdx.x % slices;
  const int lo = part * kSlice, hi = min(p.vocab, lo + kSlice);
  const T* src = static_cast<const T*>(p.logits) + (long)row * p.ld;
  T* dst = p.out != nullptr ? static_cast<T*>(p.out) + (long)row * p.ldo : nullptr;
  const uint32_t* allowed = p.allowed != nullptr ? p.allowed + (long)row * p.ld_allowed : nullptr;

  // The lists' bounds, all of them on their way before the first is looked at.
  const bool penal = p.repetition != nullptr || p.frequency != nullptr || p.presence != nullptr;
  const TokenLists* lists[3] = {&p.prompt, &p.output, &p.bias};
  const bool used[3] = {p.repetition != nullptr && p.prompt.tokens != nullptr, penal && p.output.tokens != nullptr,
                        p.bias.tokens != nullptr};
  int begin[3], end[3];
#pragma unroll
  for (int l = 0; l < 3; ++l) {
    begin[l] = used[l] ? __ldg(lists[l]->starts + row) : 0;
    end[l] = used[l] ? __ldg(lists[l]->starts + row + 1) : 0;
  }
  const float rep = p.repetition != nullptr ? __ldg(p.repetition + row) : 1.f;
  const float freq = p.frequency != nullptr ? __ldg(p.frequency + row) : 0.f;
  const float pres = p.presence != nullptr ? __ldg(p.presence + row) : 0.f;

  // A slice begins at a multiple of 32 tokens, so every slice has the row's alignment: `head` tokens
  // before the first 16-byte boundary. Vectors are used where the output (if any) has the same one;
  // the table is shifted so that a vector's words are aligned too.
  const uintptr_t a = reinterpret_cast<uintptr_t>(src) & 15;
  const bool vec = a % sizeof(T) == 0 && (dst == nullptr || (reinterpret_cast<uintptr_t>(dst) & 15) == a);
  const int head = (int)(((16 - a) & 15) / sizeof(T));
  const int shift = (4 - head % 4) % 4;
  const int v0 = vec ? min(hi, lo + head) : hi;
  const int v1 = v0 + (hi - v0) / V::kN * V::kN;
  const int first = v0 + V::kN * threadIdx.x;  // vector i of this thread begins i * kThreads * kN further

  uint32_t bits[kBatch];
  uint4 raw[kBatch];
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    const int t = first + i * kThreads * V::kN;
    bits[i] = t < v1 ? (1u << V::kN) - 1 : 0u;
    if (allowed != nullptr && t < v1) {
      const int sh = t & 31;
      uint32_t w = __ldg(allowed + (t >> 5)) >> sh;
      if (sh + V::kN > 32) w |= __ldg(allowed + (t >> 5) + 1) << (32 - sh);
      bits[i] &= w;
    }
  }
#pragma unroll
  for (int i = 0; i < kBatch; ++i)
    if (bits[i] != 0u) raw[i] = *reinterpret_cast<const uint4*>(src + first + i * kThreads * V::kN);

#pragma unroll
  for (int l = 0; l < 3; ++l)
    if (begin[l] < 0 || end[l] < begin[l] || end[l] > lists[l]->count) {  // outside the tokens: an empty list
      record_status(p.status, kBadArgument);
      begin[l] = end[l] = 0;
    }
  const bool counted = end[0] > begin[0] || end[1] > begin[1];
  const bool biased = end[2] > begin[2];
  // Places of biases: in the words above the counts, or in words of their own (count_bits 0).
  uint32_t* counts = table;
  uint32_t* places = count_bits > 0 || !penal ? table : table + kSlice + 4;
  const bool words_read = counted || (biased && count_bits > 0);
  const bool apart = biased && count_bits == 0;
  if (counted || biased) {
    const int words = (kSlice + 4) * (apart && penal ? 2 : 1);
    for (int i = 4 * threadIdx.x; i < words; i += 4 * kThreads) *reinterpret_cast<uint4*>(table + i) = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    // The tokens of this CTA's slice (those outside the vocabulary are padding).
    auto scan = [&](int l, auto add) {
      const int32_t* tokens = lists[l]->tokens;
#pragma unroll 4
      for (int i = begin[l] + threadIdx.x; i < end[l]; i += kThreads) {
        const int t = __ldg(tokens + i);
        if (t >= lo && t < hi) add(t - lo + shift, i);
      }
    };
    scan(2, [&](int at, int i) { atomicMax(places + at, (uint32_t)(i - begin[2] + 1) << count_bits); });
    if (biased && count_bits > 0) __syncthreads();  // maxima first where counts share the words
    scan(0, [&](int at, int) { atomicOr(counts + at, kPrompt); });
    scan(1, [&](int at, int) { atomicAdd(counts + at, 1u); });
    __syncthreads();
  }
  const int to_word = shift - lo;  // token -> its word
  auto adjust = [&](float v, uint32_t w, uint32_t b) {
    if ((w | b) == 0u) return v;
    if (count_bits > 0) {
      b = (w & ~kPrompt) >> count_bits;
      w &= kPrompt | ((1u << count_bits) - 1);
    }
    return adjusted(v, w, b != 0u ? p.bias_values + begin[2] + (int)b - 1 : nullptr, rep, freq, pres);
  };
  float bv = -INFINITY;
  int bi = INT_MAX;
  auto single = [&](int t) {
    const bool ok = allowed == nullptr || (allowed[t >> 5] >> (t & 31) & 1u);
    const float v = ok ? adjust(V::one(src + t), words_read ? counts[t + to_word] : 0u, apart ? places[t + to_word] : 0u)
                       : -INFINITY;
    better(bv, bi, v, t);
    if (dst != nullptr) V::put(dst + t, v);
  };
  for (int t = lo + threadIdx.x; t < v0; t += kThreads) single(t);
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    const int t = first + i * kThreads * V::kN;
    if (t >= v1) continue;
    float x[V::kN];
    if (bits[i] != 0u) {
      V::unpack(raw[i], x);
      if (words_read || apart) {
        // The words of four tokens at a time; most are zero.
#pragma unroll
        for (int e = 0; e < V::kN; e += 4) {
          uint4 w = make_uint4(0u, 0u, 0u, 0u), b = w;
          if (words_read) w = *reinterpret_cast<const uint4*>(counts + t + e + to_word);
          if (apart) b = *reinterpret_cast<const uint4*>(places + t + e + to_word);
          if ((w.x | w.y | w.z | w.w | b.x | b.y | b.z | b.w) != 0u) {
            x[e] = adjust(x[e], w.x, b.x);
            x[e + 1] = adjust(x[e + 1], w.y, b.y);
            x[e + 2] = adjust(x[e + 2], w.z, b.z);
            x[e + 3] = adjust(x[e + 3], w.w, b.w);
          }
        }
      }
      float m = -INFINITY;
#pragma unroll
      for (int e = 0; e < V::kN; ++e) {
        if (!(bits[i] >> e & 1u)) x[e] = -INFINITY;
        m = fmaxf(m, x[e]);
      }
      if (m > bv || (m == bv && t < bi)) {
        bv = m;
#pragma unroll
        for (int e = V::kN - 1; e >= 0; --e)
          if (x[e] == m) bi = t + e;
      }
    } else {
#pragma unroll
      for (int e = 0; e < V::kN; ++e) x[e] = -INFINITY;
    }
    if (dst != nullptr) V::store(dst + t, x);
  }
  for (int t = v1 + threadIdx.x; t < hi; t += kThreads) single(t);

#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
    const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
    better(bv, bi, ov, oi);
  }
  __shared__ float sv[kThreads / 32];
  __shared__ int si[kThreads / 32];
  if ((threadIdx.x & 31) == 0) {
    sv[threadIdx.x >> 5] = bv;
    si[threadIdx.x >> 5] = bi;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) better(bv, bi, sv[w], si[w]);
    if (slices == 1) {
      p.index[row] = bv == -INFINITY ? -1 : bi;
      p.value[row] = bv;
    } else {
      p.partial[(long)row * slices + part] = make_float2(bv, __int_as_float(bi));
    }
  }
}

// The first maximum of a row's slices, a warp a row.
__global__ void __launch_bounds__(128) first_maximum_kernel(const LogitsArgs p, int slices) {
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  float bv = -INFINITY;
  int bi = INT_MAX;
  for (int s = threadIdx.x & 31; s < slices; s += 32) {
    const float2 x = p.partial[(long)row * slices + s];
    better(bv, bi, x.x, __float_as_int(x.y));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
    const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
    better(bv, bi, ov, oi);
  }
  if ((threadIdx.x & 31) == 0) {
    p.index[row] = bv == -INFINITY ? -1 : bi;
    p.value[row] = bv;
  }
}

template <typename T>
int launch(const LogitsArgs& p, cudaStream_t stream) {
  const bool penal = p.repetition != nullptr || p.frequency != nullptr || p.presence != nullptr;
  const bool biases = p.bias.tokens != nullptr;
  // One word a token where a count (at most the outputs' tokens) and a place (at most the biases')
  // fit into 31 bits.
  auto width = [](int n) {
    int b = 1;
    while ((1L << b) <= n) ++b;
    return b;
  };
  const int count_bits = biases && width(p.output.count) + width(p.bias.count + 1) <= 31 ? width(p.output.count) : 0;
  const int words = penal && biases && count_bits == 0 ? 2 : penal || biases ? 1 : 0;
  const int smem = 4 * words * (kSlice + 4);  // (with room for the shift)
  const int slices = logits_slices(p.vocab);
  if (slices > 1 && (p.partial == nullptr || p.partial_count < (size_t)p.rows * slices)) return -3;
  const auto kernel = process_logits_kernel<T>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * (kSlice + 4)) != cudaSuccess) return -5;
    configured[dev & 63] = true;
  }
  if (launch_pdl(kernel, dim3((unsigned)((long)p.rows * slices)), dim3(kThreads), smem, stream, p, slices, count_bits) != cudaSuccess)
    return -5;
  if (slices > 1 && launch_pdl(first_maximum_kernel, dim3((p.rows + 3) / 4), dim3(128), 0, stream, p, slices) != cudaSuccess)
    return -5;
  return 0;
}

}  // namespace

int logits_slices(int vocab) { return (vocab + kSlice - 1) / kSlice; }

int process_logits(const LogitsArgs& p, cudaStream_t stream) {
  if (p.rows <= 0) return 0;
  // Indexes run past the vocabulary and the lists by a CTA's stride: kept inside 32 bits.
  if (p.rows > (1 << 24) || p.vocab <= 0 || p.vocab > (1 << 30)) return -2;
  if ((long)p.rows * logits_slices(p.vocab) > 2147483647L) return -2;
  if (p.prompt.count > (1 << 30) || p.output.count > (1 << 30) || p.bias.count > (1 << 30)) return -2;
  return p.half ? launch<__nv_bfloat16>(p, stream) : launch<float>(p, stream);
}

}  // namespace foa
