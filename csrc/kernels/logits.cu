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
// Listed tokens, each once, are then valued by a thread each, so the pass over the vectors only skips
// them (their bit joins the mask) and stays free of branches. A second kernel takes the first of a
// row's maxima.
//
// Bound by HBM where lists are short: every logit is read once (none where a mask leaves nothing and
// no output is written), mask words once, lists once a slice (from L2). What costs beside that is the
// way to the logits: lists' bounds, tokens, their logits, three barriers. So a thread's vectors, all of
// its slice, are loaded before the table is built, the first tokens of all lists before any is looked
// at, the slice that follows on the SM is fetched to L2 meanwhile, and five CTAs share an SM (four of
// FP32), some building while others stream. 64 rows of 128256 FP32 logits with all features: 23.6 us
// (11 without lists); 256 rows of 151936 BF16 logits, in and out, with masks and lists: 54.5 us (35
// without lists, 28.6 without masks too, which is 5440 GB/s). Before the listed tokens had threads of
// their own: 28.5 and 75.8. Slices of 4096 tokens: 28.4 and 56.1; 512 threads: 26.4 and 68.3; six
// CTAs an SM, with spills: 53.6 of BF16. With a cluster of CTAs a row (a part of the lists each, added
// through distributed shared memory): 45 and 228 us for sixteen CTAs, of whose clusters the GPU holds
// 14, 35 and 112 us for eight without the remote adds.

#include <climits>
#include <type_traits>

#include "decode_ops.cuh"
#include "launch.cuh"
#include "sm100.cuh"

namespace foa {
namespace {

constexpr int kSlice = 8192;   // tokens of a CTA
constexpr int kTable = kSlice + 8;  // their words, with room for the shift
constexpr int kThreads = 256;
constexpr int kOrder = 2048;   // listed tokens of a slice that are kept as a list
constexpr uint32_t kPrompt = 0x80000000u;

__device__ __forceinline__ void better(float& bv, int& bi, float v, int i) {
  if (v > bv || (v == bv && i < bi)) {
    bv = v;
    bi = i;
  }
}

// Sixteen bytes of logits.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int kN = 4, kResident = 4;  // elements; CTAs an SM
  // Elements without their bit become -inf; the largest of the rest.
  static __device__ __forceinline__ void mask(uint4& v, uint32_t bits) {
    constexpr uint32_t kNone = 0xff800000u;
    v.x = bits & 1u ? v.x : kNone, v.y = bits & 2u ? v.y : kNone, v.z = bits & 4u ? v.z : kNone, v.w = bits & 8u ? v.w : kNone;
  }
  static __device__ __forceinline__ float largest(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static __device__ __forceinline__ int find(const uint4& v, float x) {
    return __uint_as_float(v.x) == x ? 0 : __uint_as_float(v.y) == x ? 1 : __uint_as_float(v.z) == x ? 2 : 3;
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8, kResident = 5;
  static __device__ __forceinline__ void mask(uint4& v, uint32_t bits) {
    // Byte selectors of a pair by its two bits: an element's own bytes, or those of -inf.
    constexpr uint64_t kPick = 0x3210'3254'7610'7654ull;
    auto pick = [&](uint32_t w, uint32_t two) { return __byte_perm(w, 0xff80ff80u, (uint32_t)(kPick >> (two & 0x30u))); };
    v.x = pick(v.x, bits << 4), v.y = pick(v.y, bits << 2), v.z = pick(v.z, bits), v.w = pick(v.w, bits >> 2);
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float largest(const uint4& v) {
    const uint32_t m = max2(max2(v.x, v.y), max2(v.z, v.w));
    return fmaxf(bf16_lo(m), bf16_hi(m));
  }
  static __device__ __forceinline__ int find(const uint4& v, float x) {
    return bf16_lo(v.x) == x ? 0 : bf16_hi(v.x) == x ? 1 : bf16_lo(v.y) == x ? 2 : bf16_hi(v.y) == x ? 3
         : bf16_lo(v.z) == x ? 4 : bf16_hi(v.z) == x ? 5 : bf16_lo(v.w) == x ? 6 : 7;
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
};

// The penalties and the bias of a token.
__device__ __forceinline__ float adjusted(float v, uint32_t word, const float* bias, float rep, float freq, float pres) {
  if (word != 0u) {
    v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
    const uint32_t n = word & ~kPrompt;
    if (n != 0u) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)n)), pres);
  }
  return bias != nullptr ? __fadd_rn(v, *bias) : v;
}

template <typename A>
constexpr int kCount = std::extent_v<std::remove_reference_t<A>>;

// The whole 16-byte units of a range, from HBM to L2.
__device__ __forceinline__ void prefetch_l2(const void* from, int bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(from), b = (a + 15) & ~15ull, e = (a + bytes) & ~15ull;
  if (e > b) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(b), "r"((uint32_t)(e - b)) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kThreads, Vec<T>::kResident)
    process_logits_kernel(const LogitsArgs p, int slices, int count_bits, int ahead) {
  extern __shared__ __align__(16) uint32_t table[];
  __shared__ uint32_t listed[kSlice / 32 + 1];  // a bit a token that some list names
  __shared__ uint16_t order[kOrder];             // those tokens, each once
  __shared__ int named;                          // how many there are
  using V = Vec<T>;
  constexpr int kBatch = kSlice / (kThreads * V::kN);  // vectors of a thread
  pdl_wait();
  pdl_trigger();
  // The slice that takes this one's place on the SM begins its way from HBM.
  if (threadIdx.x == 0 && gridDim.x - blockIdx.x > (unsigned)ahead) {
    const int row1 = (blockIdx.x + ahead) / slices, lo1 = (blockIdx.x + ahead) % slices * kSlice, n = min(kSlice, p.vocab - lo1);
    if (p.allowed != nullptr) prefetch_l2(p.allowed + (long)row1 * p.ld_allowed + lo1 / 32, n / 32 * 4);
    if (p.allowed == nullptr) prefetch_l2(static_cast<const T*>(p.logits) + (long)row1 * p.ld + lo1, n * (int)sizeof(T));
  }
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
  const int shift = (V::kN - head % V::kN) % V::kN;
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
    raw[i] = bits[i] == 0u ? make_uint4(0u, 0u, 0u, 0u) : *reinterpret_cast<const uint4*>(src + first + i * kThreads * V::kN);

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
  uint32_t* places = count_bits > 0 || !penal ? table : table + kTable;
  const bool apart = biased && count_bits == 0;
  const bool any = counted || biased;
  // Every listed token once: from the list, or all bits where the list is too short for them.
  auto each = [&](auto f) {
    const bool kept = named <= kOrder;
    const int n = kept ? named : kTable;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int at = kept ? order[i] : i;
      if (kept || (listed[at >> 5] >> (at & 31) & 1u)) f(at);
    }
  };
  if (any) {
    // The first tokens of every list are on their way before any is looked at.
    auto load = [&](int l, int from, auto& t) {
#pragma unroll
      for (int j = 0; j < kCount<decltype(t)>; ++j) {
        const int i = from + j * kThreads + threadIdx.x;
        t[j] = i < end[l] ? __ldg(lists[l]->tokens + i) : -1;
      }
    };
    int prompt[4], output[4], bias[1];
    load(2, begin[2], bias);
    load(0, begin[0], prompt);
    load(1, begin[1], output);
    const int words = kTable * (apart && penal ? 2 : 1);
    for (int i = 4 * threadIdx.x; i < words; i += 4 * kThreads) *reinterpret_cast<uint4*>(table + i) = make_uint4(0u, 0u, 0u, 0u);
    for (int i = threadIdx.x; i <= kSlice / 32; i += kThreads) listed[i] = 0u;
    if (threadIdx.x == 0) named = 0;
    __syncthreads();
    // The tokens of this CTA's slice (those outside the vocabulary are padding).
    auto scan = [&](int l, auto& t, auto add) {
      constexpr int kN = kCount<decltype(t)>;
      for (int from = begin[l]; from < end[l];) {
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          if (from + j * kThreads >= end[l]) break;
          if (t[j] >= lo && t[j] < hi) {
            const int at = t[j] - lo + shift;
            const uint32_t bit = 1u << (at & 31);
            add(at, from + j * kThreads + (int)threadIdx.x);
            if ((atomicOr(listed + (at >> 5), bit) & bit) == 0u) {
              const int n = atomicAdd(&named, 1);
              if (n < kOrder) order[n] = (uint16_t)at;
            }
          }
        }
        from += kN * kThreads;
        if (from < end[l]) load(l, from, t);
      }
    };
    scan(2, bias, [&](int at, int i) { atomicMax(places + at, (uint32_t)(i - begin[2] + 1) << count_bits); });
    if (biased && count_bits > 0) __syncthreads();  // maxima first where counts share the words
    scan(0, prompt, [&](int at, int) { atomicOr(counts + at, kPrompt); });
    scan(1, output, [&](int at, int) { atomicAdd(counts + at, 1u); });
    __syncthreads();
    // The values of the listed tokens, in their words' place; the vectors pass them over.
    each([&](int at) {
      uint32_t w = counted || count_bits > 0 ? counts[at] : 0u, b = apart ? places[at] : 0u;
      if (count_bits > 0) {
        b = (w & ~kPrompt) >> count_bits;
        w &= kPrompt | ((1u << count_bits) - 1);
      }
      const int t = at - shift + lo;
      const bool ok = allowed == nullptr || (__ldg(allowed + (t >> 5)) >> (t & 31) & 1u);
      const float v = adjusted(V::one(src + t), w, b != 0u ? p.bias_values + begin[2] + (int)b - 1 : nullptr, rep, freq, pres);
      table[at] = ok ? __float_as_uint(v) : 0xff800000u;
    });
    __syncthreads();
  }
  const int to_word = shift - lo;  // token -> its word
  float bv = -INFINITY;
  int bt = 0;  // the vector of this thread's first maximum
  uint4 best = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    const int t = first + i * kThreads * V::kN;
    if (t >= v1) continue;
    if (any) {
      const int at = t + to_word;  // (a multiple of kN)
      bits[i] &= ~(listed[at >> 5] >> (at & 31));
    }
    V::mask(raw[i], bits[i]);
    const float m = V::largest(raw[i]);
    if (m > bv) {
      bv = m;
      bt = t;
      best = raw[i];
    }
    if (dst != nullptr) *reinterpret_cast<uint4*>(dst + t) = raw[i];
  }
  int bi = bv > -INFINITY ? bt + V::find(best, bv) : INT_MAX;
  auto single = [&](int t) {
    const int at = t + to_word;
    if (any && (listed[at >> 5] >> (at & 31) & 1u)) return;
    const bool ok = allowed == nullptr || (allowed[t >> 5] >> (t & 31) & 1u);
    const float v = ok ? V::one(src + t) : -INFINITY;
    better(bv, bi, v, t);
    if (dst != nullptr) V::put(dst + t, v);
  };
  for (int t = lo + threadIdx.x; t < v0; t += kThreads) single(t);
  for (int t = v1 + threadIdx.x; t < hi; t += kThreads) single(t);
  if (any) {
    __syncthreads();  // after the vectors' stores
    each([&](int at) {
      const int t = at - to_word;
      const float v = __uint_as_float(table[at]);
      better(bv, bi, v, t);
      if (dst != nullptr) V::put(dst + t, v);
    });
  }
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
  const int smem = 4 * words * kTable;
  const int slices = logits_slices(p.vocab);
  if (slices > 1 && (p.partial == nullptr || p.partial_count < (size_t)p.rows * slices)) return -3;
  const auto kernel = process_logits_kernel<T>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * kTable) != cudaSuccess) return -5;
    configured[dev & 63] = true;
  }
  if (launch_pdl(kernel, dim3((unsigned)((long)p.rows * slices)), dim3(kThreads), smem, stream, p, slices, count_bits, 148 * Vec<T>::kResident) != cudaSuccess)
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
