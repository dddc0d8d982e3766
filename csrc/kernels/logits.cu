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
// A cluster of CTAs shares a row; each owns a slice of the vocabulary with a 32-bit word a token in
// shared memory: bit 31 "in the prompt", the rest its count (a second word where biases are given:
// 1 + the place of the token's last bias). The CTAs read the row's token lists once, each its part,
// and add to the owner's words through distributed shared memory; integer adds and maxima, so their
// order does not matter. A slice that does not fit is handled in several passes over the lists.
// Bound by HBM: every logit is read once (none where a mask leaves nothing and no output is
// written), lists and mask words once.

#include <cooperative_groups.h>

#include <climits>

#include "decode_ops.cuh"
#include "launch.cuh"
#include "sm100.cuh"

namespace foa {
namespace {

constexpr int kCtas = 8;       // CTAs of a row's cluster
constexpr int kThreads = 512;
constexpr uint32_t kPrompt = 0x80000000u;

__device__ __forceinline__ void better(float& bv, int& bi, float v, int i) {
  if (v > bv || (v == bv && i < bi)) {
    bv = v;
    bi = i;
  }
}

struct Range {
  int begin, end;
};

__device__ __forceinline__ Range list_of(const TokenLists& l, int row, int* status) {
  Range r{0, 0};
  if (l.tokens == nullptr) return r;
  r.begin = l.starts[row];
  r.end = l.starts[row + 1];
  if (r.begin < 0 || r.end < r.begin || r.end > l.count) {  // lists outside the tokens read as empty
    record_status(status, kBadArgument);
    r.begin = r.end = 0;
  }
  return r;
}

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void load(const float* p, float (&x)[4]) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
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
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
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

template <typename T>
__global__ void __launch_bounds__(kThreads) process_logits_kernel(const LogitsArgs p, int slice, int passes) {
  namespace cg = cooperative_groups;
  extern __shared__ uint32_t tables[];
  using V = Vec<T>;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int row = blockIdx.x / kCtas;
  pdl_wait();
  pdl_trigger();
  const bool penal = p.repetition != nullptr || p.frequency != nullptr || p.presence != nullptr;
  Range prompt{0, 0}, output{0, 0}, bias{0, 0};
  if (penal) {
    if (p.repetition != nullptr) prompt = list_of(p.prompt, row, p.status);
    output = list_of(p.output, row, p.status);
  }
  bias = list_of(p.bias, row, p.status);
  const bool counted = prompt.end > prompt.begin || output.end > output.begin;
  const bool biased = bias.end > bias.begin;
  uint32_t* count_s = tables;
  uint32_t* bias_s = tables + (penal ? slice : 0);
  const float rep = p.repetition != nullptr ? p.repetition[row] : 1.f;
  const float freq = p.frequency != nullptr ? p.frequency[row] : 0.f;
  const float pres = p.presence != nullptr ? p.presence[row] : 0.f;
  const T* src = static_cast<const T*>(p.logits) + (long)row * p.ld;
  T* dst = p.out != nullptr ? static_cast<T*>(p.out) + (long)row * p.ldo : nullptr;
  const uint32_t* allowed = p.allowed != nullptr ? p.allowed + (long)row * p.ld_allowed : nullptr;
  float bv = -INFINITY;
  int bi = INT_MAX;

  for (int pass = 0; pass < passes; ++pass) {
    const int base = pass * kCtas * slice;  // first token of the pass
    const int lo = min(p.vocab, base + rank * slice), hi = min(p.vocab, lo + slice);
    if (counted || biased) {
      if (counted)
        for (int i = threadIdx.x; i < slice; i += kThreads) count_s[i] = 0u;
      if (biased)
        for (int i = threadIdx.x; i < slice; i += kThreads) bias_s[i] = 0u;
      cluster.sync();
      // This CTA's part of the lists; tokens outside the vocabulary (padding) are left out.
      auto scan = [&](const int32_t* tokens, Range r, auto add) {
        for (int i = r.begin + rank * kThreads + threadIdx.x; i < r.end; i += kCtas * kThreads) {
          const int t = tokens[i];
          if (t < 0 || t >= p.vocab) continue;
          const int at = t - base;
          if (at < 0 || at >= kCtas * slice) continue;
          add(at / slice, at % slice, i);
        }
      };
      scan(p.prompt.tokens, prompt, [&](int owner, int at, int) { atomicOr(cluster.map_shared_rank(count_s + at, owner), kPrompt); });
      scan(p.output.tokens, output, [&](int owner, int at, int) { atomicAdd(cluster.map_shared_rank(count_s + at, owner), 1u); });
      scan(p.bias.tokens, bias, [&](int owner, int at, int i) {
        atomicMax(cluster.map_shared_rank(bias_s + at, owner), (uint32_t)(i - bias.begin + 1));
      });
      cluster.sync();
    }
    auto adjust = [&](float x, int t, bool ok) {
      if (counted) {
        const uint32_t w = count_s[t - lo];
        if (w != 0u) {
          x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
          const uint32_t n = w & ~kPrompt;
          if (n != 0u) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, (float)n)), pres);
        }
      }
      if (biased) {
        const uint32_t b = bias_s[t - lo];
        if (b != 0u) x = __fadd_rn(x, p.bias_values[bias.begin + (int)b - 1]);
      }
      return ok ? x : -INFINITY;
    };
    auto single = [&](int t) {
      const bool ok = allowed == nullptr || (allowed[t >> 5] >> (t & 31) & 1u);
      const float x = adjust(V::one(src + t), t, ok);
      better(bv, bi, x, t);
      if (dst != nullptr) V::put(dst + t, x);
    };
    // 16-byte accesses between the slice's first and last aligned places, where the output (if any)
    // has the same alignment.
    const uintptr_t a = reinterpret_cast<uintptr_t>(src + lo) & 15;
    const bool vec = a % sizeof(T) == 0 && (dst == nullptr || (reinterpret_cast<uintptr_t>(dst + lo) & 15) == a);
    const int v0 = vec ? min(hi, lo + (int)(((16 - a) & 15) / sizeof(T))) : hi;
    const int v1 = v0 + (hi - v0) / V::kN * V::kN;
    for (int t = lo + threadIdx.x; t < v0; t += kThreads) single(t);
    for (int t = v1 + threadIdx.x; t < hi; t += kThreads) single(t);
    for (int t = v0 + V::kN * threadIdx.x; t < v1; t += V::kN * kThreads) {
      uint32_t bits = ~0u;
      if (allowed != nullptr) {
        const int sh = t & 31;
        bits = allowed[t >> 5] >> sh;
        if (sh + V::kN > 32) bits |= allowed[(t >> 5) + 1] << (32 - sh);
        bits &= (1u << V::kN) - 1;
      }
      float x[V::kN];
      if (bits == 0u) {
        if (dst == nullptr) continue;
#pragma unroll
        for (int e = 0; e < V::kN; ++e) x[e] = -INFINITY;
      } else {
        V::load(src + t, x);
#pragma unroll
        for (int e = 0; e < V::kN; ++e) {
          x[e] = adjust(x[e], t + e, bits >> e & 1u);
          better(bv, bi, x[e], t + e);
        }
      }
      if (dst != nullptr) V::store(dst + t, x);
    }
    __syncthreads();  // the tables are read before the next pass clears them
  }

#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
    const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
    better(bv, bi, ov, oi);
  }
  __shared__ float sv[kThreads / 32];
  __shared__ int si[kThreads / 32];
  __shared__ float cta_v;
  __shared__ int cta_i;
  if ((threadIdx.x & 31) == 0) {
    sv[threadIdx.x >> 5] = bv;
    si[threadIdx.x >> 5] = bi;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) better(bv, bi, sv[w], si[w]);
    cta_v = bv;
    cta_i = bi;
  }
  cluster.sync();  // every CTA's pair is in its shared memory
  if (rank == 0 && threadIdx.x == 0) {
    for (int c = 1; c < kCtas; ++c) better(bv, bi, *cluster.map_shared_rank(&cta_v, c), *cluster.map_shared_rank(&cta_i, c));
    p.index[row] = bv == -INFINITY ? -1 : bi;
    p.value[row] = bv;
  }
  cluster.sync();  // no CTA leaves while CTA 0 still reads its shared memory
}

constexpr int kTableBytes = 200 * 1024;  // shared memory that the tables may take

template <typename T>
int launch(const LogitsArgs& p, cudaStream_t stream) {
  const bool penal = p.repetition != nullptr || p.frequency != nullptr || p.presence != nullptr;
  const int words = (penal ? 1 : 0) + (p.bias.tokens != nullptr ? 1 : 0);
  // Slices of a multiple of 32 tokens, so that a mask word belongs to one CTA.
  int slice = ((p.vocab + kCtas - 1) / kCtas + 31) / 32 * 32;
  if (words > 0) slice = min(slice, kTableBytes / (4 * words) / 32 * 32);
  const int passes = (int)(((long)p.vocab + (long)kCtas * slice - 1) / ((long)kCtas * slice));
  const int smem = 4 * words * slice;
  const auto kernel = process_logits_kernel<T>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTableBytes) != cudaSuccess) return -5;
  return launch_pdl_cluster(kernel, dim3(kCtas * p.rows), dim3(kThreads), kCtas, smem, stream, p, slice, passes) == cudaSuccess
             ? 0
             : -5;
}

}  // namespace

int process_logits(const LogitsArgs& p, cudaStream_t stream) {
  if (p.rows <= 0) return 0;
  // Indexes run past the vocabulary and the lists by a cluster's stride: kept inside 32 bits.
  if (p.rows > (1 << 24) || p.vocab <= 0 || p.vocab > (1 << 30)) return -2;
  if (p.prompt.count > (1 << 30) || p.output.count > (1 << 30) || p.bias.count > (1 << 30)) return -2;
  return p.half ? launch<__nv_bfloat16>(p, stream) : launch<float>(p, stream);
}

}  // namespace foa
