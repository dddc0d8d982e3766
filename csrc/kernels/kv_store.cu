// Attention front with a quantizing paged store: per-head RMSNorm of q and k (optional), rotation,
// and K/V rows written as E4M3 codes with one FP32 scale a (row, head), or as BF16.
//
//   y = turn(norm(x)),  scale = max(amax |y|, 1e-10) / 448,  code = e4m3(y / scale)
//
// The rotation turns pairs (j, j + r/2) or (2j, 2j + 1) of the head's first r elements by
// position * inv_freq[j]; that product is formed and reduced by 2 pi in 64 bits, since at position
// 100,000 its FP32 form is off by up to 0.004 rad. Everything between the BF16 input and the stored
// value stays FP32: q rounds once to BF16, k and v once to their codes. A scale covers the finite
// elements of its row; an element that is not finite gets the NaN code, so it stays visible.
//
// Bound by HBM: a row's bytes are read once and written once (BF16 in; BF16 q, one byte a cached
// element and 4 bytes a scale out). d / 8 lanes hold a head, 8 elements (16 bytes) each.

#include <cuda_fp8.h>

#include "decode_ops.cuh"
#include "launch.cuh"
#include "sm100.cuh"

namespace foa {
namespace {

template <int kHD, bool kQuantized>
__global__ void __launch_bounds__(128) kv_store_kernel(const KvStore p, int groups) {
  constexpr int kLanes = kHD / 8;        // lanes of one head
  constexpr int kPerWarp = 32 / kLanes;  // heads of one warp pass
  __shared__ float2 turn[kHD / 2];       // (cos, sin) of the row's position
  const int row = blockIdx.x / groups, group = blockIdx.x % groups;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane / kLanes, hl = lane % kLanes;
  const int heads = p.q_heads + 2 * p.kv_heads;
  pdl_wait();
  pdl_trigger();
  const int half = p.rotary_dim / 2;
  const double pos = (double)p.positions[row];
  for (int j = threadIdx.x; j < half; j += blockDim.x) {
    const double a = pos * (double)p.inv_freq[j];
    const double r = fma(-rint(a * 0.15915494309189535), 6.283185307179586, a);
    float s, c;
    sincosf((float)r, &s, &c);
    turn[j] = make_float2(c * p.attention_factor, s * p.attention_factor);
  }
  __syncthreads();
  const int slot = p.slots[row];
  const bool past = slot >= 0 && slot >= p.cache_slots;
  if (past && group == 0 && threadIdx.x == 0) record_status(p.status, kBadIndex);
  const bool cached = slot >= 0 && !past;
  const int per_group = (heads + groups - 1) / groups;
  const int h_end = min(heads, (group + 1) * per_group);
  // The rotation partner of this lane's elements (half layout), and the pair index of its first.
  const int rl = p.rotary_dim / 8;  // lanes that turn
  const bool turns = hl < rl;
  const bool second = hl >= rl / 2;
  const int partner = !turns || p.interleaved ? lane : second ? lane - rl / 2 : lane + rl / 2;
  for (int h0 = group * per_group + warp * kPerWarp; h0 < h_end; h0 += 4 * kPerWarp) {
    const int head = h0 + sub;
    const bool valid = head < h_end;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (valid) raw = __ldcs(reinterpret_cast<const uint4*>(p.qkv + (long)row * p.ld_qkv + (long)head * kHD) + hl);
    const uint32_t rw[4] = {raw.x, raw.y, raw.z, raw.w};
    float x[8];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      x[2 * t] = bf16_lo(rw[t]);
      x[2 * t + 1] = bf16_hi(rw[t]);
    }
    const bool is_q = head < p.q_heads;
    const bool roped = head < p.q_heads + p.kv_heads;
    const __nv_bfloat16* nw = is_q ? p.q_norm : p.k_norm;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (roped && nw != nullptr) {
      const float inv = rsqrtf(ss / (float)kHD + p.eps);
      const uint4 wv = __ldg(reinterpret_cast<const uint4*>(nw) + hl);
      const uint32_t ww[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        x[2 * t] *= inv * bf16_lo(ww[t]);
        x[2 * t + 1] *= inv * bf16_hi(ww[t]);
      }
    }
    if (p.interleaved) {
      if (roped && turns) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const float2 cs = turn[hl * 4 + t];
          const float a = x[2 * t], b = x[2 * t + 1];
          x[2 * t] = a * cs.x - b * cs.y;
          x[2 * t + 1] = b * cs.x + a * cs.y;
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float other = __shfl_sync(0xffffffffu, x[e], partner);
        if (roped && turns) {
          const float2 cs = turn[(second ? hl - rl / 2 : hl) * 8 + e];
          x[e] = second ? x[e] * cs.x + other * cs.y : x[e] * cs.x - other * cs.y;
        }
      }
    }
    if (valid && is_q) {
      reinterpret_cast<uint4*>(p.q_out + ((long)row * p.q_heads + head) * kHD)[hl] =
          make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
    }
    const bool store = valid && !is_q && cached;
    const int kvh = head - p.q_heads - (roped ? 0 : p.kv_heads);
    const long place = (long)(slot >> 4) * 2 * p.kv_heads + (roped ? 0 : p.kv_heads) + kvh;  // page of (block, K or V, head)
    if constexpr (kQuantized) {
      // (A group's heads may mix q and cached ones in a warp: every lane takes part in the maximum.)
      float amax = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float m = fabsf(x[e]);
        if (m < INFINITY) amax = fmaxf(amax, m);
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      if (store) {
        const float scale = fmaxf(amax, 1e-10f) * (1.f / 448.f);
        uint16_t c[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          // The conversion saturates infinities: they become NaN first.
          float2 v = make_float2(__fdiv_rn(x[2 * t], scale), __fdiv_rn(x[2 * t + 1], scale));
          if (!(fabsf(v.x) < INFINITY)) v.x = __int_as_float(0x7fffffff);
          if (!(fabsf(v.y) < INFINITY)) v.y = __int_as_float(0x7fffffff);
          c[t] = __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
        }
        uint8_t* page = static_cast<uint8_t*>(p.cache) + place * (16 * kHD + kScaleBytes);
        reinterpret_cast<uint2*>(page + (slot & 15) * kHD)[hl] =
            make_uint2(c[0] | (uint32_t)c[1] << 16, c[2] | (uint32_t)c[3] << 16);
        if (hl == 0) reinterpret_cast<float*>(page + 16 * kHD)[slot & 15] = scale;
      }
    } else if (store) {
      __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.cache) + (place * 16 + (slot & 15)) * kHD;
      reinterpret_cast<uint4*>(dst)[hl] =
          make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
    }
  }
}

template <int kHD>
int launch(const KvStore& p, cudaStream_t stream) {
  const int heads = p.q_heads + 2 * p.kv_heads;
  const int pass = 4 * (256 / kHD);  // heads that a CTA handles at once
  int groups = (heads + pass - 1) / pass;
  if ((long)p.rows * groups > 148L * 16) groups = 1;
  const auto kernel = p.quantized ? kv_store_kernel<kHD, true> : kv_store_kernel<kHD, false>;
  if ((long)p.rows * groups > 2147483647L) return -2;
  return launch_pdl(kernel, dim3(p.rows * groups), dim3(128), 0, stream, p, groups) == cudaSuccess ? 0 : -5;
}

}  // namespace

int kv_store(const KvStore& p, cudaStream_t stream) {
  if (p.rows <= 0) return 0;
  if (p.q_heads < 0 || p.kv_heads <= 0 || p.ld_qkv % 8 != 0) return -2;
  if (p.rotary_dim < 16 || p.rotary_dim > p.head_dim || p.rotary_dim % 16 != 0) return -2;
  if ((reinterpret_cast<uintptr_t>(p.qkv) | reinterpret_cast<uintptr_t>(p.q_out) | reinterpret_cast<uintptr_t>(p.cache) |
       reinterpret_cast<uintptr_t>(p.q_norm) | reinterpret_cast<uintptr_t>(p.k_norm)) & 15)
    return -2;
  switch (p.head_dim) {
    case 64: return launch<64>(p, stream);
    case 128: return launch<128>(p, stream);
    default: return -2;
  }
}

}  // namespace foa
