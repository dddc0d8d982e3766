// Attention front with a quantizing paged store: per-head RMSNorm of q and k (optional), rotation,
// and K/V rows written as E4M3 codes with one FP32 scale a (row, head), or as BF16.
//
//   y = turn(norm(x)),  scale = max(amax |y|, 1e-10) / 448,  code = e4m3(y * (1 / scale))
//
// The rotation turns pairs (j, j + r/2) or (2j, 2j + 1) of the head's first r elements by
// position * inv_freq[j]; that product is formed and reduced by 2 pi in 64 bits, since at position
// 100,000 its FP32 form is off by up to 0.004 rad. Everything between the BF16 input and the stored
// value stays FP32: q rounds once to BF16, k and v once to their codes. A scale covers the finite
// elements of its row; an element that is not finite gets the NaN code, so it stays visible.
//
// Bound by HBM (a row's bytes are read once and written once: BF16 in; BF16 q, one byte a cached
// element and 4 bytes a scale out). d / 16 lanes hold a head, 16 elements each: eight first elements of
// rotated pairs and their eight partners, so the rotation needs no exchange between lanes, takes the
// same (cos, sin) for every head of the row, and runs on pairs of FP32 operations. A warp takes a row by
// itself (a part of one when rows are few): nothing waits for another warp, three passes' loads are in
// flight at any time, and the first are under way while the angles are formed. 8192 rows of 32 + 2 x 8
// heads of 128, normed: 37.5 us (4930 GB/s). A CTA a row, its warps joined by a barrier after the
// angles: 47.6 us, and 71 with partners that came by eight shuffles.

#include <cuda_fp8.h>

#include "decode_ops.cuh"
#include "launch.cuh"
#include "sm100.cuh"

namespace foa {
namespace {

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 w, {%6, %7};\n"
      " fma.rn.f32x2 z, x, y, w;\n mov.b64 {%0, %1}, z;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// A lane's sixteen elements as pairs' first elements a (four float2) and their partners b: of the half
// layout the two 16-byte words, of the interleaved one the low and high halves of every 32 bits.
template <bool kInterleaved>
__device__ __forceinline__ void unpack(const uint4& r0, const uint4& r1, float2 (&a)[4], float2 (&b)[4]) {
  const uint32_t w[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if constexpr (kInterleaved) {
      a[t] = make_float2(bf16_lo(w[2 * t]), bf16_lo(w[2 * t + 1]));
      b[t] = make_float2(bf16_hi(w[2 * t]), bf16_hi(w[2 * t + 1]));
    } else {
      a[t] = make_float2(bf16_lo(w[t]), bf16_hi(w[t]));
      b[t] = make_float2(bf16_lo(w[t + 4]), bf16_hi(w[t + 4]));
    }
  }
}
// Pair t of eight in the order of memory (pairs 0 .. 3 from e0, 4 .. 7 from e1).
template <bool kInterleaved>
__device__ __forceinline__ float2 in_order(const float2 (&a)[4], const float2 (&b)[4], int t) {
  if constexpr (kInterleaved) return t & 1 ? make_float2(a[t >> 1].y, b[t >> 1].y) : make_float2(a[t >> 1].x, b[t >> 1].x);
  return t < 4 ? a[t & 3] : b[t & 3];
}
template <bool kInterleaved>
__device__ __forceinline__ uint4 bf16_words(const float2 (&a)[4], const float2 (&b)[4], int from) {
  uint32_t w[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const float2 x = in_order<kInterleaved>(a, b, from + t);
    w[t] = pack_bf16x2(x.x, x.y);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int kHD, bool kQuantized, bool kInterleaved>
__global__ void __launch_bounds__(128) kv_store_kernel(const KvStore p, int groups) {
  constexpr int kLanes = kHD / 16;       // lanes of one head
  constexpr int kPerWarp = 32 / kLanes;  // heads of one warp pass
  constexpr int kAhead = 3;              // passes whose loads are in flight together
  __shared__ __align__(16) float turns_s[4][2][kHD / 2];  // a warp's row: cos, sin of its position
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long task = (long)blockIdx.x * 4 + warp;  // a part of a row's heads
  const int row = (int)(task / groups), group = (int)(task % groups);
  if (row >= p.rows) return;
  float(&turn)[2][kHD / 2] = turns_s[warp];
  const int sub = lane / kLanes, hl = lane % kLanes;
  const int heads = p.q_heads + 2 * p.kv_heads;
  const int per_group = (heads + groups - 1) / groups;
  const int h_begin = group * per_group, h_end = min(heads, h_begin + per_group);
  // This lane's elements: e0 .. e0 + 7 and e1 .. e1 + 7. Of the half layout's r / 16 turning lanes the
  // second eight are the partners of the first; otherwise the sixteen lie together.
  const bool turns = hl < p.rotary_dim / 16;
  const bool apart = turns && !kInterleaved;
  const int e0 = apart ? 8 * hl : 16 * hl, e1 = apart ? p.rotary_dim / 2 + 8 * hl : 16 * hl + 8;
  const __nv_bfloat16* src = p.qkv + (long)row * p.ld_qkv;
  uint4 raw[kAhead][2];
  auto load = [&](int i, int first) {
    const int head = first + sub;
    raw[i][0] = raw[i][1] = make_uint4(0u, 0u, 0u, 0u);
    if (head < h_end) {
      raw[i][0] = __ldcs(reinterpret_cast<const uint4*>(src + head * kHD + e0));
      raw[i][1] = __ldcs(reinterpret_cast<const uint4*>(src + head * kHD + e1));
    }
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(i, h_begin + i * kPerWarp);
  const int slot = p.slots[row];
  const double pos = (double)p.positions[row];
  for (int j = lane; j < p.rotary_dim / 2; j += 32) {
    // The angle in turns, of which only the fraction counts; as half turns in [-1, 1].
    const double turns64 = pos * ((double)p.inv_freq[j] * 0.15915494309189535);
    float s, c;
    sincospif(2.f * (float)(turns64 - rint(turns64)), &s, &c);
    turn[0][j] = c * p.attention_factor;
    turn[1][j] = s * p.attention_factor;
  }
  const bool past = slot >= 0 && slot >= p.cache_slots;
  if (past && group == 0 && lane == 0) record_status(p.status, kBadIndex);
  const bool cached = slot >= 0 && !past;
  __syncwarp();
  // cos and sin of this lane's pairs, in either layout pairs 8 hl .. 8 hl + 7.
  float2 co[4], si[4];
  if (turns) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      co[t] = *reinterpret_cast<const float2*>(turn[0] + 8 * hl + 2 * t);
      si[t] = *reinterpret_cast<const float2*>(turn[1] + 8 * hl + 2 * t);
    }
  }
  __nv_bfloat16* q_row = p.q_out + (long)row * p.q_heads * kHD;
  const long block = (long)(slot >> 4) * 2 * p.kv_heads;
  for (int h0 = h_begin; h0 < h_end; h0 += kAhead * kPerWarp) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int first = h0 + i * kPerWarp;  // the warp's first head of this pass
      if (first >= h_end) break;
      const int head = first + sub;
      const bool valid = head < h_end;
      const bool is_q = head < p.q_heads;
      const bool roped = head < p.q_heads + p.kv_heads;
      float2 a[4], b[4];
      unpack<kInterleaved>(raw[i][0], raw[i][1], a, b);
      load(i, first + kAhead * kPerWarp);
      if (p.q_norm != nullptr && first < p.q_heads + p.kv_heads) {
        float2 s2 = mul2(a[0], a[0]);
#pragma unroll
        for (int t = 1; t < 4; ++t) s2 = fma2(a[t], a[t], s2);
#pragma unroll
        for (int t = 0; t < 4; ++t) s2 = fma2(b[t], b[t], s2);
        float ss = s2.x + s2.y;
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (roped) {
          const float inv = rsqrtf(ss * (1.f / (float)kHD) + p.eps);
          const __nv_bfloat16* nw = is_q ? p.q_norm : p.k_norm;
          float2 wa[4], wb[4];
          unpack<kInterleaved>(__ldg(reinterpret_cast<const uint4*>(nw + e0)), __ldg(reinterpret_cast<const uint4*>(nw + e1)), wa, wb);
          const float2 inv2 = make_float2(inv, inv);
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            a[t] = mul2(mul2(a[t], wa[t]), inv2);
            b[t] = mul2(mul2(b[t], wb[t]), inv2);
          }
        }
      }
      if (roped && turns) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const float2 u = fma2(b[t], make_float2(-si[t].x, -si[t].y), mul2(a[t], co[t]));
          b[t] = fma2(a[t], si[t], mul2(b[t], co[t]));
          a[t] = u;
        }
      }
      if (is_q && valid) {
        __nv_bfloat16* dst = q_row + head * kHD;
        *reinterpret_cast<uint4*>(dst + e0) = bf16_words<kInterleaved>(a, b, 0);
        *reinterpret_cast<uint4*>(dst + e1) = bf16_words<kInterleaved>(a, b, 4);
      }
      if (first + kPerWarp <= p.q_heads || !cached) continue;  // (all of the warp's heads, or all of the row's)
      const bool store = valid && !is_q;
      const long place = block + head - p.q_heads;  // page of (block, K or V, head): V's heads follow K's
      if constexpr (kQuantized) {
        // (A warp's heads may mix q and cached ones: every lane takes part in the maximum.)
        float amax = 0.f;
        float2 odd = make_float2(0.f, 0.f);
        const float2 none = odd;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          amax = fmaxf(amax, fmaxf(fabsf(a[t].x), fabsf(a[t].y)));
          amax = fmaxf(amax, fmaxf(fabsf(b[t].x), fabsf(b[t].y)));
          odd = fma2(b[t], none, fma2(a[t], none, odd));  // NaN once an element is not finite
        }
        if (odd.x + odd.y != 0.f) {  // (rare) the scale is of the finite elements, the others get the NaN code
          amax = 0.f;
          auto look = [&](float& x) {
            if (fabsf(x) < INFINITY)
              amax = fmaxf(amax, fabsf(x));
            else
              x = __int_as_float(0x7fffffff);  // (the conversion saturates infinities)
          };
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            look(a[t].x);
            look(a[t].y);
            look(b[t].x);
            look(b[t].y);
          }
        }
        __syncwarp();
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (store) {
          const float scale = fmaxf(amax, 1e-10f) * (1.f / 448.f);
          const float inv = __fdiv_rn(1.f, scale);
          const float2 inv2 = make_float2(inv, inv);
          uint32_t c[4];
#pragma unroll
          for (int t = 0; t < 4; ++t)
            c[t] = __nv_cvt_float2_to_fp8x2(mul2(in_order<kInterleaved>(a, b, 2 * t), inv2), __NV_SATFINITE, __NV_E4M3) |
                   (uint32_t)__nv_cvt_float2_to_fp8x2(mul2(in_order<kInterleaved>(a, b, 2 * t + 1), inv2), __NV_SATFINITE, __NV_E4M3) << 16;
          uint8_t* page = static_cast<uint8_t*>(p.cache) + place * (16 * kHD + kScaleBytes);
          uint8_t* dst = page + (slot & 15) * kHD;
          *reinterpret_cast<uint2*>(dst + e0) = make_uint2(c[0], c[1]);
          *reinterpret_cast<uint2*>(dst + e1) = make_uint2(c[2], c[3]);
          if (hl == 0) reinterpret_cast<float*>(page + 16 * kHD)[slot & 15] = scale;
        }
      } else if (store) {
        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.cache) + (place * 16 + (slot & 15)) * kHD;
        *reinterpret_cast<uint4*>(dst + e0) = bf16_words<kInterleaved>(a, b, 0);
        *reinterpret_cast<uint4*>(dst + e1) = bf16_words<kInterleaved>(a, b, 4);
      }
    }
  }
}

template <int kHD>
int launch(const KvStore& p, cudaStream_t stream) {
  const int heads = p.q_heads + 2 * p.kv_heads;
  // A warp a row, or for few rows a warp every few heads: as many parts as there are passes, while the
  // GPU has warps to spare (sixteen an SM).
  const int passes = (heads + 512 / kHD - 1) / (512 / kHD);
  int groups = (int)(148L * 16 / p.rows);
  groups = groups < 1 ? 1 : groups > passes ? passes : groups;
  const long ctas = ((long)p.rows * groups + 3) / 4;
  const auto kernel = p.interleaved ? (p.quantized ? kv_store_kernel<kHD, true, true> : kv_store_kernel<kHD, false, true>)
                                    : (p.quantized ? kv_store_kernel<kHD, true, false> : kv_store_kernel<kHD, false, false>);
  if (ctas > 2147483647L) return -2;
  return launch_pdl(kernel, dim3((unsigned)ctas), dim3(128), 0, stream, p, groups) == cudaSuccess ? 0 : -5;
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
