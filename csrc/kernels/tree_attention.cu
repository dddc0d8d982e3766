// Attention of decode rows, chunks and drafted token trees over the paged cache, BF16 or quantized
// (E4M3 codes with one FP32 scale a (position, head) for K and for V).
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale * q_i . k_j) where row i sees key j
//
// Row i of a segment sees the whole history and the appended rows j its mask names (or j <= i). A
// row that sees nothing gets zeros. What a row does not see does not reach it, NaN included.
//
// This is the mma.sync form, one CTA per (segment, key/value head, 16 (token, head) rows, split of
// the keys); its warps take the split's 16-key pages in turn, each streaming them through its own
// cp.async ring, and merge at the end. Splits meet in a second kernel, in split order.
//
// Quantized pages are half the bytes of BF16 ones, so the same HBM rate brings twice the keys; the
// codes become FP16 exactly in registers (cvt.rn.f16x2.e4m3x2):
// - Q is scaled a row by a power of two (exact) so that FP16 holds it; S = Q K^T * (k scale * ...).
// - V's scales join the exponent: with w_j = log2(v scale of j), the weights exp2(s_j + w_j - m) of
//   the codes have their own running maximum m of s + w, so FP16 (scaled by 2^14) holds them with
//   an underflow of 2^-38 of the largest; the sum of probabilities adds each weight / v scale.
// - K fragments are read 16 codes a lane: the MMA's k index runs over the head's elements in the
//   order that makes each lane's codes contiguous (Q's fragments follow the same order). V
//   fragments come from ldmatrix.trans over byte pairs, one prmt apart.
// Sums and statistics are FP32; P rounds to FP16 (BF16 over a BF16 cache), o once to BF16.

#include <cfloat>

#include "decode_ops.cuh"
#include "launch.cuh"
#include "sm100.cuh"

namespace foa {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 4;
constexpr float kLift = 14.f;  // weights are scaled by 2^14 (at most 2^14 of FP16's 65504)

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_b16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float lds_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// 16-byte async copy; `bytes` 0 fills the destination with zeros.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Two E4M3 codes (low 16 bits of `v`) as FP16, exactly.
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t v) {
  uint32_t r;
  asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n}" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_f16x2_hi(uint32_t v) {
  uint32_t r;
  asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, hi;\n}" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// Layout of one 16-key page of K or V in shared memory: rows of kRow bytes in 16-byte chunks, XOR
// swizzled so that the reads below meet no bank twice.
template <int D, bool kQ>
struct Page {
  static constexpr int kRow = kQ ? D : 2 * D;  // bytes of a key's row
  static constexpr int kChunks = kRow / 16;    // 16-byte chunks of a row
  static constexpr int kCodes = 16 * kRow;
  static constexpr int kBytes = kCodes + (kQ ? kScaleBytes : 0);  // in the cache and in shared memory
  static __device__ __forceinline__ uint32_t at(int r, int c) {
    int x;
    if constexpr (kChunks >= 8)
      x = ((r & 1) << 2) | ((r >> 1) & 3);  // K: lanes of two keys fall in different halves of the banks
    else
      x = (r >> 1) & 3;  // 64-byte rows: two rows fill the banks
    return (uint32_t)(r * kRow + ((c ^ x) << 4));
  }
};

struct Item {  // what a CTA works on
  Segment seg;
  int kvh, m0, split;
  bool ok;  // the segment's fields fit the launch
};

// Whether the segment's rows lie in q, and whether all of it fits the launch's sizes.
__device__ __forceinline__ bool rows_fit(const TreeAttention& p, const Segment& s) {
  return s.row_start >= 0 && s.len > 0 && (long)s.row_start + s.len <= p.rows;
}
__device__ __forceinline__ bool segment_fits(const TreeAttention& p, const Segment& s) {
  return s.cached >= 0 && s.len <= p.max_len && (long)s.cached + s.len <= p.max_keys && s.table_start >= 0 &&
         s.nblocks >= 0 && (long)s.table_start + s.nblocks <= p.table_len &&
         (long)s.nblocks * 16 >= (long)s.cached + s.len;
}

// Whether row `tok` of the segment sees appended row `j` (0 <= j < len).
__device__ __forceinline__ bool sees(const TreeAttention& p, const Segment& s, int tok, int j) {
  if (p.mask == nullptr) return j <= tok;
  if (j >= 32 * p.mask_words) return false;
  return p.mask[(long)(s.row_start + tok) * p.mask_words + (j >> 5)] >> (j & 31) & 1u;
}

// ------------------------------------------------------------------------------------ main kernel
template <int D, bool kQ, int kStages>
__global__ void __launch_bounds__(32 * kWarps, kQ ? 3 : 2)
    tree_attention_kernel(const TreeAttention p, int mtiles, int max_splits) {
  using P = Page<D, kQ>;
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kSteps = D / 16;   // 16-wide k-steps of Q K^T
  constexpr int kNt = D / 8;       // 8-wide column tiles of O
  const int G = p.q_heads / p.kv_heads;
  int item = blockIdx.x;
  const int mt = item % mtiles;
  item /= mtiles;
  const int kvh = item % p.kv_heads;
  const int si = item / p.kv_heads;
  const int split = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  pdl_wait();
  pdl_trigger();
  const Segment seg = p.segments[si];
  if (seg.len == 0) return;
  if (!rows_fit(p, seg) || !segment_fits(p, seg)) {
    // Rows of a segment that does not fit the launch are zeros (where they lie in o).
    if (mt == 0 && split == 0) {
      if (threadIdx.x == 0) record_status(p.status, kBadArgument);
      if (rows_fit(p, seg))
        for (long i = threadIdx.x; i < (long)seg.len * G * D; i += 32 * kWarps)
          p.o[(long)(seg.row_start + i / (G * D)) * p.ld_o + (long)kvh * G * D + i % (G * D)] = __float2bfloat16_rn(0.f);
    }
    return;
  }
  const int M = seg.len * G;
  const int m0 = mt * 16;
  const int keys = seg.cached + seg.len;
  const int nsplit = (keys + p.keys_per_split - 1) / p.keys_per_split;
  if (m0 >= M || split >= nsplit) return;
  const int k0 = split * p.keys_per_split;
  const int k1 = min(keys, k0 + p.keys_per_split);

  // Q fragments of rows m0 + g and m0 + g + 8 (zeros past M). k-step s of the quantized form takes
  // of lane t the elements 16 (t + 4 h) + 4 i .. + 3 with s = 4 h + i.
  uint32_t qa[kSteps][4];
  float qscale[2];
  const int row0 = m0 + g, row1 = m0 + g + 8;
  const int tok0 = row0 / G, tok1 = row1 / G;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int m = r ? row1 : row0;
    const __nv_bfloat16* src =
        m < M ? p.q + (long)(seg.row_start + m / G) * p.ld_q + (long)(kvh * G + m % G) * D : nullptr;
    // Each lane's elements: D / 4 of the row in 8-byte pieces, in the order of the k-steps.
    uint2 raw[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int e = kQ ? 16 * (t + 4 * (s >> 2)) + 4 * (s & 3) : 8 * (t + 4 * (s >> 1)) + 4 * (s & 1);
      raw[s] = src != nullptr ? *reinterpret_cast<const uint2*>(src + e) : make_uint2(0u, 0u);
    }
    if constexpr (kQ) {
      float amax = 0.f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        amax = fmaxf(amax, fmaxf(fmaxf(fabsf(bf16_lo(raw[s].x)), fabsf(bf16_hi(raw[s].x))),
                                 fmaxf(fabsf(bf16_lo(raw[s].y)), fabsf(bf16_hi(raw[s].y)))));
      amax = quad_max(amax);
      // 2^e <= amax < 2^(e+1): q * 2^(14 - e) stays below FP16's 65504 and loses only what lies
      // 2^-38 below the row's largest.
      const int e = min(max((int)(__float_as_uint(amax) >> 23), 15), 254) - 127;
      const float down = __uint_as_float((uint32_t)(127 + 14 - e) << 23);  // 14 - e in [-113, 126]
      qscale[r] = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        qa[s][r] = pack_f16x2(bf16_lo(raw[s].x) * down, bf16_hi(raw[s].x) * down);
        qa[s][r + 2] = pack_f16x2(bf16_lo(raw[s].y) * down, bf16_hi(raw[s].y) * down);
      }
    } else {
      qscale[r] = 1.f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        qa[s][r] = raw[s].x;
        qa[s][r + 2] = raw[s].y;
      }
    }
  }
  const float c0 = p.scale * kLog2e * qscale[0], c1 = p.scale * kLog2e * qscale[1];

  float o[kNt][4];
#pragma unroll
  for (int j = 0; j < kNt; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
  float m_[2] = {-INFINITY, -INFINITY}, l_[2] = {0.f, 0.f};

  const uint32_t wbase = smem_u32(smem) + warp * kStages * 2 * P::kBytes;
  const long page = (long)P::kBytes;
  const uint8_t* cache = static_cast<const uint8_t*>(p.cache);
  const int b_first = k0 / 16, b_last = (k1 - 1) / 16;
  const int32_t* table = p.table + seg.table_start;

  auto issue = [&](int b, int stage) {
    int id = table[b];
    // A block ID outside the cache reads zeros and records the bad index.
    const bool valid = id >= 0 && id < p.cache_blocks;
    if (!valid) {
      if (lane == 0) record_status(p.status, kBadIndex);
      id = 0;
    }
    const uint8_t* kp = cache + ((long)id * 2 * p.kv_heads + kvh) * page;
    const uint8_t* vp = kp + (long)p.kv_heads * page;
    const uint32_t kt = wbase + stage * 2 * P::kBytes, vt = kt + P::kBytes;
#pragma unroll
    for (int i = 0; i < (16 * P::kChunks) / 32; ++i) {
      const int chunk = lane + i * 32;
      const uint32_t dst = P::at(chunk / P::kChunks, chunk % P::kChunks);
      cp_async16(kt + dst, kp + chunk * 16, valid ? 16 : 0);
      cp_async16(vt + dst, vp + chunk * 16, valid ? 16 : 0);
    }
    if constexpr (kQ) {
      if (lane < 8)
        cp_async16((lane < 4 ? kt : vt) + P::kCodes + (lane & 3) * 16, (lane < 4 ? kp : vp) + P::kCodes + (lane & 3) * 16,
                   valid ? 16 : 0);
    }
    cp_async_commit();
  };

  int b = b_first + warp;
  bool odd_v = false;  // this warp left values that are not finite out of the products
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (b + i * kWarps <= b_last)
      issue(b + i * kWarps, i);
    else
      cp_async_commit();
  }
  for (int stage = 0; b <= b_last; b += kWarps, stage = stage + 1 == kStages ? 0 : stage + 1) {
    const int ahead = b + (kStages - 1) * kWarps;
    if (ahead <= b_last)
      issue(ahead, stage == 0 ? kStages - 1 : stage - 1);
    else
      cp_async_commit();
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const uint32_t kt = wbase + stage * 2 * P::kBytes, vt = kt + P::kBytes;
    const bool inner = b * 16 + 16 <= min(seg.cached, k1);  // every row sees every key of the page
    if (!inner) {
      // A product with a zero weight must stay zero: rows past the keys are cleared, and values
      // of appended rows that are not finite (each row adds those it sees at the end).
#pragma unroll
      for (int i = 0; i < (16 * P::kChunks) / 32; ++i) {
        const int chunk = lane + i * 32;
        const int key = b * 16 + chunk / P::kChunks;
        if (key < seg.cached) continue;
        const uint32_t a = vt + P::at(chunk / P::kChunks, chunk % P::kChunks);
        uint4 v = lds128(a);
        uint32_t* w = &v.x;
        bool change = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t bad = 0u;  // bytes (or halves) that are not finite
          if (key >= k1) {
            bad = ~0u;
          } else if constexpr (kQ) {
            for (int y = 0; y < 32; y += 8)
              if ((w[e] >> y & 0x7fu) == 0x7fu) bad |= 0xffu << y;
          } else {
            if ((w[e] & 0x7f80u) == 0x7f80u) bad |= 0xffffu;
            if ((w[e] & 0x7f800000u) == 0x7f800000u) bad |= 0xffff0000u;
          }
          if (bad != 0u) {
            change = true;
            if (key < k1) odd_v = true;
            w[e] &= ~bad;
          }
        }
        if (change) sts128(a, v);
      }
      __syncwarp();
    }

    // S = Q K^T of the page's two 8-key tiles.
    float s[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
      if constexpr (kQ) {
#pragma unroll
        for (int h = 0; h < kSteps / 4; ++h) {
          const uint4 w = lds128(kt + P::at(n * 8 + g, t + 4 * h));
          mma_f16(s[n], qa[4 * h], e4m3x2_f16x2(w.x), e4m3x2_f16x2_hi(w.x));
          mma_f16(s[n], qa[4 * h + 1], e4m3x2_f16x2(w.y), e4m3x2_f16x2_hi(w.y));
          mma_f16(s[n], qa[4 * h + 2], e4m3x2_f16x2(w.z), e4m3x2_f16x2_hi(w.z));
          mma_f16(s[n], qa[4 * h + 3], e4m3x2_f16x2(w.w), e4m3x2_f16x2_hi(w.w));
        }
      } else {
#pragma unroll
        for (int h = 0; h < kSteps / 2; ++h) {
          const uint4 w = lds128(kt + P::at(n * 8 + g, t + 4 * h));
          mma_b16(s[n], qa[2 * h], w.x, w.y);
          mma_b16(s[n], qa[2 * h + 1], w.z, w.w);
        }
      }
    }

    // Scaled scores (log2 units) with V's exponents, masked; the rows' maxima.
    float inv_v[2][2];  // 1 / v scale of this lane's keys
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float ks = 1.f, w = 0.f;
        inv_v[n][i] = 1.f;
        if constexpr (kQ) {
          ks = lds_f32(kt + P::kCodes + (n * 8 + 2 * t + i) * 4);
          const float vs = lds_f32(vt + P::kCodes + (n * 8 + 2 * t + i) * 4);
          if (vs > 0.f) {  // (a page of zeros has zero scales, whose codes are zeros too)
            w = __log2f(vs);
            inv_v[n][i] = __fdividef(1.f, vs);
          }
        }
        s[n][i] = fmaf(s[n][i], c0 * ks, w);
        s[n][i + 2] = fmaf(s[n][i + 2], c1 * ks, w);
      }
    if (!inner) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int key = b * 16 + n * 8 + 2 * t + i;
          const int j = key - seg.cached;
          if (key >= k1) inv_v[n][i] = 0.f;
          if (key >= k1 || (j >= 0 && (row0 >= M || !sees(p, seg, tok0, j)))) s[n][i] = -INFINITY;
          if (key >= k1 || (j >= 0 && (row1 >= M || !sees(p, seg, tok1, j)))) s[n][i + 2] = -INFINITY;
        }
    }
    float n0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
    float n1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
    n0 = fmaxf(m_[0], quad_max(n0));
    n1 = fmaxf(m_[1], quad_max(n1));
    // A row with no visible key yet keeps a zero state.
    const float f0 = n0 == -INFINITY ? 1.f : ex2(m_[0] - n0);
    const float f1 = n1 == -INFINITY ? 1.f : ex2(m_[1] - n1);
    const float z0 = n0 == -INFINITY ? 0.f : n0 - kLift, z1 = n1 == -INFINITY ? 0.f : n1 - kLift;
    m_[0] = n0;
    m_[1] = n1;
    float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s[n][i] = ex2(s[n][i] - z0);
        s[n][i + 2] = ex2(s[n][i + 2] - z1);
        sum0 = fmaf(s[n][i], inv_v[n][i], sum0);
        sum1 = fmaf(s[n][i + 2], inv_v[n][i], sum1);
      }
    l_[0] = l_[0] * f0 + sum0;
    l_[1] = l_[1] * f1 + sum1;
    if (__any_sync(0xffffffffu, f0 != 1.f || f1 != 1.f)) {
#pragma unroll
      for (int j = 0; j < kNt; ++j) {
        o[j][0] *= f0;
        o[j][1] *= f0;
        o[j][2] *= f1;
        o[j][3] *= f1;
      }
    }

    // O += P V: the 16 keys are one k-step.
    uint32_t pa[4];
    if constexpr (kQ) {
      pa[0] = pack_f16x2(s[0][0], s[0][1]);
      pa[1] = pack_f16x2(s[0][2], s[0][3]);
      pa[2] = pack_f16x2(s[1][0], s[1][1]);
      pa[3] = pack_f16x2(s[1][2], s[1][3]);
    } else {
      pa[0] = pack_bf16x2(s[0][0], s[0][1]);
      pa[1] = pack_bf16x2(s[0][2], s[0][3]);
      pa[2] = pack_bf16x2(s[1][0], s[1][1]);
      pa[3] = pack_bf16x2(s[1][2], s[1][3]);
    }
    // ldmatrix.trans: lanes 0-7 keys 0-7 chunk c, 8-15 keys 8-15 chunk c, 16-31 the same of c + 1.
#pragma unroll
    for (int c = 0; c < P::kChunks; c += 2) {
      uint32_t r[4];
      ldsm_x4_t(r, vt + P::at(lane & 15, c + (lane >> 4)));
      if constexpr (kQ) {
        // A register holds (two keys) x (two neighbouring elements): prmt makes them (two elements)
        // x (two keys). Tile 2c takes a chunk's even elements, 2c + 1 its odd ones.
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t lo = __byte_perm(r[2 * w], 0u, 0x3120), hi = __byte_perm(r[2 * w + 1], 0u, 0x3120);
          mma_f16(o[2 * (c + w)], pa, e4m3x2_f16x2(lo), e4m3x2_f16x2(hi));
          mma_f16(o[2 * (c + w) + 1], pa, e4m3x2_f16x2_hi(lo), e4m3x2_f16x2_hi(hi));
        }
      } else {
        mma_b16(o[c], pa, r[0], r[1]);
        mma_b16(o[c + 1], pa, r[2], r[3]);
      }
    }
    __syncwarp();
  }

  // Merge the warps: row statistics, then the rescaled sums, through shared memory.
  l_[0] = quad_sum(l_[0]);
  l_[1] = quad_sum(l_[1]);
  cp_async_wait<0>();
  __syncthreads();  // every warp is done with its pages
  float* sm_m = reinterpret_cast<float*>(smem);  // [kWarps][16]
  float* sm_l = sm_m + 16 * kWarps;
  float* sm_o = sm_l + 16 * kWarps;  // [16][D]
  if (t == 0) {
    sm_m[warp * 16 + g] = m_[0];
    sm_m[warp * 16 + g + 8] = m_[1];
    sm_l[warp * 16 + g] = l_[0];
    sm_l[warp * 16 + g + 8] = l_[1];
  }
  const bool fix = __syncthreads_or(odd_v);
  float top[2], w_[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float mm = -INFINITY;
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm_m[w * 16 + g + 8 * h]);
    top[h] = mm;
    w_[h] = m_[h] == -INFINITY ? 0.f : ex2(m_[h] - mm);
  }
  for (int w = 0; w < kWarps; ++w) {
    if (warp == w) {
#pragma unroll
      for (int j = 0; j < kNt; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int c = kQ ? 16 * (j >> 1) + 4 * t + 2 * i + (j & 1) : j * 8 + 2 * t + i;
            float* dst = sm_o + (g + 8 * h) * D + c;
            const float v = o[j][2 * h + i] * w_[h];
            *dst = w == 0 ? v : *dst + v;
          }
    }
    __syncthreads();
  }
  const int rows = min(16, M - m0);
  for (int i = threadIdx.x; i < rows * D; i += 32 * kWarps) {
    const int r = i / D, c = i % D;
    const int m = m0 + r, tok = m / G, head = kvh * G + m % G;
    float mm = -INFINITY, ll = 0.f;
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm_m[w * 16 + r]);
    for (int w = 0; w < kWarps; ++w) {
      const float mw = sm_m[w * 16 + r];
      ll += mw == -INFINITY ? 0.f : sm_l[w * 16 + r] * ex2(mw - mm);
    }
    float v = sm_o[i];
    if (fix) {
      for (int j = max(0, k0 - seg.cached); j < min(seg.len, k1 - seg.cached); ++j) {
        if (!sees(p, seg, tok, j)) continue;
        const int key = seg.cached + j, id = table[key >> 4];
        if (id < 0 || id >= p.cache_blocks) continue;
        const uint8_t* vp = cache + ((long)id * 2 * p.kv_heads + p.kv_heads + kvh) * page + (key & 15) * P::kRow;
        if constexpr (kQ) {
          if ((vp[c] & 0x7fu) == 0x7fu) v = __int_as_float(0x7fffffff);
        } else {
          const float x = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(vp)[c]);
          if (!(fabsf(x) < INFINITY)) v += x;
        }
      }
    }
    const long at = (long)(seg.row_start + tok);
    if (nsplit == 1) {
      p.o[at * p.ld_o + (long)head * D + c] = __float2bfloat16_rn(mm == -INFINITY ? 0.f : v / ll);
    } else {
      const long idx = (at * p.q_heads + head) * max_splits + split;
      p.partial_o[idx * D + c] = v;
      if (c == 0) p.partial_ml[idx] = make_float2(mm, ll);
    }
  }
}

// Joins the splits of each (row, head), in split order: one warp each.
template <int D>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeAttention p, int max_splits) {
  pdl_wait();
  pdl_trigger();
  const Segment seg = p.segments[blockIdx.x / p.max_len];
  const int tok = blockIdx.x % p.max_len;
  const int head = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (tok >= seg.len || head >= p.q_heads || !rows_fit(p, seg) || !segment_fits(p, seg)) return;
  const int nsplit = (seg.cached + seg.len + p.keys_per_split - 1) / p.keys_per_split;
  if (nsplit == 1) return;  // written in place
  const long row = seg.row_start + tok;
  const long base = (row * p.q_heads + head) * max_splits;
  float top = -INFINITY;
  for (int s = lane; s < nsplit; s += 32) top = fmaxf(top, p.partial_ml[base + s].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  constexpr int E = D / 32;
  float acc[E], den = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  if (top > -INFINITY) {
#pragma unroll 4
    for (int s = 0; s < nsplit; ++s) {
      const float2 ml = p.partial_ml[base + s];
      const float w = ex2(ml.x - top);
      den = fmaf(w, ml.y, den);
      const float* src = p.partial_o + (base + s) * D + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(w, src[e], acc[e]);
    }
  } else {
    den = 1.f;
  }
  __nv_bfloat16* dst = p.o + row * p.ld_o + (long)head * D + lane * E;
  const float inv = 1.f / den;
#pragma unroll
  for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
}

template <int D, bool kQ>
int launch(const TreeAttention& p, cudaStream_t stream) {
  constexpr int kStages = kQ ? 4 : 3;
  const int G = p.q_heads / p.kv_heads;
  const int splits = (p.max_keys + p.keys_per_split - 1) / p.keys_per_split;
  if (splits > 65535) return -2;
  if (splits > 1) {
    const size_t need = (size_t)p.rows * p.q_heads * splits;
    if (p.partial_o == nullptr || p.partial_ml == nullptr || need > p.partial_capacity) return -3;
  }
  const long mtiles = ((long)p.max_len * G + 15) / 16;
  const long ctas = mtiles * p.kv_heads * p.num_segments;
  if (ctas > 2147483647L || (long)p.num_segments * p.max_len > 2147483647L) return -2;
  constexpr int smem = kWarps * kStages * 2 * Page<D, kQ>::kBytes;
  const auto kernel = tree_attention_kernel<D, kQ, kStages>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -5;
  if (launch_pdl(kernel, dim3((unsigned)ctas, splits), dim3(32 * kWarps), smem, stream, p, (int)mtiles, splits) != cudaSuccess)
    return -5;
  if (splits > 1 && launch_pdl(tree_merge_kernel<D>, dim3(p.num_segments * p.max_len, (p.q_heads + 7) / 8), dim3(256), 0,
                               stream, p, splits) != cudaSuccess)
    return -5;
  return 0;
}

}  // namespace

int tree_attention_split(int num_segments, int q_heads, int kv_heads, int head_dim, int quantized, int max_keys,
                         int max_len) {
  if (num_segments <= 0 || kv_heads <= 0 || max_keys <= 0) return 16;
  const long tiles = ((long)max_len * (q_heads / kv_heads) + 15) / 16;
  const long items = tiles * kv_heads * num_segments;
  // About four CTAs for each that the GPU holds at once, of at least 64 keys a warp.
  const long want = 148L * 3 * 4;
  const long per = (long)max_keys * items / want;
  long keys = per < 256 ? 256 : per;
  keys = (keys + 63) / 64 * 64;
  return (int)(keys > max_keys ? (max_keys + 15) / 16 * 16 : keys);
}

int tree_attention(const TreeAttention& p, cudaStream_t stream) {
  if (p.num_segments <= 0 || p.rows <= 0) return 0;
  if (p.kv_heads <= 0 || p.q_heads <= 0 || p.q_heads % p.kv_heads != 0) return -2;
  if (p.max_keys <= 0 || p.max_len <= 0 || p.keys_per_split <= 0 || p.keys_per_split % 16 != 0) return -2;
  if (p.ld_q % 8 != 0 || p.ld_o % 8 != 0) return -2;
  if ((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.o) | reinterpret_cast<uintptr_t>(p.cache)) & 15)
    return -2;
  if (p.head_dim == 64) return p.quantized ? launch<64, true>(p, stream) : launch<64, false>(p, stream);
  if (p.head_dim == 128) return p.quantized ? launch<128, true>(p, stream) : launch<128, false>(p, stream);
  return -2;
}

}  // namespace foa
