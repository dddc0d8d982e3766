// Attention of decode rows, chunks and drafted token trees over the paged cache, BF16 or quantized
// (E4M3 codes with one FP32 scale a (position, head) for K and for V).
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale * q_i . k_j) where row i sees key j
//
// Row i of a segment sees the whole history and the appended rows j its mask names (or j <= i). A
// row that sees nothing gets zeros. What a row does not see does not reach it, NaN included.
//
// This is the mma.sync form, one CTA per (segment, key/value head, tile of 8 or 16 (token, head)
// rows, split of the keys); its warps take the split's 16-key pages in turn, each streaming them
// through its own cp.async ring, and merge at the end. Splits meet in a second kernel, in split order.
//
// Keys are the MMA's M (a page's 16) and query rows its N (8 a tile), so few rows waste little:
// S^T = K Q^T, and O^T = V^T P^T with P^T from S^T by movmatrix. A decode row of eight heads a
// key/value head takes half of the products and accumulators of the form with rows as M.
//
// Quantized pages are half the bytes of BF16 ones, so the same HBM rate brings twice the keys; what
// the warps issue a page decides. The codes become FP16 exactly in registers (cvt.rn.f16x2.e4m3x2):
// - Q is scaled a row by a power of two (exact) so that FP16 holds it; K's scales multiply S.
// - V's scales multiply the weights before they round to FP16, by way of a power of two that keeps
//   the largest scale that the row has seen near one; that and the rows' maxima move only when a page
//   exceeds them (the maxima by 2^4), which one vote a page finds. Weights stay below 2^15 of FP16's
//   65504 and lose what lies 2^-34 below the largest.
// - K fragments are read 16 codes a lane: the MMA's k index runs over the head's elements in the
//   order that makes each lane's codes contiguous (Q's fragments follow the same order). V
//   fragments come from ldmatrix.trans over byte pairs, one prmt apart.
// Sums and statistics are FP32; P rounds to FP16 (BF16 over a BF16 cache), o once to BF16.
//
// Bound by HBM for batches of long histories (64 uniform sequences of 8192 keys, 32 x 8 heads: 6100
// GB/s over codes, 6800 over BF16), by uneven CTAs where lengths differ (64 sequences of 1152 to 9216
// keys: 112 us, 5400 GB/s), by the chain of one CTA and the join for few (one of 1000 keys: 8.2 us).
// Two pages in flight a warp and five CTAs an SM take 110 us where three pages, four CTAs and
// addresses computed for each access take 123.

#include "decode_ops.cuh"
#include "launch.cuh"
#include "sm100.cuh"
#include "tree_split.cuh"

namespace foa {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 4;
constexpr float kLift = 10.f;   // weights are scaled by 2^10 ...
constexpr float kSlack = 4.f;   // ... and may exceed the row's reference maximum by 2^4

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
// Transposes the warp's 8 x 8 matrix of 16-bit values (row g, columns 2t and 2t + 1 a lane).
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Layout of one 16-key page of K or V in shared memory: rows of kRow bytes in 16-byte chunks, XOR
// swizzled so that the reads below meet no bank twice.
template <int D, bool kQ>
struct Page {
  static constexpr int kRow = kQ ? D : 2 * D;  // bytes of a key's row
  static constexpr int kChunks = kRow / 16;    // 16-byte chunks of a row
  static constexpr int kCodes = 16 * kRow;
  static constexpr int kBytes = kCodes + (kQ ? kScaleBytes : 0);  // in the cache
  // In shared memory: pages begin where an XOR of an address's swizzled bits is one of its offset's.
  static constexpr int kAlign = kRow >= 128 ? kRow : 128;
  static constexpr int kSlot = (kBytes + kAlign - 1) / kAlign * kAlign;
  static __device__ __forceinline__ uint32_t at(int r, int c) {
    int x;
    if constexpr (kChunks >= 8)
      x = ((r & 1) << 2) | ((r >> 1) & 3);  // K: lanes of two keys fall in different halves of the banks
    else
      x = (r >> 1) & 3;  // 64-byte rows: two rows fill the banks
    return (uint32_t)(r * kRow + ((c ^ x) << 4));
  }
  // Chunk lane + 32 i of the page lies at (at(lane / kChunks, lane % kChunks) ^ flip(i)) + 512 i.
  static __device__ __forceinline__ constexpr uint32_t flip(int i) {
    return kChunks == 16 ? (uint32_t)(i & 3) << 4 : kChunks == 8 ? (uint32_t)(i & 1) << 5 : 0u;
  }
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
template <int D, bool kQ, int NT>
struct Shape {
  // Two stages and many warps rather than three and fewer: what a warp waits for is mostly its own
  // last instruction, not memory.
  static constexpr int kStages = 2;
  static constexpr int kCtas = NT == 1 ? (kQ ? 5 : 3) : (kQ ? 3 : 2);  // of an SM, by registers and shared memory
  static constexpr int kSmem = kWarps * kStages * 2 * Page<D, kQ>::kSlot;
};

template <int D, bool kQ, int NT>
__global__ void __launch_bounds__(32 * kWarps, Shape<D, kQ, NT>::kCtas)
    tree_attention_kernel(const TreeAttention p, int mtiles, int max_splits) {
  using P = Page<D, kQ>;
  constexpr int kStages = Shape<D, kQ, NT>::kStages;
  extern __shared__ __align__(256) uint8_t smem[];
  constexpr int kSteps = D / 16;  // 16-wide k-steps of K Q^T, and 16-row tiles of O^T
  constexpr int kRows = 8 * NT;
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
  const int m0 = mt * kRows;
  const int keys = seg.cached + seg.len;
  const Parts parts(keys, p.keys_per_split, false);
  const int nsplit = parts.count;
  if (m0 >= M || split >= nsplit) return;
  const int k0 = split * parts.width;
  const int k1 = min(keys, k0 + parts.width);

  const uint32_t wbase = smem_u32(smem) + warp * kStages * 2 * P::kSlot;
  const uint8_t* cache = static_cast<const uint8_t*>(p.cache);
  const int32_t* table = p.table + seg.table_start;
  const int b_last = (k1 - 1) / 16;
  const int b_first = k0 / 16 + warp;  // this warp's pages: b_first, b_first + kWarps, ...
  // Block IDs of 32 of the warp's pages, one a lane.
  int ids = 0, ids_at = b_first;
  if (b_first + lane * kWarps <= b_last) ids = table[b_first + lane * kWarps];

  const uint8_t* from = cache + (long)kvh * P::kBytes + lane * 16;
  const uint32_t block = (uint32_t)(2 * p.kv_heads * P::kBytes), v_off = (uint32_t)(p.kv_heads * P::kBytes);
  const uint32_t to = P::at(lane / P::kChunks, lane % P::kChunks);
  auto issue = [&](int b, int stage) {
    if (b >= ids_at + 32 * kWarps) {
      ids_at = b;
      if (b + lane * kWarps <= b_last) ids = table[b + lane * kWarps];
    }
    int id = __shfl_sync(0xffffffffu, ids, (b - ids_at) / kWarps);
    // A block ID outside the cache reads zeros and records the bad index.
    const bool valid = id >= 0 && id < p.cache_blocks;
    if (!valid) {
      if (lane == 0) record_status(p.status, kBadIndex);
      id = 0;
    }
    const uint8_t* kp = from + (uint64_t)id * block;
    const uint8_t* vp = kp + v_off;
    const uint32_t kt = wbase + stage * 2 * P::kSlot, vt = kt + P::kSlot;
    const int n = valid ? 16 : 0;
#pragma unroll
    for (int i = 0; i < (16 * P::kChunks) / 32; ++i) {
      cp_async16(((kt + to) ^ P::flip(i)) + i * 512, kp + i * 512, n);
      cp_async16(((vt + to) ^ P::flip(i)) + i * 512, vp + i * 512, n);
    }
    if constexpr (kQ) {
      if (lane < 4) {
        cp_async16(kt + P::kCodes + lane * 16, kp + P::kCodes, n);
        cp_async16(vt + P::kCodes + lane * 16, vp + P::kCodes, n);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (b_first + i * kWarps <= b_last)
      issue(b_first + i * kWarps, i);
    else
      cp_async_commit();
  }

  // Q fragments: column g of tile n is row m0 + 8 n + g (zeros past M). k-step s of the quantized
  // form takes of lane t the elements 16 (t + 4 h) + 4 i .. + 3 with s = 4 h + i.
  uint32_t qb[NT][kSteps][2];
  float c_[NT][2];  // scale to log2 units of this lane's columns 2t, 2t + 1
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int m = m0 + 8 * n + g;
    const __nv_bfloat16* src =
        m < M ? p.q + (long)(seg.row_start + m / G) * p.ld_q + (long)(kvh * G + m % G) * D : nullptr;
    uint2 raw[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int e = kQ ? 16 * (t + 4 * (s >> 2)) + 4 * (s & 3) : 8 * (t + 4 * (s >> 1)) + 4 * (s & 1);
      raw[s] = src != nullptr ? *reinterpret_cast<const uint2*>(src + e) : make_uint2(0u, 0u);
    }
    // The row's largest magnitude, as BF16 bits.
    uint32_t most = 0u;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) most = __vmaxu2(most, __vmaxu2(raw[s].x & 0x7fff7fffu, raw[s].y & 0x7fff7fffu));
    most = max(most >> 16, most & 0xffffu);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // A row with an element that is not finite has no finite score: what it sees makes it NaN (of an
    // infinity's products those of one sign would pass for keys that are not seen).
    float c = most >= 0x7f80u ? __int_as_float(0x7fffffff) : p.scale * kLog2e;
    if constexpr (kQ) {
      // 2^e <= the largest < 2^(e+1): q * 2^(14 - e) stays below FP16's 65504 and loses only what lies
      // 2^-38 below the row's largest.
      const int e = min(max((int)(most >> 7), 15), 254) - 127;
      const float down = __uint_as_float((uint32_t)(127 + 14 - e) << 23);  // 14 - e in [-113, 126]
      c *= __uint_as_float((uint32_t)(127 - 14 + e) << 23);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        qb[n][s][0] = pack_f16x2(bf16_lo(raw[s].x) * down, bf16_hi(raw[s].x) * down);
        qb[n][s][1] = pack_f16x2(bf16_lo(raw[s].y) * down, bf16_hi(raw[s].y) * down);
      }
    } else {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        qb[n][s][0] = raw[s].x;
        qb[n][s][1] = raw[s].y;
      }
    }
    c_[n][0] = __shfl_sync(0xffffffffu, c, 8 * t);
    c_[n][1] = __shfl_sync(0xffffffffu, c, 8 * t + 4);
  }

  // O^T: tile c, entries (row, column) = (g, 2t), (g, 2t + 1), (g + 8, 2t), (g + 8, 2t + 1).
  float o[NT][kSteps][4];
  float m_[NT][2], l_[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < kSteps; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][c][i] = 0.f;
    m_[n][0] = m_[n][1] = -INFINITY;
    l_[n][0] = l_[n][1] = 0.f;
  }
  // 2^-e, e the exponent of the largest V scale that the row has seen (a drafted node's values may be
  // far larger than those of rows that do not see it), and the least 2^(e + 1) of this lane's rows.
  float v_inv[NT][2];
  float v_lim = 0x1p-125f;
#pragma unroll
  for (int n = 0; n < NT; ++n) v_inv[n][0] = v_inv[n][1] = 0x1p126f;
  bool odd_v = false;          // this lane left values that are not finite out of the products

  // Addresses of this lane's fragments in a page; others of them differ in swizzled bits alone.
  const uint32_t k_at = P::at(g, t);
  const uint32_t v_at = kQ ? P::at(lane & 15, lane >> 4) : P::at((lane & 7) + 8 * (lane >> 4), lane >> 3 & 1);
  int stage = 0;
  for (int b = b_first; b <= b_last; b += kWarps, stage = stage + 1 == kStages ? 0 : stage + 1) {
    const int ahead = b + (kStages - 1) * kWarps;
    if (ahead <= b_last)
      issue(ahead, stage == 0 ? kStages - 1 : stage - 1);
    else
      cp_async_commit();
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const uint32_t kt = wbase + stage * 2 * P::kSlot, vt = kt + P::kSlot;
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
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
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
        if (change) sts128(a, make_uint4(w[0], w[1], w[2], w[3]));
      }
      __syncwarp();
    }

    // S^T of the page: rows are keys g and g + 8.
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
    if constexpr (kQ) {
#pragma unroll
      for (int h = 0; h < kSteps / 4; ++h) {
        const uint32_t at = (kt + k_at) ^ (h << 6);
        const uint4 x = lds128(at), y = lds128(at + 8 * P::kRow);
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a[4] = {e4m3x2_f16x2(xw[i]), e4m3x2_f16x2(yw[i]), e4m3x2_f16x2_hi(xw[i]), e4m3x2_f16x2_hi(yw[i])};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(s[n], a, qb[n][4 * h + i][0], qb[n][4 * h + i][1]);
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < kSteps / 2; ++h) {
        const uint32_t at = (kt + k_at) ^ (h << 6);
        const uint4 x = lds128(at), y = lds128(at + 8 * P::kRow);
        const uint32_t a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_b16(s[n], a0, qb[n][2 * h][0], qb[n][2 * h][1]);
          mma_b16(s[n], a1, qb[n][2 * h + 1][0], qb[n][2 * h + 1][1]);
        }
      }
    }

    // Scores in log2 units; masked ones are -inf.
    float ks[2] = {1.f, 1.f}, vs[2] = {1.f, 1.f};
    if constexpr (kQ) {
      ks[0] = lds_f32(kt + P::kCodes + g * 4);
      ks[1] = lds_f32(kt + P::kCodes + g * 4 + 32);
      vs[0] = lds_f32(vt + P::kCodes + g * 4);
      vs[1] = lds_f32(vt + P::kCodes + g * 4 + 32);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] *= kQ ? c_[n][i & 1] * ks[i >> 1] : c_[n][i & 1];
    if (!inner) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int key = b * 16 + g + 8 * r;
        const int j = key - seg.cached;
        if (key >= k1) vs[r] = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int m = m0 + 8 * n + 2 * t + i;
            if (key >= k1 || (j >= 0 && (m >= M || !sees(p, seg, m / G, j)))) s[n][2 * r + i] = -INFINITY;
          }
      }
    }
    // One vote finds whether a row's maximum or V's reference scale must move.
    bool move = kQ && (vs[0] >= v_lim || vs[1] >= v_lim);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) move = move || fmaxf(s[n][i], s[n][i + 2]) > m_[n][i] + kSlack;
    if (__any_sync(0xffffffffu, move)) {
      v_lim = INFINITY;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x = fmaxf(s[n][i], s[n][i + 2]);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(m_[n][i], fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16)));
          // A row with no visible key yet keeps a zero state.
          const float f = x == -INFINITY ? 1.f : ex2(m_[n][i] - x);
          m_[n][i] = x;
          l_[n][i] *= f;
          float fv = 1.f;
          if constexpr (kQ) {
            float top = fmaxf(s[n][i] > -INFINITY ? vs[0] : 0.f, s[n][i + 2] > -INFINITY ? vs[1] : 0.f);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const int was = 127 - (int)(__float_as_uint(v_inv[n][i]) >> 23);
            const int e = max(was, min(max((int)(__float_as_uint(top) >> 23), 1), 253) - 127);
            fv = ex2((float)(was - e));
            v_inv[n][i] = __uint_as_float((uint32_t)(127 - e) << 23);  // e <= 126
            v_lim = fminf(v_lim, __uint_as_float((uint32_t)(128 + e) << 23));
          }
#pragma unroll
          for (int c = 0; c < kSteps; ++c) {
            o[n][c][i] *= f * fv;
            o[n][c][i + 2] *= f * fv;
          }
        }
    }

    // Weights, their sums, and P^T as the B operand (rows are keys).
    uint32_t pb[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float z = m_[n][i & 1] == -INFINITY ? 0.f : m_[n][i & 1] - kLift;
        w[i] = ex2(s[n][i] - z);
        l_[n][i & 1] += w[i];
        if constexpr (kQ) w[i] *= !inner && s[n][i] == -INFINITY ? 0.f : vs[i >> 1] * v_inv[n][i & 1];
      }
      if constexpr (kQ) {
        pb[n][0] = transpose8(pack_f16x2(w[0], w[1]));
        pb[n][1] = transpose8(pack_f16x2(w[2], w[3]));
      } else {
        pb[n][0] = transpose8(pack_bf16x2(w[0], w[1]));
        pb[n][1] = transpose8(pack_bf16x2(w[2], w[3]));
      }
    }

    // O^T += V^T P^T.
    if constexpr (kQ) {
      // ldmatrix.trans: lanes 0-7 keys 0-7 chunk c, 8-15 keys 8-15 chunk c, 16-31 the same of c + 1.
      // A register holds (two keys) x (two neighbouring elements): prmt makes them (two elements)
      // x (two keys). A tile's rows 0-7 are a chunk's even elements, 8-15 its odd ones.
#pragma unroll
      for (int c = 0; c < P::kChunks; c += 2) {
        uint32_t r[4];
        ldsm_x4_t(r, (vt + v_at) ^ (c << 4));
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t lo = __byte_perm(r[2 * w], 0u, 0x3120), hi = __byte_perm(r[2 * w + 1], 0u, 0x3120);
          const uint32_t a[4] = {e4m3x2_f16x2(lo), e4m3x2_f16x2_hi(lo), e4m3x2_f16x2(hi), e4m3x2_f16x2_hi(hi)};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(o[n][c + w], a, pb[n][0], pb[n][1]);
        }
      }
    } else {
      // ldmatrix.trans: lanes 0-15 keys 0-7 of chunks 2c and 2c + 1, 16-31 keys 8-15 of them.
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        uint32_t r[4];
        ldsm_x4_t(r, (vt + v_at) ^ (2 * c << 4));
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_b16(o[n][c], r, pb[n][0], pb[n][1]);
      }
    }
    __syncwarp();
  }

  // Merge the warps: row statistics, then the rescaled sums, through shared memory.
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l_[n][i] += __shfl_xor_sync(0xffffffffu, l_[n][i], x);
  cp_async_wait<0>();
  __syncthreads();  // every warp is done with its pages
  float* sm_m = reinterpret_cast<float*>(smem);  // [kWarps][kRows]
  float* sm_l = sm_m + kRows * kWarps;
  float* sm_o = sm_l + kRows * kWarps;  // [kWarps][kRows][D]
  static_assert((2 * 16 * kWarps + kWarps * 16 * D) * 4 <= Shape<D, kQ, 2>::kSmem, "merge fits the ring");
  static_assert((2 * 8 * kWarps + kWarps * 8 * D) * 4 <= Shape<D, kQ, 1>::kSmem, "merge fits the ring");
  if (g == 0) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sm_m[warp * kRows + 8 * n + 2 * t + i] = m_[n][i];
        sm_l[warp * kRows + 8 * n + 2 * t + i] = l_[n][i];
      }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float* dst = sm_o + (warp * kRows + 8 * n + 2 * t + i) * D;
      const float back = kQ ? __uint_as_float((254u << 23) - __float_as_uint(v_inv[n][i])) : 1.f;  // 2^e
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        if constexpr (kQ) {
          *reinterpret_cast<float2*>(dst + 16 * c + 2 * g) = make_float2(o[n][c][i] * back, o[n][c][i + 2] * back);
        } else {
          dst[16 * c + g] = o[n][c][i];
          dst[16 * c + g + 8] = o[n][c][i + 2];
        }
      }
    }
  const bool fix = __syncthreads_or(odd_v);
  const int rows = min(kRows, M - m0);
  for (int i = threadIdx.x; i < rows * (D / 2); i += 32 * kWarps) {
    const int r = i / (D / 2), c = 2 * (i % (D / 2));
    const int m = m0 + r, tok = m / G, head = kvh * G + m % G;
    float mm = -INFINITY, ll = 0.f;
    float2 v = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm_m[w * kRows + r]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = sm_m[w * kRows + r];
      const float f = mw == -INFINITY ? 0.f : ex2(mw - mm);
      const float2 x = *reinterpret_cast<const float2*>(sm_o + (w * kRows + r) * D + c);
      ll = fmaf(f, sm_l[w * kRows + r], ll);
      v.x = fmaf(f, x.x, v.x);
      v.y = fmaf(f, x.y, v.y);
    }
    if (fix) {
      for (int j = max(0, k0 - seg.cached); j < min(seg.len, k1 - seg.cached); ++j) {
        if (!sees(p, seg, tok, j)) continue;
        const int key = seg.cached + j, id = table[key >> 4];
        if (id < 0 || id >= p.cache_blocks) continue;
        const uint8_t* vp = cache + ((long)id * 2 * p.kv_heads + p.kv_heads + kvh) * P::kBytes + (key & 15) * P::kRow;
        if constexpr (kQ) {
          if ((vp[c] & 0x7fu) == 0x7fu) v.x = __int_as_float(0x7fffffff);
          if ((vp[c + 1] & 0x7fu) == 0x7fu) v.y = __int_as_float(0x7fffffff);
        } else {
          const float x = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(vp)[c]);
          const float y = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(vp)[c + 1]);
          if (!(fabsf(x) < INFINITY)) v.x += x;
          if (!(fabsf(y) < INFINITY)) v.y += y;
        }
      }
    }
    const long at = (long)(seg.row_start + tok);
    if (nsplit == 1) {
      const float inv = mm == -INFINITY ? 0.f : 1.f / ll;
      *reinterpret_cast<uint32_t*>(p.o + at * p.ld_o + (long)head * D + c) = pack_bf16x2(v.x * inv, v.y * inv);
    } else {
      const long idx = (at * p.q_heads + head) * max_splits + split;
      *reinterpret_cast<float2*>(p.partial_o + idx * D + c) = v;
      if (c == 0) p.partial_ml[idx] = make_float2(mm, ll);
    }
  }
}

// Joins the splits of each (row, head): a CTA each, whose warps take the splits in turn and meet in
// a fixed order. (One warp a head took 20 us for 64 splits of 192 heads: it waits for one load
// after another.) Rows of more than sixteen splits get sixteen warps: with four, one sequence of 131072
// keys and 16 heads in 256 splits took 77 us, with sixteen 60. How many take part follows from the
// row's own splits, so that the order of its sums is the same in every call.
template <int D, int W>
__global__ void __launch_bounds__(32 * W) tree_merge_kernel(const TreeAttention p, int max_splits, int longest, bool even) {
  constexpr int E = D / 32;
  __shared__ float sm_acc[W - 1][D], sm_den[W - 1];
  pdl_wait();
  pdl_trigger();
  const Segment seg = p.segments[blockIdx.x / longest];
  const int tok = blockIdx.x % longest;
  const int head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (tok >= seg.len || !rows_fit(p, seg) || !segment_fits(p, seg)) return;
  const int nsplit = Parts(seg.cached + seg.len, p.keys_per_split, even).count;
  if (nsplit == 1) return;  // written in place
  const int warps = nsplit > 16 ? 16 : 4;  // (the launch has sixteen when a row may need them)
  const long row = seg.row_start + tok;
  const long base = (row * p.q_heads + head) * max_splits;
  // A part whose scores are all NaN has the maximum of one that sees nothing, and a sum that is NaN.
  float top = -INFINITY;
  bool nan = false;
  for (int s = lane; s < nsplit; s += 32) {
    const float2 ml = p.partial_ml[base + s];
    top = fmaxf(top, ml.x);
    nan = nan || ml.y != ml.y;
  }
  nan = __any_sync(0xffffffffu, nan);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float acc[E], den = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  if (top > -INFINITY) {
#pragma unroll 4
    for (int s = warp < warps ? warp : nsplit; s < nsplit; s += warps) {
      const float2 ml = p.partial_ml[base + s];
      const float w = ex2(ml.x - top);
      den = fmaf(w, ml.y, den);
      const float* src = p.partial_o + (base + s) * D + lane * E;
      float x[E];
      if constexpr (E == 4) {
        const float4 v = *reinterpret_cast<const float4*>(src);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
      } else {
        const float2 v = *reinterpret_cast<const float2*>(src);
        x[0] = v.x, x[1] = v.y;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(w, x[e], acc[e]);
    }
  }
  if (warp > 0) {
#pragma unroll
    for (int e = 0; e < E; ++e) sm_acc[warp - 1][lane * E + e] = acc[e];
    if (lane == 0) sm_den[warp - 1] = den;
  }
  __syncthreads();
  if (warp > 0) return;
#pragma unroll
  for (int w = 0; w < W - 1; ++w) {
    if (w + 1 >= warps) break;
    den += sm_den[w];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += sm_acc[w][lane * E + e];
  }
  __nv_bfloat16* dst = p.o + row * p.ld_o + (long)head * D + lane * E;
  if (nan) den = __int_as_float(0x7fffffff);
  const float inv = top > -INFINITY || nan ? 1.f / den : 0.f;
#pragma unroll
  for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
}

template <int D>
int merge(const TreeAttention& p, int splits, bool even, cudaStream_t stream) {
  if (splits == 1) return 0;
  const int longest = longest_segment(p);
  const dim3 grid(p.num_segments * longest, p.q_heads);
  const cudaError_t rc = splits > 16 ? launch_pdl(tree_merge_kernel<D, 16>, grid, dim3(512), 0, stream, p, splits, longest, even)
                                     : launch_pdl(tree_merge_kernel<D, 4>, grid, dim3(128), 0, stream, p, splits, longest, even);
  return rc == cudaSuccess ? 0 : -5;
}

template <int D, bool kQ, int NT>
int launch(const TreeAttention& p, cudaStream_t stream) {
  const int G = p.q_heads / p.kv_heads;
  const int splits = ((long)p.max_keys + p.keys_per_split - 1) / p.keys_per_split;
  const long mtiles = ((long)longest_segment(p) * G + 8 * NT - 1) / (8 * NT);
  const long ctas = mtiles * p.kv_heads * p.num_segments;
  if (ctas > 2147483647L) return -2;
  constexpr int smem = Shape<D, kQ, NT>::kSmem;
  const auto kernel = tree_attention_kernel<D, kQ, NT>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -5;
    configured[dev & 63] = true;
  }
  if (launch_pdl(kernel, dim3((unsigned)ctas, splits), dim3(32 * kWarps), smem, stream, p, (int)mtiles, splits) != cudaSuccess)
    return -5;
  return merge<D>(p, splits, false, stream);
}

// Whether a segment may have more rows than the mma.sync form holds in one tile, or in two over codes,
// where a second pass over the pages (from L2) costs less than a tcgen05 tile that is a quarter full:
// 64 trees of 5 nodes, 4 heads a key/value head, up to 4096 keys: 116 us in two tiles, 175 by tcgen05;
// 16 of 8 nodes, up to 8192 keys: 80 and 95. (BF16: 89 and 85.)
bool tc_rows(int max_len, int group, bool quantized) { return (long)max_len * group > (quantized ? 32 : 16); }

template <int D, bool kQ>
int pick(const TreeAttention& p, cudaStream_t stream) {
  if (tc_rows(p.max_len, p.q_heads / p.kv_heads, kQ) && tree_attention_tc_supported(p)) {
    const int rc = tree_attention_tc(p, stream);
    return rc != 0 ? rc : merge<D>(p, (p.max_keys + p.keys_per_split - 1) / p.keys_per_split, true, stream);
  }
  return (long)p.max_len * (p.q_heads / p.kv_heads) <= 8 ? launch<D, kQ, 1>(p, stream) : launch<D, kQ, 2>(p, stream);
}

}  // namespace

int tree_attention_split(int num_segments, int q_heads, int kv_heads, int head_dim, int quantized, int max_keys,
                         int max_len) {
  if (num_segments <= 0 || kv_heads <= 0 || max_keys <= 0) return 16;
  const long rows = (long)max_len * (q_heads / kv_heads);
  const bool tc = tc_rows(max_len, (int)(q_heads / kv_heads), quantized != 0);
  const long tile = tc ? 256 : 16;
  const long items = (rows + tile - 1) / tile * kv_heads * num_segments;
  // About two (tcgen05) or three CTAs for each that the GPU holds at once (segments may differ in
  // length), of at least so many keys that a CTA's start and end do not count; fewer where the GPU is
  // far from full (one sequence of 1000 keys, 8 heads: 8.2 us in splits of 128, 9.5 of 256; four of
  // 2048: 11.4 and 10.8). Long histories are cut into 96 parts at most, since each is joined again, and
  // where a key/value head has more than 8 rows, each part of which leaves as much as 60 keys take,
  // into 32 (one of 32768 keys, 16 rows: 26 us in splits of 1024, 39 of 256).
  const bool wide = !tc && rows > 8;
  const long want = tc ? 148L * 2 : wide ? 148L * 9 : 148L * 16;
  const long parts = tc ? max_keys : wide ? 32 : 96;
  const long thin = items * (((long)max_keys + 127) / 128) <= 148L * 2 ? 128 : 256;
  const long least = tc ? 512 : (max_keys + parts - 1) / parts > thin ? (max_keys + parts - 1) / parts : thin;
  const long per = ((long)max_keys * items + want - 1) / want;
  const long keys = ((per < least ? least : per) + 127) / 128 * 128;
  return (int)(keys > max_keys ? (max_keys + 15) / 16 * 16 : keys);
}

int tree_attention(const TreeAttention& p, cudaStream_t stream) {
  if (p.num_segments <= 0 || p.rows <= 0) return 0;
  if (p.kv_heads <= 0 || p.q_heads <= 0 || p.q_heads % p.kv_heads != 0) return -2;
  if (p.max_keys <= 0 || p.max_len <= 0 || p.keys_per_split <= 0 || p.keys_per_split % 16 != 0) return -2;
  if ((long)p.num_segments * longest_segment(p) > 2147483647L || p.q_heads > 65535) return -2;
  const long splits = ((long)p.max_keys + p.keys_per_split - 1) / p.keys_per_split;
  if (splits > 65535) return -2;
  if (splits > 1 && (p.partial_o == nullptr || p.partial_ml == nullptr ||
                     (size_t)p.rows * p.q_heads * splits > p.partial_capacity || (reinterpret_cast<uintptr_t>(p.partial_o) & 15)))
    return -3;
  if (p.ld_q % 8 != 0 || p.ld_o % 8 != 0) return -2;
  if ((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.o) | reinterpret_cast<uintptr_t>(p.cache)) & 15)
    return -2;
  if (p.head_dim == 64) return p.quantized ? pick<64, true>(p, stream) : pick<64, false>(p, stream);
  if (p.head_dim == 128) return p.quantized ? pick<128, true>(p, stream) : pick<128, false>(p, stream);
  return -2;
}

}  // namespace foa
