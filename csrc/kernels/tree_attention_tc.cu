// Attention of chunks and drafted token trees over the paged cache on the tcgen05 tensor cores, for
// segments of more than 16 (token, head) rows a key/value head, 32 over codes; tree_attention.cu states
// the operator, the rule and takes the others.
//
// One CTA per (segment, key/value head, 256 rows, split of the keys), 128-key tiles:
// - Two softmax warpgroups, a thread a row, each with its own S and O in TMEM. With more than 128
//   rows they take a row tile each and share every key tile (A); with fewer they take the key tiles
//   in turn for the same rows (B) and join their sums at the end. So one of them works on its
//   scores while the tensor cores work for the other.
// - P replaces S in TMEM (16 bits, half the columns) and is the A operand of O += P V from there.
//   One thread issues every MMA, in an order that has P_w V before the next S_w.
// - Quantized pages: K's codes are the B operand of S as they lie in the cache (kind::f8f6f4); Q
//   enters as two E4M3 parts, hi = e4m3(q), lo = e4m3(q - hi), of rows scaled by a power of two to
//   [128, 256). Two parts hold BF16's 8 bits exactly; what lies below 2^-17 of the row's largest is
//   lost. V's codes become FP16 (exactly) in shared memory, by four helper warps, since weights in
//   E4M3 would lose a long tail of small probabilities; they write the keys' scales beside it.
// - BF16 pages: TMA brings K and V as the MMAs read them; the helpers only clear V rows past the
//   keys and values that are not finite.
// - Row maxima move when a tile exceeds them by 2^kSlack, the reference exponent of V's scales when the
//   largest that the row sees does; O is rescaled in TMEM then, which takes 3000 cycles beside 3700 of a
//   pair of tiles. With slack 2^4 that happened to a warp in every third tile early on; FP16 weights of
//   slack 2^8 still hold 2^-20 of the reference in full and 2^-30 at all. Both are part of the unit that
//   O and the row's sum are held in. So a seen key whose V scale is 2^20 times the others' costs those
//   bits, however small its weight; and since weights before V's scale are FP32 in units of V's
//   reference 2^e, those below 2^(e - 132) of the row's largest flush (e > 100: values near BF16's end).
// - Every wait is bounded; a timeout records a status and every role leaves through the same end.
//
// What bounds it: the chain of one warpgroup (128 scores a thread, P to TMEM, P V, the next S, which
// overwrites P), overlapped with the other one's; over codes the shared-memory pipe beside it, since
// every thread reads every key's two scales (a broadcast of 16 bytes takes as long as 512 bytes) while
// the MMAs read Q, K and V there. 24 trees of 32 to 64 nodes over 4.5 to 16.4 thousand keys, 32 x 8
// heads of 128: 432 us over codes, 326 over BF16 pages (604 TFLOP/s); 16 of 16 to 31 nodes: 117 and 112. A CTA holds its SM alone, so its start and
// end (5 and 6 us before both warpgroups converted Q and rows were written 128 bytes at a time) and
// unequal parts show in full: 462 and 128 us with parts cut every keys_per_split keys.
// An mbarrier wait costs the MMA thread 200 cycles even for a phase long complete, so what is surely
// there (K, V, scales) is waited for before what is not (P, S): 496 -> 462 us. Tried and slower, over
// the same trees with the kernel of that day: S in halves of 64 keys so that S overlaps the softmax
// (BF16 450 us for 336: N = 64 reads Q twice as often), K and V dequantized to FP16 by the helpers (530
// for 502), two MMA threads (527), scores in fragments of 16 x 256 bits (534), weights in a rolled loop
// of two passes (526).

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "decode_ops.cuh"
#include "launch.cuh"
#include "sm100.cuh"
#include "tmap.cuh"
#include "tree_split.cuh"

namespace foa {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kLeastExp = -90;  // least exponent of V's reference scale (sums stay below 2^127)
constexpr int kTile = 128;      // rows and keys of an MMA tile
constexpr int kThreads = 512;   // 8 softmax warps, MMA, loader, 4 helpers, 2 idle (whole warpgroups)
// Registers a thread: 128 at the launch (512 x 128 is the SM's file), moved between warpgroups.
constexpr int kSoftmaxRegs = 192, kOtherRegs = 64;
static_assert(256 * kSoftmaxRegs + 256 * kOtherRegs == kThreads * 128, "the shares are the launch's registers");
constexpr int kSlots = 4;       // key tiles whose scales are held

template <int D, bool kQ>
struct Cfg {
  // Weights are scaled by 2^kLift and may exceed the row's reference by 2^kSlack: below 2^15 over codes,
  // where V's scale, under 2 in the reference's units, still multiplies them before they are FP16.
  static constexpr float kLift = kQ ? 6.f : 0.f, kSlack = kQ ? 8.f : 14.f;
  static constexpr int kHalf = kTile * 128;            // a tile's 64 16-bit columns
  static constexpr int kTile16 = kTile * D * 2;        // a 16-bit tile
  static constexpr int kTile8 = kTile * D;             // an 8-bit tile
  static constexpr int kQTile = kTile16;               // (hi and lo, or BF16)
  static constexpr int kKStages = kQ ? 3 : 2;
  static constexpr int kKStage = kQ ? kTile8 : kTile16;
  static constexpr int kVStages = 2;
  static constexpr int kRaw = kQ ? 2 : 0;              // stages of V's codes
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = kOffQ + 2 * kQTile;
  static constexpr int kOffV = kOffK + kKStages * kKStage;
  static constexpr int kOffRaw = kOffV + kVStages * kTile16;
  static constexpr int kOffScale = kOffRaw + kRaw * kTile8;       // [slots][2 (K, V)][128], then [slots][4] maxima
  static constexpr int kOffRow = kOffScale + kSlots * (2 * kTile + 4) * 4;  // [2 (maximum, sum)][128]
  static constexpr int kOffBar = (kOffRow + 2 * kTile * 4 + 15) / 16 * 16;
  static constexpr int kBytes = kOffBar + 256 + 1024;  // 1 KiB of alignment slack
  // One CTA an SM: it holds all of TMEM.
  static constexpr int kSmem = kBytes < 120 * 1024 ? 120 * 1024 : kBytes;
  static constexpr int kColO = 2 * kTile;              // TMEM: S0, S1, then O0, O1 (128 columns apart)
};

struct Maps {
  CUtensorMap cache;  // codes: [pages][16][D] bytes; BF16: [pages * 16][D]
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
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
// Pairs of FP32 operations in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}"
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
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// tcgen05.wait::ld whose loaded values cannot be used before it.
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}

// Shared-memory descriptors: a K-major 8-bit operand in rows of `kRowBytes` (128 or 64, swizzled over
// as many bytes), and an MN-major 16-bit one (see the prefill kernel's layout: rows of 64 elements,
// groups of 64 `lbo` bytes apart).
template <int kRowBytes>
__device__ __forceinline__ uint64_t desc_k8(const void* smem) {
  uint64_t d = (smem_u32(smem) >> 4) & 0x3FFFull;
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)((8 * kRowBytes) >> 4) << 32;              // eight rows
  d |= (uint64_t)1 << 46;                                   // descriptor version of sm_100
  d |= (uint64_t)(kRowBytes == 128 ? 2 : 4) << 61;          // 128- or 64-byte swizzle
  return d;
}
__device__ __forceinline__ uint64_t desc_mn16(const void* smem, uint32_t lbo, uint32_t sbo) {
  uint64_t d = (smem_u32(smem) >> 4) & 0x3FFFull;
  d |= (uint64_t)((lbo >> 4) & 0x3FFF) << 16;
  d |= (uint64_t)((sbo >> 4) & 0x3FFF) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// D[tmem] (+)= A[tmem] * B[smem]^T for 16-bit operands.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Bounded waits of one thread and of a whole warp, in few instructions (sm100's with its clock, at
// twenty places beside five roles' code, pushed the softmax loop out of the instruction cache). A
// poll blocks for 1.4 us by itself, so the limit on their number is one of 3 s.
constexpr uint32_t kPolls = 1u << 21;
__device__ __forceinline__ bool gave_up(uint32_t polls, int* status, int site, volatile int* abort) {
  if (polls & 63u) return false;
  if (abort != nullptr && *abort) return true;
  if (polls < kPolls) return false;
  record_status(status, site);
  if (abort != nullptr) *abort = 1;
  return true;
}
__device__ __forceinline__ bool wait1(uint64_t* bar, uint32_t parity, int* status, int site, volatile int* abort) {
  const uint32_t at = smem_u32(bar);
  uint32_t polls = 0;
  while (!mbar_try_wait(at, parity))
    if (gave_up(++polls, status, site, abort)) return false;
  return true;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status, int site, volatile int* abort) {
  const uint32_t at = smem_u32(bar);
  uint32_t polls = 0;
  while (!__all_sync(0xffffffffu, mbar_try_wait(at, parity)))
    if (__any_sync(0xffffffffu, gave_up(++polls, status, site, abort))) return false;
  return true;
}

// 16-byte chunk `c` of row `r` in rows of kRowBytes as TMA swizzles them.
template <int kRowBytes>
__device__ __forceinline__ uint32_t at8(int r, int c) {
  return kRowBytes == 128 ? (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)) : (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}
// 16-byte chunk `c` (8 elements) of row `r` of a 16-bit tile: halves of 64 columns.
__device__ __forceinline__ uint32_t at16(int r, int c) {
  return (uint32_t)((c >> 3) * kTile * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ bool rows_fit(const TreeAttention& p, const Segment& s) {
  return s.row_start >= 0 && s.len > 0 && (long)s.row_start + s.len <= p.rows;
}
__device__ __forceinline__ bool segment_fits(const TreeAttention& p, const Segment& s) {
  return s.cached >= 0 && s.len <= p.max_len && (long)s.cached + s.len <= p.max_keys && s.table_start >= 0 &&
         s.nblocks >= 0 && (long)s.table_start + s.nblocks <= p.table_len &&
         (long)s.nblocks * 16 >= (long)s.cached + s.len;
}
__device__ __forceinline__ uint32_t mask_word(const TreeAttention& p, const Segment& s, int tok, int w) {
  if (p.mask == nullptr) {  // causal: bits 0 .. tok
    const int n = tok + 1 - 32 * w;
    return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1;
  }
  return w < p.mask_words ? p.mask[(long)(s.row_start + tok) * p.mask_words + w] : 0u;
}
// The keys of [key, key + 32) that row `tok` sees, below k1.
__device__ __forceinline__ uint32_t visible(const TreeAttention& p, const Segment& s, int tok, int key, int k1) {
  const int j = key - s.cached;  // place of the first among the appended rows
  uint32_t v;
  if (j <= -32) {
    v = ~0u;
  } else if (j < 0) {
    v = (1u << -j) - 1 | mask_word(p, s, tok, 0) << -j;
  } else {
    v = mask_word(p, s, tok, j >> 5) >> (j & 31);
    if (j & 31) v |= mask_word(p, s, tok, (j >> 5) + 1) << (32 - (j & 31));
  }
  const int left = k1 - key;
  return left <= 0 ? 0u : left >= 32 ? v : v & ((1u << left) - 1);
}

template <int D, bool kQ>
__global__ void __launch_bounds__(kThreads, 1)
    tree_attention_tc_kernel(const __grid_constant__ Maps maps, const TreeAttention p, int mtiles, int max_splits,
                             int num_pages) {
  using C = Cfg<D, kQ>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* q_full = bars + 0;
  uint64_t* k_full = bars + 1;    // [3]
  uint64_t* k_empty = bars + 4;   // [3]
  uint64_t* v_land = bars + 7;    // [2] TMA brought V (raw codes, or BF16)
  uint64_t* v_full = bars + 9;    // [2] V as the MMA reads it
  uint64_t* v_empty = bars + 11;  // [2]
  uint64_t* r_empty = bars + 13;  // [2] raw codes converted
  uint64_t* s_full = bars + 15;   // [2]
  uint64_t* p_full = bars + 17;   // [2]
  uint64_t* c_full = bars + 19;   // [4] the tile's scales are written
  uint64_t* done = bars + 23;     // every MMA completed
  uint64_t* joined = bars + 24;   // (B) the second warpgroup's sums are in shared memory
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 25);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* odd_v = reinterpret_cast<int*>(tmem_slot + 2);  // values or scales that are not finite were left out
  float* scales = reinterpret_cast<float*>(smem + C::kOffScale);
  int* exps = reinterpret_cast<int*>(scales + kSlots * 2 * kTile);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.q_heads / p.kv_heads;
  int item = blockIdx.x;
  const int mt = item % mtiles;
  item /= mtiles;
  const int kvh = item % p.kv_heads;
  const int split = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  const Segment seg = p.segments[item / p.kv_heads];
  if (seg.len == 0) return;
  if (!rows_fit(p, seg) || !segment_fits(p, seg)) {
    if (mt == 0 && split == 0) {
      if (threadIdx.x == 0) record_status(p.status, kBadArgument);
      if (rows_fit(p, seg))
        for (int r = 0; r < seg.len; ++r)
          for (int x = threadIdx.x; x < G * D; x += kThreads)
            p.o[(long)(seg.row_start + r) * p.ld_o + (long)kvh * G * D + x] = __float2bfloat16_rn(0.f);
    }
    return;
  }
  const int M = seg.len * G;
  const int m0 = mt * 2 * kTile;
  const int keys = seg.cached + seg.len;
  const Parts parts(keys, p.keys_per_split, true);
  const int nsplit = parts.count;
  if (m0 >= M || split >= nsplit) return;
  const int k0 = split * parts.width;
  const int k1 = min(keys, k0 + parts.width);
  const int ntiles = (k1 - k0 + kTile - 1) / kTile;
  const bool two = M - m0 > kTile;          // (A) two row tiles
  const int steps = two ? 2 * ntiles : ntiles;  // (warpgroup, key tile) pairs in turn
  const int32_t* table = p.table + seg.table_start;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 256);
    for (int s = 0; s < 3; ++s) {
      mbar_init(k_full + s, 1);
      mbar_init(k_empty + s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(v_land + s, 1);
      mbar_init(v_full + s, 128);
      mbar_init(v_empty + s, 1);
      mbar_init(r_empty + s, 128);
      mbar_init(s_full + s, 1);
      mbar_init(p_full + s, 128);
    }
    for (int s = 0; s < kSlots; ++s) mbar_init(c_full + s, 128);
    mbar_init(done, 1);
    mbar_init(joined, 128);
    *abort = 0;
    *odd_v = 0;
    fence_barrier_init();
    tma_prefetch_desc(&maps.cache);
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ------------------------------------------------------------------ softmax, a thread a row
    const int w = warp >> 2;                          // warpgroup
    const int row = threadIdx.x & 127;                // TMEM lane
    const int m = m0 + (two ? w * kTile : 0) + row;
    const bool real = m < M;
    const int tok = real ? m / G : 0, head = kvh * G + (real ? m % G : 0);
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_col = lane_base + w * kTile, o_col = lane_base + C::kColO + w * kTile;
    // Q: this row into its tile (half of its columns where both warpgroups share the tile).
    float c = fmaxf(fabsf(p.scale) * kLog2e, 1.2e-38f);  // (a negative scale turns q's sign)
    {
      const __nv_bfloat16* src = p.q + (long)(seg.row_start + tok) * p.ld_q + (long)head * D;
      const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
      const uint32_t dst = smem_u32(smem + C::kOffQ + (two ? w : 0) * C::kQTile);
      // Chunk x of n is this warpgroup's.
      auto mine = [&](int x, int n) { return two || (x >= n / 2) == (w == 1); };
      uint4 raw[D / 8];  // the whole row, in one trip to L2
#pragma unroll
      for (int ch = 0; ch < D / 8; ++ch) raw[ch] = real ? reinterpret_cast<const uint4*>(src)[ch] : make_uint4(0u, 0u, 0u, 0u);
      // The largest magnitude, as BF16 bits.
      uint32_t most = 0u;
#pragma unroll
      for (int ch = 0; ch < D / 8; ++ch) {
        const uint4 v = raw[ch];
        most = __vmaxu2(most, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
      }
      most = max(most >> 16, most & 0xffffu);
      // A row with an element that is not finite has no finite score: it is NaN throughout (E4M3 would
      // saturate an infinity, and of its products those of one sign would pass for keys that are not seen).
      const bool finite = most < 0x7f80u;
      if constexpr (kQ) {
        const int e = min(max((int)(most >> 7), 8), 254) - 127;
        const float down = finite ? __uint_as_float((uint32_t)(127 + 7 - e) << 23) : __int_as_float(0x7fffffff);  // 7 - e in [-120, 126]
        c = fmaxf(c * __uint_as_float((uint32_t)(127 - 7 + e) << 23), 1.2e-38f);
#pragma unroll
        for (int ch = 0; ch < D / 16; ++ch) {
          if (!mine(ch, D / 16)) continue;
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint4 v = raw[2 * ch + half];
            const uint32_t vw[4] = {v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip};
            uint16_t h[4], l[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float2 f = make_float2(bf16_lo(vw[x]) * down, bf16_hi(vw[x]) * down);
              h[x] = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
              const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(h[x], __NV_E4M3);
              const float2 hf = __half22float2(*reinterpret_cast<const __half2*>(&hr));
              l[x] = __nv_cvt_float2_to_fp8x2(make_float2(f.x - hf.x, f.y - hf.y), __NV_SATFINITE, __NV_E4M3);
            }
            hi[2 * half] = h[0] | (uint32_t)h[1] << 16;
            hi[2 * half + 1] = h[2] | (uint32_t)h[3] << 16;
            lo[2 * half] = l[0] | (uint32_t)l[1] << 16;
            lo[2 * half + 1] = l[2] | (uint32_t)l[3] << 16;
          }
          sts128(dst + at8<D>(row, ch), make_uint4(hi[0], hi[1], hi[2], hi[3]));
          sts128(dst + C::kTile8 + at8<D>(row, ch), make_uint4(lo[0], lo[1], lo[2], lo[3]));
        }
      } else {
#pragma unroll
        for (int ch = 0; ch < D / 8; ++ch) {
          if (!mine(ch, D / 8)) continue;
          const uint4 v = raw[ch];
          const uint32_t nan = finite ? 0u : 0x7fff7fffu;
          sts128(dst + at16(row, ch), make_uint4(v.x ^ flip | nan, v.y ^ flip | nan, v.z ^ flip | nan, v.w ^ flip | nan));
        }
      }
      fence_proxy_async();
      mbar_arrive(q_full);
    }
    const bool idle = !__any_sync(0xffffffffu, real);  // none of the warp's rows counts
    float top = -INFINITY, sum = 0.f;
    int v_exp = kQ ? kLeastExp : 0;  // O and the sums are in units of 2^(top + v_exp - kLift)
    bool ok = true;
    int i = 0;
    for (int n = w; n < steps; n += 2, ++i) {
      const int j = two ? i : n, kb = k0 + j * kTile;
      const int slot = j % kSlots;
      // (A wait costs some 200 cycles even for what is there: the last to come is waited for last.)
      if ((kQ && !warp_wait(c_full + slot, (j / kSlots) & 1, p.status, kTimeoutTmemFull, abort)) ||
          !warp_wait(s_full + w, i & 1, p.status, kTimeoutTmemFull, abort)) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (!idle) {
        const float* sk = scales + slot * 2 * kTile;
        const bool inner = kb + kTile <= min(seg.cached, k1);
        int e = v_exp;
        if constexpr (kQ) {
          const int4 warps = *reinterpret_cast<const int4*>(exps + slot * 4);
          e = max(v_exp, min(max(max(warps.x, warps.y), max(warps.z, warps.w)) >> 23, 253) - 127);
        }
        // The row's 128 scores stay in registers: K's scales, the mask and the largest as they arrive
        // (c is positive, so the largest needs no scaling), then the weights.
        uint32_t r[kTile];
        float mx0 = -INFINITY, mx1 = -INFINITY;
        tmem_ld_32x32b_x32(s_col, *reinterpret_cast<uint32_t(*)[32]>(r));
#pragma unroll
        for (int c0 = 0; c0 < kTile; c0 += 32) {
          tmem_wait16(*reinterpret_cast<uint32_t(*)[16]>(r + c0));
          tmem_wait16(*reinterpret_cast<uint32_t(*)[16]>(r + c0 + 16));
          if (c0 + 32 < kTile) tmem_ld_32x32b_x32(s_col + c0 + 32, *reinterpret_cast<uint32_t(*)[32]>(r + (c0 + 32) % kTile));
#pragma unroll
          for (int x = c0; x < c0 + 32; x += 4) {
            float2 a = make_float2(__uint_as_float(r[x]), __uint_as_float(r[x + 1]));
            float2 b = make_float2(__uint_as_float(r[x + 2]), __uint_as_float(r[x + 3]));
            if constexpr (kQ) {
              const float4 k4 = *reinterpret_cast<const float4*>(sk + x);
              a = mul2(a, make_float2(k4.x, k4.y));
              b = mul2(b, make_float2(k4.z, k4.w));
              r[x] = __float_as_uint(a.x);
              r[x + 1] = __float_as_uint(a.y);
              r[x + 2] = __float_as_uint(b.x);
              r[x + 3] = __float_as_uint(b.y);
            }
            mx0 = fmaxf(mx0, fmaxf(a.x, a.y));
            mx1 = fmaxf(mx1, fmaxf(b.x, b.y));
          }
        }
        if (!inner) {
          mx0 = mx1 = -INFINITY;
          // V's reference is of the scales that the row sees: a drafted node's may be far larger.
          float most = 0.f;
#pragma unroll
          for (int c0 = 0; c0 < kTile; c0 += 32) {
            const uint32_t seen = visible(p, seg, tok, kb + c0, k1);
#pragma unroll
            for (int x = 0; x < 32; ++x) {
              const float t = seen >> x & 1u ? __uint_as_float(r[c0 + x]) : -INFINITY;
              r[c0 + x] = __float_as_uint(t);
              mx0 = fmaxf(mx0, t);
              if constexpr (kQ) most = fmaxf(most, seen >> x & 1u ? sk[kTile + c0 + x] : 0.f);
            }
          }
          if constexpr (kQ) e = max(v_exp, min((int)(__float_as_uint(most) >> 23), 253) - 127);
          __syncwarp();
        }
        float mx = fmaxf(mx0, mx1), f = 1.f;
        if (mx > -INFINITY) mx *= c;
        if (mx > top + C::kSlack) {
          f = top == -INFINITY ? 0.f : ex2(top - mx);
          top = mx;
        }
        if (e != v_exp) {
          f *= ex2((float)(v_exp - e));
          v_exp = e;
        }
        sum *= f;
        // (S_w of this step follows P_w V of the one before: O may be changed.)
        if (i > 0 && __any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += 16) {
            uint32_t y[16];
            tmem_ld_32x32b_x16(o_col + c0, y);
            tmem_wait16(y);
#pragma unroll
            for (int x = 0; x < 16; ++x) y[x] = __float_as_uint(__uint_as_float(y[x]) * f);
            tmem_st_32x32b_x16(o_col + c0, y);
          }
        }
        const float z = top == -INFINITY ? 0.f : top + (float)v_exp - C::kLift;
        const float2 c2 = make_float2(c, c), z2 = make_float2(-z, -z);
        float2 acc0 = make_float2(0.f, 0.f), acc1 = acc0;
        // P takes the columns of S.
#pragma unroll
        for (int c0 = 0; c0 < kTile; c0 += 32) {
          uint32_t out[16];
#pragma unroll
          for (int x = 0; x < 32; x += 4) {
            float2 a = fma2(make_float2(__uint_as_float(r[c0 + x]), __uint_as_float(r[c0 + x + 1])), c2, z2);
            float2 b = fma2(make_float2(__uint_as_float(r[c0 + x + 2]), __uint_as_float(r[c0 + x + 3])), c2, z2);
            a = make_float2(ex2(a.x), ex2(a.y));
            b = make_float2(ex2(b.x), ex2(b.y));
            acc0 = add2(acc0, a);
            acc1 = add2(acc1, b);
            if constexpr (kQ) {
              const float4 v4 = *reinterpret_cast<const float4*>(sk + kTile + c0 + x);
              a = mul2(a, make_float2(v4.x, v4.y));
              b = mul2(b, make_float2(v4.z, v4.w));
              out[x / 2] = pack_f16x2(a.x, a.y);
              out[x / 2 + 1] = pack_f16x2(b.x, b.y);
            } else {
              out[x / 2] = pack_bf16x2(a.x, a.y);
              out[x / 2 + 1] = pack_bf16x2(b.x, b.y);
            }
          }
          tmem_st_32x32b_x16(s_col + c0 / 2, out);
        }
        sum += (acc0.x + acc0.y) + (acc1.x + acc1.y);
        tmem_st_wait();
      }
      tc_fence_before();
      mbar_arrive(p_full + w);
    }
    // Every MMA done, O holds the sums (none for a warpgroup without a step).
    bool fine = ok && warp_wait(done, 0, p.status, kTimeoutTmemFull, abort);
    tc_fence_after();
    top += (float)v_exp;
    float* row_top = reinterpret_cast<float*>(smem + C::kOffRow);
    float* row_sum = row_top + kTile;
    // (B) The second warpgroup's sums go through the key and value stages, free by now.
    float* other = reinterpret_cast<float*>(smem + C::kOffK);
    static_assert(kTile * D * 4 <= C::kOffScale - C::kOffK, "the join fits the stages");
    static_assert(8 * 4096 <= C::kOffK - C::kOffQ, "the warps' boxes fit Q's tiles");
    auto other_at = [&](int ch) { return other + row * D + ((ch ^ row) & (D / 4 - 1)) * 4; };  // 4 columns
    if (!two && w == 1) {
      if (fine) {
        row_top[row] = i > 0 ? top : -INFINITY;
        row_sum[row] = sum;
        if (i > 0 && !idle) {
#pragma unroll
          for (int c0 = 0; c0 < D; c0 += 32) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(o_col + c0, r);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 32; x += 4)
              *reinterpret_cast<float4*>(other_at((c0 + x) / 4)) =
                  make_float4(__uint_as_float(r[x]), __uint_as_float(r[x + 1]), __uint_as_float(r[x + 2]),
                              __uint_as_float(r[x + 3]));
          }
        }
      }
      mbar_arrive(joined);
    } else {
      if (!two && fine) fine = warp_wait(joined, 0, p.status, kTimeoutTmemFull, abort);
      if (fine && !idle) {
        float f0 = 1.f, f1 = 0.f;
        if (!two) {
          const float t1 = row_top[row], both = fmaxf(top, t1);
          f0 = top == -INFINITY ? 0.f : ex2(top - both);
          f1 = t1 == -INFINITY ? 0.f : ex2(t1 - both);
          sum = sum * f0 + row_sum[row] * f1;
          top = both;
        }
        const bool fix = *reinterpret_cast<volatile int*>(odd_v) != 0;
        // (Scores that are all NaN leave the maximum of a row that sees nothing, and a sum that is NaN.)
        const float norm = nsplit > 1 ? 1.f : top == -INFINITY && sum == 0.f ? 0.f : 1.f / sum;
        const long at = (long)(seg.row_start + tok);
        const long idx = (at * p.q_heads + head) * max_splits + split;
        __nv_bfloat16* dst = p.o + at * p.ld_o + (long)head * D;
        float* part = p.partial_o + idx * D;
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t r[32];
          __syncwarp();
          tmem_ld_32x32b_x32(o_col + c0, r);
          tmem_ld_wait();
          float v[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) v[x] = __uint_as_float(r[x]) * f0;
          if (f1 > 0.f) {
#pragma unroll
            for (int x = 0; x < 32; x += 4) {
              const float4 y = *reinterpret_cast<const float4*>(other_at((c0 + x) / 4));
              v[x] = fmaf(y.x, f1, v[x]);
              v[x + 1] = fmaf(y.y, f1, v[x + 1]);
              v[x + 2] = fmaf(y.z, f1, v[x + 2]);
              v[x + 3] = fmaf(y.w, f1, v[x + 3]);
            }
          }
          if (real && fix) {
            const uint8_t* cache = static_cast<const uint8_t*>(p.cache);
            const long pb = kQ ? 16L * D + kScaleBytes : 32L * D;
            for (int a = max(0, k0 - seg.cached); a < min(seg.len, k1 - seg.cached); ++a) {
              if (!(mask_word(p, seg, tok, a >> 5) >> (a & 31) & 1u)) continue;
              const int key = seg.cached + a, id = table[key >> 4];
              if (id < 0 || id >= p.cache_blocks) continue;
              const uint8_t* vp = cache + ((long)id * 2 * p.kv_heads + p.kv_heads + kvh) * pb + (long)(key & 15) * D * (kQ ? 1 : 2);
              // A value, or all of them by their scale: left out of the products, added where seen.
              const float s = kQ ? *reinterpret_cast<const float*>(vp + (16 - (key & 15)) * D + (key & 15) * 4) : 1.f;
              const bool all = !(fabsf(s) < INFINITY);
#pragma unroll
              for (int x = 0; x < 32; ++x) {
                if constexpr (kQ) {
                  if (all || (vp[c0 + x] & 0x7fu) == 0x7fu)
                    v[x] += __half2float(__half(__nv_cvt_fp8_to_halfraw(vp[c0 + x], __NV_E4M3))) * s;
                } else {
                  const float y = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(vp)[c0 + x]);
                  if (!(fabsf(y) < INFINITY)) v[x] += y;
                }
              }
            }
          }
          if (real && nsplit == 1) {
#pragma unroll
            for (int x = 0; x < 32; x += 8)
              *reinterpret_cast<uint4*>(dst + c0 + x) =
                  make_uint4(pack_bf16x2(v[x] * norm, v[x + 1] * norm), pack_bf16x2(v[x + 2] * norm, v[x + 3] * norm),
                             pack_bf16x2(v[x + 4] * norm, v[x + 5] * norm), pack_bf16x2(v[x + 6] * norm, v[x + 7] * norm));
          } else if (nsplit > 1) {
            // Through Q's tile, free by now, so that eight lanes write a row's 128 bytes.
            const uint32_t box = smem_u32(smem + C::kOffQ) + warp * 4096;
#pragma unroll
            for (int x = 0; x < 8; ++x)
              sts128(box + lane * 128 + ((x ^ lane & 7) << 4),
                     make_uint4(__float_as_uint(v[4 * x]), __float_as_uint(v[4 * x + 1]), __float_as_uint(v[4 * x + 2]),
                                __float_as_uint(v[4 * x + 3])));
            __syncwarp();
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const int r1 = 4 * x + (lane >> 3);
              float* to = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, real ? reinterpret_cast<uint64_t>(part) : 0ull, r1));
              const uint4 y = lds128(box + r1 * 128 + (((lane & 7) ^ (r1 & 7)) << 4));
              if (to != nullptr) *reinterpret_cast<uint4*>(to + c0 + 4 * (lane & 7)) = y;
            }
          }
        }
        if (real && nsplit > 1) p.partial_ml[idx] = make_float2(top, sum);
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 9) {
      // ------------------------------------------------------------------ loader, a lane a page
      auto page_of = [&](int j) -> int {  // K's page index of this lane's page of tile j, or one past the last
        const int b = k0 / 16 + j * 8 + lane;
        if (j >= ntiles || lane >= 8 || b * 16 >= k1) return num_pages;
        const int id = table[b];
        if (id < 0 || id >= p.cache_blocks) {
          record_status(p.status, kBadIndex);  // reads as zeros
          return num_pages;
        }
        return id * 2 * p.kv_heads + kvh;
      };
      auto load = [&](uint8_t* dst, uint64_t* bar, int page) {
        if (lane == 0) mbar_arrive_expect_tx(bar, C::kKStage);
        __syncwarp();
        if (lane < 8) {
          if constexpr (kQ) {
            tma_load_3d(dst + lane * 16 * D, &maps.cache, bar, 0, 0, page);
          } else {
#pragma unroll
            for (int h = 0; h < D / 64; ++h)
              tma_load_2d(dst + h * C::kHalf + lane * 2048, &maps.cache, bar, h * 64, page * 16);
          }
        }
        __syncwarp();
      };
      int got_k = 0, got_v = 0;
      auto load_k = [&](int j, int page) {
        const int ks = j % C::kKStages;
        if (j >= C::kKStages && !warp_wait(k_empty + ks, (j / C::kKStages + 1) & 1, p.status, kTimeoutSmemEmpty, abort)) return false;
        load(smem + C::kOffK + ks * C::kKStage, k_full + ks, page);
        ++got_k;
        return true;
      };
      // K runs two tiles ahead of V: the S of tile j + 2 is issued behind the P V of tile j.
      int page0 = page_of(0), page1 = page_of(1), page2 = page_of(2);
      load_k(0, page0);
      if (ntiles > 1) load_k(1, page1);
      for (int j = 0; j < ntiles; ++j) {
        const int vs = j & 1;
        if (j >= 2 && !warp_wait((kQ ? r_empty : v_empty) + vs, (j / 2 + 1) & 1, p.status, kTimeoutSmemEmpty, abort)) break;
        load(smem + (kQ ? C::kOffRaw + vs * C::kTile8 : C::kOffV + vs * C::kTile16), v_land + vs,
             page0 == num_pages ? num_pages : page0 + p.kv_heads);
        ++got_v;
        if (j + 2 < ntiles && !load_k(j + 2, page2)) break;
        page0 = page1;
        page1 = page2;
        page2 = page_of(j + 3);
      }
      // Let the loads in flight land before the CTA may exit (an abort stops the loop early).
      for (int j = got_k > C::kKStages ? got_k - C::kKStages : 0; j < got_k; ++j)
        warp_wait(k_full + j % C::kKStages, (j / C::kKStages) & 1, p.status, kTimeoutDrain, nullptr);
      for (int j = got_v > 2 ? got_v - 2 : 0; j < got_v; ++j)
        warp_wait(v_land + (j & 1), (j / 2) & 1, p.status, kTimeoutDrain, nullptr);
    } else if (warp == 8) {
      // ------------------------------------------------------------------ MMA issuer
      if (elect_one()) {
        constexpr uint32_t idesc_s = kQ ? idesc_e4m3_f32(kTile, kTile) : idesc_bf16_f32(kTile, kTile);
        // P V: FP16 (format 0) over codes, BF16 else; B (V) MN-major.
        constexpr uint32_t idesc_o = (kQ ? idesc_bf16_f32(kTile, D) & ~((1u << 7) | (1u << 10)) : idesc_bf16_f32(kTile, D)) | (1u << 16);
        const bool ok = wait1(q_full, 0, p.status, kTimeoutTmemFull, abort);
        auto scores = [&](int n) {
          const int w = n & 1, j = two ? n >> 1 : n, ks = j % C::kKStages;
          // (Descriptors of a tile's steps differ in their address field alone.)
          const uint8_t* kt = smem + C::kOffK + ks * C::kKStage;
          const uint8_t* qt = smem + C::kOffQ + (two ? w : 0) * C::kQTile;
          const uint64_t kd = kQ ? desc_k8<D>(kt) : sdesc_kmajor_sw128(kt);
          const uint64_t qd = kQ ? desc_k8<D>(qt) : sdesc_kmajor_sw128(qt);
          if constexpr (kQ) {
#pragma unroll
            for (int part = 0; part < 2; ++part)
#pragma unroll
              for (int kk = 0; kk < D / 32; ++kk)
                mma_e4m3(tmem + w * kTile, qd + ((part * C::kTile8 + kk * 32) >> 4), kd + (kk * 32 >> 4), idesc_s,
                         part > 0 || kk > 0 ? 1u : 0u);
          } else {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const int step = ((kk >> 2) * C::kHalf + (kk & 3) * 32) >> 4;
              mma_bf16(tmem + w * kTile, qd + step, kd + step, idesc_s, kk > 0 ? 1u : 0u);
            }
          }
          mma_commit(s_full + w);
          if (!two || w == 1) mma_commit(k_empty + ks);
        };
        for (int n = -2; ok && n < steps; ++n) {
          const int w = n & 1, jk = two ? (n + 2) >> 1 : n + 2;
          if (n + 2 < steps && !wait1(k_full + jk % C::kKStages, (jk / C::kKStages) & 1, p.status, kTimeoutTmaFull, abort)) break;
          if (n >= 0) {
            const int j = two ? n >> 1 : n, vs = j & 1;
            if (!wait1(v_full + vs, (j / 2) & 1, p.status, kTimeoutTmaFull, abort) ||
                !wait1(p_full + w, (n >> 1) & 1, p.status, kTimeoutTmemFull, abort))
              break;
            tc_fence_after();
            const uint64_t vd = desc_mn16(smem + C::kOffV + vs * C::kTile16, C::kHalf, 1024);
#pragma unroll
            for (int kk = 0; kk < kTile / 16; ++kk)
              mma_f16_ts(tmem + C::kColO + w * kTile, tmem + w * kTile + kk * 8, vd + (kk * 2048 >> 4), idesc_o,
                         n >= 2 || kk > 0 ? 1u : 0u);
            if (!two || w == 1) mma_commit(v_empty + vs);
          }
          if (n + 2 < steps) scores(n + 2);
        }
        // No MMA may still write TMEM when it is read or freed (an abort can leave some in flight).
        mma_commit(done);
        wait1(done, 0, p.status, kTimeoutDrain, nullptr);
      }
    } else if (warp < 14) {
      // ------------------------------------------------------------------ helpers
      const int i = threadIdx.x - 320;  // 0 .. 127: a key of the tile
      const uint8_t* cache = static_cast<const uint8_t*>(p.cache);
      float ks = 0.f, vs_ = 0.f;
      auto fetch = [&](int j) {  // the scales of this thread's key of tile j
        ks = vs_ = 0.f;
        const int key = k0 + j * kTile + i;
        if (j >= ntiles || key >= k1) return;
        const int id = table[key >> 4];
        if (id < 0 || id >= p.cache_blocks) return;
        const long pb = 16L * D + kScaleBytes;
        const uint8_t* at = cache + ((long)id * 2 * p.kv_heads + kvh) * pb + 16 * D + (key & 15) * 4;
        ks = __ldg(reinterpret_cast<const float*>(at));
        vs_ = __ldg(reinterpret_cast<const float*>(at + p.kv_heads * pb));
      };
      if constexpr (kQ) fetch(0);
      bool odd = false;
      for (int j = 0; j < ntiles; ++j) {
        const int vs = j & 1, kb = k0 + j * kTile;
        const bool inner = kb + kTile <= min(seg.cached, k1);
        uint8_t* vt = smem + C::kOffV + vs * C::kTile16;
        if constexpr (kQ) {
          // The V stage's last reader (tile j - 2) is done, and with it the slot's (tile j - 4).
          if (j >= 2 && !warp_wait(v_empty + vs, (j / 2 + 1) & 1, p.status, kTimeoutTmemEmpty, abort)) break;
          const int slot = j % kSlots;
          float* sk = scales + slot * 2 * kTile;
          // (Not even a weight of zero may meet an appended row's scale that is not finite.)
          if (kb + i >= seg.cached && !(fabsf(vs_) < INFINITY)) {
            vs_ = 0.f;
            odd = true;
          }
          const uint32_t mine = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(vs_, 0.f)));
          sk[i] = ks;
          sk[kTile + i] = vs_;
          // Each warp's largest V scale, by its bits (scales are not negative).
          if (lane == 0) exps[slot * 4 + (i >> 5)] = (int)mine;
          mbar_arrive(c_full + slot);
          fetch(j + 1);
        }
        if (!warp_wait(v_land + vs, (j / 2) & 1, p.status, kTimeoutTmaFull, abort)) break;
        if constexpr (kQ) {
          const uint32_t raw = smem_u32(smem + C::kOffRaw + vs * C::kTile8);
          const uint32_t dst = smem_u32(vt);
          constexpr int kCh = D / 16;
          auto convert = [&](const uint32_t (&w)[4], int key, int rc) {
            const uint4 lo = make_uint4(e4m3x2_f16x2(w[0]), e4m3x2_f16x2_hi(w[0]), e4m3x2_f16x2(w[1]), e4m3x2_f16x2_hi(w[1]));
            const uint4 hi = make_uint4(e4m3x2_f16x2(w[2]), e4m3x2_f16x2_hi(w[2]), e4m3x2_f16x2(w[3]), e4m3x2_f16x2_hi(w[3]));
            // Lanes of the upper half of the columns store their chunks in the other order, so
            // that a store's lanes fall in different banks.
            const bool swap = kCh > 4 && rc >= 4;
            sts128(dst + at16(key, 2 * rc + (swap ? 1 : 0)), swap ? hi : lo);
            sts128(dst + at16(key, 2 * rc + (swap ? 0 : 1)), swap ? lo : hi);
          };
          if (inner) {
#pragma unroll 2
            for (int u = i; u < kTile * kCh; u += 128) {
              const uint4 x = lds128(raw + at8<D>(u / kCh, u % kCh));
              const uint32_t w[4] = {x.x, x.y, x.z, x.w};
              convert(w, u / kCh, u % kCh);
            }
          } else {
#pragma unroll 1
            for (int u = i; u < kTile * kCh; u += 128) {
              const int key = u / kCh;
              const uint4 x = lds128(raw + at8<D>(key, u % kCh));
              uint32_t w[4] = {x.x, x.y, x.z, x.w};
              if (kb + key >= seg.cached) {
                // A product with a zero weight must stay zero.
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  if (kb + key >= k1) w[e] = 0u;
#pragma unroll 1
                  for (int y = 0; y < 32; y += 8)
                    if ((w[e] >> y & 0x7fu) == 0x7fu) {
                      w[e] &= ~(0xffu << y);
                      odd = true;
                    }
                }
              }
              convert(w, key, u % kCh);
            }
          }
          mbar_arrive(r_empty + vs);
        } else if (!inner) {
          const uint32_t dst = smem_u32(vt);
          constexpr int kCh = D / 8;
          for (int u = i; u < kTile * kCh; u += 128) {
            const int key = u / kCh;
            if (kb + key < seg.cached) continue;
            const uint32_t a = dst + at16(key, u % kCh);
            uint4 x = lds128(a);
            uint32_t w[4] = {x.x, x.y, x.z, x.w};
            bool change = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t bad = 0u;
              if (kb + key >= k1) {
                bad = ~0u;
              } else {
                if ((w[e] & 0x7f80u) == 0x7f80u) bad |= 0xffffu;
                if ((w[e] & 0x7f800000u) == 0x7f800000u) bad |= 0xffff0000u;
                if (bad != 0u) odd = true;
              }
              change = change || bad != 0u;
              w[e] &= ~bad;
            }
            if (change) sts128(a, make_uint4(w[0], w[1], w[2], w[3]));
          }
        }
        if (odd) atomicExch(odd_v, 1);
        fence_proxy_async();
        mbar_arrive(v_full + vs);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Codes: [pages][16 rows][D] bytes, a page's rows together and its scales behind them.
bool encode_codes(CUtensorMap* map, const void* base, long pages, int d) {
  auto fn = tmap_encoder();
  if (fn == nullptr) return false;
  cuuint64_t dims[3] = {(cuuint64_t)d, 16, (cuuint64_t)pages};
  cuuint64_t strides[2] = {(cuuint64_t)d, (cuuint64_t)quantized_page_bytes(d)};
  cuuint32_t box[3] = {(cuuint32_t)d, 16, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool kQ>
int launch(const TreeAttention& p, int splits, cudaStream_t stream) {
  using C = Cfg<D, kQ>;
  static_assert(C::kSmem <= 232448, "shared memory");
  const int G = p.q_heads / p.kv_heads;
  const long mtiles = ((long)longest_segment(p) * G + 2 * kTile - 1) / (2 * kTile);
  const long ctas = mtiles * p.kv_heads * p.num_segments;
  if (ctas > 2147483647L) return -2;
  const long pages = p.cache_blocks * 2 * p.kv_heads;
  Maps maps;
  if (kQ ? !encode_codes(&maps.cache, p.cache, pages, D)
         : !encode_tmap_2d(&maps.cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.cache, pages * 16, D, D, 16, 64,
                           CU_TENSOR_MAP_SWIZZLE_128B))
    return -4;
  const auto kernel = tree_attention_tc_kernel<D, kQ>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess) return -5;
    configured[dev & 63] = true;
  }
  return launch_pdl(kernel, dim3((unsigned)ctas, splits), dim3(kThreads), C::kSmem, stream, maps, p, (int)mtiles, splits,
                    (int)pages) == cudaSuccess
             ? 0
             : -5;
}

}  // namespace

bool tree_attention_tc_supported(const TreeAttention& p) {
  const long pages = p.cache_blocks * 2 * p.kv_heads;
  return p.cache_blocks > 0 && pages * 16 < (1L << 31) - 16 && (p.head_dim == 64 || p.head_dim == 128);
}

int tree_attention_tc(const TreeAttention& p, cudaStream_t stream) {
  if (!tree_attention_tc_supported(p)) return -2;
  const int splits = (p.max_keys + p.keys_per_split - 1) / p.keys_per_split;
  if (p.head_dim == 64) return p.quantized ? launch<64, true>(p, splits, stream) : launch<64, false>(p, splits, stream);
  return p.quantized ? launch<128, true>(p, splits, stream) : launch<128, false>(p, splits, stream);
}

}  // namespace foa
