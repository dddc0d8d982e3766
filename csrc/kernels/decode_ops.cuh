// Host-visible interface of the decode-step operators over the quantized KV cache: the quantizing
// store, attention of decode rows, chunks and drafted token trees, and constrained greedy logits.
//
// A quantized cache is pages of bytes [blocks][2 (K, V)][kv_heads][16 * d + 64]: a block's 16 rows
// of one key/value head as E4M3 codes [16][d], then their 16 FP32 scales; an element's value is
// code * scale.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "attention.cuh"

namespace foa {

constexpr int kScaleBytes = 64;  // 16 FP32 scales behind a page's codes
inline long quantized_page_bytes(int head_dim) { return 16L * head_dim + kScaleBytes; }

// Per-head norm (optional), rotation and paged store of packed q/k/v rows
// [rows][(q_heads + 2 kv_heads) * head_dim].
struct KvStore {
  const __nv_bfloat16* qkv = nullptr;
  long ld_qkv = 0;
  int rows = 0, q_heads = 0, kv_heads = 0, head_dim = 128;
  const __nv_bfloat16* q_norm = nullptr;  // [head_dim] or null
  const __nv_bfloat16* k_norm = nullptr;
  float eps = 0.f;
  const int32_t* positions = nullptr;
  const float* inv_freq = nullptr;  // [rotary_dim / 2]
  float attention_factor = 1.f;
  int rotary_dim = 128;  // leading elements of a head that turn (a multiple of 16)
  int interleaved = 0;   // pairs (2j, 2j + 1) instead of (j, j + rotary_dim / 2)
  __nv_bfloat16* q_out = nullptr;  // [rows][q_heads][head_dim]
  void* cache = nullptr;           // quantized pages, or BF16 pages when quantized == 0
  int quantized = 1;
  const int32_t* slots = nullptr;  // negative: the row is not cached
  long cache_slots = 0;
  int* status = nullptr;
};
int kv_store(const KvStore& args, cudaStream_t stream);

// Attention of every segment's rows over its history (all of it visible) and the segment's own
// rows (visible by `mask`, or causally without one).
struct TreeAttention {
  const __nv_bfloat16* q = nullptr;  // [rows] rows of q_heads * head_dim, ld_q apart
  long ld_q = 0;
  __nv_bfloat16* o = nullptr;
  long ld_o = 0;
  int rows = 0;
  const void* cache = nullptr;
  int quantized = 0;
  long cache_blocks = 0;
  const int32_t* table = nullptr;
  long table_len = 0;
  const Segment* segments = nullptr;
  int num_segments = 0;
  int q_heads = 0, kv_heads = 0, head_dim = 128;
  float scale = 0.f;
  const uint32_t* mask = nullptr;  // [rows][mask_words]: bit j of row i, row i sees appended row j
  int mask_words = 0;
  int max_keys = 0;        // bounds every segment's cached + len
  int max_len = 0;         // bounds every segment's len
  int keys_per_split = 0;  // a multiple of 16
  // Partial outputs of the splits (unnormalized sums, and (maximum, sum) pairs) when
  // max_keys > keys_per_split: rows * q_heads * splits of each.
  float* partial_o = nullptr;
  float2* partial_ml = nullptr;
  size_t partial_capacity = 0;
  int* status = nullptr;
};
int tree_attention(const TreeAttention& args, cudaStream_t stream);
// What the grids are laid out for: max_len may be a bound far above any segment that fits the rows.
inline int longest_segment(const TreeAttention& args) { return args.max_len < args.rows ? args.max_len : args.rows; }
// The split width that tree_attention works best with for these sizes.
int tree_attention_split(int num_segments, int q_heads, int kv_heads, int head_dim, int quantized, int max_keys,
                         int max_len);
// The tcgen05 form, for segments of more (token, head) rows a key/value head than 16 (BF16 pages) or 32
// (codes): 256 rows a CTA, so the fewest fill an eighth of its tiles, and still come out ahead.
bool tree_attention_tc_supported(const TreeAttention& args);
int tree_attention_tc(const TreeAttention& args, cudaStream_t stream);

// A list of tokens per row: row r's are tokens[starts[r] .. starts[r + 1]).
struct TokenLists {
  const int32_t* tokens = nullptr;
  const int32_t* starts = nullptr;
  int count = 0;  // tokens of all lists
};

// Penalties, biases and an allowed-token mask on rows of logits, and each row's first maximum.
struct LogitsArgs {
  const void* logits = nullptr;  // FP32, or BF16 when half != 0
  void* out = nullptr;           // adjusted logits in the same type (may be `logits`), or null
  int half = 0;
  long ld = 0, ldo = 0;
  int rows = 0, vocab = 0;
  TokenLists prompt, output, bias;
  const float* bias_values = nullptr;
  const float* repetition = nullptr;  // [rows] or null
  const float* frequency = nullptr;
  const float* presence = nullptr;
  const uint32_t* allowed = nullptr;  // [rows][ld_allowed] words, bit t % 32 of word t / 32
  long ld_allowed = 0;
  int32_t* index = nullptr;  // -1 where no token is left
  float* value = nullptr;
  float2* partial = nullptr;  // rows * logits_slices(vocab), when that is more than one a row
  size_t partial_count = 0;
  int* status = nullptr;
};
int logits_slices(int vocab);
int process_logits(const LogitsArgs& args, cudaStream_t stream);

}  // namespace foa
