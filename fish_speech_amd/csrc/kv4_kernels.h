// kv4_kernels.h -- launch wrappers of the 4-bit K/V cache kernels (kv4.hip).
#pragma once
#include "common.h"
#include "dualar_kernels.h"   // KV_PAGE

namespace fmi {

// One layer's cache.  A page holds KV_PAGE tokens: [n_kv_head][K, V] blocks of kv4_block_bytes(D), a block =
// [KV_PAGE][D / 2] code bytes (value 2 i in the low nibble of byte i, value 2 i + 1 in the high one) followed by
// [KV_PAGE][D / 32] scale bytes (2^(b - 127); 255 = the 32 values are NaN).
struct Kv4Cache {
  uint8_t* pool;
  const int32_t* block_table;   // [slots][max_pages]; an id outside [0, n_pages) = no page
  int n_pages, KVH, D, n_slots, max_pages;
};

__host__ __device__ constexpr int kv4_block_bytes(int D) { return KV_PAGE * (D / 2 + D / 32); }

struct Kv4AppendArgs {
  Kv4Cache c;
  const bf16_t *q, *k, *v;                  // rows of [heads][D]; q may be nullptr
  int64_t q_stride, k_stride, v_stride;     // elements between rows
  bf16_t* q_out;                            // [rows][H][D], q_out_stride elements between rows
  int64_t q_out_stride;
  int H;                                    // query heads (0 when q == nullptr)
  const bf16_t *q_norm, *k_norm;            // head RMSNorm weights [D] or nullptr
  double eps;
  const bf16_t* rope;                       // [rope_len][rot / 2][2] (cos, sin) or nullptr
  int rope_len, rot, half;
  const int32_t *row_seq, *row_pos;
  // launch_kv4_step only: row_pos == nullptr: slot_pos[row_seq[r]]; rows of a slot with a set flag are not stored (nullptr: none)
  const int32_t *slot_pos, *slot_done;
  int rows;
};
int launch_kv4_append(const Kv4AppendArgs& a, hipStream_t s);

struct Kv4ReadArgs {
  Kv4Cache c;
  const int32_t *row_seq, *row_pos;         // row_seq == nullptr: row r = position r of sequence seq0
  int seq0;
  int rows;
  bf16_t *k, *v;                            // [rows][KVH][D]
};
int launch_kv4_read(const Kv4ReadArgs& a, hipStream_t s);

constexpr int KV4_MAX_SPLITS = 256;
constexpr int KV4_SINGLE_PAGES = 12;   // tiles of fewer pages are never split, whatever `splits` says

struct Kv4AttnArgs {
  Kv4Cache c;
  const bf16_t* q;                          // rows of [H][D]
  bf16_t* out;
  int64_t q_stride, out_stride;
  const int32_t* seq_slot;                  // [n_seqs] slot of each sequence, nullptr = identity
  const int32_t* q_start;                   // [n_seqs + 1] first query row of each sequence
  const int32_t* kv_len;                    // [n_seqs] keys of each sequence
  int n_seqs, total_q, max_q, max_kv, H;
  float scale;
  int splits;                               // most key ranges per query tile (kv4_attn_splits), >= 1
  float* part;                              // splits > 1: kv4_attn_part_floats
  bool wide;                                // wide tiles whatever max_q is
  int tile_cols;                            // set by the launch: query columns per tile
  // set by launch_kv4_step: one row per sequence seq_slot[i], at row_pos[i] (nullptr: slot_pos) if that is below step_len
  const int32_t *row_pos, *slot_pos;
  int step_len;
};
// most key ranges a call of these sizes is split into: a function of the host's sizes only
int kv4_attn_splits(int n_seqs, int max_q, int max_kv, int H, int KVH);
int64_t kv4_attn_part_floats(int total_q, int H, int D, int splits);
int launch_kv4_attn(const Kv4AttnArgs& a, hipStream_t s);

// append p's rows (one per sequence; q_out is not used) and attend from them; of `a`: out, out_stride, scale, splits, part
int launch_kv4_step(const Kv4AppendArgs& p, const Kv4AttnArgs& a, hipStream_t s);

}  // namespace fmi
