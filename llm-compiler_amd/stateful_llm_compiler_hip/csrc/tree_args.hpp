// Arguments of the tree attention kernels, between the entry points (tree_attention.hip)
// and the kernels' translation units.
#pragma once
#include "common.hpp"

namespace slc_tree {

// Rows that a piece has at least, 32 KB of K: shorter ones cost more in their results than
// they save (in a graph: 16 nodes on one sequence of 2000 rows of 128 bytes, 256 rows 12.4
// us, 128 rows 13.5; one node on 9 of up to 392 of 512 bytes, 256 rows 20.8 us, 64 rows 13.0).
constexpr int min_piece_rows(int padded_row_bytes) { return padded_row_bytes >= 512 ? 64 : 32768 / padded_row_bytes; }

struct TreeArgs {
  const void* query;
  const void* key;
  const void* value;
  const int32_t* table;  // null: contiguous buffers
  const void* lengths;
  const uint8_t* tree;  // null: node i sees nodes 0 .. i
  const void* mask;
  void* output;
  int64_t table_sb, num_pages, tree_sb, tree_si, tree_sj, mask_sb, mask_ss;
  int64_t q_sb, q_sh, q_st, kv_sb, kv_ss, kv_sh, o_sb, o_sh, o_st;
  int64_t rows;  // rows that may be seen: the capacity, or the mask's length
  int page_shift, lengths_dtype, mask_dtype;
  int batch, q_heads, kv_heads, nodes, head_dim;
  float scale;
  bool vector_kv, vector_q, vector_o;  // rows that 16-byte loads (8- or 16-byte stores) take
  // The split: `slots` pieces per KV head and row block at most.
  int slots, row_blocks;
  float inverse_slots;
  int extra;  // large batches: slots of further pieces, before one of each sequence's first; else -1
  float* partial;  // [place, KV head, row block][rows][DP], then their (max, sum) pairs (see Piece)
  float2* stats;
  int* counters;  // [sequence, KV head, row block], zero between calls; null: a merge kernel
  int2* pieces;   // for that: per sequence the place of its second piece, and how many
};

// The kernel for `rows` query rows per KV head, and its launch; one pair per type, in
// a translation unit each.
struct Plan {
  int rows_per_block, padded_dim;
};
Plan plan_bf16(int rows, int head_dim);
Plan plan_f16(int rows, int head_dim);
Plan plan_f32(int rows, int head_dim);
int launch_bf16(const TreeArgs& a, const Plan& plan, hipStream_t stream);
int launch_f16(const TreeArgs& a, const Plan& plan, hipStream_t stream);
int launch_f32(const TreeArgs& a, const Plan& plan, hipStream_t stream);

}  // namespace slc_tree
