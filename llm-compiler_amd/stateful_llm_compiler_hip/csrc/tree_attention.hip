// tree_attention: attention of a tree of drafted tokens over a KV cache, contiguous or
// paged: the entry points (argument checks, the split, the workspace).  The kernels are
// in tree_kernel.hpp.
#include <algorithm>
#include <cmath>

#include "tree_args.hpp"

namespace {

using slc_tree::Plan;
using slc_tree::TreeArgs;

Plan plan_for(int dtype, int rows, int head_dim) {
  if (dtype == SLC_BF16) return slc_tree::plan_bf16(rows, head_dim);
  if (dtype == SLC_F16) return slc_tree::plan_f16(rows, head_dim);
  return slc_tree::plan_f32(rows, head_dim);
}

// The split of a call: row blocks, pieces (a workgroup per CU, but room for each sequence
// and some more) and the workspace for their partial results.
struct Split {
  int64_t row_blocks, slots, extra, partial_bytes, stats_bytes, pieces_bytes;
  int64_t bytes() const { return partial_bytes + stats_bytes + pieces_bytes; }
};
Split split_for(const Plan& plan, int64_t batch, int64_t kv_heads, int64_t rows) {
  Split s;
  s.row_blocks = slc_host::ceil_div(rows, plan.rows_per_block);
  const int64_t cus = slc_host::device_cu_count(), each = kv_heads * s.row_blocks;
  // Where whole sequences are enough for all CUs only those far longer than the others are
  // cut: more workgroups than CUs are a second round (128 sequences of 500 to 2000 rows, 8
  // nodes, 2 KV heads: 25 us, pieces of even length in 160 slots 39; 1024 of 100 to 600 rows, one
  // node: 87 us, 239).
  s.extra = batch * each >= cus ? batch / 4 : -1;
  s.slots = s.extra >= 0 ? batch + s.extra : std::max<int64_t>(cus / each, batch + batch / 4);
  // Of these only the pieces of a sequence that is cut have partial results: the further
  // ones, and as many first ones at most (1024 sequences of 64 nodes, 32 heads on 8 of 128: 545
  // MB; places for all of them were 1.36 GB).
  const int64_t places = (s.extra >= 0 ? 2 * s.extra : s.slots) * kv_heads * s.row_blocks * plan.rows_per_block;
  s.partial_bytes = places * plan.padded_dim * 4;
  s.stats_bytes = places * 8;
  s.pieces_bytes = batch * 8;
  return s;
}

int run(const char* what, TreeArgs a, void* workspace, int64_t workspace_bytes, int64_t num_counters, int dtype, int64_t batch,
        int64_t q_heads, int64_t kv_heads, int64_t nodes, int64_t head_dim, int64_t capacity, int64_t mask_len,
        void* stream) {
  SLC_REQUIRE(slc_host::is_float_dtype(dtype), "%s: bad dtype %d", what, dtype);
  SLC_REQUIRE(a.lengths_dtype == SLC_I64 || a.lengths_dtype == SLC_I32, "%s: lengths must be int32 or int64", what);
  SLC_REQUIRE(batch >= 0 && batch <= 32768, "%s: batch must be 0 to 32768", what);
  SLC_REQUIRE(nodes >= 0 && nodes <= (a.tree == nullptr ? SLC_CHAIN_MAX_NODES : SLC_TREE_MAX_NODES),
              "%s: a tree has at most %d nodes, a chain %d", what, SLC_TREE_MAX_NODES, SLC_CHAIN_MAX_NODES);
  SLC_REQUIRE(kv_heads > 0 && q_heads > 0 && q_heads % kv_heads == 0 && q_heads <= 65535, "%s: bad head counts", what);
  SLC_REQUIRE(head_dim >= 1 && head_dim <= 256, "%s: head_dim must be 1 to 256", what);
  SLC_REQUIRE(capacity >= 1 && capacity <= (int64_t{1} << 30), "%s: capacity must be 1 to 2^30", what);
  SLC_REQUIRE(batch * capacity <= (int64_t{1} << 34), "%s: batch times capacity above 2^34", what);
  SLC_REQUIRE(a.scale > 0.0f && std::isfinite(a.scale), "%s: scale must be positive and finite", what);
  if (batch == 0 || nodes == 0) return SLC_OK;
  SLC_REQUIRE(a.query && a.key && a.value && a.lengths && a.output, "%s: null pointer", what);
  a.rows = capacity;
  if (a.mask != nullptr) {
    SLC_REQUIRE(slc_host::is_float_dtype(a.mask_dtype), "%s: bad mask dtype %d", what, a.mask_dtype);
    SLC_REQUIRE(mask_len >= 0 && mask_len <= capacity, "%s: the mask is longer than the cache", what);
    a.rows = mask_len;
  }
  a.batch = static_cast<int>(batch);
  a.q_heads = static_cast<int>(q_heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.nodes = static_cast<int>(nodes);
  a.head_dim = static_cast<int>(head_dim);
  const int64_t rows = q_heads / kv_heads * nodes;
  const Plan plan = plan_for(dtype, static_cast<int>(rows), a.head_dim);
  const Split split = split_for(plan, batch, kv_heads, rows);
  SLC_REQUIRE(rows < (1 << 24) && split.slots <= 65535 && split.row_blocks <= 65535, "%s: too many query rows", what);
  SLC_REQUIRE(workspace != nullptr && workspace_bytes >= split.bytes() &&
                  (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
              "%s: workspace too small or not on 16 bytes", what);
  SLC_REQUIRE(a.counters != nullptr && num_counters >= batch * kv_heads * split.row_blocks, "%s: too few counters", what);
  a.row_blocks = static_cast<int>(split.row_blocks);
  a.slots = static_cast<int>(split.slots);
  a.extra = static_cast<int>(split.extra);
  // Pieces are rounded up to whole ones; the search for their size starts as if that took
  // a third of a slot per sequence.
  a.inverse_slots = 1.0f / (static_cast<float>(split.slots) - 0.3f * static_cast<float>(batch));
  char* place = static_cast<char*>(workspace);
  a.partial = reinterpret_cast<float*>(place);
  a.stats = reinterpret_cast<float2*>(place + split.partial_bytes);
  a.pieces = reinterpret_cast<int2*>(place + split.partial_bytes + split.stats_bytes);
  const int es = slc_host::dtype_size(dtype);
  // What the last piece of a sequence would put together at most, and how many pieces would
  // release their results, each a write-back of its L2: from 64 KB or 32 pieces on a merge
  // kernel does it (see tree_merge_kernel).
  const int64_t whole = slc_host::ceil_div(a.rows, slc_tree::min_piece_rows(plan.padded_dim * es));
  const int64_t most_pieces = std::min(split.slots - batch + 1, whole > 1 ? whole + 1 : 1);
  const int64_t all_pieces = std::min(split.slots, batch * most_pieces) * kv_heads * split.row_blocks;
  if (most_pieces * std::min<int64_t>(rows, plan.rows_per_block) * plan.padded_dim * 4 > 65536 || all_pieces > 32)
    a.counters = nullptr;
  const auto on = [es](int64_t bytes, std::initializer_list<const void*> pointers, std::initializer_list<int64_t> sizes) {
    uint64_t bits = 0;
    for (const void* p : pointers) bits |= reinterpret_cast<uintptr_t>(p);
    for (int64_t n : sizes) bits |= static_cast<uint64_t>(n * es);
    return bits % static_cast<uint64_t>(bytes) == 0;
  };
  // (The 256 rows of a step lie within 2^30 bytes.)
  a.vector_kv = on(16, {a.key, a.value}, {a.kv_sb, a.kv_ss, a.kv_sh, head_dim}) && a.kv_ss * es <= (1 << 22);
  a.vector_q = on(16, {a.query}, {a.q_sb, a.q_sh, a.q_st, head_dim});
  a.vector_o = on(4 * es, {a.output}, {a.o_sb, a.o_sh, a.o_st, head_dim});
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == SLC_BF16) return slc_tree::launch_bf16(a, plan, s);
  if (dtype == SLC_F16) return slc_tree::launch_f16(a, plan, s);
  return slc_tree::launch_f32(a, plan, s);
}

}  // namespace

extern "C" int64_t slc_hip_tree_attention_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                         int64_t nodes, int64_t head_dim, int dtype) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || nodes <= 0 || head_dim <= 0 || !slc_host::is_float_dtype(dtype))
    return 0;
  const int64_t rows = q_heads / kv_heads * nodes;
  return split_for(plan_for(dtype, static_cast<int>(rows), static_cast<int>(head_dim)), batch, kv_heads, rows).bytes();
}

extern "C" int64_t slc_hip_tree_attention_counter_count(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t nodes,
                                                        int64_t head_dim, int dtype) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || nodes <= 0 || head_dim <= 0 || !slc_host::is_float_dtype(dtype))
    return 0;
  const int64_t rows = q_heads / kv_heads * nodes;
  const Plan plan = plan_for(dtype, static_cast<int>(rows), static_cast<int>(head_dim));
  return batch * kv_heads * slc_host::ceil_div(rows, plan.rows_per_block);
}

extern "C" int slc_hip_tree_attention(
    const void* query, const void* key_buffer, const void* value_buffer, const void* lengths, int lengths_dtype,
    const uint8_t* tree, const void* mask, int mask_dtype, void* output, void* workspace, int64_t workspace_bytes,
    int* counters, int64_t num_counters, int dtype, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t nodes, int64_t head_dim, int64_t capacity,
    int64_t mask_len, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t, int64_t kv_stride_b,
    int64_t kv_stride_s, int64_t kv_stride_h, int64_t tree_stride_b, int64_t tree_stride_i, int64_t tree_stride_j,
    int64_t mask_stride_b, int64_t mask_stride_s, int64_t out_stride_b, int64_t out_stride_h, int64_t out_stride_t,
    float scale, void* stream) {
  TreeArgs a{};
  a.query = query;
  a.key = key_buffer;
  a.value = value_buffer;
  a.lengths = lengths;
  a.lengths_dtype = lengths_dtype;
  a.tree = tree;
  a.mask = mask;
  a.mask_dtype = mask_dtype;
  a.output = output;
  a.q_sb = q_stride_b, a.q_sh = q_stride_h, a.q_st = q_stride_t;
  a.kv_sb = kv_stride_b, a.kv_ss = kv_stride_s, a.kv_sh = kv_stride_h;
  a.tree_sb = tree_stride_b, a.tree_si = tree_stride_i, a.tree_sj = tree_stride_j;
  a.mask_sb = mask_stride_b, a.mask_ss = mask_stride_s;
  a.o_sb = out_stride_b, a.o_sh = out_stride_h, a.o_st = out_stride_t;
  a.counters = counters;
  a.scale = scale;
  return run("slc_hip_tree_attention", a, workspace, workspace_bytes, num_counters, dtype, batch, q_heads, kv_heads, nodes, head_dim,
             capacity, mask_len, stream);
}

extern "C" int slc_hip_paged_tree_attention(
    const void* query, const void* key_pool, const void* value_pool, const int32_t* block_table,
    int64_t table_stride_b, int64_t pages_per_seq, int64_t page_tokens, int64_t num_pages, int64_t page_stride,
    const void* lengths, int lengths_dtype, const uint8_t* tree, const void* mask, int mask_dtype, void* output,
    void* workspace, int64_t workspace_bytes, int* counters, int64_t num_counters, int dtype, int64_t batch,
    int64_t q_heads, int64_t kv_heads, int64_t nodes, int64_t head_dim, int64_t mask_len, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t,
    int64_t kv_stride_s, int64_t kv_stride_h, int64_t tree_stride_b, int64_t tree_stride_i, int64_t tree_stride_j,
    int64_t mask_stride_b, int64_t mask_stride_s, int64_t out_stride_b, int64_t out_stride_h, int64_t out_stride_t,
    float scale, void* stream) {
  const char* what = "slc_hip_paged_tree_attention";
  SLC_REQUIRE(page_tokens >= 16 && (page_tokens & (page_tokens - 1)) == 0 && page_tokens <= (int64_t{1} << 30),
              "%s: page_tokens must be a power of two of 16 or more", what);
  SLC_REQUIRE(pages_per_seq >= 1 && num_pages >= 0 && pages_per_seq <= (int64_t{1} << 30) / page_tokens, "%s: bad pages",
              what);
  SLC_REQUIRE(block_table != nullptr || batch == 0 || nodes == 0, "%s: null pointer", what);
  TreeArgs a{};
  a.query = query;
  a.key = key_pool;
  a.value = value_pool;
  a.table = block_table;
  a.table_sb = table_stride_b;
  a.num_pages = num_pages;
  a.page_shift = __builtin_ctzll(static_cast<uint64_t>(page_tokens));
  a.lengths = lengths;
  a.lengths_dtype = lengths_dtype;
  a.tree = tree;
  a.mask = mask;
  a.mask_dtype = mask_dtype;
  a.output = output;
  a.q_sb = q_stride_b, a.q_sh = q_stride_h, a.q_st = q_stride_t;
  a.kv_sb = page_stride, a.kv_ss = kv_stride_s, a.kv_sh = kv_stride_h;
  a.tree_sb = tree_stride_b, a.tree_si = tree_stride_i, a.tree_sj = tree_stride_j;
  a.mask_sb = mask_stride_b, a.mask_ss = mask_stride_s;
  a.o_sb = out_stride_b, a.o_sh = out_stride_h, a.o_st = out_stride_t;
  a.counters = counters;
  a.scale = scale;
  return run(what, a, workspace, workspace_bytes, num_counters, dtype, batch, q_heads, kv_heads, nodes, head_dim,
             pages_per_seq * page_tokens, mask_len, stream);
}
