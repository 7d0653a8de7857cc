// tree_attention: attention of a tree of drafted tokens over a KV cache.
//
//   out[b, h, i] = sum_s softmax_s(t)[s] value[s],  t[s] = scale q[b, h, i].key[s] (+ mask[b, s])
//
// over the rows s that node i sees: the sequence's, s < lengths[b], and of the
// nodes' own rows lengths[b] + j those with tree[i, j].  fp32 throughout, one
// rounding of the output; no row seen: NaN.
//
// One workgroup per (node, query head, sequence): a thread per key for the scores of
// 256 keys, then a thread per dim for their weighted values.
#include <algorithm>
#include <cmath>

#include "common.hpp"

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 256;

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
  int q_heads, kv_heads, nodes, head_dim;
  float scale;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void tree_attention_kernel(TreeArgs a) {
  __shared__ float q[256], p[kThreads], part[kThreads / 64];
  __shared__ int64_t at[kThreads];
  const int i = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int64_t b = blockIdx.z;
  const int kvh = h / (a.q_heads / a.kv_heads);
  int64_t length = slc::load_length(a.lengths, b, a.lengths_dtype);
  length = length < 0 ? 0 : (length > a.rows ? a.rows : length);
  const int64_t end = length + a.nodes < a.rows ? length + a.nodes : a.rows;
  const T* key = static_cast<const T*>(a.key) + kvh * a.kv_sh;
  const T* value = static_cast<const T*>(a.value) + kvh * a.kv_sh;
  if (tid < a.head_dim)
    q[tid] = slc::to_f32(static_cast<const T*>(a.query)[b * a.q_sb + h * a.q_sh + i * a.q_st + tid]) * a.scale;
  float top = -INFINITY, sum = 0.0f, acc = 0.0f;
  for (int64_t base = 0; base < end; base += kThreads) {
    __syncthreads();
    const int64_t s = base + tid;
    int64_t row = -1;
    if (s < end) {
      const int64_t j = s - length;
      const bool seen = j < 0 || (a.tree == nullptr ? j <= i : a.tree[b * a.tree_sb + i * a.tree_si + j * a.tree_sj] != 0);
      if (seen && a.table != nullptr) {
        const int64_t page = a.table[b * a.table_sb + (s >> a.page_shift)];
        if (page >= 0 && page < a.num_pages)
          row = page * a.kv_sb + (s & ((int64_t{1} << a.page_shift) - 1)) * a.kv_ss;
      } else if (seen) {
        row = b * a.kv_sb + s * a.kv_ss;
      }
    }
    float t = -INFINITY;
    if (row >= 0) {
      const float m = a.mask == nullptr ? 0.0f : slc::load_as_f32(a.mask, b * a.mask_sb + s * a.mask_ss, a.mask_dtype);
      if (m == -INFINITY) {
        row = -1;
      } else {
        t = 0.0f;
        for (int d = 0; d < a.head_dim; ++d) t = fmaf(q[d], slc::to_f32(key[row + d]), t);
        t += m;
      }
    }
    at[tid] = row;
    float most = slc::wave_max(t);
    if ((tid & 63) == 0) part[tid >> 6] = most;
    __syncthreads();
    most = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    most = fmaxf(most, top);
    const float shift = most == -INFINITY ? 0.0f : most;
    const float alpha = exp2f((top - shift) * kLog2e);
    p[tid] = row >= 0 ? exp2f((t - shift) * kLog2e) : 0.0f;
    top = most;
    __syncthreads();
    sum *= alpha;
    acc *= alpha;
    const int keys = static_cast<int>(end - base < kThreads ? end - base : kThreads);
    for (int k = 0; k < keys; ++k) {
      sum += p[k];
      if (tid < a.head_dim && at[k] >= 0) acc = fmaf(p[k], slc::to_f32(value[at[k] + tid]), acc);
    }
  }
  if (tid < a.head_dim)
    static_cast<T*>(a.output)[b * a.o_sb + h * a.o_sh + i * a.o_st + tid] = slc::from_f32<T>(acc / sum);
}

int run(const char* what, TreeArgs a, void* workspace, int64_t workspace_bytes, int dtype, int64_t batch,
        int64_t q_heads, int64_t kv_heads, int64_t nodes, int64_t head_dim, int64_t capacity, int64_t mask_len,
        void* stream) {
  SLC_REQUIRE(slc_host::is_float_dtype(dtype), "%s: bad dtype %d", what, dtype);
  SLC_REQUIRE(a.lengths_dtype == SLC_I64 || a.lengths_dtype == SLC_I32, "%s: lengths must be int32 or int64", what);
  SLC_REQUIRE(batch >= 0 && batch <= 65535 && nodes >= 0 && nodes <= SLC_TREE_MAX_NODES, "%s: bad batch or node count",
              what);
  SLC_REQUIRE(kv_heads > 0 && q_heads > 0 && q_heads % kv_heads == 0 && q_heads <= 65535, "%s: bad head counts", what);
  SLC_REQUIRE(head_dim >= 1 && head_dim <= 256, "%s: head_dim must be 1 to 256", what);
  SLC_REQUIRE(capacity >= 1 && capacity <= (int64_t{1} << 30), "%s: capacity must be 1 to 2^30", what);
  SLC_REQUIRE(a.scale > 0.0f && std::isfinite(a.scale), "%s: scale must be positive and finite", what);
  if (batch == 0 || nodes == 0) return SLC_OK;
  SLC_REQUIRE(a.query && a.key && a.value && a.lengths && a.output, "%s: null pointer", what);
  a.rows = capacity;
  if (a.mask != nullptr) {
    SLC_REQUIRE(slc_host::is_float_dtype(a.mask_dtype), "%s: bad mask dtype %d", what, a.mask_dtype);
    SLC_REQUIRE(mask_len >= 0 && mask_len <= capacity, "%s: the mask is longer than the cache", what);
    a.rows = mask_len;
  }
  (void)workspace;
  (void)workspace_bytes;
  a.q_heads = static_cast<int>(q_heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.nodes = static_cast<int>(nodes);
  a.head_dim = static_cast<int>(head_dim);
  const dim3 grid(a.nodes, a.q_heads, static_cast<unsigned>(batch));
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case SLC_BF16:
      hipLaunchKernelGGL(tree_attention_kernel<slc::bf16_t>, grid, dim3(kThreads), 0, s, a);
      break;
    case SLC_F16:
      hipLaunchKernelGGL(tree_attention_kernel<slc::f16_t>, grid, dim3(kThreads), 0, s, a);
      break;
    default:
      hipLaunchKernelGGL(tree_attention_kernel<float>, grid, dim3(kThreads), 0, s, a);
  }
  return slc_host::check_launch(what);
}

}  // namespace

extern "C" int64_t slc_hip_tree_attention_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                         int64_t nodes, int64_t head_dim, int dtype) {
  (void)batch, (void)q_heads, (void)kv_heads, (void)nodes, (void)head_dim, (void)dtype;
  return 0;
}

extern "C" int slc_hip_tree_attention(
    const void* query, const void* key_buffer, const void* value_buffer, const void* lengths, int lengths_dtype,
    const uint8_t* tree, const void* mask, int mask_dtype, void* output, void* workspace, int64_t workspace_bytes,
    int dtype, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t nodes, int64_t head_dim, int64_t capacity,
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
  a.scale = scale;
  return run("slc_hip_tree_attention", a, workspace, workspace_bytes, dtype, batch, q_heads, kv_heads, nodes, head_dim,
             capacity, mask_len, stream);
}

extern "C" int slc_hip_paged_tree_attention(
    const void* query, const void* key_pool, const void* value_pool, const int32_t* block_table,
    int64_t table_stride_b, int64_t pages_per_seq, int64_t page_tokens, int64_t num_pages, int64_t page_stride,
    const void* lengths, int lengths_dtype, const uint8_t* tree, const void* mask, int mask_dtype, void* output,
    void* workspace, int64_t workspace_bytes, int dtype, int64_t batch, int64_t q_heads, int64_t kv_heads,
    int64_t nodes, int64_t head_dim, int64_t mask_len, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t,
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
  a.scale = scale;
  return run(what, a, workspace, workspace_bytes, dtype, batch, q_heads, kv_heads, nodes, head_dim,
             pages_per_seq * page_tokens, mask_len, stream);
}
