// kv_commit: the accepted nodes' rows of every layer's KV cache moved to their
// places behind the sequence, and the lengths after it.
//
// Node n of a tree was stored at row lengths[b] + n; the accepted ones,
// path[b, 0 .. counts[b]) in ascending order, belong at lengths[b] + 0 .. counts[b).
// Pure data movement of the few rows whose place changes: the bytes are small
// and a call is the latency of two dependent round trips, so one launch takes
// all layers (24 layers of 2 KV heads of 64, bf16, in a graph: 2.7 us for 3 rows of one
// sequence, 4.1 us for 11 rows of each of 32, in pages).  A workgroup owns one layer of one
// sequence (it reads the length once and may write it in place) and moves chunks in path
// order, a batch of loads, a barrier, their stores: a row's source lies behind its place,
// so what a batch overwrites no later batch reads.
#include "common.hpp"

namespace {

constexpr int kMaxLayers = SLC_KV_COMMIT_MAX_LAYERS;
constexpr int kMaxNodes = SLC_VERIFY_MAX_NODES;
constexpr int kThreads = 256;
constexpr int kInFlight = 4;  // chunks a thread holds between load and store
typedef uint32_t chunk16_t __attribute__((ext_vector_type(4)));

struct CommitArgs {
  void* key[kMaxLayers];
  void* value[kMaxLayers];
  const int64_t* lengths[kMaxLayers];
  int64_t* lengths_out[kMaxLayers];
  const int32_t* table;  // null: contiguous buffers
  const int64_t* path;   // [B, nodes]
  const int64_t* counts;
  int* overflow;
  int64_t table_sb, pages_per_seq, num_pages;
  int64_t sb, ss, sh;  // in units of the chunk
  int64_t capacity;
  int page_shift, nodes, heads, head_units;
};

template <typename U>
__global__ __launch_bounds__(kThreads) void kv_commit_kernel(CommitArgs a) {
  __shared__ int from[kMaxNodes], to[kMaxNodes];
  __shared__ int moves;
  const int layer = blockIdx.x;
  const int64_t b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t length = a.lengths[layer][b];
  const int64_t asked = a.counts[b];
  const int64_t count = asked < 0 ? 0 : (asked > a.nodes ? a.nodes : asked);
  // What the new length counts without a row of its own sets the flag.
  bool lost = asked != count;
  if (tid < 64) {
    // The rows that move: sources behind their places, inside the cache.
    int found = 0;
    for (int base = 0; base < count; base += 64) {
      const int j = base + lane;
      const int64_t n = j < count ? a.path[b * a.nodes + j] : -1;
      const bool there = n >= j && n < a.nodes && length >= 0 && length < a.capacity - n;
      const bool move = there && n > j;
      lost |= j < count && !there;
      const uint64_t hits = __ballot(move);
      if (move) {
        const int at = found + __popcll(hits & ((uint64_t{1} << lane) - 1));
        from[at] = static_cast<int>(n);
        to[at] = j;
      }
      found += __popcll(hits);
    }
    if (lane == 0) moves = found;
  }
  __syncthreads();
  // Offset of the sequence's row s, or -1 where its page is none of the pool's.
  auto offset = [&](int64_t s) -> int64_t {
    if (a.table == nullptr) return b * a.sb + s * a.ss;
    const int64_t page = a.table[b * a.table_sb + (s >> a.page_shift)];
    if (page < 0 || page >= a.num_pages) return -1;
    return page * a.sb + (s & ((int64_t{1} << a.page_shift) - 1)) * a.ss;
  };
  const int row_units = 2 * a.heads * a.head_units;
  const int total = moves * row_units;  // under 2^31: 1023 rows of 2^21 elements
  U* key = static_cast<U*>(a.key[layer]);
  U* value = static_cast<U*>(a.value[layer]);
  for (int base = 0; base < total; base += kThreads * kInFlight) {
    U chunk[kInFlight];
    U* place[kInFlight];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      const int item = base + i * kThreads + tid;
      place[i] = nullptr;
      if (item >= total) continue;
      const int move = item / row_units;
      int unit = item - move * row_units;
      U* buffer = unit < row_units / 2 ? key : value;
      unit = unit < row_units / 2 ? unit : unit - row_units / 2;
      const int64_t source = offset(length + from[move]), target = offset(length + to[move]);
      if (source < 0 || target < 0) {
        lost = true;
        continue;
      }
      const int64_t column = unit / a.head_units * a.sh + unit % a.head_units;
      chunk[i] = buffer[source + column];
      place[i] = buffer + target + column;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kInFlight; ++i)
      if (place[i] != nullptr) *place[i] = chunk[i];
  }
  if (tid == 0) {
    const int64_t next = static_cast<int64_t>(static_cast<uint64_t>(length) + static_cast<uint64_t>(count));
    if (a.lengths_out[layer] != nullptr) a.lengths_out[layer][b] = next;
    lost |= length > a.capacity - count || next < 0;
  }
  if (lost && a.overflow != nullptr) *a.overflow = 1;
}

}  // namespace

extern "C" int slc_hip_kv_commit(
    void* const* key, void* const* value, const int64_t* const* lengths, int64_t* const* lengths_out,
    const int32_t* block_table, int64_t table_stride_b, int64_t pages_per_seq, int64_t page_tokens,
    int64_t num_pages, const int64_t* path, const int64_t* counts, int* overflow, int dtype,
    int64_t layers, int64_t batch, int64_t nodes, int64_t heads, int64_t head_dim, int64_t capacity,
    int64_t stride_b, int64_t stride_s, int64_t stride_h, void* stream) {
  const char* what = "slc_hip_kv_commit";
  SLC_REQUIRE(slc_host::is_float_dtype(dtype), "%s: bad dtype %d", what, dtype);
  SLC_REQUIRE(layers >= 0 && batch >= 0 && batch <= 65535 && heads > 0 && head_dim > 0 && capacity > 0 &&
                  heads <= (1 << 20) && head_dim <= (1 << 20) && heads * head_dim <= (1 << 20),
              "%s: bad sizes", what);
  SLC_REQUIRE(nodes >= 1 && nodes <= kMaxNodes, "%s: 1 to %d nodes", what, kMaxNodes);
  if (block_table != nullptr)
    SLC_REQUIRE(page_tokens >= 16 && (page_tokens & (page_tokens - 1)) == 0 && num_pages >= 0 &&
                    pages_per_seq >= 0 && pages_per_seq * page_tokens >= capacity,
                "%s: bad pages", what);
  if (layers == 0 || batch == 0) return SLC_OK;
  SLC_REQUIRE(key && value && lengths && lengths_out && path && counts, "%s: null pointer", what);
  const int es = slc_host::dtype_size(dtype);
  uint64_t bits = 0;
  for (int64_t l = 0; l < layers; ++l) {
    SLC_REQUIRE(key[l] && value[l] && lengths[l], "%s: null pointer in layer %d", what,
                static_cast<int>(l));
    bits |= reinterpret_cast<uintptr_t>(key[l]) | reinterpret_cast<uintptr_t>(value[l]);
  }
  SLC_REQUIRE(bits % es == 0, "%s: misaligned cache", what);
  bits |= static_cast<uint64_t>((stride_b | stride_s | stride_h | head_dim) * es);
  const int unit = bits % 16 == 0 ? 16 : es;
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (int64_t first = 0; first < layers; first += kMaxLayers) {
    CommitArgs a{};
    const int n = static_cast<int>(layers - first < kMaxLayers ? layers - first : kMaxLayers);
    for (int l = 0; l < n; ++l) {
      a.key[l] = key[first + l];
      a.value[l] = value[first + l];
      a.lengths[l] = lengths[first + l];
      a.lengths_out[l] = lengths_out[first + l];
    }
    a.table = block_table;
    a.path = path;
    a.counts = counts;
    a.overflow = overflow;
    a.table_sb = table_stride_b;
    a.pages_per_seq = pages_per_seq;
    a.num_pages = num_pages;
    a.sb = stride_b * es / unit;
    a.ss = stride_s * es / unit;
    a.sh = stride_h * es / unit;
    a.capacity = capacity;
    a.page_shift = block_table == nullptr ? 0 : __builtin_ctzll(static_cast<uint64_t>(page_tokens));
    a.nodes = static_cast<int>(nodes);
    a.heads = static_cast<int>(heads);
    a.head_units = static_cast<int>(head_dim * es / unit);
    const dim3 grid(n, static_cast<unsigned>(batch));
    if (unit == 16) {
      hipLaunchKernelGGL(kv_commit_kernel<chunk16_t>, grid, dim3(kThreads), 0, s, a);
    } else if (unit == 4) {
      hipLaunchKernelGGL(kv_commit_kernel<uint32_t>, grid, dim3(kThreads), 0, s, a);
    } else {
      hipLaunchKernelGGL(kv_commit_kernel<uint16_t>, grid, dim3(kThreads), 0, s, a);
    }
    const int status = slc_host::check_launch(what);
    if (status != SLC_OK) return status;
  }
  return SLC_OK;
}
