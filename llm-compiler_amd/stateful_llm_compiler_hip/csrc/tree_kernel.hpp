// tree_kernel.hpp: the tree attention kernel on the matrix cores and its merge.
// Instantiated per element type in tree_attention*.hip (translation units built in
// parallel).
//
//   out[b, h, i] = sum_s softmax_s(t)[s] value[s],  t[s] = scale q[b, h, i].key[s] (+ mask[b, s])
//
// over the rows s that node i sees: the sequence's, s < lengths[b], and of the nodes'
// own rows lengths[b] + j those with tree[i, j].
//
// A workgroup owns one KV head of one sequence, a block of query rows (all nodes of all
// query heads of that KV head; row = node * group + head) and a piece of the cache rows,
// so K and V are read once for all of them.  Producer waves stream steps of K and V
// into an LDS ring with direct-to-LDS loads (16-byte chunks, XOR-swizzled by row; rows
// past the last one read as zero).  WR x WK consumer waves own 16 QB query rows and one
// of the step's WK tiles of KT keys each, so that few query rows still keep several waves
// busy: of up to 16, four of rows of 128 bytes, whose 32 KB steps hold four tiles, two of
// 256 and one of wider ones:
//  * S^T[key, query] = K . Q^T, Q^T in registers;
//  * softmax with a running maximum that moves only when a score passes it by more than
//    kThreshold, in fp32, maxima in units of the score itself so that a mask of the
//    type's lowest value stays finite;
//  * O^T[dim, query] += V^T . P^T: the score tile's C layout is the product's B layout
//    once V's rows are taken in the same order.  The matrix cores take 16-bit weights: bf16
//    and fp16 round them, unnormalised, and their sum is that of the rounded ones, so that
//    an error of all of them alike cancels (as in the online order of the other attention
//    kernels).  Against 64 bits the outputs are off by 2.3e-3 of their norm in bf16, 2.0e-4 in
//    fp16.  Weights in two parts, a product for each, leave the output's own rounding alone,
//    1.7e-3 and 1.8e-4, but cost 41.5 us for 32.5 (16 nodes, long caches) and 34.5 for 29.3 (64
//    nodes): not taken.
// The WK partial results meet in LDS; the pieces' partial results, where a sequence
// has several, in the last of them to end or in a kernel of their own.
//
// What bounds it, in a graph, 14 query heads on 2 of 64, bf16: 32 sequences of 4096 to
// 8192 rows (101 MB) take 24.0 us with 2 nodes, 4.2 TB/s, and 32.0 with 16, whose 112
// query rows' products, then exponentials, maxima and packing, are as long as the stream: a
// step's consumers pass one barrier and do them in the same order, so that the matrix cores
// and the VALU take turns; of 16 sequences with 64 nodes, 29.4 us, some 19 us are those
// steps, of which the products alone take 6 and the vector instructions 6 to 11.  Before the first tile
// lies about 4 us (the pieces, the descriptors, the first loads), behind the last one 3 to
// 6 us (results through LDS and memory): one sequence of 600 rows and 8 nodes takes 10.1.
#pragma once
#include <cmath>
#include <type_traits>

#include "tree_args.hpp"

namespace slc_tree {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kThreshold = 5.5f;  // weights stay under e^5.5 = 245, fp16's range is 65504

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef short v4s_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4_t mfma(slc::bf16_t, uint4 a, uint4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mfma(slc::f16_t, uint4 a, uint4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                0, 0);
}

__device__ __forceinline__ f32x4_t mfma(uint32_t a, uint32_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a), __uint_as_float(b), c, 0, 0, 0);
}

__device__ __forceinline__ uint4 lds_read(const unsigned char* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ uint2 lds_read_tr(const unsigned char* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) v4s_t*)(p)));
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, int bytes) {
  const uint64_t address = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(address));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(address >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(static_cast<uint64_t>(hi) << 32 | lo), 0,
                                           __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}
__device__ __forceinline__ void lds_dma16(__amdgpu_buffer_rsrc_t rsrc, unsigned char* lds, int voffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)lds, 16, voffset, 0, 0, 0);
}

// Whether any of the 16-bit (fp32) values of a dword is NaN or infinite.
template <typename T>
__device__ __forceinline__ bool has_special(uint32_t w) {
  if constexpr (sizeof(T) == 4) {
    return (w & 0x7f800000u) == 0x7f800000u;
  } else {
    constexpr uint32_t kExp = std::is_same_v<T, slc::bf16_t> ? 0x7f80u : 0x7c00u;
    return (w & kExp) == kExp || ((w >> 16) & kExp) == kExp;
  }
}
// The dword with such values set to zero.
template <typename T>
__device__ __forceinline__ uint32_t without_special(uint32_t w) {
  if constexpr (sizeof(T) == 4) {
    return has_special<T>(w) ? 0u : w;
  } else {
    constexpr uint32_t kExp = std::is_same_v<T, slc::bf16_t> ? 0x7f80u : 0x7c00u;
    if ((w & kExp) == kExp) w &= 0xffff0000u;
    if (((w >> 16) & kExp) == kExp) w &= 0x0000ffffu;
    return w;
  }
}
template <typename T>
__device__ __forceinline__ uint4 without_special(uint4 v) {
  return make_uint4(without_special<T>(v.x), without_special<T>(v.y), without_special<T>(v.z), without_special<T>(v.w));
}

// Sums up to and with this lane, in the VALU: rows of 16 lanes by shifts, then the rows
// below by broadcasts of their last lanes.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return v;
}
__device__ __forceinline__ int wave_sum(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

// Four neighbouring dims of an output row.
template <typename T>
__device__ __forceinline__ void store_quad(T* row, int dim, int head_dim, bool vector, float4 v) {
  if (vector) {
    if (dim >= head_dim) return;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(row + dim) = v;
    } else {
      *reinterpret_cast<uint2*>(row + dim) = make_uint2(slc::pack2<T>(v.x, v.y), slc::pack2<T>(v.z, v.w));
    }
    return;
  }
  const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (dim + i < head_dim) row[dim + i] = slc::from_f32<T>(e[i]);
}
// First dim of the i-th four neighbouring outputs that a lane of group g holds.
template <typename T>
__device__ __forceinline__ int quad_dim(int i, int g) {
  return sizeof(T) == 4 ? 64 * (i / 4) + 16 * g + 4 * (i % 4) : 16 * i + 4 * g;
}
// A sum of weights of zero: a node that sees no row, NaN.
__device__ __forceinline__ float4 divided(float4 v, float sum) {
  const float by = sum == 0.0f ? __builtin_nanf("") : 1.0f / sum;
  return make_float4(v.x * by, v.y * by, v.z * by, v.w * by);
}

// n / d from d's rounded inverse, n < 2^24.
__device__ __forceinline__ int quotient(int n, int d, float inverse) {
  const int q = static_cast<int>(static_cast<float>(n) * inverse);
  const int rest = n - q * d;
  return q + (rest >= d) - (rest < 0);
}

// The tail, whose rows only some nodes see, takes as long as so many steps more: a step
// with masks has twice the instructions, and wide trees span several short steps (64
// nodes, batch of 16: 32.5 us with 2, 31.2 with 5 or 6).
template <int STEP>
constexpr int kTailSteps = STEP <= 64 ? 5 : 2;

struct Piece {
  int sequence;  // -1: none
  int index, count;
  // Places of the partial results of the first piece and of the second, which the others
  // follow: the slots, but in large batches the first piece's lies behind all further ones', as
  // far as the second's from the start.
  int head, tail;
  int length, end;  // rows of the sequence, and with its nodes'
};

// The piece of slot x.  Sequences are cut into pieces of about q steps, q the smallest
// tried for which all pieces fit the slots; every wave finds its own for itself, by the
// same arithmetic (fp32: what counts is that all agree and that no sequence has none).
template <int STEP>
__device__ __forceinline__ Piece find_piece(const TreeArgs& a, int x, float min_steps) {
  const int lane = threadIdx.x & 63;
  const int rows = static_cast<int>(a.rows);
  auto length_of = [&](int b) {
    const int64_t n = b < a.batch ? slc::load_length(a.lengths, b, a.lengths_dtype) : 0;
    return static_cast<int>(n < 0 ? 0 : (n > rows ? rows : n));
  };
  auto end_of = [&](int length) { return length + a.nodes < rows ? length + a.nodes : rows; };
  auto steps_of = [&](int b, int length) {
    const int n = (end_of(length) + STEP - 1) / STEP + kTailSteps<STEP>;
    return b < a.batch ? n : 0;
  };
  // Pieces of one: no more than whole smallest ones, and one for the tail where there are several.
  const float inverse_min = 1.0f / min_steps;
  auto most_of = [&](int steps) {
    const int n = static_cast<int>(static_cast<float>(steps - kTailSteps<STEP>) * inverse_min + 0.9999f);
    return n > 1 ? n + 1 : 1;
  };
  Piece p{-1, 0, 0, 0, 0, 0, 0};
  if (a.extra >= 0) {
    // A large batch: n - 1 < steps / q further pieces of each sequence fit the extra slots
    // for q = sum of steps / extra, so that nothing is searched for.
    int sum = 0;
#pragma unroll 4
    for (int b = lane; b < a.batch; b += 64) sum += steps_of(b, length_of(b));
    sum = wave_sum(sum);
    const float inverse = 1.0f / fmaxf(static_cast<float>(sum) * 1.001f / static_cast<float>(a.extra), min_steps);
    auto further = [&](int steps) {
      const int n = static_cast<int>(static_cast<float>(steps) * inverse + 0.9999f), most = most_of(steps);
      return a.extra > 0 && steps > 0 ? max(1, min(n, most)) - 1 : 0;
    };
    if (x >= a.extra) {
      p.sequence = x - a.extra;
      p.length = __builtin_amdgcn_readfirstlane(length_of(p.sequence));
      p.count = 1 + __builtin_amdgcn_readfirstlane(further(steps_of(p.sequence, p.length)));
    }
    int before = 0;
    for (int base = 0; base < a.batch && p.count != 1; base += 64) {
      const int length = length_of(base + lane), n = further(steps_of(base + lane, length));
      const int upto = before + wave_scan(n);
      const uint64_t hits = x < a.extra ? __ballot(upto > x) : __ballot(base + lane == p.sequence);
      if (hits != 0) {
        const int at = __builtin_ctzll(hits);
        p.sequence = base + at;
        p.count = 1 + __builtin_amdgcn_readlane(n, at);
        p.tail = __builtin_amdgcn_readlane(upto - n, at);
        p.length = __builtin_amdgcn_readlane(length, at);
        break;
      }
      before = __builtin_amdgcn_readlane(upto, 63);
    }
    p.head = a.extra + p.tail;
    p.index = x < a.extra ? x - p.tail + 1 : 0;
    p.end = end_of(p.length);
    return p;
  }
  // Of the first 64 sequences; more are read again in every pass.
  const int own_length = length_of(lane), own = steps_of(lane, own_length);
  int total = wave_sum(own);
  for (int base = 64; base < a.batch; base += 64) total += wave_sum(steps_of(base + lane, length_of(base + lane)));
  float q = fmaxf(static_cast<float>(total) * a.inverse_slots, min_steps);
  for (;;) {
    // Pieces up to and with each sequence; found on the way: the sequence of slot x.
    const float inverse = __builtin_amdgcn_rcpf(q);
    int before = 0;
    p.sequence = -1;
    for (int base = 0; base < a.batch; base += 64) {
      const int length = base == 0 ? own_length : length_of(base + lane);
      const int steps = base == 0 ? own : steps_of(base + lane, length);
      // Rounded up, past rounding errors; at least one.
      int n = static_cast<int>(static_cast<float>(steps) * inverse + 0.9999f);
      const int most = most_of(steps);
      n = n < most ? n : most;
      n = n < 1 ? (steps > 0 ? 1 : 0) : (n < steps ? n : steps);
      const int upto = before + wave_scan(n);
      const uint64_t hits = __ballot(upto > x);
      if (hits != 0 && p.sequence < 0) {
        const int at = __builtin_ctzll(hits);
        p.sequence = base + at;
        p.count = __builtin_amdgcn_readlane(n, at);
        p.head = __builtin_amdgcn_readlane(upto, at) - p.count;
        p.length = __builtin_amdgcn_readlane(length, at);
      }
      before = __builtin_amdgcn_readlane(upto, 63);
    }
    if (before <= a.slots) break;
    q *= 1.05f;
  }
  p.index = x - p.head;
  p.tail = p.head + 1;
  p.end = end_of(p.length);
  return p;
}

// Units of 16 rows and 16 dims that a row block has.
template <int DP, int ROWS>
__device__ __forceinline__ int block_units(const TreeArgs& a, int block) {
  const int rows = a.q_heads / a.kv_heads * a.nodes - block * ROWS;
  return ((rows < ROWS ? rows : ROWS) + 15) / 16 * (DP / 16);
}
// Units unit, unit + step, .. (kUnits of them, those below `units`) of a sequence's row
// block (each float4 of a wave's lanes) put together from the
// `count` pieces at place `head` and from place `tail` on, kBatch at a time.
template <typename T, int DP, int ROWS, int kUnits, int kBatch>
__device__ __forceinline__ void merge_units(const TreeArgs& a, int64_t b, int kvh, int block, int head, int tail, int count,
                                            int unit, int step, int units) {
  constexpr int kQuads = DP / 16;
  const int lane = threadIdx.x & 63;
  const int group = a.q_heads / a.kv_heads;
  const float inverse_group = __builtin_amdgcn_rcpf(static_cast<float>(group));
  const int64_t stride = static_cast<int64_t>(a.kv_heads) * a.row_blocks * ROWS;  // between pieces
  const int64_t place = (static_cast<int64_t>(kvh) * a.row_blocks + block) * ROWS;
  const float2* stats = a.stats + place + (lane & 15);
  const float4* partial = reinterpret_cast<const float4*>(a.partial + place * DP) + lane;
  float top[kUnits], sum[kUnits];
  float4 v[kUnits];
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    top[j] = -INFINITY;
    sum[j] = 0.0f;
    v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll 1
  for (int at = 0; at < count; at += kBatch) {
    float2 s[kUnits][kBatch];
    float4 o[kUnits][kBatch];
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      const int u = unit + j * step < units ? unit + j * step : unit;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int piece = at + i < count ? at + i : at;
        const int64_t k = (piece == 0 ? head : tail + piece - 1) * stride;
        s[j][i] = stats[k + u / kQuads * 16];
        o[j][i] = partial[k * (DP / 4) + u * 64];
      }
    }
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      float most = top[j];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (at + i >= count) {
          s[j][i] = make_float2(-INFINITY, 0.0f);
          o[j][i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        most = fmaxf(most, s[j][i].x);
      }
      const float use = most == -INFINITY ? 0.0f : most;
      const float own = __builtin_amdgcn_exp2f((top[j] - use) * kLog2e);
      top[j] = most;
      sum[j] *= own;
      v[j] = make_float4(v[j].x * own, v[j].y * own, v[j].z * own, v[j].w * own);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float w = __builtin_amdgcn_exp2f((s[j][i].x - use) * kLog2e);
        sum[j] = fmaf(w, s[j][i].y, sum[j]);
        v[j].x = fmaf(w, o[j][i].x, v[j].x);
        v[j].y = fmaf(w, o[j][i].y, v[j].y);
        v[j].z = fmaf(w, o[j][i].z, v[j].z);
        v[j].w = fmaf(w, o[j][i].w, v[j].w);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    const int u = unit + j * step;
    const int row = block * ROWS + u / kQuads * 16 + (lane & 15);
    if (u >= units || row >= group * a.nodes) continue;
    const int n = quotient(row, group, inverse_group);
    const int h = kvh * group + row - n * group;
    store_quad<T>(static_cast<T*>(a.output) + b * a.o_sb + h * a.o_sh + n * a.o_st, quad_dim<T>(u % kQuads, lane >> 4),
                  a.head_dim, a.vector_o, divided(v[j], sum[j]));
  }
}
// The same by workgroups of their own, for large results and many pieces.  One CU takes in
// about 10 bytes a cycle, so that the last piece alone is slow from some 64 KB on (8 sequences
// of up to 8 pieces of 112 rows, 229 KB: 24.2 us, with this kernel 14.7), and each piece's
// release is a write-back of its L2 (17 sequences of 2 pieces, 49 nodes: 31.5 us, with this
// kernel 17.1; 4 of up to 8, 64 in all, in a graph: 13.7 and 12.3).  Below, a second launch
// costs the host more than it saves: 3 pieces of 56 rows (42 KB) 10.5 us a call, 12.8 with it.
template <typename T, int DP, int ROWS>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
  const int64_t b = blockIdx.z;
  const int2 pieces = a.pieces[b];
  const int kvh = blockIdx.y / a.row_blocks, block = blockIdx.y % a.row_blocks;
  const int unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int units = block_units<DP, ROWS>(a, block);
  if (pieces.y <= 1 || unit >= units) return;
  const int head = a.extra >= 0 ? a.extra + pieces.x : pieces.x - 1;
  merge_units<T, DP, ROWS, 1, 8>(a, b, kvh, block, head, pieces.x, pieces.y, unit, 1, unit + 1);
}

// Sizes of a kernel: DP the padded head dim, QB blocks of 16 query rows a wave, WR waves
// along the rows, KT keys a tile.
template <typename T, int DP, int QB, int WR, int KT>
struct Shape {
  static constexpr bool kWide = sizeof(T) == 4;
  static constexpr int kRowBytes = DP * static_cast<int>(sizeof(T));
  static constexpr int kTileBytes = KT * kRowBytes;  // of K or of V
  // Tiles side by side: eight waves (four of wide rows, whose registers no more than
  // two a SIMD have), 32 KB a step at most.
  static constexpr int kWaves = kRowBytes <= 256 ? 8 : 4;
  static constexpr int kFit = 32768 / (2 * kTileBytes);
  static constexpr int WK = kWaves / WR < kFit ? kWaves / WR : kFit;
  static constexpr int kConsumers = WR * WK;
  static constexpr int kStep = WK * KT;
  // Producers, each of a part of a step's rows that no page is smaller than.  One wave
  // issues a load in 90 to 140 cycles, 8 bytes a cycle; four keep up with the memory (32
  // sequences of 4096 to 8192 rows, 2 nodes, in a graph: 24.1 us, 25.5 with one).
  static constexpr int kProducers = kStep >= 64 ? 4 : kStep / 16;
  static constexpr int kThreads = (kConsumers + kProducers) * 64;
  static constexpr int kStageBytes = WK * 2 * kTileBytes;
  static constexpr int kOps = kStageBytes / 1024 / kProducers;  // a producer's loads of a step
  static constexpr int kRows = 16 * QB * WR;
  static constexpr int kMaskRows = kConsumers * 64;  // of the mask in LDS at a time, twice
  static constexpr int kWords = SLC_TREE_MAX_NODES / 32 + 2;  // of a node's row of the tree, as bits
  // Up to eight stages in what the rest leaves of 160 KB, and no more loads in flight than
  // the wait can count.
  static constexpr int kFree = 160 * 1024 - (kRows + 1) * kWords * 4 - 2 * kMaskRows * 4 - 64;
  static constexpr int kFill = kFree / kStageBytes < 8 ? kFree / kStageBytes : 8;
  static constexpr int kStages = (kFill - 2) * kOps < 64 ? kFill : 63 / kOps + 2;
  static constexpr int kQuads = DP / 16;           // float4 of a lane's outputs per query block
  static constexpr int kMergeBytes = WK > 1 ? WK * WR * QB * (kQuads * 4 + 2) * 256 : 0;
  static constexpr int kLds = kStages * kStageBytes > kMergeBytes ? kStages * kStageBytes : kMergeBytes;
  // The chunks of a row lie XORed with this.  A transposing read takes two neighbouring
  // chunks of each of 8 rows, which in rows of 256 bytes and more must differ in more than
  // the lowest bit to lie on banks of their own.
  __device__ static int swizzle(int row) { return kRowBytes >= 256 ? (row & 7) * 2 : row & 7; }
  static_assert((kStages - 2) * kOps < 64, "the wait counts at most 63 loads");
  static_assert(kMaskRows % kStep == 0, "whole steps of the mask are loaded by a thread per row");
};

// MASKED: with a mask; by itself the form without one has fewer registers and less code (16
// sequences, 64 nodes 30.5 -> 29.4 us, one sequence 10.5 -> 10.1).  The widest 16-bit form
// with one spills 13 registers; fp32 rows of 1024 bytes and 64 query rows spill 39, with one 115.
template <typename T, int DP, int QB, int WR, int KT, bool MASKED>
__global__ __launch_bounds__((Shape<T, DP, QB, WR, KT>::kThreads)) void tree_attention_kernel(TreeArgs a, float min_steps) {
  using S = Shape<T, DP, QB, WR, KT>;
  constexpr bool kWide = S::kWide;
  constexpr int WK = S::WK;
  constexpr int SUB = KT < 32 ? KT : 32, KB = SUB / 16, kSubs = KT / SUB;  // keys at a time
  constexpr int kRowBytes = S::kRowBytes, kTileBytes = S::kTileBytes;
  constexpr int kChunks = kRowBytes / 16, kOpRows = 1024 / kRowBytes;
  constexpr int ES = sizeof(T);
  __shared__ __attribute__((aligned(16))) unsigned char lds[S::kLds];
  constexpr int kMaxWords = S::kWords;
  __shared__ uint32_t tree_bits[(S::kRows + 1) * kMaxWords];
  constexpr int kMaskRows = S::kMaskRows, kMaskSteps = kMaskRows / S::kStep;
  __shared__ __attribute__((aligned(16))) float mask_room[2][MASKED ? kMaskRows : 4];
  __shared__ int arrived;

  const int kvh = blockIdx.x, slot = blockIdx.y, block = blockIdx.z;
  const Piece piece = find_piece<S::kStep>(a, slot, min_steps);
  if (piece.sequence < 0) return;
  const int64_t b = piece.sequence;
  // Its steps: the sequence's and its tail's, shared out as evenly as whole steps go; the
  // last pieces take the spare ones, the tail's count with the last step.
  const int steps = (piece.end + S::kStep - 1) / S::kStep;
  const int shared = steps + kTailSteps<S::kStep>;
  const int share = static_cast<int>(static_cast<unsigned>(shared) / static_cast<unsigned>(piece.count));
  const int shorter = piece.count - (shared - share * piece.count);  // pieces without a spare one
  auto first_step = [&](int index) { return max(0, min(steps - 1, index * share + max(0, index - shorter))); };
  int count = piece.count;
  while (count > 1 && first_step(count - 1) == first_step(count - 2)) --count;
  if (piece.index >= count) return;
  const int step0 = first_step(piece.index);
  const int nsteps = (piece.index + 1 < count ? first_step(piece.index + 1) : steps) - step0;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (a.counters == nullptr && tid == 0 && piece.index == 0 && kvh == 0 && block == 0)
    a.pieces[b] = make_int2(piece.tail, count);

  if (wave >= S::kConsumers) {
    // ---- producers ------------------------------------------------------------
    constexpr int kTileOps = kTileBytes / 1024;
    const T* kbase = static_cast<const T*>(a.key) + kvh * a.kv_sh;
    const T* vbase = static_cast<const T*>(a.value) + kvh * a.kv_sh;
    constexpr int kPart = S::kStep / S::kProducers;  // rows of a step that this producer loads
    const int part0 = (wave - S::kConsumers) * kPart;
    const int row_in_op = lane / kChunks;
    const bool paged = a.table != nullptr;
    const int page_rows = paged ? 1 << a.page_shift : kPart;
    const int segment = page_rows < kPart ? page_rows : kPart;  // rows with one base
    const int row_bytes = static_cast<int>(a.kv_ss) * ES;
    // Lane L of load n fills row kOpRows n + L / kChunks of the step, chunk L % kChunks, with
    // that row's chunk (L % kChunks) ^ S::swizzle(row); columns past the head dim lie past every range.
    // Rows kOpRows apart have another swizzle unless kOpRows is a multiple of 8.
    constexpr int kSwizzles = kOpRows >= 8 ? 1 : 8 / kOpRows;
    int voffset[kSwizzles];
#pragma unroll
    for (int i = 0; i < kSwizzles; ++i) {
      const int row = i * kOpRows + row_in_op;
      const int chunk = (lane % kChunks) ^ S::swizzle(row);
      voffset[i] = chunk * (16 / ES) < a.head_dim ? row * row_bytes + chunk * 16 : 0x40000000;
    }
    for (int t = 1 - S::kStages; t < nsteps; ++t) {
      if (t >= 0) {
        // Step t has landed: the kStages - 2 later ones (kOps each) may still fly.
        asm volatile("s_waitcnt vmcnt(%0)" ::"i"((S::kStages - 2) * S::kOps) : "memory");
        __syncthreads();
      }
      const int step = t + S::kStages - 1;
      unsigned char* dst = lds + step % S::kStages * S::kStageBytes;
      const int s0 = (step0 + step) * S::kStep;
      const int end = step < nsteps ? piece.end : 0;
      if (__builtin_expect(a.vector_kv, 1)) {
        for (int first = part0; first < part0 + kPart; first += segment) {
          int rows = end - s0 - first;  // rows past the last one read as zero
          rows = rows < segment ? rows : segment;
          int64_t at = b * a.kv_sb + static_cast<int64_t>(s0 + first) * a.kv_ss;
          if (paged && rows > 0) {
            typedef const __attribute__((address_space(4))) int32_t* ConstInts;
            const int page = ((ConstInts)(a.table))[b * a.table_sb + ((s0 + first) >> a.page_shift)];
            at = page * a.kv_sb + ((s0 + first) & (page_rows - 1)) * a.kv_ss;
            if (page < 0 || page >= a.num_pages) rows = 0;
          }
          const int bytes = rows > 0 ? (rows - 1) * row_bytes + a.head_dim * ES : 0;
          const __amdgpu_buffer_rsrc_t rk = make_rsrc(kbase + (rows > 0 ? at : 0), bytes);
          const __amdgpu_buffer_rsrc_t rv = make_rsrc(vbase + (rows > 0 ? at : 0), bytes);
          const int first_op = first / kOpRows;
          auto load = [&](int n, int i) {  // load n of the segment, n % kSwizzles == i
            const int op = first_op + n;
            unsigned char* place = dst + op / kTileOps * 2 * kTileBytes + op % kTileOps * 1024;
            const int offset = voffset[i] + (n - i) * kOpRows * row_bytes;
            lds_dma16(rk, place, offset);
            lds_dma16(rv, place + kTileBytes, offset);
          };
          constexpr int kGroup = 16 / kOpRows;  // loads of 16 rows, the smallest page
          for (int n = 0; n < segment / kOpRows; n += kGroup) {
#pragma unroll
            for (int i = 0; i < kGroup; ++i) load(n + i, i % kSwizzles);
          }
        }
      } else {
        // Any alignment: elements, a chunk of LDS per lane at a time.
        constexpr int kPer = 16 / ES;
#pragma unroll 1
        for (int n = part0 / kOpRows; n < (part0 + kPart) / kOpRows; ++n) {
          const int row = n * kOpRows + row_in_op;
          const int chunk = (lane % kChunks) ^ S::swizzle(row);
          const int s = s0 + row;
          int64_t at = -1;
          if (s < end) {
            at = b * a.kv_sb + s * a.kv_ss;
            if (paged) {
              const int page = a.table[b * a.table_sb + (s >> a.page_shift)];
              at = page >= 0 && page < a.num_pages ? page * a.kv_sb + (s & (page_rows - 1)) * a.kv_ss : -1;
            }
          }
          unsigned char* place = dst + n / kTileOps * 2 * kTileBytes + n % kTileOps * 1024 + lane * 16;
#pragma unroll 1
          for (int side = 0; side < 2; ++side) {
            const T* from = (side == 0 ? kbase : vbase) + (at < 0 ? 0 : at) + chunk * kPer;
            T v[kPer];
#pragma unroll
            for (int e = 0; e < kPer; ++e) v[e] = at >= 0 && chunk * kPer + e < a.head_dim ? from[e] : T{};
            *reinterpret_cast<uint4*>(place + side * kTileBytes) = __builtin_bit_cast(uint4, v);
          }
        }
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (WK > 1) {
      __syncthreads();
      __syncthreads();
    }
    return;
  }

  // ---- consumers ----------------------------------------------------------------
  const int wr = wave % WR, wk = wave / WR;
  const int g = lane >> 4, c = lane & 15;
  const int group = a.q_heads / a.kv_heads;
  const int rows = group * a.nodes;
  const float inverse_group = __builtin_amdgcn_rcpf(static_cast<float>(group));
  const int node0 = quotient(block * S::kRows, group, inverse_group);  // the block's first
  int node[QB], head[QB];
  bool real[QB];
  // Q^T: 16-bit types hold 8 dims 32 kk + 8 g of a block, fp32 4 dims 16 kk + 4 g.
  constexpr int kDims = kWide ? 16 : 32, kParts = DP / kDims;
  uint4 qv[QB][kParts];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int row = block * S::kRows + wr * 16 * QB + 16 * qb + c;
    real[qb] = row < rows;
    node[qb] = real[qb] ? quotient(row, group, inverse_group) : node0;
    head[qb] = kvh * group + (real[qb] ? row - node[qb] * group : 0);
    const T* qp = static_cast<const T*>(a.query) + b * a.q_sb + head[qb] * a.q_sh + node[qb] * a.q_st;
#pragma unroll
    for (int kk = 0; kk < kParts; ++kk) {
      constexpr int kPer = 16 / ES;
      const int dim = kk * kDims + kPer * g;
      if (__builtin_expect(a.vector_q, 1)) {
        qv[qb][kk] = dim < a.head_dim ? *reinterpret_cast<const uint4*>(qp + dim) : make_uint4(0, 0, 0, 0);
      } else {
        T e[kPer] = {};
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (dim + i < a.head_dim) e[i] = qp[dim + i];
        qv[qb][kk] = __builtin_bit_cast(uint4, e);
      }
    }
  }

  // Accumulators.  16-bit: acc[i] holds dims 16 i + 4 g + r, and acc[kQuads] the sum of
  // the rounded weights (a product with ones, so that the matrix cores do it).  fp32:
  // acc[4 d + j] holds dims 64 d + 16 g + 4 r + j, the sums are each lane's own.
  constexpr int kAcc = kWide ? S::kQuads : S::kQuads + 1;
  f32x4_t acc[kAcc][QB];
  float m_run[QB], l_part[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    m_run[qb] = -INFINITY;
    l_part[qb] = 0.0f;
#pragma unroll
    for (int i = 0; i < kAcc; ++i) acc[i][qb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t one2 = std::is_same_v<T, slc::bf16_t> ? 0x3f803f80u : 0x3c003c00u;
  const uint4 ones = make_uint4(one2, one2, one2, one2);
  const float scale_log2 = a.scale * kLog2e;

  // S^T of SUB keys at kt.
  auto scores = [&](const unsigned char* kt, f32x4_t (&st)[KB][QB]) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) st[kb][qb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int kk = 0; kk < kParts; ++kk) {
        const uint4 ka = lds_read(kt + (16 * kb + c) * kRowBytes + (((4 * kk + g) ^ S::swizzle(c)) << 4));
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          if constexpr (kWide) {
            st[kb][qb] = mfma(ka.x, qv[qb][kk].x, st[kb][qb]);
            st[kb][qb] = mfma(ka.y, qv[qb][kk].y, st[kb][qb]);
            st[kb][qb] = mfma(ka.z, qv[qb][kk].z, st[kb][qb]);
            st[kb][qb] = mfma(ka.w, qv[qb][kk].w, st[kb][qb]);
          } else {
            st[kb][qb] = mfma(T{}, ka, qv[qb][kk], st[kb][qb]);
          }
        }
      }
  };
  // The running maximum after scores of at most mx in this lane.  It spans the 4 lane
  // groups, but matters only when some lane passes the threshold.
  auto raise = [&](int qb, float mx) {
    if (!__any(mx > m_run[qb] + kThreshold)) return;
    mx = slc::max_xor32(slc::max_xor16(mx));
    const float m_new = fmaxf(m_run[qb], mx);
    const float alpha = __builtin_amdgcn_exp2f((m_run[qb] - (m_new == -INFINITY ? 0.0f : m_new)) * kLog2e);
#pragma unroll
    for (int i = 0; i < kAcc; ++i) acc[i][qb] = acc[i][qb] * alpha;
    l_part[qb] *= alpha;
    m_run[qb] = m_new;
  };
  // O^T += V^T . P^T with weights exp2(score * factor - shift); DIRTY: without V's NaNs
  // and infinities.
  auto weigh = [&](auto dirty_tag, const unsigned char* vt, const f32x4_t (&st)[KB][QB], float factor,
                   const float (&shift)[QB]) {
    constexpr bool kDirty = decltype(dirty_tag)::value;
    if constexpr (kWide) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float p[QB];
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) {
            p[qb] = __builtin_amdgcn_exp2f(fmaf(st[kb][qb][r], factor, -shift[qb]));
            l_part[qb] += p[qb];
          }
          const int row = 16 * kb + 4 * g + r;
#pragma unroll
          for (int d = 0; d < DP / 64; ++d) {
            uint4 va = lds_read(vt + row * kRowBytes + (((16 * d + c) ^ S::swizzle(row)) << 4));
            if constexpr (kDirty) va = without_special<T>(va);
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
              const uint32_t pb = __float_as_uint(p[qb]);
              acc[4 * d][qb] = mfma(va.x, pb, acc[4 * d][qb]);
              acc[4 * d + 1][qb] = mfma(va.y, pb, acc[4 * d + 1][qb]);
              acc[4 * d + 2][qb] = mfma(va.z, pb, acc[4 * d + 2][qb]);
              acc[4 * d + 3][qb] = mfma(va.w, pb, acc[4 * d + 3][qb]);
            }
          }
        }
    } else {
      uint4 pv[QB];
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(st[i / 4][qb][i % 4], factor, -shift[qb]));
        pv[qb] = make_uint4(slc::pack2<T>(p[0], p[1]), slc::pack2<T>(p[2], p[3]), slc::pack2<T>(p[4], p[5]),
                            slc::pack2<T>(p[6], p[7]));
      }
      // Lane c of group g addresses 4 dims of key 4 g + c / 4 and gets dim c of the
      // group's 4 keys; the second read's keys lie 16 further.
      const int row = 4 * g + (c >> 2);
#pragma unroll
      for (int i = 0; i < S::kQuads; ++i) {
        const int dim = 16 * i + 4 * (c & 3);
        const unsigned char* at = vt + row * kRowBytes + (((dim >> 3) ^ S::swizzle(row)) << 4) + (dim & 7) * 2;
        const uint2 lo = lds_read_tr(at), hi = lds_read_tr(at + 16 * kRowBytes);
        uint4 va = make_uint4(lo.x, lo.y, hi.x, hi.y);
        if constexpr (kDirty) va = without_special<T>(va);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) acc[i][qb] = mfma(T{}, va, pv[qb], acc[i][qb]);
      }
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) acc[S::kQuads][qb] = mfma(T{}, ones, pv[qb], acc[S::kQuads][qb]);
    }
  };

  // The steps whose rows all nodes see and that have no mask.
  int plain_steps = MASKED ? 0 : piece.length / S::kStep - step0;
  plain_steps = plain_steps < 0 ? 0 : (plain_steps < nsteps ? plain_steps : nsteps);

  // What the others need: the block's nodes' rows of the tree as bits (a word of ones in
  // front, for the sequence's rows, a word of zeros behind), and the mask, a row a thread,
  // loaded steps ahead (32 sequences, 8 nodes, a mask: 36.9 us, a step ahead 42.3).
  const int words = (a.nodes + 31) / 32 + 2;
  if (plain_steps < nsteps && a.tree != nullptr) {
    int count = quotient(block * S::kRows + S::kRows - 1, group, inverse_group);
    count = (count < a.nodes ? count : a.nodes - 1) - node0 + 1;
    const int parts = (a.nodes + 63) / 64;
#pragma unroll 2
    for (int item = wave; item < count * parts; item += S::kConsumers) {
      const int i = item / parts, part = item % parts;
      const int j = part * 64 + lane;
      const bool seen = j < a.nodes && a.tree[b * a.tree_sb + (node0 + i) * a.tree_si + j * a.tree_sj] != 0;
      const uint64_t bits = __ballot(seen);
      uint32_t* row = tree_bits + i * kMaxWords;
      if (lane == 0) {
        row[1 + 2 * part] = static_cast<uint32_t>(bits);
        row[2 + 2 * part] = static_cast<uint32_t>(bits >> 32);
        if (part == 0) row[0] = ~0u;
        if (part == parts - 1) row[words - 1 + (words & 1)] = 0;
      }
    }
  }
  auto mask_of = [&](int part) {  // this thread's row of the steps from part * kMaskSteps on
    const int s = step0 * S::kStep + part * kMaskRows + tid;
    return s < piece.end ? slc::load_as_f32(a.mask, b * a.mask_sb + s * a.mask_ss, a.mask_dtype) : -INFINITY;
  };
  float mask_next = 0.0f;
  if constexpr (MASKED) {
    mask_room[0][tid] = mask_of(0);
    mask_next = mask_of(1);
  }

  int stage = 0;
  for (int step = 0; step < plain_steps; ++step) {
    __syncthreads();  // this step's tiles are in the ring
    const unsigned char* kt = lds + stage * S::kStageBytes + wk * 2 * kTileBytes;
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
    f32x4_t st[kSubs][KB][QB];
    float shift[QB];
#pragma unroll
    for (int u = 0; u < kSubs; ++u) scores(kt + u * SUB * kRowBytes, st[u]);
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      float mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < kSubs; ++u)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, st[u][kb][qb][r]);
      raise(qb, mx * a.scale);
      shift[qb] = m_run[qb] == -INFINITY ? 0.0f : m_run[qb] * kLog2e;
    }
#pragma unroll
    for (int u = 0; u < kSubs; ++u)
      weigh(std::false_type{}, kt + kTileBytes + u * SUB * kRowBytes, st[u], scale_log2, shift);
  }

  for (int step = plain_steps; step < nsteps; ++step) {
    __syncthreads();
    const unsigned char* kt = lds + stage * S::kStageBytes + wk * 2 * kTileBytes;
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
    const int part = step / kMaskSteps, in_part = step % kMaskSteps;
    if (MASKED && in_part == kMaskSteps - 1) {
      mask_room[(part + 1) & 1][tid] = mask_next;
      mask_next = mask_of(part + 2);
    }
    const float* masks = MASKED ? &mask_room[part & 1][in_part * S::kStep + wk * KT] : nullptr;  // of the wave's keys
    if constexpr (MASKED) {
      bool open = false, masked = false;  // of this lane's keys: not all masked out, some
      f32x4_t add[kSubs][KB];
#pragma unroll
      for (int u = 0; u < kSubs; ++u)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          add[u][kb] = *reinterpret_cast<const f32x4_t*>(masks + u * SUB + 16 * kb + 4 * g);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            open |= add[u][kb][r] != -INFINITY;
            masked |= add[u][kb][r] == -INFINITY;
          }
        }
      // (Of the padding itself: a mask of -inf in part of that batch 43.7 us, without this 66.)
      if (!__any(open)) continue;
      if ((step0 + step) * S::kStep + (wk + 1) * KT <= piece.length && !__any(masked)) {
        // All nodes see all of them: of padded batches, most (16 sequences, 64 nodes, a mask:
        // 43.6 us; by the selections below, 32 keys at a time, 50.4).
        f32x4_t st[kSubs][KB][QB];
        float shift[QB];
#pragma unroll
        for (int u = 0; u < kSubs; ++u) scores(kt + u * SUB * kRowBytes, st[u]);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          float mx = -INFINITY;
#pragma unroll
          for (int u = 0; u < kSubs; ++u)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                st[u][kb][qb][r] = fmaf(st[u][kb][qb][r], a.scale, add[u][kb][r]);
                mx = fmaxf(mx, st[u][kb][qb][r]);
              }
          raise(qb, mx);
          // The lowest value times log2 e has no place in fp32; less the maximum it has.
          const float m_use = m_run[qb] == -INFINITY ? 0.0f : m_run[qb];
#pragma unroll
          for (int u = 0; u < kSubs; ++u)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
              for (int r = 0; r < 4; ++r) st[u][kb][qb][r] -= m_use;
          shift[qb] = 0.0f;
        }
#pragma unroll
        for (int u = 0; u < kSubs; ++u)
          weigh(std::false_type{}, kt + kTileBytes + u * SUB * kRowBytes, st[u], kLog2e, shift);
        continue;
      }
    }
#pragma unroll 1
    for (int u = 0; u < kSubs; ++u) {
      const int s0 = (step0 + step) * S::kStep + wk * KT + u * SUB;
      if (s0 >= piece.end) break;
      f32x4_t st[KB][QB];
      scores(kt + u * SUB * kRowBytes, st);
      // Scores t = score * scale + mask, -inf where the row is not seen, less the maximum.
      const float* mask = MASKED ? masks + u * SUB : nullptr;
      f32x4_t add[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
        add[kb] = MASKED ? *reinterpret_cast<const f32x4_t*>(mask + 16 * kb + 4 * g) : f32x4_t{0.f, 0.f, 0.f, 0.f};
      const int j0 = s0 - piece.length;  // of the first key, as a node
      const uint32_t inside = piece.end - s0 >= 32 ? ~0u : (1u << (piece.end - s0)) - 1;
      uint32_t seen[QB];
      bool hidden = false;
      float shift[QB];
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        seen[qb] = inside;
        if (j0 > -32) {
          if (a.tree == nullptr) {
            const int n = node[qb] - j0 + 1;
            seen[qb] &= n >= 32 ? ~0u : (n <= 0 ? 0u : (1u << n) - 1);
          } else {
            const uint32_t* row = tree_bits + (node[qb] - node0) * kMaxWords + ((j0 + 32) >> 5);
            seen[qb] &= __builtin_amdgcn_alignbit(row[1], row[0], (j0 + 32) & 31);
          }
        }
        hidden |= (~seen[qb] & (SUB == 32 ? ~0u : (1u << SUB) - 1)) != 0;
        const uint32_t mine = seen[qb] >> (4 * g);
        float mx = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            hidden |= MASKED && add[kb][r] == -INFINITY;
            const bool sees = (mine >> (16 * kb + r) & 1) != 0 && (!MASKED || add[kb][r] != -INFINITY);
            const float t = sees ? fmaf(st[kb][qb][r], a.scale, add[kb][r]) : -INFINITY;
            st[kb][qb][r] = t;
            mx = fmaxf(mx, t);
          }
        raise(qb, mx);
        const float m_use = m_run[qb] == -INFINITY ? 0.0f : m_run[qb];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) st[kb][qb][r] -= m_use;
        shift[qb] = 0.0f;
      }
      const unsigned char* vt = kt + kTileBytes + u * SUB * kRowBytes;
      bool dirty = false;
      if (__any(hidden)) {
        // A weight of zero times NaN or infinity is NaN: where a row is hidden from a
        // query, V is searched for them.
        bool special = false;
        for (int at = lane * 16; at < SUB * kRowBytes; at += 1024) {
          const uint4 v = lds_read(vt + at);
          special |= has_special<T>(v.x) || has_special<T>(v.y) || has_special<T>(v.z) || has_special<T>(v.w);
        }
        dirty = __any(special);
      }
      if (__builtin_expect(!dirty, 1)) {
        weigh(std::false_type{}, vt, st, kLog2e, shift);
        continue;
      }
      weigh(std::true_type{}, vt, st, kLog2e, shift);
      // V's NaNs and infinities, for the queries that see their rows.
#pragma unroll 1
      for (int row = 0; row < SUB; ++row) {
        const bool open = !MASKED || mask[row] != -INFINITY;
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          const bool sees = open && (seen[qb] >> row & 1) != 0;
#pragma unroll
          for (int i = 0; i < S::kQuads; ++i) {
            const int dim = quad_dim<T>(i, g);
            const unsigned char* at = vt + row * kRowBytes + (((dim * ES >> 4) ^ S::swizzle(row)) << 4) + (dim * ES & 15);
            T v[4];
            if constexpr (kWide) {
              *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(at);
            } else {
              *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(at);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float f = slc::to_f32(v[e]);
              const float extra = sees && !(fabsf(f) < INFINITY) ? f : 0.0f;
              if constexpr (kWide) {
                acc[4 * (i / 4) + e][qb][i % 4] += extra;
              } else {
                acc[i][qb][e] += extra;
              }
            }
          }
        }
      }
    }
  }

  float l_run[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
    l_run[qb] = kWide ? slc::sum_xor32(slc::sum_xor16(l_part[qb])) : acc[kAcc - 1][qb][0];
  // Quad i of a query block: 4 neighbouring dims.
  auto quad = [&](int i, int qb) {
    if constexpr (kWide) {
      const int d = 4 * (i / 4), r = i % 4;
      return make_float4(acc[d][qb][r], acc[d + 1][qb][r], acc[d + 2][qb][r], acc[d + 3][qb][r]);
    } else {
      return make_float4(acc[i][qb][0], acc[i][qb][1], acc[i][qb][2], acc[i][qb][3]);
    }
  };
  const int own = piece.index == 0 ? piece.head : piece.tail + piece.index - 1;
  const int64_t place = (static_cast<int64_t>(own) * a.kv_heads + kvh) * a.row_blocks + block;
  auto store = [&](int i, int qb, float4 v, float top, float sum) {
    if (!real[qb]) return;
    const int dim = quad_dim<T>(i, g);
    if (count > 1) {
      // As the lanes hold them, so that a wave writes whole lines.
      reinterpret_cast<float4*>(a.partial + place * S::kRows * DP)[((wr * QB + qb) * S::kQuads + i) * 64 + lane] = v;
      if (g == 0 && i == 0) a.stats[place * S::kRows + wr * 16 * QB + 16 * qb + c] = make_float2(top, sum);
    } else {
      T* row = static_cast<T*>(a.output) + b * a.o_sb + head[qb] * a.o_sh + node[qb] * a.o_st;
      store_quad<T>(row, dim, a.head_dim, a.vector_o, divided(v, sum));
    }
  };
  if constexpr (WK == 1) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
      for (int i = 0; i < S::kQuads; ++i) store(i, qb, quad(i, qb), m_run[qb], l_run[qb]);
  } else {
    // The tiles' results meet in LDS, where each wave takes a share of the outputs.
    constexpr int kFloats = S::kQuads * 256 + 128;  // of a wave's query block
    __syncthreads();  // the ring is free
    float* room = reinterpret_cast<float*>(lds) + wr * QB * kFloats;
    constexpr int kTile = WR * QB * kFloats;  // from one tile's results to the next's
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      float* mine = room + wk * kTile + qb * kFloats;
#pragma unroll
      for (int i = 0; i < S::kQuads; ++i) reinterpret_cast<float4*>(mine)[i * 64 + lane] = quad(i, qb);
      mine[S::kQuads * 256 + lane] = m_run[qb];
      mine[S::kQuads * 256 + 64 + lane] = l_run[qb];
    }
    __syncthreads();
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const float* from = room + qb * kFloats;
      float top = -INFINITY, sum = 0.0f, w[WK];
#pragma unroll
      for (int k = 0; k < WK; ++k) {
        w[k] = from[k * kTile + S::kQuads * 256 + lane];
        top = fmaxf(top, w[k]);
      }
      const float use = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int k = 0; k < WK; ++k) {
        w[k] = __builtin_amdgcn_exp2f((w[k] - use) * kLog2e);
        sum = fmaf(w[k], from[k * kTile + S::kQuads * 256 + 64 + lane], sum);
      }
#pragma unroll
      for (int n = 0; n < (S::kQuads + WK - 1) / WK; ++n) {
        // One of wave wk's, a quad number known only at run time.
        const int i = n * WK + wk;
        if (i >= S::kQuads) break;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < WK; ++k) {
          const float4 o = reinterpret_cast<const float4*>(from + k * kTile)[i * 64 + lane];
          v.x = fmaf(w[k], o.x, v.x);
          v.y = fmaf(w[k], o.y, v.y);
          v.z = fmaf(w[k], o.z, v.z);
          v.w = fmaf(w[k], o.w, v.w);
        }
        store(i, qb, v, top, sum);
      }
    }
  }
  if (count == 1 || a.counters == nullptr) return;

  // The last of a sequence's pieces to arrive puts all of them together: every wave's
  // results come before the barrier, each piece's count releases them, and the last one
  // acquires them all.
  __syncthreads();
  if (tid == 0) {
    int* const counter = a.counters + (piece.sequence * a.kv_heads + kvh) * a.row_blocks + block;
    arrived = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_AGENT);
    if (arrived == count - 1) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (__builtin_amdgcn_readfirstlane(arrived) != count - 1) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  const int units = block_units<DP, S::kRows>(a, block);
#pragma unroll 1
  for (int unit = wave; unit < units; unit += 2 * S::kConsumers)
    merge_units<T, DP, S::kRows, 2, 4>(a, b, kvh, block, piece.head, piece.tail, count, unit, S::kConsumers, units);
}

template <typename T, int DP, int QB, int WR, int KT>
int launch_shape(const TreeArgs& a, hipStream_t stream) {
  using S = Shape<T, DP, QB, WR, KT>;
  const float min_steps = static_cast<float>((min_piece_rows(S::kRowBytes) + S::kStep - 1) / S::kStep);
  const auto kernel = a.mask != nullptr ? tree_attention_kernel<T, DP, QB, WR, KT, true>
                                        : tree_attention_kernel<T, DP, QB, WR, KT, false>;
  hipLaunchKernelGGL(kernel, dim3(a.kv_heads, a.slots, a.row_blocks), dim3(S::kThreads), 0, stream, a, min_steps);
  const int status = slc_host::check_launch("tree attention");
  // Its pieces are put together by the last of them, or by another kernel; there are none
  // where every sequence is one.
  if (status != SLC_OK || a.counters != nullptr || a.slots <= a.batch || a.rows <= min_piece_rows(S::kRowBytes)) return status;
  hipLaunchKernelGGL((tree_merge_kernel<T, DP, S::kRows>),
                     dim3((S::kRows * DP / 256 + 3) / 4, a.kv_heads * a.row_blocks, a.batch), dim3(256), 0, stream, a);
  return slc_host::check_launch("tree attention merge");
}

// The waves along the rows and their query blocks, by the query rows and the padded
// row's bytes.  Of 128-byte rows a wave takes two blocks of 16 query rows, each K and V
// fragment from LDS serving both (in a graph, 14 query heads on 2, bf16: 32 sequences, 16
// nodes, 112 rows 32.7 us, with one 35.8; 16 sequences, 64 nodes 30.6 us, with one 47.3),
// but one of up to 16 rows (32 sequences, 2 nodes 24.1 us, with two 24.5) and from 33 to 64,
// where four waves along the rows are as many as with two of 128 (one sequence, 8 nodes
// 10.2 us, with two 10.9).  Wider rows leave no registers for two.
template <int BYTES>
constexpr bool kTwo = BYTES <= 128;
template <int BYTES>
constexpr int most_waves() { return BYTES <= 256 ? 8 : 4; }

template <typename T, int DP>
int rows_per_block(int rows) {
  constexpr int kBytes = DP * static_cast<int>(sizeof(T));
  constexpr int kWhole = (kTwo<kBytes> ? 32 : 16) * most_waves<kBytes>();
  for (int size = 16; size < kWhole; size *= 2)
    if (rows <= size) return size;
  // Whole blocks where they need no more padding than halves.
  return (rows + kWhole - 1) / kWhole * 2 == (rows + kWhole / 2 - 1) / (kWhole / 2) ? kWhole : kWhole / 2;
}

// Tiles are of 32 keys (16 of rows of 1024 bytes); of 64 where all eight waves lie along
// 128-byte rows, a step of 32 keys being short (16 sequences, 64 nodes 30.6 us, with 32
// keys 31.8; where two tiles are side by side 32 keys are better: 8 sequences, 16 nodes
// 14.0 us, with 64 keys 15.1).
template <typename T, int DP>
int launch_dim(const TreeArgs& a, int rows, hipStream_t stream) {
  constexpr int kBytes = DP * static_cast<int>(sizeof(T));
  constexpr int kKeys = kBytes == 1024 ? 16 : 32;
  if (rows == 16) return launch_shape<T, DP, 1, 1, kKeys>(a, stream);
  if constexpr (kTwo<kBytes>) {
    if (rows == 32) return launch_shape<T, DP, 2, 1, kKeys>(a, stream);
    if (rows == 64) return launch_shape<T, DP, 1, 4, kKeys>(a, stream);
    if (rows == 128) return launch_shape<T, DP, 2, 4, kKeys>(a, stream);
    return launch_shape<T, DP, 2, 8, 64>(a, stream);
  } else {
    if (rows == 32) return launch_shape<T, DP, 1, 2, kKeys>(a, stream);
    if constexpr (most_waves<kBytes>() == 8)
      if (rows == 128) return launch_shape<T, DP, 1, 8, kKeys>(a, stream);
    return launch_shape<T, DP, 1, 4, kKeys>(a, stream);
  }
}

template <typename T>
Plan plan_impl(int rows, int head_dim) {
  if (head_dim <= 64) return {rows_per_block<T, 64>(rows), 64};
  if (head_dim <= 128) return {rows_per_block<T, 128>(rows), 128};
  return {rows_per_block<T, 256>(rows), 256};
}
template <typename T>
int launch_impl(const TreeArgs& a, const Plan& plan, hipStream_t stream) {
  if (plan.padded_dim == 64) return launch_dim<T, 64>(a, plan.rows_per_block, stream);
  if (plan.padded_dim == 128) return launch_dim<T, 128>(a, plan.rows_per_block, stream);
  return launch_dim<T, 256>(a, plan.rows_per_block, stream);
}

}  // namespace
}  // namespace slc_tree
