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
// so K and V are read once for all of them.  One producer wave streams steps of K and V
// into an LDS ring with direct-to-LDS loads (16-byte chunks, XOR-swizzled by row; rows
// past the last one read as zero).  WR x WK consumer waves own 16 QB query rows and one
// of the step's WK tiles of KT keys each, so few query rows still keep all waves busy:
//  * S^T[key, query] = K . Q^T, Q^T in registers;
//  * softmax with a running maximum that moves only when a score passes it by more than
//    kThreshold, in fp32, maxima in units of the score itself so that a mask of the
//    type's lowest value stays finite;
//  * O^T[dim, query] += V^T . P^T: the score tile's C layout is the product's B layout
//    once V's rows are taken in the same order.
// The WK partial results meet in LDS; the pieces' partial results, where a sequence
// has several, in tree_merge_kernel.
#pragma once
#include <cmath>
#include <type_traits>

#include "tree_args.hpp"

namespace slc_tree {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kThreshold = 5.5f;  // weights stay under e^5.5 = 245, fp16's range is 65504
constexpr int kMinPieceRows = 256;

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

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) v += __shfl_xor(v, offset, 64);
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_scan(int v) {  // sums up to and with this lane
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int offset = 1; offset < 64; offset <<= 1) {
    const int below = __shfl_up(v, offset, 64);
    if (lane >= offset) v += below;
  }
  return v;
}

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
// A sum of weights of zero: a node that sees no row, NaN.
__device__ __forceinline__ float4 divided(float4 v, float sum) {
  const float by = sum == 0.0f ? __builtin_nanf("") : 1.0f / sum;
  return make_float4(v.x * by, v.y * by, v.z * by, v.w * by);
}

struct Piece {
  int sequence;  // -1: none
  int index, count, first;
  int length, end;  // rows of the sequence, and with its nodes'
};

// The piece of slot x.  Sequences are cut into pieces of at most q steps, q the smallest
// tried for which all pieces fit the slots; every wave finds its own for itself.
template <int STEP>
__device__ __forceinline__ Piece find_piece(const TreeArgs& a, int x, int min_steps) {
  const int lane = threadIdx.x & 63;
  auto bounds = [&](int b, int& length, int& end) {
    const int64_t n = slc::load_length(a.lengths, b, a.lengths_dtype);
    const int64_t rows = a.rows;
    length = static_cast<int>(n < 0 ? 0 : (n > rows ? rows : n));
    end = static_cast<int>(length + a.nodes < rows ? length + a.nodes : rows);
  };
  auto steps_of = [&](int b) {
    if (b >= a.batch) return 0;
    int length, end;
    bounds(b, length, end);
    return end > STEP ? (end + STEP - 1) / STEP : 1;
  };
  const int own = steps_of(lane);  // of the first 64 sequences
  int64_t total = 0;
  for (int base = 0; base < a.batch; base += 64) total += wave_sum(base == 0 ? own : steps_of(base + lane));
  int q = static_cast<int>((total + a.slots - 1) / a.slots);
  q = q < min_steps ? min_steps : q;
  auto pieces_of = [&](int n) { return n == 0 ? 0 : (n + q - 1) / q; };
  for (;;) {
    int64_t pieces = 0;
    for (int base = 0; base < a.batch; base += 64)
      pieces += wave_sum(pieces_of(base == 0 ? own : steps_of(base + lane)));
    if (pieces <= a.slots) break;
    q += (q + 7) / 8;
  }
  Piece p{-1, 0, 0, 0, 0, 0};
  int before = 0;
  for (int base = 0; base < a.batch; base += 64) {
    const int n = pieces_of(base == 0 ? own : steps_of(base + lane));
    const int upto = before + wave_scan(n);
    const uint64_t hits = __ballot(upto > x);
    if (hits != 0) {
      const int at = __builtin_ctzll(hits);
      p.sequence = base + at;
      p.count = __builtin_amdgcn_readlane(n, at);
      p.first = __builtin_amdgcn_readlane(upto, at) - p.count;
      p.index = x - p.first;
      bounds(p.sequence, p.length, p.end);
      p.length = __builtin_amdgcn_readfirstlane(p.length);
      p.end = __builtin_amdgcn_readfirstlane(p.end);
      break;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return p;
}

// Sizes of a kernel: DP the padded head dim, QB blocks of 16 query rows a wave, WR waves
// along the rows, KT keys a tile.
template <typename T, int DP, int QB, int WR, int KT>
struct Shape {
  static constexpr bool kWide = sizeof(T) == 4;
  static constexpr int kRowBytes = DP * static_cast<int>(sizeof(T));
  static constexpr int kTileBytes = KT * kRowBytes;  // of K or of V
  // Tiles side by side: eight waves (four of wide rows, whose registers no more than
  // two a SIMD have), 64 KB a step at most.
  static constexpr int kWaves = kRowBytes <= 256 ? 8 : 4;
  static constexpr int kFit = 65536 / (2 * kTileBytes);
  static constexpr int WK = kWaves / WR < kFit ? kWaves / WR : kFit;
  static constexpr int kConsumers = WR * WK;
  static constexpr int kThreads = (kConsumers + 1) * 64;
  static constexpr int kStep = WK * KT;
  static constexpr int kStageBytes = WK * 2 * kTileBytes;
  static constexpr int kStages = kStageBytes <= 16384 ? 4 : (kStageBytes <= 32768 ? 3 : 2);
  static constexpr int kOps = kStageBytes / 1024;  // loads of a step
  static constexpr int kRows = 16 * QB * WR;
  static constexpr int kQuads = DP / 16;           // float4 of a lane's outputs per query block
  static constexpr int kMergeBytes = WK > 1 ? (WK - 1) * WR * QB * (kQuads * 4 + 2) * 256 : 0;
  static constexpr int kLds = kStages * kStageBytes > kMergeBytes ? kStages * kStageBytes : kMergeBytes;
  static_assert((kStages - 2) * kOps < 64, "the wait counts at most 63 loads");
  static_assert(kLds <= 160 * 1024, "LDS");
};

template <typename T, int DP, int QB, int WR, int KT>
__global__ __launch_bounds__((Shape<T, DP, QB, WR, KT>::kThreads)) void tree_attention_kernel(TreeArgs a, int min_steps) {
  using S = Shape<T, DP, QB, WR, KT>;
  constexpr bool kWide = S::kWide;
  constexpr int WK = S::WK, KB = KT / 16;
  constexpr int kRowBytes = S::kRowBytes, kTileBytes = S::kTileBytes;
  constexpr int kChunks = kRowBytes / 16, kOpRows = 1024 / kRowBytes;
  constexpr int ES = sizeof(T);
  __shared__ __attribute__((aligned(16))) unsigned char lds[S::kLds];

  // Row blocks of one piece run on one XCD (workgroup ids that differ by 8), whose L2
  // then holds the K and V rows that they share.
  const int id = blockIdx.x;
  const int across = 8 * a.row_blocks;
  const int unit = id / across * 8 + id % across % 8;
  const int block = id % across / 8;
  const int kvh = unit % a.kv_heads;
  const int slot = unit / a.kv_heads;
  if (slot >= a.slots) return;
  const Piece piece = find_piece<S::kStep>(a, slot, min_steps);
  if (piece.sequence < 0) return;
  const int64_t b = piece.sequence;
  const int steps = piece.end > S::kStep ? (piece.end + S::kStep - 1) / S::kStep : 1;
  const int step0 = static_cast<int>(static_cast<int64_t>(steps) * piece.index / piece.count);
  const int nsteps = static_cast<int>(static_cast<int64_t>(steps) * (piece.index + 1) / piece.count) - step0;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (tid == 0 && piece.index == 0 && kvh == 0 && block == 0) a.pieces[b] = make_int2(piece.first, piece.count);

  if (wave == S::kConsumers) {
    // ---- producer -------------------------------------------------------------
    constexpr int kTileOps = kTileBytes / 1024;
    const T* kbase = static_cast<const T*>(a.key) + kvh * a.kv_sh;
    const T* vbase = static_cast<const T*>(a.value) + kvh * a.kv_sh;
    const int row_in_op = lane / kChunks;
    const bool paged = a.table != nullptr;
    const int page_rows = paged ? 1 << a.page_shift : S::kStep;
    const int segment = page_rows < S::kStep ? page_rows : S::kStep;  // rows of a step with one base
    const int row_bytes = static_cast<int>(a.kv_ss) * ES;
    // Lane L of load n fills row kOpRows n + L / kChunks of the step, chunk L % kChunks, with
    // that row's chunk (L % kChunks) ^ (row & 7); columns past the head dim lie past every range.
    // Rows kOpRows apart have another swizzle unless kOpRows is a multiple of 8.
    constexpr int kSwizzles = kOpRows >= 8 ? 1 : 8 / kOpRows;
    int voffset[kSwizzles];
#pragma unroll
    for (int i = 0; i < kSwizzles; ++i) {
      const int row = i * kOpRows + row_in_op;
      const int chunk = (lane % kChunks) ^ (row & 7);
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
      if (a.vector_kv) {
        for (int first = 0; first < S::kStep; first += segment) {
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
        for (int n = 0; n < S::kOps / 2; ++n) {
          const int row = n * kOpRows + row_in_op;
          const int chunk = (lane % kChunks) ^ (row & 7);
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
  int node[QB], head[QB];
  bool real[QB];
  // Q^T: 16-bit types hold 8 dims 32 kk + 8 g of a block, fp32 4 dims 16 kk + 4 g.
  constexpr int kDims = kWide ? 16 : 32, kParts = DP / kDims;
  uint4 qv[QB][kParts];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int row = block * S::kRows + wr * 16 * QB + 16 * qb + c;
    real[qb] = row < rows;
    node[qb] = real[qb] ? row / group : 0;
    head[qb] = kvh * group + (real[qb] ? row % group : 0);
    const T* qp = static_cast<const T*>(a.query) + b * a.q_sb + head[qb] * a.q_sh + node[qb] * a.q_st;
#pragma unroll
    for (int kk = 0; kk < kParts; ++kk) {
      constexpr int kPer = 16 / ES;
      const int dim = kk * kDims + kPer * g;
      if (a.vector_q) {
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
  // First dim of a lane's i-th four neighbouring outputs.
  auto quad_dim = [&](int i) { return kWide ? 64 * (i / 4) + 16 * g + 4 * (i % 4) : 16 * i + 4 * g; };
  const uint32_t one2 = std::is_same_v<T, slc::bf16_t> ? 0x3f803f80u : 0x3c003c00u;
  const uint4 ones = make_uint4(one2, one2, one2, one2);
  const float scale_log2 = a.scale * kLog2e;

  for (int step = 0; step < nsteps; ++step) {
    __syncthreads();  // this step's tiles are in the ring
    const int s0 = (step0 + step) * S::kStep + wk * KT;
    if (s0 >= piece.end) continue;
    const unsigned char* kt = lds + step % S::kStages * S::kStageBytes + wk * 2 * kTileBytes;
    const unsigned char* vt = kt + kTileBytes;

    f32x4_t st[KB][QB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) st[kb][qb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int kk = 0; kk < kParts; ++kk) {
        const uint4 ka = lds_read(kt + (16 * kb + c) * kRowBytes + (((4 * kk + g) ^ (c & 7)) << 4));
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          if constexpr (kWide) {
            st[kb][qb] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ka.x), __uint_as_float(qv[qb][kk].x), st[kb][qb], 0, 0, 0);
            st[kb][qb] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ka.y), __uint_as_float(qv[qb][kk].y), st[kb][qb], 0, 0, 0);
            st[kb][qb] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ka.z), __uint_as_float(qv[qb][kk].z), st[kb][qb], 0, 0, 0);
            st[kb][qb] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ka.w), __uint_as_float(qv[qb][kk].w), st[kb][qb], 0, 0, 0);
          } else {
            st[kb][qb] = mfma(T{}, ka, qv[qb][kk], st[kb][qb]);
          }
        }
      }

    // A weight is exp2(score * factor - shift).
    float factor = scale_log2, shift[QB];
    int seen_bits[QB];
    bool dirty = false;
    const bool plain = a.mask == nullptr && s0 + KT <= piece.length;
    if (plain) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        float mx = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, st[kb][qb][r]);
        mx *= a.scale;
        if (__any(mx > m_run[qb] + kThreshold)) {
          mx = slc::max_xor32(slc::max_xor16(mx));
          const float m_new = fmaxf(m_run[qb], mx);
          const float alpha = __builtin_amdgcn_exp2f((m_run[qb] - (m_new == -INFINITY ? 0.0f : m_new)) * kLog2e);
#pragma unroll
          for (int i = 0; i < kAcc; ++i) acc[i][qb] = acc[i][qb] * alpha;
          l_part[qb] *= alpha;
          m_run[qb] = m_new;
        }
        shift[qb] = m_run[qb] == -INFINITY ? 0.0f : m_run[qb] * kLog2e;
      }
    } else {
      // The tail of a sequence, or a mask: scores t = score * scale + mask, -inf where
      // the row is not seen, then t - max.
      factor = kLog2e;
      bool hidden = false;
      float add[KB][4];
      auto masks = [&](auto load) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int s = s0 + 16 * kb + 4 * g + r;
            add[kb][r] = s < piece.end ? load(s) : -INFINITY;
            hidden |= add[kb][r] == -INFINITY;
          }
      };
      const int64_t mask_at = b * a.mask_sb;
      if (a.mask == nullptr) {
        masks([](int) { return 0.0f; });
      } else if (a.mask_dtype == SLC_F32) {
        masks([&](int s) { return static_cast<const float*>(a.mask)[mask_at + s * a.mask_ss]; });
      } else if (a.mask_dtype == SLC_BF16) {
        masks([&](int s) { return slc::to_f32(static_cast<const slc::bf16_t*>(a.mask)[mask_at + s * a.mask_ss]); });
      } else {
        masks([&](int s) { return slc::to_f32(static_cast<const slc::f16_t*>(a.mask)[mask_at + s * a.mask_ss]); });
      }
      const bool tail = s0 + KT > piece.length;
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        float mx = -INFINITY;
        seen_bits[qb] = 0;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            bool seen = add[kb][r] != -INFINITY;
            const int j = s0 + 16 * kb + 4 * g + r - piece.length;
            if (tail && seen && j >= 0) {
              seen = a.tree == nullptr ? j <= node[qb]
                                       : a.tree[b * a.tree_sb + node[qb] * a.tree_si + j * a.tree_sj] != 0;
              hidden |= !seen;
            }
            seen_bits[qb] |= static_cast<int>(seen) << (4 * kb + r);
            const float t = seen ? fmaf(st[kb][qb][r], a.scale, add[kb][r]) : -INFINITY;
            st[kb][qb][r] = t;
            mx = fmaxf(mx, t);
          }
        if (__any(mx > m_run[qb] + kThreshold)) {
          mx = slc::max_xor32(slc::max_xor16(mx));
          const float m_new = fmaxf(m_run[qb], mx);
          const float alpha = __builtin_amdgcn_exp2f((m_run[qb] - (m_new == -INFINITY ? 0.0f : m_new)) * kLog2e);
#pragma unroll
          for (int i = 0; i < kAcc; ++i) acc[i][qb] = acc[i][qb] * alpha;
          l_part[qb] *= alpha;
          m_run[qb] = m_new;
        }
        const float m_use = m_run[qb] == -INFINITY ? 0.0f : m_run[qb];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) st[kb][qb][r] -= m_use;
        shift[qb] = 0.0f;
      }
      if (__any(hidden)) {
        // A weight of zero times NaN or infinity is NaN: where some row of the tile is
        // hidden from some query, V is searched for them.
        bool special = false;
        for (int at = lane * 16; at < kTileBytes; at += 1024) {
          const uint4 v = lds_read(vt + at);
          special |= has_special<T>(v.x) || has_special<T>(v.y) || has_special<T>(v.z) || has_special<T>(v.w);
        }
        dirty = __any(special);
      }
    }

    // O^T += V^T . P^T; DIRTY: without V's NaNs and infinities.
    auto weigh = [&](auto dirty_tag) {
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
              uint4 va = lds_read(vt + row * kRowBytes + (((16 * d + c) ^ (row & 7)) << 4));
              if constexpr (kDirty) va = without_special<T>(va);
#pragma unroll
              for (int qb = 0; qb < QB; ++qb) {
                acc[4 * d][qb] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(va.x), p[qb], acc[4 * d][qb], 0, 0, 0);
                acc[4 * d + 1][qb] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(va.y), p[qb], acc[4 * d + 1][qb], 0, 0, 0);
                acc[4 * d + 2][qb] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(va.z), p[qb], acc[4 * d + 2][qb], 0, 0, 0);
                acc[4 * d + 3][qb] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(va.w), p[qb], acc[4 * d + 3][qb], 0, 0, 0);
              }
            }
          }
      } else {
#pragma unroll
        for (int half = 0; half < KB / 2; ++half) {
          uint4 pv[QB];
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) {
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              p[i] = __builtin_amdgcn_exp2f(fmaf(st[2 * half + i / 4][qb][i % 4], factor, -shift[qb]));
            pv[qb] = make_uint4(slc::pack2<T>(p[0], p[1]), slc::pack2<T>(p[2], p[3]), slc::pack2<T>(p[4], p[5]),
                                slc::pack2<T>(p[6], p[7]));
          }
          // Lane c of group g addresses 4 dims of key 4 g + c / 4 and gets dim c of the
          // group's 4 keys; the second read's keys lie 16 further.
          const int row = 32 * half + 4 * g + (c >> 2);
#pragma unroll
          for (int i = 0; i < S::kQuads; ++i) {
            const int dim = 16 * i + 4 * (c & 3);
            const unsigned char* at = vt + row * kRowBytes + (((dim >> 3) ^ (row & 7)) << 4) + (dim & 7) * 2;
            const uint2 lo = lds_read_tr(at), hi = lds_read_tr(at + 16 * kRowBytes);
            uint4 va = make_uint4(lo.x, lo.y, hi.x, hi.y);
            if constexpr (kDirty) va = without_special<T>(va);
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) acc[i][qb] = mfma(T{}, va, pv[qb], acc[i][qb]);
          }
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) acc[S::kQuads][qb] = mfma(T{}, ones, pv[qb], acc[S::kQuads][qb]);
        }
      }
    };
    if (!dirty) {
      weigh(std::false_type{});
    } else {
      weigh(std::true_type{});
      // V's NaNs and infinities, for the queries that see their rows.
#pragma unroll 1
      for (int row = 0; row < KT; ++row) {
        // Row 16 kb + 4 from + r: bit 4 kb + r of the lanes of group `from`.
        const int from = (row & 15) >> 2, bit = (row >> 4) * 4 + (row & 3);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          const bool seen = (__shfl(seen_bits[qb], 16 * from + c, 64) >> bit & 1) != 0;
#pragma unroll
          for (int i = 0; i < S::kQuads; ++i) {
            const int dim = quad_dim(i);
            const unsigned char* at = vt + row * kRowBytes + (((dim * ES >> 4) ^ (row & 7)) << 4) + (dim * ES & 15);
            T v[4];
            if constexpr (kWide) {
              *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(at);
            } else {
              *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(at);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float f = slc::to_f32(v[e]);
              const float extra = seen && !(fabsf(f) < INFINITY) ? f : 0.0f;
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
  float4 out[S::kQuads][QB];
#pragma unroll
  for (int i = 0; i < S::kQuads; ++i)
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) out[i][qb] = quad(i, qb);

  if constexpr (WK > 1) {
    // The first tile's waves take in the others' results.
    constexpr int kFloats = S::kQuads * 4 + 2;
    __syncthreads();  // the ring is free
    float* room = reinterpret_cast<float*>(lds);
    if (wk > 0) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        float* mine = room + (((wk - 1) * WR + wr) * QB + qb) * kFloats * 64;
#pragma unroll
        for (int i = 0; i < S::kQuads; ++i) reinterpret_cast<float4*>(mine)[i * 64 + lane] = out[i][qb];
        mine[S::kQuads * 256 + lane] = m_run[qb];
        mine[S::kQuads * 256 + 64 + lane] = l_run[qb];
      }
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      float top = m_run[qb];
#pragma unroll
      for (int k = 1; k < WK; ++k)
        top = fmaxf(top, room[(((k - 1) * WR + wr) * QB + qb) * kFloats * 64 + S::kQuads * 256 + lane]);
      const float use = top == -INFINITY ? 0.0f : top;
      const float own = __builtin_amdgcn_exp2f((m_run[qb] - use) * kLog2e);
      l_run[qb] *= own;
#pragma unroll
      for (int i = 0; i < S::kQuads; ++i) {
        out[i][qb].x *= own;
        out[i][qb].y *= own;
        out[i][qb].z *= own;
        out[i][qb].w *= own;
      }
#pragma unroll 1
      for (int k = 1; k < WK; ++k) {
        const float* other = room + (((k - 1) * WR + wr) * QB + qb) * kFloats * 64;
        const float w = __builtin_amdgcn_exp2f((other[S::kQuads * 256 + lane] - use) * kLog2e);
        l_run[qb] = fmaf(w, other[S::kQuads * 256 + 64 + lane], l_run[qb]);
#pragma unroll
        for (int i = 0; i < S::kQuads; ++i) {
          const float4 o = reinterpret_cast<const float4*>(other)[i * 64 + lane];
          out[i][qb].x = fmaf(w, o.x, out[i][qb].x);
          out[i][qb].y = fmaf(w, o.y, out[i][qb].y);
          out[i][qb].z = fmaf(w, o.z, out[i][qb].z);
          out[i][qb].w = fmaf(w, o.w, out[i][qb].w);
        }
      }
      m_run[qb] = top;
    }
  }

  const int64_t place = (static_cast<int64_t>(slot) * a.kv_heads + kvh) * a.row_blocks + block;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int row = wr * 16 * QB + 16 * qb + c;
    if (!real[qb]) continue;
    if (piece.count > 1) {
      float* partial = a.partial + (place * S::kRows + row) * DP;
#pragma unroll
      for (int i = 0; i < S::kQuads; ++i) {
        const int dim = quad_dim(i);
        if (dim < a.head_dim) *reinterpret_cast<float4*>(partial + dim) = out[i][qb];
      }
      if (g == 0) a.stats[place * S::kRows + row] = make_float2(m_run[qb], l_run[qb]);
      continue;
    }
    T* op = static_cast<T*>(a.output) + b * a.o_sb + head[qb] * a.o_sh + node[qb] * a.o_st;
#pragma unroll
    for (int i = 0; i < S::kQuads; ++i) {
      const int dim = quad_dim(i);
      store_quad<T>(op, dim, a.head_dim, a.vector_o, divided(out[i][qb], l_run[qb]));
    }
  }
}

// The pieces of a sequence together: a thread per four dims of a row.
template <typename T, int DP, int ROWS>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
  const int64_t b = blockIdx.z;
  const int kvh = blockIdx.y;
  const int2 pieces = a.pieces[b];
  if (pieces.y <= 1) return;
  const int quads = (a.head_dim + 3) / 4;
  const int item = blockIdx.x * 256 + threadIdx.x;
  const int row = item / quads, dim = item % quads * 4;
  const int group = a.q_heads / a.kv_heads;
  if (row >= group * a.nodes) return;
  const int64_t stride = static_cast<int64_t>(a.kv_heads) * a.row_blocks;
  const int64_t place = pieces.x * stride + static_cast<int64_t>(kvh) * a.row_blocks + row / ROWS;
  const float2* stats = a.stats + place * ROWS + row % ROWS;
  const float* partial = a.partial + (place * ROWS + row % ROWS) * DP + dim;
  float top = -INFINITY, sum = 0.0f;
  float4 out = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int kBatch = 8;
  for (int first = 0; first < pieces.y; first += kBatch) {
    float2 s[kBatch];
    float4 o[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t at = (first + i < pieces.y ? first + i : first) * stride * ROWS;
      s[i] = stats[at];
      o[i] = *reinterpret_cast<const float4*>(partial + at * DP);
      if (first + i >= pieces.y) s[i] = make_float2(-INFINITY, 0.0f);
    }
    float most = top;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) most = fmaxf(most, s[i].x);
    const float use = most == -INFINITY ? 0.0f : most;
    const float own = __builtin_amdgcn_exp2f((top - use) * kLog2e);
    top = most;
    sum *= own;
    out = make_float4(out.x * own, out.y * own, out.z * own, out.w * own);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (first + i >= pieces.y) continue;
      const float w = __builtin_amdgcn_exp2f((s[i].x - use) * kLog2e);
      sum = fmaf(w, s[i].y, sum);
      out.x = fmaf(w, o[i].x, out.x);
      out.y = fmaf(w, o[i].y, out.y);
      out.z = fmaf(w, o[i].z, out.z);
      out.w = fmaf(w, o[i].w, out.w);
    }
  }
  const int node = row / group, head = kvh * group + row % group;
  store_quad<T>(static_cast<T*>(a.output) + b * a.o_sb + head * a.o_sh + node * a.o_st, dim, a.head_dim, a.vector_o,
                divided(out, sum));
}

template <typename T, int DP, int QB, int WR, int KT>
int launch_shape(const TreeArgs& a, hipStream_t stream) {
  using S = Shape<T, DP, QB, WR, KT>;
  // Groups of 8 units (a piece of a KV head), each with its row blocks.
  const int units = a.slots * a.kv_heads;
  const int min_steps = (kMinPieceRows + S::kStep - 1) / S::kStep;
  hipLaunchKernelGGL((tree_attention_kernel<T, DP, QB, WR, KT>), dim3((units + 7) / 8 * 8 * a.row_blocks),
                     dim3(S::kThreads), 0, stream, a, min_steps);
  int status = slc_host::check_launch("tree attention");
  if (status != SLC_OK || a.slots <= a.batch || (a.rows + S::kStep - 1) / S::kStep <= min_steps) return status;
  const int items = a.q_heads / a.kv_heads * a.nodes * ((a.head_dim + 3) / 4);
  hipLaunchKernelGGL((tree_merge_kernel<T, DP, S::kRows>), dim3((items + 255) / 256, a.kv_heads, a.batch), dim3(256), 0,
                     stream, a);
  return slc_host::check_launch("tree attention merge");
}

// Query blocks of 16 rows a wave by the padded row's bytes: two of 128-byte rows (each
// K and V fragment read from LDS serves both); wider rows leave no registers for that.
template <int BYTES>
constexpr int query_blocks() { return BYTES <= 128 ? 2 : 1; }
template <int BYTES>
constexpr int most_waves() { return BYTES <= 256 ? 8 : 4; }

template <typename T, int DP>
int rows_per_block(int rows) {
  constexpr int kBytes = DP * static_cast<int>(sizeof(T));
  constexpr int kRows = 16 * query_blocks<kBytes>(), kMost = most_waves<kBytes>();
  if (rows <= 16) return 16;
  for (int wr = 1; wr < kMost; wr *= 2)
    if (rows <= kRows * wr) return kRows * wr;
  // Whole blocks where they need no more padding than halves.
  const int whole = kRows * kMost, half = whole / 2;
  return (rows + whole - 1) / whole * 2 == (rows + half - 1) / half ? whole : half;
}

template <typename T, int DP>
int launch_dim(const TreeArgs& a, int rows, hipStream_t stream) {
  constexpr int kBytes = DP * static_cast<int>(sizeof(T));
  constexpr int kQb = query_blocks<kBytes>(), kRows = 16 * kQb;
  constexpr int kKeys = kBytes == 1024 ? 16 : 32;
  if constexpr (kQb > 1)
    if (rows == 16) return launch_shape<T, DP, 1, 1, kKeys>(a, stream);
  if (rows == kRows) return launch_shape<T, DP, kQb, 1, kKeys>(a, stream);
  if (rows == 2 * kRows) return launch_shape<T, DP, kQb, 2, kKeys>(a, stream);
  if constexpr (most_waves<kBytes>() > 4)
    if (rows == 8 * kRows) return launch_shape<T, DP, kQb, 8, kKeys>(a, stream);
  return launch_shape<T, DP, kQb, 4, kKeys>(a, stream);
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
