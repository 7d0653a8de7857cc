// linear_q8: Y[M, N] = (X[M, K] . W[N, K]^T) * sx[M] * sw[N] (+ bias[N]), X and
// W 8-bit codes, the sum exact in 32-bit integers.
//
// The sum of a dot product of codes is a whole number of at most K * 128^2, which
// 32 bits hold up to K = 131071; so its value does not depend on the order in
// which tiles, waves or k-steps add it, and every variant below gives the same
// bits.  The epilogue is fp32: float(sum) * sx * sw + bias, one rounding to the
// output type.
//
// X and W rows are K-contiguous, the operand layout of v_mfma_i32_16x16x64_i8
// (16 consecutive k per lane), so neither operand is transposed.
#include <type_traits>

#include "common.hpp"

namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));

constexpr int kBK = 128;           // k per tile row: 128 bytes
constexpr int kChunks = kBK / 16;  // 16-byte chunks per tile row

// Byte offset of (row, 16-byte chunk) in a tile, swizzled so that 16 rows' reads
// of one chunk fall on all banks.
__device__ __forceinline__ int lds_offset(int row, int chunk) {
  return row * kBK + ((chunk ^ (row & 7)) << 4);
}

__device__ __forceinline__ i32x4_t mfma(i32x4_t a, i32x4_t b, i32x4_t c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// float(sum) * sx * sw + bias; the last two in one fma (and one rounding) in
// every kernel, so that all give the same bits.  The result is an fp32 value before
// it is rounded to T: the compiler would else round fp16 outputs from the unrounded
// fma, where it sees both.
template <typename T>
__device__ __forceinline__ float finish(int sum, float sx, float sw, float bias) {
  float y = fmaf(static_cast<float>(sum) * sx, sw, bias);
  if constexpr (std::is_same<T, slc::f16_t>::value) asm("" : "+v"(y));
  return y;
}

struct Problem {
  const int8_t* x;
  const float* sx;
  const int8_t* w;
  const float* sw;
  const void* bias;
  void* y;
  int M, N, K;
  int64_t x_rs, y_rs;
};

// ---- any sizes, strides and alignment -----------------------------------------------
// 16 codes of a row of K from code k on, zeros past K: all but the last chunk as they lie
// (at any address), the last as the 16 codes that end the row, moved down by `shift`.  No
// load leaves the row, and none waits for a branch.
struct Chunk {
  int at, shift;
  __device__ __forceinline__ Chunk(int k, int K) : at(k < K - 16 ? k : K - 16), shift(k - at < 16 ? k - at : 16) {}
};
__device__ __forceinline__ uint4 moved_down(const uint4& v, int shift) {
  uint64_t lo = static_cast<uint64_t>(v.y) << 32 | v.x, hi = static_cast<uint64_t>(v.w) << 32 | v.z;
  const int bits = 8 * (shift & 7);
  if (shift >= 8) {
    lo = hi;
    hi = 0;
  }
  if (shift >= 16) lo = 0;
  if (bits > 0) {
    lo = lo >> bits | hi << (64 - bits);
    hi >>= bits;
  }
  return make_uint4(static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32), static_cast<uint32_t>(hi),
                    static_cast<uint32_t>(hi >> 32));
}
// A row of fewer than 16 codes.
__device__ __forceinline__ uint4 short_row(const int8_t* p, int K) {
  uint32_t word[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 15; ++i)
    if (i < K) word[i / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(p[i])) << (8 * (i % 4));
  return make_uint4(word[0], word[1], word[2], word[3]);
}

// BM x BN tiles staged through registers into one LDS tile pair, the next k-tile on its
// way while this one is multiplied; four waves of 2 x 2.  Rows past M and N repeat the
// last one (their outputs are not stored).  4096 x 9727 x 1001 91 us (880 TOPS), bound by
// unaligned loads; 301 x 1003 x 1001 7.7, by the latency of eight k-tiles one after the other.
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256) void tile_kernel(Problem p) {
  constexpr int TM = BM / 2, TN = BN / 2, FM = TM / 16, FN = TN / 16;
  constexpr int XPT = BM * kChunks / 256, WPT = BN * kChunks / 256;
  constexpr int kStep = 256 / kChunks;  // rows between a thread's chunks
  __shared__ __attribute__((aligned(16))) unsigned char xs[BM * kBK];
  __shared__ __attribute__((aligned(16))) unsigned char ws[BN * kBK];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wm = wave >> 1, wn = wave & 1;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * BM, n0 = static_cast<int64_t>(blockIdx.x) * BN;
  const int row = tid / kChunks, chunk = tid % kChunks;

  const int8_t* xp[XPT];
  const int8_t* wp[WPT];
#pragma unroll
  for (int i = 0; i < XPT; ++i) {
    const int64_t m = m0 + row + kStep * i;
    xp[i] = p.x + (m < p.M ? m : p.M - 1) * p.x_rs;
  }
#pragma unroll
  for (int i = 0; i < WPT; ++i) {
    const int64_t n = n0 + row + kStep * i;
    wp[i] = p.w + (n < p.N ? n : p.N - 1) * p.K;
  }
  uint4 xr[XPT], wr[WPT];
  auto fetch = [&](int k0) {
    const Chunk ch(k0 + chunk * 16, p.K);
#pragma unroll
    for (int i = 0; i < XPT; ++i) __builtin_memcpy(&xr[i], xp[i] + ch.at, 16);
#pragma unroll
    for (int i = 0; i < WPT; ++i) __builtin_memcpy(&wr[i], wp[i] + ch.at, 16);
  };
  auto stash = [&](int k0) {
    if (p.K - k0 < kBK) {  // the last k-tile, and K is no multiple of it
      const Chunk ch(k0 + chunk * 16, p.K);
#pragma unroll
      for (int i = 0; i < XPT; ++i) xr[i] = moved_down(xr[i], ch.shift);
#pragma unroll
      for (int i = 0; i < WPT; ++i) wr[i] = moved_down(wr[i], ch.shift);
    }
#pragma unroll
    for (int i = 0; i < XPT; ++i)
      *reinterpret_cast<uint4*>(xs + lds_offset(row + kStep * i, chunk)) = xr[i];
#pragma unroll
    for (int i = 0; i < WPT; ++i)
      *reinterpret_cast<uint4*>(ws + lds_offset(row + kStep * i, chunk)) = wr[i];
  };

  i32x4_t acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};
  auto multiply = [&]() {
#pragma unroll
    for (int kk = 0; kk < kBK / 64; ++kk) {
      i32x4_t a[FM], b[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i)
        a[i] = *reinterpret_cast<const i32x4_t*>(xs + lds_offset(wm * TM + i * 16 + c, kk * 4 + g));
#pragma unroll
      for (int j = 0; j < FN; ++j)
        b[j] = *reinterpret_cast<const i32x4_t*>(ws + lds_offset(wn * TN + j * 16 + c, kk * 4 + g));
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma(a[i], b[j], acc[i][j]);
    }
  };

  // The wave's scales and bias, requested behind the first loads: lane l holds row l's and
  // column l's.  (Asked for in the epilogue they cost 1 us of 301 x 1003 x 1001's 9.)
  static_assert(TM <= 64 && TN <= 64, "a lane for each row and column");
  float own_x = 0.0f, own_w = 0.0f, own_bias = 0.0f;
  auto scales = [&]() {
    const int64_t m = m0 + wm * TM + lane % TM, n = n0 + wn * TN + lane % TN;
    own_x = p.sx[m < p.M ? m : p.M - 1];
    own_w = p.sw[n < p.N ? n : p.N - 1];
    if (p.bias != nullptr) own_bias = slc::to_f32(static_cast<const T*>(p.bias)[n < p.N ? n : p.N - 1]);
  };
  if (p.K < 16) {
    const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < XPT; ++i)
      *reinterpret_cast<uint4*>(xs + lds_offset(row + kStep * i, chunk)) = chunk == 0 ? short_row(xp[i], p.K) : none;
#pragma unroll
    for (int i = 0; i < WPT; ++i)
      *reinterpret_cast<uint4*>(ws + lds_offset(row + kStep * i, chunk)) = chunk == 0 ? short_row(wp[i], p.K) : none;
    scales();
    __syncthreads();
    multiply();
  } else {
    fetch(0);
    scales();
    for (int k0 = 0; k0 < p.K; k0 += kBK) {
      stash(k0);
      __syncthreads();
      if (k0 + kBK < p.K) fetch(k0 + kBK);
      multiply();
      __syncthreads();  // every wave's reads of the tiles are done
    }
  }
  // Lane (c, g) of a 16 x 16 fragment: column c, rows 4g .. 4g + 3.
  float sx[FM][4];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) sx[i][r] = __shfl(own_x, i * 16 + 4 * g + r, 64);
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    const float sw = __shfl(own_w, j * 16 + c, 64), bias = __shfl(own_bias, j * 16 + c, 64);
    const int64_t n = n0 + wn * TN + j * 16 + c;
    if (n >= p.N) continue;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t m = m0 + wm * TM + i * 16 + 4 * g + r;
        if (m >= p.M) continue;
        static_cast<T*>(p.y)[m * p.y_rs + n] = slc::from_f32<T>(finish<T>(acc[i][j][r], sx[i][r], sw, bias));
      }
  }
}

// ---- prefill: tiles streamed through an LDS ring -----------------------------------
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, int64_t bytes) {
  const uint64_t address = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(address));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(address >> 32));
  const int clamped = bytes > 0x7fffffff ? 0x7fffffff : static_cast<int>(bytes);
  return __builtin_amdgcn_make_buffer_rsrc(
      reinterpret_cast<void*>(static_cast<uint64_t>(hi) << 32 | lo), 0,
      __builtin_amdgcn_readfirstlane(clamped), 0x00020000);
}

__device__ __forceinline__ void lds_dma16(__amdgpu_buffer_rsrc_t rsrc, unsigned char* lds,
                                          int voffset, int soffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      rsrc, (__attribute__((address_space(3))) void*)lds, 16, voffset, soffset, 0, 0);
}

// Tile id -> (m_blk, n_blk): workgroup ids go round-robin to the 8 XCDs, each with
// its own L2, so ids are gathered per XCD, then run in groups of kGroupM M-tiles (a power
// of two), N-tile-major inside a group.  One division, but in a last, smaller group.
template <int kGroupM>
__device__ __forceinline__ void xcd_tile_of(int id, int n_tiles, int m_tiles, int& m_blk,
                                            int& n_blk) {
  static_assert((kGroupM & (kGroupM - 1)) == 0, "a power of two");
  constexpr uint32_t kXcds = 8;
  const uint32_t u = static_cast<uint32_t>(id), per = static_cast<uint32_t>(n_tiles * m_tiles) / kXcds;
  const uint32_t t = u < per * kXcds ? (u % kXcds) * per + u / kXcds : u;
  const uint32_t span = static_cast<uint32_t>(kGroupM * n_tiles);
  const uint32_t group = t / span, rest = t - group * span;
  const int first_m = static_cast<int>(group) * kGroupM;
  if (first_m + kGroupM <= m_tiles) {
    m_blk = first_m + static_cast<int>(rest % kGroupM);
    n_blk = static_cast<int>(rest / kGroupM);
  } else {
    const uint32_t gm = static_cast<uint32_t>(m_tiles - first_m);
    n_blk = static_cast<int>(rest / gm);
    m_blk = first_m + static_cast<int>(rest % gm);
  }
}

// Swizzle of the W tile: the 16 rows of a fragment are four runs of four, eight
// apart, so the key takes row bits 0, 1 and 3.
__device__ __forceinline__ int w_key(int row) { return (row & 3) | ((row >> 1) & 4); }

// Element n of the bias as it is stored (0 past its range, of 0 bytes without a
// bias), and its value: converted at its use, so that the load is not waited for
// where it is issued.
template <typename T>
__device__ __forceinline__ uint32_t load_bias(const __amdgpu_buffer_rsrc_t& rbias, int n) {
  if constexpr (sizeof(T) == 4) return __builtin_amdgcn_raw_buffer_load_b32(rbias, n * 4, 0, 0);
  return static_cast<uint16_t>(__builtin_amdgcn_raw_buffer_load_b16(rbias, n * 2, 0, 0));
}
template <typename T>
__device__ __forceinline__ float bias_value(uint32_t bits) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(bits);
  } else {
    T v;
    v.bits = static_cast<uint16_t>(bits);
    return slc::to_f32(v);
  }
}

// Rows whose span is under this are reached by 32-bit offsets.
constexpr int64_t kRangeLimit = (int64_t{1} << 31) - (1 << 20);
constexpr int kNoPath = -2;
// An offset past every such range that stays below 2^31 with K added.
constexpr int kPastRange = 0x7fffffff - (1 << 18);

// Four consecutive elements of the bias (0 without one), in words of two where the
// outputs are whole runs of eight.
template <typename T, bool PAIRS>
struct BiasRun {
  static constexpr int kWords = PAIRS && sizeof(T) == 2 ? 2 : 4;
  uint32_t raw[kWords] = {};
  __device__ __forceinline__ void load(const __amdgpu_buffer_rsrc_t& rbias, int n) {
    if constexpr (kWords == 2) {
      const auto two = __builtin_amdgcn_raw_buffer_load_b64(rbias, n * 2, 0, 0);
      raw[0] = two[0];
      raw[1] = two[1];
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) raw[r] = load_bias<T>(rbias, n + r);
    }
  }
  __device__ __forceinline__ void wait() {
#pragma unroll
    for (int r = 0; r < kWords; ++r) asm volatile("" : "+v"(raw[r]));
  }
  __device__ __forceinline__ float value(int r) const {
    return bias_value<T>(kWords == 2 ? raw[r / 2] >> (16 * (r % 2)) & 0xffffu : raw[r]);
  }
};

// A lane's run of eight consecutive outputs at a byte offset from the tile's first.
// VST, 16-byte stores: what is outside the tile has an offset past the range (a run is
// inside its row as a whole or not at all; 4 x 2 fp32 of it at `half`).  Else `left` of
// the run are inside.
template <typename T, bool VST>
__device__ __forceinline__ void store_run(const __amdgpu_buffer_rsrc_t& ry, const float (&v)[8],
                                          uint32_t offset, uint32_t half, int left) {
  constexpr int kSize = static_cast<int>(sizeof(T));
  if constexpr (VST) {
#pragma unroll
    for (int h = 0; h < kSize / 2; ++h) {
      i32x4_t packed;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        if constexpr (kSize == 4)
          packed[d] = __float_as_int(v[4 * h + d]);
        else
          packed[d] = static_cast<int>(slc::pack2<T>(v[2 * d], v[2 * d + 1]));
      }
      __builtin_amdgcn_raw_buffer_store_b128(packed, ry, static_cast<int>(h == 0 ? offset : half), 0, 0);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e >= left) continue;
      if constexpr (kSize == 4)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(v[e]), ry, static_cast<int>(offset + 4 * e), 0, 0);
      else
        __builtin_amdgcn_raw_buffer_store_b16(static_cast<short>(slc::from_f32<T>(v[e]).bits), ry, static_cast<int>(offset + 2 * e), 0, 0);
    }
  }
}

// 16-byte aligned rows of codes.  PW producer waves stream X and W k-tiles of
// 128 codes straight into an S-stage LDS ring (buffer_load ... lds), without a
// break at tile boundaries; CWM x CWN consumer waves read LDS and issue MFMAs.
// Workgroups walk the output tiles id, id + grid, ....  One barrier per k-tile:
// before it the producers wait until their loads of tile q have landed, after it
// they refill the stage that every consumer has finished reading.  The consumers
// multiply with W rows as the A operand, the W rows of two fragments interleaved
// in runs of four, so that a lane holds eight consecutive outputs of one row and
// stores them from registers.  Past K the X chunks are loaded as zeros (an offset
// past the range), whatever the W chunks beside them hold.
//
// 4096 x 9728 x 896 43.5 us (1640 TOPS) where one buffer takes the outputs of call after call:
// loads and stores alone take 33, products and stores 32; 56 us where outputs spread over 640
// MB, past the caches.  fp32 outputs 62.  8 x 151936 x 896 28 us, 4.9 TB/s of weight.  Stores of
// single elements (N that no 16 bytes divide) cost more than the products: 4096 x 9727 x 896
// 112 us, in fp32 144.
template <typename T, int BM, int BN, int CWM, int CWN, int PW, int S, int GM, bool VST>
__global__ __launch_bounds__((CWM * CWN + PW) * 64) void stream_kernel(Problem p, int n_tiles,
                                                                       int m_tiles) {
  constexpr int CW = CWM * CWN;
  constexpr int TM = BM / CWM, TN = BN / CWN;
  constexpr int FM = TM / 16, FN = TN / 16;
  constexpr int XB = BM * kBK;
  constexpr int kStage = (BM + BN) * kBK;
  constexpr int XO = BM / 8 / PW, WO = BN / 8 / PW, kOps = XO + WO;
  static_assert(XO * PW * 8 == BM && WO * PW * 8 == BN, "operands split evenly over the producers");
  static_assert((S - 2) * kOps <= 63, "the wait count fits vmcnt");
  static_assert(TM % 16 == 0 && TN % 32 == 0, "whole fragments, in pairs over N");
  __shared__ __attribute__((aligned(16))) unsigned char ring[S * kStage];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int total = n_tiles * m_tiles;
  const int ktiles = (p.K + kBK - 1) / kBK;
  const int first = blockIdx.x, step = gridDim.x;

  if (wave >= CW) {
    const int pw = wave - CW;
    int voff[kOps];
#pragma unroll
    for (int i = 0; i < kOps; ++i) {
      const int local = i < XO ? i : i - XO;
      const int row = 8 * (pw + PW * local) + lane / 8;
      const int chunk = (lane % 8) ^ (i < XO ? row & 7 : w_key(row));
      voff[i] = (i < XO ? static_cast<int>(row * p.x_rs) : row * p.K) + chunk * 16;
    }
    // Whether this lane's X chunk of the last k-tile is past K: the chunk index
    // depends on the lane alone (rows step by 8 over the instructions).
    const int last_chunk = (lane % 8) ^ ((lane / 8) & 7);
    const bool past = (ktiles - 1) * kBK + last_chunk * 16 >= p.K;
    // The tile's ranges as base + bytes, rebuilt into scalars at every issue.
    const int8_t* xb = p.x;
    const int8_t* wb = p.w;
    int64_t x_bytes = 0, w_bytes = 0;
    int load_id = first, load_k = 0, slot = 0;
    auto set_tile = [&](int id) {
      x_bytes = w_bytes = 0;
      if (id >= total) return;
      int m_blk, n_blk;
      xcd_tile_of<GM>(id, n_tiles, m_tiles, m_blk, n_blk);
      const int64_t m0 = static_cast<int64_t>(m_blk) * BM, n0 = static_cast<int64_t>(n_blk) * BN;
      const int64_t x_rows = p.M - m0 < BM ? p.M - m0 : BM;
      const int64_t w_rows = p.N - n0 < BN ? p.N - n0 : BN;
      xb = p.x + m0 * p.x_rs;
      x_bytes = (x_rows - 1) * p.x_rs + p.K;
      wb = p.w + n0 * p.K;
      w_bytes = w_rows * p.K;
    };
    set_tile(load_id);
    auto issue = [&]() {
      unsigned char* dst = ring + __builtin_amdgcn_readfirstlane(slot) * kStage;
      const int kb = __builtin_amdgcn_readfirstlane(load_id < total ? load_k * kBK : 0);
      const __amdgpu_buffer_rsrc_t rx = make_rsrc(xb, x_bytes);
      const __amdgpu_buffer_rsrc_t rw = make_rsrc(wb, w_bytes);
      const bool cut = load_k == ktiles - 1 && past;
#pragma unroll
      for (int i = 0; i < kOps; ++i) {
        if (i < XO)
          lds_dma16(rx, dst + (pw + PW * i) * 1024, cut ? kPastRange : voff[i], kb);
        else
          lds_dma16(rw, dst + XB + (pw + PW * (i - XO)) * 1024, voff[i], kb);
      }
      slot = slot == S - 1 ? 0 : slot + 1;
      if (++load_k == ktiles) {
        load_k = 0;
        load_id += step;
        set_tile(load_id);
      }
    };
#pragma clang loop unroll(disable)
    for (int t = 0; t < S - 1; ++t) issue();
    const int64_t steps = static_cast<int64_t>((total - 1 - first) / step + 1) * ktiles;
#pragma clang loop unroll(disable)
    for (int64_t q = 0; q < steps; ++q) {
      asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"((S - 2) * kOps) : "memory");
      issue();
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    return;
  }

  const int c = lane & 15, g = lane >> 4;
  const int wm = wave / CWN, wn = wave % CWN;
  int slot = 0;
  for (int id = first; id < total; id += step) {
    int m_blk, n_blk;
    xcd_tile_of<GM>(id, n_tiles, m_tiles, m_blk, n_blk);
    const int64_t m0 = static_cast<int64_t>(m_blk) * BM, n0 = static_cast<int64_t>(n_blk) * BN;
    const int rows = p.M - m0 < BM ? static_cast<int>(p.M - m0) : BM;
    const int cols = p.N - n0 < BN ? static_cast<int>(p.N - n0) : BN;
    // Scales and bias of this lane's outputs, requested before the k loop.
    const __amdgpu_buffer_rsrc_t rsx = make_rsrc(p.sx + m0, rows * 4);
    const __amdgpu_buffer_rsrc_t rsw = make_rsrc(p.sw + n0, cols * 4);
    float sx[FM], sw[FN][4];
    BiasRun<T, VST> bias[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
      sx[i] = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsx, (wm * TM + i * 16 + c) * 4, 0, 0));
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = wn * TN + (j >> 1) * 32 + 8 * g + (j & 1) * 4;
      const auto four = __builtin_amdgcn_raw_buffer_load_b128(rsw, n * 4, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) sw[j][r] = __int_as_float(static_cast<int>(four[r]));
    }
    if (p.bias != nullptr) {
      const __amdgpu_buffer_rsrc_t rbias =
          make_rsrc(static_cast<const T*>(p.bias) + n0, cols * static_cast<int>(sizeof(T)));
#pragma unroll
      for (int j = 0; j < FN; ++j) bias[j].load(rbias, wn * TN + (j >> 1) * 32 + 8 * g + (j & 1) * 4);
    }
    i32x4_t acc[FN][FM];
    auto k_tile = [&](auto is_first) {
      constexpr bool FIRST = decltype(is_first)::value;
      // Tile kt is in its stage; the stage read before may be refilled.  No wait
      // on stores: the previous tile's output may still be in flight.
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      const unsigned char* xs = ring + slot * kStage;
      const unsigned char* ws = xs + XB;
      slot = slot == S - 1 ? 0 : slot + 1;
#pragma unroll
      for (int kk = 0; kk < kBK / 64; ++kk) {
        i32x4_t a[FM], b[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i)
          a[i] = *reinterpret_cast<const i32x4_t*>(xs + lds_offset(wm * TM + i * 16 + c, kk * 4 + g));
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const int wrow = wn * TN + (j >> 1) * 32 + 8 * (c >> 2) + (j & 1) * 4 + (c & 3);
          b[j] = *reinterpret_cast<const i32x4_t*>(ws + wrow * kBK + (((kk * 4 + g) ^ w_key(wrow)) << 4));
        }
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int i = 0; i < FM; ++i) acc[j][i] = mfma(b[j], a[i], FIRST && kk == 0 ? i32x4_t{0, 0, 0, 0} : acc[j][i]);
      }
    };
    k_tile(std::true_type{});
#pragma clang loop unroll(disable)
    for (int kt = 1; kt < ktiles; ++kt) k_tile(std::false_type{});
    // The scales have arrived while the tile was multiplied: waited for here, as a
    // later wait would count this tile's stores too.
#pragma unroll
    for (int i = 0; i < FM; ++i) asm volatile("" : "+v"(sx[i]));
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) asm volatile("" : "+v"(sw[j][r]));
#pragma unroll
    for (int j = 0; j < FN; ++j) bias[j].wait();
    constexpr int kSize = static_cast<int>(sizeof(T));
    const __amdgpu_buffer_rsrc_t ry =
        make_rsrc(static_cast<T*>(p.y) + m0 * p.y_rs + n0, (static_cast<int64_t>(rows) - 1) * p.y_rs * kSize + cols * kSize);
    const uint32_t rows16 = static_cast<uint32_t>(16 * p.y_rs) * kSize;  // 16 rows further down
#pragma unroll
    for (int q = 0; q < FN / 2; ++q) {
      const int n = wn * TN + q * 32 + 8 * g;
      const uint32_t at = static_cast<uint32_t>((wm * TM + c) * p.y_rs + n) * kSize;
      const uint32_t whole = !VST || n < cols ? at : kPastRange, half = n + 4 < cols ? at + 16 : kPastRange;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int m = wm * TM + i * 16 + c;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = 2 * q + (e >> 2), r = e & 3;
          v[e] = finish<T>(acc[j][i][r], sx[i], sw[j][r], bias[j].value(r));
        }
        store_run<T, VST>(ry, v, whole + i * rows16, half + i * rows16, m < rows ? cols - n : 0);
      }
    }
  }
}

// N loads of 1 KB into LDS, 8 KB apart from `lds` on, as one statement without results:
// the compiler, which would wait for open loads into LDS before every read of it, does
// not see them, and the kernel counts them itself.  (Five wait states between a vector
// instruction's scalar result and its use here, one after each write of m0.)
template <int N>
__device__ __forceinline__ void lds_dma_batch(i32x4_t rsrc, uint32_t lds, const int (&voff)[N], int soffset) {
  static_assert(N == 2 || N == 4, "the forms below");
  uint32_t m0;  // put back: the compiler may not be told of its change
  if constexpr (N == 4) {
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %6, %7 offen lds\n\t"
        "s_add_u32 m0, m0, 0x2000\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %6, %7 offen lds\n\t"
        "s_add_u32 m0, m0, 0x2000\n\ts_nop 0\n\tbuffer_load_dwordx4 %4, %6, %7 offen lds\n\t"
        "s_add_u32 m0, m0, 0x2000\n\ts_nop 0\n\tbuffer_load_dwordx4 %5, %6, %7 offen lds\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(m0)
        : "s"(lds), "v"(voff[0]), "v"(voff[1]), "v"(voff[2]), "v"(voff[3]), "s"(rsrc), "s"(soffset)
        : "memory", "scc");
  } else {
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %4, %5 offen lds\n\t"
        "s_add_u32 m0, m0, 0x2000\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %4, %5 offen lds\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(m0)
        : "s"(lds), "v"(voff[0]), "v"(voff[1]), "s"(rsrc), "s"(soffset)
        : "memory", "scc");
  }
}
__device__ __forceinline__ i32x4_t descriptor(const void* base, int64_t bytes) {
  const uint64_t address = reinterpret_cast<uint64_t>(base);
  i32x4_t r;
  r[0] = __builtin_amdgcn_readfirstlane(static_cast<int>(address));
  r[1] = __builtin_amdgcn_readfirstlane(static_cast<int>((address >> 32) & 0xffff));
  r[2] = __builtin_amdgcn_readfirstlane(bytes > 0x7fffffff ? 0x7fffffff : static_cast<int>(bytes));
  r[3] = 0x00020000;
  return r;
}

// 16-byte aligned rows of codes, several k-tiles.  Eight waves, two on each SIMD, in
// two groups of four that take turns: while one group's waves multiply a k-step from
// registers, the other's read their next k-step from LDS and issue the loads of a
// tile ahead (global -> LDS, no registers); a barrier ends each turn.  Group 0 holds
// the upper half of the BM rows of the output tile, group 1 the lower.
//
// Turns (one barrier after each), k-tile q, k-step s of it: group 0 reads (q, s) in
// turn 4q + 2s and multiplies it in the next, group 1 one turn later.  So what tile
// q - 1 occupied is free from turn 4q on.  X has three slots and W two, which fill the
// LDS: with (q, 0) a wave issues its part of W tile q + 1, with (q, 1) of X tile q + 2,
// each into the slot of tile q - 1.  Every wave waits for its part of tile q + 1 before
// the barrier that ends turn 4q + 3 (group 0 after multiplying (q, 1), group 1 after
// reading it).  Memory operations complete in order, so the wait leaves open what was
// issued later: X tile q + 2.  At the end of an output tile the next W tile is issued
// before the stores, so that the first such wait leaves the stores open too.
//
// Workgroups walk the output tiles id, id + grid, ...; the loads run on across tile
// boundaries.  The MFMA's A operand is W, the rows of two fragments interleaved in runs
// of four, so that a lane holds eight consecutive outputs of one row and stores them
// from registers.  Past K the X chunks are loaded as zeros (an offset past the range),
// whatever the W chunks beside them hold.
//
// 8192 x 8192 x 8192 404 us (2720 TOPS; on another card 391), 32768 x 896 x 4864 128 (2230).
// Bound by the clock that the card's power leaves: codes of all zeros take 330 and 101.
constexpr int kTurnsTile = 256, kTurnsGroup = 4;
template <typename T, bool VST>
__global__ __launch_bounds__(512, 2) void turns_kernel(Problem p, int n_tiles, int m_tiles) {
  constexpr int BM = kTurnsTile, BN = kTurnsTile, GM = kTurnsGroup;
  constexpr int CW = 8, CWN = 4, XS = 3, WS = 2;
  constexpr int TM = BM / 2, TN = BN / CWN;
  constexpr int FM = TM / 16, FN = TN / 16;
  constexpr int XB = BM * kBK, WB = BN * kBK;
  constexpr int XO = BM / 8 / CW, WO = BN / 8 / CW;
  constexpr int kSize = static_cast<int>(sizeof(T));
  constexpr int kStores = VST ? FM * FN / 2 * (kSize / 2) : 0;
  constexpr int kOpen = XO;
  static_assert(XO * CW * 8 == BM && WO * CW * 8 == BN, "operands split evenly over the waves");
  static_assert(TM % 64 == 0 && TN % 32 == 0 && TN <= 64, "whole fragments, in pairs over N; scales by lane");
  static_assert(kOpen + kStores <= 63, "the wait count fits vmcnt");
  static_assert(XS * XB + WS * WB <= 160 * 1024, "the slots fit the LDS");
  __shared__ __attribute__((aligned(16))) unsigned char ring[XS * XB + WS * WB];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int c = lane & 15, g = lane >> 4;
  const int wm = wave / CWN, wn = wave % CWN;
  const bool late = wm != 0;
  const int total = n_tiles * m_tiles;
  const int ktiles = (p.K + kBK - 1) / kBK;
  const int first = blockIdx.x, step = gridDim.x;
  const uint32_t base = static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)ring));

  // ---- loads: each operand walks the tiles and k-tiles by itself --------------------
  int xoff[XO], woff[WO];
#pragma unroll
  for (int i = 0; i < XO; ++i) {
    const int row = 8 * (wave + CW * i) + lane / 8;
    xoff[i] = static_cast<int>(row * p.x_rs) + ((lane % 8) ^ (row & 7)) * 16;
  }
#pragma unroll
  for (int i = 0; i < WO; ++i) {
    const int row = 8 * (wave + CW * i) + lane / 8;
    woff[i] = row * p.K + ((lane % 8) ^ w_key(row)) * 16;
  }
  // Whether this lane's X chunk of the last k-tile is past K: the chunk index
  // depends on the lane alone (rows step by 8 over the instructions).
  const bool past = (ktiles - 1) * kBK + ((lane % 8) ^ ((lane / 8) & 7)) * 16 >= p.K;
  struct Walk {
    const int8_t* from;
    int64_t bytes;
    int id, k, slot;
  };
  Walk wx{p.x, 0, first, 0, 0}, ww{p.w, 0, first, 0, 0};
  auto aim_x = [&]() {
    wx.bytes = 0;
    if (wx.id >= total) return;
    int m_blk, n_blk;
    xcd_tile_of<GM>(wx.id, n_tiles, m_tiles, m_blk, n_blk);
    const int64_t m0 = static_cast<int64_t>(m_blk) * BM;
    wx.from = p.x + m0 * p.x_rs;
    wx.bytes = ((p.M - m0 < BM ? p.M - m0 : BM) - 1) * p.x_rs + p.K;
  };
  auto aim_w = [&]() {
    ww.bytes = 0;
    if (ww.id >= total) return;
    int m_blk, n_blk;
    xcd_tile_of<GM>(ww.id, n_tiles, m_tiles, m_blk, n_blk);
    const int64_t n0 = static_cast<int64_t>(n_blk) * BN;
    ww.from = p.w + n0 * p.K;
    ww.bytes = (p.N - n0 < BN ? p.N - n0 : BN) * p.K;
  };
  auto advance = [&](Walk& w, int slots, auto aim) {
    w.slot = w.slot == slots - 1 ? 0 : w.slot + 1;
    if (++w.k == ktiles) {
      w.k = 0;
      w.id += step;
      aim();
    }
  };
  auto issue_x = [&]() {
    int off[XO];
    const bool cut = wx.k == ktiles - 1 && past;
#pragma unroll
    for (int i = 0; i < XO; ++i) off[i] = cut ? kPastRange : xoff[i];
    lds_dma_batch<XO>(descriptor(wx.from, wx.bytes),
                      __builtin_amdgcn_readfirstlane(base + wx.slot * XB + wave * 1024), off,
                      __builtin_amdgcn_readfirstlane(wx.id < total ? wx.k * kBK : 0));
    advance(wx, XS, aim_x);
  };
  auto issue_w = [&]() {
    lds_dma_batch<WO>(descriptor(ww.from, ww.bytes),
                      __builtin_amdgcn_readfirstlane(base + XS * XB + ww.slot * WB + wave * 1024), woff,
                      __builtin_amdgcn_readfirstlane(ww.id < total ? ww.k * kBK : 0));
    advance(ww, WS, aim_w);
  };
  auto barrier = []() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // This wave's part of the next tile; `stores`: its stores may be open too.
  auto landed = [&](bool stores) {
    __builtin_amdgcn_sched_barrier(0);
    if (stores)
      asm volatile("s_waitcnt vmcnt(%0)" ::"i"(kOpen + kStores) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(%0)" ::"i"(kOpen) : "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  aim_x();
  aim_w();
  issue_x();
  issue_w();
  issue_x();
  landed(false);
  barrier();
  if (late) barrier();
  int x_slot = 0, w_slot = 0;
  const int x_read = lds_offset(wm * TM + c, g);
  const int w_row = wn * TN + 8 * (c >> 2) + (c & 3);
  const int w_read = XS * XB + w_row * kBK + ((g ^ w_key(w_row)) << 4);
  for (int id = first; id < total; id += step) {
    int m_blk, n_blk;
    xcd_tile_of<GM>(id, n_tiles, m_tiles, m_blk, n_blk);
    const int64_t m0 = static_cast<int64_t>(m_blk) * BM, n0 = static_cast<int64_t>(n_blk) * BN;
    const int rows = p.M - m0 < BM ? static_cast<int>(p.M - m0) : BM;
    const int cols = p.N - n0 < BN ? static_cast<int>(p.N - n0) : BN;
    i32x4_t acc[FN][FM];
    uint32_t own_x[TM / 64], own_w = 0, own_bias = 0;
    auto k_tile = [&](int kt, auto is_first) {
      constexpr bool FIRST = decltype(is_first)::value;
      const int x_at = x_read + x_slot * XB, w_at = w_read + w_slot * WB;
      x_slot = x_slot == XS - 1 ? 0 : x_slot + 1;
      w_slot = w_slot == WS - 1 ? 0 : w_slot + 1;
#pragma unroll
      for (int kk = 0; kk < kBK / 64; ++kk) {
        // Fragments are constant distances apart; the second k-step is 64 bytes across
        // (bit 2 of the swizzled chunk).
        i32x4_t a[FM], b[FN];
        const unsigned char* ws = ring + (w_at ^ (kk * 64));
        const unsigned char* xs = ring + (x_at ^ (kk * 64));
#pragma unroll
        for (int j = 0; j < FN; ++j)
          b[j] = *reinterpret_cast<const i32x4_t*>(ws + ((j >> 1) * 32 + (j & 1) * 4) * kBK);
#pragma unroll
        for (int i = 0; i < FM; ++i) a[i] = *reinterpret_cast<const i32x4_t*>(xs + i * 16 * kBK);
        __builtin_amdgcn_sched_barrier(0);
        if (kk == 0) {
          if (!FIRST || id == first) issue_w();
          if constexpr (FIRST) {
            // Lane l of a load holds the scale of row l, or of column l, of the wave's.
            const __amdgpu_buffer_rsrc_t rsx = make_rsrc(p.sx + m0, rows * 4);
            const __amdgpu_buffer_rsrc_t rsw = make_rsrc(p.sw + n0, cols * 4);
            const __amdgpu_buffer_rsrc_t rbias =
                make_rsrc(p.bias != nullptr ? static_cast<const T*>(p.bias) + n0 : nullptr,
                          p.bias != nullptr ? cols * kSize : 0);
#pragma unroll
            for (int r = 0; r < TM / 64; ++r)
              own_x[r] = __builtin_amdgcn_raw_buffer_load_b32(rsx, (wm * TM + 64 * r + lane) * 4, 0, 0);
            own_w = __builtin_amdgcn_raw_buffer_load_b32(rsw, (wn * TN + lane) * 4, 0, 0);
            own_bias = load_bias<T>(rbias, wn * TN + lane);
          }
        } else {
          issue_x();
          // Nobody may still read the tile when its slots are refilled.
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          if (late) landed(FIRST && id != first);
        }
        barrier();
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[j][i] = mfma(b[j], a[i], FIRST && kk == 0 ? i32x4_t{0, 0, 0, 0} : acc[j][i]);
        __builtin_amdgcn_s_setprio(0);
        if (kk == 1 && !late) landed(FIRST && id != first);
        if (kk == 0 || kt + 1 < ktiles || !late) barrier();
      }
    };
    k_tile(0, std::true_type{});
#pragma clang loop unroll(disable)
    for (int kt = 1; kt < ktiles; ++kt) k_tile(kt, std::false_type{});
    // The scales, waited for before the next loads are issued.
#pragma unroll
    for (int r = 0; r < TM / 64; ++r) asm volatile("" : "+v"(own_x[r]));
    asm volatile("" : "+v"(own_w), "+v"(own_bias));
    issue_w();
    const __amdgpu_buffer_rsrc_t ry =
        make_rsrc(static_cast<T*>(p.y) + m0 * p.y_rs + n0,
                  (static_cast<int64_t>(rows) - 1) * p.y_rs * kSize + cols * kSize);
    float sx[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i)
      sx[i] = __uint_as_float(__shfl(own_x[i / 4], (i % 4) * 16 + c, 64));
    const uint32_t rows16 = static_cast<uint32_t>(16 * p.y_rs) * kSize;  // 16 rows further down
#pragma unroll
    for (int q = 0; q < FN / 2; ++q) {
      const int n = wn * TN + q * 32 + 8 * g;
      float sw[8], bs[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sw[e] = __uint_as_float(__shfl(own_w, q * 32 + 8 * g + e, 64));
        bs[e] = bias_value<T>(__shfl(own_bias, q * 32 + 8 * g + e, 64));
      }
      const uint32_t at = static_cast<uint32_t>((wm * TM + c) * p.y_rs + n) * kSize;
      const uint32_t whole = !VST || n < cols ? at : kPastRange, half = n + 4 < cols ? at + 16 : kPastRange;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int m = wm * TM + i * 16 + c;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = finish<T>(acc[2 * q + (e >> 2)][i][e & 3], sx[i], sw[e], bs[e]);
        store_run<T, VST>(ry, v, whole + i * rows16, half + i * rows16, m < rows ? cols - n : 0);
      }
    }
    if (late) barrier();
  }
  if (!late) barrier();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <typename T>
int launch_turns(const Problem& p, hipStream_t stream) {
  constexpr int BM = kTurnsTile, BN = kTurnsTile;
  const int64_t m_tiles = (static_cast<int64_t>(p.M) + BM - 1) / BM;
  const int64_t n_tiles = (static_cast<int64_t>(p.N) + BN - 1) / BN;
  if (BM * p.x_rs >= kRangeLimit || BM * p.y_rs * static_cast<int64_t>(sizeof(T)) >= kRangeLimit ||
      m_tiles * n_tiles >= (int64_t{1} << 30))
    return kNoPath;
  const int64_t total = m_tiles * n_tiles;
  const int cus = slc_host::device_cu_count() / 8 * 8;
  const int grid = static_cast<int>(total < cus || cus <= 0 ? total : cus);
  const int64_t unit = 16 / static_cast<int64_t>(sizeof(T));
  const bool vectors = p.N % unit == 0 && p.y_rs % unit == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
#define SLC_TURNS(VST)                                                                             \
  hipLaunchKernelGGL((turns_kernel<T, VST>), dim3(static_cast<unsigned>(grid)), \
                     dim3(512), 0, stream, p, static_cast<int>(n_tiles), static_cast<int>(m_tiles))
  if (vectors) {
    SLC_TURNS(true);
  } else {
    SLC_TURNS(false);
  }
#undef SLC_TURNS
  return slc_host::check_launch("slc_hip_linear_q8(turns)");
}

// kNoPath (nothing launched) where 32-bit offsets do not reach over a tile's rows.
template <typename T, int BM, int BN, int CWM, int CWN, int PW, int S, int GM>
int launch_stream(const Problem& p, hipStream_t stream) {
  const int64_t m_tiles = (static_cast<int64_t>(p.M) + BM - 1) / BM;
  const int64_t n_tiles = (static_cast<int64_t>(p.N) + BN - 1) / BN;
  if (BM * p.x_rs >= kRangeLimit || BM * p.y_rs * static_cast<int64_t>(sizeof(T)) >= kRangeLimit ||
      m_tiles * n_tiles >= (int64_t{1} << 30))
    return kNoPath;
  const int64_t total = m_tiles * n_tiles;
  const int cus = slc_host::device_cu_count() / 8 * 8;
  const int grid = static_cast<int>(total < cus || cus <= 0 ? total : cus);
  const int64_t unit = 16 / static_cast<int64_t>(sizeof(T));
  const bool vectors = p.N % unit == 0 && p.y_rs % unit == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
#define SLC_STREAM(VST)                                                                       \
  hipLaunchKernelGGL((stream_kernel<T, BM, BN, CWM, CWN, PW, S, GM, VST>),                    \
                     dim3(static_cast<unsigned>(grid)), dim3((CWM * CWN + PW) * 64), 0, stream, p, \
                     static_cast<int>(n_tiles), static_cast<int>(m_tiles))
  if (vectors) {
    SLC_STREAM(true);
  } else {
    SLC_STREAM(false);
  }
#undef SLC_STREAM
  return slc_host::check_launch("slc_hip_linear_q8(stream)");
}

// ---- decode: few rows, the weight streamed once -----------------------------------
// A workgroup owns a block of rows and `feat` consecutive features (up to 16 * TILES; MFMA
// rows past them are masked off by the buffer range) and splits K over its waves; the waves' sums meet
// in LDS by integer adds, whose order does not matter.  Each wave keeps U k-steps of 64
// codes in flight while it multiplies the U before.  Bound by the weight's bytes where
// it is wide, by latency where it is narrow: 1 x 151936 x 896 25 us (5.4 TB/s), 8 x 1152 x
// 896 3.3, 1 x 896 x 4864 4.6, 32 x 896 x 4864 8.5.
constexpr int kRowBlock = 32;
template <typename T, int MB, int TILES, int U>
__global__ __launch_bounds__(1024) void rows_kernel(Problem p, int feat) {
  __shared__ int sums[TILES * MB * 256];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int waves = blockDim.x >> 6;
  const int lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * feat;
  const int cols = p.N - n0 < feat ? static_cast<int>(p.N - n0) : feat;
  const int steps = (p.K + 63) / 64, per = (steps + waves - 1) / waves;
  const int begin = wave * per, end = begin + per < steps ? begin + per : steps;

  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kRowBlock;
  const int rows = p.M - m0 < kRowBlock ? static_cast<int>(p.M - m0) : kRowBlock;
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x + m0 * p.x_rs, (rows - 1) * p.x_rs + p.K);
  const __amdgpu_buffer_rsrc_t rw = make_rsrc(p.w + n0 * p.K, static_cast<int64_t>(cols) * p.K);
  int x_off[MB], w_off[TILES];
#pragma unroll
  for (int i = 0; i < MB; ++i) x_off[i] = static_cast<int>((i * 16 + c) * p.x_rs) + g * 16;
#pragma unroll
  for (int t = 0; t < TILES; ++t) w_off[t] = (t * 16 + c) * p.K + g * 16;
  i32x4_t acc[TILES][MB];
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[t][i] = i32x4_t{0, 0, 0, 0};

  // Zeros for X past K and past this wave's steps, whatever W holds there.
  i32x4_t wa[U][TILES], wb[U][TILES], xa[U][MB], xb[U][MB];
  auto load16 = [](const __amdgpu_buffer_rsrc_t& r, int at) {
    return __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
  };
  auto fetch = [&](int s0, i32x4_t (&w)[U][TILES], i32x4_t (&x)[U][MB]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u;
      const bool live = s < end;
      const bool in = live && s * 64 + g * 16 < p.K;
#pragma unroll
      for (int t = 0; t < TILES; ++t) w[u][t] = load16(rw, live ? w_off[t] + s * 64 : kPastRange);
#pragma unroll
      for (int i = 0; i < MB; ++i) x[u][i] = load16(rx, in ? x_off[i] + s * 64 : kPastRange);
    }
  };
  auto multiply = [&](const i32x4_t (&w)[U][TILES], const i32x4_t (&x)[U][MB]) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int i = 0; i < MB; ++i) acc[t][i] = mfma(x[u][i], w[u][t], acc[t][i]);
  };
  int s0 = begin;
  fetch(s0, wa, xa);
  // This thread's first output's scales, behind the first loads: element e of the
  // fragments is row 4 * (l / 16) + r of block i, column l % 16 of tile t.
  auto place = [&](int e, int& m, int& n) {
    const int l = (e / 4) & 63;
    m = (e / 256 % MB) * 16 + 4 * (l >> 4) + e % 4;
    n = e / (256 * MB) * 16 + (l & 15);
  };
  int m, n;
  place(tid, m, n);
  float sx = 0.0f, sw = 0.0f;
  uint32_t bias = 0;
  auto scales = [&]() {
    sx = p.sx[m0 + m];
    sw = p.sw[n0 + n];
    if (p.bias != nullptr) {
      if constexpr (sizeof(T) == 4)
        bias = static_cast<const uint32_t*>(p.bias)[n0 + n];
      else
        bias = static_cast<const uint16_t*>(p.bias)[n0 + n];
    }
  };
  const bool mine = tid < TILES * MB * 256 && m < rows && n < cols;
  if (mine) scales();
  for (int e = tid; e < TILES * MB * 256; e += blockDim.x) sums[e] = 0;
  __syncthreads();
  while (s0 < end) {
    fetch(s0 + U, wb, xb);
    multiply(wa, xa);
    s0 += U;
    if (s0 >= end) break;
    fetch(s0 + U, wa, xa);
    multiply(wb, xb);
    s0 += U;
  }
  if (begin < end) {
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) atomicAdd(&sums[((t * MB + i) * 64 + lane) * 4 + r], acc[t][i][r]);
  }
  __syncthreads();
  for (int e = tid; e < TILES * MB * 256; e += blockDim.x) {
    if (e != tid) place(e, m, n);
    if (m >= rows || n >= cols) continue;
    if (e != tid) scales();
    static_cast<T*>(p.y)[(m0 + m) * p.y_rs + n0 + n] =
        slc::from_f32<T>(finish<T>(sums[e], sx, sw, bias_value<T>(bias)));
  }
}

// About a workgroup per CU, of equal shares of the features, 32 at most; eight waves, fewer
// where K has fewer steps (16 waves: 1 x 896 x 896 3.9 us for 3.4, 8 x 896 x 4864 6.4 for
// 5.5; four: 3.4 and 5.7).
template <typename T>
int launch_rows(const Problem& p, hipStream_t stream) {
  if (kRowBlock * p.x_rs >= kRangeLimit) return kNoPath;
  const int64_t blocks = (static_cast<int64_t>(p.M) + kRowBlock - 1) / kRowBlock;
  const int64_t cus = slc_host::device_cu_count(), share = (p.N * blocks + cus - 1) / cus;
  const int feat = static_cast<int>(share > 32 ? 32 : share);
  const int steps = (p.K + 63) / 64, waves = steps < 8 ? steps : 8;
  const int64_t groups = (static_cast<int64_t>(p.N) + feat - 1) / feat;
  if (groups * waves * 64 >= (int64_t{1} << 32)) return kNoPath;  // threads of one launch
  const dim3 grid(static_cast<unsigned>(groups), static_cast<unsigned>(blocks));
#define SLC_ROWS(MB, TILES, U) \
  hipLaunchKernelGGL((rows_kernel<T, MB, TILES, U>), grid, dim3(waves * 64), 0, stream, p, feat)
  if (feat <= 16) {
    if (p.M <= 16) SLC_ROWS(1, 1, 4);
    else SLC_ROWS(2, 1, 2);
  } else {
    SLC_ROWS(1, 2, 2);  // a vocabulary: choose() sends 4 rows at most here
  }
#undef SLC_ROWS
  return slc_host::check_launch("slc_hip_linear_q8(rows)");
}

// Which kernel takes a shape of aligned rows, all giving the same bits.
//
// rows_kernel where 16 x 16 fragments of the outputs are no more than CUs: tiles would leave
// most CUs idle (us, rows | 64 x 64 tiles: 8 x 1152 x 896 3.4 | 4.1, 16 x 896 x 4864 6.1 | 8.9,
// 16 x 4096 x 4096 7.5 | 9.6, 48 x 896 x 896 4.0 | 4.2, 250 x 256 x 4864 9.0 | 9.4; past that 16 x
// 6000 x 2048 6.4 | 5.9, 32 x 4096 x 4096 10.7 | 10.3), but for many rows of few features, whose
// tiles are as many (1900 x 32 x 896 4.7 | 4.3).  And for up to 4 rows of a vocabulary, whose
// weight it reads a little faster (1 x 50257 x 896 10.7 | 12.1, 1 x 151936 x 896 25.3 | 26.7; 2 x
// 32768 x 896 8.0 | 7.8, 8 x 151936 x 896 29.7 | 28.2).  Else up to 32 rows 64 x 64 tiles, which
// the others' empty rows make no faster (64 x 64 | 128 x 128: 8 x 151936 x 896 28.1 | 29.0, 16 x
// 151936 x 896 29.5 | 30.1).  Operands and outputs of every call apart, 600 MB of them.
//
// Else the tile that costs least: a start, and rounds over the CUs of a fixed part and one per
// k-tile (us; fitted to every tile's time at 123 shapes of 9 to 32768 rows, 896 to 151936
// features and K 896 to 11008, where the choice is the fastest tile or within 5 %, 0.2 % off on
// average, one buffer taking the outputs).  Rounds, not tiles: 8192 x 896 x 896 12.3 us as one
// round of 256 x 128, 12.6 as two of 128 x 128 (outputs apart, as above: 13.4 and 14.3); 4096 x
// 9728 x 896 43.5 as five rounds of 256 x 128, 50 as three of 256 x 256 (56 and 57); 32768 x 896 x
// 4864 127 as two of 256 x 256, 137 as four of 256 x 128; 65 x 896 x 896 4.5 as 64 x 64, 7.9 as
// 256 x 128.
enum Kernel { kRows, k64x64, k128x64, k128x128, k256x128, k256x256 };
inline Kernel choose(int64_t M, int64_t N, int64_t K) {
  const int64_t cus = slc_host::device_cu_count();
  if ((M + 15) / 16 * ((N + 15) / 16) <= cus && (M <= 32 || N >= 128)) return kRows;
  if (M <= 32) return M <= 4 && N >= 50000 ? kRows : k64x64;
  struct Cost {
    Kernel kernel;
    int bm, bn;
    double start, fixed, per_k;
  };
  constexpr Cost costs[] = {{k64x64, 64, 64, 2.7, 0.74, 0.20},
                            {k128x64, 128, 64, 2.4, 0.88, 0.31},
                            {k128x128, 128, 128, 2.7, 0.69, 0.50},
                            {k256x128, 256, 128, 4.5, 1.24, 0.74},
                            {k256x256, 256, 256, 2.9, 4.9, 1.36}};
  const int64_t k_tiles = (K + kBK - 1) / kBK;
  Kernel best = k64x64;
  double least = 0.0;
  for (const Cost& c : costs) {
    const int64_t tiles = ((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
    const double rounds = static_cast<double>((tiles + cus - 1) / cus);
    const double cost = c.start + rounds * (c.fixed + c.per_k * static_cast<double>(k_tiles));
    if (c.kernel == k64x64 || cost < least) {
      best = c.kernel;
      least = cost;
    }
  }
  return best;
}

template <typename T>
int launch(const Problem& p, hipStream_t stream) {
  const bool aligned = ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.w)) & 15) == 0 &&
                       p.K % 16 == 0 && p.x_rs % 16 == 0;
  if (aligned) {
    // Rings no deeper than the loads' latency asks for: a deeper one puts off the first tile (us,
    // 64 x 64 with 4 | 5 | 6 | 9 stages: 512 x 896 x 896 4.7 | 4.8 | 5.0 | 5.4, 16 x 151936 x 896
    // 29.7 | 28.4 | 28.5 | 29.1; 128 x 128 with 3 | 4: 2048 x 1152 x 896 7.5 | 7.8).  Four producers
    // issue them sooner than two (512 x 896 x 4864 10.5 | 11.1).
    int rc = kNoPath;
    switch (choose(p.M, p.N, p.K)) {
      case kRows:
        rc = launch_rows<T>(p, stream);
        break;
      case k64x64:
        rc = launch_stream<T, 64, 64, 2, 2, 4, 5, 8>(p, stream);
        break;
      case k128x64:
        rc = launch_stream<T, 128, 64, 2, 2, 4, 4, 8>(p, stream);
        break;
      case k128x128:
        rc = launch_stream<T, 128, 128, 2, 4, 4, 3, 8>(p, stream);
        break;
      case k256x128:
        rc = launch_stream<T, 256, 128, 4, 2, 4, 3, 4>(p, stream);
        break;
      default:
        rc = launch_turns<T>(p, stream);
    }
    if (rc != kNoPath) return rc;
  }
  // Other rows: 128 x 128 tiles from a round of them over the CUs on, where they are not half
  // empty; else 64 x 64, of which several share a CU (us, 64 x 64 | 128 x 128: 301 x 1003 x 1001
  // 7.7 | 14.2, 2000 x 1003 x 1001 11.4 | 16.0, 500 x 9727 x 1001 22.0 | 23.0, 5 x 151937 x 897 40
  // | 44; 4096 x 1003 x 1001 20.0 | 17.9, 4096 x 9727 x 1001 138 | 91, 32768 x 897 x 3001 323 |
  // 204).
  auto any = [&](auto kernel, int64_t tile) -> int {
    // One grid holds 65535 tiles of rows, and fewer than 2^32 threads across the features.
    const int64_t most_m = 65535 * tile, most_n = ((1 << 24) - 1) * tile;
    Problem part = p;
    for (int64_t n0 = 0; n0 < p.N; n0 += most_n) {
      part.w = p.w + n0 * p.K;
      part.sw = p.sw + n0;
      part.bias = p.bias == nullptr ? nullptr : static_cast<const T*>(p.bias) + n0;
      part.N = static_cast<int>(p.N - n0 < most_n ? p.N - n0 : most_n);
      for (int64_t m0 = 0; m0 < p.M; m0 += most_m) {
        part.x = p.x + m0 * p.x_rs;
        part.sx = p.sx + m0;
        part.y = static_cast<T*>(p.y) + m0 * p.y_rs + n0;
        part.M = static_cast<int>(p.M - m0 < most_m ? p.M - m0 : most_m);
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((part.N + tile - 1) / tile), static_cast<unsigned>((part.M + tile - 1) / tile)),
                           dim3(256), 0, stream, part);
        const int rc = slc_host::check_launch("slc_hip_linear_q8(any)");
        if (rc != SLC_OK) return rc;
      }
    }
    return SLC_OK;
  };
  const int64_t large = ((static_cast<int64_t>(p.M) + 127) / 128) * ((static_cast<int64_t>(p.N) + 127) / 128);
  if (p.M > 64 && p.N > 64 && large >= slc_host::device_cu_count()) return any(tile_kernel<T, 128, 128>, 128);
  return any(tile_kernel<T, 64, 64>, 64);
}

}  // namespace

extern "C" int slc_hip_linear_q8(const int8_t* input, const float* in_scales, const int8_t* weight,
                                 const float* weight_scales, const void* bias, void* output,
                                 int dtype, int64_t rows, int64_t out_features, int64_t in_features,
                                 int64_t in_stride_row, int64_t out_stride_row, void* stream) {
  SLC_REQUIRE(slc_host::is_float_dtype(dtype), "slc_hip_linear_q8: bad dtype %d", dtype);
  SLC_REQUIRE(rows >= 0 && out_features > 0 && in_features > 0 && in_features <= SLC_Q8_MAX_K,
              "slc_hip_linear_q8: bad sizes M=%lld N=%lld K=%lld", (long long)rows,
              (long long)out_features, (long long)in_features);
  SLC_REQUIRE(rows < (1LL << 31) && out_features < (1LL << 31),
              "slc_hip_linear_q8: sizes exceed 2^31");
  SLC_REQUIRE(rows <= 1 || (in_stride_row >= 0 && out_stride_row >= out_features),
              "slc_hip_linear_q8: rows of %lld outputs overlap, or a stride is negative", (long long)out_features);
  if (rows == 0) return SLC_OK;
  SLC_REQUIRE(input && in_scales && weight && weight_scales && output,
              "slc_hip_linear_q8: null pointer");
  const uint64_t element = static_cast<uint64_t>(slc_host::dtype_size(dtype));
  SLC_REQUIRE((reinterpret_cast<uintptr_t>(in_scales) | reinterpret_cast<uintptr_t>(weight_scales)) % 4 == 0 &&
                  (reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(output)) % element == 0,
              "slc_hip_linear_q8: misaligned pointer");
  // The kernels tell rows past the last by their offsets; one row's strides say nothing.
  const Problem p{input, in_scales, weight, weight_scales, bias, output, static_cast<int>(rows),
                  static_cast<int>(out_features), static_cast<int>(in_features),
                  rows == 1 ? in_features : in_stride_row, rows == 1 ? out_features : out_stride_row};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == SLC_BF16) return launch<slc::bf16_t>(p, s);
  if (dtype == SLC_F16) return launch<slc::f16_t>(p, s);
  return launch<float>(p, s);
}
