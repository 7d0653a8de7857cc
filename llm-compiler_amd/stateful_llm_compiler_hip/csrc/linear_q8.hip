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

// 16 codes from any address, zeros past `left` of them.
__device__ __forceinline__ uint4 load_codes(const int8_t* p, int left) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (left >= 16) {
    __builtin_memcpy(&v, p, 16);
  } else if (left > 0) {
    uint32_t word[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 15; ++i)
      if (i < left) word[i / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(p[i])) << (8 * (i % 4));
    v = make_uint4(word[0], word[1], word[2], word[3]);
  }
  return v;
}

// float(sum) * sx * sw + bias; the last two in one fma (and one rounding) in
// every kernel, so that all give the same bits.
__device__ __forceinline__ float finish(int sum, float sx, float sw, float bias) {
  return fmaf(static_cast<float>(sum) * sx, sw, bias);
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

// Any sizes, strides and alignment: BM x BN tiles staged through registers into
// one LDS tile pair, four waves of 2 x 2.
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256) void tile_kernel(Problem p) {
  constexpr int TM = BM / 2, TN = BN / 2, FM = TM / 16, FN = TN / 16;
  constexpr int XPT = BM * kChunks / 256, WPT = BN * kChunks / 256;
  __shared__ __attribute__((aligned(16))) unsigned char xs[BM * kBK];
  __shared__ __attribute__((aligned(16))) unsigned char ws[BN * kBK];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wm = wave >> 1, wn = wave & 1;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * BM, n0 = static_cast<int64_t>(blockIdx.x) * BN;

  i32x4_t acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};

  for (int k0 = 0; k0 < p.K; k0 += kBK) {
    uint4 xr[XPT], wr[WPT];
#pragma unroll
    for (int i = 0; i < XPT; ++i) {
      const int id = tid + 256 * i, row = id / kChunks, k = k0 + (id % kChunks) * 16;
      xr[i] = load_codes(p.x + (m0 + row) * p.x_rs + k, m0 + row < p.M ? p.K - k : 0);
    }
#pragma unroll
    for (int i = 0; i < WPT; ++i) {
      const int id = tid + 256 * i, row = id / kChunks, k = k0 + (id % kChunks) * 16;
      wr[i] = load_codes(p.w + (n0 + row) * p.K + k, n0 + row < p.N ? p.K - k : 0);
    }
    __syncthreads();  // the tiles before are read
#pragma unroll
    for (int i = 0; i < XPT; ++i) {
      const int id = tid + 256 * i;
      *reinterpret_cast<uint4*>(xs + lds_offset(id / kChunks, id % kChunks)) = xr[i];
    }
#pragma unroll
    for (int i = 0; i < WPT; ++i) {
      const int id = tid + 256 * i;
      *reinterpret_cast<uint4*>(ws + lds_offset(id / kChunks, id % kChunks)) = wr[i];
    }
    __syncthreads();
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
  }
  // Lane (c, g) of a 16 x 16 fragment: column c, rows 4g .. 4g + 3.
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    const int64_t n = n0 + wn * TN + j * 16 + c;
    if (n >= p.N) continue;
    const float sw = p.sw[n];
    const float bias = p.bias != nullptr ? slc::to_f32(static_cast<const T*>(p.bias)[n]) : 0.0f;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t m = m0 + wm * TM + i * 16 + 4 * g + r;
        if (m >= p.M) continue;
        static_cast<T*>(p.y)[m * p.y_rs + n] = slc::from_f32<T>(finish(acc[i][j][r], p.sx[m], sw, bias));
      }
  }
}

template <typename T>
int launch(const Problem& p, hipStream_t stream) {
  const int64_t m_tiles = (static_cast<int64_t>(p.M) + 63) / 64;
  const int64_t n_tiles = (static_cast<int64_t>(p.N) + 63) / 64;
  SLC_REQUIRE(m_tiles <= 65535, "slc_hip_linear_q8: %d rows exceed one launch's grid", p.M);
  hipLaunchKernelGGL((tile_kernel<T, 64, 64>),
                     dim3(static_cast<unsigned>(n_tiles), static_cast<unsigned>(m_tiles)), dim3(256),
                     0, stream, p);
  return slc_host::check_launch("slc_hip_linear_q8");
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
  if (rows == 0) return SLC_OK;
  SLC_REQUIRE(input && in_scales && weight && weight_scales && output,
              "slc_hip_linear_q8: null pointer");
  const uint64_t element = static_cast<uint64_t>(slc_host::dtype_size(dtype));
  SLC_REQUIRE((reinterpret_cast<uintptr_t>(in_scales) | reinterpret_cast<uintptr_t>(weight_scales)) % 4 == 0 &&
                  (reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(output)) % element == 0,
              "slc_hip_linear_q8: misaligned pointer");
  const Problem p{input, in_scales, weight, weight_scales, bias, output, static_cast<int>(rows),
                  static_cast<int>(out_features), static_cast<int>(in_features), in_stride_row,
                  out_stride_row};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == SLC_BF16) return launch<slc::bf16_t>(p, s);
  if (dtype == SLC_F16) return launch<slc::f16_t>(p, s);
  return launch<float>(p, s);
}
