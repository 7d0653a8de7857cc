// Rows to 8-bit codes with one scale per row: of a tensor, of its RMSNorm (with
// the residual's addition), or of a SwiGLU product.
//
// With y the row that is coded (float for the tensor itself, h * w * rstd for
// the norm, silu(g) * u for SwiGLU) and a = max |y|:
//   scale = a / 127,   code = nearest whole number, ties to even, of 127 y / a.
// rstd divides every y of a row alike, so the norm's codes are those of h * w
// and do not wait for the statistic.
//
// Every code is the formula's, not that of a rounded y: a code is decided in
// fp32 from v ~ y and 1 / a (one fma rounds v * 127 / a to a whole number, a
// second gives the exact distance r to it), and where |r| comes within the
// error of the fp32 form of 1/2 it is decided again in fp64 from the inputs,
// with a itself in fp64.  The fp32 form's error: products of two 16-bit values
// are exact in fp32, so 127 / a and nothing else rounds, 127 * 2^-23; products
// of fp32 values add 2 * 127 * 2^-24; SwiGLU's exp, sum, quotient and product
// add at most 8 * 127 * 2^-24.  kBorder covers each; about one element in 5000
// (SwiGLU) is decided twice.  Rows whose a is 0, not finite, or so small or
// large that fp32 products round or overflow run in fp64 as a whole.
//
// One workgroup of W waves holds a row (a wave each of four rows for W = 1) in
// registers, NV 16-byte vectors per lane, so every input is read once and every
// output written once: HBM-bound from about a thousand rows, bound by the launch
// and two dependent reductions below.  Rows past 16 waves' registers are read
// twice (LOOP).  The sum of squares is held in fp64: it costs a conversion and
// an fma per element, and no square overflows.
#include <float.h>

#include "common.hpp"

namespace {

enum Source { kPlain = 0, kNorm = 1, kAddNorm = 2, kSwiglu = 3 };

struct Args {
  const void* a;       // input, or gate
  const void* b;       // residual, or up
  const void* w;       // norm weight
  void* summed;        // a + b
  int8_t* codes;
  float* scales;
  int64_t rows, a_rs, b_rs;
  int hidden;
  float eps;
};

constexpr float kMagic = 12582912.0f;   // 1.5 * 2^23: adding it rounds to a whole number
constexpr float kLow = 0x1p-60f, kHigh = 0x1p100f;  // a in fp32: products neither lost nor infinite
// SwiGLU: where exp(-g) overflows fp32, |silu(g)| < 2^-121 counts as 0; with
// |u| up to this the product is under 2^-31 of the least a.
constexpr float kMostUp = 0x1p30f;

template <typename T, int SRC>
struct Traits {
  static constexpr int VEC = 16 / sizeof(T);
  static constexpr bool kHasB = SRC == kAddNorm || SRC == kSwiglu;
  static constexpr bool kHasW = SRC == kNorm || SRC == kAddNorm;
  // Whether the fp32 v may differ from y (then a is taken again in fp64).
  static constexpr bool kInexact = SRC == kSwiglu || (kHasW && sizeof(T) == 4);
  static constexpr float kBorder = 0.5f - (SRC == kSwiglu ? 0x1.8p-14f : 0x1p-14f);
  // v within this factor below the largest v may be the largest y.
  static constexpr float kNear = 1.0f - 0x1p-19f;
};

template <typename T>
struct Raw {
  uint4 a, b, w;
};

// 16 bytes from an address of any alignment that T allows, zeros past `left`
// elements.
template <typename T>
__device__ __forceinline__ uint4 load_vec(const T* p, int left) {
  constexpr int VEC = 16 / sizeof(T);
  uint4 v = make_uint4(0, 0, 0, 0);
  if (left >= VEC) {
    __builtin_memcpy(&v, p, 16);
  } else {
    T e[VEC] = {};
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (k < left) e[k] = p[k];
    __builtin_memcpy(&v, e, 16);
  }
  return v;
}

template <typename T>
__device__ __forceinline__ float elem(const uint4& v, int k) {
  T e[16 / sizeof(T)];
  __builtin_memcpy(e, &v, 16);
  return slc::to_f32(e[k]);
}

// round(a + b) in T, element by element.
template <typename T>
__device__ __forceinline__ uint4 add_vec(const uint4& a, const uint4& b) {
  constexpr int VEC = 16 / sizeof(T);
  T o[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) o[k] = slc::from_f32<T>(elem<T>(a, k) + elem<T>(b, k));
  uint4 v;
  __builtin_memcpy(&v, o, 16);
  return v;
}

__device__ __forceinline__ float swiglu_f32(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// v of element k of a vector (after the residual's addition).
template <typename T, int SRC>
__device__ __forceinline__ float value(const Raw<T>& r, int k) {
  if constexpr (SRC == kPlain) return elem<T>(r.a, k);
  if constexpr (SRC == kSwiglu) return swiglu_f32(elem<T>(r.a, k), elem<T>(r.b, k));
  return elem<T>(r.a, k) * elem<T>(r.w, k);
}

// y of element i of a row in fp64, without the norm's rstd, from memory.
template <typename T, int SRC>
__device__ __forceinline__ double value64(const Args& p, int64_t row, int i) {
  const float a = slc::to_f32(static_cast<const T*>(p.a)[row * p.a_rs + i]);
  if constexpr (SRC == kPlain) return a;
  if constexpr (SRC == kNorm)
    return static_cast<double>(a) * slc::to_f32(static_cast<const T*>(p.w)[i]);
  const float b = slc::to_f32(static_cast<const T*>(p.b)[row * p.b_rs + i]);
  if constexpr (SRC == kAddNorm)
    return static_cast<double>(slc::round_to<T>(a + b)) * slc::to_f32(static_cast<const T*>(p.w)[i]);
  return a / (1.0 + exp(-static_cast<double>(a))) * b;
}

__device__ __forceinline__ double shfl_xor64(double v, int offset) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __shfl_xor(static_cast<uint32_t>(bits), offset, 64);
  const uint32_t hi = __shfl_xor(static_cast<uint32_t>(bits >> 32), offset, 64);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// The row's sums and maxima over its W waves.  Each use of an array of `slots`
// is followed by a barrier before its next.
struct Shared {
  double sum[16];
  double max64[16];
  uint32_t max32[16];
  uint32_t max_up[16];
};

template <typename T, int SRC, int W, int NV, bool LOOP>
__global__ __launch_bounds__(W == 1 ? 256 : W * 64) void quantize_kernel(Args p) {
  using TR = Traits<T, SRC>;
  constexpr int VEC = TR::VEC;
  constexpr int kLanes = W * 64;
  __shared__ Shared shared;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int64_t row = W == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + wave : blockIdx.x;
  if (row >= p.rows) return;  // whole waves, and whole workgroups for W > 1
  const int t = W == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int hidden = p.hidden;
  const int rounds = LOOP ? (hidden + kLanes * VEC - 1) / (kLanes * VEC) : NV;
  const T* a = static_cast<const T*>(p.a) + row * p.a_rs;
  const T* b = static_cast<const T*>(p.b) + row * p.b_rs;
  const T* w = static_cast<const T*>(p.w);
  T* summed = static_cast<T*>(p.summed) + row * hidden;
  int8_t* codes = p.codes + row * hidden;

  auto load = [&](int i, Raw<T>& r) {
    const int e = (t + kLanes * i) * VEC;
    const int left = hidden - e;
    r.a = load_vec<T>(a + e, left);
    if constexpr (TR::kHasW) r.w = load_vec<T>(w + e, left);
    if constexpr (TR::kHasB) r.b = load_vec<T>(b + e, left);
  };

  // ---- the row's largest |v|, its sum of squares, the sum h ------------------
  Raw<T> raw[LOOP ? 1 : NV];
  float v[(LOOP || SRC != kSwiglu) ? 1 : NV][VEC];
  double sq = 0.0;
  uint32_t top = 0, top_up = 0;
  if constexpr (!LOOP) {
#pragma unroll
    for (int i = 0; i < NV; ++i) load(i, raw[i]);
  }
  auto gather = [&](int i, Raw<T>& r, float (&keep)[VEC]) {
    const int e = (t + kLanes * i) * VEC;
    const int left = hidden - e;
    if (left <= 0) return;
    if constexpr (SRC == kAddNorm) {
      r.a = add_vec<T>(r.a, r.b);
      if (left >= VEC) {
        __builtin_memcpy(summed + e, &r.a, 16);
      } else {
        T o[VEC];
        __builtin_memcpy(o, &r.a, 16);
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          if (k < left) summed[e + k] = o[k];
      }
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const float x = value<T, SRC>(r, k);
      if constexpr (SRC == kSwiglu) {
        keep[k] = x;
        top_up = max(top_up, __float_as_uint(fabsf(elem<T>(r.b, k))));
      }
      // As bits: a NaN is above infinity and stays.
      top = max(top, __float_as_uint(fabsf(x)));
      if constexpr (TR::kHasW) {
        const double h = elem<T>(r.a, k);
        sq = fma(h, h, sq);
      }
    }
  };
  if constexpr (LOOP) {
    for (int i = 0; i < rounds; ++i) {
      load(i, raw[0]);
      gather(i, raw[0], v[0]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) gather(i, raw[i], v[SRC == kSwiglu ? i : 0]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    top = max(top, static_cast<uint32_t>(__shfl_xor(top, o, 64)));
    if constexpr (SRC == kSwiglu) top_up = max(top_up, static_cast<uint32_t>(__shfl_xor(top_up, o, 64)));
    if constexpr (TR::kHasW) sq += shfl_xor64(sq, o);
  }
  if constexpr (W > 1) {
    if ((t & 63) == 0) {
      shared.max32[wave] = top;
      shared.max_up[wave] = top_up;
      shared.sum[wave] = sq;
    }
    __syncthreads();
    top = top_up = 0;
    sq = 0.0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      top = max(top, shared.max32[i]);
      top_up = max(top_up, shared.max_up[i]);
      sq += shared.sum[i];
    }
  }
  // Every wave of the row holds the same values from here on.
  const float vmax = __uint_as_float(top);
  bool fast = vmax >= kLow && vmax <= kHigh;
  if constexpr (SRC == kSwiglu) fast = fast && __uint_as_float(top_up) <= kMostUp;

  // ---- a in fp64 ---------------------------------------------------------------
  double a64 = vmax;
  if (TR::kInexact || !fast) {
    a64 = 0.0;
    bool bad = false;
    auto take = [&](int e) {
      const double y = fabs(value64<T, SRC>(p, row, e));
      bad = bad || !(y <= DBL_MAX);
      a64 = y > a64 ? y : a64;
    };
    if (fast) {
      if constexpr (TR::kInexact) {
        const float near = vmax * TR::kNear;
        auto pick = [&](int i, const Raw<T>& r, const float (&kept)[VEC]) {
          const int e = (t + kLanes * i) * VEC;
          uint32_t mask = 0;
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            const float x = SRC == kSwiglu && !LOOP ? kept[k] : value<T, SRC>(r, k);
            mask |= fabsf(x) >= near ? 1u << k : 0u;
          }
          if (e >= hidden) mask = 0;
          while (mask != 0) {  // elements past the row hold 0, under `near`
            take(e + __builtin_ctz(mask));
            mask &= mask - 1;
          }
        };
        if constexpr (LOOP) {
          for (int i = 0; i < rounds; ++i) {
            load(i, raw[0]);
            if constexpr (SRC == kAddNorm) raw[0].a = add_vec<T>(raw[0].a, raw[0].b);
            pick(i, raw[0], v[0]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < NV; ++i) pick(i, raw[i], v[SRC == kSwiglu ? i : 0]);
        }
      }
    } else {
      for (int e = t; e < hidden; e += kLanes) take(e);
    }
    if (bad) a64 = __builtin_inf();
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const double other = shfl_xor64(a64, o);
      a64 = other > a64 ? other : a64;
    }
    if constexpr (W > 1) {
      if ((t & 63) == 0) shared.max64[wave] = a64;
      __syncthreads();
      a64 = 0.0;
#pragma unroll
      for (int i = 0; i < W; ++i) a64 = shared.max64[i] > a64 ? shared.max64[i] : a64;
    }
  }

  // ---- the scale ---------------------------------------------------------------
  double scale = a64 / 127.0;
  if constexpr (TR::kHasW) scale /= sqrt(sq / static_cast<double>(hidden) + static_cast<double>(p.eps));
  const bool coded = scale <= static_cast<double>(FLT_MAX);  // false for NaN
  if (t == 0) p.scales[row] = coded ? static_cast<float>(scale) : __builtin_nanf("");

  // ---- the codes ---------------------------------------------------------------
  auto code64 = [&](int e) {
    return static_cast<int>(rint(value64<T, SRC>(p, row, e) * 127.0 / a64));
  };
  if (!fast) {
    for (int e = t; e < hidden; e += kLanes)
      codes[e] = static_cast<int8_t>(coded && a64 > 0.0 ? code64(e) : 0);
    return;
  }
  const float inv = 127.0f / static_cast<float>(a64);
  auto emit = [&](int i, const Raw<T>& r, const float (&kept)[VEC]) {
    const int e = (t + kLanes * i) * VEC;
    const int left = hidden - e;
    if (left <= 0) return;
    uint32_t bits[VEC];
    float off[VEC], worst = 0.0f;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const float x = SRC == kSwiglu && !LOOP ? kept[k] : value<T, SRC>(r, k);
      const float whole = fmaf(x, inv, kMagic);
      bits[k] = __float_as_uint(whole);
      off[k] = fabsf(fmaf(x, inv, kMagic - whole));
      worst = fmaxf(worst, off[k]);
    }
    uint64_t packed = 0;
#pragma unroll
    for (int k = 0; k < VEC; ++k) packed |= static_cast<uint64_t>(bits[k] & 0xff) << (8 * k);
    if (worst > TR::kBorder) {
      uint32_t mask = 0;
#pragma unroll
      for (int k = 0; k < VEC; ++k) mask |= off[k] > TR::kBorder ? 1u << k : 0u;
      while (mask != 0) {  // elements past the row hold 0, at no border
        const int k = __builtin_ctz(mask);
        const uint64_t code = static_cast<uint64_t>(code64(e + k) & 0xff);
        packed = (packed & ~(uint64_t{0xff} << (8 * k))) | code << (8 * k);
        mask &= mask - 1;
      }
    }
    if (!coded) packed = 0;
    if (left >= VEC) {
      __builtin_memcpy(codes + e, &packed, VEC);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (k < left) codes[e + k] = static_cast<int8_t>(packed >> (8 * k));
    }
  };
  if constexpr (LOOP) {
    for (int i = 0; i < rounds; ++i) {
      load(i, raw[0]);
      if constexpr (SRC == kAddNorm) raw[0].a = add_vec<T>(raw[0].a, raw[0].b);
      emit(i, raw[0], v[0]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) emit(i, raw[i], v[SRC == kSwiglu ? i : 0]);
  }
}

template <typename T, int SRC>
int launch(const Args& p, const char* what, hipStream_t stream) {
  const int vecs = (p.hidden + Traits<T, SRC>::VEC - 1) / Traits<T, SRC>::VEC;
#define SLC_Q8(W, NV, LOOP)                                                              \
  hipLaunchKernelGGL((quantize_kernel<T, SRC, W, NV, LOOP>),                             \
                     dim3(static_cast<unsigned>(W == 1 ? (p.rows + 3) / 4 : p.rows)),    \
                     dim3(W == 1 ? 256 : W * 64), 0, stream, p)
  if (vecs <= 64) {
    SLC_Q8(1, 1, false);
  } else if (vecs <= 128) {
    SLC_Q8(1, 2, false);
  } else if (vecs <= 256) {
    SLC_Q8(4, 1, false);
  } else if (vecs <= 512) {
    SLC_Q8(4, 2, false);
  } else if (vecs <= 768) {
    SLC_Q8(4, 3, false);
  } else if (vecs <= 2048) {
    SLC_Q8(16, 2, false);
  } else if (vecs <= 4096) {
    SLC_Q8(16, 4, false);
  } else {
    SLC_Q8(16, 1, true);
  }
#undef SLC_Q8
  return slc_host::check_launch(what);
}

template <int SRC>
int dispatch(const Args& p, int dtype, const char* what, void* stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == SLC_BF16) return launch<slc::bf16_t, SRC>(p, what, s);
  if (dtype == SLC_F16) return launch<slc::f16_t, SRC>(p, what, s);
  return launch<float, SRC>(p, what, s);
}

int check(const char* what, int dtype, int64_t rows, int64_t hidden) {
  SLC_REQUIRE(slc_host::is_float_dtype(dtype), "%s: bad dtype %d", what, dtype);
  SLC_REQUIRE(rows >= 0 && rows <= INT32_MAX && hidden > 0 && hidden <= SLC_Q8_MAX_K,
              "%s: bad sizes rows=%lld hidden=%lld", what, (long long)rows, (long long)hidden);
  return SLC_OK;
}

bool aligned(const void* p, int dtype) {
  return reinterpret_cast<uintptr_t>(p) % slc_host::dtype_size(dtype) == 0;
}

}  // namespace

extern "C" int slc_hip_quantize_q8(const void* input, int8_t* codes, float* scales, int dtype,
                                   int64_t rows, int64_t hidden, int64_t in_stride_row,
                                   void* stream) {
  const char* what = "slc_hip_quantize_q8";
  const int rc = check(what, dtype, rows, hidden);
  if (rc != SLC_OK || rows == 0) return rc;
  SLC_REQUIRE(input && codes && scales, "%s: null pointer", what);
  SLC_REQUIRE(aligned(input, dtype) && aligned(scales, SLC_F32), "%s: misaligned pointer", what);
  Args p{};
  p.a = input;
  p.codes = codes;
  p.scales = scales;
  p.rows = rows;
  p.a_rs = in_stride_row;
  p.hidden = static_cast<int>(hidden);
  return dispatch<kPlain>(p, dtype, what, stream);
}

extern "C" int slc_hip_rms_norm_q8(const void* input, const void* residual, const void* weight,
                                   void* summed, int8_t* codes, float* scales, int dtype,
                                   int64_t rows, int64_t hidden, int64_t in_stride_row,
                                   int64_t residual_stride_row, float epsilon, void* stream) {
  const char* what = "slc_hip_rms_norm_q8";
  const int rc = check(what, dtype, rows, hidden);
  if (rc != SLC_OK || rows == 0) return rc;
  SLC_REQUIRE(input && weight && codes && scales, "%s: null pointer", what);
  SLC_REQUIRE((residual == nullptr) == (summed == nullptr),
              "%s: a residual comes with a place for the sum, and the other way round", what);
  SLC_REQUIRE(aligned(input, dtype) && aligned(residual, dtype) && aligned(weight, dtype) &&
                  aligned(summed, dtype) && aligned(scales, SLC_F32),
              "%s: misaligned pointer", what);
  Args p{};
  p.a = input;
  p.b = residual;
  p.w = weight;
  p.summed = summed;
  p.codes = codes;
  p.scales = scales;
  p.rows = rows;
  p.a_rs = in_stride_row;
  p.b_rs = residual_stride_row;
  p.hidden = static_cast<int>(hidden);
  p.eps = epsilon;
  if (residual == nullptr) return dispatch<kNorm>(p, dtype, what, stream);
  return dispatch<kAddNorm>(p, dtype, what, stream);
}

extern "C" int slc_hip_swiglu_q8(const void* gate, const void* up, int8_t* codes, float* scales,
                                 int dtype, int64_t rows, int64_t hidden, int64_t gate_stride_row,
                                 int64_t up_stride_row, void* stream) {
  const char* what = "slc_hip_swiglu_q8";
  const int rc = check(what, dtype, rows, hidden);
  if (rc != SLC_OK || rows == 0) return rc;
  SLC_REQUIRE(gate && up && codes && scales, "%s: null pointer", what);
  SLC_REQUIRE(aligned(gate, dtype) && aligned(up, dtype) && aligned(scales, SLC_F32),
              "%s: misaligned pointer", what);
  Args p{};
  p.a = gate;
  p.b = up;
  p.codes = codes;
  p.scales = scales;
  p.rows = rows;
  p.a_rs = gate_stride_row;
  p.b_rs = up_stride_row;
  p.hidden = static_cast<int>(hidden);
  return dispatch<kSwiglu>(p, dtype, what, stream);
}
