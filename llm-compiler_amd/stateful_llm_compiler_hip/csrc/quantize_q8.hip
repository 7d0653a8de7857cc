// Rows to 8-bit codes with one scale per row: of a tensor, of its RMSNorm (with
// the residual's addition), or of a SwiGLU product.
//
// With y the row that is coded (the tensor itself, h * w * rstd for the norm,
// silu(g) * u for SwiGLU) and a = max |y|:
//   scale = a / 127,   code = nearest whole number, ties to even, of 127 y / a.
// rstd divides every y of a row alike, so the norm's codes are those of h * w
// and do not wait for the statistic.
//
// Every code is the formula's, not that of a rounded y: with v ~ y in fp32, v * 127 / a
// is rounded to a whole number (one fma) with the factor just below and just above 127 /
// a, far enough apart to cover every error of the fp32 form, and where the two differ
// the code is decided again in fp64 from the inputs, with a itself in fp64.  In units of
// 2^-24: a and 127 / a round by 1 each, the factor's distance by 1, v by 0 where both
// factors have 16 bits, by 1 in the norm of fp32 values, by 8 in SwiGLU (silu_f32);
// kApart covers the sum.  About one element in 30000 (SwiGLU) is decided twice.  Rows
// whose a is 0, not finite, or so small or large that fp32 products round or overflow
// run in fp64 as a whole.
//
// One workgroup holds a row in registers, NV 16-byte vectors per lane, so every
// input is read once and every output written once: HBM-bound from about a
// thousand rows, bound by the launch and two dependent reductions below.  Rows
// past 16 waves' registers are read twice (LOOP).  All loads are issued before
// the first use, without branches: buffer loads whose range ends with the row.
// Graphs over six sets of inputs: 16384 x 896 fp16 9.5 us (4.7 TB/s), SwiGLU 4096 x 4864 bf16
// 23.8 (4.2 TB/s, with 14 us of vector instructions), norm of 9001 x 1001 fp32 11.2 (4.0
// TB/s), addition and norm of 4096 x 896 bf16 8.0, of one row 2.4.  Where that fp32 norm's
// time goes, over sixteen sets: 12.4, a plain copy of as many bytes 11.2; without the fp64
// maximum 11.6, without the fp64 squares 12.1, without second decisions 11.8, without all
// three 11.3.
#include <float.h>

#include <initializer_list>
#include <type_traits>

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
  int64_t row0, a_rs, b_rs;
  double per_hidden;   // 1 / hidden
  int hidden;
  float eps;
};

constexpr int kMaxWaves = 16;
constexpr float kMagic = 12582912.0f;   // 1.5 * 2^23: adding it rounds to a whole number
// a in fp32 between these: no product is lost or infinite.
constexpr float kLow = 0x1p-60f, kHigh = 0x1p60f;
// SwiGLU: where 1 + exp(-g) has no normal fp32 reciprocal, |silu(g)| < 2^-119
// counts as 0; with |u| up to this the product is under 2^-31 of the least a.
constexpr float kMostUp = 0x1p28f;

template <typename T, int SRC>
struct Traits {
  static constexpr int VEC = 16 / sizeof(T);
  static constexpr bool kHasB = SRC == kAddNorm || SRC == kSwiglu;
  static constexpr bool kHasW = SRC == kNorm || SRC == kAddNorm;
  // Whether the fp32 v may differ from y.  Then a is taken in fp64: of products of two fp32
  // values, exact there, beside v (norm 9001 x 1001, one set of inputs | several: 10.9 us |
  // 11.8; in a second pass over the values near the largest, behind a second barrier, 13.1 |
  // 12.9); of SwiGLU, whose fp64 values cost too much for that, in such a second pass.
  static constexpr bool kWide = kHasW && sizeof(T) == 4;
  static constexpr bool kInexact = SRC == kSwiglu || kWide;
  static constexpr float kApart = (SRC == kSwiglu ? 14 : kInexact ? 6 : 4) * 0x1p-24f;
  // v within this factor below the largest v may be the largest y.
  static constexpr float kNear = 1.0f - 0x1p-19f;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(const void* row, int bytes) {
  const uint64_t address = reinterpret_cast<uint64_t>(row);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(address));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(address >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(
      reinterpret_cast<void*>(static_cast<uint64_t>(hi) << 32 | lo), 0,
      __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

// One row of an operand: 16-byte vectors, zeros past its end.  The range holds
// whole 4-byte words; an odd 16-bit element at the end is loaded by itself.
template <typename T>
struct Row {
  const T* base;
  __amdgpu_buffer_rsrc_t rsrc;
  __device__ __forceinline__ Row(const void* p, int64_t offset, int hidden)
      : base(static_cast<const T*>(p) + offset),
        rsrc(row_rsrc(base, hidden * static_cast<int>(sizeof(T)) & ~3)) {}
  __device__ __forceinline__ u32x4 load(int vec) const {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, vec * 16, 0, 0));
  }
  // The odd element into the vector that it belongs to.
  __device__ __forceinline__ void patch(u32x4& v, int vec, int hidden) const {
    if constexpr (sizeof(T) == 2) {
      const int last = hidden - 1;
      if (last / 8 != vec) return;
      const uint32_t bits = __builtin_bit_cast(uint16_t, base[last]);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (last % 8 == 2 * k) v[k] = bits;
    }
  }
};

// Element k of a vector as fp32.
template <typename T>
__device__ __forceinline__ float elem(const u32x4& v, int k) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(v[k]);
  } else {
    T e;
    e.bits = static_cast<uint16_t>(v[k / 2] >> (16 * (k % 2)));
    return slc::to_f32(e);
  }
}

// round(a + b) in T, element by element.
template <typename T>
__device__ __forceinline__ u32x4 add_vec(const u32x4& a, const u32x4& b) {
  u32x4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) {
      v[k] = __float_as_uint(elem<T>(a, k) + elem<T>(b, k));
    } else {
      v[k] = slc::pack2<T>(elem<T>(a, 2 * k) + elem<T>(b, 2 * k), elem<T>(a, 2 * k + 1) + elem<T>(b, 2 * k + 1));
    }
  }
  return v;
}

// silu(g) to 7 * 2^-24 of itself: exp(-g) = 2^t (1 + d), where t is -g log2(e) in fp32
// and d the rest of it times ln 2.  (2^t is off by 2 * 2^-24, which the quotient keeps at
// most, its product with 1 + d by 1, the sum by 1, the reciprocal by 2, the product by 1.)
// A bf16 g times the first 15 bits of log2(e) is exact, so the rest is one product; d^2 / 2
// is left out, under 2^-24 down to g = -66, where |silu| is under 2^-89 and, with |u| up to
// kMostUp, the product below the least a that comes here.  Where 2^t is infinite the
// quotient is 0 (d is positive there in bf16; else it is not looked at).
template <typename T>
__device__ __forceinline__ float silu_f32(float g) {
  constexpr float kLn2 = 0x1.62e430p-1f;
  float e;
  if constexpr (std::is_same<T, slc::bf16_t>::value) {
    constexpr float kLog2e = 0x1.7154p+0f, kRestLn2 = 0x1.d94ae1p-18f * kLn2;
    const float p = __builtin_amdgcn_exp2f(-g * kLog2e);
    e = fmaf(p, -g * kRestLn2, p);
  } else {
    constexpr float kLog2e = 0x1.715476p+0f, kLog2eLow = 0x1.4ae0c0p-26f;
    const float t = -g * kLog2e;
    const float p = __builtin_amdgcn_exp2f(t);
    e = t < 128.0f ? fmaf(p, fmaf(-g, kLog2eLow, fmaf(-g, kLog2e, -t)) * kLn2, p) : p;
  }
  return g * __builtin_amdgcn_rcpf(1.0f + e);
}

// h (the input, or its rounded sum with the residual) and y, without the norm's
// rstd, of element i of a row in fp64, from memory.
template <typename T, int SRC>
__device__ __forceinline__ double summed_value(const Args& p, int64_t row, int i) {
  const float a = slc::to_f32(static_cast<const T*>(p.a)[row * p.a_rs + i]);
  if constexpr (SRC != kAddNorm) return a;
  return slc::round_to<T>(a + slc::to_f32(static_cast<const T*>(p.b)[row * p.b_rs + i]));
}
template <typename T, int SRC>
__device__ __forceinline__ double value64(const Args& p, int64_t row, int i) {
  const double h = summed_value<T, SRC>(p, row, i);
  if constexpr (Traits<T, SRC>::kHasW) return h * slc::to_f32(static_cast<const T*>(p.w)[i]);
  if constexpr (SRC == kSwiglu)
    return h / (1.0 + exp(-h)) * slc::to_f32(static_cast<const T*>(p.b)[row * p.b_rs + i]);
  return h;
}

// 1 / sqrt(x) to a few units of 2^-52: the instruction's 2^-24 or better, squared
// by a Newton step.  (NaN for 0 and infinity, whose rows have no scale.)
__device__ __forceinline__ double rsqrt64(double x) {
  double r = __builtin_amdgcn_rsq(x);
  r = fma(r * 0.5, fma(-x * r, r, 1.0), r);
  return fma(r * 0.5, fma(-x * r, r, 1.0), r);
}

// The largest magnitude so far (as its bits, a pair of them for 16-bit types) and one
// more word of the operand; and that magnitude as fp32 bits in the end.
template <typename T>
__device__ __forceinline__ void up_max(uint32_t& most, uint32_t word) {
  if constexpr (sizeof(T) == 4) {
    most = max(most, word & 0x7fffffffu);
  } else {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    most = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, most),
                                                                  __builtin_bit_cast(u16x2, word & 0x7fff7fffu)));
  }
}
template <typename T>
__device__ __forceinline__ uint32_t up_bits(uint32_t most) {
  if constexpr (sizeof(T) == 4) {
    return most;
  } else {
    T e;
    e.bits = static_cast<uint16_t>(max(most & 0xffffu, most >> 16));
    return __float_as_uint(slc::to_f32(e));
  }
}

// ---- reductions over a wave in the VALU --------------------------------------------
// Lane pairs one apart, two apart, mirrored in eight, mirrored in sixteen (DPP),
// then rows of 16 and halves of 32 (lane swaps): every lane ends with the total.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, true);
}
constexpr int kPairs = 0xB1, kQuads = 0x4E, kHalfMirror = 0x141, kMirror = 0x140;

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t x) {
  x = max(x, dpp<kPairs>(x));
  x = max(x, dpp<kQuads>(x));
  x = max(x, dpp<kHalfMirror>(x));
  x = max(x, dpp<kMirror>(x));
  auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(r[0], r[1]);
  r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max(r[0], r[1]);
}

template <typename OP>
__device__ __forceinline__ double wave_reduce64(double v, OP op) {
  auto both = [](uint32_t lo, uint32_t hi) {
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
  };
  auto split = [](double x, uint32_t& lo, uint32_t& hi) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, x);
    lo = static_cast<uint32_t>(bits);
    hi = static_cast<uint32_t>(bits >> 32);
  };
  uint32_t lo, hi;
  split(v, lo, hi);
  v = op(v, both(dpp<kPairs>(lo), dpp<kPairs>(hi)));
  split(v, lo, hi);
  v = op(v, both(dpp<kQuads>(lo), dpp<kQuads>(hi)));
  split(v, lo, hi);
  v = op(v, both(dpp<kHalfMirror>(lo), dpp<kHalfMirror>(hi)));
  split(v, lo, hi);
  v = op(v, both(dpp<kMirror>(lo), dpp<kMirror>(hi)));
  split(v, lo, hi);
  auto l = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
  auto h = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
  v = op(both(l[0], h[0]), both(l[1], h[1]));
  split(v, lo, hi);
  l = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
  h = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
  return op(both(l[0], h[0]), both(l[1], h[1]));
}

struct Shared {
  double sum[kMaxWaves];
  double most64[kMaxWaves];
  double max64[kMaxWaves];
  uint32_t max32[kMaxWaves];
  uint32_t max_up[kMaxWaves];
};

// Low bytes of eight (four) words, first lowest.
__device__ __forceinline__ uint32_t pack4(const uint32_t* b) {
  const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
  return lo | hi;
}

// Three vectors a lane with up to eight waves, whose registers then suffice.
__host__ __device__ constexpr int max_waves(int nv) { return nv == 3 ? 8 : kMaxWaves; }

// One workgroup of whole waves per row.
template <typename T, int SRC, int NV, bool LOOP>
__global__ __launch_bounds__(max_waves(NV) * 64) void quantize_kernel(Args p) {
  using TR = Traits<T, SRC>;
  constexpr int VEC = TR::VEC;
  __shared__ Shared shared;
  const int lanes = blockDim.x, waves = lanes >> 6;
  const int t = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int64_t row = p.row0 + blockIdx.x;
  const int hidden = p.hidden;
  const int rounds = LOOP ? (hidden + lanes * VEC - 1) / (lanes * VEC) : NV;
  const bool odd = sizeof(T) == 2 && (hidden & 1) != 0;
  const Row<T> ra(p.a, row * p.a_rs, hidden);
  const Row<T> rb(TR::kHasB ? p.b : p.a, TR::kHasB ? row * p.b_rs : 0, TR::kHasB ? hidden : 0);
  const Row<T> rw(TR::kHasW ? p.w : p.a, 0, TR::kHasW ? hidden : 0);
  T* summed = static_cast<T*>(p.summed) + row * hidden;
  int8_t* codes = p.codes + row * hidden;

  u32x4 a[LOOP ? 1 : NV], b[TR::kHasB && !LOOP ? NV : 1], w[TR::kHasW && !LOOP ? NV : 1];
  float v[LOOP ? 1 : NV][VEC];
  auto load = [&](int i, int slot) {
    const int vec = t + lanes * i;
    a[slot] = ra.load(vec);
    if constexpr (TR::kHasW) w[slot] = rw.load(vec);
    if constexpr (TR::kHasB) b[slot] = rb.load(vec);
  };
  auto patch = [&](int i, int slot) {
    const int vec = t + lanes * i;
    ra.patch(a[slot], vec, hidden);
    if constexpr (TR::kHasW) rw.patch(w[slot], vec, hidden);
    if constexpr (TR::kHasB) rb.patch(b[slot], vec, hidden);
  };
  // The slot's v (and h, in a) from its vectors; zeros past the row stay zeros.
  auto evaluate = [&](int slot) {
    if constexpr (SRC == kAddNorm) a[slot] = add_vec<T>(a[slot], b[slot]);
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const float x = elem<T>(a[slot], k);
      if constexpr (SRC == kPlain) v[slot][k] = x;
      if constexpr (TR::kHasW) v[slot][k] = x * elem<T>(w[slot], k);
      if constexpr (SRC == kSwiglu) v[slot][k] = silu_f32<T>(x) * elem<T>(b[slot], k);
    }
  };

  // ---- the largest |v|, the sum of squares, the sum h --------------------------
  // As bits, in two halves: the largest positive (and positive NaNs above) by
  // signed order, the largest negative by unsigned order.
  // Squares are summed in fp64, so that the scale is rounded once (inputs of four sets,
  // fp32 chains of eight | fp64: addition and norm of 4096 x 896 bf16 7.2 us | 7.3, norm of it
  // 4.35 | 4.5, norm of 2100 x 4864 bf16 7.75 | 8.15, of 9001 x 1001 fp32 10.4 | 10.4; the
  // chains were off by up to five half steps); no square leaves the range of fp64.
  int most = 0;
  uint32_t least = 0, most_up = 0;
  double sq = 0.0, most64 = 0.0;
  auto gather = [&](int i, int slot) {
    evaluate(slot);
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const uint32_t bits = __float_as_uint(v[slot][k]);
      most = max(most, static_cast<int>(bits));
      least = max(least, bits);
      if constexpr (TR::kHasW) {
        const double h = elem<T>(a[slot], k);
        sq = fma(h, h, sq);
        if constexpr (TR::kWide) most64 = fmax(most64, fabs(h * elem<T>(w[slot], k)));
      }
    }
    if constexpr (SRC == kSwiglu) {
#pragma unroll
      for (int k = 0; k < 4; ++k) up_max<T>(most_up, b[slot][k]);
    }
    if constexpr (SRC == kAddNorm) {
      const int e = (t + lanes * i) * VEC;
      if (e + VEC <= hidden) {
        __builtin_memcpy(summed + e, &a[slot], 16);
      } else if (e < hidden) {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          if (e + k < hidden) summed[e + k] = slc::from_f32<T>(elem<T>(a[slot], k));
      }
    }
  };
  if constexpr (LOOP) {
    for (int i = 0; i < rounds; ++i) {
      load(i, 0);
      if (odd) patch(i, 0);
      gather(i, 0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) load(i, i);
    if (odd) {
#pragma unroll
      for (int i = 0; i < NV; ++i) patch(i, i);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) gather(i, i);
  }
  uint32_t top = max(static_cast<uint32_t>(most), (least >> 31) != 0 ? least & 0x7fffffffu : 0u);
  const uint32_t own_top = top;  // this lane's largest
  top = wave_max_u32(top);
  if constexpr (SRC == kSwiglu) most_up = wave_max_u32(up_bits<T>(most_up));
  auto add = [](double x, double y) { return x + y; };
  auto larger = [](double x, double y) { return x > y ? x : y; };
  if constexpr (TR::kHasW) sq = wave_reduce64(sq, add);
  if constexpr (TR::kWide) most64 = wave_reduce64(most64, larger);
  if (waves > 1) {
    if ((t & 63) == 0) {
      shared.max32[wave] = top;
      if constexpr (SRC == kSwiglu) shared.max_up[wave] = most_up;
      if constexpr (TR::kHasW) shared.sum[wave] = sq;
      if constexpr (TR::kWide) shared.most64[wave] = most64;
    }
    __syncthreads();
    for (int i = 0; i < waves; ++i) {
      top = max(top, shared.max32[i]);
      if constexpr (SRC == kSwiglu) most_up = max(most_up, shared.max_up[i]);
      if constexpr (TR::kWide) most64 = larger(most64, shared.most64[i]);
    }
  }
  // Every wave of the row holds the same top from here on.
  const float vmax = __uint_as_float(top);
  bool fast = vmax >= kLow && vmax <= kHigh;
  if constexpr (SRC == kSwiglu) fast = fast && __uint_as_float(most_up) <= kMostUp;

  // ---- a in fp64: of SwiGLU's values near the largest, or of all that are not zero -----
  double a64 = TR::kWide ? most64 : vmax;
  if (SRC == kSwiglu || !fast) {
    a64 = 0.0;
    const float near = vmax * TR::kNear;
    auto pick = [&](int i, int slot) {
      uint32_t mask = 0;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        // NaNs and infinities are not zero; 0 stays 0 whatever it is multiplied
        // by, but an infinity (whose product is NaN in v too).
        const bool live = fast ? fabsf(v[slot][k]) >= near
                               : elem<T>(a[slot], k) != 0.0f || v[slot][k] != 0.0f;
        mask |= live ? 1u << k : 0u;
      }
      while (mask != 0) {  // elements past the row hold 0
        const int k = __builtin_ctz(mask), e = (t + lanes * i) * VEC + k;
        mask &= mask - 1;
        double y = fabs(value64<T, SRC>(p, row, e));
        if (!(y <= DBL_MAX)) y = __builtin_inf();
        a64 = y > a64 ? y : a64;
      }
    };
    if (!fast || __uint_as_float(own_top) >= near) {
      if constexpr (LOOP) {
        for (int i = 0; i < rounds; ++i) {
          load(i, 0);
          if (odd) patch(i, 0);
          evaluate(0);
          pick(i, 0);
        }
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) pick(i, i);
      }
    }
    a64 = wave_reduce64(a64, larger);
    if (waves > 1) {
      if ((t & 63) == 0) shared.max64[wave] = a64;
      __syncthreads();
      for (int i = 0; i < waves; ++i) a64 = shared.max64[i] > a64 ? shared.max64[i] : a64;
    }
  }
  // a / 127, times the norm's rstd; 1 / 127 rounds far below fp32.
  auto scale_of_row = [&]() {
    double scale = a64 * (1.0 / 127.0);
    if constexpr (TR::kHasW) {
      double squares = sq;
      if (waves > 1) {
        squares = 0.0;
        for (int i = 0; i < waves; ++i) squares += shared.sum[i];
      }
      scale *= rsqrt64(fma(squares, p.per_hidden, static_cast<double>(p.eps)));
    }
    return scale;
  };

  // ---- the codes ---------------------------------------------------------------
  auto code64 = [&](int e) {
    return static_cast<int>(rint(value64<T, SRC>(p, row, e) * 127.0 / a64));
  };
  if (!fast) {
    const double scale = scale_of_row();
    const bool coded = scale <= static_cast<double>(FLT_MAX);  // false for NaN
    if (t == 0) p.scales[row] = coded ? static_cast<float>(scale) : __builtin_nanf("");
    const bool zero = !coded || a64 == 0.0;
    for (int e = t; e < hidden; e += lanes) codes[e] = static_cast<int8_t>(zero ? 0 : code64(e));
    return;
  }
  const float inv = 127.0f / static_cast<float>(a64);
  const float below = inv * (1.0f - TR::kApart), above = inv * (1.0f + TR::kApart);
  auto emit = [&](int i, int slot) {
    const int e = (t + lanes * i) * VEC;
    if (e >= hidden) return;
    uint32_t lo[VEC], hi[VEC], packed[VEC / 4], differ = 0, apart[VEC / 4];
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      lo[k] = __float_as_uint(fmaf(v[slot][k], below, kMagic));
      hi[k] = __float_as_uint(fmaf(v[slot][k], above, kMagic));
    }
#pragma unroll
    for (int j = 0; j < VEC / 4; ++j) {
      packed[j] = pack4(lo + 4 * j);
      apart[j] = packed[j] ^ pack4(hi + 4 * j);
      differ |= apart[j];
    }
    if (differ != 0) {  // elements past the row hold 0, at no border
#pragma unroll
      for (int j = 0; j < VEC / 4; ++j) {
        uint32_t rest = apart[j];
        while (rest != 0) {
          const int k = __builtin_ctz(rest) / 8;
          const uint32_t byte = 0xffu << (8 * k);
          packed[j] = (packed[j] & ~byte) | static_cast<uint32_t>(code64(e + 4 * j + k) & 0xff) << (8 * k);
          rest &= ~byte;
        }
      }
    }
    if (e + VEC <= hidden) {
      __builtin_memcpy(codes + e, packed, VEC);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (e + k < hidden) codes[e + k] = static_cast<int8_t>(packed[k / 4] >> (8 * (k % 4)));
    }
  };
  if constexpr (LOOP) {
    for (int i = 0; i < rounds; ++i) {
      load(i, 0);
      if (odd) patch(i, 0);
      evaluate(0);
      emit(i, 0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) emit(i, i);
  }

  // ---- the scale: not waited for by the codes ------------------------------------
  if (wave != 0) return;
  const double scale = scale_of_row();
  if (t == 0) p.scales[row] = scale <= static_cast<double>(FLT_MAX) ? static_cast<float>(scale) : __builtin_nanf("");
}

// Vectors per lane for rows of `vecs` vectors, or 0 for rows that no registers hold.  Few
// rows leave CUs idle, so as many waves as the row fills share it (us, one | two vectors a
// lane: SwiGLU 32 x 4864 bf16 4.7 | 5.0, norm 128 x 1001 3.8 | 4.4).  Many rows: a wave's
// reductions cost about as much as a vector does, so more vectors share them, while the
// row's waves still suffice to hide its loads (one | two | three | four: SwiGLU 4096 x 4864
// bf16 35.8 | 24.7 | 23.3 | 24.6, codes 19.3 | 13.0 | 12.6 | 12.6, norm 4096 x 896 8.0 | 8.1
// | 8.7 | 9.2, SwiGLU 4096 x 4864 fp32 two 40.7, three 34.0, four 33.0).
inline int vectors_per_lane(int vecs, int64_t rows) {
  auto waves = [&](int nv) { return (vecs + 64 * nv - 1) / (64 * nv); };
  for (int nv : {1, 2, 4})
    if (waves(nv) <= max_waves(nv) && rows * waves(nv) <= 2048) return nv;
  if (vecs <= 256) return 2;
  if (waves(3) <= max_waves(3)) return 3;
  return waves(4) <= max_waves(4) ? 4 : 0;
}

template <typename T, int SRC>
int launch(Args p, int64_t rows, const char* what, hipStream_t stream) {
  const int vecs = (p.hidden + Traits<T, SRC>::VEC - 1) / Traits<T, SRC>::VEC;
  auto waves = [&](int nv) { return (vecs + 64 * nv - 1) / (64 * nv); };
  // A grid holds fewer than 2^32 threads.
  auto go = [&](auto kernel, int w) {
    const int64_t most = ((int64_t{1} << 32) - 1) / (64 * w);
    for (p.row0 = 0; p.row0 < rows; p.row0 += most) {
      const int64_t part = rows - p.row0 < most ? rows - p.row0 : most;
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(part)), dim3(static_cast<unsigned>(w) * 64), 0,
                         stream, p);
      const int rc = slc_host::check_launch(what);
      if (rc != SLC_OK) return rc;
    }
    return static_cast<int>(SLC_OK);
  };
  switch (vectors_per_lane(vecs, rows)) {
    case 1:
      return go(quantize_kernel<T, SRC, 1, false>, waves(1));
    case 2:
      return go(quantize_kernel<T, SRC, 2, false>, waves(2));
    case 3:
      return go(quantize_kernel<T, SRC, 3, false>, waves(3));
    case 4:
      return go(quantize_kernel<T, SRC, 4, false>, waves(4));
    default:
      return go(quantize_kernel<T, SRC, 1, true>, kMaxWaves);
  }
}

template <int SRC>
int dispatch(const Args& p, int64_t rows, int dtype, const char* what, void* stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == SLC_BF16) return launch<slc::bf16_t, SRC>(p, rows, what, s);
  if (dtype == SLC_F16) return launch<slc::f16_t, SRC>(p, rows, what, s);
  return launch<float, SRC>(p, rows, what, s);
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
  p.a_rs = in_stride_row;
  p.hidden = static_cast<int>(hidden);
  return dispatch<kPlain>(p, rows, dtype, what, stream);
}

extern "C" int slc_hip_rms_norm_q8(const void* input, const void* residual, const void* weight,
                                   void* summed, int8_t* codes, float* scales, int dtype,
                                   int64_t rows, int64_t hidden, int64_t in_stride_row,
                                   int64_t residual_stride_row, float epsilon, void* stream) {
  const char* what = "slc_hip_rms_norm_q8";
  const int rc = check(what, dtype, rows, hidden);
  if (rc != SLC_OK || rows == 0) return rc;
  SLC_REQUIRE(input && weight && codes && scales, "%s: null pointer", what);
  SLC_REQUIRE(epsilon >= 0.0f && epsilon <= FLT_MAX, "%s: epsilon must be finite and not negative", what);
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
  p.a_rs = in_stride_row;
  p.b_rs = residual_stride_row;
  p.hidden = static_cast<int>(hidden);
  p.per_hidden = 1.0 / static_cast<double>(hidden);
  p.eps = epsilon;
  if (residual == nullptr) return dispatch<kNorm>(p, rows, dtype, what, stream);
  return dispatch<kAddNorm>(p, rows, dtype, what, stream);
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
  p.a_rs = gate_stride_row;
  p.b_rs = up_stride_row;
  p.hidden = static_cast<int>(hidden);
  return dispatch<kSwiglu>(p, rows, dtype, what, stream);
}
