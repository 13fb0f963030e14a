// Softmax weights of logits in 64 bits, and the entries of rows that start at any
// element: shared by the kernels that decide a token by where a running sum over the
// vocabulary passes a border (verify.hip, choose.hip).
#pragma once

#include "slab_common.hpp"

namespace rrl {
namespace {

// 2^r for |r| <= 1/2: the polynomial through 2^r at the nine Chebyshev nodes of
// that interval, within 1.1e-12 of it, relative.
__device__ __forceinline__ double exp2_poly(double r) {
  double p = 0x1.63d1363942fefp-20;
  p = fma(p, r, 0x1.00dc4a534288bp-16);
  p = fma(p, r, 0x1.4308ac85a7a46p-13);
  p = fma(p, r, 0x1.5d8745a7281dep-10);
  p = fma(p, r, 0x1.3b2ab7181b773p-7);
  p = fma(p, r, 0x1.c6b08dd6fd237p-5);
  p = fma(p, r, 0x1.ebfbdff823cedp-3);
  p = fma(p, r, 0x1.62e42fef84cf0p-1);
  return fma(p, r, 1.0);
}

// Takes a whole number n, held in the low word of 1.5 2^52 + n, as an exponent.
__device__ __forceinline__ double with_exponent(double p, double whole) {
  return __hiloint2double(__double2hiint(p) + (int)((uint32_t)__double2loint(whole) << 20),
                          __double2loint(p));
}

// 2^max(t, -1000) for t <= 0.
__device__ __forceinline__ double exp2_neg(double t) {
  t = fmax(t, -1000.0);
  const double whole = t + 0x1.8p52;
  return with_exponent(exp2_poly(t - (whole - 0x1.8p52)), whole);
}

// max(a, b) of numbers that are not NaN: one instruction, where fmaxf spends a
// second on quieting its operand.
__device__ __forceinline__ float max2(float a, float b) {
  return __builtin_amdgcn_fmed3f(a, b, M<float>::inf());
}

// k 2^(c (x - m)) for the entries x <= m of a row.  With i = rint(c m), and x
// lifted to where its weight is 2^-1000 (so are impossible entries, -inf),
//   w = 1.5 2^52 - i + c x    holds rint(c x) - i in its low word
//   r = c x - rint(c x)       one fma, exact but for its rounding
// so an entry takes no reduction by its own maximum: 2^(i - c m) goes into k.
// Outside the range of that (c m past 2^20, or c so small that no float weighs
// 2^-1000, or so large that only subnormal steps below a maximum next to 0 weigh more)
// c (x - m) is formed first.
struct Weight {
  double c, scale, k, m, magic;  // k: scale 2^(i - c m)
  float least;
  bool direct;
  __device__ __forceinline__ Weight() {}
  __device__ __forceinline__ Weight(float max, double c_, double scale_)
      : c(c_), scale(scale_), k(scale_), m(max), magic(0x1.8p52) {
    const double mc = m * c, low = m - 1000.0 / c;
    direct = fabs(mc) < 0x1p20 && low > -3e38 && c < 0x1p100;
    least = (float)low;
    if (direct) {
      const double i = rint(mc);
      magic -= i;
      k *= exp2_poly(fma(-m, c, i));
    }
  }
  template <bool DIRECT>
  __device__ __forceinline__ double factor() const { return DIRECT ? k : scale; }
  template <bool DIRECT>
  __device__ __forceinline__ double unscaled(float x) const {
    if constexpr (DIRECT) {
      const double v = max2(x, least);
      const double whole = fma(v, c, magic);
      return with_exponent(exp2_poly(fma(v, c, magic - whole)), whole);
    } else {
      return exp2_neg(((double)x - m) * c);
    }
  }
  __device__ __forceinline__ double one(float x) const {
    return direct ? unscaled<true>(x) * k : unscaled<false>(x) * scale;
  }
};

// A row may start at any element: these 16 bytes are one global_load_dwordx4 at
// any address.
struct __attribute__((packed, aligned(2))) Any16 {
  u32x4 v;
};

// Entries i..i+EPV of a row, -inf past its end.
template <class Tag>
__device__ __forceinline__ void load_entries(const char* row, int64_t i, int64_t V,
                                             float (&x)[Pack16<Tag>::EPV]) {
  constexpr int EPV = Pack16<Tag>::EPV, SZ = 16 / EPV;
  if (i + EPV <= V) {
    Pack16<Tag>::unpack(reinterpret_cast<const Any16*>(row + i * SZ)->v, x);
    return;
  }
#pragma unroll
  for (int k = 0; k < EPV; ++k) {
    x[k] = -M<float>::inf();
    if (i + k < V) {
      if constexpr (SZ == 4) {
        x[k] = reinterpret_cast<const float*>(row)[i + k];
      } else {
        x[k] = Pack16<Tag>::one(reinterpret_cast<const uint16_t*>(row)[i + k]);
      }
    }
  }
}
template <class Tag>
__device__ __forceinline__ float load_entry(const char* row, int64_t i) {
  if constexpr (16 / Pack16<Tag>::EPV == 4) return reinterpret_cast<const float*>(row)[i];
  else return Pack16<Tag>::one(reinterpret_cast<const uint16_t*>(row)[i]);
}

// Butterfly over a row of 16 lanes, and over the wave.
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
  return __hiloint2double(dpp_i<CTRL>(__double2hiint(v)), dpp_i<CTRL>(__double2loint(v)));
}
__device__ __forceinline__ double row16_sum(double v) {
  v += dpp_d<kDppXor1>(v);
  v += dpp_d<kDppXor2>(v);
  v += dpp_d<kDppHalfMirror>(v);
  return v + dpp_d<kDppMirror>(v);
}
__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, dpp_f<kDppXor1>(v));
  v = fmaxf(v, dpp_f<kDppXor2>(v));
  v = fmaxf(v, dpp_f<kDppHalfMirror>(v));
  return fmaxf(v, dpp_f<kDppMirror>(v));
}
__device__ __forceinline__ int row16_min(int v) {
  v = min(v, dpp_i<kDppXor1>(v));
  v = min(v, dpp_i<kDppXor2>(v));
  v = min(v, dpp_i<kDppHalfMirror>(v));
  return min(v, dpp_i<kDppMirror>(v));
}
__device__ __forceinline__ double lane_read_d(double v, int l) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), l),
                          __builtin_amdgcn_readlane(__double2loint(v), l));
}
__device__ __forceinline__ double wave_sum_d(double v) {
  v = row16_sum(v);
  return (lane_read_d(v, 0) + lane_read_d(v, 16)) + (lane_read_d(v, 32) + lane_read_d(v, 48));
}

}  // namespace
}  // namespace rrl
