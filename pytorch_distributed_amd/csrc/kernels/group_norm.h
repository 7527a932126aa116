// What the group norm kernels share: coefficients, activations, vectors of channels.
//   mu, var over the m = S*D elements of a (sample, group); r = 1/sqrt(var + eps); xh = (x - mu) r
//   z = xh*gamma_c + beta_c + res;  out = act(z)
//   g = dout*act'(z): dres = g, dbeta_c = sum g, dgamma_c = sum g xh, with A = sum_{group} gamma g, B = sum_{group} gamma g xh
//   dx = r (gamma g - (A + xh B)/m)
#pragma once
#include "common.h"

#include <math.h>
#include <type_traits>

// Activations (the codes of the Python side).
enum GnAct : int { GN_NONE = 0, GN_RELU = 1, GN_CAP = 2, GN_SILU = 3 };
constexpr bool gn_is_relu(int act) { return act == GN_RELU || act == GN_CAP; }

struct GnStat { double mean, rstd; };

// Statistics of a group of m elements, from fp64 sums A of d = x - p and B of d^2.  B/m - (A/m)^2 as such would leave 2^-53 mean^2,
// which is more than the variance of values that are nearly alike.
// fp32: p is the group's first element (its first channel at the sample's first position), taken off each value in fp64, and
// (p - mean)^2 is at most m var: the variance is good to some m 2^-53 of itself wherever the mean lies.
// 16 bits: p is 0 (subtracting costs 400x28x28x128 fp16, D = 4, 60 us for 49).  All terms are multiples of q^2, q the last place
// of the least |x|: where m x^2 <= 2^53 q^2 for the largest one, A and B are exact, and with c = A/m as rounded and e = A - m c,
// m var = B - c A - c e, each difference rounded once.  Where that fails, then (m < 2^27) the least |x| is below a quarter of the
// largest, x^2 is at most 4 m var, and 2^-53 of it no more than above.
struct GnPair { double a, b; };
template <typename T> __device__ __forceinline__ void gn_add(GnPair& s, float x, double p) {
  const double d = sizeof(T) == 4 ? (double)x - p : (double)x;
  s.a += d;
  s.b += d * d;
}
__device__ __forceinline__ GnStat gn_stat(const GnPair& s, double p, double m, double im, double eps) {
  const double c = s.a * im, e = fma(-m, c, s.a);
  double var = (fma(-c, s.a, s.b) - c * e) * im;
  var = var < 0.0 ? 0.0 : var;  // (a NaN stays one)
  return GnStat{p + fma(e, im, c), 1.0 / sqrt(var + eps)};
}
// fp32: the first element of channel c's group; xn: the sample.
template <typename T> __device__ __forceinline__ double gn_first(const T* xn, int c, int D) {
  return sizeof(T) == 4 ? (double)ElemTraits<T>::to_f32(xn[c / D * D]) : 0.0;
}

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) GnVec {
  T v[VEC];
  __device__ __forceinline__ float f(int e) const { return ElemTraits<T>::to_f32(v[e]); }
};

// 16 bytes as four registers.  A vector that lives across branches and barriers is kept like this: as elements the
// compiler unpacks it at once, into twice the registers.
template <typename T> struct GnRaw {
  u32x4 u;
  __device__ __forceinline__ float f(int e) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(u[e]);
    else {
      const unsigned short h = (unsigned short)(e & 1 ? u[e >> 1] >> 16 : u[e >> 1]);
      return ElemTraits<T>::to_f32(__builtin_bit_cast(T, h));
    }
  }
  // f(e) - s.  fp16: one multiply-add that reads the half where it lies (one: 1.0 that the compiler does not see as such)
  __device__ __forceinline__ float sub(int e, float s, float one) const {
    if constexpr (sizeof(T) == 2 && ElemTraits<T>::code == PDA_F16) return __builtin_fmaf(f(e), one, -s);
    return f(e) - s;
  }
  // a + f(e)
  __device__ __forceinline__ float add(int e, float a, float one) const {
    if constexpr (sizeof(T) == 2 && ElemTraits<T>::code == PDA_F16) return __builtin_fmaf(f(e), one, a);
    return f(e) + a;
  }
  // elements whose bit is not set become 0
  __device__ __forceinline__ void keep(const bool (&on)[16 / sizeof(T)]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) u[i] = on[i] ? u[i] : 0u;
      else u[i] &= (on[2 * i] ? 0xffffu : 0u) | (on[2 * i + 1] ? 0xffff0000u : 0u);
    }
  }
  __device__ __forceinline__ void set(const float (&x)[16 / sizeof(T)]) {
    GnVec<T, 16 / sizeof(T)> v;
#pragma unroll
    for (int e = 0; e < (int)(16 / sizeof(T)); ++e) v.v[e] = ElemTraits<T>::from_f32(x[e]);
    u = __builtin_bit_cast(u32x4, v);
  }
};
template <typename T> __device__ __forceinline__ GnRaw<T> gn_ld_raw(const T* p) {
  return GnRaw<T>{*reinterpret_cast<const u32x4*>(p)};
}
template <typename T> __device__ __forceinline__ void gn_st_raw(T* p, const GnRaw<T>& v) { *reinterpret_cast<u32x4*>(p) = v.u; }

template <typename T, int VEC>
__device__ __forceinline__ GnVec<T, VEC> gn_ld(const T* p) { return *reinterpret_cast<const GnVec<T, VEC>*>(p); }
template <typename T, int VEC>
__device__ __forceinline__ void gn_st(T* p, const GnVec<T, VEC>& v) { *reinterpret_cast<GnVec<T, VEC>*>(p) = v; }

// The vector of a pass over rows, loaded ahead of its use.
template <typename T, int VEC>
using GnHeld = typename std::conditional<VEC * sizeof(T) == 16, GnRaw<T>, GnVec<T, VEC>>::type;
template <typename T, int VEC> __device__ __forceinline__ GnHeld<T, VEC> gn_ld_held(const T* p) {
  return *reinterpret_cast<const GnHeld<T, VEC>*>(p);
}

// The channel at a place of a row, where a row may be several positions next to each other.
__device__ __forceinline__ int gn_channel(int c, int C) {
  while (c >= C) c -= C;
  return c;
}

// Coefficients of the VEC channels of one thread: z = (x - mh)*sc + sh.  The mean is the fp32 pair (mh, ml), ml folded into
// sh.  UG: the channels lie in one group, whose mean is held once.
template <int VEC, bool UG> struct GnCoef {
  static constexpr int NG = UG ? 1 : VEC;
  float mh[NG], sc[VEC], sh[VEC];
  __device__ __forceinline__ float shmax() const {
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) m = fmaxf(m, fabsf(sh[e]));
    return m;
  }
  __device__ __forceinline__ void load(const GnStat* st /* of this sample */, const float* gamma, const float* beta, int c0,
                                       int D, int C) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int c = gn_channel(c0 + e, C);
      const GnStat s = st[(UG ? c0 : c) / D];
      const float m = (float)s.mean;
      mh[UG ? 0 : e] = m;
      sc[e] = (float)(s.rstd * (double)(gamma ? gamma[c] : 1.f));
      sh[e] = (beta ? beta[c] : 0.f) - (float)(s.mean - (double)m) * sc[e];
    }
  }
};

// sum g (x - mh) of a channel -> sum g xh
__device__ __forceinline__ float gn_centre(float gt, float g, const GnStat& s) {
  return (gt - (float)(s.mean - (double)(float)s.mean) * g) * (float)s.rstd;
}
// dx = g*sc + pa + (x - mh)*pb, from A/m and B/m
__device__ __forceinline__ void gn_dx_coefs(float A, float B, const GnStat& s, float& pa, float& pb) {
  const float r = (float)s.rstd;
  pb = -B * r * r;
  pa = -A * r - (float)(s.mean - (double)(float)s.mean) * pb;
}

// With the hardware's 2^x and 1/x: some 2^-22 in all, nothing to a 16-bit result and four steps of an fp32 one.
__device__ __forceinline__ float gn_sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f));
}

template <int ACT> __device__ __forceinline__ float gn_act(float z, float cap) {
  if constexpr (ACT == GN_SILU) return z * gn_sigmoid(z);
  if constexpr (gn_is_relu(ACT)) z = z < 0.f ? 0.f : z;  // a NaN stays one
  if constexpr (ACT == GN_CAP) z = z > cap ? cap : z;
  return z;
}

// Which of a vector's pre-activations lie between the borders 0 and cap, in fp64 from the fp64 statistics.
template <typename T, int VEC>
__device__ __forceinline__ unsigned gn_inside(const T* x, const T* res, const GnStat* st, const float* gamma, const float* beta,
                                              int c0, int D, int C, float cap) {
  unsigned on = 0;
#pragma unroll 1
  for (int e = 0; e < VEC; ++e) {
    const int c = gn_channel(c0 + e, C);
    const GnStat s = st[c / D];
    const double z = ((double)ElemTraits<T>::to_f32(x[e]) - s.mean) * s.rstd * (gamma ? (double)gamma[c] : 1.0) +
                     (beta ? (double)beta[c] : 0.0) + (res ? (double)ElemTraits<T>::to_f32(res[e]) : 0.0);
    on |= z > 0.0 && z < (double)cap ? 1u << e : 0u;
  }
  return on;
}

// The ReLUs' act'(z) of one element, and what decides whether its vector is looked at again: on which side of a border z
// lies decides over an element's whole gradient.  With z = t + sh + res, z's rounding error is below 6 u (|t| + |sh| + |res|),
// u = 2^-24, and next to 0 |t| is at most |sh| + |res| (next to the cap: and the cap).  So a vector whose least |z| is below
// 2e-6 (max |sh| + max |res|) is decided by gn_inside.
struct GnNear {
  float lo = INFINITY, hi = INFINITY, res = 0.f;
  template <int ACT> __device__ __forceinline__ bool inside(float z, float cap) {
    lo = fminf(lo, fabsf(z));
    if constexpr (ACT == GN_CAP) {
      hi = fminf(hi, fabsf(z - cap));
      return z > 0.f && z < cap;
    }
    return z > 0.f;
  }
  template <int ACT> __device__ __forceinline__ bool again(float shmax, float cap) const {
    const float tol = 2e-6f * (shmax + res);
    return lo < tol || (ACT == GN_CAP && hi < tol + 2e-6f * cap);
  }
};
// t = x - mh
template <typename V, int VEC, bool UG>
__device__ __forceinline__ float gn_silu_slope(float t, const V& w, bool wr, const GnCoef<VEC, UG>& k, int e) {
  float z = t * k.sc[e] + k.sh[e];
  if (wr) z += w.f(e);
  const float s = gn_sigmoid(z);
  return s * (1.f + z * (1.f - s));
}

// g = dout*act'(z) of a vector; x and res where they stand, c0 the channel of x[0].
template <int ACT, typename T, int VEC, bool UG, typename V>
__device__ __forceinline__ void gn_grads(float (&g)[VEC], const V& d, const V& v, const V& w, bool wr,
                                         const GnCoef<VEC, UG>& k, const T* x, const T* res, const GnStat* st,
                                         const float* gamma, const float* beta, int c0, int D, int C, float cap) {
  unsigned on = 0;
  if constexpr (gn_is_relu(ACT)) {
    GnNear near;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float z = (v.f(e) - k.mh[UG ? 0 : e]) * k.sc[e] + k.sh[e];
      if (wr) {
        const float r = w.f(e);
        z += r;
        near.res = fmaxf(near.res, fabsf(r));
      }
      on |= near.inside<ACT>(z, cap) ? 1u << e : 0u;
    }
    if (near.again<ACT>(k.shmax(), cap)) on = gn_inside<T, VEC>(x, wr ? res : nullptr, st, gamma, beta, c0, D, C, cap);
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const float dy = d.f(e);
    if constexpr (ACT == GN_NONE) g[e] = dy;
    if constexpr (gn_is_relu(ACT)) g[e] = (on >> e) & 1u ? dy : 0.f;
    if constexpr (ACT == GN_SILU) g[e] = dy * gn_silu_slope(v.f(e) - k.mh[UG ? 0 : e], w, wr, k, e);
  }
}

// Makes the compiler take a vector (or an offset) as new: what was computed from it - its elements in fp32, the addresses of
// a pass - is not kept in registers for the next pass.
template <typename T> __device__ __forceinline__ void gn_renew(GnRaw<T>& v) { asm volatile("" : "+v"(v.u)); }
__device__ __forceinline__ void gn_renew(unsigned& v) { asm volatile("" : "+v"(v)); }

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
