// What the group norm kernels share: coefficients, activations, vectors of channels.
//   mu, var over the m = S*D elements of a (sample, group); r = 1/sqrt(var + eps); xh = (x - mu) r
//   z = xh*gamma_c + beta_c + res;  out = act(z)
//   g = dout*act'(z): dres = g, dbeta_c = sum g, dgamma_c = sum g xh, with A = sum_{group} gamma g, B = sum_{group} gamma g xh
//   dx = r (gamma g - (A + xh B)/m)
#pragma once
#include "common.h"

// Activation classes.  GN_CAP is every clipped ReLU; the plain one is clipped at infinity.
enum GnAct : int { GN_NONE = 0, GN_CAP = 1, GN_SILU = 2 };

struct GnStat { double mean, rstd; };

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) GnVec { T v[VEC]; };

template <typename T, int VEC>
__device__ __forceinline__ GnVec<T, VEC> gn_ld(const T* p) { return *reinterpret_cast<const GnVec<T, VEC>*>(p); }
template <typename T, int VEC>
__device__ __forceinline__ void gn_st(T* p, const GnVec<T, VEC>& v) { *reinterpret_cast<GnVec<T, VEC>*>(p) = v; }

// Coefficients of the VEC channels of one thread.  UG: they lie in one group, whose mean and deviation are held once.
//   forward: z = (x - mh)*sc + sh;  the mean is the fp32 pair (mh, ml), ml folded into sh
template <int VEC, bool UG> struct GnCoef {
  static constexpr int NG = UG ? 1 : VEC;
  float mh[NG], ml[NG], r[NG], sc[VEC], sh[VEC];
  __device__ __forceinline__ void load(const GnStat* st /* of this sample */, const float* gamma, const float* beta, int c0,
                                       int D) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int k = UG ? 0 : e;
      const GnStat s = st[(UG ? c0 : c0 + e) / D];
      mh[k] = (float)s.mean;
      ml[k] = (float)(s.mean - (double)mh[k]);
      r[k] = (float)s.rstd;
      sc[e] = (float)(s.rstd * (double)(gamma ? gamma[c0 + e] : 1.f));
      sh[e] = (beta ? beta[c0 + e] : 0.f) - ml[k] * sc[e];
    }
  }
};

// The pre-activation in fp64, z = x*sc + sh: on which side of an activation's border a value lies decides over the whole
// gradient of the element, and fp64 multiply-adds cost what fp32 ones do.
template <int VEC> struct GnBorder {
  double sc[VEC], sh[VEC];
  __device__ __forceinline__ void load(const GnStat* st, const float* gamma, const float* beta, int c0, int D) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const GnStat s = st[(c0 + e) / D];
      sc[e] = s.rstd * (double)(gamma ? gamma[c0 + e] : 1.f);
      sh[e] = (double)(beta ? beta[c0 + e] : 0.f) - s.mean * sc[e];
    }
  }
};
struct GnNoBorder {
  __device__ __forceinline__ void load(const GnStat*, const float*, const float*, int, int) {}
};
template <int ACT, int VEC> struct GnBorderOf { typedef GnNoBorder type; };
template <int VEC> struct GnBorderOf<GN_CAP, VEC> { typedef GnBorder<VEC> type; };

__device__ __forceinline__ float gn_sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f));
}

template <int ACT> __device__ __forceinline__ float gn_act(float z, float cap) {
  if constexpr (ACT == GN_SILU) return z * gn_sigmoid(z);
  if constexpr (ACT == GN_CAP) {
    z = z < 0.f ? 0.f : z;      // a NaN stays one
    z = z > cap ? cap : z;
  }
  return z;
}

// g of one element; x as stored, t = x - mh.
template <int ACT, int VEC, typename B>
__device__ __forceinline__ float gn_grad(float dy, float x, float t, float res, float sc, float sh, const B& b, int e,
                                         double cap) {
  if constexpr (ACT == GN_NONE) return dy;
  if constexpr (ACT == GN_SILU) {
    const float z = t * sc + sh + res, s = gn_sigmoid(z);
    return dy * (s * (1.f + z * (1.f - s)));
  }
  if constexpr (ACT == GN_CAP) {
    const double z = (double)x * b.sc[e] + b.sh[e] + (double)res;
    return z > 0.0 && z < cap ? dy : 0.f;
  }
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
