// Group norm with a sample's groups held in registers: one workgroup takes a slab of whole groups of one sample, reads it
// once, forms the sums over it and writes the result from the registers.
//
// Against the passes over row chunks this saves one read of x forward, one of x, dout and res backward, and two launches
// each way.  It holds S x W elements (W channels of the slab) in up to 1024 threads x NV 16-byte vectors; gn_resident_plan
// chooses W, the block and NV.  Neighbouring slabs share memory lines (W channels are 32 bytes or more of a row), so the
// workgroups of a sample run on one XCD next to each other.
#pragma once
#include "group_norm.h"

#include <math.h>

struct GnPlan {
  int W, threads, nv;  // nv = 0: does not fit
};

// Resident vectors of one thread: what stays below the 128 registers that 1024 threads leave each.
constexpr int GN_NV_FWD = 13, GN_NV_BWD = 7;

inline GnPlan gn_resident_plan(int esize, long long N, long long S, int C, int G, bool bwd) {
  GnPlan best{0, 0, 0};
  const int vec = 16 / esize, D = C / G;
  if (C % vec || S > 1024 * GN_NV_FWD) return best;
  int a = D, b = vec;
  while (b) { const int t = a % b; a = b; b = t; }
  const int unit = D / a * vec;  // whole groups and whole vectors
  const int units = C / unit, most = bwd ? GN_NV_BWD : GN_NV_FWD;
  for (int k = units; k >= 1; --k) {
    if (units % k) continue;
    const int W = unit * k, vt = W / vec;
    if (vt > 1024 || (W * esize < 32 && W != C)) continue;
    int threads = 0;
    for (int nt = 64; nt <= 1024 && !threads; nt *= 2)
      if (nt >= vt && (S + nt / vt - 1) / (nt / vt) <= most) threads = nt;
    if (!threads) continue;
    // spread a slab over more threads while the vectors of each stay two or more
    while (threads < 1024 && (S + threads / vt - 1) / (threads / vt) > 4 && S * vt <= 2048) threads *= 2;
    const int nv = (int)((S + threads / vt - 1) / (threads / vt));
    best = GnPlan{W, threads, nv};
    // wide enough a launch, and two workgroups or more on a CU, so that one's loads cover the other's sums
    if (N * (units / k) >= 1024 && threads <= 512) break;
  }
  return best;
}

// Totals of every channel of the slab: buf [RS][W] (written, not yet synchronised) -> buf[0..W).  tmp: max(threads, W).
template <typename V> __device__ __forceinline__ void gn_channel_totals(V* buf, V* tmp, int W, int RS) {
  const int NT = blockDim.x, parts = NT > W ? NT / W : 1;
  __syncthreads();
  for (int i = threadIdx.x; i < W * parts; i += NT) {
    const int c = i % W, p = i / W;
    V a = 0;
    for (int r = p; r < RS; r += parts) a += buf[r * W + c];
    tmp[i] = a;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < W; c += NT) {
    V a = tmp[c];
    for (int p = 1; p < parts; ++p) a += tmp[p * W + c];
    buf[c] = a;
  }
  __syncthreads();
}

inline size_t gn_fwd_lds(int W, int threads, int vec, int D) {
  if (D % vec == 0) return 16ull * (threads + (size_t)(threads / 64 + 1) * (W / D));
  return 8ull * ((size_t)(threads / (W / vec)) * W + (threads > W ? threads : W) + 2 * (W / D));
}
inline size_t gn_bwd_lds(int W, int threads, int vec, int D) {
  return 4ull * (2 * (size_t)(threads / (W / vec)) * W + 2 * (threads > W ? threads : W) + 2 * (W / D));
}

struct GnPair { double a, b; };

// Sums over every group of the slab: s[e] of every thread that is on -> s[e] of the group of slot e (UG: one slot).
template <int VEC, bool UG>
__device__ __forceinline__ void gn_group_totals(GnPair (&s)[UG ? 1 : VEC], double* lds, int W, int D, int RS, int col, int rl,
                                                bool on, bool shuffles) {
  const int VT = W / VEC, Gs = W / D, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, NW = blockDim.x >> 6;
  if constexpr (UG) {
    GnPair* buf = reinterpret_cast<GnPair*>(lds);
    const int dv = D / VEC;
    double a = on ? s[0].a : 0.0, b = on ? s[0].b : 0.0;
    if (shuffles) {  // powers of two: the lanes of a group reduce among themselves, then one value a wave
      for (int o = 1; o < dv; o <<= 1) {
        a += __shfl_xor(a, o, 64);
        b += __shfl_xor(b, o, 64);
      }
      for (int o = VT; o < 64; o <<= 1) {
        a += __shfl_xor(a, o, 64);
        b += __shfl_xor(b, o, 64);
      }
      if (lane < VT && lane % dv == 0) buf[wave * Gs + lane / dv] = GnPair{a, b};
      __syncthreads();
      const int g = col / dv;
      s[0] = buf[g];
      for (int w = 1; w < NW; ++w) {
        s[0].a += buf[w * Gs + g].a;
        s[0].b += buf[w * Gs + g].b;
      }
      return;
    }
    // a wave takes a group: RS x dv values
    GnPair* grp = buf + RS * VT;
    if (on) buf[rl * VT + col] = GnPair{a, b};
    __syncthreads();
    for (int g = wave; g < Gs; g += NW) {
      a = b = 0.0;
      for (int j = lane; j < RS * dv; j += 64) {
        const GnPair t = buf[(j / dv) * VT + g * dv + j % dv];
        a += t.a;
        b += t.b;
      }
      a = wave_sum_f64(a);
      b = wave_sum_f64(b);
      if (lane == 0) grp[g] = GnPair{a, b};
    }
    __syncthreads();
    if (on) s[0] = grp[col / dv];
  } else {
    double* tmp = lds + RS * W;
    double* grp = tmp + (blockDim.x > W ? blockDim.x : W);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (on)
#pragma unroll
        for (int e = 0; e < VEC; ++e) lds[rl * W + col * VEC + e] = h ? s[e].b : s[e].a;
      gn_channel_totals(lds, tmp, W, RS);
      for (int g = wave; g < Gs; g += NW) {
        double t = 0.0;
        for (int d = lane; d < D; d += 64) t += lds[g * D + d];
        t = wave_sum_f64(t);
        if (lane == 0) grp[g] = t;
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < VEC; ++e) (h ? s[e].b : s[e].a) = grp[(col * VEC + e) / D];
    }
  }
}

template <typename T, int NV, bool UG, int ACT>
__global__ void __launch_bounds__(1024)
gn_resident_fwd_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ out, const float* __restrict__ gamma,
                       const float* __restrict__ beta, int S, int C, int G, int W, double eps, float cap, int shuffles,
                       GnStat* __restrict__ stats) {
  extern __shared__ double lds[];
  constexpr int VEC = 16 / sizeof(T), NG = UG ? 1 : VEC;
  const int slabs = C / W, D = C / G, VT = W / VEC, RS = blockDim.x / VT;
  const int id = xcd_remap(blockIdx.x, gridDim.x), n = id / slabs, c0 = (id % slabs) * W;
  const int col = threadIdx.x % VT, rl = threadIdx.x / VT;
  const bool on = rl < RS;
  // addresses: one for the workgroup, one offset a thread, one step a vector
  const long long slab = (long long)n * S * C + c0;
  unsigned off = (unsigned)(rl * C + col * VEC);
  const auto at = [&](int i) { return slab + (long long)i * RS * C; };
  GnRaw<T> v[NV];
  const auto in = [&](int i) { return on && rl + i * RS < S; };
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (in(i)) v[i] = gn_ld_raw<T>(x + at(i) + off);
  // A thread's rows relative to its first one, in fp32 (an outlier there raises the variance with its own rounding); from
  // there in fp64, where the square of a mean may be taken off the mean of the squares.
  float s1[VEC], s2[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) s1[e] = s2[e] = 0.f;
  int cnt = in(0) ? 1 : 0;
#pragma unroll
  for (int i = 1; i < NV; ++i)
    if (in(i)) {
      ++cnt;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = v[i].f(e) - v[0].f(e);
        s1[e] += d;
        s2[e] += d * d;
      }
    }
  GnPair tot[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i) tot[i] = GnPair{0.0, 0.0};
  if (cnt)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const double p = (double)v[0].f(e), kp = (double)cnt * p, d = (double)s1[e];
      tot[UG ? 0 : e].a += d + kp;
      tot[UG ? 0 : e].b += (double)s2[e] + p * (d + d + kp);
    }
  gn_group_totals<VEC, UG>(tot, lds, W, D, RS, col, rl, on, shuffles);
  const double im = 1.0 / ((double)S * D);
  float mh[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    tot[i].a *= im;
    mh[i] = (float)tot[i].a;
  }
  if (!on) return;
  float sc[VEC], sh[VEC];
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const double mean = tot[i].a, ml = mean - (double)mh[i];
    double var = tot[i].b * im - mean * mean;
    var = var < 0.0 ? 0.0 : var;  // (a NaN stays one)
    const double r = 1.0 / sqrt(var + eps);
    if (rl == 0) {
      const int c = c0 + col * VEC + i;  // the thread of a group's first channel writes its statistics
      if (c % D == 0) stats[(long long)n * G + c / D] = GnStat{mean, r};
    }
#pragma unroll
    for (int e = UG ? 0 : i; e < (UG ? VEC : i + 1); ++e) {
      const int c = c0 + col * VEC + e;
      sc[e] = (float)(r * (double)(gamma ? gamma[c] : 1.f));
      sh[e] = (beta ? beta[c] : 0.f) - (float)ml * sc[e];
    }
  }
  gn_renew(off);
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (gn_renew(v[i]), in(i)) {
      GnRaw<T> w;
      if (res) w = gn_ld_raw<T>(res + at(i) + off);
      float y[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float z = (v[i].f(e) - mh[UG ? 0 : e]) * sc[e] + sh[e];
        if (res) z += w.f(e);
        y[e] = gn_act<ACT>(z, cap);
      }
      v[i].set(y);
      gn_st_raw<T>(out + at(i) + off, v[i]);
    }
}

// dx and dres of a slab, and its channels' {sum g, sum g xh} -> part[n][c].
template <typename T, int NV, bool UG, int ACT>
__global__ void __launch_bounds__(1024)
gn_resident_bwd_kernel(const T* __restrict__ x, const T* __restrict__ res, const T* __restrict__ dout, T* __restrict__ dx,
                       T* __restrict__ dres, const float* __restrict__ gamma, const float* __restrict__ beta,
                       const GnStat* __restrict__ stats, int S, int C, int G, int W, float cap, float2* __restrict__ part) {
  extern __shared__ float ldsf[];
  constexpr int VEC = 16 / sizeof(T);
  const int slabs = C / W, D = C / G, VT = W / VEC, RS = blockDim.x / VT, Gs = W / D;
  const int id = xcd_remap(blockIdx.x, gridDim.x), n = id / slabs, c0 = (id % slabs) * W;
  const int col = threadIdx.x % VT, rl = threadIdx.x / VT, ct = c0 + col * VEC;
  const bool on = rl < RS;
  const long long slab = (long long)n * S * C + c0;
  unsigned off = (unsigned)(rl * C + col * VEC);
  const auto at = [&](int i) { return slab + (long long)i * RS * C; };
  const auto in = [&](int i) { return on && rl + i * RS < S; };
  const bool wr = ACT != GN_NONE && res;
  const GnStat* stn = stats + (long long)n * G;
  GnRaw<T> v[NV], d[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (in(i)) {
      v[i] = gn_ld_raw<T>(x + at(i) + off);
      d[i] = gn_ld_raw<T>(dout + at(i) + off);
    }
  GnCoef<VEC, UG> k;
  k.load(stn, gamma, beta, on ? ct : c0, D);
  float a[VEC], b[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) a[e] = b[e] = 0.f;
  // clipped ReLU: one bit an element says where g = dout, the rest is 0; vectors to be decided again are remembered
  unsigned bits[(NV + 32 / VEC - 1) / (32 / VEC)], again = 0;
#pragma unroll
  for (unsigned& q : bits) q = 0;
  gn_renew(off);
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (in(i)) {
      GnRaw<T> w;
      if (wr) w = gn_ld_raw<T>(res + at(i) + off);
      unsigned on = 0;
      if constexpr (ACT == GN_CAP) {
        bool near;
        on = gn_bits(v[i], w, wr, k, cap, near);
        bits[i / (32 / VEC)] |= on << (i % (32 / VEC) * VEC);
        again |= near ? 1u << i : 0u;
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float gr = d[i].f(e);
        if constexpr (ACT == GN_CAP) gr = (on >> e) & 1u ? gr : 0.f;
        if constexpr (ACT == GN_SILU) gr *= gn_silu_slope(v[i], w, wr, k, e);
        a[e] += gr;
        b[e] += gr * (v[i].f(e) - k.mh[UG ? 0 : e]);
      }
    }
  float* bufa = ldsf;
  float* bufb = bufa + RS * W;
  float* tmp = bufb + RS * W;
  const int nt = blockDim.x > W ? blockDim.x : W;
  float* grp = tmp + 2 * nt;
  if (on)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      bufa[rl * W + col * VEC + e] = a[e];
      bufb[rl * W + col * VEC + e] = gn_centre(b[e], a[e], stn[(UG ? ct : ct + e) / D]);
    }
  if constexpr (ACT == GN_CAP)
    if (again) {  // rare: what fp64 says otherwise is taken from this thread's sums, and its bits are changed
#pragma unroll 1
      for (int i = 0; i < NV; ++i) {
        if (!((again >> i) & 1u)) continue;
        const long long o = at(i) + off;
        const unsigned on = gn_inside<T, VEC>(x + o, wr ? res + o : nullptr, stn, gamma, beta, ct, D, cap);
        unsigned old = 0;
#pragma unroll
        for (int q = 0; q < (int)(sizeof(bits) / 4); ++q)
          if (i / (32 / VEC) == q) {
            old = (bits[q] >> (i % (32 / VEC) * VEC)) & ((1u << VEC) - 1u);
            bits[q] ^= (old ^ on) << (i % (32 / VEC) * VEC);
          }
#pragma unroll 1
        for (int e = 0; e < VEC; ++e) {
          if (!(((old ^ on) >> e) & 1u)) continue;
          const float dy = ((on >> e) & 1u ? 1.f : -1.f) * ElemTraits<T>::to_f32(dout[o + e]);
          const GnStat st = stn[(ct + e) / D];
          bufa[rl * W + col * VEC + e] += dy;
          bufb[rl * W + col * VEC + e] += dy * (float)(((double)ElemTraits<T>::to_f32(x[o + e]) - st.mean) * st.rstd);
        }
      }
    }
  gn_channel_totals(bufa, tmp, W, RS);
  gn_channel_totals(bufb, tmp + nt, W, RS);
  if (part)
    for (int c = threadIdx.x; c < W; c += blockDim.x) part[(long long)n * C + c0 + c] = make_float2(bufa[c], bufb[c]);
  if (!dx) return;
  for (int g = threadIdx.x >> 6; g < Gs; g += blockDim.x >> 6) {
    double ta = 0.0, tb = 0.0;
    for (int j = threadIdx.x & 63; j < D; j += 64) {
      const double ga = gamma ? (double)gamma[c0 + g * D + j] : 1.0;
      ta += ga * (double)bufa[g * D + j];
      tb += ga * (double)bufb[g * D + j];
    }
    ta = wave_sum_f64(ta);
    tb = wave_sum_f64(tb);
    if ((threadIdx.x & 63) == 0) {
      const double m = (double)S * D;
      grp[2 * g] = (float)(ta / m);
      grp[2 * g + 1] = (float)(tb / m);
    }
  }
  __syncthreads();
  if (!on) return;
  float pa[k.NG], pb[k.NG];
#pragma unroll
  for (int i = 0; i < k.NG; ++i) {
    const int g = (col * VEC + i) / D;
    gn_dx_coefs(grp[2 * g], grp[2 * g + 1], stn[c0 / D + g], pa[i], pb[i]);
  }
  gn_renew(off);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    gn_renew(v[i]);
    gn_renew(d[i]);
    if (in(i)) {
      GnRaw<T> w;
      if (ACT == GN_SILU && wr) w = gn_ld_raw<T>(res + at(i) + off);
      float y[VEC], gs[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int j = UG ? 0 : e;
        float gr = d[i].f(e);
        if constexpr (ACT == GN_CAP) gr = (bits[i / (32 / VEC)] >> (i % (32 / VEC) * VEC + e)) & 1u ? gr : 0.f;
        if constexpr (ACT == GN_SILU) gr *= gn_silu_slope(v[i], w, wr, k, e);
        const float t = v[i].f(e) - k.mh[j];
        y[e] = gr * k.sc[e] + (t * pb[j] + pa[j]);
        gs[e] = gr;
      }
      v[i].set(y);
      gn_st_raw<T>(dx + at(i) + off, v[i]);
      if (dres) {
        d[i].set(gs);
        gn_st_raw<T>(dres + at(i) + off, d[i]);
      }
    }
  }
}

// What one call gets; act is a GnAct, T is chosen by the three instantiating files.
struct GnResidentArgs {
  const void *x, *res, *dout;
  void *out, *dx, *dres;
  const float *gamma, *beta;
  long long N, S;
  int C, G, act;
  double eps;
  float cap;
  GnStat* stats;
  float2* part;
  hipStream_t st;
};
template <typename T> int gn_resident_fwd(const GnPlan& p, const GnResidentArgs& a);
template <typename T> int gn_resident_bwd(const GnPlan& p, const GnResidentArgs& a);

#ifdef GN_INSTANTIATE
template <typename K> static int gn_allow_lds(K kernel, size_t lds) {
  if (lds <= 64 * 1024) return 0;
  return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
}

template <typename T, int NV, bool UG, int ACT> static int gn_launch_fwd(const GnPlan& p, const GnResidentArgs& a) {
  constexpr int VEC = 16 / sizeof(T);
  const int D = a.C / a.G, vt = p.W / VEC, dv = D / VEC;
  const int shuffles = UG && vt <= 64 && (vt & (vt - 1)) == 0 && (dv & (dv - 1)) == 0;
  const size_t lds = gn_fwd_lds(p.W, p.threads, VEC, D);
  if (int rc = gn_allow_lds(gn_resident_fwd_kernel<T, NV, UG, ACT>, lds)) return rc;
  hipLaunchKernelGGL((gn_resident_fwd_kernel<T, NV, UG, ACT>), dim3((unsigned)(a.N * (a.C / p.W))), dim3(p.threads), lds, a.st,
                     (const T*)a.x, (const T*)a.res, (T*)a.out, a.gamma, a.beta, (int)a.S, a.C, a.G, p.W, a.eps, a.cap, shuffles,
                     a.stats);
  return pda_check_launch();
}
template <typename T, int NV, bool UG, int ACT> static int gn_launch_bwd(const GnPlan& p, const GnResidentArgs& a) {
  constexpr int VEC = 16 / sizeof(T);
  const size_t lds = gn_bwd_lds(p.W, p.threads, VEC, a.C / a.G);
  if (int rc = gn_allow_lds(gn_resident_bwd_kernel<T, NV, UG, ACT>, lds)) return rc;
  hipLaunchKernelGGL((gn_resident_bwd_kernel<T, NV, UG, ACT>), dim3((unsigned)(a.N * (a.C / p.W))), dim3(p.threads), lds, a.st,
                     (const T*)a.x, (const T*)a.res, (const T*)a.dout, (T*)a.dx, (T*)a.dres, a.gamma, a.beta, a.stats, (int)a.S,
                     a.C, a.G, p.W, a.cap, a.part);
  return pda_check_launch();
}
#define GN_RES_ACT(FN, NV, UG)                                                      \
  switch (a.act) {                                                                  \
    case GN_NONE: return FN<T, NV, UG, GN_NONE>(p, a);                              \
    case GN_CAP: return FN<T, NV, UG, GN_CAP>(p, a);                                \
    default: return FN<T, NV, UG, GN_SILU>(p, a);                                   \
  }
#define GN_RES_UG(FN, NV)                                                           \
  if ((a.C / a.G) % (16 / (int)sizeof(T)) == 0) { GN_RES_ACT(FN, NV, true) }        \
  GN_RES_ACT(FN, NV, false)
template <typename T> int gn_resident_fwd(const GnPlan& p, const GnResidentArgs& a) {
  if (p.nv <= 2) { GN_RES_UG(gn_launch_fwd, 2) }
  if (p.nv <= 4) { GN_RES_UG(gn_launch_fwd, 4) }
  if (p.nv <= 8) { GN_RES_UG(gn_launch_fwd, 8) }
  GN_RES_UG(gn_launch_fwd, GN_NV_FWD)
}
template <typename T> int gn_resident_bwd(const GnPlan& p, const GnResidentArgs& a) {
  if (p.nv <= 2) { GN_RES_UG(gn_launch_bwd, 2) }
  if (p.nv <= 4) { GN_RES_UG(gn_launch_bwd, 4) }
  GN_RES_UG(gn_launch_bwd, GN_NV_BWD)
}
#endif
