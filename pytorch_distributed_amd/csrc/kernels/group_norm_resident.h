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
  int fold = 1;        // positions that make up a row
};

// Resident vectors of one thread: what stays below the 128 registers that 1024 threads leave each.  Backward, up to
// GN_NV_BOTH vectors of x and dout stay; above that x alone does, and dout is read again (it has just passed through the
// caches).
constexpr int GN_NV_FWD = 13, GN_NV_BWD = 13, GN_NV_BOTH = 7;

// Shared memory of a workgroup: the larger of what the ways of gn_group_totals use; gn_channel_totals with its input.
inline size_t gn_fwd_lds(int W, int threads, int vec, int D) {
  const size_t waves = 16ull * (threads / 64) * (W / D);  // a pair for each wave and group
  const size_t all = D % vec == 0 ? 16ull * (threads + W / D)
                                  : 8ull * ((size_t)(threads / (W / vec)) * W + (threads > W ? threads : W) + W / D);
  return waves > all ? waves : all;
}
inline size_t gn_bwd_lds(int W, int threads, int vec, int D) {
  return 8ull * ((size_t)(threads / (W / vec)) * W + (threads > W ? threads : W) + W / D);
}

// Measured on 400 samples, fp16, forward / backward: the width of a slab's rows counts most (56x56x256 with residual:
// 16 bytes 701 / 1381 us, 32 bytes 530 / 941, 64 bytes 441 / 736 next to each other; on its own 472 / 781 = 4.1 TB/s), up to 128 bytes (14x14x1024: 32 bytes 114 / 202, 64 bytes
// 101 / 183, 128 bytes 108 / 194), then few threads with many vectors (28x28x512: 512 threads 197, 1024 230 us).
inline GnPlan gn_resident_plan(int esize, long long N, long long S, int C, int G, bool bwd) {
  GnPlan best{0, 0, 0};
  const int vec = 16 / esize, D = C / G;
  if (C > (1 << 20)) return best;  // offsets in a workgroup are 32 bits
  // channels that fill no whole vectors: as many positions a row as make them whole, and a slab is the whole row
  int fold = 1;
  while (C * fold % vec) fold *= 2;
  if (S % fold || (fold > 1 && C > 4096)) return best;
  S /= fold;
  if (S > 1024 * GN_NV_FWD) return best;
  int a = D, b = vec;
  while (b) { const int t = a % b; a = b; b = t; }
  const int unit = fold > 1 ? C * fold : D / a * vec;  // whole groups and whole vectors
  const int units = C * fold / unit;
  double top = 0.0;
  for (int k = 1; k <= units; ++k) {
    if (units % k) continue;
    const int W = unit * k, vt = W / vec, row = W * esize;
    if (vt > 1024 || (row < 32 && W != C * fold)) continue;
    const long long blocks = N * (units / k);
    // both tensors in registers where 512 threads do (two workgroups on a CU), else x alone
    int threads = 0, most = bwd ? GN_NV_BOTH : GN_NV_FWD;
    for (int pass = 0; pass < 2 && !threads; ++pass) {
      for (int nt = 64; nt <= (bwd && pass == 0 ? 512 : 1024) && !threads; nt *= 2)
        if (nt >= vt && (S + nt / vt - 1) / (nt / vt) <= most) threads = nt;
      most = bwd ? GN_NV_BWD : GN_NV_FWD;
    }
    if (!threads) continue;
    if ((bwd ? gn_bwd_lds(W, 1024, vec, D) : gn_fwd_lds(W, 1024, vec, D)) > 156 * 1024) continue;
    // few blocks: more threads each, while their vectors stay two or more
    while (threads < 1024 && blocks * threads < 256 * 512 && (S + threads / vt - 1) / (threads / vt) > 3) threads *= 2;
    const int nv = (int)((S + threads / vt - 1) / (threads / vt));
    const double fill = (double)blocks * threads / (256.0 * 512.0), used = (double)(S * vt) / ((double)threads * nv);
    double score = (row < 64 ? 0.75 : row < 128 ? 0.92 : row <= 256 ? 1.0 : 0.97) * (fill < 1.0 ? fill : 1.0);
    score *= used;                                                          // rows that do not fill the block
    if (S * vt < 256 && blocks > 1024) score *= sqrt((double)(S * vt) / 256.0);  // a workgroup costs, too
    if (threads > 512) score *= D % vec ? 0.75 : 0.92;  // (several groups a vector: more registers, spills at 13 vectors)
    if (bwd && nv > GN_NV_BOTH) score *= 0.9;
    if (score > top) {
      top = score;
      best = GnPlan{W, threads, nv, fold};
    }
  }
  return best;
}

// Totals of every channel of the slab: buf [RS][W] (written, not yet synchronised) -> buf[0..W).  tmp: max(threads, W).
template <typename V> __device__ __forceinline__ void gn_channel_totals(V* buf, V* tmp, int W, int RS) {
  // (V: a number or a pair of them)
  const int NT = blockDim.x, parts = NT < W ? 1 : NT / W < RS ? NT / W : RS;
  __syncthreads();
  for (int i = threadIdx.x; i < W * parts; i += NT) {
    const int c = i % W, p = i / W;
    V a = buf[p * W + c];  // p < RS: a part has a row at least
    for (int r = p + parts; r < RS; r += parts) a += buf[r * W + c];
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

// Sums over every group of the slab: s[e] of every thread that is on -> s[e] of the group of slot e (UG: one slot).
template <int VEC, bool UG>
__device__ __forceinline__ void gn_group_totals(GnPair (&s)[UG ? 1 : VEC], double* lds, int W, int D, int C, int fold, int RS,
                                                int col, int rl, bool on, bool shuffles) {
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
  } else if (shuffles) {  // a vector holds whole groups (D divides it), columns are a power of two
    GnPair* buf = reinterpret_cast<GnPair*>(lds);
    const int per = VEC / D, c0 = col * per;
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (!on) s[e] = GnPair{0.0, 0.0};
    if (D > 1)  // into a group's first slot
#pragma unroll
      for (int e = 0; e + 1 < VEC; e += 2) s[e] = GnPair{s[e].a + s[e + 1].a, s[e].b + s[e + 1].b};
    if (D > 2)
#pragma unroll
      for (int e = 0; e + 2 < VEC; e += 4) s[e] = GnPair{s[e].a + s[e + 2].a, s[e].b + s[e + 2].b};
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (e % D == 0) {
        for (int o = VT; o < 64; o <<= 1) {
          s[e].a += __shfl_xor(s[e].a, o, 64);
          s[e].b += __shfl_xor(s[e].b, o, 64);
        }
        if (lane < VT) buf[wave * Gs + c0 + e / D] = s[e];
      }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      s[e] = buf[c0 + e / D];
      for (int w = 1; w < NW; ++w) {
        s[e].a += buf[w * Gs + c0 + e / D].a;
        s[e].b += buf[w * Gs + c0 + e / D].b;
      }
    }
  } else {
    double* tmp = lds + RS * W;
    double* grp = tmp + (blockDim.x > W ? blockDim.x : W);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (on)
#pragma unroll
        for (int e = 0; e < VEC; ++e) lds[rl * W + col * VEC + e] = h ? s[e].b : s[e].a;
      gn_channel_totals(lds, tmp, W, RS);
      for (int g = wave; g < Gs / fold; g += NW) {
        double t = 0.0;
        for (int d = lane; d < D; d += 64)
          for (int f = 0; f < fold; ++f) t += lds[f * C + g * D + d];
        t = wave_sum_f64(t);
        if (lane == 0) grp[g] = t;
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < VEC; ++e) (h ? s[e].b : s[e].a) = grp[(fold > 1 ? gn_channel(col * VEC + e, C) : col * VEC + e) / D];
    }
  }
}

template <typename T, int NV, bool UG, int ACT>
__global__ void __launch_bounds__(1024)
gn_resident_fwd_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ out, const float* __restrict__ gamma,
                       const float* __restrict__ beta, int S, int C, int G, int W, int fold, double eps, float cap, int shuffles,
                       GnStat* __restrict__ stats) {
  extern __shared__ double lds[];
  constexpr int VEC = 16 / sizeof(T), NG = UG ? 1 : VEC;
  const int row = C * fold, slabs = row / W, D = C / G, VT = W / VEC, RS = blockDim.x / VT;
  const int id = xcd_remap(blockIdx.x, gridDim.x), n = id / slabs, c0 = (id % slabs) * W;
  const int col = threadIdx.x % VT, rl = threadIdx.x / VT;
  const bool on = rl < RS;
  // addresses: one for the workgroup, one offset a thread, one step a vector
  const long long slab = (long long)n * S * row + c0;
  unsigned off = (unsigned)(rl * row + col * VEC);
  const auto at = [&](int i) { return slab + (long long)i * RS * row; };
  float one = 1.f;
  asm volatile("" : "+s"(one));
  GnRaw<T> v[NV];
  const auto in = [&](int i) { return on && rl + i * RS < S; };
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (in(i)) v[i] = gn_ld_raw<T>(x + at(i) + off);
  // Sums in fp64: a spread far below the mean is kept, and the side of an activation's border on which an element lies can be
  // decided by what comes out (a sum of squares in fp32, joined in fp64, put one element of 300 million on the wrong one).
  double first[NG];
  GnPair tot[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    first[i] = gn_first(x + (long long)n * S * row, gn_channel(c0 + col * VEC + i, C), D);
    tot[i] = GnPair{0.0, 0.0};
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (in(i))
#pragma unroll
      for (int e = 0; e < VEC; ++e) gn_add<T>(tot[UG ? 0 : e], v[i].f(e), first[UG ? 0 : e]);
  gn_group_totals<VEC, UG>(tot, lds, W, D, C, fold, RS, col, rl, on, shuffles);
  const double m = (double)S * fold * D, im = 1.0 / m;
  if (!on) return;
  float mh[NG], sc[VEC], sh[VEC];
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const GnStat st = gn_stat(tot[i], first[i], m, im, eps);
    const double r = st.rstd;
    mh[i] = (float)st.mean;
    const double ml = st.mean - (double)mh[i];
    if (rl == 0) {
      const int c = c0 + col * VEC + i;  // the thread of a group's first channel writes its statistics
      if (c < C && c % D == 0) stats[(long long)n * G + c / D] = st;
    }
#pragma unroll
    for (int e = UG ? 0 : i; e < (UG ? VEC : i + 1); ++e) {
      const int c = gn_channel(c0 + col * VEC + e, C);
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
        float z = v[i].sub(e, mh[UG ? 0 : e], one) * sc[e] + sh[e];
        if (res) z = w.add(e, z, one);
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
                       const GnStat* __restrict__ stats, int S, int C, int G, int W, int fold, float cap, float2* __restrict__ part) {
  extern __shared__ float2 lds2[];
  constexpr int VEC = 16 / sizeof(T);
  constexpr bool BOTH = NV <= GN_NV_BOTH;  // x and dout stay; otherwise x and (ReLUs) one bit an element of act'(z)
  const int row = C * fold, slabs = row / W, D = C / G, VT = W / VEC, RS = blockDim.x / VT, Gs = W / fold / D;
  const int id = xcd_remap(blockIdx.x, gridDim.x), n = id / slabs, c0 = (id % slabs) * W;
  const int col = threadIdx.x % VT, rl = threadIdx.x / VT, ct = c0 + col * VEC;
  const bool on = rl < RS;
  const long long slab = (long long)n * S * row + c0;
  unsigned off = (unsigned)(rl * row + col * VEC);
  const auto at = [&](int i) { return slab + (long long)i * RS * row; };
  const auto in = [&](int i) { return on && rl + i * RS < S; };
  const bool wr = ACT != GN_NONE && res;
  const GnStat* stn = stats + (long long)n * G;
  float one = 1.f;
  asm volatile("" : "+s"(one));
  GnRaw<T> v[NV], d[BOTH ? NV : 1];
  unsigned bits[BOTH ? 1 : (NV * VEC + 31) / 32];
#pragma unroll
  for (unsigned& q : bits) q = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (in(i)) {
      v[i] = gn_ld_raw<T>(x + at(i) + off);
      if constexpr (BOTH) d[i] = gn_ld_raw<T>(dout + at(i) + off);
    }
  GnCoef<VEC, UG> k;
  k.load(stn, gamma, beta, on ? ct : c0, D, C);
  float a[VEC], b[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) a[e] = b[e] = 0.f;
  // ReLUs: dout becomes g here (0 or as it was); vectors to be decided again are remembered
  const float shmax = gn_is_relu(ACT) ? k.shmax() : 0.f;
  unsigned again = 0;
  gn_renew(off);
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (in(i)) {
      GnRaw<T> w;
      GnRaw<T>& dy = d[BOTH ? i : 0];
      if (wr) w = gn_ld_raw<T>(res + at(i) + off);
      if constexpr (!BOTH) dy = gn_ld_raw<T>(dout + at(i) + off);
      float t[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) t[e] = v[i].sub(e, k.mh[UG ? 0 : e], one);
      if constexpr (gn_is_relu(ACT)) {
        GnNear near;
        bool on[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          float z = t[e] * k.sc[e] + k.sh[e];
          if (wr) {
            z = w.add(e, z, one);
            near.res = fmaxf(near.res, fabsf(w.f(e)));
          }
          on[e] = near.inside<ACT>(z, cap);
        }
        dy.keep(on);
        if constexpr (!BOTH)
#pragma unroll
          for (int e = 0; e < VEC; ++e) bits[(i * VEC + e) / 32] |= on[e] ? 1u << ((i * VEC + e) % 32) : 0u;
        again |= near.again<ACT>(shmax, cap) ? 1u << i : 0u;
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if constexpr (ACT == GN_SILU) {
          const float gr = dy.f(e) * gn_silu_slope(t[e], w, wr, k, e);
          a[e] += gr;
          b[e] += gr * t[e];
        } else {
          a[e] = dy.add(e, a[e], one);
          b[e] = __builtin_fmaf(dy.f(e), t[e], b[e]);
        }
      }
    }
  float2* buf = lds2;
  float2* tmp = buf + RS * W;
  float2* grp = tmp + (blockDim.x > W ? blockDim.x : W);
  if (on)
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      buf[rl * W + col * VEC + e] = make_float2(a[e], gn_centre(b[e], a[e], stn[(UG ? ct : gn_channel(ct + e, C)) / D]));
  if constexpr (gn_is_relu(ACT))
    if (again) {  // rare: what fp64 says otherwise is put right in this thread's sums, in g and in the bits
#pragma unroll 1
      for (int i = 0; i < NV; ++i) {
        if (!((again >> i) & 1u)) continue;
        const long long o = at(i) + off;
        const unsigned on = gn_inside<T, VEC>(x + o, wr ? res + o : nullptr, stn, gamma, beta, ct, D, C, cap);
        unsigned was = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (j == i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              if constexpr (BOTH) {
                was |= d[j].f(e) != 0.f ? 1u << e : 0u;
              } else {
                const unsigned bit = 1u << ((j * VEC + e) % 32);
                unsigned& q = bits[(j * VEC + e) / 32];
                was |= q & bit ? 1u << e : 0u;
                q = (on >> e) & 1u ? q | bit : q & ~bit;
              }
            }
#pragma unroll 1
        for (int e = 0; e < VEC; ++e) {
          const float dy = ElemTraits<T>::to_f32(dout[o + e]);
          if (!(((on ^ was) >> e) & 1u) || dy == 0.f) continue;
          const float more = (on >> e) & 1u ? dy : -dy;
          const GnStat st = stn[gn_channel(ct + e, C) / D];
          buf[rl * W + col * VEC + e] += make_float2(more, more * (float)(((double)ElemTraits<T>::to_f32(x[o + e]) - st.mean) * st.rstd));
        }
        if constexpr (BOTH) {
          GnRaw<T> now = gn_ld_raw<T>(dout + o);
          bool keep[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) keep[e] = (on >> e) & 1u;
          now.keep(keep);
#pragma unroll
          for (int j = 0; j < NV; ++j)
            if (j == i) d[j] = now;
        }
      }
    }
  gn_channel_totals(buf, tmp, W, RS);
  if (fold > 1) {
    for (int c = threadIdx.x; c < C; c += blockDim.x)
      for (int f = 1; f < fold; ++f) buf[c] += buf[f * C + c];
    __syncthreads();
  }
  if (part)
    for (int c = threadIdx.x; c < W / fold; c += blockDim.x) part[(long long)n * C + c0 + c] = buf[c];
  if (!dx) return;
  for (int g = threadIdx.x >> 6; g < Gs; g += blockDim.x >> 6) {
    double ta = 0.0, tb = 0.0;
    for (int j = threadIdx.x & 63; j < D; j += 64) {
      const double ga = gamma ? (double)gamma[c0 + g * D + j] : 1.0;
      const float2 t = buf[g * D + j];
      ta += ga * (double)t.x;
      tb += ga * (double)t.y;
    }
    ta = wave_sum_f64(ta);
    tb = wave_sum_f64(tb);
    if ((threadIdx.x & 63) == 0) {
      const double m = (double)S * fold * D;
      grp[g] = make_float2((float)(ta / m), (float)(tb / m));
    }
  }
  __syncthreads();
  if (!on) return;
  float pa[k.NG], pb[k.NG];
#pragma unroll
  for (int i = 0; i < k.NG; ++i) {
    const int g = (fold > 1 ? gn_channel(col * VEC + i, C) : col * VEC + i) / D;
    gn_dx_coefs(grp[g].x, grp[g].y, stn[c0 / D + g], pa[i], pb[i]);
  }
  gn_renew(off);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    gn_renew(v[i]);
    if constexpr (BOTH) gn_renew(d[i]);
    if (in(i)) {
      GnRaw<T> w;
      GnRaw<T>& dy = d[BOTH ? i : 0];
      if constexpr (!BOTH) {
        dy = gn_ld_raw<T>(dout + at(i) + off);
        if constexpr (gn_is_relu(ACT)) {
          bool on[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) on[e] = (bits[(i * VEC + e) / 32] >> ((i * VEC + e) % 32)) & 1u;
          dy.keep(on);
        }
      }
      if (ACT == GN_SILU && wr) w = gn_ld_raw<T>(res + at(i) + off);
      float y[VEC], gs[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int j = UG ? 0 : e;
        const float t = v[i].sub(e, k.mh[j], one);
        gs[e] = ACT == GN_SILU ? dy.f(e) * gn_silu_slope(t, w, wr, k, e) : 0.f;
        const float rest = t * pb[j] + pa[j];
        y[e] = ACT == GN_SILU ? gs[e] * k.sc[e] + rest : __builtin_fmaf(dy.f(e), k.sc[e], rest);
      }
      v[i].set(y);
      gn_st_raw<T>(dx + at(i) + off, v[i]);
      if (dres) {
        if constexpr (ACT == GN_SILU) dy.set(gs);
        gn_st_raw<T>(dres + at(i) + off, dy);
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
  const int shuffles = p.fold == 1 && vt <= 64 && (vt & (vt - 1)) == 0 && (UG ? (dv & (dv - 1)) == 0 : VEC % D == 0);
  const size_t lds = gn_fwd_lds(p.W, p.threads, VEC, D);
  if (int rc = gn_allow_lds(gn_resident_fwd_kernel<T, NV, UG, ACT>, lds)) return rc;
  hipLaunchKernelGGL((gn_resident_fwd_kernel<T, NV, UG, ACT>), dim3((unsigned)(a.N * (a.C * p.fold / p.W))), dim3(p.threads), lds,
                     a.st, (const T*)a.x, (const T*)a.res, (T*)a.out, a.gamma, a.beta, (int)(a.S / p.fold), a.C, a.G, p.W, p.fold, a.eps, a.cap, shuffles,
                     a.stats);
  return pda_check_launch();
}
template <typename T, int NV, bool UG, int ACT> static int gn_launch_bwd(const GnPlan& p, const GnResidentArgs& a) {
  constexpr int VEC = 16 / sizeof(T);
  const size_t lds = gn_bwd_lds(p.W, p.threads, VEC, a.C / a.G);
  if (int rc = gn_allow_lds(gn_resident_bwd_kernel<T, NV, UG, ACT>, lds)) return rc;
  hipLaunchKernelGGL((gn_resident_bwd_kernel<T, NV, UG, ACT>), dim3((unsigned)(a.N * (a.C * p.fold / p.W))), dim3(p.threads), lds,
                     a.st, (const T*)a.x, (const T*)a.res, (const T*)a.dout, (T*)a.dx, (T*)a.dres, a.gamma, a.beta, a.stats,
                     (int)(a.S / p.fold), a.C, a.G, p.W, p.fold, a.cap, a.part);
  return pda_check_launch();
}
#define GN_RES_ACT(FN, NV, UG)                                                      \
  switch (a.act) {                                                                  \
    case GN_NONE: return FN<T, NV, UG, GN_NONE>(p, a);                              \
    case GN_RELU: return FN<T, NV, UG, GN_RELU>(p, a);                              \
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
  if (p.nv <= GN_NV_BOTH) { GN_RES_UG(gn_launch_bwd, GN_NV_BOTH) }
  GN_RES_UG(gn_launch_bwd, GN_NV_BWD)
}
#endif
