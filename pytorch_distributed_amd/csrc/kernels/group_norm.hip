// Group norm with an optional residual and activation, channels last: x [N][S][C], C = G groups of D channels.  The formulas
// are those of group_norm.h.
//
// Statistics are fp64 sums (gn_stat) and are kept in fp64: a value next to an activation's border is placed by them.  The element
// passes take mu as an fp32 pair (hi subtracted from x, lo folded into the shift).
//
// Memory-bound throughout: the work is split over (sample, row chunk), a thread owns one vector of channels and walks
// rows, so the per-channel coefficients stay in registers; 2048 blocks of two or four rows in flight a thread measured
// best.  The element passes take the blocks from the last to the first: what the sums read last is still in the memory-side
// cache.  128x112x112x64 bf16 with SiLU: sums 47 us = 4.4 TB/s, apply 77 us = 5.3, backward sums 97 us = 4.2 (113 with the
// blocks in order), backward apply 114 us = 5.4 (121).  No atomics: results repeat bit for bit.
#include "group_norm_resident.h"

#include <initializer_list>
#include <math.h>

namespace {

// Where a block's threads stand: VT vectors of channels side by side, RS rows at a time (threads beyond VT*RS idle).
struct GnGeom {
  int VT, RS, col, rl;
  __device__ explicit GnGeom(int vpr) {
    VT = vpr < 256 ? vpr : 256;
    RS = 256 / VT;
    col = threadIdx.x % VT;
    rl = threadIdx.x / VT;
  }
};

// Per-channel sums of one row chunk -> part[n][chunk][c].
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
gn_partial_kernel(const T* __restrict__ x, long long S, int C, int G, int chunks, GnPair* __restrict__ part) {
  __shared__ GnPair sm[256 * VEC];
  const int n = blockIdx.x / chunks, ch = blockIdx.x % chunks;
  const long long r0 = S * ch / chunks, r1 = S * (ch + 1) / chunks;
  const int vpr = C / VEC, D = C / G;
  const GnGeom g(vpr);
  const T* xn = x + (long long)n * S * C;
  for (int c0 = 0; c0 < vpr; c0 += g.VT) {
    const int vec = c0 + g.col;
    const bool active = g.rl < g.RS && vec < vpr;
    GnPair s[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[e] = GnPair{0.0, 0.0};
    if (active) {
      const T* p = xn + (long long)vec * VEC;
      double first[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) first[e] = gn_first(xn, vec * VEC + e, D);
      const auto add = [&](const GnHeld<T, VEC>& v) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) gn_add<T>(s[e], v.f(e), first[e]);
      };
      long long r = r0 + g.rl;
      for (; r + 3 * g.RS < r1; r += 4 * g.RS) {
        GnHeld<T, VEC> v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = gn_ld_held<T, VEC>(p + (r + u * g.RS) * C);
#pragma unroll
        for (int u = 0; u < 4; ++u) add(v[u]);
      }
      for (; r < r1; r += g.RS) add(gn_ld_held<T, VEC>(p + r * C));
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) sm[e * 256 + threadIdx.x] = s[e];
    __syncthreads();
    int h = 1;
    while (h < g.RS) h <<= 1;
    for (h >>= 1; h > 0; h >>= 1) {
      if (g.rl < h && g.rl + h < g.RS) {
        const int o = threadIdx.x + h * g.VT;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          s[e].a += sm[e * 256 + o].a;
          s[e].b += sm[e * 256 + o].b;
          sm[e * 256 + threadIdx.x] = s[e];
        }
      }
      __syncthreads();
    }
    if (active && g.rl == 0) {
      GnPair* o = part + (long long)blockIdx.x * C + (long long)vec * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = s[e];
    }
  }
}

// One wave per (sample, group): chunks x D sums -> {mu, r} in fp64.  5 us for 32 groups a sample; one wide group is a long walk (one
// group of 128x14x14x1024 fp16 68 us, of 1x56x56x256 64, and as much again backward), more than the passes beside it.
template <typename T>
__global__ void __launch_bounds__(64)
gn_finalize_kernel(const T* __restrict__ x, const GnPair* __restrict__ part, long long S, int C, int G, int chunks, double eps,
                   GnStat* __restrict__ stats) {
  const int D = C / G;
  const int n = blockIdx.x / G, g = blockIdx.x % G;
  const GnPair* p = part + (long long)n * chunks * C + (long long)g * D;
  const long long pairs = (long long)chunks * D;
  double a = 0.0, b = 0.0;
  for (long long j = threadIdx.x; j < pairs; j += 64) {
    const GnPair v = p[(j / D) * C + j % D];
    a += v.a;
    b += v.b;
  }
  const double m = (double)S * D;
  const GnPair s{wave_sum_f64(a), wave_sum_f64(b)};
  if (threadIdx.x == 0) stats[blockIdx.x] = gn_stat(s, gn_first(x + (long long)n * S * C, g * D, D), m, 1.0 / m, eps);
}

template <typename T, int VEC, bool UG, int ACT>
__global__ void __launch_bounds__(256)
gn_apply_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ out, const float* __restrict__ gamma,
                const float* __restrict__ beta, const GnStat* __restrict__ stats, long long S, int C, int G, int chunks,
                float cap) {
  constexpr int U = 2;  // rows in flight
  const int blk = gridDim.x - 1 - blockIdx.x;
  const int n = blk / chunks, ch = blk % chunks;
  const long long r0 = S * ch / chunks, r1 = S * (ch + 1) / chunks;
  const int vpr = C / VEC, D = C / G;
  const GnGeom g(vpr);
  if (g.rl >= g.RS) return;
  for (int vec = g.col; vec < vpr; vec += g.VT) {
    GnCoef<VEC, UG> k;
    k.load(stats + (long long)n * G, gamma, beta, vec * VEC, D, C);
    const long long base = (long long)n * S * C + (long long)vec * VEC;
    const auto row = [&](const GnHeld<T, VEC>& v, const GnHeld<T, VEC>& w, long long o) {
      GnVec<T, VEC> y;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float z = (v.f(e) - k.mh[UG ? 0 : e]) * k.sc[e] + k.sh[e];
        if (res) z += w.f(e);
        y.v[e] = ElemTraits<T>::from_f32(gn_act<ACT>(z, cap));
      }
      gn_st<T, VEC>(out + o, y);
    };
    long long r = r0 + g.rl;
    for (; r + (U - 1) * g.RS < r1; r += U * g.RS) {
      GnHeld<T, VEC> v[U], w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        v[u] = gn_ld_held<T, VEC>(x + base + (r + u * g.RS) * C);
        if (res) w[u] = gn_ld_held<T, VEC>(res + base + (r + u * g.RS) * C);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) row(v[u], w[u], base + (r + u * g.RS) * C);
    }
    for (; r < r1; r += g.RS) {
      GnHeld<T, VEC> v = gn_ld_held<T, VEC>(x + base + r * C), w;
      if (res) w = gn_ld_held<T, VEC>(res + base + r * C);
      row(v, w, base + r * C);
    }
  }
}

// Per-channel {sum g, sum g xh} of one row chunk of one sample -> part[n][chunk][c].  fp32 over a thread's rows and the block's
// tree; what joins chunks, channels and samples is fp64.
template <typename T, int VEC, bool UG, int ACT>
__global__ void __launch_bounds__(256)
gn_bwd_partial_kernel(const T* __restrict__ x, const T* __restrict__ res, const T* __restrict__ dout,
                      const float* __restrict__ gamma, const float* __restrict__ beta, const GnStat* __restrict__ stats,
                      long long S, int C, int G, int chunks, float cap, float2* __restrict__ part) {
  constexpr int U = 2;
  __shared__ float sa[256 * VEC], sb[256 * VEC];
  const int n = blockIdx.x / chunks, ch = blockIdx.x % chunks;
  const long long r0 = S * ch / chunks, r1 = S * (ch + 1) / chunks;
  const int vpr = C / VEC, D = C / G;
  const GnGeom g(vpr);
  for (int c0 = 0; c0 < vpr; c0 += g.VT) {
    const int vec = c0 + g.col;
    const bool active = g.rl < g.RS && vec < vpr;
    float a[VEC], b[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) a[e] = b[e] = 0.f;
    if (active) {
      GnCoef<VEC, UG> k;
      const GnStat* stn = stats + (long long)n * G;
      k.load(stn, gamma, beta, vec * VEC, D, C);
      const long long base = (long long)n * S * C + (long long)vec * VEC;
      const bool wr = ACT != GN_NONE && res;
      const auto row = [&](const GnHeld<T, VEC>& v, const GnHeld<T, VEC>& d, const GnHeld<T, VEC>& w, long long o) {
        float gr[VEC];
        gn_grads<ACT>(gr, d, v, w, wr, k, x + o, res + o, stn, gamma, beta, vec * VEC, D, C, cap);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          a[e] += gr[e];
          b[e] += gr[e] * (v.f(e) - k.mh[UG ? 0 : e]);
        }
      };
      long long r = r0 + g.rl;
      for (; r + (U - 1) * g.RS < r1; r += U * g.RS) {
        GnHeld<T, VEC> v[U], d[U], w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const long long o = base + (r + u * g.RS) * C;
          v[u] = gn_ld_held<T, VEC>(x + o);
          d[u] = gn_ld_held<T, VEC>(dout + o);
          if (wr) w[u] = gn_ld_held<T, VEC>(res + o);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) row(v[u], d[u], w[u], base + (r + u * g.RS) * C);
      }
      for (; r < r1; r += g.RS) {
        const long long o = base + r * C;
        const GnHeld<T, VEC> v = gn_ld_held<T, VEC>(x + o), d = gn_ld_held<T, VEC>(dout + o);
        GnHeld<T, VEC> w;
        if (wr) w = gn_ld_held<T, VEC>(res + o);
        row(v, d, w, o);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) b[e] = gn_centre(b[e], a[e], stn[(vec * VEC + (UG ? 0 : e)) / D]);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sa[e * 256 + threadIdx.x] = a[e];
      sb[e * 256 + threadIdx.x] = b[e];
    }
    __syncthreads();
    int h = 1;
    while (h < g.RS) h <<= 1;
    for (h >>= 1; h > 0; h >>= 1) {
      if (g.rl < h && g.rl + h < g.RS) {
        const int o = threadIdx.x + h * g.VT;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          sa[e * 256 + threadIdx.x] = a[e] += sa[e * 256 + o];
          sb[e * 256 + threadIdx.x] = b[e] += sb[e * 256 + o];
        }
      }
      __syncthreads();
    }
    if (active && g.rl == 0) {
      float2* o = part + (long long)blockIdx.x * C + (long long)vec * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = make_float2(a[e], b[e]);
    }
  }
}

// One wave per (sample, group): {A/m, B/m}.
__global__ void __launch_bounds__(64)
gn_bwd_finalize_kernel(const float2* __restrict__ part, const float* __restrict__ gamma, long long S, int C, int G,
                       int chunks, float2* __restrict__ ab) {
  const int D = C / G;
  const int n = blockIdx.x / G, g = blockIdx.x % G;
  const float2* p = part + (long long)n * chunks * C + (long long)g * D;
  double a = 0.0, b = 0.0;
  const long long pairs = (long long)chunks * D;
  for (long long j = threadIdx.x; j < pairs; j += 64) {
    const int d = (int)(j % D);
    const float2 v = p[(j / D) * C + d];
    const double ga = gamma ? (double)gamma[g * D + d] : 1.0;
    a += ga * (double)v.x;
    b += ga * (double)v.y;
  }
  a = wave_sum_f64(a);
  b = wave_sum_f64(b);
  const double m = (double)S * D;
  if (threadIdx.x == 0) ab[blockIdx.x] = make_float2((float)(a / m), (float)(b / m));
}

// dgamma_c, dbeta_c: the column sums of part [rows][C].  A block takes 4 channels with 256 lanes of rows each: with one
// block a channel group the walk over the rows (thousands at large batch) has to be short.  Many rows are summed in two
// steps: blockIdx.y takes `span` rows and leaves their sums in the first of them (rounded to fp32 there, 2^-24 of each), which no
// other block reads; the second step (dbeta given) takes those, `step` rows apart.
__global__ void __launch_bounds__(1024)
gn_params_kernel(float2* part, long long rows, long long span, long long step, int C, float* __restrict__ dgamma,
                 float* __restrict__ dbeta) {
  __shared__ double ra[16][4], rb[16][4];
  const int cl = threadIdx.x & 3, lane = threadIdx.x >> 2;
  const int c = blockIdx.x * 4 + cl;
  const long long r0 = blockIdx.y * span, r1 = r0 + span < rows ? r0 + span : rows, row = step * C;
  double a = 0.0, b = 0.0;
  if (c < C) {
    long long r = r0 + lane;
    for (; r + 768 < r1; r += 1024) {
      float2 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = part[(r + u * 256) * row + c];
#pragma unroll
      for (int u = 0; u < 4; ++u) { a += (double)v[u].x; b += (double)v[u].y; }
    }
    for (; r < r1; r += 256) {
      const float2 v = part[r * row + c];
      a += (double)v.x;
      b += (double)v.y;
    }
  }
#pragma unroll
  for (int o = 4; o < 64; o <<= 1) {
    a += __shfl_xor(a, o, 64);
    b += __shfl_xor(b, o, 64);
  }
  const int wv = threadIdx.x >> 6;
  if ((threadIdx.x & 63) < 4) { ra[wv][cl] = a; rb[wv][cl] = b; }
  __syncthreads();
  if (threadIdx.x < 4 && c < C) {
#pragma unroll
    for (int w = 1; w < 16; ++w) { a += ra[w][cl]; b += rb[w][cl]; }
    if (dbeta) {
      dbeta[c] = (float)a;
      dgamma[c] = (float)b;
    } else {
      part[r0 * row + c] = make_float2((float)a, (float)b);
    }
  }
}

template <typename T, int VEC, bool UG, int ACT>
__global__ void __launch_bounds__(256)
gn_bwd_apply_kernel(const T* __restrict__ x, const T* __restrict__ res, const T* __restrict__ dout, T* __restrict__ dx,
                    T* __restrict__ dres, const float* __restrict__ gamma, const float* __restrict__ beta,
                    const GnStat* __restrict__ stats, const float2* __restrict__ ab, long long S, int C, int G, int chunks,
                    float cap) {
  constexpr int U = 2;
  const int blk = gridDim.x - 1 - blockIdx.x;
  const int n = blk / chunks, ch = blk % chunks;
  const long long r0 = S * ch / chunks, r1 = S * (ch + 1) / chunks;
  const int vpr = C / VEC, D = C / G;
  const GnGeom g(vpr);
  if (g.rl >= g.RS) return;
  for (int vec = g.col; vec < vpr; vec += g.VT) {
    GnCoef<VEC, UG> k;
    const GnStat* stn = stats + (long long)n * G;
    k.load(stn, gamma, beta, vec * VEC, D, C);
    float pa[k.NG], pb[k.NG];
#pragma unroll
    for (int i = 0; i < k.NG; ++i) {
      const int gi = (vec * VEC + i) / D;
      const float2 v = ab[(long long)n * G + gi];
      gn_dx_coefs(v.x, v.y, stn[gi], pa[i], pb[i]);
    }
    const long long base = (long long)n * S * C + (long long)vec * VEC;
    const bool wr = ACT != GN_NONE && res;
    const auto row = [&](const GnHeld<T, VEC>& v, const GnHeld<T, VEC>& d, const GnHeld<T, VEC>& w, long long o) {
      GnVec<T, VEC> yx, yr;
      float gr[VEC];
      gn_grads<ACT>(gr, d, v, w, wr, k, x + o, res + o, stn, gamma, beta, vec * VEC, D, C, cap);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int i = UG ? 0 : e;
        const float t = v.f(e) - k.mh[i];
        yx.v[e] = ElemTraits<T>::from_f32(gr[e] * k.sc[e] + (t * pb[i] + pa[i]));
        yr.v[e] = ElemTraits<T>::from_f32(gr[e]);
      }
      gn_st<T, VEC>(dx + o, yx);
      if (dres) gn_st<T, VEC>(dres + o, yr);
    };
    long long r = r0 + g.rl;
    for (; r + (U - 1) * g.RS < r1; r += U * g.RS) {
      GnHeld<T, VEC> v[U], d[U], w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long o = base + (r + u * g.RS) * C;
        v[u] = gn_ld_held<T, VEC>(x + o);
        d[u] = gn_ld_held<T, VEC>(dout + o);
        if (wr) w[u] = gn_ld_held<T, VEC>(res + o);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        row(v[u], d[u], w[u], base + (r + u * g.RS) * C);
      }
    }
    for (; r < r1; r += g.RS) {
      const long long o = base + r * C;
      GnHeld<T, VEC> v = gn_ld_held<T, VEC>(x + o), d = gn_ld_held<T, VEC>(dout + o), w;
      if (wr) w = gn_ld_held<T, VEC>(res + o);
      row(v, d, w, o);
    }
  }
}

// Widest vector (elements) that divides the channels and that every address allows.
int gn_vec(int C, int esize, std::initializer_list<const void*> ptrs) {
  for (int vec = 16 / esize; vec > 1; vec >>= 1) {
    if (C % vec) continue;
    bool ok = true;
    for (const void* p : ptrs) ok = ok && reinterpret_cast<uintptr_t>(p) % (size_t)(vec * esize) == 0;
    if (ok) return vec;
  }
  return 1;
}

bool gn_aligned(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return true;
}

bool gn_args_ok(long long N, long long S, int C, int G, int chunks, int act) {
  return N > 0 && S > 0 && C > 0 && G > 0 && C % G == 0 && chunks >= 0 && chunks <= S && act >= GN_NONE && act <= GN_SILU &&
         N * chunks < (1ll << 31) && N * G < (1ll << 31);
}

}  // namespace

#define GN_VEC_CASE(T, V, ...) case V: { constexpr int VEC = V; typedef T E; __VA_ARGS__; } break;
#define GN_DISPATCH(dtype, vec, ...)                                                                                  \
  switch (dtype) {                                                                                                    \
    case PDA_F32: switch (vec) { GN_VEC_CASE(float, 4, __VA_ARGS__) GN_VEC_CASE(float, 2, __VA_ARGS__)                \
                                 default: { constexpr int VEC = 1; typedef float E; __VA_ARGS__; } } break;           \
    case PDA_F16: switch (vec) { GN_VEC_CASE(f16, 8, __VA_ARGS__) GN_VEC_CASE(f16, 4, __VA_ARGS__)                    \
                                 GN_VEC_CASE(f16, 2, __VA_ARGS__)                                                     \
                                 default: { constexpr int VEC = 1; typedef f16 E; __VA_ARGS__; } } break;             \
    case PDA_BF16: switch (vec) { GN_VEC_CASE(bf16, 8, __VA_ARGS__) GN_VEC_CASE(bf16, 4, __VA_ARGS__)                 \
                                  GN_VEC_CASE(bf16, 2, __VA_ARGS__)                                                   \
                                  default: { constexpr int VEC = 1; typedef bf16 E; __VA_ARGS__; } } break;           \
    default: return -6;                                                                                               \
  }
// ... and over the activation class and whether a vector of channels lies in one group
#define GN_DISPATCH_ACT(act, ug, ...)                                                          \
  switch (act) {                                                                               \
    case GN_NONE: { constexpr int ACT = GN_NONE; GN_UG(ug, __VA_ARGS__) } break;               \
    case GN_RELU: { constexpr int ACT = GN_RELU; GN_UG(ug, __VA_ARGS__) } break;               \
    case GN_CAP: { constexpr int ACT = GN_CAP; GN_UG(ug, __VA_ARGS__) } break;                 \
    default: { constexpr int ACT = GN_SILU; GN_UG(ug, __VA_ARGS__) } break;                    \
  }
#define GN_UG(ug, ...)                                                                                        \
  if (ug && VEC * sizeof(E) == 16) { constexpr bool UG = VEC * sizeof(E) == 16; __VA_ARGS__; }                \
  else { constexpr bool UG = false; __VA_ARGS__; }

// How a call runs: 0 = a slab of a sample in registers (group_norm_resident.h), > 0 = that many row chunks a sample, in
// passes.  aligned: every tensor starts on 16 bytes.
PDA_EXPORT int pda_group_norm_plan(int dtype, long long N, long long S, int C, int G, int bwd, int aligned) {
  if (N <= 0 || S <= 0 || C <= 0 || C > (1 << 28) || G <= 0 || C % G) return -1;
  const int es = dtype == PDA_F32 ? 4 : 2;
  if (aligned && gn_resident_plan(es, N, S, C, G, bwd != 0).nv) return 0;
  // about 2048 blocks over the chip, at least 8 rows for each thread of a block
  const int vpr = (C * es + 15) / 16;
  const int rs = vpr >= 256 ? 1 : 256 / vpr;
  long long want = (2048 + N - 1) / N, most = S / (rs * 8ll);
  if (want > most) want = most;
  return (int)(want < 1 ? 1 : want > 1024 ? 1024 : want);
}

// A launch holds fewer than 2^32 threads: samples of `threads` threads each go in steps, one after the other.
template <typename F> static int gn_each_step(long long N, long long threads, F launch) {
  const long long step = (1ll << 31) / threads;  // at least 32: 2^20 channels, a wave a group at most
  if (step < 1) return -1;
  int rc = 0;
  for (long long n0 = 0; n0 < N && rc == 0; n0 += step) rc = launch(n0, N - n0 < step ? N - n0 : step);
  return rc;
}
static long long gn_threads(const GnPlan& p, int C, int G, int chunks) {
  if (chunks == 0) return (long long)p.threads * (C * p.fold / p.W);
  return 256ll * chunks > 64ll * G ? 256ll * chunks : 64ll * G;
}
static const char* gn_at(const void* p, long long bytes) { return p ? static_cast<const char*>(p) + bytes : nullptr; }
static char* gn_at(void* p, long long bytes) { return p ? static_cast<char*>(p) + bytes : nullptr; }

// chunks: from pda_group_norm_plan, as are those of the backward pass.  part: two fp64 [N][chunks][C] (none at 0 chunks);
// stats: {fp64 mean, fp64 1/std} [N][G]
PDA_EXPORT int pda_group_norm_fwd(int dtype, const void* x_, const void* res_, void* out_, const float* gamma,
                                  const float* beta, long long N_, long long S, int C, int G, double eps, int act, float cap,
                                  int chunks, void* part_, void* stats_, hipStream_t st) {
  if (!gn_args_ok(N_, S, C, G, chunks, act)) return -1;
  const int es = dtype == PDA_F32 ? 4 : 2;
  const int vec = gn_vec(C, es, {x_, res_, out_});
  GnPlan p{0, 0, 0};
  if (chunks == 0) {
    p = gn_resident_plan(es, N_, S, C, G, false);
    if (!p.nv || !gn_aligned({x_, res_, out_})) return -1;
  }
  return gn_each_step(N_, gn_threads(p, C, G, chunks), [&](long long n0, long long N) -> int {
    const long long from = n0 * S * C * es;
    const char *x = gn_at(x_, from), *res = gn_at(res_, from);
    char* out = gn_at(out_, from);
    GnStat* stats = (GnStat*)stats_ + n0 * G;
    GnPair* part = (GnPair*)part_ + n0 * chunks * C;
    if (chunks == 0) {
      const GnResidentArgs a{x, res, nullptr, out, nullptr, nullptr, gamma, beta, N, S, C, G, act, eps, cap, stats, nullptr, st};
      return dtype == PDA_F32 ? gn_resident_fwd<float>(p, a) : dtype == PDA_F16 ? gn_resident_fwd<f16>(p, a)
             : dtype == PDA_BF16 ? gn_resident_fwd<bf16>(p, a) : -6;
    }
    const int blocks = (int)(N * chunks);
    GN_DISPATCH(dtype, vec, hipLaunchKernelGGL((gn_partial_kernel<E, VEC>), dim3(blocks), dim3(256), 0, st, (const E*)x, S, C, G,
                                               chunks, part));
    GN_DISPATCH(dtype, 1, hipLaunchKernelGGL((gn_finalize_kernel<E>), dim3((int)(N * G)), dim3(64), 0, st, (const E*)x,
                                             (const GnPair*)part, S, C, G, chunks, eps, stats));
    const bool ug = (C / G) % vec == 0;
    GN_DISPATCH(dtype, vec, GN_DISPATCH_ACT(act, ug, hipLaunchKernelGGL((gn_apply_kernel<E, VEC, UG, ACT>), dim3(blocks),
                dim3(256), 0, st, (const E*)x, (const E*)res, (E*)out, gamma, beta, (const GnStat*)stats, S, C, G, chunks, cap)));
    return pda_check_launch();
  });
}

// part: float2 [N][max(chunks, 1)][C]; ab: float2 [N][G] (none at 0 chunks).  dgamma / dbeta: both or none.
PDA_EXPORT int pda_group_norm_bwd(int dtype, const void* x_, const void* res_, const void* dout_, void* dx_, void* dres_,
                                  const float* gamma, const float* beta, const void* stats_, long long N_, long long S, int C,
                                  int G, int act, float cap, int chunks, void* part_, void* ab_, float* dgamma, float* dbeta,
                                  hipStream_t st) {
  if (!gn_args_ok(N_, S, C, G, chunks, act) || (dres_ && !dx_)) return -1;
  const int es = dtype == PDA_F32 ? 4 : 2;
  const int vec = gn_vec(C, es, {x_, res_, dout_, dx_, dres_});
  const float top = act == GN_CAP ? cap : INFINITY;
  GnPlan p{0, 0, 0};
  if (chunks == 0) {
    p = gn_resident_plan(es, N_, S, C, G, true);
    if (!p.nv || !gn_aligned({x_, res_, dout_, dx_, dres_})) return -1;
  }
  const int rc = gn_each_step(N_, gn_threads(p, C, G, chunks), [&](long long n0, long long N) -> int {
    const long long from = n0 * S * C * es;
    const char *x = gn_at(x_, from), *res = gn_at(res_, from), *dout = gn_at(dout_, from);
    char *dx = gn_at(dx_, from), *dres = gn_at(dres_, from);
    const GnStat* stats = (const GnStat*)stats_ + n0 * G;
    float2* part = (float2*)part_ + n0 * (chunks ? chunks : 1) * C;
    if (chunks == 0) {
      const GnResidentArgs a{x, res, dout, nullptr, dx, dres, gamma, beta, N, S, C, G, act, 0.0, top, const_cast<GnStat*>(stats),
                             dgamma ? part : nullptr, st};
      return dtype == PDA_F32 ? gn_resident_bwd<float>(p, a) : dtype == PDA_F16 ? gn_resident_bwd<f16>(p, a)
             : dtype == PDA_BF16 ? gn_resident_bwd<bf16>(p, a) : -6;
    }
    float2* ab = (float2*)ab_ + n0 * G;
    const int blocks = (int)(N * chunks);
    const bool ug = (C / G) % vec == 0;
    GN_DISPATCH(dtype, vec, GN_DISPATCH_ACT(act, ug, hipLaunchKernelGGL((gn_bwd_partial_kernel<E, VEC, UG, ACT>), dim3(blocks),
                dim3(256), 0, st, (const E*)x, (const E*)res, (const E*)dout, gamma, beta, stats, S, C, G, chunks, top, part)));
    hipLaunchKernelGGL(gn_bwd_finalize_kernel, dim3((int)(N * G)), dim3(64), 0, st, (const float2*)part, gamma, S, C, G, chunks,
                       ab);
    if (dx)
      GN_DISPATCH(dtype, vec, GN_DISPATCH_ACT(act, ug, hipLaunchKernelGGL((gn_bwd_apply_kernel<E, VEC, UG, ACT>), dim3(blocks),
                  dim3(256), 0, st, (const E*)x, (const E*)res, (const E*)dout, (E*)dx, (E*)dres, gamma, beta, stats,
                  (const float2*)ab, S, C, G, chunks, top)));
    return pda_check_launch();
  });
  if (rc || !dgamma) return rc;
  // two steps where one block a channel group would walk far (2^20 x 16 channels 1280 us in one)
  long long rows = N_ * (chunks ? chunks : 1), step = 1;
  const dim3 grid((C + 3) / 4), block(1024);
  if (rows > 4096) {
    const long long span = rows > 512 * 1024ll ? (rows + 1023) / 1024 : 512, parts = (rows + span - 1) / span;
    hipLaunchKernelGGL(gn_params_kernel, dim3(grid.x, (unsigned)parts), block, 0, st, (float2*)part_, rows, span, step, C, nullptr,
                       nullptr);
    rows = parts;
    step = span;
  }
  hipLaunchKernelGGL(gn_params_kernel, grid, block, 0, st, (float2*)part_, rows, rows, step, C, dgamma, dbeta);
  return pda_check_launch();
}
