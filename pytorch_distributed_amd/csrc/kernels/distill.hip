// Distillation from a teacher's top logits: the selection of a row's k largest logits (with the log-sum-exp of the others)
// and the Kullback-Leibler loss of a student against them, forward and backward.
//
// Rows have one stride, their elements are adjacent; a row starts anywhere (odd class counts).  The 16-byte accesses are
// typed as element-aligned; where a row is written, its first elements are taken alone up to the next 16 bytes.  (Where one is
// summed up they are not: that costs 5 % on rows of 50001 16-bit classes, but sums do not depend on where a tensor lies.)
//
// One block takes one row.  Sums S of a row's exponentials are fp32: a thread adds V/256 terms (512 at 131072 classes, 4096 at
// 2^20), N = 4 or 8 of a vector first, so S is off by at most (V/(256 N) + N + 16) 2^-24 of itself - 5e-6 at 131072 16-bit
// classes - and as a rule by the root of so many roundings; each term is good to some 2^-22, and c = log2(e)/T, rounded once, acts as
// a T off by 2^-24 of itself.  That is what bounds the loss (T^2 times it) of a student that has nearly become its teacher.  What
// is formed from S, the k entries and their log-sum-exps is fp64: logarithms that cancel add nothing to it.
#include "common.h"

#include <float.h>

namespace {

constexpr int MAX_K = 1024;          // entries of a row
constexpr int MAX_CLASSES = 1 << 20;  // one bit a class in shared memory

template <typename T> struct RowVec {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};
template <typename T>
__device__ __forceinline__ RowVec<T> row_ld(const T* p) {
  RowVec<T> r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
template <typename T>
__device__ __forceinline__ void row_st(T* p, const RowVec<T>& r) { __builtin_memcpy(p, &r, 16); }

// Elements in front of the first one on a 16-byte address.
template <typename T> __device__ __forceinline__ int row_head(const T* p, int V) {
  const int h = (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T);
  return h < V ? h : V;
}

// Running maximum (raw logit) and sum of exp((z - m)/T).  m starts at the lowest finite number, so that neither a row of
// infinities nor a difference of two of them makes a NaN that the row has not got.
struct MaxSum {
  float m, s;
};
// exp((z - m)/T) with c = log2(e)/T; 1 for m itself, an infinite one too
__device__ __forceinline__ float ms_exp(float z, float m, float c) { return z == m ? 1.f : exp2f((z - m) * c); }
__device__ __forceinline__ void ms_merge(MaxSum& a, float m2, float s2, float c) {
  const float m = fmaxf(a.m, m2);
  a.s = a.s * ms_exp(a.m, m, c) + s2 * ms_exp(m2, m, c);
  a.m = m;
}
__device__ __forceinline__ void ms_add(MaxSum& a, float z, float c) {
  if (z > a.m) {
    a.s *= exp2f((a.m - z) * c);
    a.m = z;
  }
  a.s += ms_exp(z, a.m, c);
}
// 2^x.  The hardware's own is enough for 16-bit logits; fp32 gradients may be denormal, which it flushes.
template <typename T> __device__ __forceinline__ float fast_exp2(float x) {
  return sizeof(T) == 4 ? exp2f(x) : __builtin_amdgcn_exp2f(x);
}
// The same running pair for whole vectors, on the scale that the exponential takes: sum of 2^(z*c - mc) with one
// multiply-add an element.  mc is the rounded product of the maximum and c; flush() takes its rounding out of the sum.  Where
// the product is so large that its rounding matters by itself (masks of the type's lowest value, tiny temperatures), and
// where a NaN or +inf came by, the sum is given as NaN: the caller then looks again with ms_add, which takes differences first.
// So does a thread that meets nothing but large finite masks (below about -1e9) in its first vectors, at most temperatures: the
// exponent of such a term is the rounding of mc, and where that overflows the sum stays no number.
struct FastSum {
  float m = -INFINITY, mc = 0.f, s = 0.f;
  template <int N> __device__ __forceinline__ void add(const float (&z)[N], float c) {
    float top = z[0];
#pragma unroll
    for (int e = 1; e < N; ++e) top = fmaxf(top, z[e]);
    if (top > m) {
      const float mc2 = fmaxf(top * c, -FLT_MAX);  // (finite: a thread that meets masks first goes on from its next maximum)
      s *= s == 0.f ? 0.f : __builtin_amdgcn_exp2f(mc - mc2);
      m = top;
      mc = mc2;
    }
    float a = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) a += __builtin_amdgcn_exp2f(__builtin_fmaf(z[e], c, -mc));
    s += a;
  }
  __device__ __forceinline__ MaxSum flush(float c) const {
    if (m == -INFINITY) return MaxSum{-FLT_MAX, s};  // nothing, or infinities below (or NaN alone: s is one)
    if (!(fabsf(mc) <= 16777216.f)) return MaxSum{m, NAN};
    return MaxSum{m, s * __builtin_amdgcn_exp2f(-__builtin_fmaf(m, c, -mc))};
  }
};
// Over the lanes of a wave, which are all there, to every one of them.  The values go from lane to lane with the instruction
// that adds them (from the 1, 2, 4 and 8 lanes below, then from the ends of the rows of 16), not through shared memory.
template <int FROM, int ROWS> __device__ __forceinline__ float lane_below(float v, float none) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), FROM, ROWS, 0xf, false));
}
__device__ __forceinline__ float last_lane(float v) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float lanes_sum(float v) {
  v += lane_below<0x111, 0xf>(v, 0.f);
  v += lane_below<0x112, 0xf>(v, 0.f);
  v += lane_below<0x114, 0xf>(v, 0.f);
  v += lane_below<0x118, 0xf>(v, 0.f);
  v += lane_below<0x142, 0xa>(v, 0.f);
  v += lane_below<0x143, 0xc>(v, 0.f);
  return last_lane(v);
}
__device__ __forceinline__ float lanes_max(float v) {
  v = fmaxf(v, lane_below<0x111, 0xf>(v, v));
  v = fmaxf(v, lane_below<0x112, 0xf>(v, v));
  v = fmaxf(v, lane_below<0x114, 0xf>(v, v));
  v = fmaxf(v, lane_below<0x118, 0xf>(v, v));
  v = fmaxf(v, lane_below<0x142, 0xa>(v, v));
  v = fmaxf(v, lane_below<0x143, 0xc>(v, v));
  return last_lane(v);
}
__device__ __forceinline__ MaxSum ms_wave(MaxSum a, float c) {
  const float m = lanes_max(a.m);
  return MaxSum{m, lanes_sum(a.s * ms_exp(a.m, m, c))};
}
template <int NT>
__device__ __forceinline__ MaxSum ms_block(MaxSum a, float c, float* scratch /* 2*NT/64 */) {
  a = ms_wave(a, c);
  const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63;
  __syncthreads();
  if (lane == 0) {
    scratch[2 * wid] = a.m;
    scratch[2 * wid + 1] = a.s;
  }
  __syncthreads();
  const bool on = lane < NT / 64;
  return ms_wave(MaxSum{on ? scratch[2 * lane] : -FLT_MAX, on ? scratch[2 * lane + 1] : 0.f}, c);
}

// ------------------------------------------------------------------------------------------------ top logits
// A value as a whole number of the same order: NaN above everything, -0 equal to +0.  0 is below every value.
__device__ __forceinline__ unsigned order_key(float v) {
  const unsigned b = __float_as_uint(v);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if ((b << 1) == 0u) return 0x80000000u;
  return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}

// The value of a key: NaN for a key of none, +0 for both zeros.
__device__ __forceinline__ float key_value(unsigned q) { return __uint_as_float(q & 0x80000000u ? q ^ 0x80000000u : ~q); }

// The digit (0..255) at which a count from the top (or, with ascending, from the bottom) reaches need; need becomes what
// is still to be taken inside that digit.  hist[256] -> every thread.
template <int NT>
__device__ __forceinline__ int radix_digit(unsigned* hist, int& need, bool ascending, int* out /* 2 ints */) {
  __syncthreads();
  if (threadIdx.x < 64) {
    const int l = threadIdx.x;
    int h[4], own = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = l * 4 + i;
      h[i] = (int)hist[ascending ? d : 255 - d];
      own += h[i];
    }
    int before = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int t = __shfl_up(before, o, 64);
      if (l >= o) before += t;
    }
    before -= own;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (before < need && need <= before + h[i]) {
        out[0] = ascending ? l * 4 + i : 255 - (l * 4 + i);
        out[1] = need - before;
      }
      before += h[i];
    }
  }
  __syncthreads();
  need = out[1];
  return out[0];
}

constexpr int MAX_CAND = 1536;  // elements that are ranked

struct TopShared {
  unsigned hist[256];
  int pick[2];
  int count;
  alignas(16) unsigned long long cand[MAX_CAND];  // key, then the class from the last to the first: larger is better
};
__device__ __forceinline__ unsigned long long cand_of(unsigned key, int j) {
  return ((unsigned long long)key << 32) | (0xffffffffu - (unsigned)j);
}

// For any row: the k-th largest key is found digit by digit (a histogram of 256 counts a pass over the row), then, where
// more values equal it than are wanted, the highest class that still belongs, digit by digit of the class.  Leaves the K
// elements in sh.cand and returns the pair of all others.
template <typename T, int NT>
__device__ MaxSum top_by_digits(const T* row, int V, int K, float c, TopShared& sh) {
  unsigned key = 0;
  int need = K;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += NT) sh.hist[i] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < V; j += NT) {
      const unsigned q = order_key(ElemTraits<T>::to_f32(row[j]));
      if (shift == 24 || (q >> (shift + 8)) == key) atomicAdd(&sh.hist[(q >> shift) & 255], 1u);
    }
    key = (key << 8) | (unsigned)radix_digit<NT>(sh.hist, need, false, sh.pick);
    __syncthreads();
  }
  // need of the elements that equal key are wanted, those of the lowest classes
  unsigned last = 0;
  int top_shift = 0;
  while (((V - 1) >> top_shift) > 255) top_shift += 8;
  for (int shift = top_shift; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += NT) sh.hist[i] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < V; j += NT) {
      if (order_key(ElemTraits<T>::to_f32(row[j])) != key) continue;
      if (shift == top_shift || ((unsigned)j >> (shift + 8)) == last) atomicAdd(&sh.hist[((unsigned)j >> shift) & 255], 1u);
    }
    last = (last << 8) | (unsigned)radix_digit<NT>(sh.hist, need, true, sh.pick);
    __syncthreads();
  }
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  MaxSum ms{-FLT_MAX, 0.f};
  for (int j = threadIdx.x; j < V; j += NT) {
    const float v = ElemTraits<T>::to_f32(row[j]);
    const unsigned q = order_key(v);
    if (q > key || (q == key && (unsigned)j <= last)) {
      const int p = atomicAdd(&sh.count, 1);
      if (p < MAX_CAND) sh.cand[p] = cand_of(q, j);
    } else {
      ms_add(ms, v, c);
    }
  }
  __syncthreads();
  return ms;
}

// One block a row, one read of it from memory.  A thread's vectors are cut into CELLS runs; of each run it keeps the
// maximum and the sum of exponentials.  The K-th largest of the threads' maxima is a bound that at least K elements reach,
// and not many more do: only the runs that reach it are read again (from the caches), their elements at or above the bound
// become candidates, and the K best are found by counting for each candidate how many are better.  The log-sum-exp of the
// others is joined from the runs without a candidate and the single elements of the others, nothing is taken off a sum.
// 4096 rows of 131072 bf16, K = 64: 211 us = 5.1 TB/s, bound by memory; one row 16 us, bound by one CU's bandwidth and the
// latency of the steps after the read: some 11 000 cycles a block, of which counting ranks takes 2700, the bound 2700 and the
// second reading 2000 to 4000 (400 x 1000 fp32 7 us, 16384 x 8000 fp16 107 us = 2.5 TB/s).  8 loads are in flight.
// Rows that do not fit this (more candidates than MAX_CAND: many equal values, K near the number of threads or above it) go
// digit by digit: K = 600 takes 4096 x 131072 bf16 4.8 ms.
template <typename T, int NT, int CELLS>
__global__ void __launch_bounds__(NT)
top_logits_kernel(const T* __restrict__ z, long long ld, int V, int K, float c, double temperature, T* __restrict__ values,
                  long long* __restrict__ indices, float* __restrict__ rest) {
  constexpr int VN = RowVec<T>::N, U = CELLS < 8 ? CELLS : 8;  // U: loads in flight
  __shared__ TopShared sh;
  __shared__ int waves[NT / 64];
  __shared__ unsigned tops[NT];
  __shared__ union {
    unsigned short run[CELLS * NT];  // the list of runs
    unsigned key[MAX_CAND];          // later: the keys of candidates that are not among the K
  } list;
  __shared__ float scratch[2 * NT / 64];
  const T* row = z + (long long)blockIdx.x * ld;
  const int nv = V / VN;                                 // whole vectors; a thread each takes what is left
  const int per = (nv + CELLS * NT - 1) / (CELLS * NT);  // vectors of a run: thread + NT*(run*per + 0 .. per-1)
  const int extra = nv * VN + threadIdx.x;
  const unsigned inv = 0xffffffffu / (unsigned)max(per, 1) + 1u;  // w / per = the upper half of w * inv, per > 1, w * per < 2^32
  MaxSum cell[CELLS];
  float most = -INFINITY;
#pragma unroll
  for (int q0 = 0; q0 < CELLS; q0 += U) {
    FastSum fs[U];
    for (int p = 0; p < per; ++p) {
      RowVec<T> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = row_ld(row + (long long)min(threadIdx.x + NT * ((q0 + u) * per + p), nv - 1) * VN);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if ((int)threadIdx.x + NT * ((q0 + u) * per + p) < nv) {
          float zf[VN];
#pragma unroll
          for (int e = 0; e < VN; ++e) zf[e] = ElemTraits<T>::to_f32(v[u].v[e]);
          fs[u].add(zf, c);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      cell[q0 + u] = fs[u].flush(c);
      most = cell[q0 + u].s == 0.f ? most : fmaxf(most, cell[q0 + u].m);
    }
  }
  if (threadIdx.x == 0) sh.count = 0;
  // a NaN or +inf leaves a sum that is no number: such a thread looks for its maximum again
  bool odd = false;
#pragma unroll
  for (int q = 0; q < CELLS; ++q) odd |= !(cell[q].s < INFINITY);
  unsigned mine = order_key(most);
  if (odd) {
    mine = 0;
    for (int i = threadIdx.x; i < nv; i += NT)
      for (int e = 0; e < VN; ++e) mine = max(mine, order_key(ElemTraits<T>::to_f32(row[i * VN + e])));
  }
  if (extra < V) mine = max(mine, order_key(ElemTraits<T>::to_f32(row[extra])));
  // the bound, to the upper 16 bits of the key: one wave counts, bit by bit, how many of the maxima reach it
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  bool fits = K <= NT;
  unsigned bound = 0;
  if (fits) {
    tops[threadIdx.x] = mine >> 16;
    __syncthreads();
    if (wave == 0) {
      unsigned t[NT / 64];
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) t[w] = tops[w * 64 + lane];
      const auto reach = [&](unsigned b) {
        int m = 0;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) m += __popcll(__ballot(t[w] >= b));
        return m;
      };
      int n = 0;
#pragma unroll 1
      for (int bits = 14; bits >= 0 && n != K; bits -= 2) {
        const unsigned b1 = bound | 1u << bits, b2 = bound | 2u << bits, b3 = bound | 3u << bits;
        const int n1 = reach(b1), n2 = reach(b2), n3 = reach(b3);
        if (n1 >= K) {
          bound = n3 >= K ? b3 : n2 >= K ? b2 : b1;
          n = n3 >= K ? n3 : n2 >= K ? n2 : n1;
        }
      }
      if (lane == 0) sh.pick[0] = (int)bound;
    }
    __syncthreads();
    bound = (unsigned)sh.pick[0] << 16;
  }
  MaxSum ms{-FLT_MAX, 0.f};
  if (fits) {
    // the runs to read again, as a list in the order of wave, run and lane: all their vectors are then fetched at once
    const float low = key_value(bound);
    unsigned long long mask[CELLS];
    int own = 0;
    float base = -FLT_MAX, sum = 0.f;
#pragma unroll
    for (int q = 0; q < CELLS; ++q) {
      // (a sum of 0: -inf alone)
      const bool some = (int)threadIdx.x + NT * q * per < nv;
      const bool again = some && (!(cell[q].s < INFINITY) || !((cell[q].s == 0.f ? -INFINITY : cell[q].m) < low));
      mask[q] = __ballot(again);
      own += __popcll(mask[q]);
      if (!some || again) cell[q] = MaxSum{-FLT_MAX, 0.f};
      base = fmaxf(base, cell[q].m);
    }
#pragma unroll
    for (int q = 0; q < CELLS; ++q) sum += cell[q].s * __builtin_amdgcn_exp2f((cell[q].m - base) * c);  // all finite
    ms = MaxSum{base, sum};
    if (lane == 0) waves[wave] = own;
    __syncthreads();
    int at = 0, runs = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
      const int n = waves[w];
      at += w < wave ? n : 0;
      runs += n;
    }
#pragma unroll
    for (int q = 0; q < CELLS; ++q) {
      if ((mask[q] >> lane) & 1ull) list.run[at + __popcll(mask[q] & ((1ull << lane) - 1ull))] = (unsigned short)(q * NT + threadIdx.x);
      at += __popcll(mask[q]);
    }
    __syncthreads();
    const int todo = runs * per;
    // elements that reach the bound (NaN does) become candidates, the others are summed
    const auto vector = [&](int w) {
      const int q = per == 1 ? w : (int)__umulhi((unsigned)w, inv), e0 = list.run[q];
      return (e0 % NT) + NT * ((e0 / NT) * per + (w - q * per));
    };
    FastSum fs;
    for (int w0 = wave * 64; w0 < todo; w0 += NT) {
      const int w = w0 + lane, i = w < todo ? vector(w) : nv;
      float zf[VN];
#pragma unroll
      for (int e = 0; e < VN; ++e) zf[e] = -INFINITY;
      if (i < nv) {
        const RowVec<T> v = row_ld(row + (long long)i * VN);
#pragma unroll
        for (int e = 0; e < VN; ++e) zf[e] = ElemTraits<T>::to_f32(v.v[e]);
      }
      // one count a wave; of each element the lanes below and the elements before
      unsigned long long hit[VN];
      int hits = 0;
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        hit[e] = __ballot(i < nv && !(zf[e] < low));
        hits += __popcll(hit[e]);
      }
      int at = 0;
      if (hits) {
        if (lane == 0) at = atomicAdd(&sh.count, hits);
        at = __builtin_amdgcn_readfirstlane(at);
      }
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        if ((hit[e] >> lane) & 1ull) {
          const int p = at + __popcll(hit[e] & ((1ull << lane) - 1ull));
          if (p < MAX_CAND) sh.cand[p] = cand_of(order_key(zf[e]), i * VN + e);
          zf[e] = -INFINITY;
        }
        at += __popcll(hit[e]);
      }
      fs.add(zf, c);
    }
    MaxSum again = fs.flush(c);
    if (!(again.s < INFINITY)) {  // rare: from differences
      again = MaxSum{-FLT_MAX, 0.f};
      for (int w = threadIdx.x; w < todo; w += NT) {
        const int i = vector(w);
        if (i >= nv) continue;
        for (int e = 0; e < VN; ++e) {
          const float v = ElemTraits<T>::to_f32(row[i * VN + e]);
          if (v < low) ms_add(again, v, c);
        }
      }
    }
    ms_merge(ms, again.m, again.s, c);
    if (extra < V) {
      const float v = ElemTraits<T>::to_f32(row[extra]);
      if (!(v < low)) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < MAX_CAND) sh.cand[at] = cand_of(order_key(v), extra);
      } else {
        ms_add(ms, v, c);
      }
    }
    __syncthreads();
    fits = sh.count >= K && sh.count <= MAX_CAND;
  }
  if (!fits) {
    __syncthreads();
    ms = top_by_digits<T, NT>(row, V, K, c, sh);
  }
  // in order of rank (the list's own order is that of the atomics): what comes after the K-th joins the others
  const int n = sh.count;
  if (threadIdx.x < 8 && n + threadIdx.x < MAX_CAND) sh.cand[n + threadIdx.x] = 0;  // worse than every candidate
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT) {
    const unsigned long long me = sh.cand[i];
    int r = 0;
    for (int o = 0; o < n; o += 8) {
      ulonglong2 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = reinterpret_cast<const ulonglong2*>(sh.cand + o)[u];
#pragma unroll
      for (int u = 0; u < 4; ++u) r += (v[u].x > me ? 1 : 0) + (v[u].y > me ? 1 : 0);
    }
    const unsigned j = 0xffffffffu - (unsigned)me, key = (unsigned)(me >> 32);
    if (r < K) {
      // (the row's own NaN, and its sign of a zero)
      const T v = key == 0xffffffffu || key == 0x80000000u ? row[j] : ElemTraits<T>::from_f32(key_value(key));
      values[(long long)blockIdx.x * K + r] = v;
      indices[(long long)blockIdx.x * K + r] = (long long)j;
    } else {
      list.key[r - K] = key;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n - K; i += NT) ms_add(ms, key_value(list.key[i]), c);
  ms = ms_block<NT>(ms, c, scratch);
  if (threadIdx.x == 0)
    rest[blockIdx.x] = ms.s == 0.f ? -INFINITY : (float)((double)ms.m / temperature + log((double)ms.s));
}

// ------------------------------------------------------------------------------------------------ distillation loss
__device__ __forceinline__ float rd_value(const void* p, int dtype, long long i) {
  if (dtype == PDA_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == PDA_F16) return (float)reinterpret_cast<const f16*>(p)[i];
  return (float)reinterpret_cast<const bf16*>(p)[i];
}
__device__ __forceinline__ long long rd_index(const void* p, int is64, long long i) {
  return is64 ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// maximum that keeps a NaN
__device__ __forceinline__ double max_nan(double a, double b) { return (b > a || b != b) ? b : a; }
__device__ __forceinline__ double wave_max_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max_nan(v, __shfl_xor(v, o, 64));
  return v;
}

// What a row leaves for its backward pass: dz_j = T (exp((z_j - shift)/T) * factor) g outside the entries, T dtop_k g at
// entry k (dtop = q - p).  A factor of 0 is a row whose gradient is zero everywhere outside the entries.
struct RowStat { float shift, factor; };

// Shared memory of a row: the entries, then one bit a class.
struct RowEntries {
  double* p;        // [K] the teacher's logits over T
  int* idx;         // [K] class, -1 for an empty entry
  int* first;       // [K] the first entry of the same class
  float* z;         // [K] the student's logit there
  unsigned* bits;   // [(V + 31)/32]
  __device__ RowEntries(char* mem, int K) {
    p = reinterpret_cast<double*>(mem);
    idx = reinterpret_cast<int*>(mem + 8ll * K);
    first = idx + K;
    z = reinterpret_cast<float*>(first + K);
    bits = reinterpret_cast<unsigned*>(z + K);
  }
};
inline size_t row_entries_bytes(int K, int V) { return 20ull * K + 4ull * ((V + 31) / 32) + 16; }

// One block a row, one read of it: 8192 x 131072 bf16 375 us = 5.7 TB/s, bound by memory; 400 x 1000 by the latency of the row's
// few fp64 steps, which one wave takes.  With rest, classes that are entries stay out of (m, s): the student's remainder is summed by itself, since one minus
// the entries' sum would keep no digits where the entries hold nearly everything.
template <typename T, int NT>
__global__ void __launch_bounds__(NT)
distill_fwd_kernel(const T* __restrict__ z, long long ld, int V, const void* __restrict__ values, int vdtype, long long vld,
                   const void* __restrict__ indices, int idx64, long long ild, const float* __restrict__ rest, int K,
                   double temperature, float c, float* __restrict__ row_loss, RowStat* __restrict__ stat,
                   float* __restrict__ dtop) {
  extern __shared__ __align__(16) char mem[];
  __shared__ float scratch[2 * NT / 64];
  __shared__ int twice;
  const RowEntries en(mem, K);
  const long long rowi = blockIdx.x;
  const T* row = z + rowi * ld;
  constexpr int VN = RowVec<T>::N;
  for (int i = threadIdx.x; i < (V + 31) / 32; i += NT) en.bits[i] = 0u;
  if (threadIdx.x == 0) twice = 0;
  const double it = 1.0 / temperature;
  __syncthreads();
  for (int k = threadIdx.x; k < K; k += NT) {
    const long long i = rd_index(indices, idx64, rowi * ild + k);
    const int j = (i >= 0 && i < V) ? (int)i : -1;
    en.idx[k] = j;
    en.first[k] = k;
    en.p[k] = (double)rd_value(values, vdtype, rowi * vld + k) * it;
    if (j >= 0) {
      en.z[k] = ElemTraits<T>::to_f32(row[j]);
      if (atomicOr(&en.bits[j >> 5], 1u << (j & 31)) & (1u << (j & 31))) twice = 1;
    }
  }
  __syncthreads();
  const int nv = V / VN;
  const unsigned char* bytes = reinterpret_cast<const unsigned char*>(en.bits);
  const auto fetch = [&](int i) { return row_ld(row + (long long)i * VN); };
  FastSum fs;
  const auto take = [&](const RowVec<T>& v, int i) {
    float zf[VN];
#pragma unroll
    for (int e = 0; e < VN; ++e) zf[e] = ElemTraits<T>::to_f32(v.v[e]);
    if (rest) {
      const unsigned skip = VN == 8 ? bytes[i] : (bytes[i >> 1] >> ((i & 1) * 4)) & 15u;
      if (skip)
#pragma unroll
        for (int e = 0; e < VN; ++e) zf[e] = (skip >> e) & 1u ? -INFINITY : zf[e];
    }
    fs.add(zf, c);
  };
  constexpr int U = 4;  // loads in flight
  int i = threadIdx.x;
  for (; i + (U - 1) * NT < nv; i += U * NT) {
    RowVec<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = fetch(i + u * NT);
#pragma unroll
    for (int u = 0; u < U; ++u) take(v[u], i + u * NT);
  }
  for (; i < nv; i += NT) take(fetch(i), i);
  MaxSum ms = fs.flush(c);
  const bool odd = !(ms.s < INFINITY);
  const auto skipped = [&](int j) { return rest && ((en.bits[j >> 5] >> (j & 31)) & 1u); };
  const int from = __syncthreads_or(odd) ? 0 : nv * VN;  // the last elements, or all of them again
  if (from == 0) ms = MaxSum{-FLT_MAX, 0.f};
  for (int j = from + threadIdx.x; j < V; j += NT)
    if (!skipped(j)) ms_add(ms, ElemTraits<T>::to_f32(row[j]), c);
  ms = ms_block<NT>(ms, c, scratch);
  if (twice)  // rare: entries of one class are one class of the distribution
    for (int k = threadIdx.x; k < K; k += NT)
      if (en.idx[k] >= 0)
        for (int o = 0; o < k; ++o)
          if (en.idx[o] == en.idx[k]) { en.first[k] = o; break; }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const int lane = threadIdx.x;
  // Student: log q of an entry is (z - M)/T - lS with the maximum M of everything and S = sum exp((z - M)/T); all logarithms
  // are taken next to a maximum, where masks of -1e38 do not swallow them.  (A softmax that holds +inf is NaN, as
  // everywhere else.)
  const double m = (double)ms.m, ls = log((double)ms.s);
  double M = m, S = ms.m == INFINITY ? (double)NAN : (double)ms.s;
  if (rest) {
    double me = -DBL_MAX;
    for (int k = lane; k < K; k += 64)
      if (en.idx[k] >= 0) me = max_nan(me, (double)en.z[k]);
    me = wave_max_d(me);
    double se = 0.0;
    for (int k = lane; k < K; k += 64)
      if (en.idx[k] >= 0 && en.first[k] == k) se += exp(((double)en.z[k] - me) * it);
    se = wave_sum_d(se);
    M = max_nan(m, me);
    S = S * exp((m - M) * it) + (se == 0.0 ? 0.0 : se * exp((me - M) * it));
  }
  const double lS = log(S);
  // teacher
  const double R = rest ? (double)rest[rowi] : -INFINITY;
  double tm = -INFINITY;
  int any = 0;
  for (int k = lane; k < K; k += 64)
    if (en.idx[k] >= 0) {
      any = 1;
      tm = max_nan(tm, en.p[k]);
    }
  any = __any(any);
  tm = max_nan(wave_max_d(tm), R);
  if (!any || tm == -INFINITY) {  // nothing to learn from
    for (int k = lane; k < K; k += 64) dtop[rowi * K + k] = 0.f;
    if (lane == 0) {
      row_loss[rowi] = 0.f;
      stat[rowi] = RowStat{0.f, 0.f};
    }
    return;
  }
  double ts = 0.0;
  for (int k = lane; k < K; k += 64)
    if (en.idx[k] >= 0) ts += exp(en.p[k] - tm);
  ts = wave_sum_d(ts);
  if (rest) ts += exp(R - tm);
  const double lts = log(ts);
  double loss = 0.0;
  for (int k = lane; k < K; k += 64) {
    const int j = en.idx[k];
    double d = 0.0;
    if (j >= 0) {
      double lp = (en.p[k] - tm) - lts, p = exp(lp);
      if (twice) {
        p = 0.0;
        for (int o = 0; o < K; ++o)
          if (en.idx[o] == j) p += exp((en.p[o] - tm) - lts);
        lp = log(p);
      }
      const double lq = ((double)en.z[k] - M) * it - lS;
      if (en.first[k] == k && p != 0.0) loss += p * (lp - lq);
      d = exp(lq) - p;
    }
    dtop[rowi * K + k] = (float)d;
  }
  loss = wave_sum_d(loss);
  // q of the remainder against its own maximum: q_j = exp((z_j - m)/T) * factor
  double factor = exp((m - M) * it - lS);
  if (rest) {
    const double pr = exp((R - tm) - lts);
    if (pr != 0.0) {
      loss += pr * (((R - tm) - lts) - ((m - M) * it + ls - lS));
      factor -= pr / (double)ms.s;
    }
    if (ms.s == 0.f) factor = 0.0;
  }
  if (lane == 0) {
    row_loss[rowi] = (float)(loss * temperature * temperature);
    stat[rowi] = RowStat{ms.m, (float)factor};
  }
}

// dz of a row: one value for every class, then the entries' own over it (the barrier orders the two writes).  Bound by memory:
// 8192 x 131072 bf16 778 us = 5.5 TB/s.
// Rows go from the last to the first: what the forward pass read last is still in the memory-side cache, and a gradient too
// large to stay there itself passes it by (stream: non-temporal stores; 2047 x 50001 bf16 160 -> 144 us with the forward pass,
// 8192 x 131072 1250 -> 1212 us).
template <typename T, int NT>
__global__ void __launch_bounds__(NT)
distill_bwd_kernel(const T* __restrict__ z, long long ld, int V, const void* __restrict__ indices, int idx64, long long ild,
                   int K, float c, const RowStat* __restrict__ stat, const float* __restrict__ dtop,
                   const float* __restrict__ g, int gstride, float gscale, int stream, T* __restrict__ dz) {
  const long long rowi = gridDim.x - 1 - blockIdx.x;
  const T* row = z + rowi * ld;
  T* out = dz + rowi * V;
  constexpr int VN = RowVec<T>::N;
  const float gr = g[rowi * gstride] * gscale;
  const RowStat st = stat[rowi];
  const float f = st.factor * gr;
  const int head = row_head(out, V), nv = (V - head) / VN;
  const auto end = [&](int o) { return o < head ? o : nv * VN + o; };  // the o-th of the elements outside the vectors
  if (st.factor == 0.f) {  // not read: what stands in a row without entries may be anything
    RowVec<T> v;
#pragma unroll
    for (int e = 0; e < VN; ++e) v.v[e] = ElemTraits<T>::from_f32(0.f);
    for (int i = threadIdx.x; i < nv; i += NT) row_st(out + head + (long long)i * VN, v);
    for (int o = threadIdx.x; o < V - nv * VN; o += NT) out[end(o)] = ElemTraits<T>::from_f32(0.f);
  } else {
    const auto value = [&](float zf) { return fast_exp2<T>((zf - st.shift) * c) * f; };
    const auto put = [&](RowVec<T>& v, int i) {
#pragma unroll
      for (int e = 0; e < VN; ++e) v.v[e] = ElemTraits<T>::from_f32(value(ElemTraits<T>::to_f32(v.v[e])));
      T* o = out + head + (long long)i * VN;
      if (stream) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), reinterpret_cast<u32x4*>(o));
      else row_st(o, v);
    };
    constexpr int U = 4;
    int i = threadIdx.x;
    for (; i + (U - 1) * NT < nv; i += U * NT) {
      RowVec<T> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = row_ld(row + head + (long long)(i + u * NT) * VN);
#pragma unroll
      for (int u = 0; u < U; ++u) put(v[u], i + u * NT);
    }
    for (; i < nv; i += NT) {
      RowVec<T> v = row_ld(row + head + (long long)i * VN);
      put(v, i);
    }
    for (int o = threadIdx.x; o < V - nv * VN; o += NT) out[end(o)] = ElemTraits<T>::from_f32(value(ElemTraits<T>::to_f32(row[end(o)])));
  }
  __syncthreads();
  for (int k = threadIdx.x; k < K; k += NT) {
    const long long j = rd_index(indices, idx64, rowi * ild + k);
    if (j >= 0 && j < V) out[j] = ElemTraits<T>::from_f32(dtop[rowi * K + k] * gr);
  }
}

// out = scale * sum of x: one block, fp64 (8192 rows 5.6 us, 2^20 rows 288 us).
__global__ void __launch_bounds__(1024)
row_total_kernel(const float* __restrict__ x, long long n, double scale, float* __restrict__ out) {
  __shared__ double red[16];
  double a = 0.0;
  for (long long i = threadIdx.x; i < n; i += 1024) a += (double)x[i];
  a = wave_sum_d(a);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) a += red[w];
    *out = (float)(a * scale);
  }
}

}  // namespace

#define DISTILL_DISPATCH(dtype, ...)                        \
  switch (dtype) {                                          \
    case PDA_F32: { typedef float T; __VA_ARGS__; } break;  \
    case PDA_F16: { typedef f16 T; __VA_ARGS__; } break;    \
    case PDA_BF16: { typedef bf16 T; __VA_ARGS__; } break;  \
    default: return -6;                                     \
  }

static const double LOG2E = 1.4426950408889634;

// A launch holds fewer than 2^32 threads: rows of one block each go in steps of 2^21.
constexpr long long ROW_STEP = 1ll << 21;
template <typename F> static int each_step(long long rows, F launch) {
  int rc = 0;
  for (long long r0 = 0; r0 < rows && rc == 0; r0 += ROW_STEP) rc = launch(r0, rows - r0 < ROW_STEP ? rows - r0 : ROW_STEP);
  return rc;
}
static const char* bytes_at(const void* p, long long bytes) { return p ? static_cast<const char*>(p) + bytes : nullptr; }
static char* bytes_at(void* p, long long bytes) { return static_cast<char*>(p) + bytes; }
static int size_of(int dtype) { return dtype == PDA_F32 ? 4 : 2; }

PDA_EXPORT int pda_top_logits(int dtype, const void* z, long long ld, long long rows, int V, int K, double temperature,
                              void* values, long long* indices, float* rest, hipStream_t st) {
  if (rows <= 0 || rows >= (1ll << 31) || V <= 0 || V > MAX_CLASSES || K <= 0 || K > V || K > MAX_K || !(temperature > 0.0))
    return -1;
  const float c = (float)(LOG2E / temperature);
  const long long es = size_of(dtype), bytes = V * es;
#define TOP_LAUNCH(NT, CELLS)                                                                                                  \
  DISTILL_DISPATCH(dtype, hipLaunchKernelGGL((top_logits_kernel<T, NT, CELLS>), dim3((unsigned)n), dim3(NT), 0, st,             \
                                             (const T*)bytes_at(z, r0 * ld * es), ld, V, K, c, temperature,                     \
                                             (T*)bytes_at(values, r0 * K * es), indices + r0 * K, rest + r0))
  // Threads: enough that the K-th largest of their maxima is close to the K-th largest element (the candidates are about
  // NT log(NT/(NT - K))), few where rows are short, since the steps after the read take as long for any row and other
  // rows' blocks fill the time (256 / 512 threads: 8192 x 20000 fp16 95 / 144 us, 512 x 50000 bf16 18.5 / 20.1,
  // 4096 x 131072 bf16 231 / 211, one row of it 21 / 16).  Short rows: no more runs than they have vectors.
  return each_step(rows, [&](long long r0, long long n) {
    if (bytes <= 8 * 1024) {
      TOP_LAUNCH(256, 2)
    } else if (K > 160 || bytes > 128 * 1024) {
      TOP_LAUNCH(512, 8)
    } else if (bytes <= 32 * 1024) {
      TOP_LAUNCH(256, 4)
    } else {
      TOP_LAUNCH(256, 8)
    }
    return pda_check_launch();
  });
}

template <typename T, int NT>
static int launch_distill_fwd(const void* z, long long ld, long long rows, int V, const void* values, int vdtype,
                              long long vld, const void* indices, int idx64, long long ild, const float* rest, int K,
                              double temperature, float* row_loss, void* stat, float* dtop, hipStream_t st) {
  const size_t lds = row_entries_bytes(K, V);
  if (lds > 64 * 1024) {
    hipError_t r = hipFuncSetAttribute(reinterpret_cast<const void*>(distill_fwd_kernel<T, NT>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (r != hipSuccess) return (int)r;
  }
  hipLaunchKernelGGL((distill_fwd_kernel<T, NT>), dim3((unsigned)rows), dim3(NT), lds, st, (const T*)z, ld, V, values, vdtype,
                     vld, indices, idx64, ild, rest, K, temperature, (float)(LOG2E / temperature), row_loss, (RowStat*)stat,
                     dtop);
  return pda_check_launch();
}

// stat: {fp32 shift, fp32 factor} [rows]; dtop: fp32 [rows][K].  loss (may be null): scale * sum of row_loss.
PDA_EXPORT int pda_distill_fwd(int dtype, const void* z, long long ld, long long rows, int V, const void* values, int vdtype,
                               long long vld, const void* indices, int idx64, long long ild, const float* rest, int K,
                               double temperature, float* row_loss, void* stat, float* dtop, float* loss, double scale,
                               hipStream_t st) {
  if (rows <= 0 || rows >= (1ll << 31) || V <= 0 || V > MAX_CLASSES || K <= 0 || K > MAX_K || !(temperature > 0.0)) return -1;
  if (vdtype != PDA_F32 && vdtype != PDA_F16 && vdtype != PDA_BF16) return -6;
  int rc = each_step(rows, [&](long long r0, long long n) {
    const void* zr = bytes_at(z, r0 * ld * size_of(dtype));
    const void* vr = bytes_at(values, r0 * vld * size_of(vdtype));
    const void* ir = bytes_at(indices, r0 * ild * (idx64 ? 8 : 4));
    DISTILL_DISPATCH(dtype, return (launch_distill_fwd<T, 256>(zr, ld, n, V, vr, vdtype, vld, ir, idx64, ild, rest ? rest + r0 : nullptr,
                                                               K, temperature, row_loss + r0, (RowStat*)stat + r0, dtop + r0 * K, st)));
    return 0;
  });
  if (rc == 0 && loss) {
    hipLaunchKernelGGL(row_total_kernel, dim3(1), dim3(1024), 0, st, row_loss, rows, scale, loss);
    rc = pda_check_launch();
  }
  return rc;
}

// g: fp32, one for all rows (gstride 0) or one a row (gstride 1); gscale: what it is multiplied with.
PDA_EXPORT int pda_distill_bwd(int dtype, const void* z, long long ld, long long rows, int V, const void* indices, int idx64,
                               long long ild, int K, double temperature, const void* stat, const float* dtop, const float* g,
                               int gstride, float gscale, void* dz, hipStream_t st) {
  if (rows <= 0 || rows >= (1ll << 31) || V <= 0 || V > MAX_CLASSES || K <= 0 || K > MAX_K || !(temperature > 0.0)) return -1;
  const float c = (float)(LOG2E / temperature);
  const long long es = size_of(dtype);
  const int stream = rows * V * es > pda_stream_min_bytes();
#define DISTILL_BWD(NT)                                                                                                          \
  DISTILL_DISPATCH(dtype, hipLaunchKernelGGL((distill_bwd_kernel<T, NT>), dim3((unsigned)n), dim3(NT), 0, st,                      \
                                             (const T*)bytes_at(z, r0 * ld * es), ld, V,                                          \
                                             bytes_at(indices, r0 * ild * (idx64 ? 8 : 4)), idx64, ild, K, c,                     \
                                             (const RowStat*)stat + r0, dtop + r0 * K, g + r0 * gstride, gstride, gscale, stream,  \
                                             (T*)dz + r0 * V))
  // long rows: fewer of them at once (256 / 1024 threads: 8192 x 131072 bf16 861 / 778 us, 2047 x 50001 72 / 66,
  // 32 x 131072 17 / 11, 1024 x 20000 15 / 15)
  return each_step(rows, [&](long long r0, long long n) {
    if (V * es < 32 * 1024) {
      DISTILL_BWD(256)
    } else {
      DISTILL_BWD(1024)
    }
    return pda_check_launch();
  });
}
