// aq_sample.hip - one token for each row of logits: temperature, top-k, top-p and
// min-p, from given random numbers.
//
// A row's tokens are ordered by logit, of equal ones the lowest token first; a
// token's weight is e^((x - max) / T).  What top-k, top-p and min-p keep are
// beginnings of that order, so the kept set is the shortest of three beginnings,
// all that is left of it is its sum, and the token is the first whose running sum
// exceeds u times it.  Every step is one question: the first token of the order up
// to which the count, or the sum, reaches a number.
//
// Weights are formed in 64 bits and added as whole multiples of 2^-kScale(n) of
// the largest (kScale(n) = 62 - bits of n; 45 for a vocabulary of 128 256), so
// sums do not depend on the order of their terms, nor on which path finds a token:
// the sum of n such roundings is off by 2^-46 n at most, 2^-29 of the largest
// weight, and by about 2^-37 of it in practice.  (In fp32 a running sum's error of
// 2^-24 would move every thousandth border between two tokens across u.)
#include <math.h>

#include "aq_internal.h"

namespace aq {
namespace {

constexpr int kWG = 1024;
constexpr int kBins = 2048;
constexpr int kCap = 4096;  // tokens that are sorted at once
constexpr double kSpan = 44.0;  // exponents that the linear bins cover: e^-44 < 2^-63

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ uint32_t key_of(float x) {  // ascending with x; 0 and -0 alike
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
// a token's place in the order, descending: its logit's key, then its number
__device__ __forceinline__ uint64_t place_of(float x, uint32_t t) {
  return (uint64_t)key_of(x) << 32 | (uint32_t)~t;
}

struct Row {
  float top;       // the largest logit
  double inv_t;    // 1 / temperature
  double scale;    // units of the sums
  double p, min_p, u;
  int64_t k;       // 0: no top-k
  float inv_bin;   // linear bins per logit
  // weight of a logit, and in units
  __device__ __forceinline__ double weight(float x) const {
    return x == top ? 1.0 : exp(((double)x - (double)top) * inv_t);
  }
  __device__ __forceinline__ uint64_t units(float x) const {
    return (uint64_t)(weight(x) * scale + 0.5);
  }
  // the linear bin: no larger for a larger logit
  __device__ __forceinline__ int bin(float x) const {
    return x == top ? 0 : (int)fminf((top - x) * inv_bin, (float)(kBins - 1));
  }
};

struct Shared {
  uint64_t mass[kBins];
  uint32_t count[kBins];
  uint64_t list[kCap];
  uint64_t wave_mass[kWG / 64];
  uint32_t wave_count[kWG / 64];
  uint64_t found;
  uint64_t before_mass;
  uint32_t before_count, bin, n_list, key_lo, key_hi, in_bin;
  float wave_max[kWG / 64];
};

// Every token above -infinity (NaNs count as that): f(x, token).
template <class F>
__device__ __forceinline__ void each_token(const float *x, int64_t n, F &&f) {
  const float lowest = -__builtin_inff();
  for (int64_t i = 4 * (int64_t)threadIdx.x; i < n; i += 4 * kWG) {
    if (i + 4 <= n) {
      const f4u v = *reinterpret_cast<const f4u *>(x + i);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (v[e] > lowest) f(v[e], (uint32_t)(i + e));
    } else {
      for (int64_t j = i; j < n; ++j)
        if (x[j] > lowest) f(x[j], (uint32_t)j);
    }
  }
}

// inclusive running sums over the workgroup, a thread's own first
__device__ __forceinline__ void running(uint64_t &mass, uint32_t &count, Shared &s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint64_t m = __shfl_up((unsigned long long)mass, off);
    const uint32_t c = __shfl_up(count, off);
    if (lane >= off) mass += m, count += c;
  }
  if (lane == 63) s.wave_mass[wave] = mass, s.wave_count[wave] = count;
  __syncthreads();
  for (int w = 0; w < wave; ++w) mass += s.wave_mass[w], count += s.wave_count[w];
  __syncthreads();
}

// What is asked: the first token of the order where the count (BY_COUNT) or the
// sum reaches `goal` >= 1.
struct Answer {
  uint64_t place;  // 0: no token
  uint64_t mass;   // the sum up to and with it
  uint64_t total;  // of all tokens (from the first pass)
};

// The bins hold counts and masses; finds the one where the goal is reached and
// what lies before it.  false: none.
__device__ __forceinline__ bool find_bin(Shared &s, bool by_count, uint64_t goal,
                                         uint64_t &before_mass, uint32_t &before_count, int &bin,
                                         uint32_t &in_bin, uint64_t *total) {
  constexpr int PER = kBins / kWG;
  const int t = threadIdx.x;
  uint64_t mass = 0;
  uint32_t count = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) mass += s.mass[PER * t + i], count += s.count[PER * t + i];
  uint64_t m = mass;
  uint32_t c = count;
  if (t == 0) s.bin = kBins;
  running(m, c, s);
  uint64_t bm = before_mass + m - mass;
  uint32_t bc = before_count + c - count;
  if ((by_count ? (uint64_t)bc : bm) < goal &&
      (by_count ? (uint64_t)(before_count + c) : before_mass + m) >= goal) {
    int i = PER * t;
    for (;; ++i) {
      if ((by_count ? (uint64_t)bc + s.count[i] : bm + s.mass[i]) >= goal) break;
      bm += s.mass[i], bc += s.count[i];
    }
    s.bin = i, s.before_mass = bm, s.before_count = bc, s.in_bin = s.count[i];
  }
  if (t == kWG - 1) s.found = before_mass + m;
  __syncthreads();
  if (total) *total = s.found;
  bin = (int)s.bin;
  if (bin < kBins) before_mass = s.before_mass, before_count = s.before_count, in_bin = s.in_bin;
  __syncthreads();
  return bin < kBins;
}

__device__ __forceinline__ void clear_bins(Shared &s) {
  for (int i = threadIdx.x; i < kBins; i += kWG) s.mass[i] = 0, s.count[i] = 0;
  __syncthreads();
}

// list[0 .. n) in descending order (n at most kCap; what is past n is scratch)
__device__ __forceinline__ void sort_list(Shared &s, int n) {
  int m = 64;
  while (m < n) m <<= 1;
  for (int i = n + threadIdx.x; i < m; i += kWG) s.list[i] = 0;
  __syncthreads();
  for (int size = 2; size <= m; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      for (int i = threadIdx.x; i < m / 2; i += kWG) {
        const int a = 2 * i - (i & (step - 1)), b = a + step;
        const uint64_t x = s.list[a], y = s.list[b];
        if ((x < y) == ((a & size) == 0)) s.list[a] = y, s.list[b] = x;
      }
      __syncthreads();
    }
}

__device__ Answer ask(const float *x, int64_t n, const Row &r, Shared &s, bool by_count,
                      uint64_t goal) {
  const int t = threadIdx.x;
  Answer a = {0, 0, 0};
  uint64_t before_mass = 0;
  uint32_t before_count = 0, in_bin = 0;
  int bin;
  clear_bins(s);
  each_token(x, n, [&](float v, uint32_t) {
    const int b = r.bin(v);
    atomicAdd(&s.count[b], 1u);
    atomicAdd((unsigned long long *)&s.mass[b], (unsigned long long)r.units(v));
  });
  __syncthreads();
  if (!find_bin(s, by_count, goal, before_mass, before_count, bin, in_bin, &a.total)) return a;
  // the bin's tokens have the keys lo .. hi
  if (t == 0) s.key_lo = 0xFFFFFFFFu, s.key_hi = 0;
  __syncthreads();
  each_token(x, n, [&](float v, uint32_t) {
    if (r.bin(v) == bin) atomicMin(&s.key_lo, key_of(v)), atomicMax(&s.key_hi, key_of(v));
  });
  __syncthreads();
  uint32_t lo = s.key_lo, hi = s.key_hi;
  __syncthreads();
  while (in_bin > kCap && lo < hi) {  // bins of equal ranges of keys, descending
    int shift = 0;
    while (((hi - lo) >> shift) >= kBins) ++shift;
    clear_bins(s);
    each_token(x, n, [&](float v, uint32_t) {
      const uint32_t key = key_of(v);
      if (key < lo || key > hi) return;
      const int b = (hi - key) >> shift;
      atomicAdd(&s.count[b], 1u);
      atomicAdd((unsigned long long *)&s.mass[b], (unsigned long long)r.units(v));
    });
    __syncthreads();
    find_bin(s, by_count, goal, before_mass, before_count, bin, in_bin, nullptr);
    hi -= (uint32_t)bin << shift;
    const uint32_t width = (1u << shift) - 1;
    lo = hi - lo > width ? hi - width : lo;
  }
  uint32_t t_lo = 0, t_hi = 0xFFFFFFFFu;
  if (in_bin > kCap) {  // of equal logits the lowest tokens first
    const uint64_t each = r.units(value_of(lo));
    int shift = 0;
    while (((n - 1) >> shift) >= kBins) ++shift;
    clear_bins(s);
    each_token(x, n, [&](float v, uint32_t i) {
      if (key_of(v) != lo) return;
      atomicAdd(&s.count[i >> shift], 1u);
      atomicAdd((unsigned long long *)&s.mass[i >> shift], (unsigned long long)each);
    });
    __syncthreads();
    find_bin(s, by_count, goal, before_mass, before_count, bin, in_bin, nullptr);
    t_lo = (uint32_t)bin << shift;
    t_hi = t_lo + ((1u << shift) - 1);
  }
  if (t == 0) s.n_list = 0;
  __syncthreads();
  each_token(x, n, [&](float v, uint32_t i) {
    const uint32_t key = key_of(v);
    if (key >= lo && key <= hi && i >= t_lo && i <= t_hi) {
      const uint32_t j = atomicAdd(&s.n_list, 1u);
      if (j < kCap) s.list[j] = place_of(v, i);
    }
  });
  __syncthreads();
  const int m = min((int)s.n_list, kCap);
  sort_list(s, m);
  constexpr int PER = kCap / kWG;
  uint64_t w[PER], mass = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = PER * t + i;
    w[i] = j < m ? r.units(value_of((uint32_t)(s.list[j] >> 32))) : 0;
    mass += w[i];
  }
  uint64_t run = mass;
  uint32_t unused = 0;
  if (t == 0) s.found = 0;
  running(run, unused, s);
  run += before_mass - mass;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = PER * t + i;
    const bool had = by_count ? before_count + (uint64_t)j >= goal : run >= goal;
    run += w[i];
    const bool has = by_count ? before_count + (uint64_t)j + 1 >= goal : run >= goal;
    if (j < m && has && !had) s.found = s.list[j], s.before_mass = run;
  }
  __syncthreads();
  a.place = s.found;
  a.mass = s.before_mass;
  __syncthreads();
  return a;
}

// One workgroup a row.
__global__ void __launch_bounds__(kWG)
    k_sample(const float *__restrict__ logits, int64_t n, const double *__restrict__ u,
             const double *__restrict__ params, int64_t params_ld, int64_t *out, float *logp) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  Shared &s = *reinterpret_cast<Shared *>(lds);
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x;
  const float *x = logits + row * n;
  const double *par = params + row * params_ld;
  float top = -__builtin_inff();
  each_token(x, n, [&](float v, uint32_t) { top = fmaxf(top, v); });
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  if ((t & 63) == 0) s.wave_max[t >> 6] = top;
  __syncthreads();
  for (int w = 0; w < kWG / 64; ++w) top = fmaxf(top, s.wave_max[w]);
  if (top == -__builtin_inff()) {  // nothing to choose from
    if (t == 0) {
      out[row] = -1;
      if (logp) logp[row] = -__builtin_inff();
    }
    return;
  }
  Row r;
  r.top = top;
  const bool greedy = !(par[0] > 0.0);
  r.inv_t = greedy ? 1.0 : 1.0 / par[0];
  r.k = greedy ? 1 : !(par[1] >= 1.0) || par[1] >= (double)n ? 0 : (int64_t)par[1];
  r.p = par[2];
  r.min_p = par[3];
  r.u = u[row] > 0.0 ? fmin(u[row], 0x1.fffffffffffffp-1) : 0.0;
  r.scale = ldexp(1.0, __builtin_clzll((unsigned long long)n) - 2);
  r.inv_bin = (float)(kBins / kSpan * r.inv_t);
  uint64_t total;
  Answer a;
  if (r.k) {
    a = ask(x, n, r, s, true, (uint64_t)r.k);
    total = a.place ? a.mass : a.total;
  } else {
    a = ask(x, n, r, s, true, 1);
    total = a.total;
  }
  if (r.p < 1.0) {
    const double goal = ceil(r.p * (double)total);
    a = ask(x, n, r, s, false, goal > 1.0 ? (uint64_t)goal : 1);
    if (a.place) total = a.mass < total ? a.mass : total;
  }
  if (r.min_p > 0.0) {
    uint64_t mass = 0;
    uint32_t count = 0;
    each_token(x, n, [&](float v, uint32_t) {
      const double w = r.weight(v);
      if (w >= r.min_p) mass += (uint64_t)(w * r.scale + 0.5);
    });
    running(mass, count, s);
    if (t == kWG - 1) s.found = mass;
    __syncthreads();
    const uint64_t kept = s.found;
    __syncthreads();
    const uint64_t first = (uint64_t)(r.scale + 0.5);  // the first token is always kept
    total = kept < total ? kept : total;
    total = total > first ? total : first;
  }
  // u = m 2^-53 of the total, rounded down: below it
  const uint64_t m53 = (uint64_t)(r.u * 0x1p53);
  const uint64_t goal = (__umul64hi(m53, total) << 11 | (m53 * total) >> 53) + 1;
  a = ask(x, n, r, s, false, goal);
  if (t == 0) {
    out[row] = a.place ? (int64_t)(uint32_t)~(uint32_t)a.place : -1;
    if (logp) {
      const float v = value_of((uint32_t)(a.place >> 32));
      logp[row] = (float)((v == top ? 0.0 : ((double)v - (double)top) * r.inv_t) -
                          log((double)total / r.scale));
    }
  }
}

}  // namespace

hipError_t launch_sample(const float *logits, int64_t rows, int64_t n, const double *u,
                         const double *params, int64_t params_ld, int64_t *out, float *logp,
                         hipStream_t s) {
  const int lds = (int)sizeof(Shared);
  hipError_t e = set_dynamic_lds(reinterpret_cast<const void *>(k_sample), lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k_sample, dim3((unsigned)rows), dim3(kWG), lds, s, logits, n, u, params,
                     params_ld, out, logp);
  return hipGetLastError();
}

}  // namespace aq
