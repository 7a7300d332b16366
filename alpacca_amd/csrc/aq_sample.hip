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
// Weights are formed in 64 bits and added as whole multiples of 2^-e of the
// largest, e = 62 - bits of n (45 for a vocabulary of 128 256), so running sums do not
// depend on the order of their terms: the sum of n such roundings is off by 2^-46 n at
// most, 2^-29 of the largest weight, and by about 2^-37 of it in practice.  The sum of a
// whole row without a top-k is one of doubles, the parts', where the row is answered
// from a list that leaves tokens out; it lies as near to the multiples' sum, which is
// taken otherwise.  Which of the two it is goes by the row and its settings alone.  (In
// fp32 a running sum's error of 2^-24 would move every thousandth border between two
// tokens across u.)
//
// Two launches.  k_sample_parts reads the logits once, wide, and leaves the largest
// logit of every 64 tokens and, without a top-k, sums.  k_sample, a workgroup a row,
// finds from these largest a logit tau above which everything asked lies (at least k
// tokens are as large as the k-th largest of them; and a sum that they alone reach
// is reached above the last of them; where they are too few for either, what lies above
// tau is counted or summed before it is used), reads the blocks that reach tau again, and
// answers from the few tokens it finds: one wave sorts up to 64, the workgroup up to
// kWG, up to kCap go into bins.  Rows so flat that more matter are read pass by pass,
// into bins too: of rows of 128256 like a model's with nothing left out 1 in 100 at a
// temperature of 1.0, 1 in 40 at 1.1, 1 in 7 at 1.3; with top-p 0.95 at 1.1 1 in 45, with
// 0.9 at 1.3 3 in 4.
#include <math.h>

#include <type_traits>

#include "aq_internal.h"

namespace aq {
namespace {

constexpr int kWG = 512;
constexpr int kWaves = kWG / 64;
constexpr int kBins = 2048;
constexpr int kCap = 4096;    // tokens of the list
constexpr int kParts = kWG;   // most parts of a row
constexpr int kPartShift = 9;  // 512 tokens a part, more where the row has too many
constexpr int kPart = 1 << kPartShift;
constexpr int kBlocks = 8;  // of a part
constexpr double kSpan = 44;  // exponents that the linear bins cover: e^-44 < 2^-63
constexpr float kNone = -__builtin_inff();

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
__device__ __forceinline__ float logit_of(uint64_t place) {
  return value_of((uint32_t)(place >> 32));
}

// a row's parts: the logarithm of their size, and how many
__host__ __device__ __forceinline__ int part_shift(int64_t n) {
  int shift = kPartShift;
  while ((n - 1) >> shift >= kParts) ++shift;
  return shift;
}
__host__ __device__ __forceinline__ int64_t parts_of(int64_t n) {
  return ((n - 1) >> part_shift(n)) + 1;
}

// e^z for z <= 0 (anything else that is no number: 0) by a table and a polynomial, after
// Tang's method: z = n ln(2) / 64 + r, |r| <= ln(2) / 128, in two steps of which the
// first is exact, and e^z = 2^(n / 64) (1 + (e^r - 1)), e^r - 1 by its series up to
// r^5 / 120 (the next term is below 2^-54).  Off by 2.2e-16 of the value at most;
// table[j] = 2^(j / 64).  Fewer operations than the library's: 64 rows of 128256 logits
// in 16 us of k_sample_parts against 19.
constexpr int kTable = 64;
__device__ __forceinline__ double exp_of(double z, const double *table) {
  z = fmax(z, -1000.0);
  const double n = rint(z * 0x1.71547652b82fep+6);
  double r = fma(n, -0x1.62e42fef00000p-7, z);
  r = fma(n, -0x1.473de6af278edp-40, r);
  double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0) * r;
  const int i = (int)n;
  const double t = table[i & (kTable - 1)];
  return ldexp(fma(t, p, t), i >> 6);
}
__device__ __forceinline__ void fill_table(double *table) {  // (a barrier behind it)
  if (threadIdx.x < kTable) table[threadIdx.x] = exp2((double)threadIdx.x / kTable);
}

// e^((x - top) / T); of an infinite top, and of -infinity, nothing is left
__device__ __forceinline__ double weight_of(float x, float top, double inv_t,
                                            const double *table) {
  const double w = exp_of(((double)x - (double)top) * inv_t, table);
  return x == top ? 1.0 : w;
}

struct Row {
  const double *table;
  float top;           // the largest logit
  double temp, inv_t;  // the temperature (greedy: 1) and 1 / it
  double scale;  // units of the sums
  double p, min_p, u;
  int64_t k;      // 0: no top-k
  float inv_bin;  // linear bins per logit
  uint32_t last;  // the highest token
  // weight of a logit, and in units
  __device__ __forceinline__ double weight(float x) const {
    return weight_of(x, top, inv_t, table);
  }
  __device__ __forceinline__ uint64_t units(double w) const { return (uint64_t)(w * scale + 0.5); }
  __device__ __forceinline__ uint64_t units(float x) const { return units(weight(x)); }
  // the sum that top-p reaches; the one that the token's exceeds u times
  __device__ __forceinline__ uint64_t share(uint64_t total) const {
    const double goal = ceil(p * (double)total);
    return goal > 1.0 ? (uint64_t)goal : 1;
  }
  __device__ __forceinline__ uint64_t goal(uint64_t total) const {
    const uint64_t m53 = (uint64_t)(u * 0x1p53);  // rounded down: below total
    return (__umul64hi(m53, total) << 11 | (m53 * total) >> 53) + 1;
  }
  // the linear bin, and its bin of bins: no larger for a larger logit
  __device__ __forceinline__ float line(float x) const {
    return x == top ? 0.f : fminf((top - x) * inv_bin, (float)(kBins - 1));
  }
  __device__ __forceinline__ int bin(float x) const { return (int)line(x); }
  __device__ __forceinline__ int sub_bin(float x) const {
    const float y = line(x);
    return (int)fminf((y - truncf(y)) * kBins, (float)(kBins - 1));
  }
};

struct Bins {
  uint64_t mass[kBins];
  uint32_t count[kBins];
};
struct Shared {
  double table[kTable];
  uint64_t list[kCap];
  uint64_t few[64];
  Bins coarse, fine;
  uint16_t block[kParts * kBlocks];  // those that reach tau
  double sum[kWaves];
  uint64_t wave_mass[kWaves];
  float wave_max[kWaves], wave_min[kWaves];
  uint64_t place, total, mass, count, all_mass;
  uint32_t bin, in_bin, n_list, key_lo, key_hi;
};

// Tokens at .. at + 3 of a row of n >= 4, without a branch: v[e] is the logit of token
// first + e, -infinity where that is below `at` (the quad is moved inside the row) or
// NaN.
struct Quad {
  f4u v;
  int64_t first;
};
__device__ __forceinline__ Quad load_quad(const float *x, int64_t at, int64_t n) {
  Quad q;
  q.first = at < n - 4 ? at : n - 4;
  q.v = *reinterpret_cast<const f4u *>(x + q.first);
  return q;
}
__device__ __forceinline__ void mask_quad(Quad &q, int64_t at) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    q.v[e] = q.first + e >= at && q.v[e] == q.v[e] ? q.v[e] : kNone;
}

// Every token above -infinity: f(x, token).  Eight loads a thread are under way.
template <class F>
__device__ __forceinline__ void each_token(const float *x, int64_t n, F &&f) {
  constexpr int U = 8;
  if (n < 4) {
    if (threadIdx.x < n && x[threadIdx.x] > kNone) f(x[threadIdx.x], threadIdx.x);
    return;
  }
  for (int64_t c = 0; c < n; c += 4 * kWG * U) {
    Quad q[U];
#pragma unroll
    for (int i = 0; i < U; ++i) q[i] = load_quad(x, c + 4 * (kWG * i + (int)threadIdx.x), n);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      mask_quad(q[i], c + 4 * (kWG * i + (int)threadIdx.x));
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (q[i].v[e] > kNone) f(q[i].v[e], (uint32_t)(q[i].first + e));
    }
  }
}

// v of lane l ^ STEP, without LDS (lane permutations of gfx9's data-parallel
// moves: xor 1, 2, 3, 7 and 15; gfx950's row swaps for 16 and 32)
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ uint32_t dppu(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int STEP>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  if constexpr (STEP == 1) return dppu<0xB1>(v);
  else if constexpr (STEP == 2) return dppu<0x4E>(v);
  else if constexpr (STEP == 4) return dppu<0x1B>(dppu<0x141>(v));
  else if constexpr (STEP == 8) return dppu<0x141>(dppu<0x140>(v));
  else {
    const auto r = STEP == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false)
                              : __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & STEP ? r[0] : r[1];
  }
}
template <int STEP>
__device__ __forceinline__ uint64_t lane_xor64(uint64_t v) {
  return (uint64_t)lane_xor<STEP>((uint32_t)(v >> 32)) << 32 | lane_xor<STEP>((uint32_t)v);
}
// the same for all sizes of values
template <int STEP>
__device__ __forceinline__ float lane_xor(float v) {
  return __uint_as_float(lane_xor<STEP>(__float_as_uint(v)));
}
template <int STEP>
__device__ __forceinline__ double lane_xor(double v) {
  return __builtin_bit_cast(double, lane_xor64<STEP>(__builtin_bit_cast(uint64_t, v)));
}
// op over lanes l ^ 1 .. l ^ (SIZE - 1), in every lane
template <int SIZE, typename T, class Op>
__device__ __forceinline__ T over_lanes(T v, Op op) {
  v = op(v, lane_xor<1>(v));
  if constexpr (SIZE > 2) v = op(v, lane_xor<2>(v));
  if constexpr (SIZE > 4) v = op(v, lane_xor<4>(v));
  if constexpr (SIZE > 8) v = op(v, lane_xor<8>(v));
  if constexpr (SIZE > 16) v = op(v, lane_xor<16>(v));
  if constexpr (SIZE > 32) v = op(v, lane_xor<32>(v));
  return v;
}
struct Max {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Min {
  __device__ __forceinline__ float operator()(float a, float b) const { return fminf(a, b); }
  __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const {
    return a < b ? a : b;
  }
};
struct Add {
  __device__ __forceinline__ double operator()(double a, double b) const { return a + b; }
};
// v of a lane that is the same for the whole wave
__device__ __forceinline__ uint64_t of_lane(uint64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), lane);
  return (uint64_t)hi << 32 | lo;
}

// inclusive running sums, a thread's own first: over the wave, over the workgroup
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return dppu<CTRL, ROWS>(v);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t moved(uint64_t v) {
  return (uint64_t)dppu<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | dppu<CTRL, ROWS>((uint32_t)v);
}
template <typename T>
__device__ __forceinline__ T running_wave(T v) {
  v += moved<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8 (0 enters a row of 16)
  v += moved<0x112, 0xF>(v);
  v += moved<0x114, 0xF>(v);
  v += moved<0x118, 0xF>(v);
  v += moved<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  v += moved<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ uint64_t running(uint64_t mass, Shared &s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  mass = running_wave(mass);
  if (lane == 63) s.wave_mass[wave] = mass;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) mass += w < wave ? s.wave_mass[w] : 0;
  __syncthreads();
  return mass;
}

// ---- the sorted list ---------------------------------------------------------------

template <int SIZE, int STEP>
__device__ __forceinline__ void sort_steps(uint64_t &v) {
  const int t = threadIdx.x & 63;
  const uint64_t y = lane_xor64<STEP>(v);
  const bool larger = ((t & STEP) == 0) == ((t & SIZE) == 0);
  v = larger == (v > y) ? v : y;
  if constexpr (STEP > 1) sort_steps<SIZE, STEP / 2>(v);
}
// one value a lane, in descending order over the wave
template <int SIZE = 2>
__device__ __forceinline__ void sort_wave(uint64_t &v) {
  sort_steps<SIZE, SIZE / 2>(v);
  if constexpr (SIZE < 64) sort_wave<2 * SIZE>(v);
}

// ---- a beginning of the order ------------------------------------------------------
//
// decide() asks for tokens of a beginning of the order that is held in a wave's
// lanes (WaveOrder), or by bins over a list in LDS or over the whole row (BinOrder):
//   ask(by_count, goal): the first token up to which the count (by_count) or the sum
//     reaches the goal (place 0: none), and the sum up to and with it
//   all(): the sum of all
//   heavier(w): the sum of those that weigh at least w

struct Answer {
  uint64_t place;  // 0: no token
  uint64_t sum;
};

template <int E>
struct WaveOrder {
  int m;  // tokens: lane l has the places l, l + 64, ..
  uint64_t v[E], sum[E];
  double w[E];
  __device__ __forceinline__ uint64_t at(const uint64_t (&x)[E], int i) const {
    uint64_t y = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) y = i / 64 == e ? x[e] : y;
    return of_lane(y, i % 64);
  }
  __device__ __forceinline__ uint64_t all() const { return at(sum, m - 1); }
  __device__ __forceinline__ Answer ask(const Row &, bool by_count, uint64_t goal) const {
    int i = 0;  // (places past m hold the last sum)
#pragma unroll
    for (int e = 0; e < E; ++e) i += __popcll(__ballot(sum[e] < goal));
    if (by_count) i = (int)goal - 1;
    if (i >= m) return {0, 0};
    return {at(v, i), at(sum, i)};
  }
  __device__ __forceinline__ uint64_t heavier(const Row &, double least) const {
    int n = 0;
#pragma unroll
    for (int e = 0; e < E; ++e)
      n += __popcll(__ballot(64 * e + (int)(threadIdx.x & 63) < m && w[e] >= least));
    return n ? at(sum, n - 1) : 0;
  }
};
// list[0 .. m), at most 64 tokens, sorted: the calling wave's
__device__ __forceinline__ WaveOrder<1> wave_order(const uint64_t *list, int m, const Row &r) {
  const int lane = threadIdx.x & 63;
  uint64_t v = lane < m ? list[lane] : 0;
  sort_wave(v);
  const double w = r.weight(logit_of(v));
  return {m, {v}, {running_wave<uint64_t>(lane < m ? r.units(w) : 0)}, {w}};
}
// How many of RUNS sorted runs of 64 places are larger than v, by halving.
template <int RUNS>
__device__ __forceinline__ int larger_than(const uint64_t *runs, uint64_t v) {
  int at[RUNS] = {}, all = 0;
#pragma unroll
  for (int step = 32; step > 0; step /= 2) {
    uint64_t y[RUNS];
#pragma unroll
    for (int w = 0; w < RUNS; ++w) y[w] = runs[64 * w + at[w] + step - 1];
#pragma unroll
    for (int w = 0; w < RUNS; ++w) at[w] += y[w] > v ? step : 0;
  }
#pragma unroll
  for (int w = 0; w < RUNS; ++w) all += at[w] + (runs[64 * w + at[w]] > v ? 1 : 0);
  return all;
}
// s.list[0 .. m), at most kWG tokens, sorted by the whole workgroup: a wave sorts 64 of
// them, and a token's place is how many of each wave's are larger.  The order lies in
// s.coarse, from where the calling wave has it.
struct Sorted {
  uint64_t runs[kWG], place[kWG], sum[kWG];
  double weight[kWG];
};
__device__ __forceinline__ WaveOrder<kWaves> sorted_order(int m, const Shared &s) {
  const Sorted &o = reinterpret_cast<const Sorted &>(s.coarse);
  WaveOrder<kWaves> w;
  w.m = m;
#pragma unroll
  for (int e = 0; e < kWaves; ++e) {
    const int i = 64 * e + (threadIdx.x & 63);
    w.v[e] = o.place[i], w.sum[e] = o.sum[i], w.w[e] = o.weight[i];
  }
  return w;
}
__device__ __forceinline__ void sort_list(int m, const Row &r, Shared &s) {
  const int t = threadIdx.x;
  Sorted &o = reinterpret_cast<Sorted &>(s.coarse);
  static_assert(sizeof(Sorted) <= sizeof(Bins) && kWaves == 8, "");
  uint64_t v = t < m ? s.list[t] : 0;
  sort_wave(v);
  o.runs[t] = v;
  o.place[t] = 0;
  __syncthreads();
  if (v)
    o.place[m <= 128   ? larger_than<2>(o.runs, v)
            : m <= 256 ? larger_than<4>(o.runs, v)
                       : larger_than<8>(o.runs, v)] = v;
  __syncthreads();
  v = o.place[t];
  const double weight = r.weight(logit_of(v));
  o.sum[t] = running(t < m ? r.units(weight) : 0, s);
  o.weight[t] = weight;
  __syncthreads();
}

// The answer from the m first tokens of the order.  total: of the whole row (without
// a top-k) on entry, of what is kept on return.  whole: there are no more tokens;
// to_min_p: what min-p keeps is among them.  With a top-k of k they are at least k, or
// the whole row, or hold what min-p keeps of a row without top-p.  0: they end too
// early.
template <class Order>
__device__ __forceinline__ uint64_t decide(const Order &order, const Row &r, int64_t m, bool whole,
                                           bool to_min_p, uint64_t &total) {
  bool open = false;  // what is kept may end behind them
#pragma unroll 1
  for (int step = 0;; ++step) {  // top-k, top-p, min-p and the token (one place that asks)
    bool by_count = false;
    uint64_t goal;
    if (step == 0) {
      if (r.k ? r.k >= m : whole) total = order.all();
      open = !r.k && !whole;
      if (!r.k || r.k >= m) continue;
      by_count = true;
      goal = (uint64_t)r.k;
    } else if (step == 1) {
      if (!(r.p < 1.0)) continue;
      goal = r.share(total);
    } else {
      if (r.min_p > 0.0 && (!open || to_min_p)) {
        const uint64_t first = r.units(1.0);  // the first token is always kept
        uint64_t kept = order.heavier(r, r.min_p);
        kept = kept > first ? kept : first;
        total = open || kept < total ? kept : total;
      }
      goal = r.goal(total);
    }
    const Answer a = order.ask(r, by_count, goal);
    if (step == 2) return a.place;
    if (step == 0) {
      total = a.place ? a.sum : order.all();
    } else if (a.place) {
      total = a.sum < total ? a.sum : total;
      open = false;
    } else if (open && !to_min_p) {
      return 0;
    }
  }
}

// ---- bins --------------------------------------------------------------------------

// Where a BinOrder's tokens are: each(f) calls f(logit, token) for all of them.
struct RowTokens {
  const float *x;
  int64_t n;
  template <class F>
  __device__ __forceinline__ void each(F &&f) const { each_token(x, n, f); }
};
struct ListTokens {
  const uint64_t *list;
  int64_t n;
  template <class F>
  __device__ __forceinline__ void each(F &&f) const {
    for (int i = threadIdx.x; i < n; i += kWG) f(logit_of(list[i]), (uint32_t)~(uint32_t)list[i]);
  }
};

struct Before {  // of a bin
  uint64_t sum, count;
};

// The bin where the count (by_count) or the sum reaches the goal, what lies before
// it (its count only if asked for, its sum then if both are), and how many tokens it
// holds.  kBins: none.
__device__ __forceinline__ int find_bin(const Bins &b, Shared &s, bool by_count, uint64_t goal,
                                        Before &before, uint32_t &in_bin, bool both = true) {
  constexpr int PER = kBins / kWG;
  const int t = threadIdx.x;
  uint64_t masses[PER], mass = 0, count = 0;
  uint32_t counts[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) masses[i] = b.mass[PER * t + i], counts[i] = b.count[PER * t + i];
#pragma unroll
  for (int i = 0; i < PER; ++i) mass += masses[i], count += counts[i];
  if (t == 0) s.bin = kBins;  // (running's barriers follow)
  uint64_t m = !by_count || both ? running(mass, s) - mass + before.sum : 0;
  uint64_t c = by_count ? running(count, s) - count + before.count : 0;
  if (t == kWG - 1) s.all_mass = m + mass;
  if ((by_count ? c : m) < goal && (by_count ? c + count : m + mass) >= goal) {
    bool found = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (!found && (by_count ? c + counts[i] : m + masses[i]) >= goal)
        found = true, s.bin = PER * t + i, s.mass = m, s.count = c, s.in_bin = counts[i];
      m += masses[i], c += counts[i];
    }
  }
  __syncthreads();
  const int bin = (int)s.bin;
  if (bin < kBins) before = {s.mass, s.count}, in_bin = s.in_bin;
  __syncthreads();
  return bin;
}

// the tokens that `has` into bins by `bin_of`
template <class Tokens, class H, class B>
__device__ __forceinline__ void fill_bins(Bins &b, const Tokens &tokens, const Row &r, H &&has,
                                          B &&bin_of) {
  for (int i = threadIdx.x; i < kBins; i += kWG) b.mass[i] = 0, b.count[i] = 0;
  __syncthreads();
  tokens.each([&](float v, uint32_t i) {
    if (!has(v, i)) return;
    const int j = bin_of(v, i);
    atomicAdd(&b.count[j], 1u);
    atomicAdd((unsigned long long *)&b.mass[j], (unsigned long long)r.units(v));
  });
  __syncthreads();
}
// those that `has` into s.few (or as many as fit); how many they are
template <class Tokens, class H>
__device__ __forceinline__ int pick(uint64_t *list, int room, const Tokens &tokens, Shared &s,
                                    H &&has) {
  if (threadIdx.x == 0) s.n_list = 0;
  __syncthreads();
  tokens.each([&](float v, uint32_t i) {
    if (!has(v, i)) return;
    const uint32_t j = atomicAdd(&s.n_list, 1u);
    if ((int)j < room) list[j] = place_of(v, i);
  });
  __syncthreads();
  const int m = (int)s.n_list;
  __syncthreads();
  return m;
}

// Tokens in the linear bins of s.coarse.  A bin of more than 64 tokens is parted into
// finer ones, by logit, by its keys and, where they are all equal, by the tokens'
// numbers.
template <class Tokens>
struct BinOrder {
  const Tokens &tokens;
  Shared &s;
  __device__ __forceinline__ void fill(const Row &r) const {
    fill_bins(s.coarse, tokens, r, [](float, uint32_t) { return true; },
              [&](float v, uint32_t) { return r.bin(v); });
  }
  __device__ __forceinline__ uint64_t all() const {
    uint64_t mass = 0;
    for (int i = threadIdx.x; i < kBins; i += kWG) mass += s.coarse.mass[i];
    return sum_of(mass);
  }
  __device__ __forceinline__ uint64_t sum_of(uint64_t mass) const {
    mass = running(mass, s);
    if (threadIdx.x == kWG - 1) s.total = mass;
    __syncthreads();
    mass = s.total;
    __syncthreads();
    return mass;
  }
  __device__ __forceinline__ uint64_t heavier(const Row &r, double least) const {
    uint64_t kept = 0;
    tokens.each([&](float v, uint32_t) {
      const double w = r.weight(v);
      if (w >= least) kept += r.units(w);
    });
    return sum_of(kept);
  }
  __device__ __forceinline__ Answer ask(const Row &r, bool by_count, uint64_t goal) const {
    Before before = {0, 0};
    uint32_t in_bin = 0;
    const int bin = find_bin(s.coarse, s, by_count, goal, before, in_bin);
    if (bin == kBins) return {0, 0};
    return narrow(tokens, r, bin, by_count, goal, before, in_bin);
  }
  // the answer among the in_bin tokens of a coarse bin
  template <class From>
  __device__ __forceinline__ Answer narrow(const From &from, const Row &r, int bin, bool by_count,
                                           uint64_t goal, Before before, uint32_t in_bin) const {
    constexpr bool row = std::is_same<From, RowTokens>::value;
    constexpr uint32_t kRest = row ? kCap : 64;
    int fine = -1;
    uint32_t lo = 0, hi = 0xFFFFFFFFu, t_lo = 0, t_hi = 0xFFFFFFFFu;
    auto has = [&](float v, uint32_t i) {
      if (r.bin(v) != bin || (fine >= 0 && r.sub_bin(v) != fine)) return false;
      const uint32_t key = key_of(v);
      return key >= lo && key <= hi && i >= t_lo && i <= t_hi;
    };
    if (in_bin > kRest) {
      fill_bins(s.fine, from, r, has, [&](float v, uint32_t) { return r.sub_bin(v); });
      fine = find_bin(s.fine, s, by_count, goal, before, in_bin);
    }
    if (in_bin > kRest) {  // bins of equal ranges of keys, descending
      if (threadIdx.x == 0) s.key_lo = 0xFFFFFFFFu, s.key_hi = 0;
      __syncthreads();
      from.each([&](float v, uint32_t i) {
        if (has(v, i)) atomicMin(&s.key_lo, key_of(v)), atomicMax(&s.key_hi, key_of(v));
      });
      __syncthreads();
      lo = s.key_lo, hi = s.key_hi;
      __syncthreads();
    }
    while (in_bin > kRest && lo < hi) {
      int shift = 0;
      while (((hi - lo) >> shift) >= kBins) ++shift;
      fill_bins(s.fine, from, r, has,
                [&](float v, uint32_t) { return (int)((hi - key_of(v)) >> shift); });
      hi -= (uint32_t)find_bin(s.fine, s, by_count, goal, before, in_bin) << shift;
      const uint32_t width = (1u << shift) - 1;
      lo = hi - lo > width ? hi - width : lo;
    }
    if (in_bin > kRest) t_hi = r.last;
    // of equal logits the lowest tokens first (one token always ends it, also where
    // another stream writes the logits meanwhile)
    while (in_bin > kRest && t_lo < t_hi) {
      int shift = 0;
      while (((t_hi - t_lo) >> shift) >= kBins) ++shift;
      fill_bins(s.fine, from, r, has,
                [&](float, uint32_t i) { return (int)((i - t_lo) >> shift); });
      t_lo += (uint32_t)find_bin(s.fine, s, by_count, goal, before, in_bin) << shift;
      const uint32_t width = (1u << shift) - 1;
      t_hi = t_hi - t_lo > width ? t_lo + width : t_hi;
    }
    if constexpr (row) {  // the rest from the list
      const ListTokens list = {s.list, min(pick(s.list, kCap, from, s, has), kCap)};
      return narrow(list, r, bin, by_count, goal, before, in_bin);
    }
    const int m = min(pick(s.few, 64, from, s, has), 64);
    if (threadIdx.x < 64) {
      const Answer a = wave_order(s.few, m, r)
                           .ask(r, by_count, goal - (by_count ? before.count : before.sum));
      if (threadIdx.x == 0) s.place = a.place, s.mass = a.sum + before.sum;
    }
    __syncthreads();
    const Answer a = {s.place, s.mass};
    __syncthreads();
    return a;
  }
};

// ---- few tokens --------------------------------------------------------------------

// All tokens >= tau into the list, from the `reach` blocks that have any (s.block); the
// list's length may pass kCap, its content does not.  First the numbers of the quads
// that have any (they lie in s.coarse), up to kQuads of a thread's under way; then, a
// thread each, their tokens: looking at every element of every quad instead took 5 us for
// 286 blocks, this 3.4.  Where a thread has two quads at most they are all looked at.
__device__ __forceinline__ int gather(const float *x, int64_t n, float tau, int reach, Shared &s) {
  constexpr int kQuads = 12;
  const int t = threadIdx.x, lane = t & 63;
  // a place in s.n_list's count for each of a lane's `mine`
  auto places = [&](uint32_t mine) {
    const uint32_t sum = running_wave(mine);
    uint32_t base = 0;
    if (lane == 63) base = atomicAdd(&s.n_list, sum);
    return sum - mine + __builtin_amdgcn_readlane(base, 63);
  };
  auto listed = [&] {
    __syncthreads();
    const int m = (int)s.n_list;
    __syncthreads();
    return m;
  };
  if (t == 0) s.n_list = 0;
  __syncthreads();
  if (n < 4) {
    if (t < n && x[t] >= tau) s.list[atomicAdd(&s.n_list, 1u)] = place_of(x[t], t);
    return listed();
  }
  uint32_t *hits = reinterpret_cast<uint32_t *>(s.coarse.mass);
  static_assert(sizeof(s.coarse.mass) >= kCap * sizeof(uint32_t), "");
  const int shift = part_shift(n) - 3 - 2;  // quads of a block
  const uint32_t quads = (uint32_t)reach << shift, end = (uint32_t)((n + 3) / 4);
  auto quad_of = [&](uint32_t j) {
    return j < quads ? (uint32_t)s.block[j >> shift] << shift | (j & ((1u << shift) - 1)) : end;
  };
  const bool all = quads <= 2 * kWG;
  for (uint32_t c = 0; c < quads && !all; c += kWG * kQuads) {
    f4u v[kQuads];
    uint32_t quad[kQuads];
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      if (c + kWG * i >= quads) continue;
      quad[i] = quad_of(c + kWG * i + t);
      const int64_t at = 4 * (int64_t)quad[i];
      v[i] = *reinterpret_cast<const f4u *>(x + (at < n - 4 ? at : n - 4));
    }
    uint32_t has = 0;
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      if (c + kWG * i >= quads) continue;
      const float top = fmaxf(fmaxf(v[i][0], v[i][1]), fmaxf(v[i][2], v[i][3]));
      if (top >= tau && quad[i] < end) has |= 1u << i;
    }
    if (!__any(has)) continue;
    uint32_t j = places(__popc(has));
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      if (c + kWG * i >= quads) continue;
      if (has >> i & 1) {
        if (j < kCap) hits[j] = quad[i];
        ++j;
      }
    }
  }
  const int m = all ? (int)quads : listed();
  if (m > kCap) return m;
  if (!all) {
    if (t == 0) s.n_list = 0;
    __syncthreads();
  }
  for (int c = 0; c < m; c += 2 * kWG) {
    int64_t first[2], at[2];
    f4u v[2];
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = c + kWG * i + t;
      first[i] = 4 * (int64_t)(j >= m ? end : all ? quad_of(j) : hits[j]);
      at[i] = first[i] < n - 4 ? first[i] : n - 4;  // (the last quad is moved inside)
      if (c + kWG * i < m) v[i] = *reinterpret_cast<const f4u *>(x + at[i]);
    }
    auto is = [&](int i, int e) { return (v[i][e] >= tau) & (at[i] + e >= first[i]); };
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (c + kWG * i < m)
#pragma unroll
        for (int e = 0; e < 4; ++e) mine += is(i, e) ? 1u : 0u;
    uint32_t j = places(mine);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (c + kWG * i < m)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (is(i, e)) {
            if (j < kCap) s.list[j] = place_of(v[i][e], (uint32_t)(at[i] + e));
            ++j;
          }
  }
  return listed();
}

// tops: the blocks' largest logits, low the smallest of them.  false: the row's answer
// takes more tokens than a list holds.
__device__ __forceinline__ bool choose_few(const float *x, int64_t n, const Row &r, Shared &s,
                                           uint64_t whole_sum, const float (&tops)[kBlocks],
                                           float low, uint64_t &place, uint64_t &total) {
  const int t = threadIdx.x;
  float floor_ = kNone;  // what min-p keeps is at least this
  if (r.min_p > 0.0) {
    // from the largest logit down, with room for the weights' rounding and floor_'s
    const double below = (fmin(log(r.min_p), 0.0) - 1e-9) * r.temp;
    floor_ = r.top == __builtin_inff()
                 ? r.top
                 : (float)((double)r.top + below - 1e-6 * (fabs((double)r.top) - below));
  }
  float tau = low;
  if (r.k || r.p < 1.0 || !(r.min_p > 0.0)) {
    // the blocks' largest in bins over their range, and of the one where they reach
    // what is asked (or of the last) the smallest
    Row br = r;
    br.inv_bin = (float)kBins / (r.top - low);
    uint32_t key = 0xFFFFFFFFu;
    for (int i = t; i < kBins; i += kWG) s.coarse.mass[i] = 0, s.coarse.count[i] = 0;
    if (t == 0) s.key_lo = 0xFFFFFFFFu;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      if (!(tops[i] > kNone)) continue;
      const int b = br.bin(tops[i]);
      atomicAdd(&s.coarse.count[b], 1u);
      if (!r.k)
        atomicAdd((unsigned long long *)&s.coarse.mass[b], (unsigned long long)r.units(tops[i]));
    }
    __syncthreads();
    uint64_t goal = r.k ? (uint64_t)r.k : r.p < 1.0 ? r.share(whole_sum) : r.goal(whole_sum);
    int last;
    for (;;) {
      Before before = {0, 0};
      uint32_t in_bin;
      last = find_bin(s.coarse, s, r.k != 0, goal, before, in_bin, false);
      // Where they alone do not reach the sum, but half of it: so much of theirs that an
      // eighth is left out of what the sum leaves out, a guess (two heavy tokens may share a
      // block) that decide() turns down if the list ends too early.  Without it such a
      // row is read pass by pass: one in 1500 of rows like a model's at a temperature of
      // 0.9 with top-p 0.9, 130 us.
      if (last < kBins || r.k || s.all_mass < goal / 2) break;
      const double left = 0.125 * (1.0 - (double)goal / (double)whole_sum);
      goal = (uint64_t)((double)s.all_mass * (1.0 - left));
      goal = goal < 1 ? 1 : goal < s.all_mass ? goal : s.all_mass;
    }
    if (last < kBins) {
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
        if (tops[i] > kNone && br.bin(tops[i]) <= last) key = min(key, key_of(tops[i]));
      key = over_lanes<64>(key, Min());
      if ((t & 63) == 0) atomicMin(&s.key_lo, key);
      __syncthreads();
      tau = value_of(s.key_lo);
    }
  } else {
    tau = floor_;
  }
  if (floor_ >= tau && !(r.k && r.p < 1.0)) tau = floor_;
  constexpr float kLowest = -3.402823466e38f;
  const bool to_min_p = floor_ >= tau;
  tau = fmaxf(tau, kLowest);
  bool whole;
  int m;
  for (;;) {
    whole = tau == kLowest;
    // the blocks that reach tau, in no order
    if (t == 0) s.n_list = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBlocks; ++i)
      if (tops[i] >= tau) s.block[atomicAdd(&s.n_list, 1u)] = (uint16_t)(i * kWG + t);
    __syncthreads();
    const int reach = (int)s.n_list;
    __syncthreads();
    m = gather(x, n, tau, reach, s);
    if (m > kCap) return false;
    // Fewer blocks than k have anything: tau is the smallest of their largest, and k
    // tokens need not reach it.  top-p's share is of all k, whatever min-p keeps, so a
    // list short of them is made of all tokens (once: it is whole then).
    if (whole || !r.k || m >= r.k || (to_min_p && !(r.p < 1.0))) break;
    tau = kLowest;
  }
  total = whole_sum;
  if (m <= kWG) {
    if (m > 64) sort_list(m, r, s);
    if (t < 64) {
      const uint64_t p = m > 64 ? decide(sorted_order(m, s), r, m, whole, to_min_p, total)
                                : decide(wave_order(s.list, m, r), r, m, whole, to_min_p, total);
      if (t == 0) s.place = p, s.total = total;
    }
    __syncthreads();
    place = s.place;
    total = s.total;
    __syncthreads();
  } else {
    Row lr = r;  // bins over the list's range, where it has an end
    if (!whole) lr.inv_bin = (float)kBins / (r.top - tau);
    const ListTokens tokens = {s.list, m};
    const BinOrder<ListTokens> order = {tokens, s};
    order.fill(lr);
    place = decide(order, lr, m, whole, to_min_p, total);
  }
  return place != 0;
}

// ---- kernels -----------------------------------------------------------------------

// A wave a part: the largest logits of its blocks and, where the row has no top-k, the
// sum of its weights relative to its largest logit.  One row of 128256 in 3.9 us (a
// launch's start and a chain of loads); 64 rows 16, bound by the vector instructions
// (of the exponentials a third); with a top-k, which needs no sums, 10.5 (3.1 TB/s).
// Several parts a wave, the next one's loads under way, 17 to 21.
__global__ void __launch_bounds__(256)
    k_sample_parts(const float *__restrict__ logits, int64_t n, const double *__restrict__ params,
                   int64_t params_ld, double *__restrict__ sums, float *__restrict__ part_tops,
                   float *__restrict__ tops) {
  __shared__ double table[kTable];
  const int lane = threadIdx.x & 63;
  const int more = part_shift(n) - kPartShift;  // a block is 64 << more tokens
  const int64_t row = blockIdx.y, parts = parts_of(n);
  const int64_t part = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const float *x = logits + row * n;
  Quad q[2];
  auto load = [&](int64_t c) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int64_t at = c + 256 * g + 4 * lane;
      if (n >= 4) {
        q[g] = load_quad(x, at, n);
      } else {
        q[g].first = at;
#pragma unroll
        for (int e = 0; e < 4; ++e) q[g].v[e] = at + e < n ? x[at + e] : kNone;
      }
    }
  };
  const int64_t first = part * ((int64_t)kPart << more), last = first + ((int64_t)kPart << more);
  if (part < parts) load(first);
  const double *par = params + row * params_ld;
  const bool sum_all = par[0] > 0.0 && !(par[1] >= 1.0 && par[1] < (double)n);
  const double inv_t = 1.0 / par[0];
  fill_table(table);
  __syncthreads();
  float top = kNone, block = kNone;
  double sum = 0.0;
  if (part >= parts) return;
  tops += (row * parts + part) * kBlocks;
  int step = 0;
  for (int64_t c = first; c < last; c += kPart, ++step) {
    float v[8];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      mask_quad(q[g], c + 256 * g + 4 * lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * g + e] = q[g].v[e];
    }
    if (c + kPart < last) load(c + kPart);
    // 64 tokens are 16 lanes' four
    float m[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      m[g] = fmaxf(fmaxf(v[4 * g], v[4 * g + 1]), fmaxf(v[4 * g + 2], v[4 * g + 3]));
      m[g] = over_lanes<16>(m[g], Max());
      const float two = fmaxf(m[g], lane_xor<16>(m[g])), four = fmaxf(two, lane_xor<32>(two));
      if (more <= 2 && (lane & ((16 << more) - 1)) == 0)
        tops[(8 * step + 4 * g + (lane >> 4)) >> more] = more == 0 ? m[g] : more == 1 ? two : four;
      m[g] = four;
    }
    const float all = fmaxf(m[0], m[1]);
    if (more > 2) {
      block = fmaxf(block, all);
      if (((step + 1) & ((1 << (more - 3)) - 1)) == 0) {
        if (lane == 0) tops[step >> (more - 3)] = block;
        block = kNone;
      }
    }
    const float next = fmaxf(top, all);
    if (sum_all && next > kNone) {
      if (next != top) sum = top > kNone ? sum * weight_of(top, next, inv_t, table) : 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += weight_of(v[e], next, inv_t, table);
    }
    top = next;
  }
  if (sum_all) sum = over_lanes<64>(sum, Add());
  if (lane == 0) {
    part_tops[row * parts + part] = top;
    sums[row * parts + part] = sum;
  }
}

// One workgroup a row.  A chain of short steps, so bound by their latency and not by
// bytes (the launch's start and the parts' results 2 us, tau 3, the blocks that reach it
// 1.5 to 3.5, the list's order 2 to 4, the answer 2): one row of 128256 9.6 us, 64 of
// them with a top-k of 40 and top-p 10, with top-p 0.9 alone, lists of up to 418 tokens,
// 15.9 (19.2 with such lists in bins); 64 of 2145 with a top-k of 309, top-p and min-p, most
// of them listed a second time and whole, 21.  A row that is read pass by pass takes 110 to
// 160, and so does its batch.
__global__ void __launch_bounds__(kWG)
    k_sample(const float *__restrict__ logits, int64_t n, const double *__restrict__ u,
             const double *__restrict__ params, int64_t params_ld, const double *__restrict__ sums,
             const float *__restrict__ part_tops, const float *__restrict__ block_tops,
             int64_t *out, float *logp) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  Shared &s = *reinterpret_cast<Shared *>(lds);
  const int64_t row = blockIdx.x, parts = parts_of(n);
  const int t = threadIdx.x;
  const float *x = logits + row * n;
  const double *par = params + row * params_ld;
  const double par0 = par[0], par1 = par[1], par2 = par[2], par3 = par[3], u_row = u[row];
  fill_table(s.table);
  float tops[kBlocks], top = kNone, low = __builtin_inff();
#pragma unroll
  for (int i = 0; i < kBlocks; ++i) {
    const int64_t j = i * kWG + t;
    tops[i] = kNone;
    if (j < parts * kBlocks) tops[i] = block_tops[row * parts * kBlocks + j];
  }
  const float part_top = t < parts ? part_tops[row * parts + t] : kNone;
  const double part_sum = t < parts ? sums[row * parts + t] : 0.0;
#pragma unroll
  for (int i = 0; i < kBlocks; ++i) {
    top = fmaxf(top, tops[i]);
    low = fminf(low, tops[i] > kNone ? tops[i] : low);
  }
  top = over_lanes<64>(top, Max());
  low = over_lanes<64>(low, Min());
  if ((t & 63) == 0) s.wave_max[t >> 6] = top, s.wave_min[t >> 6] = low;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w)
    top = fmaxf(top, s.wave_max[w]), low = fminf(low, s.wave_min[w]);
  if (top == kNone) {  // nothing to choose from
    if (t == 0) {
      out[row] = -1;
      if (logp) logp[row] = kNone;
    }
    return;
  }
  Row r;
  r.table = s.table;
  r.top = top;
  const bool greedy = !(par0 > 0.0);
  r.temp = greedy ? 1.0 : par0;
  r.inv_t = 1.0 / r.temp;
  r.k = greedy ? 1 : !(par1 >= 1.0) || par1 >= (double)n ? 0 : (int64_t)par1;
  r.last = (uint32_t)(n - 1);
  r.p = par2;
  r.min_p = par3;
  r.u = u_row > 0.0 ? fmin(u_row, 0x1.fffffffffffffp-1) : 0.0;
  r.scale = ldexp(1.0, __builtin_clzll((unsigned long long)n) - 2);
  r.inv_bin = (float)(kBins / kSpan * r.inv_t);
  uint64_t whole_sum = 0;
  if (!r.k) {  // of all weights
    double sum = t < parts ? part_sum * r.weight(part_top) : 0.0;
    sum = over_lanes<64>(sum, Add());
    if ((t & 63) == 0) s.sum[t >> 6] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < kWaves; ++w) sum += s.sum[w];
    whole_sum = (uint64_t)(sum * r.scale + 0.5);
  }
  uint64_t total, place;
  if (!choose_few(x, n, r, s, whole_sum, tops, low, place, total)) {
    __syncthreads();
    const RowTokens tokens = {x, n};
    const BinOrder<RowTokens> order = {tokens, s};
    order.fill(r);
    place = decide(order, r, n, true, true, total);
  }
  if (t == 0) {
    out[row] = place ? (int64_t)(uint32_t)~(uint32_t)place : -1;
    if (logp) {
      const float v = logit_of(place);
      logp[row] = (float)((v == top ? 0.0 : ((double)v - (double)top) * r.inv_t) -
                          log((double)total / r.scale));
    }
  }
}

}  // namespace

size_t sample_scratch(int64_t rows, int64_t n) {
  return (size_t)rows * parts_of(n) * (sizeof(double) + (1 + kBlocks) * sizeof(float));
}

hipError_t launch_sample(const float *logits, int64_t rows, int64_t n, const double *u,
                         const double *params, int64_t params_ld, void *scratch, int64_t *out,
                         float *logp, hipStream_t s) {
  const int lds = (int)sizeof(Shared);
  hipError_t e = set_dynamic_lds(reinterpret_cast<const void *>(k_sample), lds);
  if (e != hipSuccess) return e;
  const int64_t parts = parts_of(n);
  double *sums = static_cast<double *>(scratch);
  float *part_tops = reinterpret_cast<float *>(sums + rows * parts);
  float *tops = part_tops + rows * parts;
  hipLaunchKernelGGL(k_sample_parts, dim3((unsigned)((parts + 3) / 4), (unsigned)rows), dim3(256),
                     0, s, logits, n, params, params_ld, sums, part_tops, tops);
  hipLaunchKernelGGL(k_sample, dim3((unsigned)rows), dim3(kWG), lds, s, logits, n, u, params,
                     params_ld, sums, part_tops, tops, out, logp);
  return hipGetLastError();
}

}  // namespace aq
