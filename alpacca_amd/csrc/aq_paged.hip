// aq_paged.hip - the paged 16-bit KV cache: rotation and append, attention over a
// shared prefix and each sequence's own pages, read-back.
//
// A page holds page_size positions (a multiple of 32) of every kv head, K (rotated)
// and V in two arrays [n_pages][n_kv][page_size / 32][32 head_dim] of fp16 or
// bf16.  The 32 positions of a block lie in the order in which the matrix
// instructions take them as operands, 16 bytes a lane and 1 KB a wave:
//   K [2 pt][head_dim / 32 ks][4 cg][16 r][8 e]: position 16 pt + r, dimension
//     32 ks + 8 cg + e
//   V [head_dim / 16 dt][4 g][16 c][2 pt][4 r]: dimension 16 dt + c, position
//     16 pt + 4 g + r
// Position p of a sequence lies in the prefix (p < start) or in slot p - start of
// its row of the table; what has no page there (a row, slot or page number out of
// range, a negative position) is absent: not stored, not attended to.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "aq_internal.h"
#include "aq_matmul_dma.h"

namespace aq {
namespace {

constexpr int kBlk = 32;
// workgroups of one launch: a grid holds fewer than 2^32 threads, 256 a workgroup
constexpr int64_t kMaxGrid = (1 << 24) - 1;
// the end of positions that no table ends: all from 0 on are below it
constexpr uint64_t kAnyPos = (uint64_t)1 << 63;

template <int HD>
__device__ __forceinline__ int k_place(int s, int d) {
  return ((((s >> 4) * (HD / 32) + (d >> 5)) * 4 + ((d >> 3) & 3)) * 16 + (s & 15)) * 8 + (d & 7);
}
__device__ __forceinline__ int v_place(int s, int d) {
  return (((d >> 4) * 4 + ((s >> 2) & 3)) * 16 + (d & 15)) * 8 + 4 * (s >> 4) + (s & 3);
}

template <typename T>
__device__ __forceinline__ T rounded(float x) {
  return (T)x;  // to nearest, ties to even
}

// A value that no store of the kernel reaches, at a place that is the same for the
// whole wave: a scalar load.
template <typename T>
__device__ __forceinline__ T load_const(const T *p) {
  return *(const __attribute__((address_space(4))) T *)p;
}

// the block that holds slot `slot` of row `seq`: its number in the pool's blocks of
// kv head 0, or -1 (slots are below 2^31: the host sees to it)
__device__ __forceinline__ int64_t block_of(const aq_paged &c, const PagedTable &t, int64_t seq,
                                            int64_t slot) {
  const int per = c.page_size / kBlk;
  if (seq < 0 || seq >= t.seqs || slot < 0 || slot >= t.width * c.page_size) return -1;
  const uint32_t block = (uint32_t)slot / kBlk, page = block / (uint32_t)per;
  const int64_t id = load_const(t.pages + seq * t.width + page);
  if (id < 0 || id >= c.n_pages) return -1;
  return id * c.n_kv * per + (block - page * (uint32_t)per);
}

typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
template <typename T>
struct Vec;
template <>
struct Vec<_Float16> {
  typedef _Float16 four __attribute__((ext_vector_type(4)));
  typedef _Float16 eight __attribute__((ext_vector_type(8)));
};
template <>
struct Vec<__bf16> {
  typedef __bf16 four __attribute__((ext_vector_type(4)));
  typedef __bf16 eight __attribute__((ext_vector_type(8)));
};

// A call's tokens and where they go.
struct Place {
  int64_t pos, block;  // block -1: no place
  int s;               // the position in the block
};
__device__ __forceinline__ Place place_of(const aq_paged &c, const PagedTable &tab, int64_t n) {
  Place p;
  p.pos = load_const(tab.pos + n);
  const int64_t seq = tab.seq ? load_const(tab.seq + n) : n, slot = p.pos - tab.start;
  p.block = p.pos < 0 ? -1 : block_of(c, tab, seq, slot);
  p.s = (int)(slot & (kBlk - 1));
  return p;
}
// Values go four tokens at a time, where these lie side by side in a page (a prompt's do:
// group g holds tokens 4 g - lead .., so that the first token's neighbours start at a
// multiple of four), 8 bytes a dimension; other tokens one by one.
__device__ __forceinline__ int lead_of(const PagedTable &tab) {
  return (int)((load_const(tab.pos) - tab.start) & 3);
}
struct Group {
  int64_t n[4];
  Place p[4];
  bool in[4], together;
};
__device__ __forceinline__ Group group_of(const aq_paged &c, const PagedTable &tab, int64_t N,
                                          int64_t g, uint64_t n_pos) {
  Group r;
  const int64_t first = 4 * g - lead_of(tab);
  r.together = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r.in[i] = first + i >= 0 && first + i < N;
    r.n[i] = r.in[i] ? first + i : 0;
    r.p[i] = place_of(c, tab, r.n[i]);
    r.in[i] &= r.p[i].block >= 0 && (uint64_t)r.p[i].pos < n_pos;
    r.together &= r.in[i] && r.p[i].block == r.p[0].block && r.p[i].s == r.p[0].s + i;
  }
  r.together &= (r.p[0].s & 3) == 0;
  return r;
}

// ---- rotation and append -------------------------------------------------------
// A thread a unit, each value read once and written once: of a query or key 8 dimensions
// (neox: the rotated ones are four and their four partners), 16 bytes of a page; of the
// values four dimensions of four tokens.  Workgroups 0 .. n_qk - 1 take the queries and
// keys, per_token of them a token, the others the values.
//
// One token of 32 / 8 heads of 64 3.2 us (a launch's start and its chain: position, page,
// store), 64 of 32 / 8 of 128 5.9, 2048 of them 21.7, bound by memory (92 MB: 4.2 TB/s).
template <int HD, typename T>
__global__ void __launch_bounds__(256)
    k_paged_append(const float *q, const float *__restrict__ k, const float *__restrict__ v,
                   float *q_out, int64_t N, int n_head, int n_rot, int neox,
                   const float *__restrict__ cos_t, const float *__restrict__ sin_t,
                   uint64_t n_pos, PagedTable tab, aq_paged c, unsigned per_token,
                   unsigned per_group, unsigned n_qk) {
#pragma clang fp contract(off)
  const int64_t per = c.page_size / kBlk;
  if (blockIdx.x >= n_qk) {
    const unsigned b = blockIdx.x - n_qk;
    const int u = (int)(b % per_group) * 256 + threadIdx.x;
    if (u >= c.n_kv * (HD / 4)) return;
    const int h = u / (HD / 4), d = 4 * (u % (HD / 4));
    const Group g = group_of(c, tab, N, b / per_group, n_pos);
    f4v x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = *reinterpret_cast<const f4v *>(v + (g.n[i] * c.n_kv + h) * HD + d);
    T *vp = static_cast<T *>(c.v);
    if (g.together) {
      T *to = vp + (g.p[0].block + h * per) * (kBlk * HD) + v_place(g.p[0].s, d);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<typename Vec<T>::four *>(to + 8 * e) = typename Vec<T>::four{
            rounded<T>(x[0][e]), rounded<T>(x[1][e]), rounded<T>(x[2][e]), rounded<T>(x[3][e])};
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!g.in[i]) continue;
      T *to = vp + (g.p[i].block + h * per) * (kBlk * HD) + v_place(g.p[i].s, d);
#pragma unroll
      for (int e = 0; e < 4; ++e) to[8 * e] = rounded<T>(x[i][e]);
    }
    return;
  }
  const int64_t n = blockIdx.x / per_token;
  const int u = (int)(blockIdx.x % per_token) * 256 + threadIdx.x;
  const int heads = (q ? n_head : 0) + c.n_kv;
  if (u >= heads * (HD / 8)) return;
  int h = u / (HD / 8);
  const int i = u % (HD / 8), half = n_rot / 2;
  const bool is_k = h < c.n_kv;
  if (!is_k) h -= c.n_kv;
  const float *src = is_k ? k + (n * c.n_kv + h) * HD : q + (n * n_head + h) * HD;
  // the unit's two quads: side by side, or partners
  const bool pairs = neox && 8 * i < n_rot;
  const int a = pairs ? 4 * i : 8 * i, b = pairs ? a + half : a + 4;
  f4v x = *reinterpret_cast<const f4v *>(src + a), y = *reinterpret_cast<const f4v *>(src + b);
  const Place p = place_of(c, tab, n);
  if ((uint64_t)p.pos >= n_pos) return;  // (the whole workgroup; a position below 0 too)
  const float *cr = cos_t + p.pos * half, *sr = sin_t + p.pos * half;
  if (pairs) {
    const f4u cs = *reinterpret_cast<const f4u *>(cr + a);
    const f4u sn = *reinterpret_cast<const f4u *>(sr + a);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float r0 = x[e] * cs[e] - y[e] * sn[e];
      const float r1 = x[e] * sn[e] + y[e] * cs[e];
      x[e] = r0;
      y[e] = r1;
    }
  } else if (!neox && 8 * i < n_rot) {
    f4u cs, sn;  // of pairs 4 i .. 4 i + 3, those that exist
    if (8 * i + 8 <= n_rot) {
      cs = *reinterpret_cast<const f4u *>(cr + 4 * i);
      sn = *reinterpret_cast<const f4u *>(sr + 4 * i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = 4 * i + e < half ? 4 * i + e : half - 1;
        cs[e] = cr[j], sn[e] = sr[j];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (4 * i + e >= half) continue;
      const float x0 = e < 2 ? x[2 * e] : y[2 * e - 4], x1 = e < 2 ? x[2 * e + 1] : y[2 * e - 3];
      const float r0 = x0 * cs[e] - x1 * sn[e];
      const float r1 = x0 * sn[e] + x1 * cs[e];
      if (e < 2) x[2 * e] = r0, x[2 * e + 1] = r1;
      else y[2 * e - 4] = r0, y[2 * e - 3] = r1;
    }
  }
  if (!is_k) {
    float *dst = q_out + (n * n_head + h) * HD;
    *reinterpret_cast<f4v *>(dst + a) = x;
    *reinterpret_cast<f4v *>(dst + b) = y;
    return;
  }
  if (p.block < 0) return;
  T *to = static_cast<T *>(c.k) + (p.block + h * per) * (kBlk * HD);
  const typename Vec<T>::four xs = {rounded<T>(x[0]), rounded<T>(x[1]), rounded<T>(x[2]),
                                    rounded<T>(x[3])};
  const typename Vec<T>::four ys = {rounded<T>(y[0]), rounded<T>(y[1]), rounded<T>(y[2]),
                                    rounded<T>(y[3])};
  *reinterpret_cast<typename Vec<T>::four *>(to + k_place<HD>(p.s, a)) = xs;
  *reinterpret_cast<typename Vec<T>::four *>(to + k_place<HD>(p.s, b)) = ys;
}

// Neox rotation of dimensions that are no multiple of 8: a thread a pair of one head, for
// the queries and keys (the values go as above).
template <int HD, typename T>
__global__ void __launch_bounds__(256)
    k_paged_append_pairs(const float *q, const float *__restrict__ k, float *q_out, int n_head,
                         int n_rot, const float *__restrict__ cos_t,
                         const float *__restrict__ sin_t, uint64_t n_pos, PagedTable tab,
                         aq_paged c) {
#pragma clang fp contract(off)
  const int64_t n = blockIdx.x;
  const Place p = place_of(c, tab, n);
  if ((uint64_t)p.pos >= n_pos) return;
  const int half = n_rot / 2, heads = (q ? n_head : 0) + c.n_kv;
  for (int j = threadIdx.x; j < heads * (HD / 2); j += 256) {
    int h = j / (HD / 2);
    const int i = j % (HD / 2);
    const bool is_k = h < c.n_kv;
    if (!is_k) h -= c.n_kv;
    const int a = i < half ? i : n_rot + 2 * (i - half), b = i < half ? i + half : a + 1;
    const float *src = is_k ? k + (n * c.n_kv + h) * HD : q + (n * n_head + h) * HD;
    float x0 = src[a], x1 = src[b];
    if (i < half) {
      const float cs = cos_t[p.pos * half + i], sn = sin_t[p.pos * half + i];
      const float r0 = x0 * cs - x1 * sn;
      const float r1 = x0 * sn + x1 * cs;
      x0 = r0;
      x1 = r1;
    }
    if (!is_k) {
      float *dst = q_out + (n * n_head + h) * HD;
      dst[a] = x0;
      dst[b] = x1;
    } else if (p.block >= 0) {
      T *to = static_cast<T *>(c.k) + (p.block + (int64_t)h * (c.page_size / kBlk)) * (kBlk * HD);
      to[k_place<HD>(p.s, a)] = rounded<T>(x0);
      to[k_place<HD>(p.s, b)] = rounded<T>(x1);
    }
  }
}

// ---- read-back -------------------------------------------------------------------
// A thread a unit: 8 dimensions of a key, or four of four tokens' values.  1 token of 8
// heads of 64 3.2 us, 64 of 8 of 128 5.4, 2048 7.4 to 9.6 (16.8 MB: a launch's start and
// end, then memory).
template <int HD>
__global__ void __launch_bounds__(256)
    k_paged_read(int64_t N, PagedTable tab, aq_paged c, uint16_t *__restrict__ ko,
                 uint16_t *__restrict__ vo, unsigned per_token, unsigned per_group,
                 unsigned n_k) {
  typedef uint16_t four __attribute__((ext_vector_type(4)));
  const int64_t per = c.page_size / kBlk;
  if (blockIdx.x < n_k) {
    const int64_t n = blockIdx.x / per_token;
    const int u = (int)(blockIdx.x % per_token) * 256 + threadIdx.x;
    if (u >= c.n_kv * (HD / 8)) return;
    const int h = u / (HD / 8), d = 8 * (u % (HD / 8));
    const Place p = place_of(c, tab, n);
    uint4 x = make_uint4(0, 0, 0, 0);
    if (p.block >= 0)
      x = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(c.k) +
                                           (p.block + h * per) * (kBlk * HD) +
                                           k_place<HD>(p.s, d));
    *reinterpret_cast<uint4 *>(ko + (n * c.n_kv + h) * HD + d) = x;
    return;
  }
  const unsigned b = blockIdx.x - n_k;
  const int u = (int)(b % per_group) * 256 + threadIdx.x;
  if (u >= c.n_kv * (HD / 4)) return;
  const int h = u / (HD / 4), d = 4 * (u % (HD / 4));
  const int64_t first = 4 * (int64_t)(b / per_group) - lead_of(tab);
  const Group g = group_of(c, tab, N, b / per_group, kAnyPos);
  const uint16_t *vp = static_cast<const uint16_t *>(c.v);
  four x[4];
  if (g.together) {
    const uint16_t *from = vp + (g.p[0].block + h * per) * (kBlk * HD) + v_place(g.p[0].s, d);
    four y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = *reinterpret_cast<const four *>(from + 8 * e);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = four{y[0][i], y[1][i], y[2][i], y[3][i]};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = four{0, 0, 0, 0};
      if (!g.in[i]) continue;
      const uint16_t *from = vp + (g.p[i].block + h * per) * (kBlk * HD) + v_place(g.p[i].s, d);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = from[8 * e];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (first + i >= 0 && first + i < N)
      *reinterpret_cast<four *>(vo + ((first + i) * c.n_kv + h) * HD + d) = x[i];
}

// ---- attention -----------------------------------------------------------------
// Tiles of 16 query rows of one kv head, blocks of 32 positions, on the
// 16x16x32 matrix instructions of the cache's type, with every fp32 operand in
// pieces of that type (x = sum of pieces: two of fp16, 22 bits; three of bf16, 24):
//   S^T (positions x rows) = K Q^T, Q's row times log2(e) / sqrt(head_dim) and a
//     power of two (Ops<T>::shift): lane l holds row l % 16's scores at positions
//     16 pt + 4 (l / 16) + r (pt = 0, 1; r = 0 .. 3);
//   O^T (dimensions x rows) += V^T P^T: those eight weights are the lane's operand
//     as it holds them.  Lane l gets row l % 16's dimensions 16 dt + 4 (l / 16) + r.
// Weights are P = 2^(z - m + Ops<T>::kTop), m the running maximum rounded up to a whole
// number, so that rescaling is exact and rare, and the pieces hold 22 bits of what
// counts.  The sum of the weights is kept per lane, in fp32.
typedef float f2v __attribute__((ext_vector_type(2)));
typedef unsigned int u4v __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

template <typename T>
struct Ops;
template <>
struct Ops<_Float16> {
  static constexpr int NP = 2;
  static constexpr float kTop = 14.f;  // weights reach 2^14: their second piece is normal
  // The power of two that a query row is raised by, am its largest value: to
  // [2^14, 2^15) after the factor f, where the second piece's last bit is a normal one's.
  // (A row below 2^-110 keeps fewer bits of scores that are as good as 0.)
  static __device__ __forceinline__ int shift(float am, float f) {
    return min(15 - __builtin_amdgcn_frexp_expf(am * f), 125);
  }
  static __device__ __forceinline__ f4v mfma(u4v a, u4v b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a),
                                                  __builtin_bit_cast(h8, b), c, 0, 0, 0);
  }
  // a and b in two pieces.  The first is cut off (one instruction for the pair), so
  // that what it leaves has their signs and is exact; the second is rounded.
  static __device__ __forceinline__ void split(float a, float b, uint32_t (&piece)[2]) {
    const h2 h = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(a, b));
    // (a factor that the compiler does not know keeps this one mixed-precision
    // multiply-add a value instead of a conversion and a difference)
    float minus = -1.f;
    asm("" : "+v"(minus));
    const h2 l = __builtin_convertvector(
        f2v{fmaf((float)h[0], minus, a), fmaf((float)h[1], minus, b)}, h2);
    piece[0] = __builtin_bit_cast(uint32_t, h);
    piece[1] = __builtin_bit_cast(uint32_t, l);
  }
};
template <>
struct Ops<__bf16> {
  static constexpr int NP = 3;
  static constexpr float kTop = 0.f;  // values may be as large as float32: weights are not
  // bf16 has float32's exponents, and so have the keys: rows go down by 2^12, and sums of
  // their products pass float32's range only where the scores (which come back up in
  // the weights' exponents) are past it themselves.  A row whose last piece would then not
  // be normal is brought to 2^-24, from where no key takes a sum past 2^(128 + 8 - 24).
  static __device__ __forceinline__ int shift(float am, float) {
    return am < 0x1p-64f ? -24 - __builtin_amdgcn_frexp_expf(am) : -12;
  }
  static __device__ __forceinline__ f4v mfma(u4v a, u4v b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a),
                                                   __builtin_bit_cast(b8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ void split(float a, float b, uint32_t (&piece)[3]) {
#pragma unroll
    for (int n = 0; n < 3; ++n) {
      const b2 h = __builtin_convertvector(f2v{a, b}, b2);
      a -= (float)h[0];
      b -= (float)h[1];
      piece[n] = __builtin_bit_cast(uint32_t, h);
    }
  }
};

template <int OFF>
__device__ __forceinline__ float2 lane_pair(float v) {
  const unsigned u = __float_as_uint(v);
  const auto r = OFF == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false)
                           : __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// over the four lanes l, l ^ 16, l ^ 32, l ^ 48 that share a row
__device__ __forceinline__ float row_max(float v) {
  float2 p = lane_pair<16>(v);
  p = lane_pair<32>(fmaxf(p.x, p.y));
  return fmaxf(p.x, p.y);
}
__device__ __forceinline__ float row_sum(float v) {
  float2 p = lane_pair<16>(v);
  p = lane_pair<32>(p.x + p.y);
  return p.x + p.y;
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.f : m; }

// A query row of the lane's (its dimensions 32 ks + 8 (l / 16) + e) in pieces of
// q log2(e) / sqrt(HD) / back, back a power of two.  A row with an infinity or a NaN
// is NaN.
template <int HD, typename T>
struct QRow {
  static constexpr int NP = Ops<T>::NP;
  u4v piece[NP][HD / 32];
  float back;
  __device__ __forceinline__ void load(const float *q, bool live) {
    const int cg = (threadIdx.x >> 4) & 3;
    const float f = 1.44269504088896341f / __builtin_sqrtf((float)HD);
    float v[HD / 32][8];
    float am = 0.f;
#pragma unroll
    for (int ks = 0; ks < HD / 32; ++ks) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const f4v x = *reinterpret_cast<const f4v *>(q + 32 * ks + 8 * cg + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[ks][4 * i + e] = live ? x[e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // (a NaN counts as infinity here: a maximum passes over it)
        const float a = fabsf(v[ks][e]);
        am = fmaxf(am, a < INFINITY ? a : INFINITY);
      }
    }
    am = row_max(am);
    const bool bad = am == INFINITY;
    const int up = am > 0.f && !bad ? Ops<T>::shift(am, f) : 0;
    back = ldexpf(1.f, -up);
#pragma unroll
    for (int ks = 0; ks < HD / 32; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a = ldexpf(v[ks][2 * i], up) * f, b = ldexpf(v[ks][2 * i + 1], up) * f;
        a = bad ? NAN : a;
        b = bad ? NAN : b;
        uint32_t parts[NP];
        Ops<T>::split(a, b, parts);
#pragma unroll
        for (int p = 0; p < NP; ++p) piece[p][ks][i] = parts[p];
      }
  }
};

// The running softmax of a lane's row: m (the same in the row's four lanes), the
// lane's part of the sum, the numerators at dimensions 16 dt + 4 (l / 16) + r.
template <int HD>
struct RowState {
  float m, l;
  f4v o[HD / 16];
  __device__ __forceinline__ void clear() {
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) o[i] = f4v{0.f, 0.f, 0.f, 0.f};
  }
};

// raw scores of NB blocks (two tiles of positions each) to weights in pieces; the state
// moves on to the new maximum.  TAIL: positions from rem[b] on of block b do not exist.
// (back is a power of two: scores times it are exact, in the maximum and in the
// multiply-add that gives a weight's exponent.)
template <int HD, typename T, int NB, bool TAIL>
__device__ __forceinline__ void weigh(f4v (&sc)[NB][2], float back, const int (&rem)[NB],
                                      RowState<HD> &st, u4v (&w)[NB][Ops<T>::NP]) {
  const int cg = (threadIdx.x >> 4) & 3;
  float top = -INFINITY;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (TAIL && 16 * (e >> 2) + 4 * cg + (e & 3) >= rem[b]) sc[b][e >> 2][e & 3] = -INFINITY;
      top = fmaxf(top, sc[b][e >> 2][e & 3]);
    }
  top *= back;
  if (__any(top > st.m)) {
    const float m = fmaxf(st.m, ceilf(row_max(top)));
    const float f = st.m == -INFINITY ? 0.f : exp2_(st.m - m);
    st.m = m;
    st.l *= f;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) st.o[i] *= f;
  }
  const float ref = Ops<T>::kTop - finite_ref(st.m);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    float p[8], l[4];
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = exp2_(fmaf(sc[b][e >> 2][e & 3], back, ref));
#pragma unroll
    for (int e = 0; e < 4; ++e) l[e] = p[e] + p[4 + e];
    st.l += (l[0] + l[1]) + (l[2] + l[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t parts[Ops<T>::NP];
      Ops<T>::split(p[2 * i], p[2 * i + 1], parts);
#pragma unroll
      for (int n = 0; n < Ops<T>::NP; ++n) w[b][n][i] = parts[n];
    }
  }
}

// values at positions from `rem` on become 0 (whatever lies there, a weight of 0
// would not undo an infinity or a NaN)
__device__ __forceinline__ u4v only_first(u4v v, int rem) {
  const int cg = (threadIdx.x >> 4) & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int pos = 16 * (i >> 1) + 4 * cg + 2 * (i & 1);
    v[i] &= (pos < rem ? 0xFFFFu : 0u) | (pos + 1 < rem ? 0xFFFF0000u : 0u);
  }
  return v;
}

// The block numbers (see block_of, with kv head h's) of blocks first, first + 4, ..
// of a list of pages, one a lane; -1: absent.
__device__ __forceinline__ int64_t lane_block(const aq_paged &c, const int32_t *pages, int h,
                                              int64_t b, int64_t end) {
  const uint32_t per = c.page_size / kBlk, page = (uint32_t)b / per;
  if (b >= end) return -1;
  const int64_t id = pages[page];
  if (id < 0 || id >= c.n_pages) return -1;
  return (id * c.n_kv + h) * per + ((uint32_t)b - page * per);
}
__device__ __forceinline__ int64_t of_lane(int64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// A tile of rows against NB blocks: keys(b, j) is operand j = pt * HD / 32 + ks of
// block b, values(b, j) that of its dimensions 16 j ..  Products of different sums
// follow one another: one that adds to the last one's result would wait for it.
// scored() runs when the scores' products are on their way.
template <int HD, typename T, int NB, bool TAIL, class K, class Next>
__device__ __forceinline__ void score_block(const QRow<HD, T> &q, RowState<HD> &st,
                                            const int (&rem)[NB], K &&keys, Next &&scored,
                                            u4v (&w)[NB][Ops<T>::NP]) {
  constexpr int KS = HD / 32, NP = Ops<T>::NP;
  f4v sc[NB][2];
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i) sc[i >> 1][i & 1] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    u4v k[2 * NB];
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) k[i] = keys(i >> 1, (i & 1) * KS + ks);
#pragma unroll
    for (int p = NP - 1; p >= 0; --p)
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i)
        sc[i >> 1][i & 1] = Ops<T>::mfma(k[i], q.piece[p][ks], sc[i >> 1][i & 1]);
  }
  scored();
  weigh<HD, T, NB, TAIL>(sc, q.back, rem, st, w);
}
template <int HD, typename T, int NB, bool TAIL, class K, class V, class Next>
__device__ __forceinline__ void attend_block(const QRow<HD, T> &q, RowState<HD> &st,
                                             const int (&rem)[NB], K &&keys, V &&values,
                                             Next &&scored) {
  constexpr int NP = Ops<T>::NP;
  u4v w[NB][NP];
  score_block<HD, T, NB, TAIL>(q, st, rem, keys, scored, w);
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int j = 0; j < HD / 16; j += 4) {
      u4v v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = values(b, j + i);
        if (TAIL) v[i] = only_first(v[i], rem[b]);
      }
#pragma unroll
      for (int p = NP - 1; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[j + i] = Ops<T>::mfma(v[i], w[b][p], st.o[j + i]);
    }
}

// The tokens whose rows share a tile: row j is token j / G's, which sees `len` positions.
struct Tokens {
  int count, G;
  int least;  // of their lengths
  int mine;   // the lane's row's
  const int64_t *pos;
  int64_t start, room;
  __device__ __forceinline__ int len(int t) const {
    const int64_t n = load_const(pos + t) - start;
    return (int)(n < room ? n + 1 : room);
  }
};

// One tile of rows against blocks b0 + wave, b0 + wave + 4, .. below b1 of a list of
// pages, straight from memory; len: the largest of the tokens' lengths.  A wave's next
// keys are on their way while it weighs the present ones; with eight waves a CU that is
// enough to be bound by memory: 64 rows' own positions of 8 heads of 128 at 4.7 to 5.1
// TB/s, the rate of a large copy.  In blocks where a token's
// positions end, each token's sums take its own values alone: what lies behind them may
// be an infinity or a NaN, which a weight of 0 would not undo.
template <int HD, typename T>
__device__ __forceinline__ void attend_strided(const aq_paged &c, const int32_t *pages, int h,
                                               int64_t b0, int64_t b1, const Tokens &tok,
                                               const QRow<HD, T> &q, RowState<HD> &st) {
  constexpr int KS = HD / 32, DT = HD / 16, NP = Ops<T>::NP;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u4v *kp = static_cast<const u4v *>(c.k) + lane, *vp = static_cast<const u4v *>(c.v) + lane;
  for (int64_t base = b0 + wave; base < b1; base += 4 * 64) {
    const int64_t mine = lane_block(c, pages, h, base + 4 * lane, b1);
    uint64_t left = __ballot(mine >= 0);
    if (!left) continue;
    int i = __builtin_ctzll(left);
    int64_t at = of_lane(mine, i) * (kBlk * HD / 8);
    u4v k[2 * KS], v[DT];
#pragma unroll
    for (int j = 0; j < 2 * KS; ++j) k[j] = kp[at + 64 * j];
    while (left) {
      left &= left - 1;
      const int first = (int)(base + 4 * i) * kBlk;  // the block's first position
#pragma unroll
      for (int j = 0; j < DT; ++j) v[j] = vp[at + 64 * j];
      auto keys = [&](int, int j) { return k[j]; };
      auto values = [&](int, int j) { return v[j]; };
      auto next = [&] {
        if (!left) return;
        i = __builtin_ctzll(left);
        at = of_lane(mine, i) * (kBlk * HD / 8);
#pragma unroll
        for (int j = 0; j < 2 * KS; ++j) k[j] = kp[at + 64 * j];
      };
      if (first + kBlk <= tok.least) {
        const int rem[1] = {kBlk};
        attend_block<HD, T, 1, false>(q, st, rem, keys, values, next);
        continue;
      }
      const int rem[1] = {tok.mine - first};
      u4v w[1][NP];
      score_block<HD, T, 1, true>(q, st, rem, keys, next, w);
#pragma unroll 1
      for (int t = 0; t < tok.count; ++t) {
        const int len = tok.count == 1 ? tok.least : tok.len(t);
        if (len <= first) continue;
        const bool its = (lane & 15) / tok.G == t || tok.count == 1;
#pragma unroll
        for (int j = 0; j < DT; ++j) {
          const u4v x = only_first(v[j], len - first);
          f4v o = st.o[j];
#pragma unroll
          for (int p = NP - 1; p >= 0; --p) o = Ops<T>::mfma(x, w[0][p], o);
          st.o[j] = its ? o : st.o[j];
        }
      }
    }
  }
}

// The same for TW tiles of rows, a wave each, against blocks b0 .. b1 - 1,
// which go through LDS in stages of 4 / TW ways of NB blocks: the four waves bring one
// while another is computed.  64 rows of 32 / 8 heads of 128 over 8000 positions 38 us in
// fp16, 43 in bf16 (33 MB: 7 us, and as long on the matrix units): bound by a wave's own
// chain of barrier, scores, weights and sums, which one wave a SIMD beside the rows' own
// positions does not overlap.  Straight from memory 50 and 70; one block a stage 42; two
// tiles of rows a wave, or three waves a SIMD, spill registers (105, 41 to 58).
template <int HD, int TW>
struct Stage {
  static constexpr int NB = TW == 4 ? 2 : 1, WAYS = 4 / TW, BLOCKS = WAYS * NB;
  static constexpr int BLOCK = HD * 128;  // bytes of K and V
  static constexpr int BYTES = BLOCKS * BLOCK;
};
template <int HD, typename T, int TW, class Load>
__device__ __forceinline__ void attend_staged(const aq_paged &c, const int32_t *pages, int h,
                                              int64_t b0, int64_t b1, int64_t len, uint8_t *lds,
                                              QRow<HD, T> &q, RowState<HD> &st,
                                              Load &&load_rows) {
  using St = Stage<HD, TW>;
  constexpr int NB = St::NB;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t lds0 = lds_offset(lds);
  for (int64_t base = b0; base < b1; base += 64) {
    const int64_t mine = lane_block(c, pages, h, base + lane, b1) * (kBlk * HD * 2);  // bytes
    uint64_t to_bring = __ballot(mine >= 0), to_do = to_bring;
    auto bring = [&](int buf) {
#pragma unroll
      for (int p = 0; p < St::BLOCKS; ++p) {
        if (!to_bring) break;
        const int64_t at = of_lane(mine, __builtin_ctzll(to_bring));
        to_bring &= to_bring - 1;
        const char *k = static_cast<const char *>(c.k) + at;
        const char *v = static_cast<const char *>(c.v) + at;
        const uint32_t to = lds0 + buf * St::BYTES + p * St::BLOCK;
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) {
          const int x = 1024 * (4 * j + wave);
          dma16(to + x, 16 * lane, k + x);
          dma16(to + HD * 64 + x, 16 * lane, v + x);
        }
      }
    };
    __syncthreads();  // (the buffers are free)
    bring(0);
    if (base == b0) load_rows();  // beside the first stage's way
    for (int buf = 0; to_do; buf ^= 1) {
      dma_barrier<0>();  // this stage is there, and the other buffer has been used
      auto next = [&] { bring(buf ^ 1); };
      // the wave's blocks of the stage
      int rem[NB];
      bool full = true;
#pragma unroll
      for (int p = 0; p < St::BLOCKS; ++p) {
        if (p / NB == wave / TW) {
          const int64_t behind = to_do ? len - (base + __builtin_ctzll(to_do)) * kBlk : 0;
          rem[p % NB] = behind < kBlk ? (int)behind : kBlk;
          full &= behind >= kBlk;
        }
        to_do &= to_do - 1;
      }
      if (rem[0] <= 0) {
        next();
        continue;
      }
      const uint8_t *at = lds + buf * St::BYTES + (wave / TW) * (NB * St::BLOCK) + 16 * lane;
      auto keys = [&](int b, int j) { return lds_read<u4v>(at + b * St::BLOCK + 1024 * j); };
      auto values = [&](int b, int j) {
        return lds_read<u4v>(at + b * St::BLOCK + HD * 64 + 1024 * j);
      };
      if (full) attend_block<HD, T, NB, false>(q, st, rem, keys, values, next);
      else attend_block<HD, T, NB, true>(q, st, rem, keys, values, next);
    }
  }
}

// The partial state of a row: HD numerators relative to 2^(m - Ops<T>::kTop), m, l.
template <int HD>
constexpr int kState = HD + 4;

// How a call's work is split (host and kernels).
struct PagedPlan {
  int tw;          // tiles of 16 rows of the prefix that a workgroup takes
  int groups;      // groups of 16 tw rows of a kv head
  int sp, ss;      // splits of the prefix and of a row's own positions
  unsigned pre, own;  // workgroups of each, in this order
  int states() const { return sp + ss; }
};

template <int HD>
__device__ __forceinline__ void put_dead(float *state) {
  state[HD] = -INFINITY;
  state[HD + 1] = 0.f;
}

// Item `item` of the prefix: a split of a kv head, and a group of rows.  The groups
// that read the same positions follow one another eight items apart, which is on
// the same one of the eight dies, whose L2 then holds them.
__device__ __forceinline__ void pick_unit(const PagedPlan &p, unsigned units, unsigned item,
                                          unsigned &unit, unsigned &group) {
  const unsigned groups = p.groups, full = units / 8 * 8;
  if (item < full * groups) {
    unit = item / (8 * groups) * 8 + item % 8;
    group = item / 8 % groups;
  } else {
    item -= full * groups;
    unit = full + item % (units - full);
    group = item / (units - full);
  }
}

// Items of the prefix: a split, a group of rows and a kv head; own ones: a split, a kv
// head and a row, or the rows of neighbours of one sequence (a row that ends inside the
// prefix has that part of it as its own).
// Waves that share rows have their states merged through LDS.
template <int HD, typename T, int TW>
__global__ void __launch_bounds__(256, HD == 256 ? 1 : 2)
    k_paged_attn(const float *__restrict__ q, int64_t N, int n_head, PagedTable tab,
                 PagedTable pre, aq_paged c, PagedPlan plan, float *__restrict__ states,
                 float *__restrict__ out) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  auto num = reinterpret_cast<float(*)[16][HD + 4]>(lds);  // numerators, maximum, sum of 4 waves
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, cg = lane >> 4;
  const int G = n_head / c.n_kv, S = plan.sp + plan.ss;
  const bool is_pre = blockIdx.x < plan.pre;
  unsigned item = blockIdx.x - (is_pre ? 0u : plan.pre);
  int h, split;
  int64_t len, b0, b1;
  const int32_t *pages;
  Tokens tok = {1, G, 0, 0, nullptr, 0, 0};
  const int rows = (int)N * G;  // of a kv head (N * n_head is below 2^24)
  int row0 = 0;                 // of the group
  int n = 0;
  if (is_pre) {
    unsigned unit, group;
    pick_unit(plan, (unsigned)(plan.sp * c.n_kv), item, unit, group);
    split = (int)(unit % plan.sp);
    h = (int)(unit / plan.sp);
    row0 = (int)group * (16 * TW);
    pages = pre.pages;
    len = pre.start;
    const int64_t blocks = (len + kBlk - 1) / kBlk, each = (blocks + plan.sp - 1) / plan.sp;
    b0 = split * each;
    b1 = b0 + each < blocks ? b0 + each : blocks;
  } else {
    split = (int)(item % plan.ss);
    item /= plan.ss;
    h = (int)(item % c.n_kv);
    n = (int)(item / c.n_kv);
    row0 = n * G;
    const int64_t pos = load_const(tab.pos + n), seq = tab.seq ? load_const(tab.seq + n) : n;
    const int64_t room = tab.width * c.page_size;
    // (the 64 tokens about it, below, loaded at once with its own)
    const bool share = tab.seq && G <= 8;
    const int around = n & ~63;
    int64_t lp = -1, ls = -1;
    if (share && around + lane < (int)N) lp = tab.pos[around + lane], ls = tab.seq[around + lane];
    len = 0;
    pages = nullptr;
    if (pos >= 0 && pos < pre.start) {
      pages = pre.pages;
      len = pos + 1;
      tok = {1, G, (int)len, (int)len, nullptr, 0, 0};
    } else if (pos >= 0 && seq >= 0 && seq < tab.seqs) {
      pages = tab.pages + seq * tab.width;
      len = pos - tab.start < room ? pos - tab.start + 1 : room;
      tok = {1, G, (int)len, (int)len, tab.pos + n, tab.start, room};
      if (share) {
        // Neighbours of one sequence share a tile: runs inside 64 tokens, 16 / G at a
        // time, the first of them for all.
        const int i = n - around, per = 16 / G;
        const bool joins = lp >= tab.start && lp >= 0 && ls == seq;
        const uint64_t others = ~__ballot(joins);
        const uint64_t below = others & ((1ull << i) - 1);
        const int from = below ? 64 - __builtin_clzll(below) : 0;  // the run's first
        const uint64_t above = i < 63 ? others >> (i + 1) : 0;
        const int to = above ? i + 1 + __builtin_ctzll(above) : 64;
        if ((i - from) % per) return;
        tok.count = min(per, to - i);
        // the shortest and the longest of them, and the lane's row's
        const int64_t its = lp - tab.start < room ? lp - tab.start + 1 : room;
        int lo = INT32_MAX, hi = 0;
        for (int t = 0; t < tok.count; ++t) {
          const int l = __builtin_amdgcn_readlane((int)its, i + t);
          lo = min(lo, l), hi = max(hi, l);
          if (j / G == t) tok.mine = l;
        }
        tok.least = lo;
        len = hi;
      }
    }
    const int64_t blocks = (len + kBlk - 1) / kBlk;
    int64_t each = (blocks + plan.ss - 1) / plan.ss;
    each = each > 4 ? each : 4;
    b0 = split * each;
    b1 = b0 + each < blocks ? b0 + each : blocks;
    split += plan.sp;
  }
  // the states of `tiles` tiles of rows, the first one's first row `first`, wave w's
  // of tile w % tiles, to memory
  auto write = [&](const RowState<HD> &st, int tiles, int first, int end) {
    const float l = row_sum(st.l);
    __syncthreads();
#pragma unroll
    for (int d = 0; d < HD / 16; ++d)
      *reinterpret_cast<f4v *>(&num[wave][j][16 * d + 4 * cg]) = st.o[d];
    if (cg == 0) num[wave][j][HD] = st.m, num[wave][j][HD + 1] = l;
    __syncthreads();
    // 16 threads a row
    const int r = threadIdx.x >> 4, part = threadIdx.x & 15;
    for (int tile = 0; tile < tiles; ++tile) {
      const int row = first + 16 * tile + r;
      if (row >= end) break;
      float m = -INFINITY, sum = 0.f;
      for (int w = tile; w < 4; w += tiles) m = fmaxf(m, num[w][r][HD]);
      f4v o[HD / 64];
#pragma unroll
      for (int d = 0; d < HD / 64; ++d) o[d] = f4v{0.f, 0.f, 0.f, 0.f};
      for (int w = tile; w < 4; w += tiles) {
        const float mw = num[w][r][HD], lw = num[w][r][HD + 1];
        const float f = mw == -INFINITY ? 0.f : exp2_(mw - m);
        sum += lw == 0.f ? 0.f : lw * (m == -INFINITY ? 1.f : f);
#pragma unroll
        for (int d = 0; d < HD / 64; ++d)
          o[d] += f * *reinterpret_cast<const f4v *>(&num[w][r][64 * d + 4 * part]);
      }
      const int i = row / G;
      const int64_t flat = (int64_t)i * n_head + h * G + (row - i * G);
      const bool skip = is_pre && tab.pos[i] < pre.start;
      float *dst = S == 1 ? out + flat * HD : states + (flat * S + split) * kState<HD>;
      const float inv = S == 1 ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
#pragma unroll
      for (int d = 0; d < HD / 64; ++d)
        *reinterpret_cast<f4v *>(dst + 64 * d + 4 * part) = o[d] * inv;
      if (S != 1 && part == 0) {
        dst[HD] = skip ? -INFINITY : m;
        dst[HD + 1] = skip ? 0.f : sum;
      }
    }
  };
  if (is_pre) {
    QRow<HD, T> qr;
    RowState<HD> st;
    st.clear();
    auto load_rows = [&] {
      const int row = row0 + 16 * (wave % TW) + j;
      const bool live = row < rows;
      const int i = live ? row / G : 0, head = h * G + (live ? row - i * G : 0);
      qr.load(q + ((int64_t)i * n_head + head) * HD, live);
    };
    if constexpr (TW == 1) {
      load_rows();
      const Tokens one = {1, G, (int)len, (int)len, nullptr, 0, 0};
      attend_strided<HD, T>(c, pages, h, b0, b1, one, qr, st);
    } else {
      attend_staged<HD, T, TW>(c, pages, h, b0, b1, len, lds, qr, st, load_rows);
    }
    write(st, TW, row0, rows);
  } else {
    const int live = tok.count * G;
    if (b0 >= b1 && S != 1) {  // nothing of the rows here
      const int r = threadIdx.x;
      if (r < live)
        put_dead<HD>(states + (((int64_t)(n + r / G) * n_head + h * G + r % G) * S + split) *
                                  kState<HD>);
      return;
    }
    QRow<HD, T> qr;
    RowState<HD> st;
    const int r = j < live ? j : 0;
    qr.load(q + ((int64_t)(n + r / G) * n_head + h * G + r % G) * HD, j < live);
    st.clear();
    attend_strided<HD, T>(c, pages, h, b0, b1, tok, qr, st);
    write(st, 1, row0, row0 + live);
  }
}

// One row's states of its S <= 64 splits to its output: NT threads, four dimensions
// each, HD / 4 of them a state, all loads under way at once.  One wave up to 8 states,
// four from there on: 48 states of 256 rows of 128 in 4 us (13.3 in one wave, state
// after state).
template <int HD, int NT>
__global__ void __launch_bounds__(256)
    k_paged_merge(const float *__restrict__ states, int64_t rows, int S, float *__restrict__ out) {
  constexpr int TPS = HD / 4, GROUPS = NT / TPS, PER = 64 / (NT == 64 ? 8 : 1) / GROUPS;
  __shared__ __attribute__((aligned(16))) float num[NT == 256 ? 4 : 1][HD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = NT == 64 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
  if (row >= rows) return;
  states += row * S * kState<HD>;
  const int t = threadIdx.x & (NT - 1), g = t / TPS, d = 4 * (t % TPS);
  f4v x[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = g + GROUPS * i;
    x[i] = *reinterpret_cast<const f4v *>(states + (s < S ? s : 0) * kState<HD> + d);
  }
  float m = -INFINITY, l = 0.f;
  if (lane < S) {
    m = states[lane * kState<HD> + HD];
    l = states[lane * kState<HD> + HD + 1];
  }
  const bool some = m != -INFINITY || l != 0.f;  // (a sum may be NaN)
  float top = m;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  const float f = !some ? 0.f : m == -INFINITY ? 1.f : exp2_(m - top);
  float sum = some ? l * f : 0.f;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
  const uint64_t live = __ballot(some);
  f4v o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = g + GROUPS * i;
    const float fs = __shfl(f, s & 63);
    const bool use = s < S && (live >> (s & 63) & 1);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = use ? fmaf(x[i][e], fs, o[e]) : o[e];
  }
  // over the wave's groups
#pragma unroll
  for (int off = 32; off >= TPS && off > 0; off >>= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], off);
  if constexpr (NT == 256) {
    if (lane < TPS) *reinterpret_cast<f4v *>(&num[wave][d]) = o;
    __syncthreads();
    if (wave > 0 || lane >= TPS) return;
    o = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) o += *reinterpret_cast<const f4v *>(&num[w][d]);
  }
  if (lane < TPS)
    *reinterpret_cast<f4v *>(out + row * HD + d) = o * (sum == 0.f ? 0.f : 1.f / sum);
}

// Splits.  The prefix, in workgroups of four waves: up to 16 rows one tile, straight from
// memory, which the waves part the positions of (8 rows of 4 heads over 100000 positions
// 89 us in 48 splits of 8 heads, 92 in 32); up to 32 rows two tiles, two waves each, which
// share stages of two blocks in LDS; past that four tiles, a wave each, that share all
// positions through LDS, a workgroup a CU: the rows' own positions, bound by memory,
// run on the same CUs (64 rows of 32 / 8 heads over 8000 and 1024 of their own 68 us;
// with two workgroups of the prefix a CU, twice the states, 82; the two kinds in
// turn 75, where rows that own little then wait for a late start: 28 against 25).
// A row's own positions: what takes the fewest rounds of the workgroups that the GPU
// holds beside the prefix's, where a workgroup's start and end count as much as four
// blocks (24 sequences' two rows of 28 / 4 heads over 4001 positions in 8 splits 43 us, in
// 5 51; before neighbours shared a tile 59 in 3, 44 in 6).
PagedPlan paged_plan(const aq_paged &c, int64_t N, int n_head, int64_t width, int64_t start) {
  const int64_t rows = N * (n_head / c.n_kv), places = c.head_dim == 256 ? 256 : 512;
  PagedPlan p = {};
  p.tw = 1;
  if (start > 0) {
    p.tw = rows > 32 ? 4 : rows > 16 ? 2 : 1;
    p.groups = (int)((rows + 16 * p.tw - 1) / (16 * p.tw));
    const int64_t items = (int64_t)p.groups * c.n_kv, want = p.tw == 2 ? 512 : 256;
    const int64_t blocks = (start + kBlk - 1) / kBlk, least = p.tw == 4 ? 8 : 4;
    const int64_t s = std::min((want + items - 1) / items, (blocks + least - 1) / least);
    p.sp = (int)std::max<int64_t>(1, std::min<int64_t>(s, 48));
    p.pre = (unsigned)(p.sp * items);
  }
  const int64_t items = N * c.n_kv, blocks = width * c.page_size / kBlk;
  const int64_t left = std::max<int64_t>(places - p.pre, places / 2);
  const int64_t fit = items ? (kMaxGrid - p.pre) / items : 1;  // splits that one launch takes
  const int64_t most = std::min({(blocks + 3) / 4, (int64_t)(p.sp ? 16 : 64), fit});
  p.ss = 1;
  int64_t best = INT64_MAX;
  for (int64_t s = 1; s <= std::max<int64_t>(most, 1); ++s) {
    const int64_t cost = (items * s + left - 1) / left * ((blocks + s - 1) / s + 4);
    if (cost <= best) best = cost, p.ss = (int)s;
  }
  p.own = (unsigned)(p.ss * items);
  return p;
}

template <class F>
void by_shape(const aq_paged &c, F &&f) {
  auto typed = [&](auto hd) {
    if (c.dtype == AQ_F16) f(hd, _Float16());
    else f(hd, __bf16());
  };
  if (c.head_dim == 64) typed(std::integral_constant<int, 64>());
  else if (c.head_dim == 128) typed(std::integral_constant<int, 128>());
  else typed(std::integral_constant<int, 256>());
}

}  // namespace

hipError_t launch_rope_paged(const float *q, const float *k, const float *v, float *q_out,
                             int64_t N, int n_head, int n_rot, int neox, const float *cos_t,
                             const float *sin_t, int64_t n_pos, const PagedTable &tab,
                             const aq_paged &c, hipStream_t s) {
  if (n_rot == 0) neox = 0;
  const uint64_t end = n_rot ? (uint64_t)n_pos : kAnyPos;  // (no table, and no end to it)
  const bool by_pairs = neox && n_rot % 8 != 0;
  const int64_t heads = (q ? n_head : 0) + c.n_kv;
  const int64_t per_token = (heads * c.head_dim / 8 + 255) / 256;
  const int64_t per_group = ((int64_t)c.n_kv * c.head_dim / 4 + 255) / 256;
  const int64_t n_qk = by_pairs ? 0 : N * per_token, n_v = (N + 6) / 4 * per_group;
  if (n_qk + n_v > kMaxGrid || N > kMaxGrid) return hipErrorInvalidValue;
  by_shape(c, [&](auto hd, auto t) {
    constexpr int HD = decltype(hd)::value;
    typedef decltype(t) T;
    if (by_pairs)
      hipLaunchKernelGGL((k_paged_append_pairs<HD, T>), dim3((unsigned)N), dim3(256), 0, s, q, k,
                         q_out, n_head, n_rot, cos_t, sin_t, end, tab, c);
    hipLaunchKernelGGL((k_paged_append<HD, T>), dim3((unsigned)(n_qk + n_v)), dim3(256), 0, s, q,
                       k, v, q_out, N, n_head, n_rot, neox, cos_t, sin_t, end, tab, c,
                       (unsigned)per_token, (unsigned)per_group, (unsigned)n_qk);
  });
  return hipGetLastError();
}

hipError_t launch_paged_read(int64_t N, const PagedTable &tab, const aq_paged &c, void *k, void *v,
                             hipStream_t s) {
  const int64_t per_token = ((int64_t)c.n_kv * c.head_dim / 8 + 255) / 256;
  const int64_t per_group = ((int64_t)c.n_kv * c.head_dim / 4 + 255) / 256;
  const int64_t n_k = N * per_token, n_v = (N + 6) / 4 * per_group;
  if (n_k + n_v > kMaxGrid) return hipErrorInvalidValue;
  by_shape(c, [&](auto hd, auto) {
    hipLaunchKernelGGL((k_paged_read<decltype(hd)::value>), dim3((unsigned)(n_k + n_v)), dim3(256),
                       0, s, N, tab, c, static_cast<uint16_t *>(k), static_cast<uint16_t *>(v),
                       (unsigned)per_token, (unsigned)per_group, (unsigned)n_k);
  });
  return hipGetLastError();
}

bool attention_paged_fits(const aq_paged &c, int64_t N, int n_head, int64_t width,
                          int64_t start) {
  // (splits are held below the bound, and the prefix's workgroups are fewer than
  // N n_head / 16 + n_kv + 512: no plan is made for ordinary calls)
  if (N * n_head <= 1 << 22) return true;
  const PagedPlan p = paged_plan(c, N, n_head, width, start);
  return (int64_t)p.pre + p.own <= kMaxGrid && (p.states() <= 8 || N * n_head <= kMaxGrid);
}

size_t attention_paged_scratch(const aq_paged &c, int64_t N, int n_head, int64_t width,
                               int64_t start) {
  const PagedPlan p = paged_plan(c, N, n_head, width, start);
  return p.states() == 1 ? 0 : (size_t)N * n_head * p.states() * (c.head_dim + 4) * sizeof(float);
}

hipError_t launch_attention_paged(const float *q, int64_t N, int n_head, const PagedTable &tab,
                                  const PagedTable &pre, const aq_paged &c, float *states,
                                  float *out, hipStream_t s) {
  const PagedPlan p = paged_plan(c, N, n_head, tab.width, tab.start);
  hipError_t e = hipSuccess;
  by_shape(c, [&](auto hd, auto t) {
    constexpr int HD = decltype(hd)::value;
    auto go = [&](auto tw) {
      constexpr int TW = decltype(tw)::value;
      auto kern = k_paged_attn<HD, decltype(t), TW>;
      constexpr int merge = 4 * 16 * (HD + 4) * (int)sizeof(float);
      constexpr int lds = TW == 1 ? merge : std::max(merge, 2 * Stage<HD, TW>::BYTES);
      e = set_dynamic_lds(reinterpret_cast<const void *>(kern), lds);
      if (e != hipSuccess) return;
      hipLaunchKernelGGL(kern, dim3(p.pre + p.own), dim3(256), lds, s, q, N, n_head, tab, pre, c, p,
                         states, out);
    };
    if (p.tw == 1) go(std::integral_constant<int, 1>());
    else if (p.tw == 2) go(std::integral_constant<int, 2>());
    else go(std::integral_constant<int, 4>());
    if (e != hipSuccess) return;
    if (p.states() > 8)
      hipLaunchKernelGGL((k_paged_merge<HD, 256>), dim3((unsigned)(N * n_head)), dim3(256), 0, s,
                         states, N * n_head, p.states(), out);
    else if (p.states() > 1)
      hipLaunchKernelGGL((k_paged_merge<HD, 64>), dim3((unsigned)((N * n_head + 3) / 4)),
                         dim3(256), 0, s, states, N * n_head, p.states(), out);
  });
  return e == hipSuccess ? hipGetLastError() : e;
}

}  // namespace aq
