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

#include <type_traits>

#include "aq_internal.h"

namespace aq {
namespace {

constexpr int kBlk = 32;

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

// the block that holds slot `slot` of row `seq`: its number in the pool's blocks of
// kv head 0, or -1
__device__ __forceinline__ int64_t block_of(const aq_paged &c, const PagedTable &t, int64_t seq,
                                            int64_t slot) {
  const int64_t per = c.page_size / kBlk;
  if (seq < 0 || seq >= t.seqs || slot < 0 || slot >= t.width * c.page_size) return -1;
  const int64_t id = t.pages[seq * t.width + slot / c.page_size];
  if (id < 0 || id >= c.n_pages) return -1;
  return id * c.n_kv * per + slot % c.page_size / kBlk;
}

// ---- rotation and append -------------------------------------------------------
template <int HD, typename T>
__global__ void __launch_bounds__(256)
    k_paged_append(const float *q, const float *__restrict__ k, const float *__restrict__ v,
                   float *q_out, int n_head, int n_rot, int neox, const float *__restrict__ cos_t,
                   const float *__restrict__ sin_t, int64_t n_pos, PagedTable tab, aq_paged c) {
#pragma clang fp contract(off)
  const int64_t n = blockIdx.x;
  const int64_t pos = tab.pos[n], seq = tab.seq ? tab.seq[n] : n;
  if (pos < 0 || (n_rot && pos >= n_pos)) return;
  const int64_t slot = pos - tab.start, blk = block_of(c, tab, seq, slot);
  const int s = (int)(slot & (kBlk - 1)), half = n_rot / 2, pairs = HD / 2;
  const int heads = (q ? n_head : 0) + c.n_kv;
  for (int j = threadIdx.x; j < heads * pairs; j += 256) {
    int h = j / pairs;
    const int i = j % pairs;
    const bool is_k = h < c.n_kv;
    if (!is_k) h -= c.n_kv;
    if (is_k && blk < 0) continue;
    int a, b;
    if (i < half) {
      a = neox ? i : 2 * i;
      b = neox ? i + half : 2 * i + 1;
    } else {
      a = n_rot + 2 * (i - half);
      b = a + 1;
    }
    const float *src = is_k ? k + (n * c.n_kv + h) * HD : q + (n * n_head + h) * HD;
    float x0 = src[a], x1 = src[b];
    if (i < half) {
      const float cs = cos_t[pos * half + i], sn = sin_t[pos * half + i];
      const float r0 = x0 * cs - x1 * sn;
      const float r1 = x0 * sn + x1 * cs;
      x0 = r0;
      x1 = r1;
    }
    if (!is_k) {
      float *dst = q_out + (n * n_head + h) * HD;
      dst[a] = x0;
      dst[b] = x1;
      continue;
    }
    const int64_t at = (blk + (int64_t)h * (c.page_size / kBlk)) * (kBlk * HD);
    T *kp = static_cast<T *>(c.k) + at, *vp = static_cast<T *>(c.v) + at;
    const float *vs = v + (n * c.n_kv + h) * HD;
    kp[k_place<HD>(s, a)] = rounded<T>(x0);
    kp[k_place<HD>(s, b)] = rounded<T>(x1);
    vp[v_place(s, a)] = rounded<T>(vs[a]);
    vp[v_place(s, b)] = rounded<T>(vs[b]);
  }
}

// ---- read-back -------------------------------------------------------------------
template <int HD>
__global__ void __launch_bounds__(256)
    k_paged_read(PagedTable tab, aq_paged c, uint16_t *__restrict__ ko, uint16_t *__restrict__ vo) {
  const int64_t n = blockIdx.x;
  const int64_t pos = tab.pos[n], seq = tab.seq ? tab.seq[n] : n;
  const int64_t slot = pos - tab.start, blk = pos < 0 ? -1 : block_of(c, tab, seq, slot);
  const int s = (int)(slot & (kBlk - 1));
  for (int j = threadIdx.x; j < c.n_kv * HD; j += 256) {
    const int h = j / HD, d = j % HD;
    const int64_t at = (blk + (int64_t)h * (c.page_size / kBlk)) * (kBlk * HD);
    ko[n * c.n_kv * HD + j] = blk < 0 ? 0 : static_cast<uint16_t *>(c.k)[at + k_place<HD>(s, d)];
    vo[n * c.n_kv * HD + j] = blk < 0 ? 0 : static_cast<uint16_t *>(c.v)[at + v_place(s, d)];
  }
}

// ---- attention -----------------------------------------------------------------
// Tiles of 16 query rows of one kv head, blocks of 32 positions, on the
// 16x16x32 matrix instructions of the cache's type, with every fp32 operand in
// pieces of that type (x = sum of pieces: two of fp16, 22 bits; three of bf16, 24):
//   S^T (positions x rows) = K Q^T, Q's row times log2(e) / sqrt(head_dim) and a
//     power of two that brings its largest value to [2^14, 2^15): lane l holds row
//     l % 16's scores at positions 16 pt + 4 (l / 16) + r (pt = 0, 1; r = 0 .. 3);
//   O^T (dimensions x rows) += V^T P^T: those eight weights are the lane's operand
//     as it holds them.  Lane l gets row l % 16's dimensions 16 dt + 4 (l / 16) + r.
// Weights are P = 2^(z - m + 14), m the running maximum rounded up to a whole
// number, so that rescaling is exact and rare, and the pieces hold 22 bits of what
// counts.  The sum of the weights is kept per lane, in fp32.
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef unsigned int u4v __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

constexpr float kTop = 14.f;  // weights reach 2^14 in the pieces

template <typename T>
struct Ops;
template <>
struct Ops<_Float16> {
  static constexpr int NP = 2;
  static __device__ __forceinline__ f4v mfma(u4v a, u4v b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a),
                                                  __builtin_bit_cast(h8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t take(float &a, float &b) {
    const h2 h = __builtin_convertvector(f2v{a, b}, h2);
    a -= (float)h[0];
    b -= (float)h[1];
    return __builtin_bit_cast(uint32_t, h);
  }
};
template <>
struct Ops<__bf16> {
  static constexpr int NP = 3;
  static __device__ __forceinline__ f4v mfma(u4v a, u4v b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a),
                                                   __builtin_bit_cast(b8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t take(float &a, float &b) {
    const b2 h = __builtin_convertvector(f2v{a, b}, b2);
    a -= (float)h[0];
    b -= (float)h[1];
    return __builtin_bit_cast(uint32_t, h);
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
// q log2(e) / sqrt(HD) 2^-back.  A row with an infinity or a NaN is NaN.
template <int HD, typename T>
struct QRow {
  static constexpr int NP = Ops<T>::NP;
  u4v piece[NP][HD / 32];
  int back;
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
        for (int e = 0; e < 4; ++e) v[ks][4 * i + e] = live ? x[e] * f : 0.f;
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
    const int up = am > 0.f && !bad ? 15 - __builtin_amdgcn_frexp_expf(am) : 0;
    back = -up;
#pragma unroll
    for (int ks = 0; ks < HD / 32; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a = ldexpf(v[ks][2 * i], up), b = ldexpf(v[ks][2 * i + 1], up);
        a = bad ? NAN : a;
        b = bad ? NAN : b;
#pragma unroll
        for (int p = 0; p < NP; ++p) piece[p][ks][i] = Ops<T>::take(a, b);
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

// raw scores of a block (a tile of positions each) to weights in pieces; the state
// moves on to the new maximum.  Positions from `rem` on do not exist.
template <int HD, typename T>
__device__ __forceinline__ void weigh(f4v (&sc)[2], int back, int rem, RowState<HD> &st,
                                      u4v (&w)[Ops<T>::NP]) {
  const int cg = (threadIdx.x >> 4) & 3;
  float top = -INFINITY;
#pragma unroll
  for (int pt = 0; pt < 2; ++pt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float z = ldexpf(sc[pt][r], back);
      if (16 * pt + 4 * cg + r >= rem) z = -INFINITY;
      sc[pt][r] = z;
      top = fmaxf(top, z);
    }
  if (__any(top > st.m)) {
    const float m = fmaxf(st.m, ceilf(row_max(top)));
    const float f = st.m == -INFINITY ? 0.f : exp2_(st.m - m);
    st.m = m;
    st.l *= f;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) st.o[i] *= f;
  }
  const float ref = finite_ref(st.m) - kTop;
  float p[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    p[e] = exp2_(sc[e >> 2][e & 3] - ref);
    st.l += p[e];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < Ops<T>::NP; ++n) w[n][i] = Ops<T>::take(p[2 * i], p[2 * i + 1]);
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
  const int per = c.page_size / kBlk;
  if (b >= end) return -1;
  const int64_t id = pages[b / per];
  if (id < 0 || id >= c.n_pages) return -1;
  return (id * c.n_kv + h) * per + b % per;
}
__device__ __forceinline__ int64_t of_lane(int64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// RT tiles of rows against blocks b0 + wave, b0 + wave + 4, .. below b1 of a list
// of pages that holds len positions.  A wave's next keys are on their way while
// it weighs the present ones.
template <int HD, typename T, int RT>
__device__ __forceinline__ void attend_blocks(const aq_paged &c, const int32_t *pages, int h,
                                              int64_t b0, int64_t b1, int64_t len,
                                              const QRow<HD, T> (&q)[RT], RowState<HD> (&st)[RT]) {
  constexpr int KS = HD / 32, DT = HD / 16;
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
      const int64_t after = len - (base + 4 * i) * kBlk;
      const int rem = after < kBlk ? (int)after : kBlk;
#pragma unroll
      for (int j = 0; j < DT; ++j) v[j] = vp[at + 64 * j];
      f4v sc[RT][2];
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) {
          sc[t][pt] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int p = Ops<T>::NP - 1; p >= 0; --p)
              sc[t][pt] = Ops<T>::mfma(k[pt * KS + ks], q[t].piece[p][ks], sc[t][pt]);
        }
      if (left) {
        i = __builtin_ctzll(left);
        at = of_lane(mine, i) * (kBlk * HD / 8);
#pragma unroll
        for (int j = 0; j < 2 * KS; ++j) k[j] = kp[at + 64 * j];
      }
      if (rem < kBlk) {
#pragma unroll
        for (int j = 0; j < DT; ++j) v[j] = only_first(v[j], rem);
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        u4v w[Ops<T>::NP];
        weigh<HD, T>(sc[t], q[t].back, rem, st[t], w);
#pragma unroll
        for (int j = 0; j < DT; ++j)
#pragma unroll
          for (int p = Ops<T>::NP - 1; p >= 0; --p)
            st[t].o[j] = Ops<T>::mfma(v[j], w[p], st[t].o[j]);
      }
    }
  }
}

// The partial state of a row: HD numerators relative to 2^(m - kTop), m, l.
template <int HD>
constexpr int kState = HD + 4;

// How a call's work is split (host and kernels).
struct PagedPlan {
  int rt;          // tiles of 16 rows that a wave takes of the prefix
  int groups;      // groups of 16 rt rows of a kv head
  int sp, ss;      // splits of the prefix and of a row's own positions
  int states() const { return sp + ss; }
};

template <int HD>
__device__ __forceinline__ void put_dead(float *state) {
  state[HD] = -INFINITY;
  state[HD + 1] = 0.f;
}

// Workgroups 0 .. n_pre - 1: split, group of rows and kv head of the prefix; then
// split, kv head and row of the rows' own positions (a row that ends inside the
// prefix has that part of it as its own).  The four waves take every fourth block
// each and their states are merged through LDS.
template <int HD, typename T, int RT>
__global__ void __launch_bounds__(256, HD == 256 ? 1 : 2)
    k_paged_attn(const float *__restrict__ q, int64_t N, int n_head, PagedTable tab,
                 PagedTable pre, aq_paged c, PagedPlan plan, float *__restrict__ states,
                 float *__restrict__ out) {
  constexpr int LD = HD + 4;
  __shared__ __attribute__((aligned(16))) float num[4][16][LD];
  __shared__ float mm[4][16], ll[4][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, cg = lane >> 4;
  const int G = n_head / c.n_kv, S = plan.sp + plan.ss;
  const int n_pre = plan.sp * plan.groups * c.n_kv;
  const bool is_pre = (int)blockIdx.x < n_pre;
  int h, split;
  int64_t len, b0, b1;
  const int32_t *pages;
  const int64_t rows = N * G;  // of a kv head
  int64_t row0 = 0;            // of the group
  int64_t n = 0;
  if (is_pre) {
    int x = blockIdx.x;
    split = x % plan.sp;
    x /= plan.sp;
    h = x % c.n_kv;
    row0 = (int64_t)(x / c.n_kv) * (16 * RT);
    pages = pre.pages;
    len = pre.start;
    const int64_t blocks = (len + kBlk - 1) / kBlk, each = (blocks + plan.sp - 1) / plan.sp;
    b0 = split * each;
    b1 = b0 + each < blocks ? b0 + each : blocks;
  } else {
    int64_t x = (int64_t)blockIdx.x - n_pre;
    split = (int)(x % plan.ss);
    x /= plan.ss;
    h = (int)(x % c.n_kv);
    n = x / c.n_kv;
    row0 = n * G;
    const int64_t pos = tab.pos[n], seq = tab.seq ? tab.seq[n] : n;
    len = 0;
    pages = nullptr;
    if (pos >= 0 && pos < pre.start) {
      pages = pre.pages;
      len = pos + 1;
    } else if (pos >= 0 && seq >= 0 && seq < tab.seqs) {
      pages = tab.pages + seq * tab.width;
      const int64_t room = tab.width * c.page_size;
      len = pos - tab.start < room ? pos - tab.start + 1 : room;
    }
    const int64_t blocks = (len + kBlk - 1) / kBlk;
    int64_t each = (blocks + plan.ss - 1) / plan.ss;
    each = each > 4 ? each : 4;
    b0 = split * each;
    b1 = b0 + each < blocks ? b0 + each : blocks;
    split += plan.sp;
  }
  auto write = [&](auto &st, int64_t first, int64_t end) {  // rows first .. of this tile
    const float l = row_sum(st.l);
#pragma unroll
    for (int d = 0; d < HD / 16; ++d)
      *reinterpret_cast<f4v *>(&num[wave][j][16 * d + 4 * cg]) = st.o[d];
    if (cg == 0) mm[wave][j] = st.m, ll[wave][j] = l;
    __syncthreads();
    // 16 threads a row
    const int r = threadIdx.x >> 4, part = threadIdx.x & 15;
    const int64_t row = first + r;
    if (row < end) {
      const float m = fmaxf(fmaxf(mm[0][r], mm[1][r]), fmaxf(mm[2][r], mm[3][r]));
      float f[4], sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        f[w] = mm[w][r] == -INFINITY ? 0.f : exp2_(mm[w][r] - m);
        sum += ll[w][r] == 0.f ? 0.f : ll[w][r] * (m == -INFINITY ? 1.f : f[w]);
      }
      const int64_t i = row / G, head = (int64_t)h * G + row % G;
      const int64_t flat = i * n_head + head;
      const bool skip = is_pre && tab.pos[i] < pre.start;
      float *dst = S == 1 ? out + flat * HD : states + (flat * S + split) * kState<HD>;
      const float inv = S == 1 ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
#pragma unroll
      for (int d = 4 * part; d < HD; d += 64) {
        f4v o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) o += f[w] * *reinterpret_cast<const f4v *>(&num[w][r][d]);
        *reinterpret_cast<f4v *>(dst + d) = o * inv;
      }
      if (S != 1 && part == 0) {
        dst[HD] = skip ? -INFINITY : m;
        dst[HD + 1] = skip ? 0.f : sum;
      }
    }
    __syncthreads();
  };
  if (is_pre) {
    QRow<HD, T> qr[RT];
    RowState<HD> st[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int64_t row = row0 + 16 * t + j;
      const bool live = row < rows;
      const int64_t i = live ? row / G : 0, head = (int64_t)h * G + (live ? row % G : 0);
      qr[t].load(q + (i * n_head + head) * HD, live);
      st[t].clear();
    }
    attend_blocks<HD, T, RT>(c, pages, h, b0, b1, len, qr, st);
#pragma unroll
    for (int t = 0; t < RT; ++t) write(st[t], row0 + 16 * t, rows);
  } else {
    if (b0 >= b1 && S != 1) {  // nothing of the row here
      if ((int)threadIdx.x < G)
        put_dead<HD>(states + ((n * n_head + h * G + threadIdx.x) * S + split) * kState<HD>);
      return;
    }
    QRow<HD, T> qr[1];
    RowState<HD> st[1];
    qr[0].load(q + (n * n_head + h * G + (j < G ? j : 0)) * HD, j < G);
    st[0].clear();
    attend_blocks<HD, T, 1>(c, pages, h, b0, b1, len, qr, st);
    write(st[0], row0, row0 + G);
  }
}

// One wave an output row: the states of its splits, at most 64.
template <int HD>
__global__ void __launch_bounds__(256)
    k_paged_merge(const float *__restrict__ states, int64_t rows, int S, float *__restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  states += row * S * kState<HD>;
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
  constexpr int PER = HD / 64;
  float o[PER] = {};
  uint64_t left = __ballot(some);
  while (left) {
    const int s = __builtin_ctzll(left);
    left &= left - 1;
    const float fs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), s));
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = fmaf(states[s * kState<HD> + PER * lane + i], fs, o[i]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < PER; ++i) out[row * HD + PER * lane + i] = o[i] * inv;
}

PagedPlan paged_plan(const aq_paged &c, int64_t N, int n_head, int64_t width, int64_t start) {
  const int64_t rows = N * (n_head / c.n_kv), want = 512;
  PagedPlan p = {1, 0, 0, 1};
  auto splits = [&](int64_t items, int64_t blocks) {  // at least a block a wave
    int64_t s = (want + items - 1) / items;
    const int64_t most = (blocks + 3) / 4;
    s = s < most ? s : most;
    return (int)(s < 1 ? 1 : s > 32 ? 32 : s);
  };
  if (start > 0) {
    p.rt = rows > 16 && c.head_dim < 256 ? 2 : 1;
    p.groups = (int)((rows + 16 * p.rt - 1) / (16 * p.rt));
    p.sp = splits((int64_t)p.groups * c.n_kv, (start + kBlk - 1) / kBlk);
  }
  p.ss = splits(N * c.n_kv, width * c.page_size / kBlk);
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
  by_shape(c, [&](auto hd, auto t) {
    hipLaunchKernelGGL((k_paged_append<decltype(hd)::value, decltype(t)>), dim3((unsigned)N),
                       dim3(256), 0, s, q, k, v, q_out, n_head, n_rot, neox, cos_t, sin_t, n_pos,
                       tab, c);
  });
  return hipGetLastError();
}

hipError_t launch_paged_read(int64_t N, const PagedTable &tab, const aq_paged &c, void *k, void *v,
                             hipStream_t s) {
  by_shape(c, [&](auto hd, auto) {
    hipLaunchKernelGGL((k_paged_read<decltype(hd)::value>), dim3((unsigned)N), dim3(256), 0, s,
                       tab, c, static_cast<uint16_t *>(k), static_cast<uint16_t *>(v));
  });
  return hipGetLastError();
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
  const int64_t wgs = (int64_t)p.sp * p.groups * c.n_kv + (int64_t)p.ss * N * c.n_kv;
  by_shape(c, [&](auto hd, auto t) {
    constexpr int HD = decltype(hd)::value;
    auto go = [&](auto kern) {
      hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(256), 0, s, q, N, n_head, tab, pre, c, p,
                         states, out);
    };
    if constexpr (HD < 256) {
      if (p.rt == 2) go(k_paged_attn<HD, decltype(t), 2>);
      else go(k_paged_attn<HD, decltype(t), 1>);
    } else {
      go(k_paged_attn<HD, decltype(t), 1>);
    }
    if (p.states() > 1)
      hipLaunchKernelGGL((k_paged_merge<HD>), dim3((unsigned)((N * n_head + 3) / 4)), dim3(256), 0,
                         s, states, N * n_head, p.states(), out);
  });
  return hipGetLastError();
}

}  // namespace aq
