// aq_kv8.hip - the 8-bit KV cache: rotation and store, attention, read-back.
//
// Values are coded in blocks of kKv8Block = 32 positions of one kv head, K and
// V apart: s = fl32(amax / 127) over the tokens the block holds so far, and a
// value x is the whole number c nearest to x / s (ties to even), standing for
// s c.  The last block stored is kept in fp32 too (the tail), so a block that a
// token joins is coded anew from its own values: the codes are a function of
// the tokens alone, not of the calls that brought them, and no error adds up.
//
// Layouts (n_blocks = ceil(n_ctx / 32) per kv head):
//   K codes [n_kv][n_blocks][32 positions][head_dim]
//   V codes [n_kv][n_blocks][head_dim / 2][4 g][2 dimensions][8 positions],
//     the eight positions 16 pt + 4 g + r (pt = 0, 1; r = 0 .. 3) of a dimension
//     side by side: what a lane of the matrix instructions takes as its operand
//     (the scores' lanes hold the weights of these positions), two dimensions
//     per 16-byte load
//   scales [n_kv][n_blocks] fp32; tails [n_kv][32][head_dim] fp32.
#include <math.h>

#include "aq_internal.h"

namespace aq {
namespace {

constexpr int kBlk = kKv8Block;
constexpr int kWG = 256;

typedef float f4v __attribute__((ext_vector_type(4)));

// byte of position row (0 .. 31) and dimension d in a V block
__device__ __forceinline__ int v_byte(int row, int d) {
  return (d >> 1) * 64 + ((row >> 2) & 3) * 16 + (d & 1) * 8 + (row >> 4) * 4 + (row & 3);
}

// positions p0 .. p0 + n of a call that lie in the cache (n = 0: none)
struct Span {
  int64_t p0, n;
};
__device__ __forceinline__ Span span_of(const aq_decode_state *st, int64_t pos0, int64_t T,
                                        int64_t n_ctx) {
  const int64_t p0 = st ? (int64_t)st->pos : pos0;
  if (p0 < 0 || p0 >= n_ctx) return {0, 0};
  return {p0, T < n_ctx - p0 ? T : n_ctx - p0};
}

// element d of a head vector, rotated for position pos: pairs (2i, 2i + 1) or,
// neox, (i, i + n_rot / 2); products and differences rounded separately
__device__ __forceinline__ float rotated(const float *x, int d, int64_t pos, int n_rot,
                                         int neox, const float *__restrict__ cos_t,
                                         const float *__restrict__ sin_t) {
#pragma clang fp contract(off)
  if (d >= n_rot) return x[d];
  const int half = n_rot / 2;
  const int i = neox ? (d < half ? d : d - half) : d >> 1;
  const bool lo = neox ? d < half : !(d & 1);
  const int other = neox ? (lo ? d + half : d - half) : d ^ 1;
  const float c = cos_t[pos * half + i], s = sin_t[pos * half + i];
  const float a = x[d], b = x[other];
  return lo ? a * c - b * s : b * s + a * c;
}

// the whole number nearest to x / s, ties to even, exactly: rem is x - r s
// without rounding (a multiple of the smaller of their units, below 2^24 of
// it), so it tells which side of a half the quotient lies on
__device__ __forceinline__ int code_of(float x, float s) {
#pragma clang fp contract(off)
  if (!(s > 0.f)) return 0;  // an empty block's scale, or a NaN
  float r = rintf(x / s);
  const float rem = fmaf(-r, s, x), two = 2.f * fabsf(rem);
  if (two > s || (two == s && ((int)r & 1))) r += copysignf(1.f, rem);
  return (int)fminf(fmaxf(r, -127.f), 127.f);
}

// ---- rotation and store ------------------------------------------------------
// Workgroups 0 .. n_store - 1 code one block of one kv head each, K or V: the
// block's tokens go to LDS (those before the call's from the tail, the call's
// own rotated), their largest magnitude gives the scale, and every thread codes
// 16-byte units.  Slots past the last token are cleared.  The workgroup of the
// call's first block also keeps the tail: it alone reads it (before), and
// writes the tokens of the last block (after), so no two workgroups meet there.
// The rest rotate q.
template <int HD>
__global__ void __launch_bounds__(kWG)
    k_kv8_store(const float *q, const float *__restrict__ k, const float *__restrict__ v,
                float *q_out, int64_t T, int n_head,
                int n_rot, int neox, const float *__restrict__ cos_t,
                const float *__restrict__ sin_t, const aq_decode_state *st, int64_t pos0, aq_kv8 c,
                int64_t n_store) {
  __shared__ __attribute__((aligned(16))) float xs[kBlk * HD];
  __shared__ uint32_t red[kWG / 64];
  const Span sp = span_of(st, pos0, T, c.n_ctx);
  if (sp.n == 0) return;
  const int tid = threadIdx.x;
  if ((int64_t)blockIdx.x >= n_store) {  // q: one element a thread, in place allowed by pairs
    const int64_t n = sp.n * n_head * (HD / 2);
    for (int64_t i = ((int64_t)blockIdx.x - n_store) * kWG + tid; i < n;
         i += (int64_t)(gridDim.x - n_store) * kWG) {
      const int64_t t = i / (n_head * (HD / 2));
      const int r = (int)(i - t * (n_head * (HD / 2)));
      const int h = r / (HD / 2), j = r - h * (HD / 2), half = n_rot / 2;
      int a, b;
      if (j < half) {
        a = neox ? j : 2 * j;
        b = neox ? j + half : 2 * j + 1;
      } else {
        a = n_rot + 2 * (j - half);
        b = a + 1;
      }
      const float *x = q + (t * n_head + h) * HD;
      const float ra = rotated(x, a, sp.p0 + t, n_rot, neox, cos_t, sin_t);
      const float rb = rotated(x, b, sp.p0 + t, n_rot, neox, cos_t, sin_t);
      float *y = q_out + (t * n_head + h) * HD;
      y[a] = ra;
      y[b] = rb;
    }
    return;
  }
  const int which = (int)(blockIdx.x & 1);
  const int kvh = (int)((blockIdx.x >> 1) % c.n_kv);
  const int64_t b0 = sp.p0 / kBlk, bl = (sp.p0 + sp.n - 1) / kBlk;
  const int64_t b = b0 + (int64_t)(blockIdx.x >> 1) / c.n_kv;
  if (b > bl) return;
  const float *src = which ? v : k;
  float *tail = (which ? c.v_tail : c.k_tail) + (int64_t)kvh * kBlk * HD;
  // the call's value at position p (p0 <= p < p0 + n)
  auto fresh = [&](int64_t p, int d) {
    const float *x = src + ((p - sp.p0) * c.n_kv + kvh) * HD;
    return which ? x[d] : rotated(x, d, p, n_rot, neox, cos_t, sin_t);
  };
  uint32_t am = 0;  // the largest magnitude, as bits (a NaN's lie above infinity's)
  for (int i = tid; i < kBlk * HD; i += kWG) {
    const int row = i / HD, d = i - row * HD;
    const int64_t p = b * kBlk + row;
    float x = 0.f;
    if (p < sp.p0) x = tail[i];
    else if (p < sp.p0 + sp.n) x = fresh(p, d);
    xs[i] = x;
    am = max(am, __float_as_uint(x) & 0x7FFFFFFFu);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) am = max(am, (uint32_t)__shfl_xor((int)am, off));
  if ((tid & 63) == 0) red[tid >> 6] = am;
  __syncthreads();  // (and the tail has been read)
#pragma unroll
  for (int w = 0; w < kWG / 64; ++w) am = max(am, red[w]);
  const float s = am >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __uint_as_float(am) / 127.f;
  const int64_t n_blocks = (c.n_ctx + kBlk - 1) / kBlk;
  if (tid == 0) (which ? c.v_scale : c.k_scale)[kvh * n_blocks + b] = s;
  int8_t *dst = (which ? c.v : c.k) + (kvh * n_blocks + b) * (kBlk * HD);
  for (int u = tid; u < kBlk * HD / 16; u += kWG) {
    union {
      int8_t c8[16];
      uint4 w;
    } o;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      int row, d;
      if (which) {  // unit (dimension pair, g): 2 dimensions x 8 positions
        row = 16 * ((e >> 2) & 1) + 4 * (u & 3) + (e & 3);
        d = 2 * (u >> 2) + (e >> 3);
      } else {
        row = u / (HD / 16);
        d = 16 * (u % (HD / 16)) + e;
      }
      o.c8[e] = (int8_t)code_of(xs[row * HD + d], s);
    }
    reinterpret_cast<uint4 *>(dst)[u] = o.w;
  }
  if (b == b0) {  // the tail: the last block's tokens of this call
    const int64_t first = bl == b0 ? sp.p0 : bl * kBlk;
    const int n = (int)(sp.p0 + sp.n - first), r0 = (int)(first - bl * kBlk);
    for (int i = tid; i < n * HD; i += kWG) {
      const int row = i / HD, d = i - row * HD;
      tail[(r0 + row) * HD + d] = fresh(first + row, d);
    }
  }
}

// ---- read-back ---------------------------------------------------------------
// out[kvh][p - start][d] = s c, one product rounded to fp32
template <int HD>
__global__ void __launch_bounds__(kWG)
    k_kv8_read(aq_kv8 c, int64_t start, int64_t n, float *__restrict__ ko,
               float *__restrict__ vo) {
  const int64_t n_blocks = (c.n_ctx + kBlk - 1) / kBlk;
  const int64_t total = (int64_t)c.n_kv * n * HD;
  for (int64_t i = (int64_t)blockIdx.x * kWG + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * kWG) {
    const int d = (int)(i % HD);
    const int64_t pp = i / HD, kvh = pp / n, p = start + (pp - kvh * n);
    const int64_t blk = kvh * n_blocks + p / kBlk;
    const int row = (int)(p % kBlk);
    ko[i] = c.k_scale[blk] * (float)c.k[blk * (kBlk * HD) + row * HD + d];
    vo[i] = c.v_scale[blk] * (float)c.v[blk * (kBlk * HD) + v_byte(row, d)];
  }
}

// ---- attention -----------------------------------------------------------------
// Both kernels below work on tiles of 16 query rows of one kv head (row id =
// token * G + head in the group, any G up to 16) with
// v_mfma_f32_16x16x32_f16, the codes as exact fp16 operands and every fp32
// operand in two fp16 pieces (x = hi + lo, 24 bits where lo is normal):
//   S^T (positions x rows) = C_K Q^T, Q's row scaled by a power of two to a
//     largest value in [2^14, 2^15): lane l holds row l % 16's scores at
//     positions 16 pt + 4 (l / 16) + r of a block (pt = 0, 1; r = 0 .. 3);
//   O^T (dimensions x rows) += C_V^T P^T: those 8 weights are the lane's B
//     operand as it holds them (the V layout stores positions in that order).
// The block's K scale enters as the factor of its raw scores, its V scale in
// the weights: P = 2^(z - m) s_V, formed relative to the largest such product
// the row has met, 2^R, so the pieces hold 24 bits of whatever counts and no
// magnitude of V over- or underflows them.  m and R are rounded up to whole
// numbers, so every rescaling is an exact power of two.  The sum of 2^(z - m)
// is kept per lane.
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef unsigned int u4v __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kTop = 14.f;      // weights reach 2^14 in the pieces
constexpr float kLow = -1e30f;    // R before any weight

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

// four signed codes as exact fp16: 1024 + (c + 128) by its bits, less 1152
__device__ __forceinline__ void codes4(uint32_t w, uint32_t &a, uint32_t &b) {
  w ^= 0x80808080u;
  const h2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
  a = __builtin_bit_cast(
      uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + off);
  b = __builtin_bit_cast(
      uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + off);
}
// 16 codes as two operands of 8
__device__ __forceinline__ void codes16(u4v w, h8 &lo, h8 &hi) {
  u4v a, b;
  uint32_t x, y;
  codes4(w[0], x, y);
  a[0] = x, a[1] = y;
  codes4(w[1], x, y);
  a[2] = x, a[3] = y;
  codes4(w[2], x, y);
  b[0] = x, b[1] = y;
  codes4(w[3], x, y);
  b[2] = x, b[3] = y;
  lo = __builtin_bit_cast(h8, a);
  hi = __builtin_bit_cast(h8, b);
}
// (a, b) as pieces: fp16 of the value, and fp16 of what that leaves
__device__ __forceinline__ void pieces2(float a, float b, uint32_t &hi, uint32_t &lo) {
  const h2 h = __builtin_convertvector(f2v{a, b}, h2);
  const h2 l = __builtin_convertvector(
      f2v{fmaf((float)h[0], -1.f, a), fmaf((float)h[1], -1.f, b)}, h2);
  hi = __builtin_bit_cast(uint32_t, h);
  lo = __builtin_bit_cast(uint32_t, l);
}

// A lane's part of one query row: 8 dimensions 64 jj + 16 cg + 8 half .. per k
// step ks = 2 jj + half, in pieces, and the factor that turns raw scores into
// exponents of two (less the K scale).  A row with an infinity or a NaN gets
// the factor NaN.
template <int HD>
struct QRow {
  h8 hi[HD / 32], lo[HD / 32];
  float f;
  __device__ __forceinline__ void load(const float *__restrict__ q, bool live, int cg,
                                       float scale) {
    f4v v[HD / 16];
    float am = 0.f;
    bool fin = true;
#pragma unroll
    for (int ks = 0; ks < HD / 32; ++ks)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f4v x = {0.f, 0.f, 0.f, 0.f};
        if (live)
          x = *reinterpret_cast<const f4v *>(q + 64 * (ks >> 1) + 16 * cg + 8 * (ks & 1) + 4 * i);
        v[2 * ks + i] = x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          fin = fin && fabsf(x[e]) < INFINITY;
          am = fmaxf(am, fabsf(x[e]));
        }
      }
    am = row_max(am);
    const bool bad = row_max(fin ? 0.f : 1.f) != 0.f;
    const int up = am > 0.f && !bad ? 15 - __builtin_amdgcn_frexp_expf(am) : 0;
    f = bad ? __uint_as_float(0x7FC00000u) : ldexpf(scale * kLog2e, -up);
#pragma unroll
    for (int ks = 0; ks < HD / 32; ++ks) {
      u4v h, l;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f4v x = v[2 * ks + (i >> 1)];
        const float a = bad ? 0.f : ldexpf(x[2 * (i & 1)], up);
        const float b = bad ? 0.f : ldexpf(x[2 * (i & 1) + 1], up);
        uint32_t hh, ll;
        pieces2(a, b, hh, ll);
        h[i] = hh, l[i] = ll;
      }
      hi[ks] = __builtin_bit_cast(h8, h);
      lo[ks] = __builtin_bit_cast(h8, l);
    }
  }
};

// The running softmax of a lane's row: maximum m and reference R (both whole
// exponents of two, the same in the row's four lanes), the lane's part of the
// sum l, and the numerators, o[2 j + e][rr] at dimension 32 j + 8 cg + 2 rr + e,
// which stand for o 2^(R - m - kTop).
template <int HD>
struct RowState {
  float m, R, l;
  f4v o[HD / 16];
  __device__ __forceinline__ void clear() {
    m = -INFINITY, R = kLow, l = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) o[i] = f4v{0.f, 0.f, 0.f, 0.f};
  }
};

// NB blocks' raw scores sc (two tiles of positions each) to weights in pieces,
// with their K and V scales: m, R, l and o of the row move on.  MASK: only
// positions up to last[b], counted from the lane's first one in block b, exist.
template <int HD, int NB, bool MASK>
__device__ __forceinline__ void softmax_step(RowState<HD> &st, f4v (&sc)[2 * NB], float f,
                                             const float (&ks)[NB], const float (&vs)[NB],
                                             const int (&last)[NB], h8 (&ph)[NB], h8 (&pl)[NB]) {
  float c[NB], t[NB], ve[NB], mn = st.m, R = st.R;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    c[b] = ks[b] * f;
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = sc[2 * b + (i >> 2)][i & 3];
      mx = !MASK || 16 * (i >> 2) + (i & 3) <= last[b] ? fmaxf(mx, x) : mx;
    }
    mx = row_max(mx);
    t[b] = mx == -INFINITY ? mx : ceilf(mx * c[b]);  // (not through a masked block's scale)
    mn = fmaxf(mn, t[b]);
    ve[b] = (float)__builtin_amdgcn_frexp_expf(vs[b]);
    if (vs[b] > 0.f) R = fmaxf(R, t[b] + ve[b]);
  }
  const float mref = mn == -INFINITY ? 0.f : mn;
  const float corr = exp2_(st.m - mref), corr_o = exp2_(st.R - R);
  float sum = 0.f;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const float g =
        __builtin_amdgcn_frexp_mantf(vs[b]) * exp2_(fminf(ve[b] + mref - R + kTop, 120.f));
    u4v h, l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float p[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int j = 2 * i + k;
        const float e = exp2_(fmaf(sc[2 * b + (j >> 2)][j & 3], c[b], -mref));
        const bool see = !MASK || 16 * (j >> 2) + (j & 3) <= last[b];
        sum += see ? e : 0.f;
        p[k] = see ? e * g : 0.f;
      }
      uint32_t hh, ll;
      pieces2(p[0], p[1], hh, ll);
      h[i] = hh, l[i] = ll;
    }
    ph[b] = __builtin_bit_cast(h8, h);
    pl[b] = __builtin_bit_cast(h8, l);
  }
  st.l = fmaf(st.l, corr, sum);
  st.m = mn;
  st.R = R;
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) st.o[i] *= corr_o;
}

// v 2^(R - m - kTop) / den, the power in two whole parts so that neither leaves
// the range
struct OutScale {
  float a, b;
  __device__ __forceinline__ OutScale(float R, float m, float den) {
    const float x = R - m - kTop, h = floorf(0.5f * x);
    a = exp2_(h);
    b = exp2_(x - h);
    inv = 1.f / den;
  }
  float inv;
  template <class V>
  __device__ __forceinline__ V operator()(V v) const {
    return v * a * inv * b;
  }
};

// ---- few rows: the positions split over workgroups -------------------------------
// Workgroup (split j, kv head, tile of 16 rows): wave w takes blocks 4 j + w, + 4 S
// ..., straight from memory into operand order (no LDS), the next block's loads
// under way while one is computed; the waves' states meet in LDS, the splits'
// in k_kv8_combine.  One split writes the output itself.
constexpr int kWaves = 4;
template <int HD>
__global__ void __launch_bounds__(64 * kWaves)
    k_kv8_split(const float *__restrict__ q, aq_kv8 c, const aq_decode_state *st, int64_t pos0,
                int64_t T, int G, float scale, float *__restrict__ part,
                float *__restrict__ out) {
  constexpr int KJ = HD / 64, VJ = HD / 32, PS = HD + 4;
  constexpr int PARTS = HD == 256 ? 2 : 1, VP = VJ / PARTS;  // the merge's LDS: at most 32 KB
  __shared__ f4v os[kWaves][2 * VP][64];
  __shared__ float stat[kWaves][3][16];
  const Span sp = span_of(st, pos0, T, c.n_ctx);
  const int j = blockIdx.x, S = gridDim.x, kvh = blockIdx.y, n_head = gridDim.y * G;
  const int id0 = blockIdx.z * 16, rows = (int)sp.n * G;  // at most 65535 x 16
  if (id0 >= rows) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, cg = lane >> 4;
  const int id = id0 + r16, id_last = id0 + 15 < rows ? id0 + 15 : rows - 1;
  const bool live = id < rows;
  const int tok = live ? id / G : 0;
  const int g = live ? id - tok * G : 0;
  const int64_t lim = sp.p0 + tok;              // the row's last position
  const int64_t lim0 = sp.p0 + id0 / G;         // the tile's first row's
  const int nb = (int)((sp.p0 + id_last / G) / kBlk) + 1;  // blocks the tile sees
  const int64_t n_blocks = (c.n_ctx + kBlk - 1) / kBlk;
  const int8_t *kb = c.k + kvh * n_blocks * (kBlk * HD), *vb = c.v + kvh * n_blocks * (kBlk * HD);
  const float *ksc = c.k_scale + kvh * n_blocks, *vsc = c.v_scale + kvh * n_blocks;
  struct Buf {
    u4v k[2][KJ], v[VJ];
    float ks, vs;
  };
  auto load = [&](int b, Buf &x) {
    b = b < nb ? b : nb - 1;  // (past the last one: not used)
    const int8_t *kp = kb + (int64_t)b * (kBlk * HD), *vp = vb + (int64_t)b * (kBlk * HD);
#pragma unroll
    for (int pt = 0; pt < 2; ++pt)
#pragma unroll
      for (int jj = 0; jj < KJ; ++jj)
        x.k[pt][jj] = *reinterpret_cast<const u4v *>(kp + (16 * pt + r16) * HD + 64 * jj + 16 * cg);
#pragma unroll
    for (int i = 0; i < VJ; ++i)
      x.v[i] = *reinterpret_cast<const u4v *>(vp + ((16 * i + r16) * 4 + cg) * 16);
    x.ks = ksc[b];
    x.vs = vsc[b];
  };
  Buf b0, b1;
  int b = j * kWaves + wave;
  load(b, b0);
  QRow<HD> qr;
  qr.load(q + ((int64_t)tok * n_head + kvh * G + g) * HD, live, cg, scale);
  RowState<HD> s;
  s.clear();
  auto compute = [&](int blk, Buf &x) {
    f4v sc[2];
#pragma unroll
    for (int pt = 0; pt < 2; ++pt) {
      h8 kf[2 * KJ];
#pragma unroll
      for (int jj = 0; jj < KJ; ++jj) codes16(x.k[pt][jj], kf[2 * jj], kf[2 * jj + 1]);
      sc[pt] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < 2 * KJ; ++ks)
        sc[pt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[ks], qr.lo[ks], sc[pt], 0, 0, 0);
#pragma unroll
      for (int ks = 0; ks < 2 * KJ; ++ks)
        sc[pt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[ks], qr.hi[ks], sc[pt], 0, 0, 0);
    }
    h8 ph[1], pl[1];
    const float ks[1] = {x.ks}, vs[1] = {x.vs};
    const int64_t first = (int64_t)blk * kBlk;
    if (first + kBlk - 1 > lim0) {  // (uniform) some row ends inside the block or before it
      const int64_t d = lim - first - 4 * cg;
      const int last[1] = {(int)(d > 64 ? 64 : d < -1 ? -1 : d)};
      softmax_step<HD, 1, true>(s, sc, qr.f, ks, vs, last, ph, pl);
    } else {
      const int last[1] = {0};
      softmax_step<HD, 1, false>(s, sc, qr.f, ks, vs, last, ph, pl);
    }
#pragma unroll
    for (int i = 0; i < VJ; ++i) {
      h8 vf[2];
      codes16(x.v[i], vf[0], vf[1]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s.o[2 * i + e] =
            __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[e], pl[0], s.o[2 * i + e], 0, 0, 0);
        s.o[2 * i + e] =
            __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[e], ph[0], s.o[2 * i + e], 0, 0, 0);
      }
    }
  };
  const int stride = S * kWaves;
  while (b < nb) {
    load(b + stride, b1);
    compute(b, b0);
    if ((b += stride) >= nb) break;
    load(b + stride, b0);
    compute(b, b1);
    b += stride;
  }
  // the waves' states, then one state per row
  s.l = row_sum(s.l);
  if (cg == 0) {
    stat[wave][0][r16] = s.m;
    stat[wave][1][r16] = s.R;
    stat[wave][2][r16] = s.l;
  }
  float *dst = S == 1 ? out + ((int64_t)tok * n_head + kvh * G + g) * HD
                      : part + (((int64_t)kvh * T * G + id) * S + j) * PS;
  float M = -INFINITY, R = kLow, den = 0.f, fo[kWaves];
#pragma unroll
  for (int h = 0; h < PARTS; ++h) {
    if (h) __syncthreads();
#pragma unroll
    for (int i = 0; i < 2 * VP; ++i) os[wave][i][lane] = s.o[2 * VP * h + i];
    __syncthreads();
    if (h == 0) {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        M = fmaxf(M, stat[w][0][r16]);
        R = fmaxf(R, stat[w][1][r16]);
      }
      const float mref = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        den = fmaf(stat[w][2][r16], exp2_(stat[w][0][r16] - mref), den);
        fo[w] = exp2_(stat[w][1][r16] - R);
      }
    }
    const OutScale fin(R, M, den);
    for (int i = wave; i < VP; i += kWaves) {
      f4v a[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        a[e] = os[0][2 * i + e][lane] * fo[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) a[e] += os[w][2 * i + e][lane] * fo[w];
        if (S == 1) a[e] = fin(a[e]);
      }
      f4v *o4 = reinterpret_cast<f4v *>(dst + 32 * (VP * h + i) + 8 * cg);
      if (live) {
        o4[0] = f4v{a[0][0], a[1][0], a[0][1], a[1][1]};
        o4[1] = f4v{a[0][2], a[1][2], a[0][3], a[1][3]};
      }
    }
  }
  if (S > 1 && live && wave == 0 && cg == 0)
    *reinterpret_cast<f4v *>(dst + HD) = f4v{M, R, den, 0.f};
}

// One workgroup of HD threads per query row merges the splits' states.
template <int HD>
__global__ void __launch_bounds__(HD)
    k_kv8_combine(const float *__restrict__ part, const aq_decode_state *st, int64_t pos0,
                  int64_t n_ctx, int64_t T, int G, int S, float *__restrict__ out) {
  constexpr int PS = HD + 4;
  const Span sp = span_of(st, pos0, T, n_ctx);
  const int id = blockIdx.x, t = id / G;
  if (t >= sp.n) return;
  const int kvh = blockIdx.y, d = threadIdx.x, n_head = gridDim.y * G;
  const float *p = part + ((int64_t)kvh * T * G + id) * S * PS;
  float M = -INFINITY, R = kLow;
  for (int s = 0; s < S; ++s) {
    M = fmaxf(M, p[s * PS + HD]);
    R = fmaxf(R, p[s * PS + HD + 1]);
  }
  const float mref = M == -INFINITY ? 0.f : M;
  float num = 0.f, den = 0.f;
  for (int s = 0; s < S; ++s) {
    num = fmaf(p[s * PS + d], exp2_(p[s * PS + HD + 1] - R), num);
    den = fmaf(p[s * PS + HD + 2], exp2_(p[s * PS + HD] - mref), den);
  }
  out[((int64_t)t * n_head + kvh * G + (id - t * G)) * HD + d] = OutScale(R, M, den)(num);
}

// ---- many rows: tiles of rows over all positions they see -------------------------
// One workgroup of four waves per 64 NR rows (16 NR per wave) of a kv head.
// The chunks of two blocks are converted to fp16 in operand order in LDS once
// for all waves (each lane's 16 bytes at its place: no conflicts), the next
// chunk's codes in flight meanwhile.
template <int HD, int NR>
__global__ void __launch_bounds__(64 * kWaves)
    k_kv8_tiles(const float *__restrict__ q, aq_kv8 c, const aq_decode_state *st, int64_t pos0,
                int64_t T, int G, float scale, int tiles, float *__restrict__ out) {
  constexpr int KJ = HD / 64, VJ = HD / 32, KS = HD / 32, NU = HD / 64;
  __shared__ __attribute__((aligned(16))) h8 kl[4 * KS][64];   // [position tile, k step][lane]
  __shared__ __attribute__((aligned(16))) h8 vl[4 * VJ][64];   // [block, dimension tile][lane]
  const Span sp = span_of(st, pos0, T, c.n_ctx);
  // the tiles that see most first; a kv head's tiles side by side in the grid
  // are n_kv apart (workgroup id modulo 8 is the XCD: one L2 per kv head)
  const int n_kv = c.n_kv, kvh = blockIdx.x % n_kv, n_head = n_kv * G;
  const int tile = tiles - 1 - (int)(blockIdx.x / n_kv);
  const int rows = (int)sp.n * G, id0 = tile * (16 * NR * kWaves);
  if (id0 >= rows) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, cg = lane >> 4;
  const int wid0 = id0 + wave * (16 * NR);  // the wave's first row
  int id_last = id0 + 16 * NR * kWaves - 1;
  id_last = id_last < rows ? id_last : rows - 1;
  const int64_t p_last = sp.p0 + id_last / G;  // the last position any row sees
  const int nb = (int)(p_last / kBlk) + 1, nc = (nb + 1) / 2;
  const int64_t lim0 = sp.p0 + wid0 / G;       // the wave's first row's last position
  QRow<HD> qr[NR];
  RowState<HD> s[NR];
  int64_t lim[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int id = wid0 + 16 * n + r16;
    const bool live = id < rows;
    const int tok = live ? id / G : 0;
    const int g = live ? id - tok * G : 0;
    lim[n] = sp.p0 + tok;
    qr[n].load(q + ((int64_t)tok * n_head + kvh * G + g) * HD, live, cg, scale);
    s[n].clear();
  }
  const int64_t n_blocks = (c.n_ctx + kBlk - 1) / kBlk;
  const int8_t *kb = c.k + kvh * n_blocks * (kBlk * HD), *vb = c.v + kvh * n_blocks * (kBlk * HD);
  const float *ksc = c.k_scale + kvh * n_blocks, *vsc = c.v_scale + kvh * n_blocks;
  u4v rk[NU], rv[NU];
  float ks[2], vs[2], nks[2], nvs[2];
  auto fetch = [&](int ch) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      int b = 2 * ch + u;
      b = b < nb ? b : nb - 1;  // (an odd last block's partner: masked)
      nks[u] = ksc[b];
      nvs[u] = vsc[b];
    }
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int x = wave + kWaves * i;
      {
        const int pt = x / KJ, jj = x % KJ;
        int b = 2 * ch + (pt >> 1);
        b = b < nb ? b : nb - 1;
        rk[i] = *reinterpret_cast<const u4v *>(kb + (int64_t)b * (kBlk * HD) +
                                               (16 * (pt & 1) + r16) * HD + 64 * jj + 16 * cg);
      }
      {
        const int u = x / VJ, jv = x % VJ;
        int b = 2 * ch + u;
        b = b < nb ? b : nb - 1;
        rv[i] = *reinterpret_cast<const u4v *>(vb + (int64_t)b * (kBlk * HD) +
                                               ((16 * jv + r16) * 4 + cg) * 16);
      }
    }
  };
  fetch(0);
  for (int ch = 0; ch < nc; ++ch) {
    __syncthreads();  // the previous chunk is consumed
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int x = wave + kWaves * i;
      codes16(rk[i], kl[2 * x][lane], kl[2 * x + 1][lane]);
      codes16(rv[i], vl[2 * x][lane], vl[2 * x + 1][lane]);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      ks[u] = nks[u];
      vs[u] = nvs[u];
    }
    __syncthreads();
    if (ch + 1 < nc) fetch(ch + 1);
    f4v sc[NR][4];
#pragma unroll
    for (int pt = 0; pt < 4; ++pt) {
#pragma unroll
      for (int n = 0; n < NR; ++n) sc[n][pt] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const h8 kf = kl[pt * KS + k][lane];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          sc[n][pt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qr[n].lo[k], sc[n][pt], 0, 0, 0);
          sc[n][pt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qr[n].hi[k], sc[n][pt], 0, 0, 0);
        }
      }
    }
    h8 ph[NR][2], pl[NR][2];
    const int64_t first = (int64_t)ch * (2 * kBlk);
    if (first + 2 * kBlk - 1 > lim0) {  // (uniform)
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        int last[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int64_t d = lim[n] - first - 32 * u - 4 * cg;
          last[u] = (int)(d > 64 ? 64 : d < -1 ? -1 : d);
        }
        softmax_step<HD, 2, true>(s[n], sc[n], qr[n].f, ks, vs, last, ph[n], pl[n]);
      }
    } else {
      const int last[2] = {0, 0};
#pragma unroll
      for (int n = 0; n < NR; ++n)
        softmax_step<HD, 2, false>(s[n], sc[n], qr[n].f, ks, vs, last, ph[n], pl[n]);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int ht = 0; ht < 2 * VJ; ++ht) {
        const h8 vf = vl[2 * u * VJ + ht][lane];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          s[n].o[ht] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[n][u], s[n].o[ht], 0, 0, 0);
          s[n].o[ht] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[n][u], s[n].o[ht], 0, 0, 0);
        }
      }
  }
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int id = wid0 + 16 * n + r16;
    const float den = row_sum(s[n].l);
    if (id >= rows) continue;
    const int tok = id / G;
    const OutScale fin(s[n].R, s[n].m, den);
    float *dst = out + ((int64_t)tok * n_head + kvh * G + (id - tok * G)) * HD + 8 * cg;
#pragma unroll
    for (int i = 0; i < VJ; ++i) {
      const f4v a = fin(s[n].o[2 * i]), b = fin(s[n].o[2 * i + 1]);
      f4v *o4 = reinterpret_cast<f4v *>(dst + 32 * i);
      o4[0] = f4v{a[0], b[0], a[1], b[1]};
      o4[1] = f4v{a[2], b[2], a[3], b[3]};
    }
  }
}

}  // namespace

bool kv8_supported(int head_dim) { return head_dim == 64 || head_dim == 128 || head_dim == 256; }

// partials of at most this many (query row, split)s
constexpr int64_t kScratchRows = 16384;
size_t kv8_scratch_bytes(int head_dim) {
  return (size_t)2 * kScratchRows * (head_dim + 4) * sizeof(float);
}

#define AQ_HD(hd, CALL)                                   \
  switch (hd) {                                           \
    case 64: { constexpr int HD = 64; CALL; } break;      \
    case 128: { constexpr int HD = 128; CALL; } break;    \
    case 256: { constexpr int HD = 256; CALL; } break;    \
    default: return hipErrorInvalidValue;                 \
  }

hipError_t launch_rope_kv8(const float *q, const float *k, const float *v, float *q_out, int64_t T,
                           int n_head, int n_rot, int neox, const float *cos_t,
                           const float *sin_t, const aq_decode_state *st, int64_t pos0,
                           const aq_kv8 &c, hipStream_t s) {
  const int64_t blocks = (T + kBlk - 2) / kBlk + 1;  // blocks T positions can touch
  const int64_t n_store = blocks * c.n_kv * 2;
  int64_t n_q = q ? (T * n_head * (c.head_dim / 2) + kWG - 1) / kWG : 0;
  if (n_q > 8192) n_q = 8192;
  AQ_HD(c.head_dim, hipLaunchKernelGGL(k_kv8_store<HD>, dim3((unsigned)(n_store + n_q)), dim3(kWG),
                                       0, s, q, k, v, q_out, T, n_head, n_rot, neox, cos_t, sin_t,
                                       st, pos0, c, n_store))
  return hipGetLastError();
}

hipError_t launch_kv8_read(const aq_kv8 &c, int64_t start, int64_t n, float *k, float *v,
                           hipStream_t s) {
  const int64_t total = (int64_t)c.n_kv * n * c.head_dim;
  const int64_t wg = (total + kWG - 1) / kWG < 8192 ? (total + kWG - 1) / kWG : 8192;
  AQ_HD(c.head_dim, hipLaunchKernelGGL(k_kv8_read<HD>, dim3((unsigned)wg), dim3(kWG), 0, s, c,
                                       start, n, k, v))
  return hipGetLastError();
}

// The splits of the positions for T tokens: about two workgroups per CU, no
// more than the cache's blocks give every wave one of, nor than the scratch
// holds.  By the cache's length, not by the position, which the host may not
// know: a call gives the same bits however it is told where it is.
int kv8_splits(const aq_kv8 &c, int64_t T, int n_head) {
  const int64_t G = n_head / c.n_kv, tiles = (T * G + 15) / 16;
  const int64_t blocks = (c.n_ctx + kBlk - 1) / kBlk;
  int64_t S = (blocks + kWaves - 1) / kWaves;
  const int64_t fill = (512 + c.n_kv * tiles - 1) / (c.n_kv * tiles);
  const int64_t room = kScratchRows / (T * n_head);
  S = S < fill ? S : fill;
  S = S < room ? S : room;
  return (int)(S < 1 ? 1 : S);
}

hipError_t launch_attention_kv8(const float *q, const aq_kv8 &c, int64_t T, int n_head,
                                const aq_decode_state *st, int64_t pos0, float *out,
                                hipStream_t s) {
  const float scale = (float)(1.0 / sqrt((double)c.head_dim));
  const int G = n_head / c.n_kv;
  const int64_t rows = T * G;
  if (rows <= 64) {
    const int S = kv8_splits(c, T, n_head);
    AQ_HD(c.head_dim,
          hipLaunchKernelGGL(k_kv8_split<HD>, dim3((unsigned)S, (unsigned)c.n_kv,
                                                   (unsigned)((rows + 15) / 16)),
                             dim3(64 * kWaves), 0, s, q, c, st, pos0, T, G, scale, c.scratch, out);
          if (S > 1) hipLaunchKernelGGL(k_kv8_combine<HD>, dim3((unsigned)rows, (unsigned)c.n_kv),
                                        dim3(HD), 0, s, c.scratch, st, pos0, c.n_ctx, T, G, S, out))
    return hipGetLastError();
  }
  const int64_t tiles = (rows + 63) / 64;
  AQ_HD(c.head_dim, hipLaunchKernelGGL((k_kv8_tiles<HD, 1>), dim3((unsigned)(tiles * c.n_kv)),
                                       dim3(64 * kWaves), 0, s, q, c, st, pos0, T, G, scale,
                                       (int)tiles, out))
  return hipGetLastError();
}

hipError_t launch_attention_rope_kv8(const float *q, const float *k, const float *v, int n_head,
                                     int n_rot, int neox, const float *cos_t, const float *sin_t,
                                     const aq_decode_state *st, int64_t pos0, const aq_kv8 &c,
                                     float *out, hipStream_t s) {
  if (n_head > kScratchRows) return hipErrorInvalidValue;
  float *qr = c.scratch + kScratchRows * (c.head_dim + 4);
  hipError_t e = launch_rope_kv8(q, k, v, qr, 1, n_head, n_rot, neox, cos_t, sin_t, st,
                                 pos0, c, s);
  return e != hipSuccess ? e : launch_attention_kv8(qr, c, 1, n_head, st, pos0, out, s);
}

}  // namespace aq
