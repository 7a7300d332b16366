// aq_kv8.hip - the 8-bit KV cache: rotation and store, attention, read-back.
//
// Values are coded in blocks of kKv8Block = 32 positions of one kv head, K and
// V apart: s = fl32(amax / 127) over the tokens the block holds so far, and a
// value x is the whole number c nearest to x / s (ties to even), standing for
// s c.  The last block stored is kept in fp32 too (the tail), so a block that a
// token joins is coded anew from its own values: the codes are a function of
// the tokens alone, not of the calls that brought them, and no error adds up.
// A call that goes back inside an earlier block, whose fp32 values are gone,
// takes them from the codes (the tail's tag names the block it holds).
//
// Layouts (n_blocks = ceil(n_ctx / 32) per kv head):
//   K codes [n_kv][n_blocks][32 positions][head_dim]
//   V codes [n_kv][n_blocks][head_dim / 2][4 g][2 dimensions][8 positions],
//     the eight positions 16 pt + 4 g + r (pt = 0, 1; r = 0 .. 3) of a dimension
//     side by side: what a lane of the matrix instructions takes as its operand
//     (the scores' lanes hold the weights of these positions), two dimensions
//     per 16-byte load
//   scales [n_kv][n_blocks] fp32; tails [n_kv][32][head_dim] fp32, and behind
//   them the block that each kv head's tail holds, [n_kv] int32
#include <math.h>

#include <type_traits>

#include "aq_internal.h"

namespace aq {
namespace {

constexpr int kBlk = kKv8Block;
constexpr int kWG = 256;

typedef float f4v __attribute__((ext_vector_type(4)));

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

// The rotation: pairs (2i, 2i + 1) or, neox, (i, i + n_rot / 2) of a head's first
// n_rot dimensions, products and differences rounded separately.
struct Rope {
  const float *cos_t, *sin_t;
  int n_rot, neox;
};
// element d of the head vector x at position pos
__device__ __forceinline__ float rotated(const float *x, int d, int64_t pos, const Rope &r) {
#pragma clang fp contract(off)
  if (d >= r.n_rot) return x[d];
  const int half = r.n_rot / 2;
  const int i = r.neox ? (d < half ? d : d - half) : d >> 1;
  const bool lo = r.neox ? d < half : !(d & 1);
  const int other = r.neox ? (lo ? d + half : d - half) : d ^ 1;
  const float c = r.cos_t[pos * half + i], s = r.sin_t[pos * half + i];
  const float a = x[d], b = x[other];
  return lo ? a * c - b * s : b * s + a * c;
}
// elements d .. d + 3 (d a multiple of 4).  neox: n_rot a multiple of 8, so that
// a group of four has its partners side by side.  Table values are loaded at
// clamped places before they are needed, without branches between the loads.
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ f4v rotated4(const float *x, int d, int64_t pos, const Rope &r) {
#pragma clang fp contract(off)
  const int half = r.n_rot / 2;
  const f4v v = *reinterpret_cast<const f4v *>(x + d);
  if (half == 0) return v;
  const float *cr = r.cos_t + pos * half, *sr = r.sin_t + pos * half;
  f4v o = v;
  if (r.neox) {
    const bool lo = d < half, in = d < r.n_rot;
    const int i = in ? (lo ? d : d - half) : 0;
    const f4v y = *reinterpret_cast<const f4v *>(x + (in ? (lo ? d + half : d - half) : d));
    const f4v c = *reinterpret_cast<const f4u *>(cr + i), s = *reinterpret_cast<const f4u *>(sr + i);
    if (in) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = lo ? v[e] * c[e] - y[e] * s[e] : y[e] * s[e] + v[e] * c[e];
    }
  } else {
    float c[2], s[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int i = d / 2 + p < half ? d / 2 + p : half - 1;
      c[p] = cr[i];
      s[p] = sr[i];
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      if (d / 2 + p >= half) continue;
      o[2 * p] = v[2 * p] * c[p] - v[2 * p + 1] * s[p];
      o[2 * p + 1] = v[2 * p] * s[p] + v[2 * p + 1] * c[p];
    }
  }
  return o;
}
// a where mask is all ones, b where it is 0 (bits; a conditional here becomes
// branches, which part the loads and the waits)
__device__ __forceinline__ float pick(uint32_t mask, float a, float b) {
  return __uint_as_float((__float_as_uint(a) & mask) | (__float_as_uint(b) & ~mask));
}
__device__ __forceinline__ uint32_t ones_if(bool c) { return c ? 0xFFFFFFFFu : 0u; }
// elements d0 .. d0 + 15 (d0 a multiple of 16) of x: every load goes out before
// the first use
__device__ __forceinline__ void rotated16(const float *x, int d0, int64_t pos, const Rope &r,
                                          float (&o)[16]) {
#pragma clang fp contract(off)
  const int half = r.n_rot / 2;
  f4v v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const f4v *>(x + d0 + 4 * i);
  if (half == 0) {
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = v[e >> 2][e & 3];
    return;
  }
  const float *cr = r.cos_t + pos * half, *sr = r.sin_t + pos * half;
  if (r.neox) {
    f4v y[4], c[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = d0 + 4 * i;
      const bool lo = d < half, in = d < r.n_rot;
      const int t = in ? (lo ? d : d - half) : 0;
      y[i] = *reinterpret_cast<const f4v *>(x + (in ? (lo ? d + half : d - half) : d));
      c[i] = *reinterpret_cast<const f4u *>(cr + t);
      s[i] = *reinterpret_cast<const f4u *>(sr + t);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = d0 + 4 * i;
      const uint32_t in = ones_if(d < r.n_rot), minus = d < half ? 0x80000000u : 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = v[i][e] * c[i][e], b = y[i][e] * s[i][e];
        o[4 * i + e] = pick(in, a + __uint_as_float(__float_as_uint(b) ^ minus), v[i][e]);
      }
    }
    return;
  }
  float c[8], s[8];
  if (r.n_rot % 16 == 0) {  // the pairs are all rotated or none
    const int t = d0 / 2 < half ? d0 / 2 : 0;
    const f4u c0 = *reinterpret_cast<const f4u *>(cr + t),
              c1 = *reinterpret_cast<const f4u *>(cr + t + 4),
              s0 = *reinterpret_cast<const f4u *>(sr + t),
              s1 = *reinterpret_cast<const f4u *>(sr + t + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c[e] = c0[e], c[4 + e] = c1[e];
      s[e] = s0[e], s[4 + e] = s1[e];
    }
  } else {
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const int t = d0 / 2 + p < half ? d0 / 2 + p : half - 1;
      c[p] = cr[t];
      s[p] = sr[t];
    }
  }
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const float a = v[p >> 1][2 * (p & 1)], b = v[p >> 1][2 * (p & 1) + 1];
    const uint32_t in = ones_if(d0 / 2 + p < half);
    const float ra = a * c[p] - b * s[p], rb = a * s[p] + b * c[p];
    o[2 * p] = pick(in, ra, a);
    o[2 * p + 1] = pick(in, rb, b);
  }
}
// whether rotated4 takes this rotation
__device__ __forceinline__ bool rope_by4(const Rope &r) { return !r.neox || r.n_rot % 8 == 0; }

// A block's coding: c = round-half-even(x / s) over the reals.  y = x (1 / s) is
// off by less than 127 2^-23, so its nearest whole number r is the code unless it
// lies that near a half (one value in thirty thousand); then the remainder
// x - r s, which is exact (a multiple of the smaller of their units, below 2^24 of
// it), tells.  Scales below 2^-100 are lifted by 2^100, exactly, with the
// values; among the subnormals a scale can be too small, and codes end at 127.
struct Coder {
  float s, inv, lift;
  __device__ __forceinline__ explicit Coder(float scale) {
    lift = scale < 0x1p-100f ? 0x1p100f : 1.f;
    s = scale * lift;
    inv = s > 0.f ? 1.f / s : 0.f;
  }
  // 16 values as bytes: 1.5 2^23 added to y leaves its nearest whole number in
  // the sum's low bits
  __device__ __forceinline__ uint4 operator()(const float (&x)[16]) const {
    uint32_t t[16], w[4];
    if (!(s > 0.f)) return make_uint4(0, 0, 0, 0);  // (0 or NaN)
    float far = lift - 1.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float m = fmaf(x[e], inv, kMagic), r = m - kMagic;
      far = fmaxf(far, fabsf(fmaf(x[e], inv, -r)));
      t[e] = __float_as_uint(m);
    }
    if (far > 0.49998f) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float v = x[e] * lift, r = rintf(v * inv), rem = fmaf(-r, s, v);
        int c = (int)r;
        const float two = 2.f * fabsf(rem);
        const bool fix = (two > s) | ((two == s) & ((c & 1) != 0));
        c += fix ? (rem < 0.f ? -1 : 1) : 0;
        t[e] = (uint32_t)min(max(c, -127), 127);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = __builtin_amdgcn_perm(t[4 * i + 1], t[4 * i], 0x0C0C0400u);
      const uint32_t b = __builtin_amdgcn_perm(t[4 * i + 3], t[4 * i + 2], 0x0C0C0400u);
      w[i] = a | b << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static constexpr float kMagic = 12582912.f;
};
__device__ __forceinline__ float scale_of(uint32_t amax_bits) {
  return amax_bits >= 0x7F800000u ? __uint_as_float(0x7FC00000u)
                                  : __uint_as_float(amax_bits) / 127.f;
}

// The tokens of one block of one kv head's K or V, in the units of 16 codes that
// are 16 bytes of the layout: of K 16 dimensions of a position, of V two
// dimensions of the eight positions 16 pt + 4 g + r.
template <int HD>
struct BlockTokens {
  static constexpr int UNITS = kBlk * HD / 16;
  bool is_v, by4;
  float *tail;         // rows before the call's tokens, if *tag is their block
  int32_t *tag;
  const uint4 *codes;  // the block's
  const float *scale;
  const float *first;  // where the call's token of row 0 would be
  int64_t stride;      // from a token to the next
  int before, end;     // rows 0 .. before - 1 from the tail, before .. end - 1 the call's
  int64_t pos;         // the position of row 0
  Rope rope;
  // block b of a call's tokens sp at x (the head's vector of the first of them)
  __device__ __forceinline__ BlockTokens(const aq_kv8 &c, int kvh, bool is_v, bool by4,
                                         const float *x, const Span &sp, int64_t b,
                                         const Rope &rope)
      : is_v(is_v), by4(by4), stride((int64_t)c.n_kv * HD), rope(rope) {
    const int64_t n_blocks = (c.n_ctx + kBlk - 1) / kBlk;
    float *tails = is_v ? c.v_tail : c.k_tail;
    tail = tails + (int64_t)kvh * kBlk * HD;
    tag = reinterpret_cast<int32_t *>(tails + (int64_t)c.n_kv * kBlk * HD) + kvh;
    codes = reinterpret_cast<const uint4 *>((is_v ? c.v : c.k) +
                                            (kvh * n_blocks + b) * (kBlk * HD));
    scale = (is_v ? c.v_scale : c.k_scale) + kvh * n_blocks + b;
    x += kvh * HD;
    pos = b * kBlk;
    const int64_t lead = sp.p0 - pos, e = lead + sp.n;
    first = x - lead * stride;
    before = lead > 0 ? (int)lead : 0;
    end = e < kBlk ? (int)e : kBlk;
  }
  // the vector of a row (past the last token: of the last, not used)
  __device__ __forceinline__ const float *row_of(int row) const {
    const float *t = tail + row * HD, *f = first + (int64_t)min(max(row, before), end - 1) * stride;
    return row < before ? t : f;
  }
  // the unit's values (0 past the last token); the loads do not wait for any
  __device__ __forceinline__ void load(int u, float (&x)[16]) const {
    if (!is_v) {
      const int row = u / (HD / 16), d0 = 16 * (u % (HD / 16));
      const float *t = row_of(row);
      if (by4) {
        float y[16];
        rotated16(t, d0, pos + min(max(row, before), end - 1), rope, y);
        const uint32_t old = ones_if(row < before), live = ones_if(row < end);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f4v v = *reinterpret_cast<const f4v *>(t + d0 + 4 * i);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[4 * i + e] = pick(old, v[e], pick(live, y[4 * i + e], 0.f));
        }
      } else {
#pragma unroll 1
        for (int e = 0; e < 16; ++e)
          x[e] = row < before ? t[d0 + e] : row < end ? rotated(t, d0 + e, pos + row, rope) : 0.f;
      }
      return;
    }
    const int d0 = 2 * (u >> 2);
    float2 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      v[k] = *reinterpret_cast<const float2 *>(row_of(v_row(u, k)) + d0);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t live = ones_if(v_row(u, k) < end);
      x[k] = pick(live, v[k].x, 0.f);
      x[8 + k] = pick(live, v[k].y, 0.f);
    }
  }
  // whether the rows before the call's are not in the tail.  A scalar load and a
  // branch, before the workgroup, the only one to write the tag, does; the empty
  // statement holds the value, which is not to be loaded again after that.
  __device__ __forceinline__ bool gone() const {
    int32_t t = *(const __attribute__((address_space(4))) int32_t *)tag;
    asm volatile("" : "+s"(t));
    return before > 0 && t != (int32_t)(pos / kBlk);
  }
  // those rows from the codes (a unit is the 16 bytes that its thread writes later)
  __device__ __forceinline__ void reopen(int u, float (&x)[16]) const {
    const uint4 w = codes[u];
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
    const float s = *scale;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int row = is_v ? v_row(u, e & 7) : u / (HD / 16);
      if (row < before) x[e] = s * (float)(int8_t)(ws[e >> 2] >> (8 * (e & 3)));
    }
  }
  __device__ __forceinline__ static int v_row(int u, int k) {
    return 16 * (k >> 2) + 4 * (u & 3) + (k & 3);
  }
  // rows from .. end - 1 of the block into the tail
  __device__ __forceinline__ void keep(int u, int from, const float (&x)[16]) const {
    if (!is_v) {
      const int row = u / (HD / 16), d0 = 16 * (u % (HD / 16));
      if (row < from || row >= end) return;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f4v *>(tail + row * HD + d0 + 4 * i) =
            f4v{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
      return;
    }
    const int d0 = 2 * (u >> 2);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int row = v_row(u, k);
      if (row >= from && row < end)
        *reinterpret_cast<float2 *>(tail + row * HD + d0) = make_float2(x[k], x[8 + k]);
    }
  }
};
__device__ __forceinline__ uint32_t amax16(const float (&x)[16], uint32_t am) {
#pragma unroll
  for (int e = 0; e < 16; ++e) am = max(am, __float_as_uint(x[e]) & 0x7FFFFFFFu);
  return am;  // (as bits: a NaN's lie above infinity's)
}
template <int CTRL>
__device__ __forceinline__ uint32_t dppu(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  v = max(v, dppu<0xB1>(v));   // quad_perm [1,0,3,2]
  v = max(v, dppu<0x4E>(v));   // quad_perm [2,3,0,1]
  v = max(v, dppu<0x141>(v));  // row_half_mirror
  v = max(v, dppu<0x140>(v));  // row_mirror
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(b[0], b[1]);
}

// ---- rotation and store ------------------------------------------------------
// Workgroups 0 .. n_store - 1 code one block of one kv head each, K or V: every
// thread holds one or two units' values (those before the call's from the tail,
// the call's own rotated), their largest magnitude gives the scale.  Slots past
// the last token are cleared.  The workgroup of the call's first block also keeps
// the tail: it alone reads it (before), and writes the tokens of the last block
// (after), so no two workgroups meet there.  The rest rotate q, a token each.
//
// One pass over memory, one barrier a block: 2048 tokens, 32 / 8 heads of 128
// 20.3 us (50 MB in, 38 out: 4.3 TB/s; a large copy 5.15), one token of 32 / 8
// heads of 64 5.0 us (its chain: position, tail, tables, maximum).
template <int HD>
constexpr int kStoreWG = HD == 64 ? 128 : 256;
template <int HD>
__global__ void __launch_bounds__(kStoreWG<HD>, HD == 256 ? 2 : 4)
    k_kv8_store(const float *q, const float *__restrict__ k, const float *__restrict__ v,
                float *q_out, int64_t T, int n_head, Rope rope, const aq_decode_state *st,
                int64_t pos0, aq_kv8 c, int64_t n_store) {
  constexpr int NT = kStoreWG<HD>, UPT = BlockTokens<HD>::UNITS / NT;
  __shared__ uint32_t red[NT / 64];
  const Span sp = span_of(st, pos0, T, c.n_ctx);
  if (sp.n == 0) return;
  const int tid = threadIdx.x;
  if ((int64_t)blockIdx.x >= n_store) {
    const bool by4 = rope_by4(rope);
    const int half = rope.n_rot / 2;
    for (int64_t t = (int64_t)blockIdx.x - n_store; t < sp.n; t += gridDim.x - n_store) {
      const int64_t p = sp.p0 + t;
      if (by4) {  // a thread's share: four dimensions; neox: and their partners
        for (int i = tid; i < n_head * (HD / 4); i += NT) {
          const int h = i / (HD / 4), d = 4 * (i % (HD / 4));
          const float *x = q + (t * n_head + h) * HD;
          float *y = q_out + (t * n_head + h) * HD;
          if (rope.neox && d >= half && d < rope.n_rot) continue;  // its partner's thread's
          const f4v a = rotated4(x, d, p, rope);
          if (rope.neox && d < half) {
            const f4v b = rotated4(x, d + half, p, rope);
            *reinterpret_cast<f4v *>(y + d + half) = b;
          }
          *reinterpret_cast<f4v *>(y + d) = a;
        }
      } else {  // pairs (j, j + half), then the dimensions past n_rot
        for (int i = tid; i < n_head * (HD / 2); i += NT) {
          const int h = i / (HD / 2), j = i % (HD / 2);
          const float *x = q + (t * n_head + h) * HD;
          float *y = q_out + (t * n_head + h) * HD;
          const int a = j < half ? j : rope.n_rot + 2 * (j - half);
          const int b = j < half ? j + half : a + 1;
          const float ra = rotated(x, a, p, rope), rb = rotated(x, b, p, rope);
          y[a] = ra;
          y[b] = rb;
        }
      }
    }
    return;
  }
  const bool is_v = blockIdx.x & 1;
  const int kvh = (int)((blockIdx.x >> 1) % c.n_kv);
  const int64_t b0 = sp.p0 / kBlk, bl = (sp.p0 + sp.n - 1) / kBlk;
  const int64_t b = b0 + (int64_t)(blockIdx.x >> 1) / c.n_kv;
  if (b > bl) return;
  auto tokens = [&](int64_t bi) {
    return BlockTokens<HD>(c, kvh, is_v, rope_by4(rope), is_v ? v : k, sp, bi, rope);
  };
  BlockTokens<HD> blk = tokens(b);
  float x[UPT][16];
#pragma unroll
  for (int i = 0; i < UPT; ++i) blk.load(tid + NT * i, x[i]);
  const bool gone = blk.gone();
  uint32_t am = 0;
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    if (gone) blk.reopen(tid + NT * i, x[i]);
    am = amax16(x[i], am);
  }
  am = wave_umax(am);
  if ((tid & 63) == 0) red[tid >> 6] = am;
  __syncthreads();  // (and the tail, its tag and the block's scale have been read)
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) am = max(am, red[w]);
  const float s = scale_of(am);
  const Coder code(s);
  const int64_t n_blocks = (c.n_ctx + kBlk - 1) / kBlk;
  if (tid == 0) (is_v ? c.v_scale : c.k_scale)[kvh * n_blocks + b] = s;
  uint4 *dst = reinterpret_cast<uint4 *>((is_v ? c.v : c.k) + (kvh * n_blocks + b) * (kBlk * HD));
#pragma unroll
  for (int i = 0; i < UPT; ++i) dst[tid + NT * i] = code(x[i]);
  if (b != b0) return;
  if (tid == 0) *blk.tag = (int32_t)bl;
  int from = gone ? 0 : blk.before;
  if (bl != b0) {
    blk = tokens(bl);
    from = 0;
#pragma unroll
    for (int i = 0; i < UPT; ++i) blk.load(tid + NT * i, x[i]);
  }
#pragma unroll
  for (int i = 0; i < UPT; ++i) blk.keep(tid + NT * i, from, x[i]);
}

// ---- read-back ---------------------------------------------------------------
// out[kvh][p - start][d] = s c, one product rounded to fp32.  One workgroup per
// block of K and of V; a thread turns units of 16 codes into four 16-byte stores
// (K), or eight 8-byte ones to eight rows (V; 16 lanes fill 128 bytes of a row).
// Bound by its stores: 2048 positions of 8 heads of 128, 21 MB in 7.5 us; one
// position 2.4.
template <int HD>
__global__ void __launch_bounds__(kStoreWG<HD>)
    k_kv8_read(aq_kv8 c, int64_t start, int64_t n, float *__restrict__ ko,
               float *__restrict__ vo) {
  constexpr int NT = kStoreWG<HD>, UPT = BlockTokens<HD>::UNITS / NT;
  const bool is_v = blockIdx.x & 1;
  const int64_t b = start / kBlk + (blockIdx.x >> 1), n_blocks = (c.n_ctx + kBlk - 1) / kBlk;
  const int kvh = blockIdx.y;
  const uint4 *src =
      reinterpret_cast<const uint4 *>((is_v ? c.v : c.k) + (kvh * n_blocks + b) * (kBlk * HD));
  const float s = (is_v ? c.v_scale : c.k_scale)[kvh * n_blocks + b];
  // row r of the block is output row first + r, where lo <= r < hi
  const int64_t first = b * kBlk - start, left = n - first;
  const int lo = first < 0 ? (int)-first : 0, hi = left < kBlk ? (int)left : kBlk;
  float *out = (is_v ? vo : ko) + (kvh * n + first) * HD;
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    const int u = threadIdx.x + NT * i;
    const uint4 w = src[u];
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
    float x[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = s * (float)(int8_t)(ws[e >> 2] >> (8 * (e & 3)));
    if (!is_v) {
      const int row = u / (HD / 16), d0 = 16 * (u % (HD / 16));
      if (row < lo || row >= hi) continue;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *reinterpret_cast<f4u *>(out + row * HD + d0 + 4 * k) =
            f4u{x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]};
      continue;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int row = BlockTokens<HD>::v_row(u, k);
      if (row < lo || row >= hi) continue;
      typedef float f2u __attribute__((ext_vector_type(2), aligned(4)));
      *reinterpret_cast<f2u *>(out + row * HD + 2 * (u >> 2)) = f2u{x[k], x[8 + k]};
    }
  }
}

// ---- attention -----------------------------------------------------------------
// Both kernels below work on tiles of 16 query rows of one kv head (row id =
// token * G + head in the group, any G up to 16) with
// v_mfma_f32_16x16x32_f16, the codes as exact fp16 operands and every fp32
// operand in two fp16 pieces (x = hi + lo, 23 bits where lo is normal):
//   S^T (positions x rows) = C_K Q^T, Q's row scaled by a power of two to a
//     largest value in [2^14, 2^15): lane l holds row l % 16's scores at
//     positions 16 pt + 4 (l / 16) + r of a block (pt = 0, 1; r = 0 .. 3);
//   O^T (dimensions x rows) += C_V^T P^T: those 8 weights are the lane's B
//     operand as it holds them (the V layout stores positions in that order).
// The block's K scale enters as the factor of its raw scores, its V scale in
// the weights: P = 2^(z - m) s_V, formed relative to the largest such product
// the row has met, 2^D (of the same 2^m), so the pieces hold 23 bits of whatever
// counts and no magnitude of V over- or underflows them.  m and D are rounded up
// to whole numbers, so every rescaling is an exact power of two; D stays a small
// number however large the scores are.  The sum of 2^(z - m) is kept per lane.
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef unsigned int u4v __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kTop = 14.f;      // weights reach 2^14 in the pieces
constexpr float kLow = -1e30f;    // D before any weight
constexpr float kFine = 0x1p20f;  // exponents up to here are off by less than 2^-4

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
__device__ __forceinline__ float wave_max(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __uint_as_float(dppu<decltype(ctrl)::value>(__float_as_uint(x)));
  };
  v = fmaxf(v, dpp(v, std::integral_constant<int, 0xB1>()));   // quad_perm [1,0,3,2]
  v = fmaxf(v, dpp(v, std::integral_constant<int, 0x4E>()));   // quad_perm [2,3,0,1]
  v = fmaxf(v, dpp(v, std::integral_constant<int, 0x141>()));  // row_half_mirror
  v = fmaxf(v, dpp(v, std::integral_constant<int, 0x140>()));  // row_mirror
  return row_max(v);
}
// a float that no store of this kernel reaches, at a wave's common place: a
// scalar load
__device__ __forceinline__ float load_const(const float *p) {
  return *(const __attribute__((address_space(4))) float *)p;
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
  // (a factor that the compiler does not know keeps this one mixed-precision
  // fused multiply-add a value, exact, instead of a conversion and a difference)
  float minus = -1.f;
  asm("" : "+v"(minus));
  const h2 l = __builtin_convertvector(
      f2v{fmaf((float)h[0], minus, a), fmaf((float)h[1], minus, b)}, h2);
  hi = __builtin_bit_cast(uint32_t, h);
  lo = __builtin_bit_cast(uint32_t, l);
}

// A lane's part of one query row: 8 dimensions 64 jj + 16 cg + 8 half .. per k
// step ks = 2 jj + half, in pieces of the row times 2^-back.  back stays apart: as
// part of a factor it would fall among the subnormals for small rows, whose keys
// may be large.  The pieces of a row with an infinity or a NaN are NaN, and with
// them its raw scores.
template <int HD>
struct QRow {
  h8 hi[HD / 32], lo[HD / 32];
  int back;
  // ROPE: q is rotated for position pos on the way
  template <bool ROPE>
  __device__ __forceinline__ void load(const float *__restrict__ q, bool live, int cg, int64_t pos,
                                       const Rope &rope) {
    float v[HD / 64][16];
    const uint32_t exists = ones_if(live);
    uint32_t am = 0;  // the largest magnitude, as bits (infinity's and NaNs' above all)
#pragma unroll
    for (int jj = 0; jj < HD / 64; ++jj) {
      const int d0 = 64 * jj + 16 * cg;
      if constexpr (ROPE) {
        rotated16(q, d0, pos, rope, v[jj]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f4v x = *reinterpret_cast<const f4v *>(q + d0 + 4 * i);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[jj][4 * i + e] = x[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        v[jj][e] = pick(exists, v[jj][e], 0.f);  // (rows that do not exist read row 0)
        am = max(am, __float_as_uint(v[jj][e]) & 0x7FFFFFFFu);
      }
    }
    const auto r = __builtin_amdgcn_permlane16_swap(am, am, false, false);
    am = max(r[0], r[1]);
    const auto t = __builtin_amdgcn_permlane32_swap(am, am, false, false);
    am = max(t[0], t[1]);
    const bool bad = am >= 0x7F800000u;
    const int up = am > 0 && !bad ? 15 - __builtin_amdgcn_frexp_expf(__uint_as_float(am)) : 0;
    back = -up;
    const float nan = __uint_as_float(0x7FC00000u);
    const uint32_t good = ones_if(!bad);
#pragma unroll
    for (int ks = 0; ks < HD / 32; ++ks) {
      u4v h, l;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = pick(good, ldexpf(v[ks >> 1][8 * (ks & 1) + 2 * i], up), nan);
        const float b = pick(good, ldexpf(v[ks >> 1][8 * (ks & 1) + 2 * i + 1], up), nan);
        uint32_t hh, ll;
        pieces2(a, b, hh, ll);
        h[i] = hh, l[i] = ll;
      }
      hi[ks] = __builtin_bit_cast(h8, h);
      lo[ks] = __builtin_bit_cast(h8, l);
    }
  }
};

// The running softmax of a lane's row: maximum m and, counted from it, the
// reference D (both whole exponents of two, the same in the row's four lanes), the
// lane's part of the sum l, and the numerators, o[2 j + e][rr] at dimension
// 32 j + 8 cg + 2 rr + e, which stand for o 2^(D - kTop).
template <int HD>
struct RowState {
  float m, D, l;
  f4v o[HD / 16];
  __device__ __forceinline__ void clear() {
    m = -INFINITY, D = kLow, l = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) o[i] = f4v{0.f, 0.f, 0.f, 0.f};
  }
};
// differences are taken from m, 0 where the row has seen nothing
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.f : m; }
// a reference D counted from m, counted from ref >= m
__device__ __forceinline__ float moved(float D, float m, float ref) {
  return fmaxf(D + (m - ref), kLow);
}

// NB blocks' raw scores sc (two tiles of positions each) to weights in pieces,
// with their K and V scales: m, D, l and o of the row move on.  f, and 2^back of
// the row: what turns raw scores into exponents of two (but for the K scale).
// MASK: only positions up to last[b], counted from the lane's first one in block
// b, exist.
//
// An exponent is one fma, whose product is not rounded while the maximum's is:
// past kFine that would show (weights above what fp16 holds, or the largest one
// lost), so there the scores are rounded products first, for the whole wave.
template <int HD, int NB, bool MASK>
__device__ __forceinline__ void softmax_step(RowState<HD> &st, f4v (&sc)[2 * NB], float f, int back,
                                             const float (&ks)[NB], const float (&vs)[NB],
                                             const int (&last)[NB], h8 (&ph)[NB], h8 (&pl)[NB]) {
  float c[NB], t[NB], ve[NB], mn = st.m, reach = 0.f;
  auto largest = [&](int b) {  // of the row's scores in a block, -infinity for none
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = sc[2 * b + (i >> 2)][i & 3];
      mx = !MASK || 16 * (i >> 2) + (i & 3) <= last[b] ? fmaxf(mx, x) : mx;
    }
    return row_max(mx);
  };
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    c[b] = ldexpf(ks[b], back) * f;
    const float mx = largest(b);
    const bool none = MASK && mx == -INFINITY;  // (not through a masked block's scale)
    t[b] = none ? mx : ceilf(mx * c[b]);
    reach += none ? 0.f : fabsf(t[b]);
  }
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(reach < kFine)) != 0, 0)) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      c[b] = c[b] > 0x1.fffffep127f ? 0x1.fffffep127f : c[b];  // (no 0 x infinity; a NaN stays)
#pragma unroll
      for (int i = 0; i < 8; ++i) sc[2 * b + (i >> 2)][i & 3] *= c[b];
      t[b] = ceilf(largest(b));
      c[b] = 1.f;
    }
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) mn = fmaxf(mn, t[b]);
  const float mref = finite_ref(mn), old = moved(st.D, st.m, mref);
  float D = old;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    ve[b] = (float)__builtin_amdgcn_frexp_expf(vs[b]);
    if (vs[b] > 0.f) D = fmaxf(D, (t[b] - mref) + ve[b]);
  }
  // (whole exponents: an integer conversion and a ldexp, a quarter of exp2's time)
  const float corr = ldexpf(1.f, (int)(st.m - mref)), corr_o = ldexpf(1.f, (int)(old - D));
  float sum = 0.f;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const float g = ldexpf(__builtin_amdgcn_frexp_mantf(vs[b]),
                           (int)fminf(ve[b] - D + kTop, 120.f));
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
  // (whole powers of two, so seldom)
  if (__builtin_amdgcn_ballot_w64(D != old)) {
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) st.o[i] *= corr_o;
  }
  st.D = D;
}

// v 2^(D - kTop) / den, the power in two whole parts so that neither leaves
// the range
struct OutScale {
  float a, b;
  __device__ __forceinline__ OutScale(float D, float den) {
    const float x = D - kTop, h = floorf(0.5f * x);
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
// the maximum and the reference of N states joined: m(i), D(i) of each
struct Ref {
  float m, D;
};
template <int N, class M, class R>
__device__ __forceinline__ Ref joined(M m, R D) {
  Ref all{m(0), kLow};
#pragma unroll
  for (int i = 1; i < N; ++i) all.m = fmaxf(all.m, m(i));
  const float ref = finite_ref(all.m);
#pragma unroll
  for (int i = 0; i < N; ++i) all.D = fmaxf(all.D, moved(D(i), m(i), ref));
  return all;
}

// ---- few rows: the positions split over workgroups -------------------------------
// Workgroup (split j, kv head, tile of 16 rows): wave w takes blocks 4 j + w, + 4 S
// ..., straight from memory into operand order (no LDS), the next block's loads
// under way while one is computed; the waves' states meet in LDS, the splits'
// in k_kv8_combine.  One split writes the output itself.
//
// Bound by the codes' bytes, for short caches by one wave's chain.  One token of
// 32 / 8 heads of 128: 30000 positions 13.7 us (61 MB: 4.5 TB/s), 131072 42
// (268 MB: 6.4); 32 / 8 heads of 64, 2176 positions 4.4; 16 / 8 heads of 256, 3800
// 7.7, 32766 24.6 (134 MB: 5.5); 5 tokens of 28 / 4 heads of 128 at 7001 12.9
// (three tiles of rows, one or two blocks a wave, 3.2 MB of states beside 7.2 of
// codes; which of these bounds it was not measured).
//
// ROPE: one token, whose q, k and v are not rotated yet.  Every workgroup
// rotates its q rows in registers; one more workgroup per kv head (the first)
// takes the token's block, which it alone reads: it codes the block anew from
// the tail and the token (k_kv8_store's codes, bit for bit), stores it and
// attends to it from LDS, while the others go through the blocks before.  There
// a wave executes its few thousand instructions alone on its SIMD, 2 ns each,
// so four waves code the block while a fifth makes q's pieces, as long as a CU
// has one workgroup (several of five waves each load its SIMDs unevenly).  Whole
// calls, five waves against four: 32 / 8 heads of 64 at 4094 positions 9.7 us
// (10.0), at 32766 14.0 (13.0); of 128 at 4094 10.9 (11.4), at 8190 15.4 (12.9), at
// 32766 23.9 (18.9).  At 256 dimensions five waves spill: four.
constexpr int kWaves = 4;
template <int HD, bool ROPE, int NW>
__global__ void __launch_bounds__(64 * NW, HD == 64 ? 3 : 1)
    k_kv8_split(const float *__restrict__ q, aq_kv8 c, const aq_decode_state *st, int64_t pos0,
                int64_t T, int G, float f, float *__restrict__ part, float *__restrict__ out,
                const float *__restrict__ kn, const float *__restrict__ vn, Rope rope) {
  constexpr int KJ = HD / 64, VJ = HD / 32, PS = HD + 4;
  constexpr int PARTS = HD == 256 ? 2 : 1, VP = VJ / PARTS;  // the merge's LDS: at most 40 KB
  __shared__ f4v os[NW][2 * VP][64];
  __shared__ float stat[NW][3][16];
  __shared__ uint4 own[ROPE ? 2 : 1][ROPE ? BlockTokens<HD>::UNITS : 1];  // the token's block
  __shared__ uint32_t red[2][kWaves];
  const Span sp = span_of(st, pos0, T, c.n_ctx);
  const int j = blockIdx.x, S = gridDim.x, kvh = blockIdx.y, n_head = gridDim.y * G;
  const int id0 = blockIdx.z * 16, rows = (int)sp.n * G;  // at most 65535 x 16
  if (id0 >= rows) return;
  const int lane = threadIdx.x & 63, r16 = lane & 15, cg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = id0 + r16, id_last = id0 + 15 < rows ? id0 + 15 : rows - 1;
  const bool live = id < rows;
  const int tok = live ? id / G : 0;
  const int g = live ? id - tok * G : 0;
  const int lim = (int)sp.p0 + tok;             // the row's last position
  const int lim0 = (int)sp.p0 + id0 / G;        // the tile's first row's
  const int nb_all = (int)((sp.p0 + id_last / G) / kBlk) + 1;  // blocks the tile sees
  const int nb = ROPE ? nb_all - 1 : nb_all;                   // of them from memory
  const int64_t n_blocks = (c.n_ctx + kBlk - 1) / kBlk;
  const int8_t *kb = c.k + kvh * n_blocks * (kBlk * HD), *vb = c.v + kvh * n_blocks * (kBlk * HD);
  const float *ksc = c.k_scale + kvh * n_blocks, *vsc = c.v_scale + kvh * n_blocks;
  struct Buf {
    u4v k[2][KJ], v[VJ];
    float ks, vs;
  };
  auto load = [&](int b, Buf &x) {
    b = b < nb ? b : nb_all - 1;  // (past the last one: not used)
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
  const bool owner = ROPE && j == 0;
  int b = owner ? nb : (ROPE ? j - 1 : j) * NW + wave;
  if (!owner) load(b, b0);
  // the owner's tokens: on their way before q's are waited for
  constexpr int UNITS = BlockTokens<HD>::UNITS, NT = 64 * kWaves;
  constexpr int UPT = 2 * UNITS / NT;  // units of K, then V, per thread
  float x[ROPE ? UPT : 1][16];
  auto tokens = [&](int i, int &u) {  // (the same w for the wave)
    int w;
    if constexpr (UNITS < NT) {
      w = __builtin_amdgcn_readfirstlane(threadIdx.x / UNITS);
      u = threadIdx.x % UNITS;
    } else {
      w = i / (UNITS / NT);
      u = threadIdx.x + NT * (i % (UNITS / NT));
    }
    return BlockTokens<HD>(c, kvh, w == 1, true, w ? vn : kn, sp, (int64_t)nb, rope);
  };
  bool gone[2] = {false, false};  // K's and V's block
  const bool coding = owner && wave < kWaves, asking = owner && wave == NW - 1;
  if constexpr (ROPE) {
    if (coding) {
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        int u;
        tokens(i, u).load(u, x[i]);
      }
#pragma unroll
      for (int i = 0; i < UPT; ++i) {  // (awaited when all loads are on their way)
        int u;
        const BlockTokens<HD> blk = tokens(i, u);
        gone[blk.is_v] = blk.gone();
      }
    }
  }
  QRow<HD> qr;
  if (!coding || asking)
    qr.template load<ROPE>(q + ((int64_t)tok * n_head + kvh * G + g) * HD, live, cg, sp.p0, rope);
  RowState<HD> s;
  s.clear();
  auto compute = [&](int blk, Buf &x, auto mask) {
    constexpr bool MASK = decltype(mask)::value;
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
    const int first = blk * kBlk;  // (below n_ctx, and with it 2^31)
    if (MASK && first > lim0 - (kBlk - 1)) {  // (uniform) some row ends inside it or before
      const int d = lim - first - 4 * cg;
      const int last[1] = {d > 64 ? 64 : d < -1 ? -1 : d};
      softmax_step<HD, 1, true>(s, sc, f, qr.back, ks, vs, last, ph, pl);
    } else {
      const int last[1] = {0};
      softmax_step<HD, 1, false>(s, sc, f, qr.back, ks, vs, last, ph, pl);
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
  if constexpr (ROPE) {
    if (owner) {
      if (coding) {
        uint32_t am[2] = {0, 0};  // of K's and V's units (a wave's units are of one each)
#pragma unroll
        for (int i = 0; i < UPT; ++i) {
          int u;
          const BlockTokens<HD> blk = tokens(i, u);
          if (gone[blk.is_v]) {
            blk.reopen(u, x[i]);
            blk.keep(u, 0, x[i]);
          } else if (!blk.is_v) {
            blk.keep(u, blk.before, x[i]);  // (its own row; no other thread reads it)
          }
          const uint32_t a = amax16(x[i], 0);
          am[0] = max(am[0], blk.is_v ? 0u : a);
          am[1] = max(am[1], blk.is_v ? a : 0u);
        }
        for (int d = threadIdx.x; d < HD; d += NT)  // V's tail row: the token's values
          c.v_tail[((int64_t)kvh * kBlk + sp.p0 % kBlk) * HD + d] = vn[kvh * HD + d];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          am[w] = wave_umax(am[w]);
          if (lane == 0) red[w][wave] = am[w];
        }
      }
      __syncthreads();
      float sc[2];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        sc[w] = scale_of(max(max(red[w][0], red[w][1]), max(red[w][2], red[w][3])));
        if (threadIdx.x == 0) {
          (w ? c.v_scale : c.k_scale)[kvh * n_blocks + nb] = sc[w];
          reinterpret_cast<int32_t *>((w ? c.v_tail : c.k_tail) +
                                      (int64_t)c.n_kv * kBlk * HD)[kvh] = nb;
        }
      }
      if (coding) {
#pragma unroll
        for (int i = 0; i < UPT; ++i) {
          int u;
          const BlockTokens<HD> blk = tokens(i, u);
          const int w = blk.is_v ? 1 : 0;
          const uint4 cd = Coder(w ? sc[1] : sc[0])(x[i]);
          own[w][u] = cd;
          reinterpret_cast<uint4 *>((w ? c.v : c.k) + (kvh * n_blocks + nb) * (kBlk * HD))[u] = cd;
        }
      }
      __syncthreads();
      if (asking) {
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
          for (int jj = 0; jj < KJ; ++jj)
            b0.k[pt][jj] = *reinterpret_cast<const u4v *>(
                &own[0][((16 * pt + r16) * HD + 64 * jj + 16 * cg) / 16]);
#pragma unroll
        for (int i = 0; i < VJ; ++i)
          b0.v[i] = *reinterpret_cast<const u4v *>(&own[1][(16 * i + r16) * 4 + cg]);
        b0.ks = sc[0];
        b0.vs = sc[1];
        compute(nb, b0, std::true_type());
      }
    }
  }
  const int stride = (ROPE ? S - 1 : S) * NW;
  constexpr auto mask = std::integral_constant<bool, !ROPE>();  // (full blocks before the token's)
  while (b < nb) {
    load(b + stride, b1);
    compute(b, b0, mask);
    if ((b += stride) >= nb) break;
    load(b + stride, b0);
    compute(b, b1, mask);
    b += stride;
  }
  // the waves' states, then one state per row
  s.l = row_sum(s.l);
  if (cg == 0) {
    stat[wave][0][r16] = s.m;
    stat[wave][1][r16] = s.D;
    stat[wave][2][r16] = s.l;
  }
  float *dst = S == 1 ? out + ((int64_t)tok * n_head + kvh * G + g) * HD
                      : part + (((int64_t)kvh * T * G + id) * S + j) * PS;
  Ref all{-INFINITY, kLow};
  float den = 0.f, fo[NW];
#pragma unroll
  for (int h = 0; h < PARTS; ++h) {
    if (h) __syncthreads();
#pragma unroll
    for (int i = 0; i < 2 * VP; ++i) os[wave][i][lane] = s.o[2 * VP * h + i];
    __syncthreads();
    if (h == 0) {
      all = joined<NW>([&](int w) { return stat[w][0][r16]; },
                       [&](int w) { return stat[w][1][r16]; });
      const float mref = finite_ref(all.m);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        den = fmaf(stat[w][2][r16], exp2_(stat[w][0][r16] - mref), den);
        fo[w] = exp2_(moved(stat[w][1][r16], stat[w][0][r16], mref) - all.D);
      }
    }
    const OutScale fin(all.D, den);
    for (int i = wave; i < VP; i += NW) {
      f4v a[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        a[e] = os[0][2 * i + e][lane] * fo[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) a[e] += os[w][2 * i + e][lane] * fo[w];
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
    *reinterpret_cast<f4v *>(dst + HD) = f4v{all.m, all.D, den, 0.f};
}

// One workgroup per query row merges the splits' states: HD / 4 threads of 16
// bytes a split, all of a chunk's loads (and the m, D, l of every split) in
// flight at once.  Bound by a launch's start and two trips to memory: 3.0-3.9 us
// at 18 to 64 splits (loads one after the other: 31 at 64).
constexpr int kMaxSplits = 512;
template <int HD>
__global__ void __launch_bounds__(kWG)
    k_kv8_combine(const float *__restrict__ part, const aq_decode_state *st, int64_t pos0,
                  int64_t n_ctx, int64_t T, int G, int S, float *__restrict__ out) {
  constexpr int PS = HD + 4, LP = HD / 4, NG = kWG / LP, U = 8;
  __shared__ float fo[kMaxSplits + 8];
  __shared__ float red[3][kWG / 64];
  __shared__ f4v acc[NG][LP];
  const int id = blockIdx.x, t = id / G, kvh = blockIdx.y, n_head = gridDim.y * G;
  const int tid = threadIdx.x, d4 = tid % LP, grp = tid / LP;
  const float *p = part + ((int64_t)kvh * T * G + id) * S * PS;
  f4v x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int s = grp + NG * u;
    x[u] = *reinterpret_cast<const f4v *>(p + (s < S ? s : 0) * PS + 4 * d4);
  }
  f4v e[2];  // m, D, l of splits tid and tid + 256
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int s = tid + kWG * i;
    e[i] = f4v{-INFINITY, kLow, 0.f, 0.f};
    if (s < S) e[i] = *reinterpret_cast<const f4v *>(p + s * PS + HD);
  }
  const Span sp = span_of(st, pos0, T, n_ctx);
  if (t >= sp.n) return;
  // (the wave's maximum, then its reference counted from it, then the waves')
  const float wm = wave_max(fmaxf(e[0][0], e[1][0])), wref = finite_ref(wm);
  const float wd = wave_max(fmaxf(moved(e[0][1], e[0][0], wref), moved(e[1][1], e[1][0], wref)));
  if ((tid & 63) == 0) {
    red[0][tid >> 6] = wm;
    red[1][tid >> 6] = wd;
  }
  __syncthreads();
  const Ref all = joined<kWG / 64>([&](int w) { return red[0][w]; },
                                   [&](int w) { return red[1][w]; });
  const float mref = finite_ref(all.m);
  float den = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (tid + kWG * i < S) fo[tid + kWG * i] = exp2_(moved(e[i][1], e[i][0], mref) - all.D);
    den = fmaf(e[i][2], exp2_(e[i][0] - mref), den);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) den += __shfl_xor(den, off);
  if ((tid & 63) == 0) red[2][tid >> 6] = den;
  __syncthreads();
  den = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
  f4v o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0;;) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + grp + NG * u;
      if (s < S) o += x[u] * fo[s];
    }
    s0 += NG * U;
    if (s0 >= S) break;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + grp + NG * u;
      x[u] = *reinterpret_cast<const f4v *>(p + (s < S ? s : 0) * PS + 4 * d4);
    }
  }
  acc[grp][d4] = o;
  __syncthreads();
  if (tid >= LP) return;
#pragma unroll
  for (int w = 1; w < NG; ++w) o += acc[w][d4];
  const OutScale fin(all.D, den);
  reinterpret_cast<f4v *>(out + ((int64_t)t * n_head + kvh * G + (id - t * G)) * HD)[d4] = fin(o);
}

// The merge of up to kFewSplits splits of many rows: HD / 4 threads per row, all
// its loads in flight at once, no LDS.  Bound by the states' bytes: 256 tokens
// of 32 heads of 128 in 4 splits (17 MB in, 4 out, from the last-level cache)
// 5.3 us (through k_kv8_combine the whole call took 95 us, not 85).
constexpr int kFewSplits = 8;
template <int HD>
__global__ void __launch_bounds__(kWG)
    k_kv8_combine_few(const float *__restrict__ part, const aq_decode_state *st, int64_t pos0,
                      int64_t n_ctx, int64_t T, int G, int S, float *__restrict__ out) {
  constexpr int PS = HD + 4, LP = HD / 4;
  const int id = blockIdx.x * (kWG / LP) + threadIdx.x / LP, d4 = threadIdx.x % LP;
  const int kvh = blockIdx.y, n_head = gridDim.y * G, t = id / G;
  const Span sp = span_of(st, pos0, T, n_ctx);
  if (t >= sp.n) return;
  const float *p = part + ((int64_t)kvh * T * G + id) * S * PS;
  f4v x[kFewSplits], e[kFewSplits];  // numerators; m, D, l
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    const float *ps = p + (s < S ? s : 0) * PS;
    x[s] = *reinterpret_cast<const f4v *>(ps + 4 * d4);
    e[s] = *reinterpret_cast<const f4v *>(ps + HD);
  }
  // (repeats of the first split change nothing)
  const Ref all = joined<kFewSplits>([&](int s) { return e[s][0]; },
                                     [&](int s) { return e[s][1]; });
  const float mref = finite_ref(all.m);
  f4v o = {0.f, 0.f, 0.f, 0.f};
  float den = 0.f;
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    if (s >= S) break;
    o += x[s] * exp2_(moved(e[s][1], e[s][0], mref) - all.D);
    den = fmaf(e[s][2], exp2_(e[s][0] - mref), den);
  }
  const OutScale fin(all.D, den);
  reinterpret_cast<f4v *>(out + ((int64_t)t * n_head + kvh * G + (id - t * G)) * HD)[d4] = fin(o);
}

// ---- many rows: tiles of rows over all positions they see -------------------------
// One workgroup of four waves per 64 rows (16 per wave) of a kv head and split of
// the positions (gridDim.y of them; one writes the output, several their states
// for the merge).  The chunks of two blocks are converted to fp16 in operand
// order in LDS once for all waves (each lane's 16 bytes at its place: no
// conflicts).  A wave's pass over chunk ch forms the scores of chunk ch + 1 while
// the softmax of chunk ch runs (the matrix and the vector instructions of one
// pass do not wait for each other), then adds the values of chunk ch; K of chunk
// ch + 2 and V of chunk ch + 1 go to LDS meanwhile, the codes after them are on
// their way, and one barrier ends it.
//
// Bound by issue, matrix and vector instructions together (matrix cores busy 34 %
// and 38 % of the time; each useful product is two, of two pieces).  2048 tokens of
// 32 / 8 heads of 64 from the start 50-52 us a call in a row of calls, 55 traced
// (17.2 useful GFLOP: 0.33 PFLOP/s, 0.66 with both pieces); 777 of 32 / 8 heads of
// 128 behind 2901 113 us, 125 traced (0.37, 0.74).
// Slower: two row tiles per wave (74 and 182 against 66 and 146 then), eight waves
// (57 and 143), q's pieces from LDS, rescaling always (61 against 57).
template <int HD>
__global__ void __launch_bounds__(64 * kWaves, HD == 64 ? 4 : 1)
    k_kv8_tiles(const float *__restrict__ q, aq_kv8 c, const aq_decode_state *st, int64_t pos0,
                int64_t T, int G, float f, int tiles, int layer, float *__restrict__ part,
                float *__restrict__ out) {
  constexpr int KJ = HD / 64, VJ = HD / 32, KS = HD / 32;
  constexpr int NU = HD / 64;  // 1 KB units of a chunk's K (and of its V) per wave
  // 128 dimensions and more have the registers to read four operands ahead (127 us,
  // one ahead 134); at 64 it costs (59, one ahead 56)
  constexpr int AHEAD = HD >= 128 ? 4 : 1;
  extern __shared__ __attribute__((aligned(16))) h8 lds[];
  auto kl = reinterpret_cast<h8(*)[4 * KS][64]>(lds);                // [2][position tile, k step][lane]
  auto vl = reinterpret_cast<h8(*)[4 * VJ][64]>(lds + 2 * 4 * KS * 64);  // [2][block, dim. tile][lane]
  const Span sp = span_of(st, pos0, T, c.n_ctx);
  // The tiles that see most first; every other layer of `layer` tiles (what the
  // GPU's CUs take of a kv head at once) the other way round, so that CUs that
  // hold several workgroups get alike sums.  A kv head's tiles are n_kv apart in
  // the grid (workgroup id modulo 8 is the XCD: one L2 per kv head).
  const int n_kv = c.n_kv, kvh = blockIdx.x % n_kv, n_head = n_kv * G;
  int rank = (int)(blockIdx.x / n_kv);
  const int ly = rank / layer, in = rank - ly * layer;
  if ((ly & 1) && (ly + 1) * layer <= tiles) rank = ly * layer + layer - 1 - in;
  const int tile = tiles - 1 - rank;
  const int rows = (int)sp.n * G, id0 = tile * (16 * kWaves);
  if (id0 >= rows) return;
  const int lane = threadIdx.x & 63, r16 = lane & 15, cg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id_last = id0 + 16 * kWaves - 1;
  id_last = id_last < rows ? id_last : rows - 1;
  const int64_t p_last = sp.p0 + id_last / G;  // the last position any row sees
  const int nb = (int)(p_last / kBlk) + 1, nc = (nb + 1) / 2;
  // the split's chunks c0 .. c1 - 1, of which every row sees those below n_full whole
  const int S = gridDim.y, split = blockIdx.y;
  const int c0 = (int)((int64_t)nc * split / S), c1 = (int)((int64_t)nc * (split + 1) / S);
  int n_full = (int)((sp.p0 + id0 / G + 1) / (2 * kBlk));
  n_full = n_full < c1 ? n_full : c1;
  const int id = id0 + wave * 16 + r16;
  const bool live = id < rows;
  const int tok = live ? id / G : 0, g = live ? id - tok * G : 0;
  const int lim = (int)sp.p0 + tok;  // the row's last position
  const int64_t qo = ((int64_t)tok * n_head + kvh * G + g) * HD;
  const int64_t n_blocks = (c.n_ctx + kBlk - 1) / kBlk;
  const int8_t *kb = c.k + kvh * n_blocks * (kBlk * HD) + r16 * HD + 16 * cg;
  const int8_t *vb = c.v + kvh * n_blocks * (kBlk * HD) + r16 * 64 + 16 * cg;
  const float *ksc = c.k_scale + kvh * n_blocks, *vsc = c.v_scale + kvh * n_blocks;
  u4v rk[NU], rv[NU];
  // block 2 ch + u, the last one past the end (a partner that is masked, or a
  // chunk that is not used); block numbers are the wave's: scalar
  auto block = [&](int ch, int u) { return (int64_t)(2 * ch + u < nb ? 2 * ch + u : nb - 1); };
  auto fetch_k = [&](int ch) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int x = wave + kWaves * i, pt = x / KJ, jj = x % KJ;
      rk[i] = *reinterpret_cast<const u4v *>(
          kb + (block(ch, pt >> 1) * kBlk + 16 * (pt & 1)) * HD + 64 * jj);
    }
  };
  auto fetch_v = [&](int ch) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int x = wave + kWaves * i, u = x / VJ, jv = x % VJ;
      rv[i] = *reinterpret_cast<const u4v *>(vb + block(ch, u) * (kBlk * HD) + 1024 * jv);
    }
  };
  auto stage = [&](const u4v (&r)[NU], h8 (*dst)[64]) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int x = wave + kWaves * i;
      codes16(r[i], dst[2 * x][lane], dst[2 * x + 1][lane]);
    }
  };
  auto scales = [&](int ch, float (&ks)[2], float (&vs)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      ks[u] = load_const(ksc + block(ch, u));
      vs[u] = load_const(vsc + block(ch, u));
    }
  };
  QRow<HD> qr;
  RowState<HD> s;
  s.clear();
  auto scores = [&](const h8 (*k)[64], f4v (&sc)[4]) {
#pragma unroll
    for (int pt = 0; pt < 4; ++pt) sc[pt] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int p0 = 0; p0 < 4; p0 += AHEAD) {
        h8 kf[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) kf[i] = k[(p0 + i) * KS + ks][lane];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
          sc[p0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i], qr.lo[ks], sc[p0 + i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
          sc[p0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i], qr.hi[ks], sc[p0 + i], 0, 0, 0);
      }
  };
  float ks[2], vs[2];
  auto pass = [&](int ch, f4v (&sc)[4], f4v (&next)[4], auto masked) {
    constexpr bool MASK = decltype(masked)::value;
    const int odd = (ch - c0) & 1;
    stage(rk, kl[odd]);
    stage(rv, vl[odd ^ 1]);
    fetch_k(ch + 3);
    fetch_v(ch + 2);
    float nks[2], nvs[2];
    scales(ch + 1, nks, nvs);
    scores(kl[odd ^ 1], next);
    h8 ph[2], pl[2];
    int last[2] = {0, 0};
    if constexpr (MASK) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int d = lim - ((2 * ch + u) * kBlk + 4 * cg);
        last[u] = d > 64 ? 64 : d < -1 ? -1 : d;
      }
    }
    softmax_step<HD, 2, MASK>(s, sc, f, qr.back, ks, vs, last, ph, pl);
    const h8 (*v)[64] = vl[odd];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int h0 = 0; h0 < 2 * VJ; h0 += AHEAD) {
        h8 vf[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) vf[i] = v[2 * u * VJ + h0 + i][lane];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
          s.o[h0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[i], pl[u], s.o[h0 + i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
          s.o[h0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[i], ph[u], s.o[h0 + i], 0, 0, 0);
      }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      ks[u] = nks[u];
      vs[u] = nvs[u];
    }
    __syncthreads();
  };
  fetch_k(c0);
  fetch_v(c0);
  scales(c0, ks, vs);
  qr.template load<false>(q + qo, live, cg, 0, Rope{});
  stage(rk, kl[0]);
  stage(rv, vl[0]);
  fetch_k(c0 + 1);
  fetch_v(c0 + 1);
  stage(rk, kl[1]);
  fetch_k(c0 + 2);
  __syncthreads();
  f4v sa[4], sb[4];
  scores(kl[0], sa);
  __syncthreads();  // (the first chunk's keys have been read)
  int ch = c0;
  for (; ch + 1 < n_full; ch += 2) {
    pass(ch, sa, sb, std::false_type());
    pass(ch + 1, sb, sa, std::false_type());
  }
  for (; ch < c1; ++ch) {
    pass(ch, sa, sb, std::true_type());
#pragma unroll
    for (int i = 0; i < 4; ++i) sa[i] = sb[i];
  }
  const float den = row_sum(s.l);
  if (!live) return;
  const OutScale fin(s.D, den);
  float *dst = S == 1 ? out + qo : part + (((int64_t)kvh * T * G + id) * S + split) * (HD + 4);
  if (S > 1 && cg == 0) *reinterpret_cast<f4v *>(dst + HD) = f4v{s.m, s.D, den, 0.f};
#pragma unroll
  for (int i = 0; i < VJ; ++i) {
    f4v a = s.o[2 * i], b = s.o[2 * i + 1];
    if (S == 1) a = fin(a), b = fin(b);
    f4v *o4 = reinterpret_cast<f4v *>(dst + 8 * cg + 32 * i);
    o4[0] = f4v{a[0], b[0], a[1], b[1]};
    o4[1] = f4v{a[2], b[2], a[3], b[3]};
  }
}

}  // namespace

bool kv8_supported(int head_dim) { return head_dim == 64 || head_dim == 128 || head_dim == 256; }

// partials of at most this many (query row, split)s
constexpr int64_t kScratchRows = 65536;
// most rows per kv head for the split kernel: it converts every block once per
// tile of 16 rows, the tiles kernel once per 64, but by way of LDS and barriers.
// 32/8 heads of 128 after 8000 positions, split against tiles: 32 rows 14.8 / 20.5
// us, 64 18.2 / 20.6, 128 24.1 / 26.3, 256 36.0 / 38.9; 16/8 heads of 256: 64 rows
// 26.4 / 52.9, 128 38.2 / 53.7, 256 62.0 / 56.0.
constexpr int64_t kSplitRows = 256;
size_t kv8_scratch_bytes(int head_dim) {
  return (size_t)kScratchRows * (head_dim + 4) * sizeof(float);
}

#define AQ_HD(hd, ...)                                    \
  switch (hd) {                                           \
    case 64: { constexpr int HD = 64; __VA_ARGS__; } break;      \
    case 128: { constexpr int HD = 128; __VA_ARGS__; } break;    \
    case 256: { constexpr int HD = 256; __VA_ARGS__; } break;    \
    default: return hipErrorInvalidValue;                 \
  }

hipError_t launch_rope_kv8(const float *q, const float *k, const float *v, float *q_out, int64_t T,
                           int n_head, int n_rot, int neox, const float *cos_t,
                           const float *sin_t, const aq_decode_state *st, int64_t pos0,
                           const aq_kv8 &c, hipStream_t s) {
  const int64_t blocks = (T + kBlk - 2) / kBlk + 1;  // blocks T positions can touch
  const int64_t n_store = blocks * c.n_kv * 2;
  const Rope rope{cos_t, sin_t, n_rot, neox};
  const int64_t n_q = !q ? 0 : T < 65536 ? T : 65536;
  AQ_HD(c.head_dim, hipLaunchKernelGGL(k_kv8_store<HD>, dim3((unsigned)(n_store + n_q)),
                                       dim3(kStoreWG<HD>), 0, s, q, k, v, q_out, T, n_head, rope,
                                       st, pos0, c, n_store))
  return hipGetLastError();
}

hipError_t launch_kv8_read(const aq_kv8 &c, int64_t start, int64_t n, float *k, float *v,
                           hipStream_t s) {
  const int64_t blocks = (start + n - 1) / kBlk - start / kBlk + 1;
  AQ_HD(c.head_dim,
        hipLaunchKernelGGL(k_kv8_read<HD>, dim3((unsigned)(2 * blocks), (unsigned)c.n_kv),
                           dim3(kStoreWG<HD>), 0, s, c, start, n, k, v))
  return hipGetLastError();
}

// The splits of the positions.  Both rules go by the cache's length, not by the
// position, which the host may not know: a call gives the same bits however it
// is told where it is.
//
// Workgroups of the split and of the tiles kernel that a CU has the registers for
// at once: heads of 256 take more than half of a SIMD's per wave (and the tiles
// 128 KB of LDS), so one; a second turn is then no faster than a second launch.
constexpr int kv8_residents(int head_dim) { return head_dim == 256 ? 1 : 2; }
// The split kernel: as many workgroups as 256 CUs hold (rounded up to whole splits
// where that is two each and there are no others), no more than give every wave a
// block of a full cache, nor than the scratch holds.  more: workgroups per kv head
// beside them (the step's), which would else leave some for a second turn: the step
// of 32 / 8 heads of 128 at 32128 positions, 64 + 1 splits a kv head 20.3 us, 63 + 1
// 17.8.  Heads of 256, 32767 positions, 8 kv heads: 32 splits 28.8, 64 33.4; 4 kv
// heads: 64 splits 20.6, 128 27.2; the step, 8 kv heads: 31 + 1 31.4, 64 + 1 43.4.
int kv8_splits(const aq_kv8 &c, int64_t tiles, int64_t rows, int waves, int more) {
  const int64_t n_blocks = (c.n_ctx + kBlk - 1) / kBlk, groups = c.n_kv * tiles;
  const int64_t hold = 256 * kv8_residents(c.head_dim);
  int64_t S = (n_blocks + waves - 1) / waves;
  int64_t fill = (hold - more * c.n_kv) / groups;
  if (hold > 256 && !more) fill = (hold - 2 + groups) / groups;
  const int64_t room = kScratchRows / rows - 1;
  S = S < fill ? S : fill;
  S = S < room ? S : room;
  return (int)(S < 1 ? 1 : S);
}
// The tiles kernel: the smallest estimate.  A workgroup takes about head_dim / 96
// us per chunk, two on a CU 1.3 times that, where a CU holds two, else and beyond
// in turn; the splits' states go through memory once each way, in a launch of its
// own.  32/8 heads of 128: 256 tokens at 8000 172 us whole, 85 in four splits.
// Heads of 256, groups of 4: 700 tokens of 5 kv heads at 3396 (220 workgroups) 162
// whole, 166 in two; 512 of 4 at 3000 (128) 137, in two 84, in four 90; 256 (64)
// 128, in four 50, in eight 62.
int kv8_tile_splits(const aq_kv8 &c, int64_t tiles, int64_t rows, int cus) {
  const double chunks = (double)((c.n_ctx + 2 * kBlk - 1) / (2 * kBlk));
  const double beside = kv8_residents(c.head_dim) == 1 ? 1.0 : 0.65;
  double best = 0.0;
  int pick = 1;
  for (int S = 1; S <= kFewSplits && S <= chunks && (S == 1 || rows * S <= kScratchRows); ++S) {
    const double turns = ceil((double)(tiles * c.n_kv * S) / cus);
    const double t = ceil(chunks / S) * (c.head_dim / 96.0) * (turns > 1 ? beside * turns : 1.0) +
                     (S > 1 ? 4.0 + (double)rows * S * (c.head_dim + 4) * 8 / 4e6 : 0.0);
    if (S == 1 || t < best) {
      best = t;
      pick = S;
    }
  }
  return pick;
}

// scores to exponents of two
static float score_factor(int head_dim) { return (float)(1.0 / sqrt((double)head_dim)) * kLog2e; }

hipError_t launch_attention_kv8(const float *q, const aq_kv8 &c, int64_t T, int n_head,
                                const aq_decode_state *st, int64_t pos0, float *out,
                                hipStream_t s) {
  const float f = score_factor(c.head_dim);
  const int G = n_head / c.n_kv;
  const int64_t rows = T * G;
  int S;
  if (rows <= kSplitRows) {
    const int64_t tiles = (rows + 15) / 16;
    S = kv8_splits(c, tiles, T * n_head, kWaves, 0);
    AQ_HD(c.head_dim,
          hipLaunchKernelGGL((k_kv8_split<HD, false, kWaves>),
                             dim3((unsigned)S, (unsigned)c.n_kv, (unsigned)tiles),
                             dim3(64 * kWaves), 0, s, q, c, st, pos0, T, G, f, c.scratch, out,
                             nullptr, nullptr, Rope{}))
  } else {
    int dev = 0;
    if (hipError_t e = hipGetDevice(&dev)) return e;
    const int cus = device_info(dev).cus;
    const int layer = cus / c.n_kv > 1 ? cus / c.n_kv : 1;
    const int64_t tiles = (rows + 16 * kWaves - 1) / (16 * kWaves);
    S = kv8_tile_splits(c, tiles, T * n_head, cus);
    const int lds = 512 * c.head_dim;  // two chunks of K and of V in fp16
    AQ_HD(c.head_dim,
          if (hipError_t e = set_dynamic_lds(reinterpret_cast<const void *>(k_kv8_tiles<HD>), lds))
            return e;
          hipLaunchKernelGGL(k_kv8_tiles<HD>, dim3((unsigned)(tiles * c.n_kv), (unsigned)S),
                             dim3(64 * kWaves), lds, s, q, c, st, pos0, T, G, f, (int)tiles,
                             layer, c.scratch, out))
  }
  if (S > 1 && S <= kFewSplits) {
    AQ_HD(c.head_dim,
          constexpr int R = kWG / (HD / 4);
          hipLaunchKernelGGL(k_kv8_combine_few<HD>,
                             dim3((unsigned)((rows + R - 1) / R), (unsigned)c.n_kv), dim3(kWG), 0,
                             s, c.scratch, st, pos0, c.n_ctx, T, G, S, out))
  } else if (S > 1) {
    AQ_HD(c.head_dim, hipLaunchKernelGGL(k_kv8_combine<HD>, dim3((unsigned)rows, (unsigned)c.n_kv),
                                         dim3(kWG), 0, s, c.scratch, st, pos0, c.n_ctx, T, G, S,
                                         out))
  }
  return hipGetLastError();
}

hipError_t launch_attention_rope_kv8(const float *q, const float *k, const float *v, int n_head,
                                     int n_rot, int neox, const float *cos_t, const float *sin_t,
                                     const aq_decode_state *st, int64_t pos0, const aq_kv8 &c,
                                     float *out, hipStream_t s) {
  const float f = score_factor(c.head_dim);
  const int G = n_head / c.n_kv;
  // five waves where a CU gets one workgroup
  const bool five =
      c.head_dim < 256 && (kv8_splits(c, 1, n_head, kWaves + 1, 1) + 1) * c.n_kv <= 256;
  const int waves = five ? kWaves + 1 : kWaves, S = kv8_splits(c, 1, n_head, waves, 1) + 1;
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((unsigned)S, (unsigned)c.n_kv, 1u), dim3(64 * waves), 0, s, q, c,
                       st, pos0, (int64_t)1, G, f, c.scratch, out, k, v,
                       Rope{cos_t, sin_t, n_rot, neox});
  };
  AQ_HD(c.head_dim,
        if (five) go(k_kv8_split<HD, true, HD < 256 ? kWaves + 1 : kWaves>);
        else go(k_kv8_split<HD, true, kWaves>);
        hipLaunchKernelGGL(k_kv8_combine<HD>, dim3((unsigned)G, (unsigned)c.n_kv), dim3(kWG), 0, s,
                           c.scratch, st, pos0, c.n_ctx, (int64_t)1, G, S, out))
  return hipGetLastError();
}

}  // namespace aq
