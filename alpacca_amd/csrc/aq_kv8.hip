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
// One workgroup per (query token, head): 256 positions at a time, a score per
// thread, with the running maximum and sum of the softmax.
template <int HD>
__global__ void __launch_bounds__(kWG)
    k_kv8_attn(const float *__restrict__ q, aq_kv8 c, const aq_decode_state *st, int64_t pos0,
               int64_t T, int n_head, float scale, float *__restrict__ out) {
  __shared__ float qs[HD], ws[kWG], part[kWG], red[kWG / 64];
  const Span sp = span_of(st, pos0, T, c.n_ctx);
  const int64_t t = blockIdx.x;
  if (t >= sp.n) return;
  const int h = blockIdx.y, kvh = h / (n_head / c.n_kv), tid = threadIdx.x;
  const int64_t L = sp.p0 + t + 1, n_blocks = (c.n_ctx + kBlk - 1) / kBlk;
  for (int d = tid; d < HD; d += kWG) qs[d] = q[(t * n_head + h) * HD + d];
  __syncthreads();
  constexpr int NP = kWG / HD > 0 ? kWG / HD : 1;  // parts of the positions per dimension
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int64_t c0 = 0; c0 < L; c0 += kWG) {
    const int64_t p = c0 + tid;
    float z = -INFINITY, vs = 0.f;
    if (p < L) {
      const int64_t blk = kvh * n_blocks + p / kBlk;
      const int8_t *kr = c.k + blk * (kBlk * HD) + (p % kBlk) * HD;
      float a = 0.f;
      for (int d = 0; d < HD; ++d) a = fmaf(qs[d], (float)kr[d], a);
      z = a * c.k_scale[blk] * scale;
      vs = c.v_scale[blk];
    }
    float mx = z;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
    if ((tid & 63) == 0) red[tid >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float mn = fmaxf(m, mx), corr = m == -INFINITY ? 0.f : expf(m - mn);
    const float e = p < L ? expf(z - mn) : 0.f;
    l = fmaf(l, corr, e);
    ws[tid] = p < L ? e * vs : 0.f;
    m = mn;
    __syncthreads();
    o *= corr;
    const int d = tid % HD, p_part = tid / HD;
    const int np = (int)(L - c0 < kWG ? L - c0 : kWG);
    for (int j = p_part; j < np; j += NP) {
      const int64_t pj = c0 + j;
      o = fmaf(ws[j], (float)c.v[(kvh * n_blocks + pj / kBlk) * (kBlk * HD) + v_byte((int)(pj % kBlk), d)], o);
    }
    __syncthreads();
  }
  part[tid] = o;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off);
  if ((tid & 63) == 0) red[tid >> 6] = l;
  __syncthreads();
  const float den = (red[0] + red[1]) + (red[2] + red[3]);
  if (tid < HD) {
    float num = 0.f;
    for (int j = 0; j < NP; ++j) num += part[j * HD + tid];
    out[(t * n_head + h) * HD + tid] = num / den;
  }
}

}  // namespace

bool kv8_supported(int head_dim) { return head_dim == 64 || head_dim == 128 || head_dim == 256; }

// partials of at most this many (query row, split)s
constexpr int64_t kScratchRows = 16384;
size_t kv8_scratch_bytes(int head_dim) {
  return (size_t)kScratchRows * (head_dim + 4) * sizeof(float);
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

hipError_t launch_attention_kv8(const float *q, const aq_kv8 &c, int64_t T, int n_head,
                                const aq_decode_state *st, int64_t pos0, float *out,
                                hipStream_t s) {
  const float scale = (float)(1.0 / sqrt((double)c.head_dim));
  AQ_HD(c.head_dim, hipLaunchKernelGGL(k_kv8_attn<HD>, dim3((unsigned)T, (unsigned)n_head),
                                       dim3(kWG), 0, s, q, c, st, pos0, T, n_head, scale, out))
  return hipGetLastError();
}

hipError_t launch_attention_rope_kv8(const float *q, const float *k, const float *v, int n_head,
                                     int n_rot, int neox, const float *cos_t, const float *sin_t,
                                     const aq_decode_state *st, int64_t pos0, const aq_kv8 &c,
                                     float *out, hipStream_t s) {
  if (n_head > kScratchRows) return hipErrorInvalidValue;
  hipError_t e = launch_rope_kv8(q, k, v, c.scratch, 1, n_head, n_rot, neox, cos_t, sin_t, st,
                                 pos0, c, s);
  return e != hipSuccess ? e : launch_attention_kv8(c.scratch, c, 1, n_head, st, pos0, out, s);
}

}  // namespace aq
