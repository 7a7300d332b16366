// aq_logits.hip - what stands between the head and the choice of a token:
// penalties for tokens already said, biases and a grammar's mask, per row.
#include "aq_internal.h"

namespace aq {
namespace {

constexpr int kWG = 256;
constexpr int kAhead = 4;  // tokens and entries a thread loads ahead
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

// Workgroup (slice of 1024 V logits, row).  The logits and mask words of the
// slice are on their way first.  The window's tokens and the biased tokens that
// fall into it are marked in LDS (a count, and the index of the last entry, by
// integer atomics, so their order does not show) and listed once each; then the
// logits that nothing touches pass through 16 bytes at a time, and the listed
// ones, a few, are adjusted a thread each, in double and rounded once.  In place,
// only listed and masked logits are touched.
//
// Bound by the logits' bytes for a batch: 64 rows of 128256 in 16-18 us (the
// mask's and 66 MB: 3.9 TB/s; slices of 4096 and 8192 23 and 38); one row in
// 4.0 (a launch's start and a chain of loads).
template <int V>
__global__ void __launch_bounds__(kWG)
    k_logits_adjust(const float *x, int64_t n, const int64_t *__restrict__ window, int64_t last_n,
                    const double *__restrict__ pen, const int64_t *__restrict__ bias_ids,
                    const float *__restrict__ bias, const int64_t *__restrict__ bias_off,
                    int64_t n_bias, const uint32_t *__restrict__ mask, int64_t mask_ld,
                    float *out) {
#pragma clang fp contract(off)
  constexpr int SL = 1024 * V;
  __shared__ __attribute__((aligned(16))) uint32_t cnt[SL];
  __shared__ __attribute__((aligned(16))) uint32_t ent[SL];  // 1 + the last entry of the token
  __shared__ uint32_t touched[SL / 32];
  __shared__ uint16_t list[SL];
  __shared__ int n_list;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y, base = (int64_t)blockIdx.x * SL;
  const bool in_place = x == out;
  x += row * n + base;
  out += row * n + base;
  const int len = (int)(n - base < SL ? n - base : SL);  // of the slice
  const uint32_t *mw = mask ? mask + row * mask_ld + (base >> 5) : nullptr;
  f4u xv[V];
  uint32_t allow[V];  // of the thread's four logits, bits 0 .. 3
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = 4 * (v * kWG + tid);
    allow[v] = 15u;
    if (e >= len) continue;
    if (mw) allow[v] = (mw[e >> 5] >> (e & 31)) & 15u;
    if (in_place) continue;
    if (e + 4 <= len) {
      xv[v] = *reinterpret_cast<const f4u *>(x + e);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) xv[v][k] = e + k < len ? x[e + k] : 0.f;
    }
  }
  // the first tokens of the window and entries of the list, before it is known how
  // many count
  const int64_t *w = window ? window + row * (1 + last_n) : nullptr;
  int64_t tok[kAhead], id[kAhead];
  int64_t a = bias_off && n_bias ? bias_off[row] : 0, b = bias_off && n_bias ? bias_off[row + 1] : n_bias;
  a = a < 0 ? 0 : a < n_bias ? a : n_bias;  // (also: a + j below does not wrap)
  b = b < n_bias ? b : n_bias;
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int64_t j = tid + kWG * i;
    tok[i] = w && j < last_n ? w[1 + j] : -1;
    id[i] = a + j < b ? bias_ids[a + j] : -1;
  }
  const int64_t seen = !w ? 0 : w[0] < last_n ? w[0] : last_n;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    reinterpret_cast<uint4 *>(cnt)[v * kWG + tid] = make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4 *>(ent)[v * kWG + tid] = make_uint4(0, 0, 0, 0);
  }
  if (tid < SL / 32) touched[tid] = 0;
  if (tid == 0) n_list = 0;
  __syncthreads();
  auto touch = [&](int t) {
    const uint32_t bit = 1u << (t & 31);
    if (!(atomicOr(&touched[t >> 5], bit) & bit)) list[atomicAdd(&n_list, 1)] = (uint16_t)t;
  };
  auto said = [&](int64_t t) {
    t -= base;
    if (t < 0 || t >= len) return;
    atomicAdd(&cnt[t], 1u);
    touch((int)t);
  };
  auto biased = [&](int64_t t, int64_t j) {
    t -= base;
    if (t < 0 || t >= len) return;
    atomicMax(&ent[t], (uint32_t)j + 1u);
    touch((int)t);
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int64_t j = tid + kWG * i;
    if (j < seen) said(tok[i]);
    if (a + j < b) biased(id[i], a + j);
  }
  for (int64_t j = tid + kWG * kAhead; j < seen; j += kWG) said(w[1 + j]);
  for (int64_t j = a + tid + kWG * kAhead; j < b; j += kWG) biased(bias_ids[j], j);
  double rep = 1.0, pres = 0.0, freq = 0.0;
  if (w) {
    rep = pen[row * 3];
    pres = pen[row * 3 + 1];
    freq = pen[row * 3 + 2];
  }
  __syncthreads();
  const float lowest = -__builtin_inff();
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = 4 * (v * kWG + tid);
    if (e >= len) continue;
    const uint32_t mine = (touched[e >> 5] >> (e & 31)) & 15u;  // the list's, unless masked
    f4u y;
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = (allow[v] >> k) & 1u ? xv[v][k] : lowest;
    // written here: masked ones, and out of place those not listed
    const uint32_t w = (in_place ? 0u : ~mine) | ~allow[v];
    if ((w & 15u) == 15u && e + 4 <= len) {
      *reinterpret_cast<f4u *>(out + e) = y;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (((w >> k) & 1u) && e + k < len) out[e + k] = y[k];
    }
  }
  const int m = n_list;
  for (int i = tid; i < m; i += kWG) {
    const int e = list[i];
    if (mw && !((mw[e >> 5] >> (e & 31)) & 1u)) continue;
    const uint32_t c = cnt[e], j = ent[e];
    double y = (double)x[e];
    if (c) {
      if (rep != 0.0 && rep != 1.0) y = y > 0.0 ? y / rep : y * rep;
      y = y - (pres + freq * (double)c);
    }
    if (j) y = y + (double)bias[j - 1];
    out[e] = (float)y;
  }
}

}  // namespace

hipError_t launch_logits_adjust(const float *logits, int64_t rows, int64_t n,
                                const int64_t *window, int64_t last_n, const double *pen,
                                const int64_t *bias_ids, const float *bias,
                                const int64_t *bias_off, int64_t n_bias, const uint32_t *mask,
                                int64_t mask_ld, float *out, hipStream_t s) {
  // Slices of 2048 logits where they fill the GPU several times over (every slice
  // reads its row's whole window and list: 64 rows of 128256 17.9 us against 18.4),
  // else of 1024 (4 rows 4.7 us against 5.0).  Larger ones leave too few waves on
  // a CU for their LDS (4096: 23.1 us).
  auto go = [&](auto kern, int64_t slice) {
    hipLaunchKernelGGL(kern, dim3((unsigned)((n + slice - 1) / slice), (unsigned)rows), dim3(kWG),
                       0, s, logits, n, window, last_n, pen, bias_ids, bias, bias_off, n_bias,
                       mask, mask_ld, out);
  };
  if (rows * ((n + 2047) / 2048) >= 1024) go(k_logits_adjust<2>, 2048);
  else go(k_logits_adjust<1>, 1024);
  return hipGetLastError();
}

}  // namespace aq
