// aq_logits.hip - what stands between the head and the choice of a token:
// penalties for tokens already said, biases and a grammar's mask, per row.
#include "aq_internal.h"

namespace aq {
namespace {

constexpr int kWG = 256;
constexpr int kSlice = 1024;  // logits per workgroup

// Workgroup (slice, row): the window's tokens and the biased tokens that fall
// into the slice are marked in LDS (a count, and the index of the last entry:
// integer atomics, so their order does not show), then every logit of the
// slice is adjusted in double and rounded once.  In place, a logit that nothing
// touches is neither read nor written.
__global__ void __launch_bounds__(kWG)
    k_logits_adjust(const float *x, int64_t n, const int64_t *__restrict__ window, int64_t last_n,
                    const double *__restrict__ pen, const int64_t *__restrict__ bias_ids,
                    const float *__restrict__ bias, const int64_t *__restrict__ bias_off,
                    int64_t n_bias, const uint32_t *__restrict__ mask, int64_t mask_ld,
                    float *out) {
#pragma clang fp contract(off)
  __shared__ uint32_t cnt[kSlice];
  __shared__ uint32_t ent[kSlice];  // 1 + the last entry of the token
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y, base = (int64_t)blockIdx.x * kSlice;
  const bool in_place = x == out;
  x += row * n;
  out += row * n;
  for (int i = tid; i < kSlice; i += kWG) cnt[i] = ent[i] = 0;
  __syncthreads();
  double rep = 1.0, pres = 0.0, freq = 0.0;
  if (window && pen) {
    rep = pen[row * 3];
    pres = pen[row * 3 + 1];
    freq = pen[row * 3 + 2];
    const int64_t *w = window + row * (1 + last_n);
    const int64_t seen = w[0] < last_n ? w[0] : last_n;
    for (int64_t j = tid; j < seen; j += kWG) {
      const int64_t t = w[1 + j] - base;
      if (t >= 0 && t < kSlice) atomicAdd(&cnt[t], 1u);
    }
  }
  if (n_bias) {
    int64_t a = bias_off ? bias_off[row] : 0, b = bias_off ? bias_off[row + 1] : n_bias;
    a = a > 0 ? a : 0;
    b = b < n_bias ? b : n_bias;
    for (int64_t j = a + tid; j < b; j += kWG) {
      const int64_t t = bias_ids[j] - base;
      if (t >= 0 && t < kSlice) atomicMax(&ent[t], (uint32_t)j + 1u);
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSlice / kWG; ++k) {
    const int e = k * kWG + tid;
    const int64_t i = base + e;
    if (i >= n) break;
    const bool off = mask && !((mask[row * mask_ld + (i >> 5)] >> (i & 31)) & 1u);
    if (off) {
      out[i] = -__builtin_inff();
      continue;
    }
    const uint32_t c = cnt[e], j = ent[e];
    if (!c && !j) {
      if (!in_place) out[i] = x[i];
      continue;
    }
    double y = (double)x[i];
    if (c) {
      if (rep != 0.0 && rep != 1.0) y = y > 0.0 ? y / rep : y * rep;
      y = y - (pres + freq * (double)c);
    }
    if (j) y = y + (double)bias[j - 1];
    out[i] = (float)y;
  }
}

}  // namespace

hipError_t launch_logits_adjust(const float *logits, int64_t rows, int64_t n,
                                const int64_t *window, int64_t last_n, const double *pen,
                                const int64_t *bias_ids, const float *bias,
                                const int64_t *bias_off, int64_t n_bias, const uint32_t *mask,
                                int64_t mask_ld, float *out, hipStream_t s) {
  const int64_t slices = (n + kSlice - 1) / kSlice;
  hipLaunchKernelGGL(k_logits_adjust, dim3((unsigned)slices, (unsigned)rows), dim3(kWG), 0, s,
                     logits, n, window, last_n, pen, bias_ids, bias, bias_off, n_bias, mask,
                     mask_ld, out);
  return hipGetLastError();
}

}  // namespace aq
