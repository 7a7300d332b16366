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
// One workgroup a query row, 256 positions at a time.
template <int HD, typename T>
__global__ void __launch_bounds__(256)
    k_paged_attn(const float *__restrict__ q, int n_head, PagedTable tab, PagedTable pre,
                 aq_paged c, float *__restrict__ out) {
  __shared__ float qs[HD], w[256], red[4];
  __shared__ int64_t blocks[8];
  const int t = threadIdx.x, h = blockIdx.x % n_head, G = n_head / c.n_kv;
  const int64_t n = blockIdx.x / n_head;
  const int64_t pos = tab.pos[n], seq = tab.seq ? tab.seq[n] : n;
  const int64_t head = (int64_t)(h / G) * (c.page_size / kBlk);
  out += (n * n_head + h) * HD;
  if (t < HD) qs[t] = q[(n * n_head + h) * HD + t] * (1.44269504088896341f / sqrtf((float)HD));
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int part = 0; part < 2; ++part) {
    const int64_t room = part ? tab.width * c.page_size : pre.start;
    int64_t len = part ? pos + 1 - tab.start : pos + 1;
    len = len < room ? len : room;
    for (int64_t p0 = 0; p0 < len; p0 += 256) {
      __syncthreads();
      if (t < 8) blocks[t] = part ? block_of(c, tab, seq, p0 + 32 * t) : block_of(c, pre, 0, p0 + 32 * t);
      __syncthreads();
      float z = -INFINITY;
      const int64_t blk = blocks[t >> 5];
      if (p0 + t < len && blk >= 0) {
        const T *kp = static_cast<const T *>(c.k) + (blk + head) * (kBlk * HD);
        z = 0.f;
        for (int d = 0; d < HD; ++d) z = fmaf(qs[d], (float)kp[k_place<HD>(t & 31, d)], z);
      }
      float mx = z;
      for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
      if ((t & 63) == 0) red[t >> 6] = mx;
      __syncthreads();
      mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
      const float mn = fmaxf(m, mx);
      w[t] = z == -INFINITY ? 0.f : exp2f(z - mn);
      const float f = m == -INFINITY ? 0.f : exp2f(m - mn);
      m = mn;
      __syncthreads();
      if (t < HD) {
        l *= f;
        o *= f;
        for (int i = 0; i < 256; ++i) {
          if (p0 + i >= len || blocks[i >> 5] < 0) continue;
          const T *vp = static_cast<const T *>(c.v) + (blocks[i >> 5] + head) * (kBlk * HD);
          l += w[i];
          o = fmaf(w[i], (float)vp[v_place(i & 31, t)], o);
        }
      }
    }
  }
  if (t < HD) out[t] = m == -INFINITY && l == 0.f ? 0.f : o / l;
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

hipError_t launch_attention_paged(const float *q, int64_t N, int n_head, const PagedTable &tab,
                                  const PagedTable &pre, const aq_paged &c, float *out,
                                  hipStream_t s) {
  by_shape(c, [&](auto hd, auto t) {
    hipLaunchKernelGGL((k_paged_attn<decltype(hd)::value, decltype(t)>),
                       dim3((unsigned)(N * n_head)), dim3(256), 0, s, q, n_head, tab, pre, c, out);
  });
  return hipGetLastError();
}

}  // namespace aq
