// Attention of a batch of sequences over a paged KV cache.
#include "kernels.h"
#include "paged.h"

namespace mdma {
namespace {

// A workgroup per (new token, query head): scores of 256 keys at a time, one
// a thread, an online softmax over the blocks, then each thread's dims of P V.
__global__ __launch_bounds__(256) void attn_paged_kernel(const float *__restrict__ q, PagedView kv, uint32_t n_new,
                                                         uint32_t q_heads, uint32_t kv_heads, uint32_t hd, float scale,
                                                         float *__restrict__ o) {
  __shared__ float qs[256], ps[256], red[4];
  __shared__ uint64_t rows[256];
  const uint32_t t = blockIdx.x, h = blockIdx.y, s = t / n_new, j = t % n_new, tid = threadIdx.x;
  const uint32_t kvh = h / (q_heads / kv_heads), len = kv.length(s);
  const uint32_t seen = len + j + 1 > n_new ? len + j + 1 - n_new : 0;  // keys 0 .. seen - 1
  const uint64_t at = ((uint64_t)t * q_heads + h) * hd;
  if (tid < hd) qs[tid] = q[at + tid];
  float m = -INFINITY, l = 0.f, acc = 0.f;
  bool any = false;
  for (uint32_t k0 = 0; k0 < seen; k0 += 256) {
    __syncthreads();
    const uint32_t key = k0 + tid;
    float sc = -INFINITY;
    uint64_t row = ~0ull;
    if (key < seen) {
      const uint32_t id = kv.page(s, key >> kv.page_shift);
      if (id != NO_PAGE) {
        row = kv.row(id, key) + (uint64_t)kvh * hd;
        float x = 0.f;
        for (uint32_t d = 0; d < hd; d++) x = fmaf(qs[d], h2f(kv.k[row + d]), x);
        sc = x * scale;
      }
    }
    rows[tid] = row;
    const float wm = wave_max_all(sc);
    if ((tid & 63) == 0) red[tid >> 6] = wm;
    any |= __syncthreads_or(row != ~0ull) != 0;
    const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float al = m == -INFINITY ? 0.f : expf(m - mn);
    ps[tid] = row == ~0ull ? 0.f : expf(sc - mn);
    __syncthreads();
    l *= al;
    acc *= al;
    m = mn;
    for (uint32_t i = 0; i < 256; i++) {
      if (rows[i] == ~0ull) continue;
      l += ps[i];
      if (tid < hd) acc = fmaf(ps[i], h2f(kv.v[rows[i] + tid]), acc);
    }
  }
  if (tid < hd) o[at + tid] = any ? acc / l : 0.f;
}

}  // namespace

void launch_attn_paged(mdma_ctx *ctx, const float *q, const PagedView &kv, uint32_t n_new, uint32_t q_heads,
                       uint32_t kv_heads, uint32_t hd, float *o) {
  attn_paged_kernel<<<dim3(kv.n_seqs * n_new, q_heads), 256, 0, ctx->stream>>>(q, kv, n_new, q_heads, kv_heads, hd,
                                                                              1.0f / sqrtf((float)hd), o);
  hip_check(hipGetLastError(), "attn_paged launch");
}

}  // namespace mdma
