// Low-rank adapters of many requests beside a shared projection:
// y[t] = base[t] + scale_a B_a (A_a x[t]), a = ids[t].
#include "kernels.h"

namespace mdma {
namespace {

template <class W>
__device__ __forceinline__ float w2f(W w) { return (float)w; }

// u[t][r] = A_a[r] . x[t], a wave per (token, r).
template <class W>
__global__ __launch_bounds__(64) void lora_shrink_kernel(LoraView w, const uint32_t *__restrict__ ids,
                                                         const float *__restrict__ x, float *__restrict__ u) {
  const uint32_t t = blockIdx.x, r = blockIdx.y, id = ids[t];
  if (id >= w.n_slots || r >= w.info[id].rank) return;
  const W *a = static_cast<const W *>(w.a) + ((uint64_t)id * w.rank_pad + r) * w.in_pad;
  float s = 0.f;
  for (uint32_t i = threadIdx.x; i < w.n_in; i += 64) s = fmaf(w2f(a[i]), x[(uint64_t)t * w.n_in + i], s);
  s = wave_sum_all(s);
  if (threadIdx.x == 0) u[(uint64_t)t * w.rank_pad + r] = s;
}
template <class W>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraView w, const uint32_t *__restrict__ ids,
                                                          const float *__restrict__ u, const float *__restrict__ base,
                                                          float *__restrict__ y) {
  const uint32_t t = blockIdx.x, n = blockIdx.y * 256 + threadIdx.x, id = ids[t];
  if (n >= w.n_out) return;
  float s = 0.f, scale = 0.f;
  if (id < w.n_slots && w.info[id].rank) {
    const LoraSlot in = w.info[id];
    const W *b = static_cast<const W *>(w.b) + ((uint64_t)id * w.n_out) * w.rank_pad + (uint64_t)n * in.stride;
    for (uint32_t r = 0; r < in.rank; r++) s = fmaf(w2f(b[r]), u[(uint64_t)t * w.rank_pad + r], s);
    scale = in.scale;
    y[(uint64_t)t * w.n_out + n] = fmaf(s, scale, base[(uint64_t)t * w.n_out + n]);
  } else {
    y[(uint64_t)t * w.n_out + n] = base[(uint64_t)t * w.n_out + n];
  }
}

}  // namespace

uint64_t lora_scratch(const LoraView &w, uint64_t T) { return T * w.rank_pad * 4; }

void launch_lora(mdma_ctx *ctx, const LoraView &w, const uint32_t *ids, uint32_t T, const float *x, const float *base,
                 float *y, float *u) {
  const dim3 g1(T, w.rank_pad), g2(T, (w.n_out + 255) / 256);
  if (w.dtype == DT_F16) {
    lora_shrink_kernel<_Float16><<<g1, 64, 0, ctx->stream>>>(w, ids, x, u);
    lora_expand_kernel<_Float16><<<g2, 256, 0, ctx->stream>>>(w, ids, u, base, y);
  } else {
    lora_shrink_kernel<float><<<g1, 64, 0, ctx->stream>>>(w, ids, x, u);
    lora_expand_kernel<float><<<g2, 256, 0, ctx->stream>>>(w, ids, u, base, y);
  }
  hip_check(hipGetLastError(), "lora_add launch");
}

}  // namespace mdma
