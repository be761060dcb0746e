// Low-rank adapters of many requests beside a shared projection:
// y[t] = base[t] + scale_a B_a u[t], u[t] = A_a x[t], a = ids[t].
//
// Two launches: shrink leaves u (n_in split into parts, each a sum of its own),
// expand adds the parts up and writes y. What bounds them is memory: the
// adapters' values once per request batch (decode), x, base and y (prompts).
// Products run on v_mfma_f32_16x16x4_f32: x and u stay f32, F16 values are
// widened, so there is no scale to choose for x and one token's infinity or NaN stays in
// its column; at 16 and more tokens a value the f32 rate (64 operations a cycle and
// SIMD) is still ahead of memory up to rank 64.
//
// A wave works for 16 tokens of one adapter (columns of the MFMA). Up to
// GATHER tokens they are gathered from the whole batch, so requests in any order read each
// adapter once per 16 of its tokens; above, a wave takes 16 consecutive tokens and
// goes through the adapters among them one after the other (prompts come in runs).
#include "kernels.h"

namespace mdma {
namespace {

typedef float v4f_t __attribute__((ext_vector_type(4)));
typedef float v4f_u __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 v4h_t __attribute__((ext_vector_type(4)));
typedef _Float16 v8h_t __attribute__((ext_vector_type(8)));

constexpr uint32_t GATHER = 256;       // a thread a token
constexpr uint32_t NO_SLOT = ~0u, NO_TOKEN = ~0u;
constexpr uint32_t COLS = 256;         // outputs of an expand workgroup, 64 a wave and step

// The slot of token t's adapter, NO_SLOT where it has none.
__device__ __forceinline__ uint32_t slot_of(const LoraView &w, const uint32_t *ids, uint32_t t) {
  const uint32_t id = ids[t];
  return id < w.n_slots && w.info[id].rank ? id : NO_SLOT;
}

// Up to GATHER tokens: the tokens of the adapter of token `lead`, from its rank among
// them on (a multiple of 16, else false: another workgroup's), 16 at most, into tok.
__device__ __forceinline__ bool gather(const LoraView &w, const uint32_t *ids, uint32_t T, uint32_t lead,
                                       uint32_t *tok, uint32_t *slot) {
  __shared__ uint32_t all[GATHER];
  __shared__ uint64_t mask[GATHER / 64];
  const uint32_t t = threadIdx.x, wave = t >> 6;
  const uint32_t mine = t < T ? slot_of(w, ids, t) : NO_SLOT;
  all[t] = mine;
  if (t < 16) tok[t] = NO_TOKEN;
  __syncthreads();
  *slot = __builtin_amdgcn_readfirstlane(all[lead]);
  const bool same = t < T && mine == *slot;
  const uint64_t m = __ballot(same);
  if ((t & 63) == 0) mask[wave] = m;
  __syncthreads();
  uint32_t before = 0, lead_rank = 0;
#pragma unroll
  for (uint32_t v = 0; v < GATHER / 64; v++) {
    const uint64_t x = mask[v];
    if (v < wave) before += __popcll(x);
    if (v < lead / 64) lead_rank += __popcll(x);
    else if (v == lead / 64) lead_rank += __popcll(x & ((1ull << (lead & 63)) - 1));
  }
  if (lead_rank % 16) return false;
  const uint32_t rank = before + __popcll(m & ((1ull << (t & 63)) - 1));
  if (same && rank >= lead_rank && rank < lead_rank + 16) tok[rank - lead_rank] = t;
  __syncthreads();
  return true;
}

// Eight values of a row from column 8 c on, as f32.
template <class W>
struct Eight;
template <>
struct Eight<_Float16> {
  v8h_t v;
  __device__ __forceinline__ void load(const void *p, uint64_t at) {
    v = *reinterpret_cast<const v8h_t *>(static_cast<const _Float16 *>(p) + at);
  }
  __device__ __forceinline__ float operator[](int i) const { return (float)v[i]; }
};
template <>
struct Eight<float> {
  v4f_t v[2];
  __device__ __forceinline__ void load(const void *p, uint64_t at) {
    const v4f_t *q = reinterpret_cast<const v4f_t *>(static_cast<const float *>(p) + at);
    v[0] = q[0];
    v[1] = q[1];
  }
  __device__ __forceinline__ float operator[](int i) const { return v[i >> 2][i & 3]; }
};
// Four of them.
__device__ __forceinline__ v4f_t four(const _Float16 *p) {
  const v4h_t h = *reinterpret_cast<const v4h_t *>(p);
  return __builtin_convertvector(h, v4f_t);
}
__device__ __forceinline__ v4f_t four(const float *p) { return *reinterpret_cast<const v4f_t *>(p); }

// x's eight values from column k on; 0 past the row's end.
__device__ __forceinline__ void load_x(const float *row, uint32_t k, uint32_t n_in, v4f_t *x) {
  if (k + 8 <= n_in) {
    x[0] = *reinterpret_cast<const v4f_u *>(row + k);
    x[1] = *reinterpret_cast<const v4f_u *>(row + k + 4);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) x[e >> 2][e & 3] = k + e < n_in ? row[k + e] : 0.f;
  }
}

// The tokens' sums over 32-column steps s0, s0 + by, .. below s1, for ranks
// r0 + 16 i: D[i] holds ranks 4 lq + (0..3) of token l16.
template <class W, int RT>
__device__ __forceinline__ void shrink_steps(const LoraView &w, uint32_t slot, const float *xr, uint32_t r0, uint32_t s0,
                                             uint32_t s1, uint32_t by, v4f_t *D) {
  const uint32_t lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
  const uint64_t a0 = ((uint64_t)slot * w.rank_pad + r0 + l16) * w.in_pad + 8 * lq;
  Eight<W> a[RT], an[RT];
  v4f_t x[2], xn[2];
#pragma unroll
  for (int i = 0; i < RT; i++) D[i] = v4f_t{0.f, 0.f, 0.f, 0.f};
  if (s0 >= s1) return;
  auto load = [&](uint32_t s, Eight<W> *A, v4f_t *X) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < RT; i++) A[i].load(w.a, a0 + (uint64_t)16 * i * w.in_pad + 32 * s);
    load_x(xr, 32 * s + 8 * lq, w.n_in, X);
  };
  load(s0, an, xn);
  for (uint32_t s = s0; s < s1; s += by) {
#pragma unroll
    for (int i = 0; i < RT; i++) a[i] = an[i];
    x[0] = xn[0], x[1] = xn[1];
    if (s + by < s1) load(s + by, an, xn);
#pragma unroll
    for (int e = 0; e < 8; e++)
#pragma unroll
      for (int i = 0; i < RT; i++)
        D[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][e], x[e >> 2][e & 3], D[i], 0, 0, 0);
  }
}

// GATHERED: workgroup (lead token, part), its waves share the part's columns and add
// their sums up in LDS. Else workgroup (64 tokens, part), 16 tokens a wave.
template <class W, int RT, bool GATHERED>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraView w, const uint32_t *__restrict__ ids, uint32_t T,
                                                          const float *__restrict__ x, float *__restrict__ u,
                                                          uint32_t part_steps) {
  __shared__ uint32_t tok[16];
  __shared__ v4f_t sums[GATHERED ? 3 : 1][RT][64];
  const uint32_t lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t part = blockIdx.x, steps = w.in_pad / 32;
  const uint32_t s0 = part * part_steps, s1 = min(s0 + part_steps, steps);
  auto store = [&](uint32_t t, uint32_t r0, uint32_t rank, const v4f_t *D) __attribute__((always_inline)) {
    float *dst = u + ((uint64_t)part * T + t) * w.rank_pad + r0 + 4 * lq;
#pragma unroll
    for (int i = 0; i < RT; i++) {
      v4f_t v = D[i];
      if (r0 + 16 * i >= rank) break;
      // (0 past the rank, whatever x holds)
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = r0 + 16 * i + 4 * lq + e < rank ? v[e] : 0.f;
      *reinterpret_cast<v4f_t *>(dst + 16 * i) = v;
    }
  };
  v4f_t D[RT];
  if constexpr (GATHERED) {
    uint32_t slot;
    if (!gather(w, ids, T, blockIdx.y, tok, &slot) || slot == NO_SLOT) return;
    const uint32_t rank = w.info[slot].rank, t = tok[l16];
    const float *xr = x + (uint64_t)(t != NO_TOKEN ? t : tok[0]) * w.n_in;
    for (uint32_t r0 = 0; r0 < rank; r0 += 16 * RT) {  // (uniform)
      shrink_steps<W, RT>(w, slot, xr, r0, s0 + wave, s1, 4, D);
      __syncthreads();
      if (wave) {
#pragma unroll
        for (int i = 0; i < RT; i++) sums[wave - 1][i][lane] = D[i];
      }
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int i = 0; i < RT; i++) D[i] = (D[i] + sums[0][i][lane]) + (sums[1][i][lane] + sums[2][i][lane]);
        if (t != NO_TOKEN) store(t, r0, rank, D);
      }
    }
  } else {
    const uint32_t t = 64 * blockIdx.y + 16 * wave + l16;
    const uint32_t mine = t < T ? slot_of(w, ids, t) : NO_SLOT;
    const float *xr = x + (uint64_t)min(t, T - 1) * w.n_in;
    for (uint64_t todo = __ballot(mine != NO_SLOT) & 0xffff; todo;) {
      const uint32_t slot = __builtin_amdgcn_readlane((int)mine, __builtin_ctzll(todo));
      todo &= ~__ballot(mine == slot);
      const uint32_t rank = w.info[slot].rank;
      for (uint32_t r0 = 0; r0 < rank; r0 += 16 * RT) {
        shrink_steps<W, RT>(w, slot, xr, r0, s0, s1, 1, D);
        if (mine == slot) store(t, r0, rank, D);
      }
    }
  }
}

// The outputs n0 + 64 step (64 of them) of a wave's 16 tokens (rows of D; tr: the lane's
// four, NO_TOKEN for none), u's blocks of 16 ranks as operands U.
template <class W, int UB>
__device__ __forceinline__ void expand_cols(const LoraView &w, const W *b0, uint32_t stride, float scale, uint32_t blocks,
                                            const v4f_t *U, uint32_t n, const uint32_t *tr,
                                            const float *__restrict__ base, float *__restrict__ y) {
  // Lane l16 has the four outputs from n on, so it reads their rows of B and writes 16 bytes.
  v4f_t D[4], old[4];
  const uint32_t lq = (threadIdx.x & 63) >> 4;
  const bool whole = n + 4 <= w.n_out;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    old[i] = v4f_t{0.f, 0.f, 0.f, 0.f};
    if (tr[i] != NO_TOKEN) {
      const float *p = base + (uint64_t)tr[i] * w.n_out + n;
      if (whole) old[i] = *reinterpret_cast<const v4f_u *>(p);
      else
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (n + j < w.n_out) old[i][j] = p[j];
    }
  }
  v4f_t B[4][UB];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const W *row = b0 + (uint64_t)min(n + j, w.n_out - 1) * stride + 4 * lq;
#pragma unroll
    for (int b = 0; b < UB; b++)
      if (b < (int)blocks) B[j][b] = four(row + 16 * b);
    D[j] = v4f_t{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int b = 0; b < UB; b++)
    if (b < (int)blocks) {  // (uniform)
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int j = 0; j < 4; j++) D[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(U[b][e], B[j][b][e], D[j], 0, 0, 0);
    }
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (tr[i] != NO_TOKEN) {
      v4f_t v;
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = fmaf(D[j][i], scale, old[i][j]);
      float *p = y + (uint64_t)tr[i] * w.n_out + n;
      if (whole) *reinterpret_cast<v4f_u *>(p) = v;
      else
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (n + j < w.n_out) p[j] = v[j];
    }
}
// y = base for the lane's tokens, outputs n .. n + 3.
__device__ __forceinline__ void copy_cols(const LoraView &w, uint32_t n, const uint32_t *tr, const float *base, float *y) {
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (tr[i] != NO_TOKEN)
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (n + j < w.n_out) y[(uint64_t)tr[i] * w.n_out + n + j] = base[(uint64_t)tr[i] * w.n_out + n + j];
}

// Workgroup (COLS outputs, tokens): GATHERED, 16 tokens of one adapter, 64 outputs a
// wave; else 64 tokens, 16 a wave, each all the outputs. UB: blocks of 16 ranks.
template <class W, int UB, bool GATHERED>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraView w, const uint32_t *__restrict__ ids, uint32_t T,
                                                          const float *__restrict__ u, uint32_t parts,
                                                          const float *__restrict__ base, float *__restrict__ y) {
  __shared__ uint32_t tok[16];
  const uint32_t lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t n0 = COLS * blockIdx.x + 4 * l16;
  // u of the lane's token (l16), ranks 16 b + 4 lq + (0..3): its parts in order.
  auto load_u = [&](uint32_t t, uint32_t blocks, v4f_t *U) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < UB; b++) {
      U[b] = v4f_t{0.f, 0.f, 0.f, 0.f};
      if (t == NO_TOKEN || b >= (int)blocks) continue;
      const float *p = u + (uint64_t)t * w.rank_pad + 16 * b + 4 * lq;
      for (uint32_t c = 0; c < parts; c++) U[b] += *reinterpret_cast<const v4f_t *>(p + (uint64_t)c * T * w.rank_pad);
    }
  };
  v4f_t U[UB];
  uint32_t tr[4];
  if constexpr (GATHERED) {
    uint32_t slot;
    if (!gather(w, ids, T, blockIdx.y, tok, &slot)) return;
#pragma unroll
    for (int i = 0; i < 4; i++) tr[i] = tok[4 * lq + i];
    const uint32_t n = n0 + 64 * wave;
    if (n - 4 * l16 >= w.n_out) return;
    if (slot == NO_SLOT) {
      if (base != y) copy_cols(w, n, tr, base, y);
      return;
    }
    const LoraSlot in = w.info[slot];
    load_u(tok[l16], in.stride / 16, U);
    expand_cols<W, UB>(w, static_cast<const W *>(w.b) + (uint64_t)slot * w.n_out * w.rank_pad, in.stride, in.scale,
                       in.stride / 16, U, n, tr, base, y);
  } else {
    const uint32_t t0 = 64 * blockIdx.y + 16 * wave, t = t0 + l16;
    const uint32_t mine = t < T ? slot_of(w, ids, t) : NO_SLOT;
    // (the rows 4 lq + i of this lane: their slots from the lanes that looked them up)
    uint32_t of[4];
#pragma unroll
    for (int i = 0; i < 4; i++) of[i] = __shfl((int)mine, 4 * lq + i, 64);
    for (uint64_t todo = __ballot(t < T) & 0xffff; todo;) {
      const uint32_t slot = __builtin_amdgcn_readlane((int)mine, __builtin_ctzll(todo));
      todo &= ~__ballot(mine == slot);
#pragma unroll
      for (int i = 0; i < 4; i++) tr[i] = of[i] == slot && t0 + 4 * lq + i < T ? t0 + 4 * lq + i : NO_TOKEN;
      if (slot == NO_SLOT) {
        if (base != y)
          for (uint32_t k = 0; k < COLS / 64; k++) copy_cols(w, n0 + 64 * k, tr, base, y);
        continue;
      }
      const LoraSlot in = w.info[slot];
      load_u(mine == slot ? t : NO_TOKEN, in.stride / 16, U);
      for (uint32_t k = 0; k < COLS / 64 && n0 - 4 * l16 + 64 * k < w.n_out; k++)
        expand_cols<W, UB>(w, static_cast<const W *>(w.b) + (uint64_t)slot * w.n_out * w.rank_pad, in.stride, in.scale,
                           in.stride / 16, U, n0 + 64 * k, tr, base, y);
    }
  }
}

struct Plan {
  uint32_t steps, parts;  // 32-column steps of a part of n_in, and parts
};
// Gathered: a part of 256 columns, two steps a wave, at most 16 parts (the
// expand adds them up). Consecutive: as many parts as keep about 4 waves a SIMD busy, at most 8.
Plan plan_of(const LoraView &w, uint64_t T) {
  const uint32_t steps = w.in_pad / 32;
  const uint64_t most = T <= GATHER ? 16 : std::min<uint64_t>(8, std::max<uint64_t>(1, 4096 * 16 / T));
  const uint32_t parts = (uint32_t)std::min<uint64_t>(most, (steps + 7) / 8);
  const uint32_t per = (steps + parts - 1) / parts;
  return Plan{per, (steps + per - 1) / per};
}

template <class W, int UB>
void launch(mdma_ctx *ctx, const LoraView &w, const uint32_t *ids, uint32_t T, const float *x, const float *base,
            float *y, float *u) {
  constexpr int RT = UB < 4 ? UB : 4;
  const Plan p = plan_of(w, T);
  const uint32_t cols = (w.n_out + COLS - 1) / COLS;
  if (T <= GATHER) {
    lora_shrink_kernel<W, RT, true><<<dim3(p.parts, T), 256, 0, ctx->stream>>>(w, ids, T, x, u, p.steps);
    lora_expand_kernel<W, UB, true><<<dim3(cols, T), 256, 0, ctx->stream>>>(w, ids, T, u, p.parts, base, y);
  } else {
    const uint32_t tiles = (T + 63) / 64;
    lora_shrink_kernel<W, RT, false><<<dim3(p.parts, tiles), 256, 0, ctx->stream>>>(w, ids, T, x, u, p.steps);
    lora_expand_kernel<W, UB, false><<<dim3(cols, tiles), 256, 0, ctx->stream>>>(w, ids, T, u, p.parts, base, y);
  }
}
template <class W>
void launch_of(mdma_ctx *ctx, const LoraView &w, const uint32_t *ids, uint32_t T, const float *x, const float *base,
               float *y, float *u) {
  if (w.rank_pad <= 16) launch<W, 1>(ctx, w, ids, T, x, base, y, u);
  else if (w.rank_pad <= 32) launch<W, 2>(ctx, w, ids, T, x, base, y, u);
  else if (w.rank_pad <= 64) launch<W, 4>(ctx, w, ids, T, x, base, y, u);
  else launch<W, 16>(ctx, w, ids, T, x, base, y, u);
}

}  // namespace

uint64_t lora_scratch(const LoraView &w, uint64_t T) { return T * w.rank_pad * 4 * plan_of(w, T).parts; }

void launch_lora(mdma_ctx *ctx, const LoraView &w, const uint32_t *ids, uint32_t T, const float *x, const float *base,
                 float *y, float *u) {
  if (w.dtype == DT_F16) launch_of<_Float16>(ctx, w, ids, T, x, base, y, u);
  else launch_of<float>(ctx, w, ids, T, x, base, y, u);
  hip_check(hipGetLastError(), "lora_add launch");
}

}  // namespace mdma
