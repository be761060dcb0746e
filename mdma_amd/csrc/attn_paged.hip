// Attention of a batch of sequences over a paged KV cache, a prefix that all of
// them share read once.
//
// With p = the position of a query, o = sum_{x <= p} w_x v_x / sum w_x, w_x =
// exp(q . k_x / sqrt(hd)). A sum over keys splits: keys [a, b) leave m (a
// reference point near the largest score), l = sum 2^(s - m) and O = sum
// 2^(s - m) v, s the score times log2 e, and parts join with weights
// 2^(m_i - M). So the shared prefix is one job for the query rows of the
// whole batch, each sequence's own keys (the tail) are a job for its rows,
// both are cut into chunks of keys, and a second kernel joins a row's parts.
//
// Arithmetic: K and V are f16 in the cache, and S^T = K Q^T and O^T = V^T P^T
// run on v_mfma_f32_16x16x32_f16 with f32 sums. Q and P are f32; each goes in
// as two f16 parts, so nothing is rounded to less than 22 bits:
//  - a row of q times the power of two that brings its largest value into
//    [2^14, 2^15): hi has 11 bits, lo the 11 bits below, together 2^-24
//    of the row's largest value at worst, as f32 products of it would be;
//  - p times 2^10, at most 2^15 (m may lag the maximum by 5 bits): hi and lo keep 2^-22 of
//    p, and 2^-35 of the row's largest p.
// m is a whole number, so 2^(m - m') is a power of two: rescaling l and O
// and joining chunks round nothing.
#include "kernels.h"
#include "paged.h"

namespace mdma {
namespace {

typedef _Float16 v8h_t __attribute__((ext_vector_type(8)));
typedef _Float16 v4h_t __attribute__((ext_vector_type(4)));
typedef _Float16 v2h_t __attribute__((ext_vector_type(2)));
typedef float v4f_t __attribute__((ext_vector_type(4)));
typedef float v2f_t __attribute__((ext_vector_type(2)));
typedef short v4s_t __attribute__((ext_vector_type(4)));

constexpr float P_BITS = 10.f, M_LAG = 5.f;
constexpr uint32_t MAX_PARTS = 64;  // parts of a row: a lane each in the joining kernel

struct Args {
  const float *q;
  PagedView kv;
  float *o, *part;  // part: O [slot][row][hd], then (m, l) [slot][row]
  uint32_t n_new, heads, group, hd, rows;  // rows: all query rows, tokens * heads
  float scale2;                            // log2 e / sqrt(hd)
  uint32_t start;                          // the tails' first position: the shared prefix's length, 0 without
  uint32_t n_p, cp, rt_p, blocks_p;        // prefix: chunks, keys in one, row tiles, blocks
  uint32_t n_t, rt_t;                      // tails: chunks a sequence at most, row tiles
  bool wide_p, wide_t;                     // which kind of job (below) they are
};

// Keys in a chunk of a tail of n positions cut into at most n_t chunks.
__device__ __forceinline__ uint32_t tail_chunk(uint32_t n, uint32_t n_t) {
  return n_t == 1 ? max(n, 1u) : max(((n + n_t - 1) / n_t + 127) & ~127u, 256u);
}
// Keys token j of a sequence of len positions sees, the first ones.
__device__ __forceinline__ uint32_t seen_by(uint32_t len, uint32_t n_new, uint32_t j) {
  return len + j + 1 > n_new ? len + j + 1 - n_new : 0;
}

// A block's unit (what it reads) and row tile (for whom): blocks go to the
// 8 XCDs in turn, and the row tiles of one unit to the same one, whose L2 then
// holds the unit's keys and values once.
__device__ __forceinline__ void unit_of(uint32_t b, uint32_t tiles, uint32_t *unit, uint32_t *tile) {
  *unit = b / (8 * tiles) * 8 + b % 8;
  *tile = b / 8 % tiles;
}

// LDS slot of 16-byte chunk ch of a key's row of KC chunks: keys read together
// (16 rows of one chunk; 4 rows of a 32-byte column by a transposing read) fall on
// different banks.
template <int KC>
__device__ __forceinline__ uint32_t slot_of(uint32_t key, uint32_t ch) {
  if constexpr (KC == 8) return ch ^ ((key >> 1) & 7);
  else if constexpr (KC == 12) {
    const uint32_t s = ch + (key & 15) / 2;
    return s >= KC ? s - KC : s;
  } else return ch ^ (key & 15);
}

// A row in f32, key by key, over the keys [k0, k1) that exist: for rows that
// came out not finite (an infinity or a NaN, perhaps at a key that the row
// does not see: 0 times it in the MFMA is NaN), or with no weight at all. The
// whole wave; dim 64 i + lane in acc[i].
template <int NA>
__device__ __forceinline__ void row_by_keys(const Args &a, uint32_t token, uint32_t head, uint32_t k0, uint32_t k1,
                                         float *acc, float *m_out, float *l_out) {
  const uint32_t lane = threadIdx.x & 63, s = token / a.n_new, hd = a.hd;
  const float *qr = a.q + ((uint64_t)token * a.heads + head) * hd;
  const uint64_t col = (uint64_t)(head / a.group) * hd;
  auto score = [&](uint32_t key, bool *there) {
    const uint32_t id = key < k1 ? a.kv.page(s, key >> a.kv.page_shift) : NO_PAGE;
    *there = id != NO_PAGE;
    if (!*there) return -INFINITY;
    const uint16_t *kr = a.kv.k + a.kv.row(id, key) + col;
    float x = 0.f;
    for (uint32_t d = 0; d < hd; d++) x = fmaf(qr[d], h2f(kr[d]), x);
    return x;
  };
  float rm = -INFINITY, l = 0.f;
  bool any = false, there;
  for (uint32_t k = k0; k < k1; k += 64) {
    rm = fmaxf(rm, score(k + lane, &there));
    any |= __any(there) != 0;
  }
  rm = wave_max_all(rm);
  float m = rm * a.scale2;
  if (m == -INFINITY && any) m = -3.0e38f;  // every weight is 0: not a row without keys
#pragma unroll
  for (int i = 0; i < NA; i++) acc[i] = 0.f;
  for (uint32_t k = k0; k < k1; k += 64) {
    const float x = score(k + lane, &there);
    const float p = there ? __builtin_amdgcn_exp2f(fmaf(x, a.scale2, P_BITS - m)) : 0.f;
    l += p;
    for (uint64_t todo = __ballot(there); todo; todo &= todo - 1) {
      const int i = __builtin_ctzll(todo);
      const float pi = __shfl(p, i, 64);
      const uint32_t key = k + i;
      const uint16_t *vr = a.kv.v + a.kv.row(a.kv.page(s, key >> a.kv.page_shift), key) + col;
#pragma unroll
      for (int n = 0; n < NA; n++)
        if (64 * n + lane < hd) acc[n] = fmaf(pi, h2f(vr[64 * n + lane]), acc[n]);
    }
  }
  *m_out = any ? m : -INFINITY;
  *l_out = wave_sum_all(l);
}

// Scores of 32 keys (K0, K1: 16 keys' operands for dims 32 j) for M row
// blocks, q's low parts before the high ones; and their values' step for dims 16 n.
template <int M, int NC>
__device__ __forceinline__ void scores_step(int j, v8h_t K0, v8h_t K1, const v8h_t (&qh)[M][NC], const v8h_t (&ql)[M][NC],
                                            v4f_t (&S)[M][2]) {
  const v4f_t zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < M; i++) {
    S[i][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(K0, ql[i][j], j ? S[i][0] : zero, 0, 0, 0);
    S[i][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(K1, ql[i][j], j ? S[i][1] : zero, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < M; i++) {
    S[i][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(K0, qh[i][j], S[i][0], 0, 0, 0);
    S[i][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(K1, qh[i][j], S[i][1], 0, 0, 0);
  }
}
template <int M, int ND>
__device__ __forceinline__ void values_step(int n, v8h_t V, const v8h_t (&Ph)[M], const v8h_t (&Pl)[M],
                                            v4f_t (&O)[M][ND]) {
#pragma unroll
  for (int i = 0; i < M; i++) O[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(V, Pl[i], O[i][n], 0, 0, 0);
#pragma unroll
  for (int i = 0; i < M; i++) O[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(V, Ph[i], O[i][n], 0, 0, 0);
}

// Jobs come in two kinds. Narrow: up to 16 MA query rows; the workgroup's four waves take
// 32-key tiles in turn, each for all the rows, K straight from memory as MFMA operands, V
// through 32 keys of LDS of the wave's own (ds_read_b64_tr_b16 gives
// its columns), no barrier until the four join at the end. Wide: 64 MB rows,
// 16 MB a wave; the waves share 64-key tiles of K and V in two LDS buffers,
// one barrier a tile. NC: head_dim in 32s, rounded up; the dims past head_dim
// read some other dim of the same key with q 0 there.
template <int NC, int MA, int MB>
__global__ __launch_bounds__(256, NC <= 4 ? 2 : 1) void attn_paged_kernel(Args a) {
  constexpr int KC = 4 * NC, ND = 2 * NC, NA = (NC + 1) / 2;
  constexpr int MX = MA > MB ? MA : MB;
  __shared__ __attribute__((aligned(16))) char lds[16 * 1024 * NC];
  __shared__ float2 ml[4][16 * MX];
  __shared__ uint32_t flags[4];
  const uint32_t tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lq = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t kv_heads = a.heads / a.group;

  // ---- which job ----
  const bool is_p = blockIdx.x < a.blocks_p, wide = is_p ? a.wide_p : a.wide_t;
  uint32_t unit, tile, chunk, kvh, t0, n_rows, k0, k1, seq = 0;
  if (is_p) {
    unit_of(blockIdx.x, a.rt_p, &unit, &tile);
    if (unit >= a.n_p * kv_heads) return;
    kvh = unit % kv_heads;
    chunk = unit / kv_heads;
    t0 = 0;
    n_rows = a.kv.n_seqs * a.n_new * a.group;
    k0 = chunk * a.cp;
    k1 = min(k0 + a.cp, a.start);
  } else {
    unit_of(blockIdx.x - a.blocks_p, a.rt_t, &unit, &tile);
    if (unit >= a.n_t * kv_heads * a.kv.n_seqs) return;
    kvh = unit % kv_heads;
    chunk = unit / kv_heads % a.n_t;
    seq = unit / (kv_heads * a.n_t);
    t0 = seq * a.n_new;
    n_rows = a.n_new * a.group;
    const uint32_t len = a.kv.length(seq), n = len > a.start ? len - a.start : 0, ct = tail_chunk(n, a.n_t);
    // (chunk * ct below n < 2^31 or cut off here)
    const uint32_t off = (uint64_t)chunk * ct < n ? chunk * ct : n;
    k0 = a.start + off;
    k1 = a.start + min(n, off + ct);
    if (a.n_t > 1 && off == n) return;  // (the join knows)
  }
  const uint32_t slot = is_p ? chunk : a.n_p + chunk;
  const bool direct = a.part == nullptr;

  // ---- this lane's query rows: column l16 of every MFMA ----
  struct Row {
    uint32_t token, head, seen;
    bool there;
  };
  auto row_of = [&](uint32_t r) __attribute__((always_inline)) {
    Row x;
    x.there = r < n_rows;
    const uint32_t c = min(r, n_rows - 1);
    x.token = t0 + c / a.group;
    x.head = kvh * a.group + c % a.group;
    const uint32_t s = x.token / a.n_new;
    x.seen = seen_by(a.kv.length(s), a.n_new, x.token % a.n_new);  // (of the last row past the end)
    return x;
  };
  auto load_q = [&](const Row &x, v8h_t *hi, v8h_t *lo, float *c) __attribute__((always_inline)) {
    const float *qr = a.q + ((uint64_t)x.token * a.heads + x.head) * a.hd;
    v4f_t v[2 * NC];
    float big = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * NC; i++) {
      const uint32_t d = 32 * (i >> 1) + 8 * lq + 4 * (i & 1);
      v[i] = d < a.hd ? *reinterpret_cast<const v4f_t *>(qr + d) : v4f_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; e++) big = fmaxf(big, fabsf(v[i][e]));
    }
    // 2^(14 - exponent), at most 2^126 (a NaN is not seen here: it stays one below)
    const int up_exp = min(268 - (int)(__builtin_bit_cast(uint32_t, quarter_max(big)) >> 23), 253);
    const float up = __builtin_bit_cast(float, (uint32_t)up_exp << 23);
    *c = __builtin_bit_cast(float, (uint32_t)(254 - up_exp) << 23) * a.scale2;
#pragma unroll
    for (int i = 0; i < 2 * NC; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float y = v[i][e] * up;
        const _Float16 h = (_Float16)y;
        hi[i >> 1][4 * (i & 1) + e] = h;
        lo[i >> 1][4 * (i & 1) + e] = (_Float16)(y - (float)h);
      }
  };

  // ---- page ids: lane b holds that of the 16-key block id0 + b of the job ----
  uint32_t idv = 0, id0 = 1u << 31;  // (no group yet: blocks are below 2^27)
  bool holes = false;  // a block met so far has no page
  auto block_id = [&](uint32_t b) __attribute__((always_inline)) {  // (uniform)
    if (b - id0 >= 64) {
      id0 = b & ~63u;
      const uint32_t pos = k0 + 16 * (id0 + lane);
      idv = pos < k1 ? a.kv.page(seq, pos >> a.kv.page_shift) : NO_PAGE;
      holes |= __any(pos < k1 && idv == NO_PAGE) != 0;
    }
    return (uint32_t)__builtin_amdgcn_readlane((int)idv, (int)(b - id0));
  };
  const uint32_t row_bytes = a.kv.width * 2, last_ch = a.hd / 8 - 1;
  const char *Kh = reinterpret_cast<const char *>(a.kv.k) + (uint64_t)kvh * a.hd * 2;
  const char *Vh = reinterpret_cast<const char *>(a.kv.v) + (uint64_t)kvh * a.hd * 2;
  const uint32_t page_mask = (1u << a.kv.page_shift) - 1;
  // Byte offset of block b (its first key at position pos) in a pool; false
  // where it has no page (page 0 is read, and masked).
  auto block_at = [&](uint32_t pos, uint64_t *at) __attribute__((always_inline)) {
    const uint32_t id = block_id((pos - k0) >> 4);
    const bool ok = id != NO_PAGE;
    *at = (((uint64_t)(ok ? id : 0) << a.kv.page_shift) + (pos & page_mask)) * row_bytes;
    return ok;
  };

  // ---- the softmax of 32 keys' scores; the probabilities as operands ----
  // S[kb][r] is key 16 kb + 4 lq + r of the 32 keys at pos.
  auto weights = [&](v4f_t (&S)[2], float c, uint32_t seen, bool mask, bool ok0, bool ok1, uint32_t pos, float &m,
                     float &l, v4f_t *O, v8h_t &Ph, v8h_t &Pl) __attribute__((always_inline)) {
    if (mask) {  // (uniform)
#pragma unroll
      for (int kb = 0; kb < 2; kb++)
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (pos + 16 * kb + 4 * lq + r >= seen || !(kb ? ok1 : ok0)) S[kb][r] = -INFINITY;
    }
    float mx = fmaxf(fmaxf(fmaxf(S[0][0], S[0][1]), fmaxf(S[0][2], S[0][3])),
                     fmaxf(fmaxf(S[1][0], S[1][1]), fmaxf(S[1][2], S[1][3])));
    mx = quarter_max(mx) * c;
    if (__any(mx > m + M_LAG)) {  // (also the first visible key: m = -inf)
      const float mn = mx > m + M_LAG ? ceilf(mx) : m;
      const float al = mn == m ? 1.f : m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
      l *= al;
#pragma unroll
      for (int n = 0; n < ND; n++) O[n] *= al;
      m = mn;
    }
    const float t = m == -INFINITY ? 0.f : P_BITS - m;
    float ps[4];
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(S[kb][r], c, t));  // (0 for masked keys)
        const float p1 = __builtin_amdgcn_exp2f(fmaf(S[kb][r + 1], c, t));
        ps[2 * kb + r / 2] = p0 + p1;
        const v2h_t h = __builtin_convertvector((v2f_t{p0, p1}), v2h_t);
        const v2h_t w = __builtin_convertvector((v2f_t{p0 - (float)h[0], p1 - (float)h[1]}), v2h_t);
        Ph[4 * kb + r] = h[0], Ph[4 * kb + r + 1] = h[1];
        Pl[4 * kb + r] = w[0], Pl[4 * kb + r + 1] = w[1];
      }
    l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
  };
  // V's columns of 32 keys (rows of KC chunks in LDS from `v`) for dims 16 n.
  auto v_columns = [&](const char *v, int n) __attribute__((always_inline)) {
    const uint32_t key = 4 * lq + (l16 >> 2), ch = 2 * n + ((l16 & 3) >> 1);
    const uint32_t off = (key * KC + slot_of<KC>(key, ch)) * 16 + 8 * (l16 & 1);
    auto rd = [&](uint32_t at) {
      return __builtin_bit_cast(v4h_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                           (__attribute__((address_space(3))) v4s_t *)(v + at)));
    };
    const v4h_t x = rd(off), y = rd(off + 16 * KC * 16);  // (slot_of has period 16 in the key)
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  float *part_o = a.part;
  float2 *part_ml = reinterpret_cast<float2 *>(a.part + (uint64_t)(a.n_p + a.n_t) * a.rows * a.hd);
  auto out_row = [&](const Row &x) {
    const uint64_t row = (uint64_t)x.token * a.heads + x.head;
    return direct ? a.o + row * a.hd : part_o + ((uint64_t)slot * a.rows + row) * a.hd;
  };
  auto put_ml = [&](const Row &x, float m, float l) {
    if (!direct) part_ml[(uint64_t)slot * a.rows + (uint64_t)x.token * a.heads + x.head] = make_float2(m, l);
  };
  // What a row's stored values are divided by: 0 keys give zeros.
  auto over = [&](float m, float l) { return !direct || m == -INFINITY ? 1.f : l; };
  auto slow_row = [&](const Row &x) {  // (uniform row)
    float acc[NA], m, l;
    row_by_keys<NA>(a, x.token, x.head, k0, min(k1, x.seen), acc, &m, &l);
    float *dst = out_row(x);
#pragma unroll
    for (int i = 0; i < NA; i++)
      if (64 * i + lane < a.hd) dst[64 * i + lane] = acc[i] / over(m, l);
    if (lane == 0) put_ml(x, m, l);
  };

  if (!wide) {
    Row row[MA];
    v8h_t qh[MA][NC], ql[MA][NC];
    float c[MA], m[MA], l[MA];
    v4f_t O[MA][ND];
    uint32_t seen_max = 0, seen_min = ~0u;
#pragma unroll
    for (int i = 0; i < MA; i++) {
      row[i] = row_of(16 * MA * tile + 16 * i + l16);
      load_q(row[i], qh[i], ql[i], &c[i]);
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int n = 0; n < ND; n++) O[i][n] = v4f_t{0.f, 0.f, 0.f, 0.f};
      seen_max = max(seen_max, row[i].seen);
      seen_min = min(seen_min, row[i].seen);
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      seen_max = max(seen_max, (uint32_t)__shfl_xor((int)seen_max, d, 64));
      seen_min = min(seen_min, (uint32_t)__shfl_xor((int)seen_min, d, 64));
    }
    seen_max = __builtin_amdgcn_readfirstlane(seen_max);
    seen_min = __builtin_amdgcn_readfirstlane(seen_min);
    const uint32_t end = min(k1, seen_max);  // (k0 >= end: nothing to read)
    char *vs = lds + wave * (32 * KC * 16);
    u32x4 kr[2][NC], vr[2][NC];
    bool ok[2] = {true, true};
    auto gload = [&](uint32_t pos) __attribute__((always_inline)) {
      const uint32_t last = (end - 1 - k0) & ~15u;
#pragma unroll
      for (int kb = 0; kb < 2; kb++) {
        const uint32_t blk = k0 + min(pos - k0 + 16 * kb, last);  // (past the end: the last block again, masked)
        uint64_t at;
        ok[kb] = block_at(blk, &at);
        const uint32_t most = end - 1 - blk;  // rows past the end: the last one again
        const char *K = Kh + at + min(l16, most) * row_bytes, *V = Vh + at + min(lane >> 2, most) * row_bytes;
#pragma unroll
        for (int i = 0; i < NC; i++) {
          kr[kb][i] = *reinterpret_cast<const u32x4 *>(K + 16 * min(4 * i + lq, last_ch));
          vr[kb][i] = *reinterpret_cast<const u32x4 *>(V + 16 * min(4 * i + (lane & 3), last_ch));
        }
      }
    };
    uint32_t pos = k0 + 32 * wave;
    if (pos < end) gload(pos);
    for (; pos < end; pos += 128) {
#pragma unroll
      for (int kb = 0; kb < 2; kb++)
#pragma unroll
        for (int i = 0; i < NC; i++) {
          const uint32_t key = lane >> 2;
          *reinterpret_cast<u32x4 *>(vs + ((16 * kb + key) * KC + slot_of<KC>(key, 4 * i + (lane & 3))) * 16) =
              vr[kb][i];
        }
      v4f_t S[MA][2];
#pragma unroll
      for (int j = 0; j < NC; j++)
        scores_step<MA>(j, __builtin_bit_cast(v8h_t, kr[0][j]), __builtin_bit_cast(v8h_t, kr[1][j]), qh, ql, S);
      const bool ok0 = ok[0], ok1 = ok[1], mask = pos + 32 > seen_min || !ok0 || !ok1;
      __builtin_amdgcn_sched_barrier(0);
      if (pos + 128 < end) gload(pos + 128);  // in flight over the rest of this tile
      __builtin_amdgcn_sched_barrier(0);
      v8h_t Ph[MA], Pl[MA];
#pragma unroll
      for (int i = 0; i < MA; i++)
        weights(S[i], c[i], row[i].seen, mask, ok0, ok1, pos, m[i], l[i], O[i], Ph[i], Pl[i]);
#pragma unroll
      for (int n = 0; n < ND; n++) values_step<MA, ND>(n, v_columns(vs, n), Ph, Pl, O);
    }
    // ---- the four waves' parts joined ----
    __syncthreads();
    v4f_t *ob = reinterpret_cast<v4f_t *>(lds);
#pragma unroll
    for (int i = 0; i < MA; i++) {
      l[i] = quarter_sum(l[i]);
      if (lq == 0) ml[wave][16 * i + l16] = make_float2(m[i], l[i]);
#pragma unroll
      for (int n = 0; n < ND; n++) ob[((wave * MA + i) * ND + n) * 64 + lane] = O[i][n];
    }
    if (tid == 0) flags[0] = 0;
    __syncthreads();
    constexpr int NB = (ND + 3) / 4;  // 16-dim blocks a wave joins per row block: wave, wave + 4, ..
    v4f_t R[MA][NB];
    float M[MA], L[MA];
#pragma unroll
    for (int i = 0; i < MA; i++) {
      float w[4];
      M[i] = -INFINITY;
      L[i] = 0.f;
#pragma unroll
      for (int v = 0; v < 4; v++) M[i] = fmaxf(M[i], ml[v][16 * i + l16].x);
#pragma unroll
      for (int v = 0; v < 4; v++) {
        const float2 x = ml[v][16 * i + l16];
        w[v] = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - M[i]);
        L[i] = fmaf(x.y, w[v], L[i]);
      }
      float z = 0.f;  // NaN from any value that is not finite
#pragma unroll
      for (int b = 0; b < NB; b++) {
        R[i][b] = v4f_t{0.f, 0.f, 0.f, 0.f};
        const uint32_t n = 4 * b + wave;
        if (n >= ND) continue;
#pragma unroll
        for (int v = 0; v < 4; v++) R[i][b] += ob[((v * MA + i) * ND + n) * 64 + lane] * w[v];
#pragma unroll
        for (int e = 0; e < 4; e++) z = fmaf(R[i][b][e], 0.f, z);
      }
      const bool bad = row[i].there && row[i].seen > k0 && (!(fmaf(L[i], 0.f, z) == 0.f) || M[i] == -INFINITY);
      const uint64_t all = __ballot(bad);
      const uint32_t rows16 = (uint32_t)(all | all >> 16 | all >> 32 | all >> 48) & 0xffff;
      if (lane == 0 && rows16) atomicOr(&flags[0], rows16 << (16 * i));
    }
    __syncthreads();
    const uint32_t slow = flags[0];
#pragma unroll
    for (int i = 0; i < MA; i++) {
      if (!row[i].there || (slow >> (16 * i + l16) & 1)) continue;
      float *dst = out_row(row[i]);
      const float by = over(M[i], L[i]);
#pragma unroll
      for (int b = 0; b < NB; b++) {
        const uint32_t n = 4 * b + wave, d = 16 * n + 4 * lq;
        // (a row that sees no key here: zeros, whatever the other rows' keys hold)
        if (n < ND && d < a.hd)
          *reinterpret_cast<v4f_t *>(dst + d) = M[i] == -INFINITY ? v4f_t{0.f, 0.f, 0.f, 0.f} : R[i][b] / by;
      }
      if (wave == 0 && lq == 0) put_ml(row[i], M[i], L[i]);
    }
    for (uint32_t todo = slow; todo; todo &= todo - 1) {
      const uint32_t r = __builtin_ctz(todo);
      if (r % 4 == wave) slow_row(row_of(16 * MA * tile + r));
    }
    return;
  }

  // ---- wide ----
  Row row[MB];
  v8h_t qh[MB][NC], ql[MB][NC];
  float c[MB], m[MB], l[MB];
  v4f_t O[MB][ND];
  uint32_t seen_max = 0, seen_min = ~0u;
#pragma unroll
  for (int i = 0; i < MB; i++) {
    row[i] = row_of(64 * MB * tile + 16 * (MB * wave + i) + l16);
    load_q(row[i], qh[i], ql[i], &c[i]);
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int n = 0; n < ND; n++) O[i][n] = v4f_t{0.f, 0.f, 0.f, 0.f};
    seen_max = max(seen_max, row[i].seen);
    seen_min = min(seen_min, row[i].seen);
  }
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) {
    seen_max = max(seen_max, (uint32_t)__shfl_xor((int)seen_max, d, 64));
    seen_min = min(seen_min, (uint32_t)__shfl_xor((int)seen_min, d, 64));
  }
  seen_max = __builtin_amdgcn_readfirstlane(seen_max);
  seen_min = __builtin_amdgcn_readfirstlane(seen_min);
  if (lane == 0) flags[wave] = seen_max;
  __syncthreads();
  const uint32_t end = min(k1, max(max(flags[0], flags[1]), max(flags[2], flags[3])));
  const uint32_t n_tiles = end > k0 ? (end - k0 + 63) / 64 : 0;
  u32x4 kr[NC], vr[NC];
  // Wave w brings the tile's 16-key block w.
  auto gload = [&](uint32_t t) __attribute__((always_inline)) {
    const uint32_t blk = k0 + min(64 * t + 16 * wave, (end - 1 - k0) & ~15u);
    uint64_t at;
    block_at(blk, &at);
    const uint32_t off = min(lane >> 2, end - 1 - blk) * row_bytes;
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const uint32_t ch = 16 * min(4 * i + (lane & 3), last_ch);
      kr[i] = *reinterpret_cast<const u32x4 *>(Kh + at + off + ch);
      vr[i] = *reinterpret_cast<const u32x4 *>(Vh + at + off + ch);
    }
  };
  constexpr uint32_t TILE = 64 * KC * 16;  // bytes of a K or a V tile
  auto to_lds = [&](uint32_t t) __attribute__((always_inline)) {
    char *b = lds + (t & 1) * (2 * TILE);
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const uint32_t key = lane >> 2;
      const uint32_t off = ((16 * wave + key) * KC + slot_of<KC>(key, 4 * i + (lane & 3))) * 16;
      *reinterpret_cast<u32x4 *>(b + off) = kr[i];
      *reinterpret_cast<u32x4 *>(b + TILE + off) = vr[i];
    }
  };
  if (n_tiles) {
    gload(0);
    to_lds(0);
    if (n_tiles > 1) gload(1);
  }
  for (uint32_t t = 0; t < n_tiles; t++) {
    lds_barrier();  // tile t is written; the reads of tile t - 1, whose buffer comes next, are done
    if (t + 1 < n_tiles) {
      to_lds(t + 1);
      if (t + 2 < n_tiles) gload(t + 2);
    }
    const uint32_t pos0 = k0 + 64 * t;
    if (pos0 >= seen_max) continue;  // (uniform: none of this wave's rows sees the tile)
    const char *kb_ = lds + (t & 1) * (2 * TILE);
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const uint32_t pos = pos0 + 32 * half;
      bool ok0 = true, ok1 = true;
      if (holes) {
        if (pos < end) ok0 = block_id((pos - k0) >> 4) != NO_PAGE;
        if (pos + 16 < end) ok1 = block_id((pos + 16 - k0) >> 4) != NO_PAGE;
      }
      const bool mask = pos + 32 > seen_min || !ok0 || !ok1;
      v4f_t S[MB][2];
#pragma unroll
      for (int j = 0; j < NC; j++) {
        const char *k = kb_ + ((32 * half + l16) * KC + slot_of<KC>(l16, 4 * j + lq)) * 16;
        scores_step<MB>(j, *reinterpret_cast<const v8h_t *>(k), *reinterpret_cast<const v8h_t *>(k + 16 * KC * 16), qh,
                        ql, S);
      }
      v8h_t Ph[MB], Pl[MB];
#pragma unroll
      for (int i = 0; i < MB; i++)
        weights(S[i], c[i], row[i].seen, mask, ok0, ok1, pos, m[i], l[i], O[i], Ph[i], Pl[i]);
#pragma unroll
      for (int n = 0; n < ND; n++)
        values_step<MB, ND>(n, v_columns(kb_ + TILE + 32 * half * KC * 16, n), Ph, Pl, O);
    }
  }
#pragma unroll
  for (int i = 0; i < MB; i++) {
    l[i] = quarter_sum(l[i]);
    float z = 0.f;
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) z = fmaf(O[i][n][e], 0.f, z);
    const bool bad = row[i].there && row[i].seen > k0 && (!(fmaf(l[i], 0.f, z) == 0.f) || m[i] == -INFINITY);
    const uint64_t all = __ballot(bad);
    const uint32_t slow = (uint32_t)(all | all >> 16 | all >> 32 | all >> 48) & 0xffff;
    if (row[i].there && !(slow >> l16 & 1)) {
      float *dst = out_row(row[i]);
#pragma unroll
      for (int n = 0; n < ND; n++)
        if (16 * n + 4 * lq < a.hd)
          *reinterpret_cast<v4f_t *>(dst + 16 * n + 4 * lq) =
              m[i] == -INFINITY ? v4f_t{0.f, 0.f, 0.f, 0.f} : O[i][n] / over(m[i], l[i]);
      if (lq == 0) put_ml(row[i], m[i], l[i]);
    }
    for (uint32_t todo = slow; todo; todo &= todo - 1)
      slow_row(row_of(64 * MB * tile + 16 * (MB * wave + i) + __builtin_ctz(todo)));
  }
}

// The parts of every row joined: a wave per row.
__global__ __launch_bounds__(256) void attn_paged_join_kernel(Args a) {
  const uint32_t lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const uint32_t token = row / a.heads, s = token / a.n_new, slots = a.n_p + a.n_t;
  const uint32_t len = a.kv.length(s), seen = seen_by(len, a.n_new, token % a.n_new);
  const uint32_t n = len > a.start ? len - a.start : 0, ct = tail_chunk(n, a.n_t);
  const float2 *ml = reinterpret_cast<const float2 *>(a.part + (uint64_t)slots * a.rows * a.hd);
  // Which parts were written: those with a key the row sees.
  const uint64_t first = lane < a.n_p ? (uint64_t)lane * a.cp : a.start + (uint64_t)(lane - a.n_p) * ct;
  const bool mine = lane < slots && first < seen;
  float2 x = make_float2(-INFINITY, 0.f);
  if (mine) x = ml[(uint64_t)lane * a.rows + row];
  const float M = wave_max_all(x.x);
  const float w = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - M);
  const float L = wave_sum_all(x.y * w);
  const uint64_t have = __ballot(mine && x.x != -INFINITY);
  for (uint32_t d = 4 * lane; d < a.hd; d += 256) {
    v4f_t acc = {0.f, 0.f, 0.f, 0.f};
    for (uint64_t todo = have; todo; todo &= todo - 1) {
      const int i = __builtin_ctzll(todo);
      const float wi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i));
      acc += *reinterpret_cast<const v4f_t *>(a.part + ((uint64_t)i * a.rows + row) * a.hd + d) * wi;
    }
    *reinterpret_cast<v4f_t *>(a.o + (uint64_t)row * a.hd + d) = have ? acc / L : acc;
  }
}

}  // namespace

void launch_attn_paged(mdma_ctx *ctx, const float *q, const PagedView &kv, uint32_t n_new, uint32_t q_heads,
                       uint32_t kv_heads, uint32_t hd, float *o) {
  Args a{};
  a.q = q;
  a.kv = kv;
  a.o = o;
  a.n_new = n_new;
  a.heads = q_heads;
  a.group = q_heads / kv_heads;
  a.hd = hd;
  a.rows = kv.n_seqs * n_new * q_heads;
  a.scale2 = (float)(1.4426950408889634 / sqrt((double)hd));
  const uint64_t cap = (uint64_t)kv.max_pages << kv.page_shift, pre = (uint64_t)kv.n_prefix << kv.page_shift;
  const uint64_t rows_p = (uint64_t)kv.n_seqs * n_new * a.group, rows_t = (uint64_t)n_new * a.group;
  const uint32_t NC = hd <= 64 ? 2 : hd <= 96 ? 3 : hd <= 128 ? 4 : 8, MB = NC <= 4 ? 2 : 1;
  const auto tiles = [](uint64_t n, uint64_t per) { return (uint32_t)((n + per - 1) / per); };
  const uint64_t want = 2ull * ctx->cu_count;  // workgroups that fill the chip
  // A prefix of a few tiles is read again by each sequence instead.
  bool shared = kv.n_seqs > 1 && pre >= 256;
  uint64_t parts_bytes = 0;
  auto plan = [&](bool split) {
    a.start = split && shared ? (uint32_t)pre : 0;
    a.wide_t = rows_t > 32;
    a.wide_p = rows_p > 32;
    a.rt_t = a.wide_t ? tiles(rows_t, 64 * MB) : 1;
    a.rt_p = a.wide_p ? tiles(rows_p, 64 * MB) : 1;
    const uint64_t units = (uint64_t)kv.n_seqs * kv_heads * a.rt_t, keys = cap - a.start;
    a.n_p = 0;
    if (a.start) {
      const uint64_t per = (uint64_t)kv_heads * a.rt_p;
      const uint64_t n = std::min<uint64_t>({MAX_PARTS / 2, tiles(pre, 256), std::max<uint64_t>(1, want / 2 / per)});
      a.cp = tiles(tiles(pre, n), 128) * 128;
      a.n_p = tiles(pre, a.cp);
    }
    a.n_t = 1;
    if (split && keys > 768)
      a.n_t = (uint32_t)std::min<uint64_t>({MAX_PARTS / 2, tiles(keys, 256),
                                            std::max<uint64_t>(tiles(keys, 1024), tiles(want * 3 / 2, units))});
    const uint32_t slots = a.n_p + a.n_t;
    parts_bytes = slots > 1 ? (uint64_t)slots * a.rows * (hd + 2) * 4 : 0;
  };
  plan(true);
  if (parts_bytes) {
    a.part = static_cast<float *>(split_space(ctx, parts_bytes));
    if (!a.part) plan(false);
  }
  const uint32_t need = std::max(a.wide_t ? 1u : (uint32_t)rows_t, a.n_p && !a.wide_p ? (uint32_t)rows_p : 1u);
  const uint64_t blocks_p = (uint64_t)tiles((uint64_t)a.n_p * kv_heads, 8) * 8 * a.rt_p;
  const uint64_t blocks = blocks_p + (uint64_t)tiles((uint64_t)a.n_t * kv_heads * kv.n_seqs, 8) * 8 * a.rt_t;
  if (blocks > INT32_MAX) fail(MDMA_ERR_SIZE_OVERFLOW, "attn_paged: too many query rows");
  a.blocks_p = (uint32_t)blocks_p;
  const dim3 grid((uint32_t)blocks);
#define ATTN_PAGED(NC_, MB_)                                                                   \
  if (NC == NC_) {                                                                             \
    if (need <= 16) attn_paged_kernel<NC_, 1, MB_><<<grid, 256, 0, ctx->stream>>>(a);          \
    else attn_paged_kernel<NC_, 2, MB_><<<grid, 256, 0, ctx->stream>>>(a);                     \
  }
  ATTN_PAGED(2, 2)
  ATTN_PAGED(3, 2)
  ATTN_PAGED(4, 2)
  ATTN_PAGED(8, 1)
#undef ATTN_PAGED
  if (a.part) attn_paged_join_kernel<<<(a.rows + 3) / 4, 256, 0, ctx->stream>>>(a);
  hip_check(hipGetLastError(), "attn_paged launch");
}

}  // namespace mdma
