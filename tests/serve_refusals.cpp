// Every refusal of the paged cache's and adapters' entry points, without a
// GPU: contexts and buffers made here, none of whose memory a refused call
// may touch (their addresses are not mapped).
#include <cstdio>
#include <cmath>
#include <cstring>
#include <functional>

#include "../mdma_amd/csrc/internal.h"

static int failures = 0;
static void expect(const char *what, int code, int got) {
  if (got == code) return;
  failures++;
  printf("%s: status %d, expected %d (%s)\n", what, got, code, mdma_gfx950_last_error());
}

int main() {
  const int SHAPE = MDMA_ERR_SHAPE_MISMATCH, OVER = MDMA_ERR_SIZE_OVERFLOW, NOTIMP = MDMA_ERR_NOT_IMPLEMENTED;
  mdma_ctx ctx, other;
  uint64_t next = 1ull << 40;  // far from anything mapped
  auto mk = [&](uint64_t bytes) {
    mdma_buf b;
    b.ctx = &ctx;
    b.ptr = reinterpret_cast<char *>(next);
    b.len = bytes;
    next += (bytes + 4095) / 4096 * 4096 + 4096;
    return b;
  };
  // 2 layers, 10 pages of 16 positions of 64; 3 sequences of up to 5 pages; 4 heads of 32 over 2.
  mdma_buf k = mk(2 * 10 * 16 * 64 * 2), v = mk(k.len), table = mk(3 * 5 * 4), lens = mk(12), refs = mk(40);
  mdma_buf from = mk(12), keep = mk(12), grow = mk(12), status = mk(12), live = mk(4), prefix = mk(8);
  mdma_buf q = mk(3 * 2 * 128 * 4), o = mk(q.len), nk = mk(3 * 2 * 64 * 4), nv = mk(nk.len);
  mdma_kv_pages good{&k, &v, &table, &lens, &refs, 2, 10, 16, 64, 3, 5};
  mdma_attn_spec att{32, 4, 2};
  mdma_rope_spec rope{32, 1e4f};
  using P = mdma_kv_pages;
  // Every call that takes a cache refuses the same bad caches.
  struct { const char *what; int code; std::function<void(P &)> f; } bad[] = {
      {"null k", SHAPE, [](P &p) { p.k = nullptr; }}, {"null v", SHAPE, [](P &p) { p.v = nullptr; }},
      {"null table", SHAPE, [](P &p) { p.table = nullptr; }}, {"null lens", SHAPE, [](P &p) { p.lens = nullptr; }},
      {"null refs", SHAPE, [](P &p) { p.refs = nullptr; }}, {"no layers", SHAPE, [](P &p) { p.n_layers = 0; }},
      {"no pages", SHAPE, [](P &p) { p.n_pages = 0; }}, {"no sequences", SHAPE, [](P &p) { p.n_seqs = 0; }},
      {"no entries", SHAPE, [](P &p) { p.max_pages = 0; }}, {"page 8", SHAPE, [](P &p) { p.page_len = 8; }},
      {"page 24", SHAPE, [](P &p) { p.page_len = 24; }}, {"page 512", SHAPE, [](P &p) { p.page_len = 512; }},
      {"page 0", SHAPE, [](P &p) { p.page_len = 0; }}, {"width 60", SHAPE, [](P &p) { p.kv_width = 60; }},
      {"width 0", SHAPE, [](P &p) { p.kv_width = 0; }}, {"many sequences", SHAPE, [](P &p) { p.n_seqs = 1025; }},
      {"a layer more than the pool", SHAPE, [](P &p) { p.n_layers = 3; }},
      {"a page more than the pool", SHAPE, [](P &p) { p.n_pages = 11; }},
      {"an entry more than the table", SHAPE, [](P &p) { p.max_pages = 6; }},
      {"a sequence more than the books", SHAPE, [](P &p) { p.n_seqs = 4; }},
      {"2^31 pages", OVER, [](P &p) { p.n_pages = 1ull << 31; }},
      {"2^63 pages", OVER, [](P &p) { p.n_pages = 1ull << 63; }},
      {"2^31 positions", OVER, [](P &p) { p.max_pages = (1ull << 31) / 16; }},
      {"2^63 entries", OVER, [](P &p) { p.max_pages = 1ull << 63; }},
      {"2^63 layers", OVER, [](P &p) { p.n_layers = 1ull << 63; }},
      {"v is k", SHAPE, [&](P &p) { p.v = &k; }}, {"lens in refs", SHAPE, [&](P &p) { p.lens = &refs; }}};
  for (auto &b : bad) {
    P p = good;
    b.f(p);
    expect((std::string("fork, ") + b.what).c_str(), b.code, mdma_gfx950_kv_pages_fork(&ctx, &p, &from, &keep));
    expect((std::string("grow, ") + b.what).c_str(), b.code, mdma_gfx950_kv_pages_grow(&ctx, &p, &grow, &status));
    expect((std::string("compact, ") + b.what).c_str(), b.code, mdma_gfx950_kv_pages_compact(&ctx, &p, &live));
    expect((std::string("write, ") + b.what).c_str(), b.code,
           mdma_gfx950_rope_kv_write_paged(&ctx, &q, &nk, &nv, &p, 0, &rope));
    if (strcmp(b.what, "v is k") && strcmp(b.what, "lens in refs"))  // (only read there)
      expect((std::string("attn, ") + b.what).c_str(), b.code,
             mdma_gfx950_attn_paged(&ctx, &q, &p, 0, &prefix, &att, &o));
  }
  for (mdma_buf **field : {&good.k, &good.v, &good.table, &good.lens, &good.refs}) {
    mdma_buf moved = **field, *was = *field;
    *field = &moved;
    moved.ctx = &other;
    expect("another context", SHAPE, mdma_gfx950_attn_paged(&ctx, &q, &good, 0, nullptr, &att, &o));
    expect("another context", SHAPE, mdma_gfx950_kv_pages_compact(&ctx, &good, nullptr));
    moved = *was;
    moved.ptr += 2;
    expect("misaligned", SHAPE, mdma_gfx950_kv_pages_compact(&ctx, &good, nullptr));
    *field = was;
  }
  mdma_buf short12 = mk(8), odd = mk(12);
  odd.ptr += 1;
  // fork, grow, compact
  expect("null context", SHAPE, mdma_gfx950_kv_pages_fork(nullptr, &good, &from, &keep));
  expect("null pages", SHAPE, mdma_gfx950_kv_pages_fork(&ctx, nullptr, &from, &keep));
  expect("null from", SHAPE, mdma_gfx950_kv_pages_fork(&ctx, &good, nullptr, &keep));
  expect("short from", SHAPE, mdma_gfx950_kv_pages_fork(&ctx, &good, &short12, &keep));
  expect("short keep", SHAPE, mdma_gfx950_kv_pages_fork(&ctx, &good, &from, &short12));
  expect("misaligned from", SHAPE, mdma_gfx950_kv_pages_fork(&ctx, &good, &odd, nullptr));
  expect("from is lens", SHAPE, mdma_gfx950_kv_pages_fork(&ctx, &good, &lens, nullptr));
  expect("keep is lens", SHAPE, mdma_gfx950_kv_pages_fork(&ctx, &good, &from, &lens));
  expect("null context", SHAPE, mdma_gfx950_kv_pages_grow(nullptr, &good, &grow, &status));
  expect("null grow", SHAPE, mdma_gfx950_kv_pages_grow(&ctx, &good, nullptr, &status));
  expect("null status", SHAPE, mdma_gfx950_kv_pages_grow(&ctx, &good, &grow, nullptr));
  expect("short grow", SHAPE, mdma_gfx950_kv_pages_grow(&ctx, &good, &short12, &status));
  expect("short status", SHAPE, mdma_gfx950_kv_pages_grow(&ctx, &good, &grow, &short12));
  expect("status is grow", SHAPE, mdma_gfx950_kv_pages_grow(&ctx, &good, &grow, &grow));
  expect("status is refs", SHAPE, mdma_gfx950_kv_pages_grow(&ctx, &good, &grow, &refs));
  expect("null context", SHAPE, mdma_gfx950_kv_pages_compact(nullptr, &good, &live));
  expect("n_live in lens", SHAPE, mdma_gfx950_kv_pages_compact(&ctx, &good, &lens));
  // write
  auto write = [&](const char *what, int code, mdma_buf *wq, mdma_buf *wk, mdma_buf *wv, uint64_t layer,
                   const mdma_rope_spec *s) {
    expect(what, code, mdma_gfx950_rope_kv_write_paged(&ctx, wq, wk, wv, &good, layer, s));
  };
  mdma_buf cut = q, off = q, empty = mk(0);
  cut.len -= 4;
  off.ptr += 4;
  mdma_rope_spec r0{0, 1e4f}, r33{33, 1e4f}, r48{48, 1e4f}, rneg{32, -1.f}, rinf{32, INFINITY}, rnan{32, NAN};
  write("null q", SHAPE, nullptr, &nk, &nv, 0, &rope);
  write("null k", SHAPE, &q, nullptr, &nv, 0, &rope);
  write("null v", SHAPE, &q, &nk, nullptr, 0, &rope);
  write("null spec", SHAPE, &q, &nk, &nv, 0, nullptr);
  write("layer 2 of 2", SHAPE, &q, &nk, &nv, 2, &rope);
  for (auto *s : {&r0, &r33, &r48, &rneg, &rinf, &rnan}) write("rope spec", SHAPE, &q, &nk, &nv, 0, s);
  write("q not whole", SHAPE, &cut, &nk, &nv, 0, &rope);
  write("q misaligned", SHAPE, &off, &nk, &nv, 0, &rope);
  write("k not whole", SHAPE, &q, &cut, &nv, 0, &rope);
  write("no tokens", SHAPE, &q, &empty, &empty, 0, &rope);
  write("empty q", SHAPE, &empty, &nk, &nv, 0, &rope);
  write("q is k", SHAPE, &nk, &nk, &nv, 0, &rope);
  write("q in the pool", SHAPE, &k, &nk, &nv, 0, &rope);
  mdma_buf long_table = mk(3ull * ((1 << 20) + 1) * 4);
  P far = good;
  far.table = &long_table;
  far.max_pages = (1 << 20) + 1;  // 16 positions past 2^24
  expect("positions past 2^24", OVER, mdma_gfx950_rope_kv_write_paged(&ctx, &q, &nk, &nv, &far, 0, &rope));
  // attn
  auto attn = [&](const char *what, int code, const mdma_buf *aq, uint64_t layer, const mdma_buf *pre, mdma_attn_spec s,
                  mdma_buf *ao) { expect(what, code, mdma_gfx950_attn_paged(&ctx, aq, &good, layer, pre, &s, ao)); };
  mdma_buf pre3 = mk(24), preodd = mk(6);
  expect("null spec", SHAPE, mdma_gfx950_attn_paged(&ctx, &q, &good, 0, nullptr, nullptr, &o));
  attn("null q", SHAPE, nullptr, 0, nullptr, att, &o);
  attn("null o", SHAPE, &q, 0, nullptr, att, nullptr);
  attn("layer", SHAPE, &q, 2, nullptr, att, &o);
  attn("layer", SHAPE, &q, 1ull << 40, nullptr, att, &o);
  attn("head_dim 0", SHAPE, &q, 0, nullptr, {0, 4, 2}, &o);
  attn("head_dim 12", SHAPE, &q, 0, nullptr, {12, 4, 2}, &o);
  attn("head_dim 264", SHAPE, &q, 0, nullptr, {264, 4, 2}, &o);
  attn("width", SHAPE, &q, 0, nullptr, {32, 4, 4}, &o);
  attn("no kv heads", SHAPE, &q, 0, nullptr, {32, 4, 0}, &o);
  attn("kv heads that overflow", SHAPE, &q, 0, nullptr, {32, 4, (1ull << 59) + 2}, &o);
  attn("heads", SHAPE, &q, 0, nullptr, {32, 3, 2}, &o);
  attn("no heads", SHAPE, &q, 0, nullptr, {32, 0, 2}, &o);
  attn("many heads", SHAPE, &q, 0, nullptr, {32, 65536, 2}, &o);
  attn("q not whole", SHAPE, &cut, 0, nullptr, att, &o);
  attn("empty q", SHAPE, &empty, 0, nullptr, att, &o);
  attn("o short", SHAPE, &q, 0, nullptr, att, &nk);
  attn("o is q", SHAPE, &q, 0, nullptr, att, &q);
  attn("o is k", SHAPE, &q, 0, nullptr, att, &k);
  attn("prefix past max_pages", SHAPE, &q, 0, &pre3, att, &o);
  attn("prefix not whole ids", SHAPE, &q, 0, &preodd, att, &o);
  // adapters
  mdma_lora *l = nullptr;
  expect("null out", SHAPE, mdma_gfx950_lora_new(&ctx, 1, 8, 8, 8, 1, nullptr));
  expect("null context", SHAPE, mdma_gfx950_lora_new(nullptr, 1, 8, 8, 8, 1, &l));
  expect("dtype", NOTIMP, mdma_gfx950_lora_new(&ctx, 12, 8, 8, 8, 1, &l));
  expect("no columns", SHAPE, mdma_gfx950_lora_new(&ctx, 1, 0, 8, 8, 1, &l));
  expect("no rows", SHAPE, mdma_gfx950_lora_new(&ctx, 1, 8, 0, 8, 1, &l));
  expect("rank 0", SHAPE, mdma_gfx950_lora_new(&ctx, 1, 8, 8, 0, 1, &l));
  expect("rank 257", SHAPE, mdma_gfx950_lora_new(&ctx, 1, 8, 8, 257, 1, &l));
  expect("no slots", SHAPE, mdma_gfx950_lora_new(&ctx, 1, 8, 8, 8, 0, &l));
  expect("columns", OVER, mdma_gfx950_lora_new(&ctx, 1, 1ull << 40, 8, 8, 1, &l));
  expect("rows", OVER, mdma_gfx950_lora_new(&ctx, 1, 8, 1ull << 63, 8, 1, &l));
  expect("slots", OVER, mdma_gfx950_lora_new(&ctx, 1, 8, 8, 8, 1ull << 60, &l));
  expect("null adapters", SHAPE, mdma_gfx950_lora_add(&ctx, nullptr, &from, &q, &o, &o));
  expect("null adapters", SHAPE, mdma_gfx950_lora_load(nullptr, 0, nullptr, nullptr, 0, 1.f));
  expect("free of none", MDMA_OK, mdma_gfx950_lora_free(nullptr));
  if (!failures) printf("ok\n");
  return failures != 0;
}
