// Host side of the paged key-value caches: the page table and the checks of
// the slm_op_paged_* calls.  Everything a kernel indexes with (page ids,
// lengths, pool sizes, strides) is checked here, on the host's copy of the
// table, so no call reaches memory outside its buffers.
#include <algorithm>
#include <string>
#include <vector>

#include "capi.hpp"
#include "common.cuh"
#include "page_table.hpp"
#include "paged.cuh"

struct slm_table {
  slm_ctx* ctx;
  slm::PageTable host;
  std::vector<uint32_t> sent;  // what the device holds of host.words
  uint32_t* dev = nullptr;
};

namespace slm {
namespace {

// Sends what changed since the last call, in stream order.
void flush(slm_table* t) {
  PageTable& h = t->host;
  if (h.changed.empty()) return;
  const PageTable::Update u = h.update(t->sent);
  cudaStream_t st = t->ctx->stream;
  if (u.hi) {
    // Pageable source: the runtime has read it when the call returns.
    SLM_CUDA(cudaMemcpyAsync(t->dev + u.lo, h.words.data() + u.lo, (u.hi - u.lo) * sizeof(uint32_t),
                             cudaMemcpyHostToDevice, st));
    std::copy(h.words.begin() + u.lo, h.words.begin() + u.hi, t->sent.begin() + u.lo);
  } else {
    for (size_t j = 0; j < u.at.size(); j += kPutWords)
      table_put(t->dev, u.at.data() + j, u.value.data() + j, (int)std::min<size_t>(kPutWords, u.at.size() - j), st);
    for (size_t j = 0; j < u.at.size(); j++) t->sent[u.at[j]] = u.value[j];
  }
  h.settle();
}

PagedTable on_device(slm_table* t) {
  PagedTable d;
  d.lens = t->dev, d.ids = t->dev + t->host.seqs;
  d.n = (int)t->host.seqs, d.per = (int)t->host.per;
  d.set_page((uint32_t)t->host.page);
  return d;
}

void not_capturing(slm_ctx* c, const char* what) {
  cudaStreamCaptureStatus s;
  SLM_CUDA(cudaStreamIsCapturing(c->stream, &s));
  SLM_REQUIRE(s == cudaStreamCaptureStatusNone, std::string(what) + ": the stream is being captured");
}

// Buffers of this context, none twice.
void own_buffers(slm_ctx* c, std::initializer_list<const slm_buf*> bufs, const char* what) {
  for (auto a = bufs.begin(); a != bufs.end(); ++a) {
    if (!*a) continue;
    SLM_REQUIRE((*a)->ctx == c, std::string(what) + ": a buffer belongs to another context");
    for (auto b = bufs.begin(); b != a; ++b)
      SLM_REQUIRE(*a != *b, std::string(what) + ": one buffer is passed twice");
  }
}

// Checks the pool's geometry against the table and its buffers.
void pool(const slm_paged* p, const slm_table* t, const slm_buf* k, const slm_buf* v, const slm_buf* weights,
          const char* what) {
  auto require = [&](bool ok, const char* msg) { SLM_REQUIRE(ok, std::string(what) + ": " + msg); };
  require(p->type == SLM_PAGES_F32 || p->type == SLM_PAGES_BF16, "unknown page type");
  require(p->dh >= 8 && p->dh <= 256 && p->dh % 8 == 0, "head size must be a multiple of 8, at most 256");
  require(p->key_heads > 0 && p->key_heads <= 65535, "bad number of key heads");
  const size_t rows = checked_mul(checked_mul(t->host.pages, p->key_heads), t->host.page);
  require(rows < ((size_t)1 << 32), "pages x key heads x page must stay below 2^32");
  const size_t floats = p->type == SLM_PAGES_BF16 ? rows * (p->dh / 2) : rows * p->dh;
  view(k, 0, floats, "paged k");
  view(v, 0, floats, "paged v");
  if (weights) view(weights, 0, rows, "paged weights");
}

// n rows of `width` floats at off, off + ld, …
const float* rows_of(const slm_buf* b, size_t off, size_t n, size_t ld, size_t width, const char* what) {
  SLM_REQUIRE(ld >= width, std::string(what) + ": the row stride is below the row");
  SLM_REQUIRE(ld < ((size_t)1 << 40), std::string(what) + ": the row stride is too large");
  return view(b, off, n ? checked_add(checked_mul(n - 1, ld), width) : 0, what);
}

}  // namespace
}  // namespace slm

using namespace slm;

extern "C" {

int slm_table_new(slm_ctx* c, size_t seqs, size_t per_seq, size_t page, size_t pages, slm_table** out) {
  return guard([&] {
    SLM_REQUIRE(c && out, "table: bad arguments");
    Device dev(c);
    not_capturing(c, "table_new");  // a captured clearing would empty the table at every replay
    auto* t = new slm_table{c, PageTable(seqs, per_seq, page, pages)};
    try {
      const size_t bytes = t->host.words.size() * sizeof(uint32_t);
      t->sent = t->host.words;
      t->dev = static_cast<uint32_t*>(dev_alloc(bytes));
      SLM_CUDA(cudaMemsetAsync(t->dev, 0, bytes, c->stream));
    } catch (...) {
      dev_free(t->dev);
      delete t;
      throw;
    }
    ctx_retain(c);
    *out = t;
  });
}

int slm_table_free(slm_table* t) {
  return guard([&] {
    if (!t) return;
    slm_ctx* c = t->ctx;
    {
      Device dev(c);
      // The wait below would end a capture.  A query that fails keeps no table from being freed.
      cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
      cudaStreamIsCapturing(c->stream, &capture);
      SLM_REQUIRE(capture == cudaStreamCaptureStatusNone, "table_free: the stream is being captured");
      cudaStreamSynchronize(c->stream);
      dev_free(t->dev);
    }
    delete t;
    ctx_release(c);
  });
}

int slm_table_assign(slm_table* t, size_t seq, const uint32_t* ids, size_t n) {
  return guard([&] {
    SLM_REQUIRE(t, "table_assign: bad arguments");
    t->host.assign(seq, ids, n);
  });
}

int slm_table_set_lens(slm_table* t, const uint32_t* lens, size_t n) {
  return guard([&] {
    SLM_REQUIRE(t, "table_set_lens: bad arguments");
    t->host.set_lens(lens, n);
  });
}

int slm_table_lens(const slm_table* t, uint32_t* out, size_t n) {
  return guard([&] {
    SLM_REQUIRE(t && out && n == t->host.seqs, "table_lens: bad arguments");
    std::copy(t->host.words.begin(), t->host.words.begin() + n, out);
  });
}

int slm_op_paged_store(slm_ctx* c, slm_buf* k, slm_buf* v, slm_buf* weights, slm_table* t, size_t first, size_t count,
                       const slm_buf* ksrc, size_t koff, size_t ldk, const slm_buf* vsrc, size_t voff, size_t ldv,
                       size_t m, const slm_paged* p) {
  return guard([&] {
    SLM_REQUIRE(c && t && p, "paged_store: bad arguments");
    SLM_REQUIRE(t->ctx == c, "paged_store: the table belongs to another context");
    // ksrc and vsrc may be one buffer (a fused projection).
    own_buffers(c, {k, v, weights, ksrc}, "paged_store");
    own_buffers(c, {k, v, weights, vsrc}, "paged_store");
    pool(p, t, k, v, weights, "paged_store");
    t->host.check_store(first, count, m);
    const size_t width = p->key_heads * p->dh;
    PagedStoreArgs a;
    a.ks = rows_of(ksrc, koff, count * m, ldk, width, "paged_store ksrc");
    a.vs = rows_of(vsrc, voff, count * m, ldv, width, "paged_store vsrc");
    Device dev(c);
    not_capturing(c, "paged_store");
    if (!m || !count) return;
    flush(t);
    a.t = on_device(t);
    a.first = (int)first, a.count = (int)count, a.m = (int)m, a.key_heads = (int)p->key_heads, a.dh = (int)p->dh;
    a.bf16 = p->type == SLM_PAGES_BF16;
    a.ldk = (long long)ldk, a.ldv = (long long)ldv;
    a.k = k->ptr, a.v = v->ptr, a.weights = weights ? weights->ptr : nullptr;
    paged_store(a, c->stream);
  });
}

int slm_op_paged_attend(slm_ctx* c, slm_buf* y, slm_buf* scores, const slm_buf* q, size_t qoff, size_t ldq,
                        const slm_buf* k, const slm_buf* v, slm_buf* weights, slm_table* t, const slm_paged* p) {
  return guard([&] {
    SLM_REQUIRE(c && y && scores && t && p, "paged_attend: bad arguments");
    SLM_REQUIRE(t->ctx == c, "paged_attend: the table belongs to another context");
    own_buffers(c, {y, scores, q, k, v, weights}, "paged_attend");
    pool(p, t, k, v, weights, "paged_attend");
    SLM_REQUIRE(p->heads > 0 && p->heads <= 65535 && p->heads % p->key_heads == 0, "paged_attend: bad number of heads");
    SLM_REQUIRE(p->reach > 0, "paged_attend: reach is 0");
    SLM_REQUIRE(!weights || !t->host.shared, "paged_attend: weights of a page that two sequences list");
    const size_t width = p->heads * p->dh;
    PagedAttendArgs a;
    a.q = rows_of(q, qoff, t->host.seqs, ldq, width, "paged_attend q");
    Device dev(c);
    not_capturing(c, "paged_attend");
    a.t = on_device(t);
    a.host_lens = t->host.words.data();
    a.heads = (int)p->heads, a.key_heads = (int)p->key_heads, a.dh = (int)p->dh;
    a.reach = p->reach >= ((size_t)1 << 31) ? 0 : (long long)p->reach;
    a.scale = p->scale, a.bf16 = p->type == SLM_PAGES_BF16;
    a.ldq = (long long)ldq;
    a.k = k->ptr, a.v = v->ptr, a.weights = weights ? weights->ptr : nullptr;
    ensure(y, t->host.seqs * width);
    // What the scratch takes grows with the lengths: some more than that, so
    // that few of a decode loop's steps wait for a new one.
    const size_t scratch = paged_attend_scratch(a);
    if (scratch > scores->len) ensure(scores, scratch + scratch / 4);
    a.y = y->ptr, a.scratch = scores->ptr;
    flush(t);
    paged_attend(a, c->stream);
  });
}

int slm_op_paged_evict(slm_ctx* c, slm_buf* kept, slm_buf* k, slm_buf* v, slm_buf* weights, slm_table* from,
                       slm_table* to, size_t keep, size_t sinks, size_t recent, const slm_paged* p) {
  return guard([&] {
    SLM_REQUIRE(c && kept && weights && from && to && p, "paged_evict: bad arguments");
    SLM_REQUIRE(from->ctx == c && to->ctx == c, "paged_evict: a table belongs to another context");
    from->host.check_evict(to->host, keep, sinks, recent);
    own_buffers(c, {kept, k, v, weights}, "paged_evict");
    pool(p, from, k, v, weights, "paged_evict");
    const size_t words = checked_mul(checked_mul(from->host.seqs, p->key_heads), keep);
    Device dev(c);
    not_capturing(c, "paged_evict");
    ensure(kept, words);
    PagedEvictArgs a;
    a.longest = 0;
    for (size_t i = 0; i < from->host.seqs; i++) {
      to->host.set_len(i, (uint32_t)std::min<size_t>(from->host.len(i), keep));
      a.longest = std::max(a.longest, (int)from->host.len(i));
    }
    flush(from);
    flush(to);
    a.from = on_device(from), a.to = on_device(to);
    a.key_heads = (int)p->key_heads, a.dh = (int)p->dh, a.bf16 = p->type == SLM_PAGES_BF16;
    a.keep = (int)keep, a.sinks = (int)sinks, a.recent = (int)recent;
    a.k = k->ptr, a.v = v->ptr, a.weights = weights->ptr;
    a.kept = reinterpret_cast<uint32_t*>(kept->ptr);
    paged_evict(a, c->stream);
  });
}

}  // extern "C"
