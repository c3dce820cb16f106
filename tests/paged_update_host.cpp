// What a page table sends to the device, behind plain C calls: a table, and the
// words that a device which follows its updates holds.
#include "../slm.use_b200/csrc/page_table.hpp"

namespace {
struct Both {
  slm::PageTable host;
  std::vector<uint32_t> device;
};
Both* at(void* p) { return static_cast<Both*>(p); }
}  // namespace

extern "C" {
void* pu_new(size_t seqs, size_t per, size_t page, size_t pages) {
  auto* b = new Both{slm::PageTable(seqs, per, page, pages), {}};
  b->device = b->host.words;
  return b;
}
void pu_free(void* b) { delete at(b); }
void pu_assign(void* b, size_t seq, const uint32_t* ids, size_t n) { at(b)->host.assign(seq, ids, n); }
void pu_set_lens(void* b, const uint32_t* lens, size_t n) { at(b)->host.set_lens(lens, n); }
// Sends; out: the single words, and the words of the range.  1 when the device holds the table then.
int pu_send(void* b, size_t* out) {
  auto& h = at(b)->host;
  auto& d = at(b)->device;
  const auto u = h.update(d);
  out[0] = u.hi ? 0 : u.at.size(), out[1] = u.hi - u.lo;
  if (u.hi)
    std::copy(h.words.begin() + u.lo, h.words.begin() + u.hi, d.begin() + u.lo);
  else
    for (size_t j = 0; j < u.at.size(); j++) d[u.at[j]] = u.value[j];
  h.settle();
  return d == h.words;
}
}
