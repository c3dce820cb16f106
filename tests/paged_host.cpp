// The host's page table (slm.use_b200/csrc/page_table.hpp) behind plain C
// calls, so that its refusals are tested without a GPU: 0, or 1 and a message.
#include <string>

#include "../slm.use_b200/csrc/page_table.hpp"

namespace {
std::string g_error;
template <class F>
int guard(F&& f) {
  try {
    f();
    return 0;
  } catch (const std::invalid_argument& e) {
    g_error = e.what();
    return 1;
  }
}
using T = slm::PageTable;
T* at(void* p) { return static_cast<T*>(p); }
}  // namespace

extern "C" {
const char* pt_error() { return g_error.c_str(); }
int pt_new(size_t seqs, size_t per, size_t page, size_t pages, void** out) {
  return guard([&] { *out = new T(seqs, per, page, pages); });
}
void pt_free(void* t) { delete at(t); }
int pt_assign(void* t, size_t seq, const uint32_t* ids, size_t n) {
  return guard([&] { at(t)->assign(seq, ids, n); });
}
int pt_set_lens(void* t, const uint32_t* lens, size_t n) {
  return guard([&] { at(t)->set_lens(lens, n); });
}
int pt_check_store(void* t, size_t first, size_t count, size_t m) {
  return guard([&] { at(t)->check_store(first, count, m); });
}
int pt_check_evict(void* t, void* to, size_t keep, size_t sinks, size_t recent) {
  return guard([&] { at(t)->check_evict(*at(to), keep, sinks, recent); });
}
size_t pt_shared(void* t) { return at(t)->shared; }
void pt_words(void* t, uint32_t* out) { std::copy(at(t)->words.begin(), at(t)->words.end(), out); }
// The words changed since the last call, as first and last ranges' bounds and their number.
void pt_changed(void* t, size_t* out) {
  out[0] = out[1] = out[2] = 0;
  const auto& c = at(t)->changed;
  if (!c.empty()) out[0] = c.front().first, out[1] = c.back().second, out[2] = c.size();
  at(t)->settle();
}
}
