// An eviction's search on the host, one slot after the other, with the
// library's own order, digits and rule of what counts
// (slm.use_b200/csrc/evict_order.hpp): the steps of the kernel.
#include <vector>

#include "../slm.use_b200/csrc/evict_order.hpp"

namespace {
template <bool ONE>
int search(const float* w, int n, int keep, int sinks, int recent, uint32_t* out) {
  using D = slm::Digits<ONE>;
  std::vector<uint32_t> order(n);
  for (int s = 0; s < n; s++) order[s] = s < sinks || s >= n - recent ? slm::kHeld : slm::order_of(w[s]);
  uint32_t prefix = 0;
  int need = keep - sinks - recent;
  if (need == 0) prefix = slm::kHeld - 1;
  for (int pass = 0; pass < D::kPasses && need; pass++) {
    const int shift = D::shift(pass), bits = D::bits(pass);
    std::vector<int> hist(D::kCount, 0);
    for (uint32_t o : order)
      if (pass == 0 ? o != slm::kHeld : slm::counts(o, prefix, shift + bits)) hist[o >> shift & ((1 << bits) - 1)]++;
    hist[(1 << bits) - 1] -= slm::held_counted<ONE>(sinks + recent, prefix, pass);
    int digit = D::kCount - 1;
    while (digit > 0 && hist[digit] < need) need -= hist[digit--];
    prefix |= (uint32_t)digit << shift;
    if (hist[digit] == need && prefix != 0) prefix -= 1, need = 0;
  }
  int count = 0, ties = 0;
  for (int s = 0; s < n; s++)
    if (order[s] > prefix || (order[s] == prefix && ties++ < need)) {
      if (count < keep) out[count] = (uint32_t)s;
      count++;
    }
  return count;
}
}  // namespace

extern "C" {
uint32_t ev_order(float w) { return slm::order_of(w); }
// The slots kept of n > keep, ascending; returns how many the rule keeps.
int ev_kept(int one, const float* w, int n, int keep, int sinks, int recent, uint32_t* out) {
  return one ? search<true>(w, n, keep, sinks, recent, out) : search<false>(w, n, keep, sinks, recent, out);
}
}
