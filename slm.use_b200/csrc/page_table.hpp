// The host's copy of a paged cache's table: which pages a sequence has, how
// many tokens, and which sequences list a page.  Plain C++ (no CUDA), so that
// everything a kernel will index with is checked, and tested, without a GPU.
// A refused call throws std::invalid_argument and changes nothing.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

namespace slm {

inline void table_require(bool ok, const char* msg) {
  if (!ok) throw std::invalid_argument(msg);
}
inline void table_require(bool ok, const std::string& msg) {
  if (!ok) throw std::invalid_argument(msg);
}

inline size_t checked_mul(size_t a, size_t b) {
  size_t r;
  table_require(!__builtin_mul_overflow(a, b, &r), "paged: size overflows");
  return r;
}

inline size_t checked_add(size_t a, size_t b) {
  size_t r;
  table_require(!__builtin_add_overflow(a, b, &r), "paged: size overflows");
  return r;
}

class PageTable {
 public:
  PageTable(size_t seqs, size_t per, size_t page, size_t pages) : seqs(seqs), per(per), page(page), pages(pages) {
    table_require(seqs > 0 && seqs <= kSeqs, "table: 1 to 4096 sequences");
    table_require(per > 0 && page > 0 && checked_mul(per, page) < ((size_t)1 << 30), "table: bad pages per sequence");
    table_require(pages > 0 && pages < ((size_t)1 << 31), "table: bad number of pages");
    table_require(checked_add(seqs, checked_mul(seqs, per)) < ((size_t)1 << 32), "table: too many pages in all");
    words.assign(seqs + seqs * per, 0);
    held.assign(seqs, 0);
    uses.assign(pages, 0);
    listed.assign((pages + 63) / 64, 0);
  }

  const size_t seqs, per, page, pages;
  // lens[seqs], then ids[seqs][per]: the layout the kernels read.
  std::vector<uint32_t> words;
  std::vector<uint32_t> held;  // pages of each sequence
  std::vector<uint32_t> uses;  // sequences that list each page
  std::vector<uint64_t> listed;  // a bit per page: listed by any
  size_t shared = 0;           // pages listed by more than one
  // Ranges of words set since settle() (they may overlap).
  std::vector<std::pair<size_t, size_t>> changed;

  uint32_t len(size_t i) const { return words[i]; }
  const uint32_t* ids(size_t i) const { return words.data() + seqs + i * per; }
  void settle() { changed.clear(); }

  // What a device that holds `sent` lacks: words, or (hi > 0) a range to copy.
  // Words go in launch parameters, which the host never waits for (4352 of them:
  // 52 us of the host's time).  A large copy waits until the stream is idle (4 MB:
  // 0.4 ms behind an idle stream, 4.7 ms behind 4.4 ms of work); one of up to
  // kUnheld words does not, and takes no longer than words do (280 KB 33 us, 512
  // KB 50 us).  So no decode step waits: it changes kStep words at most, a length
  // and a page of every sequence there may be.
  static constexpr size_t kSeqs = 4096, kFew = 1920, kUnheld = 1 << 17, kStep = 2 * kSeqs;
  struct Update {
    std::vector<uint32_t> at, value;
    size_t lo = 0, hi = 0;
  };
  Update update(const std::vector<uint32_t>& sent) const {
    Update u;
    size_t lo = words.size(), hi = 0, marked = 0;
    for (const auto& c : changed) lo = std::min(lo, c.first), hi = std::max(hi, c.second), marked += c.second - c.first;
    const size_t most = hi - lo <= kUnheld ? kFew : kStep;
    u.at.reserve(std::min(marked, most + 1)), u.value.reserve(std::min(marked, most + 1));
    for (const auto& c : changed)
      for (size_t i = c.first; i < c.second && u.at.size() <= most; i++)
        if (words[i] != sent[i]) u.at.push_back((uint32_t)i), u.value.push_back(words[i]);
    if (u.at.size() > most) u.lo = lo, u.hi = hi;
    return u;
  }

  void assign(size_t seq, const uint32_t* list, size_t n) {
    table_require(list || n == 0, "table_assign: bad arguments");
    table_require(seq < seqs, "table_assign: no such sequence");
    table_require(n <= per, "table_assign: more pages than the table has room for");
    table_require(len(seq) <= n * page, "table_assign: the pages do not hold the sequence's length");
    uint32_t* row = words.data() + seqs + seq * per;
    size_t same = 0;  // a sequence that grew keeps its first pages
    while (same < n && same < held[seq] && row[same] == list[same]) same++;
    if (same == held[seq] && n - same <= 8) {  // a few pages more (a step of decoding): no sort
      for (size_t j = same; j < n; j++) {
        table_require(list[j] < pages, "table_assign: page id out of range");
        const uint32_t* from = uses[list[j]] ? list : list + same;  // listed by nobody: only here
        table_require(std::find(from, list + j, list[j]) == list + j, "table_assign: a page comes twice in one sequence");
      }
    } else {
      std::vector<uint32_t> sorted(list, list + n);
      std::sort(sorted.begin(), sorted.end());
      table_require(n == 0 || sorted.back() < pages, "table_assign: page id out of range");
      table_require(std::adjacent_find(sorted.begin(), sorted.end()) == sorted.end(),
                    "table_assign: a page comes twice in one sequence");
    }
    for (size_t j = same; j < held[seq]; j++) {
      const uint32_t id = row[j], left = --uses[id];
      shared -= left == 1;
      if (left == 0) listed[id / 64] &= ~((uint64_t)1 << id % 64);
    }
    for (size_t j = same; j < n; j++) {
      const uint32_t id = list[j];
      shared += ++uses[id] == 2;
      listed[id / 64] |= (uint64_t)1 << id % 64;
    }
    std::copy(list + same, list + n, row + same);
    held[seq] = (uint32_t)n;
    if (same < n) touch(seqs + seq * per + same, seqs + seq * per + n);
  }

  void set_lens(const uint32_t* lens, size_t n) {
    table_require(lens, "table_set_lens: bad arguments");
    table_require(n == seqs, "table_set_lens: one length per sequence");
    for (size_t i = 0; i < n; i++)
      if (lens[i] > held[i] * page)
        table_require(false, "table_set_lens: sequence " + std::to_string(i) + " has " + std::to_string(held[i]) +
                                 " pages, too few for " + std::to_string(lens[i]) + " tokens");
    size_t lo = n, hi = 0;  // one range: a step changes most lengths
    for (size_t i = 0; i < n; i++)
      if (words[i] != lens[i]) words[i] = lens[i], lo = std::min(lo, i), hi = i + 1;
    if (hi) touch(lo, hi);
  }

  void set_len(size_t i, uint32_t v) {
    if (words[i] == v) return;
    words[i] = v;
    touch(i, i + 1);
  }

  // The last m tokens of sequences first .. first + count - 1 may be written.
  void check_store(size_t first, size_t count, size_t m) const {
    table_require(first <= seqs && count <= seqs - first, "paged_store: no such sequences");
    table_require(m < ((size_t)1 << 31), "paged_store: too many tokens");
    if (!shared || !m) return;
    for (size_t i = first; i < first + count; i++)
      for (size_t j = (len(i) > m ? len(i) - m : 0) / page; j * page < len(i); j++)
        table_require(uses[ids(i)[j]] == 1, "paged_store: a page is listed by two sequences");
  }

  // At most `keep` tokens of each sequence may move to the pages of `to`.
  void check_evict(const PageTable& to, size_t keep, size_t sinks, size_t recent) const {
    table_require(this != &to, "paged_evict: the tables are one");
    table_require(seqs == to.seqs && page == to.page && pages == to.pages,
                  "paged_evict: the tables are of different sequences or pools");
    table_require(keep > 0 && keep < ((size_t)1 << 31), "paged_evict: bad budget");
    table_require(sinks <= keep && recent <= keep - sinks, "paged_evict: sinks and recent exceed the budget");
    for (size_t i = 0; i < seqs; i++)
      if (std::min<size_t>(len(i), keep) > to.held[i] * to.page)
        table_require(false, "paged_evict: sequence " + std::to_string(i) + " has too few pages to go to");
    table_require(to.shared == 0, "paged_evict: a page to go to is listed by two sequences");
    for (size_t w = 0; w < listed.size(); w++)
      table_require((listed[w] & to.listed[w]) == 0, "paged_evict: the tables have a page in common");
  }

 private:
  void touch(size_t a, size_t b) {
    if (!changed.empty() && changed.back().first <= a && a <= changed.back().second)
      changed.back().second = std::max(changed.back().second, b);
    else
      changed.emplace_back(a, b);
    if (changed.size() > kStep) {  // nobody has looked for long: one range for all
      size_t lo = words.size(), hi = 0;
      for (const auto& c : changed) lo = std::min(lo, c.first), hi = std::max(hi, c.second);
      changed.assign(1, {lo, hi});
    }
  }
};

}  // namespace slm
