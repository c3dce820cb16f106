// What an eviction's search compares: the order of the weights, the digits it
// looks at, and which slots it counts.  Plain C++ (no CUDA), so that the rule
// is tested without a GPU.
#pragma once

#include <stdint.h>
#include <string.h>

#ifdef __CUDACC__
#define SLM_BOTH __host__ __device__ __forceinline__
#else
#define SLM_BOTH inline
#endif

namespace slm {

// Order of the weights as unsigned integers from 1 on: NaN lowest, the two
// zeros equal.  0 stands for no slot, kHeld for one that does not compete.
constexpr uint32_t kHeld = 0xffffffffu;
SLM_BOTH uint32_t order_of(float w) {
  if (w != w) return 1;
  w += 0.0f;
  uint32_t b;
  memcpy(&b, &w, sizeof b);
  return (b & 0x80000000u ? ~b : b | 0x80000000u) + 1;
}

// A CTA alone searches four digits of 8 bits, a cluster digits of 11, 11 and 10.
template <bool ONE>
struct Digits {
  static constexpr int kPasses = ONE ? 4 : 3, kCount = ONE ? 256 : 2048;
  static constexpr int kTop = ONE ? 24 : 21;  // the lowest bit of the first digit
  static SLM_BOTH int shift(int pass) { return ONE ? 24 - 8 * pass : pass == 0 ? 21 : pass == 1 ? 10 : 0; }
  static SLM_BOTH int bits(int pass) { return ONE ? 8 : pass == 2 ? 10 : 11; }
};

// Whether a slot of order o counts after the first pass: its digits above `bit`
// are those of `prefix`.
SLM_BOTH bool counts(uint32_t o, uint32_t prefix, int bit) { return (o ^ prefix) >> bit == 0; }

// How many of the `held` slots counted with them, all at the largest digit,
// though they do not compete.  With 11 bits no weight's first digit is theirs;
// with 8 bits it is from just below 2^127 up to +inf.  (Left out slot by slot
// they took 18 registers more, and 2000 sequences of 300 took 312 us, not 260.)
template <bool ONE>
SLM_BOTH int held_counted(int held, uint32_t prefix, int pass) {
  using D = Digits<ONE>;
  return ONE && pass > 0 && counts(kHeld, prefix, D::shift(pass) + D::bits(pass)) ? held : 0;
}

}  // namespace slm
