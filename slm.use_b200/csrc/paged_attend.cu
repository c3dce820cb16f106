// Attention of one new token per sequence over a paged key-value cache.
//
//   p_s = exp(x_s - max x) / Σ exp(x - max x),  x_s = scale · q·k_s,  y = Σ p_s v_s
//
// over the visible slots, in one pass: every warp keeps a running reference
// maximum m, the sum l of exp(x - m) and the sum of exp(x - m) v, all f32.
// Keys and values are read once for every 8 query heads of a key head, so bytes
// bound the call (but for many wide heads, see Shape); the rest is arranged to
// stay under them.
//
// Work: the visible slots of every pair, a (sequence, tile of up to 8 query
// heads of one key head), lie one after the other and are shared evenly over
// all warps that fit on the GPU at once, whatever the sequences' lengths; a
// warp works alone, and a second kernel joins the pieces of cut pairs in order,
// so results do not depend on timing.  Where all pairs are short, a CTA's four
// warps share one and join it themselves.
//
// Data: a warp streams its tiles through two to four private buffers with
// 16-byte asynchronous copies, which look every row's page up (a page may end
// anywhere in a tile) and fill rows past the end and columns past the head
// size with zeros.  8 to 12 warps an SM (4 at 256-wide f32 heads) keep 64
// to 144 KB in flight.
//
// Products: mma.m16n8k8 on tf32, with the group's heads as rows.  Operands of
// f32 precision are split into two tf32 parts, x = hi + lo: of the 16 rows, 8
// hold the heads' hi parts and 8 their lo parts, so one product per part of
// the other operand gives all four partial products, and a row pair's sum is
// the result.  Two parts keep 22 of f32's 24 bits; three would leave room for 5
// heads and take three products.  Errors against 64 bits on f32 pages (in
// brackets those of plain f32, 64-wide heads): 0.8e-7 of one token (0), 2.0e-7
// of 8 (1.6e-7), 2.8e-7 of 97 (2.9e-7), 2.9e-7 of 16389 (4.3e-7).  bf16 keys and
// values are tf32 values as they are: one product, errors of 0 to 2.0e-7.  The
// tensor cores do in this form what the CUDA cores would do in 8 times the
// instructions.  With heads as rows a tcgen05 tile (64 or 128 of them) would be
// mostly empty; slots as its rows and heads times parts as columns would fill
// it, which is not built.
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"
#include "paged.cuh"

namespace slm {

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32, kHeads = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.0f;     // scores (log2 units) may exceed m by this before m moves
constexpr int kWeightKeys = 256;  // slots whose weights a CTA adds at once

// Where a launch keeps what its warps hand one another.
struct Scratch {
  float* part;       // [taker][2][heads of a tile][dh]: sums of pieces of cut (sequence, tile)s
  float* part_ml;    // [taker][2][kHeads][2]: their m and l
  float* stat;       // [n][heads][2]: final m and 1 / l, or null
  float* score;      // per sequence [heads][visible rounded up to 4], log2 units; or null
  uint32_t piece;    // floats of a piece's sums
};

__host__ __device__ inline int visible_of(uint32_t len, long long reach) {
  return reach && (long long)len > reach ? (int)reach : (int)len;
}

// Slots of a warp's tile, its buffers, and CTAs an SM, by page type and head
// size (rounded up to the next one listed: rows in shared memory are multiples
// of 128 bytes).  K and V of a tile take 6 to 16 KB.  Measured (us): at 64, three
// CTAs with two buffers against two with three, 37.5 / 38.5 for 64 ragged f32
// sequences and 13.4 / 14.7 for one of 16389; at 128, where three CTAs leave 168
// registers, two against three, 172 / 175 for 48 ragged bf16 sequences; 8-slot
// tiles at bf16 128, 187; f32 96 and 192 by themselves against rounded up to 128
// and 256, 93 / 105 for 34 sequences of 2393 and 29 / 34 for 8 of 4000.
struct Config {
  int dh, keys, stages, ctas;
};
constexpr int kMaxCtas = 3;
constexpr Config kF32[] = {{32, 16, 3, 3}, {64, 16, 2, 3}, {96, 8, 3, 3}, {128, 8, 3, 2}, {192, 8, 2, 2}, {256, 8, 2, 1}};
constexpr Config kBf16[] = {{64, 32, 2, 3}, {128, 16, 3, 2}, {192, 8, 4, 2}, {256, 8, 2, 2}};
// The first that a head size fits into.
constexpr Config config_of(bool bf16, int dh) {
  const Config* c = bf16 ? kBf16 : kF32;
  while (c->dh < dh) c++;
  return *c;
}
template <bool BF16, int DH>
struct Shape {
  static constexpr Config kCfg = config_of(BF16, DH);
  static_assert(kCfg.dh == DH && kCfg.ctas <= kMaxCtas, "configuration");
  static constexpr int kRow = DH * (BF16 ? 2 : 4);   // bytes of a row in shared memory
  static constexpr int kKeys = kCfg.keys;
  static constexpr int kStages = kCfg.stages;
  static constexpr int kTile = kKeys * kRow;         // K (or V) bytes of a tile
  static constexpr int kWarp = kStages * 2 * kTile;  // bytes of a warp's buffers
  static constexpr bool kQShared = DH > 192;         // q in shared memory, for a CTA: registers hold the sums
  // 16-byte pieces of q that stay in registers all the same: where q is shared
  // half of it for bf16 pages, whose rows are read twice as fast (24 ragged
  // sequences, 16 query heads of 256: 29.7 us against 32.1).
  static constexpr int kQHeld = !kQShared ? kRow / 64 : BF16 ? kRow / 128 : 0;
  static constexpr int kSmem = kWarps * kWarp + (kRow / 64 - kQHeld) * (BF16 ? 4 : 2) * 512;
  static constexpr int kCtas = kCfg.ctas;
  static_assert(kRow % 128 == 0 && kKeys % 8 == 0 && kKeys <= 32, "swizzles and look-ups");
};

__device__ __forceinline__ void copy16(uint32_t dst, const char* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// 16 bytes, or zeros and no read.
__device__ __forceinline__ void copy16(uint32_t dst, const char* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a));
  return r;
}

__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2_of(float x) {  // relative error 2^-22; 0 below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The upper 11 significant bits of x, and the rest, of which the tensor core
// reads the upper 11 in turn: half a step is added, so that x is kept to 2^-22
// without a bias (without it errors were 1.5 times as large).
__device__ __forceinline__ uint32_t hi_of(uint32_t x) { return x & 0xffffe000u; }
__device__ __forceinline__ uint32_t lo_of(uint32_t x) {
  return __float_as_uint(__uint_as_float(x) - __uint_as_float(hi_of(x))) + 0x1000u;
}
// The same with both parts rounded to nearest (operands that are split once).
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = (__float_as_uint(x - __uint_as_float(hi)) + 0x1000u) & 0xffffe000u;
}

// c += a · (two values of the other operand, for two columns of a): value j of
// w0 and of w1 (f32), or the two bf16 halves of one word each.
template <bool BF16>
struct Operand;
template <>
struct Operand<false> {
  static __device__ __forceinline__ void mul(float* c, const uint32_t* a, uint32_t x0, uint32_t x1) {
    mma(c, a, hi_of(x0), hi_of(x1));
    mma(c, a, lo_of(x0), lo_of(x1));
  }
};
template <>
struct Operand<true> {
  static __device__ __forceinline__ void mul(float* c, const uint32_t* a, uint32_t x0, uint32_t x1) { mma(c, a, x0, x1); }
};

// How a launch's work is laid out.  Every pair, a (sequence, tile of up to 8
// query heads of one key head), has ⌈visible / keys⌉ blocks of `keys` slots.
// Pairs lie one after the other in units: `extra` (what beginning a pair costs,
// in blocks) plus its blocks; with whole = true a pair is one unit, never cut.
// A taker is a warp, or (by_cta) a CTA whose warps take blocks in turn.
struct Work {
  uint32_t keys, extra;
  uint32_t takers;              // warps (CTAs if by_cta) that share the units:
  uint32_t each, more;          // `each` and one more for the first `more`
  int tiles;                    // pairs of a sequence
  bool whole, by_cta;
  bool direct;                  // the sequence of a unit follows from its number: one sequence, or all with `tiles` units
  __host__ __device__ uint32_t blocks_of(uint32_t visible) const { return (visible + keys - 1) / keys; }
  __host__ __device__ uint32_t units_of(uint32_t visible) const {  // of a pair
    return visible == 0 ? 0 : whole ? 1 : blocks_of(visible) + extra;
  }
  __device__ uint32_t first_unit(uint32_t w) const { return w * each + min(w, more); }
  __device__ uint32_t taker_of(uint32_t unit) const {
    const uint32_t longer = more * (each + 1);
    return unit < longer ? unit / (each + 1) : more + (unit - longer) / each;
  }
};

// Finds the sequence that holds unit `at` (every warp for itself) and what lies
// before it.
struct Place {
  int seq, len, visible;
  uint32_t unit;       // at, counted from the sequence's first unit
  long long slots;     // visible slots of the sequences before it, each rounded up to 4
  __device__ __forceinline__ void read(const PagedTable& t, long long reach) {
    len = (int)t.lens[seq];
    visible = visible_of(len, reach);
  }
};
__device__ __forceinline__ Place locate(const PagedTable& t, long long reach, const Work& wk, uint32_t at) {
  if (wk.direct) {
    const int seq = t.n == 1 ? 0 : at / wk.tiles;
    Place p{seq, 0, 0, at - seq * wk.tiles, 0};
    p.read(t, reach);
    return p;
  }
  const int lane = threadIdx.x & 31, each = (t.n + 31) / 32;
  uint32_t mine = 0;
  long long slots = 0;
#pragma unroll 4
  for (int j = 0; j < each; j++) {
    const int i = lane * each + j;
    const uint32_t v = i < t.n ? visible_of(t.lens[i], reach) : 0;
    mine += wk.units_of(v) * wk.tiles, slots += (v + 3) & ~3u;
  }
  uint32_t upto = mine;
  long long slots_upto = slots;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, upto, o);
    const long long b = __shfl_up_sync(0xffffffffu, slots_upto, o);
    if (lane >= o) upto += a, slots_upto += b;
  }
  const int src = __ffs(__ballot_sync(0xffffffffu, upto > at)) - 1;
  Place p{src * each, 0, 0, at - __shfl_sync(0xffffffffu, upto - mine, src),
          __shfl_sync(0xffffffffu, slots_upto - slots, src)};
  for (;; p.seq++) {
    p.read(t, reach);
    const uint32_t n = wk.units_of(p.visible) * wk.tiles;
    if (p.unit < n) return p;
    p.unit -= n, p.slots += (p.visible + 3) & ~3;
  }
}

template <bool BF16, int DH>
__global__ void __launch_bounds__(kThreads, Shape<BF16, DH>::kCtas)
    k_paged_attend(const __grid_constant__ PagedAttendArgs a, const __grid_constant__ Scratch sc,
                   const __grid_constant__ Work wk, bool idle, bool q16) {
  constexpr int SIZE = BF16 ? 2 : 4;
  using S = Shape<BF16, DH>;
  constexpr int kSteps = DH / 8;            // k-steps of q·k, and 8-column tiles of p·v
  constexpr int kLoad = BF16 ? 4 : 2;       // k-steps that a 16-byte piece of a key row feeds
  constexpr int kPieces = S::kRow / 16;     // 16-byte pieces of a row
  constexpr int kKeys = S::kKeys, kStages = S::kStages;
  constexpr int kSum = DH + 4;               // floats of a head's sums in shared memory
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float s_m[kWarps][kHeads], s_l[kWarps][kHeads];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group = a.heads / a.key_heads, per_key = (group + kHeads - 1) / kHeads;
  const uint32_t mine = (uint32_t)__cvta_generic_to_shared(smem) + warp * S::kWarp;
  unsigned char* q_shared = smem + kWarps * S::kWarp;
  const uint32_t q_at = (uint32_t)__cvta_generic_to_shared(q_shared) + lane * 16;
  const char *K = static_cast<const char*>(a.k), *V = static_cast<const char*>(a.v);
  const int row_bytes = a.dh * SIZE, pieces = row_bytes / 16;

  dependency_wait();
  dependents_launch();
  if (idle)  // rows of idle sequences: zeros
    for (int i = blockIdx.x; i < a.t.n; i += gridDim.x)
      if (a.t.lens[i] == 0)
        for (int e = threadIdx.x; e < a.heads * a.dh; e += kThreads) a.y[(size_t)i * a.heads * a.dh + e] = 0.0f;
  // This taker's units, and where they begin.
  const bool by_cta = S::kQShared || wk.by_cta;
  const uint32_t w = by_cta ? blockIdx.x : blockIdx.x * kWarps + warp;
  if (w >= wk.takers) return;
  const int turn = by_cta ? warp : 0, turns = by_cta ? kWarps : 1;
  const uint32_t begin = wk.first_unit(w);
  uint32_t left = wk.first_unit(w + 1) - begin;
  Place at = locate(a.t, a.reach, wk, begin);

  while (left) {
    // A segment: blocks b0 .. b1-1 of the pair's n_blocks.
    const uint32_t n_blocks = wk.blocks_of(at.visible), n_units = wk.units_of(at.visible);
    const int tile = at.unit / n_units;
    const uint32_t u0 = at.unit - tile * n_units, u1 = min(n_units, u0 + left), skip = wk.extra;
    const uint32_t b0 = u0 > skip ? u0 - skip : 0, b1 = wk.whole ? n_blocks : u1 > skip ? u1 - skip : 0;
    left -= u1 - u0;
    at.unit += u1 - u0;
    if (b0 < b1) {
    const int kh = tile / per_key, head0 = kh * group + (tile % per_key) * kHeads;
    const int heads = min(kHeads, (kh + 1) * group - head0);
    const int lo = at.len - at.visible;
    const int first = lo + b0 * kKeys, end = lo + min((uint32_t)at.visible, b1 * kKeys);
    const uint32_t* ids = a.t.ids + (size_t)at.seq * a.t.per;
    const int n_tiles = ((int)(b1 - b0) - turn + turns - 1) / turns;  // this warp's blocks
    auto key_of = [&](int j) { return first + (j * turns + turn) * kKeys; };

    // The pool row that this lane looks up for tile j.
    auto look_up = [&](int j) -> uint32_t {  // j < n_tiles
      const uint32_t s = min(key_of(j) + lane % kKeys, end - 1);
      const uint32_t page = a.t.page_of(s);
      return (ids[page] * a.key_heads + kh) * a.t.page + (s - page * a.t.page);
    };
    auto load = [&](int buffer, int n, uint32_t row) {  // n slots
      const uint32_t to = mine + buffer * (2 * S::kTile);
      const bool whole = n >= kKeys && row_bytes == S::kRow;
#pragma unroll
      for (int u = 0; u < kKeys * kPieces / 32; u++) {
        const int r = (u * 32 + lane) / kPieces, c = (u * 32 + lane) % kPieces;
        const uint64_t from = (uint64_t)__shfl_sync(0xffffffffu, row, r) * (uint32_t)row_bytes + c * 16;
        // Swizzles under which the reads below hit every bank once.
        const uint32_t kd = to + r * S::kRow + ((c ^ ((r & 1) << 2)) << 4);
        const uint32_t vd = to + S::kTile + r * S::kRow + ((c ^ (r & 6)) << 4);
        if (whole) {
          copy16(kd, K + from);
          copy16(vd, V + from);
        } else {
          const bool ok = r < n && c < pieces;
          copy16(kd, ok ? K + from : K, ok);
          copy16(vd, ok ? V + from : V, ok);
        }
      }
    };

    uint32_t row = look_up(0), row1 = n_tiles > 1 ? look_up(1) : 0;  // of the next tiles to load
    int in = 0, out = 0;  // buffers
    auto load_next = [&](int next) {
      if (next < n_tiles) {
        load(in, end - key_of(next), row);
        row = row1;
        if (next + 2 < n_tiles) row1 = look_up(next + 2);
      }
      copies_commit();
      in = in + 1 == kStages ? 0 : in + 1;
    };
    // q, scaled to log2 units and split, in the order the key rows are read:
    // rows g and g + 8 of the left operand are head g's hi and lo parts.
    uint32_t qa[S::kQHeld ? S::kQHeld * kLoad : 1][4];
    {
      const float* q = a.q + at.seq * a.ldq + (size_t)(head0 + g) * a.dh;
      auto read = [&](int i, float* v) {
        const int d = i * (kLoad * 8) + t * (kLoad * 2);
        const bool ok = g < heads && d < a.dh;  // dh is a multiple of 8
#pragma unroll
        for (int e = 0; e < kLoad * 2; e += 4) {
          float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (ok && q16)
            x = *reinterpret_cast<const float4*>(q + d + e);
          else if (ok)
            x = make_float4(q[d + e], q[d + e + 1], q[d + e + 2], q[d + e + 3]);
          v[e] = x.x, v[e + 1] = x.y, v[e + 2] = x.z, v[e + 3] = x.w;
        }
      };
      auto parts = [&](const float* v, int e, uint32_t* to) {
        split(v[2 * e] * (a.scale * kLog2e), to[0], to[1]);
        split(v[2 * e + 1] * (a.scale * kLog2e), to[2], to[3]);
      };
      // Read first, split when the first tiles' copies are on their way.  Shared:
      // the pieces that stay in registers, and every fourth of the others.
      constexpr int kRead = S::kQHeld + (S::kQShared ? (kSteps / kLoad - S::kQHeld) / kWarps : 0);
      float qr[kRead][kLoad * 2];
#pragma unroll
      for (int i = 0; i < kRead; i++) read(i < S::kQHeld ? i : S::kQHeld + (i - S::kQHeld) * kWarps + warp, qr[i]);
#pragma unroll 1
      for (int j = 0; j < kStages - 1; j++) load_next(j);
#pragma unroll
      for (int i = 0; i < kRead; i++)
#pragma unroll
        for (int e = 0; e < kLoad; e++) {
          if (i < S::kQHeld) {
            parts(qr[i], e, qa[i < S::kQHeld ? i * kLoad + e : 0]);
          } else {
            uint32_t to[4];
            parts(qr[i], e, to);
            *reinterpret_cast<uint4*>(q_shared + (((i - S::kQHeld) * kWarps + warp) * kLoad + e) * 512 + lane * 16) =
                make_uint4(to[0], to[1], to[2], to[3]);
          }
        }
    }

    if (S::kQShared) __syncthreads();
    float m = -INFINITY, l = 0.0f, o[kSteps][2];
#pragma unroll
    for (int s = 0; s < kSteps; s++) o[s][0] = o[s][1] = 0.0f;
    float* score = sc.score && g < heads
                       ? sc.score + at.slots * a.heads + (size_t)(head0 + g) * ((at.visible + 3) & ~3) - lo
                       : nullptr;

#pragma unroll 1
    for (int j = 0; j < n_tiles; j++) {
      copies_wait<kStages - 2>();
      __syncwarp();  // every lane's copies of this tile have landed, and all are done with the last one
      load_next(j + kStages - 1);

      const uint32_t kt = mine + out * (2 * S::kTile), vt = kt + S::kTile;
      out = out + 1 == kStages ? 0 : out + 1;
      const int key0 = key_of(j);
      constexpr int kBlocks = kKeys / 8;
      constexpr int kChains = BF16 ? 2 : 4;  // independent sums: products overlap, and short chains truncate little
      float x[kBlocks][2], c[kBlocks][kChains][4];
#pragma unroll
      for (int b = 0; b < kBlocks; b++)
#pragma unroll
        for (int e = 0; e < kChains; e++) c[b][e][0] = c[b][e][1] = c[b][e][2] = c[b][e][3] = 0.0f;
      const uint32_t krow = kt + g * S::kRow + t * 16;
      const int odd = (g & 1) * 64;
#pragma unroll
      for (int i = 0; i < kSteps / kLoad; i++) {
        uint4 kw[kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; b++) kw[b] = lds16(krow + b * 8 * S::kRow + i * 64 + (i & 1 ? -odd : odd));
#pragma unroll
        for (int e = 0; e < kLoad; e++) {
          const int s = i * kLoad + e;
          uint32_t qs[4];
          if (i >= S::kQHeld) {
            const uint4 qw = lds16(q_at + (s - S::kQHeld * kLoad) * 512);
            qs[0] = qw.x, qs[1] = qw.y, qs[2] = qw.z, qs[3] = qw.w;
          }
          const uint32_t* qv = i >= S::kQHeld ? qs : qa[i >= S::kQHeld ? 0 : s];
#pragma unroll
          for (int b = 0; b < kBlocks; b++) {
            const uint32_t v[4] = {kw[b].x, kw[b].y, kw[b].z, kw[b].w};
            if (BF16)
              Operand<BF16>::mul(c[b][s % kChains], qv, v[e] << 16, v[e] & 0xffff0000u);
            else
              Operand<BF16>::mul(c[b][s % kChains], qv, v[e * 2], v[e * 2 + 1]);
          }
        }
      }
#pragma unroll
      for (int b = 0; b < kBlocks; b++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float sum = 0.0f;
#pragma unroll
          for (int ch = 0; ch < kChains; ch++) sum += c[b][ch][e] + c[b][ch][e + 2];
          x[b][e] = sum;
        }
        const int s = key0 + b * 8 + 2 * t;
        if (key0 + kKeys > end) {
          if (s >= end) x[b][0] = -INFINITY;
          if (s + 1 >= end) x[b][1] = -INFINITY;
        }
        // In pairs: rows are padded, and a block ends at an odd slot only at the row's end.
        if (score && s < end) *reinterpret_cast<float2*>(score + s) = make_float2(x[b][0], x[b][1]);
      }
      float top = x[0][0];
#pragma unroll
      for (int b = 0; b < kBlocks; b++) top = fmaxf(top, fmaxf(x[b][0], x[b][1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // m moves only when a score passes it by kLazy (the first tile: from -inf).
      if (__any_sync(0xffffffffu, top > m + kLazy)) {
        const float to = top > m + kLazy ? top : m;
        const float keep = to == m ? 1.0f : exp2_of(m - to);
        m = to, l *= keep;
#pragma unroll
        for (int s = 0; s < kSteps; s++) o[s][0] *= keep, o[s][1] *= keep;
      }
      uint32_t p[kBlocks][4];
#pragma unroll
      for (int b = 0; b < kBlocks; b++) {
        const float p0 = exp2_of(x[b][0] - m), p1 = exp2_of(x[b][1] - m);
        l += p0 + p1;
        split(p0, p[b][0], p[b][1]);
        split(p1, p[b][2], p[b][3]);
      }
      // A tile's products in sums of their own: the tensor core truncates when it
      // accumulates, and over thousands of tokens that drifts (a relative error of
      // 8e-6 against 4e-7 after 3500 tokens a warp).
      const uint32_t vrow = vt + 2 * t * S::kRow + ((g ^ (2 * t)) << 4);
#pragma unroll
      for (int i = 0; i < S::kRow / 128; i++) {
        constexpr int kOf = BF16 ? 8 : 4;  // 8-column tiles a 16-byte piece feeds
        float f[kOf][4];
#pragma unroll
        for (int e = 0; e < kOf; e++) f[e][0] = f[e][1] = f[e][2] = f[e][3] = 0.0f;
#pragma unroll
        for (int b = 0; b < kBlocks; b++) {
          const uint4 w0 = lds16(vrow + b * 8 * S::kRow + i * 128), w1 = lds16(vrow + (b * 8 + 1) * S::kRow + i * 128);
          const uint32_t v0[4] = {w0.x, w0.y, w0.z, w0.w}, v1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
          for (int e = 0; e < 4; e++) {
            if (BF16) {
              Operand<BF16>::mul(f[e * 2], p[b], v0[e] << 16, v1[e] << 16);
              Operand<BF16>::mul(f[e * 2 + 1], p[b], v0[e] & 0xffff0000u, v1[e] & 0xffff0000u);
            } else {
              Operand<BF16>::mul(f[e], p[b], v0[e], v1[e]);
            }
          }
        }
        // The rows' hi and lo parts of a head are added here.
#pragma unroll
        for (int e = 0; e < kOf; e++)
          o[i * kOf + e][0] += f[e][0] + f[e][2], o[i * kOf + e][1] += f[e][1] + f[e][3];
      }
    }
    __syncwarp();  // all lanes are done with the buffers
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);

    // The sums of this taker's share of the pair: all of it, or a piece to be
    // joined with others (a taker cuts at most two pairs, the one it continues
    // and the one it begins).  A CTA's warps are joined in shared memory first.
    const bool all = b1 - b0 == n_blocks;
    const size_t slot = 2 * (size_t)w + (b0 == 0);
    const float r = all && !by_cta ? 1.0f / l : 1.0f;
    float* dst = all ? a.y + ((size_t)at.seq * a.heads + head0) * a.dh : sc.part + slot * sc.piece;
    float* ml = !all ? sc.part_ml + slot * kHeads * 2
                     : sc.stat ? sc.stat + 2 * ((size_t)at.seq * a.heads + head0) : nullptr;
    float* to = by_cta ? reinterpret_cast<float*>(smem + warp * S::kWarp) + g * kSum : dst + g * a.dh;
    if (g < heads) {
      constexpr int kWide = BF16 ? 8 : 4;  // columns of a 16-byte piece: lane t holds 2 · kWide in a row
#pragma unroll
      for (int i = 0; i < kSteps / kWide; i++)
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
          for (int c = 0; c < kWide; c += 4) {
            const int d = i * (kWide * 8) + (2 * t + e) * kWide + c;
            float v[4];
#pragma unroll
            for (int f = 0; f < 4; f++) v[f] = o[i * kWide + c + f][e] * r;
            if (d < a.dh) *reinterpret_cast<float4*>(to + d) = make_float4(v[0], v[1], v[2], v[3]);
          }
      if (t == 0 && by_cta)
        s_m[warp][g] = m, s_l[warp][g] = l;
      else if (t == 0 && ml)
        ml[2 * g] = m, ml[2 * g + 1] = all ? r : l;
    }
    if (by_cta) {
      __syncthreads();
      for (int h = warp; h < heads; h += kWarps) {
        float M = s_m[0][h], L = 0.0f, f[kWarps];
#pragma unroll
        for (int x = 1; x < kWarps; x++) M = fmaxf(M, s_m[x][h]);
#pragma unroll
        for (int x = 0; x < kWarps; x++) {
          f[x] = s_l[x][h] == 0.0f ? 0.0f : exp2_of(s_m[x][h] - M);  // 0: a warp without blocks
          L += s_l[x][h] * f[x];
        }
        const float norm = all ? 1.0f / L : 1.0f;
        for (int d = lane; d < a.dh; d += 32) {
          float v = 0.0f;
#pragma unroll
          for (int x = 0; x < kWarps; x++) v += reinterpret_cast<float*>(smem + x * S::kWarp)[h * kSum + d] * f[x];
          dst[h * a.dh + d] = v * norm;
        }
        if (ml && lane == 0) ml[2 * h] = M, ml[2 * h + 1] = all ? norm : L;
      }
      __syncthreads();  // before the next pair's copies
    }
    }
    // On to the next pair or the next sequence with tokens.
    while (left && at.unit >= wk.tiles * wk.units_of(at.visible)) {
      at.unit = 0, at.slots += (at.visible + 3) & ~3;
      at.seq++, at.read(a.t, a.reach);
    }
  }
}

// Four floats through L2, or zeros and no read; no branch, so that several are
// on their way at once.
__device__ __forceinline__ float4 load_if(const float* p, bool ok) {
  float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %5, 0;\n @p ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];\n}\n"
               : "+f"(r.x), "+f"(r.y), "+f"(r.z), "+f"(r.w)
               : "l"(p), "r"((int)ok));
  return r;
}

// (M, L) := the maximum and the sum of exp2(x - maximum) of two sets of scores.
__device__ __forceinline__ void merge(float& M, float& L, float m, float l) {
  const float to = fmaxf(M, m);
  L = (M == -INFINITY ? 0.0f : L * exp2_of(M - to)) + (m == -INFINITY ? l : l * exp2_of(m - to));
  M = to;
}
__device__ __forceinline__ void merge_warp(float& M, float& L) {
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) {
    const float m = __shfl_xor_sync(0xffffffffu, M, x), l = __shfl_xor_sync(0xffffffffu, L, x);
    merge(M, L, m, l);
  }
}

// The pair that holds unit `at` of taker `taker` is cut between w0 and w1.
struct Pieces {
  uint32_t w0, w1;
  // Piece c of the pair: the first taker's second slot, then the others' first ones.
  __device__ size_t slot_of(int c) const { return 2 * (size_t)(w0 + c) + (c == 0); }
  __device__ size_t slot_of(int c, int h) const { return slot_of(c) * kHeads + h; }
  __device__ int count() const { return w1 - w0 + 1; }
};
__device__ __forceinline__ Pieces pieces_of(const Work& wk, uint32_t origin, uint32_t blocks) {
  if (wk.whole) return Pieces{0, 0};
  return Pieces{wk.taker_of(origin + wk.extra), wk.taker_of(origin + wk.extra + blocks - 1)};
}
// First unit of a sequence (every warp for itself).
__device__ __forceinline__ uint32_t first_unit_of(const PagedTable& t, long long reach, const Work& wk,
                                                  int seq) {
  uint32_t before = 0;
  for (int i = threadIdx.x & 31; i < seq; i += 32) before += wk.units_of(visible_of(t.lens[i], reach));
  return __reduce_add_sync(0xffffffffu, before) * wk.tiles;
}

// Joins the pieces of cut pairs, a CTA per head of one.  Where there are fewer
// pairs than takers, `x` counts them; else it counts the takers, and the first
// taker of a cut pair joins it.
constexpr int kMaxTakers = 148 * kMaxCtas * kWarps;  // and pieces of a pair
template <int kJoin>
__device__ void join(const PagedAttendArgs& a, const Scratch& sc, const Work& wk, bool by_pair,
                     uint32_t x0, int y0) {
  __shared__ __align__(16) float s_sum[kJoin * 4];  // stored four at a time
  __shared__ float s_factor[kMaxTakers], s_red[2][kJoin / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = a.heads / a.key_heads, per_key = (group + kHeads - 1) / kHeads;
  int seq, tile;
  uint32_t origin, n;  // the pair's first unit, and its blocks
  if (by_pair) {
    seq = x0 / wk.tiles, tile = x0 % wk.tiles;
    const uint32_t visible = visible_of(a.t.lens[seq], a.reach);
    n = wk.blocks_of(visible);
    origin = first_unit_of(a.t, a.reach, wk, seq) + tile * wk.units_of(visible);
  } else {
    // The pair that holds the last unit of taker x0.
    const uint32_t at = wk.first_unit(x0 + 1) - 1;
    const Place p = locate(a.t, a.reach, wk, at);
    n = wk.blocks_of(p.visible);
    seq = p.seq, tile = p.unit / wk.units_of(p.visible);
    origin = at - (p.unit - tile * wk.units_of(p.visible));
  }
  dependency_wait();  // every CTA: that this kernel is done says that the one before it is
  if (n == 0) return;
  const Pieces pc = pieces_of(wk, origin, n);
  const int kh = tile / per_key, head = tile % per_key * kHeads + y0;  // of the key head's
  if (pc.w0 == pc.w1 || (!by_pair && pc.w0 != x0) || head >= group) return;
  const int parts = pc.count();

  // Threads of a group take 4 columns each, groups every so-manieth piece; the
  // first pieces are on their way while the factors are worked out.
  constexpr int kAtOnce = 8;
  const int cols = a.dh / 4, groups = kJoin / cols, mine = min(tid / cols, groups - 1), d = tid % cols * 4;
  float4 x[kAtOnce], v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto fetch = [&](int c) {
#pragma unroll
    for (int u = 0; u < kAtOnce; u++)
      x[u] = load_if(sc.part + pc.slot_of(c + u * groups) * sc.piece + y0 * a.dh + d, c + u * groups < parts);
  };
  fetch(mine);

  // M and l of the pieces, and each piece's factor.
  float M = -INFINITY, L = 0.0f;
  for (int c = tid; c < parts; c += kJoin) {
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(sc.part_ml) + pc.slot_of(c, y0));
    s_factor[c] = ml.x;
    merge(M, L, ml.x, ml.y);
  }
  merge_warp(M, L);
  if (lane == 0) s_red[0][warp] = M, s_red[1][warp] = L;
  __syncthreads();
  M = s_red[0][0], L = s_red[1][0];
#pragma unroll
  for (int w = 1; w < kJoin / 32; w++) merge(M, L, s_red[0][w], s_red[1][w]);
  for (int c = mine;;) {
#pragma unroll
    for (int u = 0; u < kAtOnce; u++) {
      const int p = c + u * groups;
      const float f = p < parts ? exp2_of(s_factor[min(p, parts - 1)] - M) : 0.0f;
      v.x = fmaf(x[u].x, f, v.x), v.y = fmaf(x[u].y, f, v.y), v.z = fmaf(x[u].z, f, v.z), v.w = fmaf(x[u].w, f, v.w);
    }
    c += groups * kAtOnce;
    if (c >= parts) break;
    fetch(c);
  }
  if (tid < groups * cols) *reinterpret_cast<float4*>(&s_sum[mine * a.dh + d]) = v;
  __syncthreads();
  const size_t row = (size_t)seq * a.heads + kh * group + head;
  for (int e = tid; e < a.dh; e += kJoin) {
    float sum = 0.0f;
    for (int w = 0; w < groups; w++) sum += s_sum[w * a.dh + e];
    a.y[row * a.dh + e] = sum / L;
  }
}

// weight[s] += Σ_h p_s over the key head's query heads, from the kept scores:
// `slots` slots (kWeightKeys at a time) of one key head and sequence, after M
// and 1 / l of its heads, kStats at a time, from the pieces or, of a pair that was not cut, as
// kept.
constexpr int kStats = 32;
template <int kThreads_>
__device__ void add_weights(const PagedAttendArgs& a, const Scratch& sc, const Work& wk, uint32_t x0, int slots) {
  __shared__ float s_stat[kStats][2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kh = x0 % a.key_heads, group = a.heads / a.key_heads, per_key = (group + kHeads - 1) / kHeads;
  const Place at =
      locate(a.t, a.reach, Work{(uint32_t)slots, 0, 0, 0, 0, 1, false, false, false}, x0 / a.key_heads);
  const uint32_t n = wk.blocks_of(at.visible), n_units = wk.units_of(at.visible);
  const uint32_t origin = first_unit_of(a.t, a.reach, wk, at.seq) + kh * per_key * n_units;
  const int padded = (at.visible + 3) & ~3, end = min(at.visible, (int)(at.unit + 1) * slots);
  const float* score = sc.score + at.slots * a.heads + (size_t)kh * group * padded;
  constexpr int kEach = kWeightKeys / kThreads_;
  for (int v0 = at.unit * slots + tid; v0 - tid < end; v0 += kWeightKeys) {
    const bool begins = v0 - tid == (int)at.unit * slots;
    int v[kEach];
    float* w[kEach];
    float was[kEach], sum[kEach];
#pragma unroll
    for (int e = 0; e < kEach; e++) {
      v[e] = min(v0 + e * kThreads_, end - 1);
      const uint32_t s = at.len - at.visible + v[e], page = a.t.page_of(s);
      w[e] = a.weights + ((size_t)a.t.ids[(size_t)at.seq * a.t.per + page] * a.key_heads + kh) * a.t.page +
             (s - page * a.t.page);
      was[e] = *w[e], sum[e] = 0.0f;
    }
    if (begins) dependency_wait();
    constexpr int kEarly = 16 / kEach;  // heads whose scores are read while the statistics are worked out
    float early[kEarly][kEach];
#pragma unroll
    for (int h = 0; h < kEarly; h++)
#pragma unroll
      for (int e = 0; e < kEach; e++) early[h][e] = __ldcg(score + (size_t)min(h, group - 1) * padded + v[e]);
    for (int h0 = 0; h0 < group; h0 += kStats) {
      const int count = min(kStats, group - h0);
      if (begins || group > kStats) {
        __syncthreads();
        for (int h = warp; h < count; h += kThreads_ / 32) {
          const Pieces pc = pieces_of(wk, origin + (h0 + h) / kHeads * n_units, n);
          const float* stat = sc.stat + 2 * ((size_t)at.seq * a.heads + kh * group + h0 + h);
          if (pc.w0 == pc.w1) {
            if (lane < 2) s_stat[h][lane] = __ldcg(stat + lane);
            continue;
          }
          float M = -INFINITY, L = 0.0f;
          for (int c = lane; c < pc.count(); c += 32) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(sc.part_ml) + pc.slot_of(c, (h0 + h) % kHeads));
            merge(M, L, ml.x, ml.y);
          }
          merge_warp(M, L);
          if (lane == 0) s_stat[h][0] = M, s_stat[h][1] = 1.0f / L;
        }
        __syncthreads();
      }
      int h = 0;
      if (h0 == 0) {
#pragma unroll
        for (; h < kEarly; h++)
          if (h < count)
#pragma unroll
            for (int e = 0; e < kEach; e++) sum[e] += exp2_of(early[h][e] - s_stat[h][0]) * s_stat[h][1];
      }
#pragma unroll 4
      for (; h < count; h++)
#pragma unroll
        for (int e = 0; e < kEach; e++)
          sum[e] += exp2_of(__ldcg(score + (size_t)(h0 + h) * padded + v[e]) - s_stat[h][0]) * s_stat[h][1];
    }
#pragma unroll
    for (int e = 0; e < kEach; e++)
      if (v0 + e * kThreads_ < end) *w[e] = was[e] + sum[e];
  }
}

// The first `joins` CTAs join (`heads` of them a pair), the others add weights.
template <int kJoin>
__global__ void __launch_bounds__(kJoin)
    k_paged_finish(const __grid_constant__ PagedAttendArgs a, const __grid_constant__ Scratch sc,
                   const __grid_constant__ Work wk, bool by_pair, uint32_t joins,
                   uint32_t heads, int slots) {
  if (blockIdx.x < joins)
    join<kJoin>(a, sc, wk, by_pair, blockIdx.x / heads, blockIdx.x % heads);
  else
    add_weights<kJoin>(a, sc, wk, blockIdx.x - joins, slots);
}

struct Plan {
  Work work;
  uint32_t weight_ctas;
  int weight_slots;  // of a CTA
  int pairs;
  bool idle, cut;
  size_t slots;  // visible slots, each sequence's rounded up to 4
};

// Beginning and ending a pair takes a warp about as long as two blocks (4200
// cycles against 1900 to 2400 a block): counted so, 16 ragged sequences of 8
// key heads take 50 us, against 52 at one and 64 without.
constexpr uint32_t kExtra = 2;
// Pairs of up to this many blocks stay whole, a CTA each, joined in shared
// memory: cut, a call of 97 slots takes 8.2 us instead of 7.7.
constexpr uint32_t kWholeBlocks = 16;

// Where a pair would be cut into more than this many pieces by CTAs, CTAs are
// the takers (a quarter of the pieces to join): one of 16389 slots 14.0 us
// against 17.7.
constexpr uint32_t kManyPieces = 8;

Plan plan_of(const PagedAttendArgs& a) {
  Plan p{};
  const int group = a.heads / a.key_heads;
  const Config cfg = config_of(a.bf16, a.dh);
  Work& wk = p.work;
  wk.keys = cfg.keys, wk.tiles = a.key_heads * ((group + kHeads - 1) / kHeads);
  p.pairs = a.t.n * wk.tiles;
  uint32_t longest = 0, busy = 0;
  for (int i = 0; i < a.t.n; i++) {
    const uint32_t v = visible_of(a.host_lens[i], a.reach);
    longest = std::max(longest, v), busy += v > 0;
    p.slots += (v + 3) & ~3u;
  }
  p.idle = busy < (uint32_t)a.t.n;
  wk.whole = wk.blocks_of(longest) <= kWholeBlocks;
  wk.by_cta = wk.whole || cfg.dh > 192 || wk.tiles * busy * kManyPieces <= 148u * cfg.ctas;
  wk.direct = a.t.n == 1 || (wk.whole && !p.idle && !a.weights);
  wk.extra = wk.whole ? 0 : wk.by_cta ? kExtra * kWarps : kExtra;
  // Weights: more slots a CTA where there would be more CTAs than fit at once
  // (19 ragged sequences of up to 28955: 34.2 us against 36.6 without).
  p.weight_slots = kWeightKeys;
  while (p.slots * a.key_heads / p.weight_slots > 2048 && p.weight_slots < 1 << 20) p.weight_slots *= 2;
  uint64_t units = 0, weight_ctas = 0;
  for (int i = 0; i < a.t.n; i++) {
    const uint32_t v = visible_of(a.host_lens[i], a.reach);
    units += (uint64_t)wk.units_of(v) * wk.tiles;
    weight_ctas += (uint64_t)(v + p.weight_slots - 1) / p.weight_slots * a.key_heads;
  }
  SLM_REQUIRE(std::max(units, weight_ctas) < (1ull << 31), "paged_attend: too much work for one call");
  p.weight_ctas = (uint32_t)weight_ctas;
  // A taker for every place on the GPU; of CTAs at most two an SM, which leaves
  // room for the second kernel's to be there when the pieces are (one sequence
  // of 16389 bf16 slots, 64 wide: 9.0 us against 10.4 with three).
  wk.takers = (uint32_t)std::min<uint64_t>(148 * (wk.by_cta ? std::min(cfg.ctas, 2) : cfg.ctas * kWarps), units);
  if (wk.takers) wk.each = (uint32_t)(units / wk.takers), wk.more = (uint32_t)(units % wk.takers);
  p.cut = !wk.whole && wk.takers > 1;
  return p;
}

size_t round4(size_t n) { return (n + 3) / 4 * 4; }

// Carves the scratch; returns the floats it takes (base may be null).
size_t carve(const PagedAttendArgs& a, const Plan& p, float* base, Scratch* sc) {
  size_t at = 0;
  auto take = [&](size_t n) {
    float* r = base + at;
    at += round4(n);
    return r;
  };
  const size_t warps = p.cut ? p.work.takers : 0;
  sc->piece = std::min(kHeads, a.heads / a.key_heads) * a.dh;
  sc->part = take(2 * warps * sc->piece);
  sc->part_ml = take(2 * warps * kHeads * 2);
  sc->stat = a.weights ? take((size_t)a.t.n * a.heads * 2) : nullptr;
  sc->score = a.weights ? take(p.slots * a.heads) : nullptr;
  return at + 4;
}

template <bool BF16, int DH>
void launch(const PagedAttendArgs& a, const Scratch& sc, const Plan& p, cudaStream_t st) {
  const bool q16 = ((uintptr_t)a.q & 15) == 0 && a.ldq % 4 == 0;  // q in 16-byte loads
  const unsigned ctas = p.work.by_cta ? p.work.takers : cdiv(p.work.takers, kWarps);
  launch_after(k_paged_attend<BF16, DH>, dim3(std::max(1u, ctas)), kThreads, Shape<BF16, DH>::kSmem, st, a, sc,
               p.work, p.idle, q16);
}

template <bool BF16, int DH>
void prepare() {
  SLM_CUDA(cudaFuncSetAttribute(k_paged_attend<BF16, DH>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                Shape<BF16, DH>::kSmem));
}

}  // namespace

void paged_prepare() {
  prepare<false, 32>();
  prepare<false, 64>();
  prepare<false, 96>();
  prepare<false, 128>();
  prepare<false, 192>();
  prepare<false, 256>();
  prepare<true, 64>();
  prepare<true, 128>();
  prepare<true, 192>();
  prepare<true, 256>();
}

size_t paged_attend_scratch(const PagedAttendArgs& a) {
  Scratch sc;
  return carve(a, plan_of(a), nullptr, &sc);
}

void paged_attend(const PagedAttendArgs& a, cudaStream_t st) {
  const Plan p = plan_of(a);
  Scratch sc;
  carve(a, p, a.scratch, &sc);
  const int dh = config_of(a.bf16, a.dh).dh;
  if (a.bf16)
    (dh == 64 ? launch<true, 64> : dh == 128 ? launch<true, 128> : dh == 192 ? launch<true, 192> : launch<true, 256>)(
        a, sc, p, st);
  else
    (dh == 32    ? launch<false, 32>
     : dh == 64  ? launch<false, 64>
     : dh == 96  ? launch<false, 96>
     : dh == 128 ? launch<false, 128>
     : dh == 192 ? launch<false, 192>
                 : launch<false, 256>)(a, sc, p, st);
  const bool by_pair = p.pairs < (int)p.work.takers;
  const uint32_t heads = std::min(kHeads, a.heads / a.key_heads);
  const uint32_t joins = p.cut ? (by_pair ? p.pairs : p.work.takers) * heads : 0;
  const uint32_t ctas = joins + (a.weights ? p.weight_ctas : 0);
  if (!ctas) return;
  // Few pieces a pair: small CTAs, since there are many; 128 threads where the
  // weights of many query heads are added (12 a key head: 21.9 us against 26.1).
  const bool few = p.work.takers / 32 < (uint32_t)p.pairs && a.dh <= 128;
  const int threads = !few ? 256 : a.weights && a.heads / a.key_heads > 4 ? 128 : 64;
  launch_after(threads == 64 ? k_paged_finish<64> : threads == 128 ? k_paged_finish<128> : k_paged_finish<256>,
               dim3(ctas), threads, 0, st, a, sc, p.work, by_pair, joins, heads, p.weight_slots);
}

}  // namespace slm
