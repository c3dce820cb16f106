// Attention of one new token per sequence over a paged key-value cache.
//
//   p_s = exp(x_s - max x) / Σ exp(x - max x),  x_s = scale · q·k_s,  y = Σ p_s v_s
//
// over the visible slots, in one pass: every warp keeps a running reference
// maximum m, the sum l of exp(x - m) and the sum of exp(x - m) v, all f32.
// Keys and values are read once, so bytes bound the call; the rest is arranged
// to stay under them.
//
// Work: the visible slots of a (sequence, tile of up to 8 query heads of one
// key head) are cut into chunks of equal length, one CTA each (4 warps, every
// warp its own tiles of the chunk); the last CTA of a cut (sequence, tile)
// joins the chunks' partials in order, so results do not depend on timing.
//
// Data: a warp streams its tiles through three private buffers with 16-byte
// asynchronous copies, which look every row's page up (a page may end
// anywhere in a tile) and fill rows past the end and columns past the head
// size with zeros.  8 warps an SM keep 128 KB or so in flight.
//
// Products: mma.m16n8k8 on tf32, with the group's heads as rows.  Operands of
// f32 precision are split into two tf32 parts, x = hi + lo: of the 16 rows, 8
// hold the heads' hi parts and 8 their lo parts, so one product per part of
// the other operand gives all four partial products, and a row pair's sum is
// the f32 result.  bf16 keys and values are tf32 values as they are: one
// product.  The tensor cores do in this form what the CUDA cores would do in
// 8 times the instructions; a tcgen05 tile (64 or 128 rows) would be mostly
// empty at 1 to 8 heads.
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"
#include "paged.cuh"

namespace slm {

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32, kHeads = 8, kStages = 3;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.0f;     // scores (log2 units) may exceed m by this before m moves
constexpr int kMaxChunks = 1024;  // chunks of one sequence
constexpr int kWeightKeys = 256;  // slots of a CTA of k_paged_weights

// Where a launch keeps what its CTAs hand one another.
struct Scratch {
  float* part;       // [CTA][heads][dh] sums, then [CTA][heads][2] (m, l), of cut sequences
  float* part_ml;
  float* stat;       // [n][heads][2]: final m and 1 / l
  float* score;      // per sequence [heads][visible rounded up to 4], log2 units; or null
  unsigned* cnt;     // [n][tiles] arrivals, zero between launches
};

__host__ __device__ inline int visible_of(uint32_t len, long long reach) {
  return reach && (long long)len > reach ? (int)reach : (int)len;
}

// Tile shape for pages of `size`-byte values and head sizes up to DH: K and V
// of a tile take 8 KB (16 KB at f32, 256).
template <int SIZE, int DH>
struct Shape {
  static constexpr int kRow = DH * SIZE;             // bytes of a row in shared memory
  static constexpr int kKeys = 4096 / kRow < 8 ? 8 : 4096 / kRow;
  static constexpr int kTile = kKeys * kRow;         // K (or V) bytes of a tile
  static constexpr int kBuffers = kWarps * kStages * 2 * kTile;
  static constexpr bool kQShared = DH > 128;         // q in shared memory: registers hold the sums
  static constexpr int kQ = kQShared ? DH / 8 * 512 : 0;
  static constexpr int kSmem = kBuffers + kQ;
  static constexpr int kCtas = kSmem <= 113 * 1024 ? 2 : 1;
};

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

// The upper 11 significant bits of x, and the rest (read by the tensor core to
// 11 bits of its own: x is kept to 2^-21).
__device__ __forceinline__ uint32_t hi_of(uint32_t x) { return x & 0xffffe000u; }
__device__ __forceinline__ uint32_t lo_of(uint32_t x) {
  return __float_as_uint(__uint_as_float(x) - __uint_as_float(hi_of(x)));
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

// The sequence and chunk of CTA-row `at`: sequences' chunks lie one after the
// other.  Also the rounded visible slots of the sequences before it.
struct Place {
  int seq, chunk, chunks, visible;
  long long before;
};
__device__ Place find_place(const PagedTable& t, long long reach, int keys, int at) {
  __shared__ int s_chunks[kThreads / 32];
  __shared__ long long s_slots[kThreads / 32];
  __shared__ Place s_place;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  const int each = (t.n + blockDim.x - 1) / blockDim.x;
  int mine = 0;
  long long slots = 0;
  for (int j = 0; j < each; j++) {
    const int i = tid * each + j;
    const int v = i < t.n ? visible_of(t.lens[i], reach) : 0;
    mine += (v + keys - 1) / keys, slots += (v + 3) & ~3;
  }
  int upto = mine;
  long long slots_upto = slots;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, upto, o);
    const long long b = __shfl_up_sync(0xffffffffu, slots_upto, o);
    if (lane >= o) upto += a, slots_upto += b;
  }
  if (lane == 31) s_chunks[warp] = upto, s_slots[warp] = slots_upto;
  __syncthreads();
  for (int w = 0; w < nw; w++)
    if (w < warp) upto += s_chunks[w], slots_upto += s_slots[w];
  if (at < upto && at >= upto - mine) {
    int c = at - (upto - mine);
    long long b = slots_upto - slots;
    for (int j = 0;; j++) {
      const int v = visible_of(t.lens[tid * each + j], reach), n = (v + keys - 1) / keys;
      if (c < n) {
        s_place = Place{tid * each + j, c, n, v, b};
        break;
      }
      c -= n, b += (v + 3) & ~3;
    }
  }
  __syncthreads();
  return s_place;
}

template <bool BF16, int DH>
__global__ void __launch_bounds__(kThreads, Shape<BF16 ? 2 : 4, DH>::kCtas)
    k_paged_attend(PagedAttendArgs a, Scratch sc, int keys, int tiles) {
  constexpr int SIZE = BF16 ? 2 : 4;
  using S = Shape<SIZE, DH>;
  constexpr int kSteps = DH / 8;            // k-steps of q·k, and 8-column tiles of p·v
  constexpr int kLoad = BF16 ? 4 : 2;       // k-steps that a 16-byte piece of a key row feeds
  constexpr int kPieces = S::kRow / 16;     // 16-byte pieces of a row
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float s_m[kWarps][kHeads], s_l[kWarps][kHeads];
  __shared__ int s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tile = blockIdx.x % tiles;
  const Place at = find_place(a.t, a.reach, keys, blockIdx.x / tiles);
  const int group = a.heads / a.key_heads, per_key = (group + kHeads - 1) / kHeads;
  const int kh = tile / per_key, head0 = kh * group + (tile % per_key) * kHeads;
  const int heads = min(kHeads, (kh + 1) * group - head0);
  const int lo = (int)a.t.lens[at.seq] - at.visible;
  const int first = lo + at.chunk * keys, end = lo + min(at.visible, (at.chunk + 1) * keys);

  // q, scaled to log2 units and split, in the order the key rows are read:
  // rows g and g + 8 of the left operand are head g's hi and lo parts.
  uint32_t qa[S::kQShared ? 1 : kSteps][4];
  const uint32_t buffers = (uint32_t)__cvta_generic_to_shared(smem);
  const uint32_t q_shared = buffers + S::kBuffers;
  {
    const float* q = a.q + at.seq * a.ldq + (size_t)(head0 + g) * a.dh;
    const float scale = a.scale * kLog2e;
#pragma unroll
    for (int s = 0; s < kSteps; s++) {
      const int d = (s / kLoad) * (BF16 ? 32 : 16) + t * (BF16 ? 8 : 4) + s % kLoad * 2;
      const bool ok = g < heads && d < a.dh;  // dh is even
      uint32_t w[4];
      split(ok ? q[d] * scale : 0.0f, w[0], w[1]);
      split(ok ? q[d + 1] * scale : 0.0f, w[2], w[3]);
      if (S::kQShared) {
        if (s % kWarps == warp)
          *reinterpret_cast<uint4*>(smem + S::kBuffers + s * 512 + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++) qa[S::kQShared ? 0 : s][j] = w[j];
      }
    }
    if (S::kQShared) __syncthreads();
  }

  // This warp's tiles: warp, warp + kWarps, … of the chunk.
  const uint32_t mine = buffers + warp * (kStages * 2 * S::kTile);
  const uint32_t* ids = a.t.ids + (size_t)at.seq * a.t.per;
  const char *K = static_cast<const char*>(a.k), *V = static_cast<const char*>(a.v);
  const int row_bytes = a.dh * SIZE, pieces = row_bytes / 16;
  const int n_tiles = first + warp * S::kKeys < end
                          ? (end - first - warp * S::kKeys + kWarps * S::kKeys - 1) / (kWarps * S::kKeys)
                          : 0;
  auto key_of = [&](int j) { return first + (j * kWarps + warp) * S::kKeys; };
  // Byte offset in the pool of the row that this lane looks up for tile j.
  auto look_up = [&](int j) -> long long {
    const int s = min(key_of(j) + lane % S::kKeys, end - 1);
    const int page = s / a.t.page;
    return (((long long)ids[page] * a.key_heads + kh) * a.t.page + (s - page * a.t.page)) * row_bytes;
  };
  auto load = [&](int j, long long off) {
    const uint32_t to = mine + j % kStages * (2 * S::kTile);
    const int n = end - key_of(j);
#pragma unroll
    for (int u = 0; u < S::kKeys * kPieces / 32; u++) {
      const int r = (u * 32 + lane) / kPieces, c = (u * 32 + lane) % kPieces;
      const long long o = __shfl_sync(0xffffffffu, off, r);
      const bool ok = r < n && c < pieces;
      const long long from = ok ? o + c * 16 : 0;
      // Swizzles under which the reads below hit every bank once.
      copy16(to + r * S::kRow + ((c ^ ((r & 1) << 2)) << 4), K + from, ok);
      copy16(to + S::kTile + r * S::kRow + ((c ^ (r & 6)) << 4), V + from, ok);
    }
  };

  float m = -INFINITY, l = 0.0f, o[kSteps][4];
#pragma unroll
  for (int s = 0; s < kSteps; s++)
#pragma unroll
    for (int j = 0; j < 4; j++) o[s][j] = 0.0f;
  float* score = sc.score ? sc.score + at.before * a.heads + (size_t)(head0 + g) * ((at.visible + 3) & ~3) - lo : nullptr;

  long long off = 0;
#pragma unroll
  for (int j = 0; j < kStages - 1; j++) {
    if (j < n_tiles) load(j, look_up(j));
    copies_commit();
  }
  if (kStages - 1 < n_tiles) off = look_up(kStages - 1);
  for (int j = 0; j < n_tiles; j++) {
    copies_wait<kStages - 2>();
    __syncwarp();  // every lane's copies of tile j have landed, and all are done with tile j - 1
    if (j + kStages - 1 < n_tiles) load(j + kStages - 1, off);
    copies_commit();
    if (j + kStages < n_tiles) off = look_up(j + kStages);

    const uint32_t kt = mine + j % kStages * (2 * S::kTile), vt = kt + S::kTile;
    const int key0 = key_of(j);
    constexpr int kBlocks = S::kKeys / 8;
    float x[kBlocks][2];
#pragma unroll
    for (int b = 0; b < kBlocks; b++) {
      constexpr int kChains = 4;  // independent sums, so that products overlap
      float c[kChains][4];
#pragma unroll
      for (int e = 0; e < kChains; e++) c[e][0] = c[e][1] = c[e][2] = c[e][3] = 0.0f;
      const uint32_t row = kt + (b * 8 + g) * S::kRow + t * 16;
      const int odd = (g & 1) * 64;
#pragma unroll
      for (int i = 0; i < kSteps / kLoad; i++) {
        const uint4 w = lds16(row + i * 64 + (i & 1 ? -odd : odd));
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < kLoad; e++) {
          const int s = i * kLoad + e;
          uint32_t qs[4];
          if (S::kQShared) {
            const uint4 qw = lds16(q_shared + s * 512 + lane * 16);
            qs[0] = qw.x, qs[1] = qw.y, qs[2] = qw.z, qs[3] = qw.w;
          }
          const uint32_t* qv = S::kQShared ? qs : qa[S::kQShared ? 0 : s];
          if (BF16)
            Operand<BF16>::mul(c[s % kChains], qv, v[e] << 16, v[e] & 0xffff0000u);
          else
            Operand<BF16>::mul(c[s % kChains], qv, v[e * 2], v[e * 2 + 1]);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float sum = 0.0f;
#pragma unroll
        for (int ch = 0; ch < kChains; ch++) sum += c[ch][e] + c[ch][e + 2];
        x[b][e] = key0 + b * 8 + 2 * t + e < end ? sum : -INFINITY;
      }
      if (score && g < heads) {
        const int s = key0 + b * 8 + 2 * t;
        if (s < end) score[s] = x[b][0];
        if (s + 1 < end) score[s + 1] = x[b][1];
      }
    }
    float top = x[0][0];
#pragma unroll
    for (int b = 0; b < kBlocks; b++) top = fmaxf(top, fmaxf(x[b][0], x[b][1]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // m moves only when a score passes it by kLazy (the first tile: from -inf).
    if (__any_sync(0xffffffffu, top > m + kLazy)) {
      const float to = top > m + kLazy ? top : m;
      const float keep = to == m ? 1.0f : exp2f(m - to);
      m = to, l *= keep;
#pragma unroll
      for (int s = 0; s < kSteps; s++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[s][e] *= keep;
    }
#pragma unroll
    for (int b = 0; b < kBlocks; b++) {
      const float p0 = exp2f(x[b][0] - m), p1 = exp2f(x[b][1] - m);
      l += p0 + p1;
      uint32_t p[4];
      split(p0, p[0], p[1]);
      split(p1, p[2], p[3]);
      const uint32_t row = vt + (b * 8 + 2 * t) * S::kRow + ((g ^ (2 * t)) << 4);
#pragma unroll
      for (int i = 0; i < S::kRow / 128; i++) {
        const uint4 w0 = lds16(row + i * 128), w1 = lds16(row + S::kRow + i * 128);
        const uint32_t v0[4] = {w0.x, w0.y, w0.z, w0.w}, v1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (BF16) {
            Operand<BF16>::mul(o[i * 8 + e * 2], p, v0[e] << 16, v1[e] << 16);
            Operand<BF16>::mul(o[i * 8 + e * 2 + 1], p, v0[e] & 0xffff0000u, v1[e] & 0xffff0000u);
          } else {
            Operand<BF16>::mul(o[i * 4 + e], p, v0[e], v1[e]);
          }
        }
      }
    }
  }
  copies_wait<0>();
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  __syncthreads();  // the buffers are free

  // Join the warps: sums through shared memory, [warp][head][DH].
  float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int s = 0; s < kSteps; s++) {
    constexpr int kWide = BF16 ? 8 : 4;  // columns of a 16-byte piece
    const int d = s / kWide * (kWide * 8) + 2 * t * kWide + s % kWide;
    float* to = sums + (warp * kHeads + g) * DH + d;
    to[0] = o[s][0] + o[s][2];
    to[kWide] = o[s][1] + o[s][3];
  }
  if (t == 0) s_m[warp][g] = m, s_l[warp][g] = l;
  __syncthreads();
  const bool cut = at.chunks > 1;
  float* part = sc.part + (size_t)blockIdx.x * kHeads * a.dh;
  float* part_ml = sc.part_ml + (size_t)blockIdx.x * kHeads * 2;
  float* y = a.y + ((size_t)at.seq * a.heads + head0) * a.dh;
  for (int e = threadIdx.x; e < heads * a.dh; e += kThreads) {
    const int h = e / a.dh, d = e % a.dh;
    float M = s_m[0][h], L = 0.0f, v = 0.0f;
#pragma unroll
    for (int w = 1; w < kWarps; w++) M = fmaxf(M, s_m[w][h]);
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
      const float f = s_l[w][h] > 0.0f ? exp2f(s_m[w][h] - M) : s_l[w][h];  // a warp without tiles: 0 (NaN stays)
      L += s_l[w][h] * f;
      v += sums[(w * kHeads + h) * DH + d] * f;
    }
    if (!cut) {
      y[e] = v / L;
      if (sc.stat && d == 0) {
        float* st = sc.stat + 2 * ((size_t)at.seq * a.heads + head0 + h);
        st[0] = M, st[1] = 1.0f / L;
      }
    } else {
      part[e] = v;
      if (d == 0) part_ml[2 * h] = M, part_ml[2 * h + 1] = L;
    }
  }
  if (!cut) return;

  // The last chunk of the (sequence, tile) to arrive joins all of them.
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned* cnt = sc.cnt + (size_t)at.seq * tiles + tile;
    s_last = atomicAdd(cnt, 1u) == (unsigned)at.chunks - 1;
    if (s_last) *cnt = 0;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  const size_t cta0 = (size_t)blockIdx.x - (size_t)at.chunk * tiles;
  const float* ml = sc.part_ml + cta0 * kHeads * 2;
  const size_t ml_step = (size_t)tiles * kHeads * 2;
  float* factor = reinterpret_cast<float*>(smem);  // [chunk][head]
  for (int h = warp; h < heads; h += kWarps) {
    float M = -INFINITY, L = 0.0f;
    for (int c = lane; c < at.chunks; c += 32) M = fmaxf(M, __ldcg(ml + c * ml_step + 2 * h));
    M = warp_max(M);
    for (int c = lane; c < at.chunks; c += 32) {
      const float f = exp2f(__ldcg(ml + c * ml_step + 2 * h) - M);
      factor[c * kHeads + h] = f;
      L += f * __ldcg(ml + c * ml_step + 2 * h + 1);
    }
    L = warp_sum(L);
    if (lane == 0) {
      s_m[0][h] = M, s_l[0][h] = 1.0f / L;
      if (sc.stat) {
        float* st = sc.stat + 2 * ((size_t)at.seq * a.heads + head0 + h);
        st[0] = M, st[1] = 1.0f / L;
      }
    }
  }
  __syncthreads();
  const float* parts = sc.part + cta0 * kHeads * a.dh;
  const size_t step = (size_t)tiles * kHeads * a.dh;
  for (int e = threadIdx.x * 4; e < heads * a.dh; e += kThreads * 4) {
    const int h = e / a.dh;  // dh is a multiple of 8
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int c = 0; c < at.chunks; c++) {
      const float4 w = __ldcg(reinterpret_cast<const float4*>(parts + c * step + e));
      const float f = factor[c * kHeads + h];
      v.x = fmaf(w.x, f, v.x), v.y = fmaf(w.y, f, v.y), v.z = fmaf(w.z, f, v.z), v.w = fmaf(w.w, f, v.w);
    }
    const float r = s_l[0][h];
    y[e] = v.x * r, y[e + 1] = v.y * r, y[e + 2] = v.z * r, y[e + 3] = v.w * r;
  }
}

// weight[s] += Σ_h p_s over the key head's query heads, from the kept scores:
// a thread per slot.
__global__ void __launch_bounds__(kThreads) k_paged_weights(PagedAttendArgs a, Scratch sc) {
  const int kh = blockIdx.x % a.key_heads, group = a.heads / a.key_heads;
  const Place at = find_place(a.t, a.reach, kWeightKeys, blockIdx.x / a.key_heads);
  const int lo = (int)a.t.lens[at.seq] - at.visible, padded = (at.visible + 3) & ~3;
  const float* score = sc.score + at.before * a.heads + (size_t)kh * group * padded;
  const float* stat = sc.stat + 2 * ((size_t)at.seq * a.heads + kh * group);
  for (int j = threadIdx.x; j < kWeightKeys; j += kThreads) {
    const int v = at.chunk * kWeightKeys + j;
    if (v >= at.visible) break;
    float sum = 0.0f;
    for (int h = 0; h < group; h++) sum += exp2f(score[(size_t)h * padded + v] - stat[2 * h]) * stat[2 * h + 1];
    const int s = lo + v, page = s / a.t.page;
    a.weights[((size_t)a.t.ids[(size_t)at.seq * a.t.per + page] * a.key_heads + kh) * a.t.page + s - page * a.t.page] +=
        sum;
  }
}

// y rows of idle sequences (their key heads have no CTA).
__global__ void k_paged_idle(PagedAttendArgs a) {
  const int i = blockIdx.x;
  if (a.t.lens[i] != 0) return;
  for (int e = threadIdx.x; e < a.heads * a.dh; e += blockDim.x) a.y[(size_t)i * a.heads * a.dh + e] = 0.0f;
}

// What a launch is cut into.
struct Plan {
  int keys, tiles, ctas;   // slots of a chunk; head tiles; CTAs in all
  int weight_ctas;
  bool cut, idle;
  size_t slots;            // visible slots, each sequence's rounded up to 4
};

int padded_dh(int dh) { return dh <= 64 ? 64 : dh <= 128 ? 128 : 256; }

Plan plan_of(const PagedAttendArgs& a) {
  Plan p{};
  const int group = a.heads / a.key_heads, size = a.bf16 ? 2 : 4, dh = padded_dh(a.dh);
  p.tiles = a.key_heads * ((group + kHeads - 1) / kHeads);
  const int row = dh * size, tile_keys = std::max(8, 4096 / row) * kWarps;
  const int room = 148 * (!a.bf16 && dh == 256 ? 1 : 2);
  long long total = 0, longest = 0, weight_ctas = 0;
  for (int i = 0; i < a.t.n; i++) {
    const int v = visible_of(a.host_lens[i], a.reach);
    total += v, longest = std::max<long long>(longest, v);
    p.slots += (v + 3) & ~3;
    p.idle |= v == 0;
    weight_ctas += (long long)cdiv(v, kWeightKeys) * a.key_heads;
  }
  // Chunks of about 256 KB when there is work for many of them, else one for
  // every place a CTA has on the GPU; at least one tile a warp.
  long long keys = std::min<long long>((total * p.tiles + room - 1) / room, std::max(1, 262144 / (2 * row)));
  keys = std::max(keys, (longest + kMaxChunks - 1) / kMaxChunks);
  keys = std::max<long long>(1, (keys + tile_keys - 1) / tile_keys) * tile_keys;
  p.keys = (int)keys;  // below 2^21: a sequence holds less than 2^30 slots
  long long chunks = 0;
  for (int i = 0; i < a.t.n; i++) {
    const long long c = (visible_of(a.host_lens[i], a.reach) + (long long)p.keys - 1) / p.keys;
    chunks += c;
    p.cut |= c > 1;
  }
  SLM_REQUIRE(std::max(chunks * p.tiles, weight_ctas) < (1ll << 31), "paged_attend: too much work for one call");
  p.weight_ctas = (int)weight_ctas;
  p.ctas = (int)(chunks * p.tiles);
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
  const size_t parts = p.cut ? (size_t)p.ctas : 0;
  sc->part = take(parts * kHeads * a.dh);
  sc->part_ml = take(parts * kHeads * 2);
  sc->stat = a.weights ? take((size_t)a.t.n * a.heads * 2) : nullptr;
  sc->score = a.weights ? take(p.slots * a.heads) : nullptr;
  sc->cnt = a.counters;
  return at + 4;
}

template <bool BF16, int DH>
void launch(const PagedAttendArgs& a, const Scratch& sc, const Plan& p, cudaStream_t st) {
  k_paged_attend<BF16, DH><<<p.ctas, kThreads, Shape<BF16 ? 2 : 4, DH>::kSmem, st>>>(a, sc, p.keys, p.tiles);
}

template <bool BF16, int DH>
void prepare() {
  SLM_CUDA(cudaFuncSetAttribute(k_paged_attend<BF16, DH>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                Shape<BF16 ? 2 : 4, DH>::kSmem));
}

}  // namespace

void paged_prepare() {
  prepare<false, 64>();
  prepare<false, 128>();
  prepare<false, 256>();
  prepare<true, 64>();
  prepare<true, 128>();
  prepare<true, 256>();
}

size_t paged_attend_scratch(const PagedAttendArgs& a) {
  Scratch sc;
  return carve(a, plan_of(a), nullptr, &sc);
}

size_t paged_attend_counters(const PagedAttendArgs& a) {
  const int group = a.heads / a.key_heads;
  return (size_t)a.t.n * a.key_heads * ((group + kHeads - 1) / kHeads);
}

void paged_attend(const PagedAttendArgs& a, cudaStream_t st) {
  const Plan p = plan_of(a);
  Scratch sc;
  carve(a, p, a.scratch, &sc);
  if (p.idle) {
    k_paged_idle<<<a.t.n, 256, 0, st>>>(a);
    SLM_LAUNCHED("k_paged_idle");
  }
  if (!p.ctas) return;
  const int dh = padded_dh(a.dh);
  if (a.bf16)
    dh == 64 ? launch<true, 64>(a, sc, p, st) : dh == 128 ? launch<true, 128>(a, sc, p, st) : launch<true, 256>(a, sc, p, st);
  else
    dh == 64 ? launch<false, 64>(a, sc, p, st) : dh == 128 ? launch<false, 128>(a, sc, p, st) : launch<false, 256>(a, sc, p, st);
  SLM_LAUNCHED("k_paged_attend");
  if (a.weights) {
    k_paged_weights<<<p.weight_ctas, kThreads, 0, st>>>(a, sc);
    SLM_LAUNCHED("k_paged_weights");
  }
}

}  // namespace slm
