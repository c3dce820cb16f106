// Storing tokens into the pages of a paged cache, evicting tokens from it, and
// updates of its tables (checked on the host, paged.cpp).
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <cstring>

#include "common.cuh"
#include "evict_order.hpp"
#include "paged.cuh"

namespace cg = cooperative_groups;

namespace slm {

namespace {

// Pool row of slot s of sequence i, key head h.
__device__ __forceinline__ size_t pool_row(const PagedTable& t, int i, int s, int h, int key_heads) {
  const uint32_t page = t.page_of(s), id = t.ids[(size_t)i * t.per + page];
  return ((size_t)id * key_heads + h) * t.page + (s - page * t.page);
}

struct Words {
  uint32_t at[kPutWords], value[kPutWords];
};

__global__ void k_table_put(uint32_t* words, const __grid_constant__ Words w, int n) {
  for (int j = threadIdx.x; j < n; j += blockDim.x) words[w.at[j]] = w.value[j];
}

// ---------------------------------------------------------------------------
// Store: bytes bound it (8 of f32 in, 4 or 8 out, a value of K and V).  A warp
// per token; a lane moves 8 values of K and of V at a time, its reads on their
// way before the token's page is looked up.
// ---------------------------------------------------------------------------
constexpr int kStoreThreads = 256;

template <bool VEC>
__device__ __forceinline__ void read8(const float* p, float* v) {
  if (VEC) {
    const float4 a = ld_stream(reinterpret_cast<const float4*>(p)), b = ld_stream(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = p[e];
  }
}

template <bool BF16>
__device__ __forceinline__ void write8(void* pool, size_t at, const float* v) {
  if (BF16) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {  // the nearest bf16, ties to even
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
      w[e] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(pool) + at) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    float4* to = reinterpret_cast<float4*>(static_cast<float*>(pool) + at);
    to[0] = make_float4(v[0], v[1], v[2], v[3]);
    to[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

template <bool BF16, bool VEC>
__global__ void __launch_bounds__(kStoreThreads) k_paged_store(const __grid_constant__ PagedStoreArgs a) {
  dependency_wait();
  dependents_launch();
  const int lane = threadIdx.x & 31, eights = a.dh / 8, total = a.key_heads * eights;
  const long long tokens = (long long)a.count * a.m, step = (long long)gridDim.x * (kStoreThreads / 32);
  for (long long tok = (long long)blockIdx.x * (kStoreThreads / 32) + (threadIdx.x >> 5); tok < tokens; tok += step) {
    const int i = a.first + (int)(tok / a.m), s = (int)((long long)a.t.lens[i] - a.m + tok % a.m);
    if (s < 0) continue;
    const uint32_t page = a.t.page_of(s);
    const uint32_t id = a.t.ids[(size_t)i * a.t.per + page];
    for (int e = lane; e < total; e += 32) {
      float kv[8], vv[8];
      read8<VEC>(a.ks + tok * a.ldk + e * 8, kv);
      read8<VEC>(a.vs + tok * a.ldv + e * 8, vv);
      const int h = e / eights;
      const size_t row = ((size_t)id * a.key_heads + h) * a.t.page + (s - page * a.t.page);
      const size_t at = row * a.dh + (e - h * eights) * 8;
      write8<BF16>(a.k, at, kv);
      write8<BF16>(a.v, at, vv);
      if (a.weights && e == h * eights) a.weights[row] = 0.0f;
    }
  }
}

// ---------------------------------------------------------------------------
// Evict.  A cluster of CTAs per pair (key head, sequence), each CTA a
// contiguous slice of its slots with their weights in shared memory, so memory
// is read once.  The lowest kept weight is found digit by digit from the top of
// an order-preserving integer: every CTA counts its slice, and one warp of each
// adds the cluster's counts through distributed shared memory.  Latency bounds
// it: three digits (11, 11, 10 bits, searched by their upper 5 bits first) in a
// cluster, where a digit costs a cluster barrier; four of 8 bits in a CTA alone
// (one of 16640: 14.9 us against 18.7 with four; 32 of 600: 19.1 against 22.3
// with three).  A second kernel moves the kept tokens' rows,
// bound by bytes (moved by the searching CTAs themselves, with too few loads in
// flight, 16 ragged sequences of up to 32768 took 150 us instead of 98).
// ---------------------------------------------------------------------------
constexpr int kSelect = 512, kMaxCluster = 8;
constexpr int kSelectKeys = 40 * 1024;  // slots of a slice that shared memory holds; longer ones are read again
constexpr int kSelectWarps = kSelect / 32;

// Inclusive sums over the lanes of a warp.
__device__ __forceinline__ int scan_up(int v) {
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, x);
    if ((threadIdx.x & 31) >= x) v += u;
  }
  return v;
}

// Counts `digit` of the lanes that compete; the first one's is likely to be
// many lanes' (weights share an exponent), so those are counted as one.
__device__ __forceinline__ void count_digit(int* hist, uint32_t digit, bool competes) {
  const unsigned lanes = __ballot_sync(0xffffffffu, competes);
  if (lanes == 0) return;
  const int leader = __ffs(lanes) - 1, lane = threadIdx.x & 31;
  const uint32_t most = __shfl_sync(0xffffffffu, digit, leader);
  const unsigned same = __ballot_sync(0xffffffffu, competes && digit == most);
  if (lane == leader) atomicAdd(hist + most, __popc(same));
  if (competes && digit != most) atomicAdd(hist + digit, 1);
}

// FITS: a slice fits into shared memory; ONE: a CTA a pair, no cluster.
template <bool FITS, bool ONE>
__global__ void __launch_bounds__(kSelect)
    k_paged_select(const __grid_constant__ PagedEvictArgs a) {
  using D = Digits<ONE>;
  constexpr int kPasses = D::kPasses, kDigits = D::kCount, kTop = D::kTop, kCoarse = 32, kGroup = kDigits / kCoarse;
  extern __shared__ uint32_t s_order[];
  // Alone, counts of every pass; in a cluster two passes' in turn, so that four
  // CTAs fit an SM (48 KB each at 8192 slots): 89.1 us against 90.3.
  constexpr int kHists = ONE ? kPasses : 2;
  __shared__ __align__(16) int s_hist[kHists][kDigits];
  __shared__ int s_coarse[kPasses][kCoarse];
  __shared__ int s_digit, s_left, s_rest, s_sure[kSelectWarps + 1], s_tie[kSelectWarps + 1];
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = ONE ? 1 : cluster.num_blocks(), part = ONE ? 0 : cluster.block_rank();
  auto sync = [&] {
    if (ONE)
      __syncthreads();
    else
      cluster.sync();
  };
  const int pair = blockIdx.x / parts, h = pair % a.key_heads, i = pair / a.key_heads;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  dependency_wait();
  dependents_launch();
  const int n = (int)a.from.lens[i];
  uint32_t* out = a.kept + ((size_t)i * a.key_heads + h) * a.keep;
  if (n <= a.keep) {  // all kept; uniform in the cluster
    const size_t keep = a.keep, step = parts * kSelect;  // a step past keep may pass 2^31
    for (size_t j = part * kSelect + t; j < keep; j += step) out[j] = j < (size_t)n ? (uint32_t)j : 0xffffffffu;
  } else {
    for (int d = t; d < kHists * kDigits; d += kSelect) (&s_hist[0][0])[d] = 0;
    // A warp's slots lie together: 32 · rounds of them.
    const int rounds = (n + parts * kSelect - 1) / (parts * kSelect);
    const int slice = part * rounds * kSelect, mine = warp * rounds * 32 + lane;
    const int lo = a.sinks, hi = n - a.recent;  // the slots that compete
    auto order_at = [&](int r) -> uint32_t {
      const int j = mine + r * 32, s = slice + j;
      if (FITS || j < kSelectKeys) return s_order[j];
      if (s >= n) return 0;
      return s < lo || s >= hi ? kHeld : order_of(a.weights[pool_row(a.from, i, s, h, a.key_heads)]);
    };
    __syncthreads();
    // Several slots' page ids, then weights, on their way at once.
    constexpr int kAtOnce = 8;
    const uint32_t* ids = a.from.ids + (size_t)i * a.from.per;
    for (int r0 = 0; r0 < rounds; r0 += kAtOnce) {
      uint32_t row[kAtOnce];
      float w[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; u++) {
        const uint32_t s = min(slice + mine + (r0 + u) * 32, n - 1), page = a.from.page_of(s);
        row[u] = (ids[page] * a.key_heads + h) * a.from.page + (s - page * a.from.page);
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; u++) w[u] = a.weights[row[u]];
#pragma unroll
      for (int u = 0; u < kAtOnce; u++) {
        const int j = mine + (r0 + u) * 32, s = slice + j;
        if (r0 + u >= rounds) break;
        const uint32_t o = s >= n ? 0 : s < lo || s >= hi ? kHeld : order_of(w[u]);
        if (FITS || j < kSelectKeys) s_order[j] = o;
        const bool competes = o != 0 && o != kHeld;
        if (ONE)
          count_digit(s_hist[0], o >> kTop, competes);
        else if (competes)
          atomicAdd(&s_hist[0][o >> kTop], 1);
      }
    }
    uint32_t prefix = 0;
    int need = a.keep - a.sinks - a.recent;  // how many of those that compete are kept
    if (need == 0) prefix = kHeld - 1;
#pragma unroll 1
    for (int pass = 0; pass < kPasses; pass++) {
      if (need == 0) break;  // uniform in the cluster
      const int shift = D::shift(pass), bits = D::bits(pass);
      int* hist = s_hist[pass % kHists];
      if (pass > 0) {
#pragma unroll 4
        for (int r = 0; r < rounds; r++) {
          const uint32_t o = order_at(r);
          if (counts(o, prefix, shift + bits)) atomicAdd(hist + (o >> shift & ((1 << bits) - 1)), 1);
        }
      }
      if (!ONE) {
        // Counts of kGroup digits at a time.
        __syncthreads();
        for (int c = warp; c < kCoarse; c += kSelectWarps) {
          const int v = __reduce_add_sync(0xffffffffu, hist[c * kGroup + lane] + hist[c * kGroup + kGroup / 2 + lane]);
          if (lane == 0) s_coarse[pass][c] = v;
        }
      }
      sync();
      // The first pass's counts have been read by all: room for the third's.
      if (!ONE && pass == 1)
        for (int d = t; d < kDigits; d += kSelect) s_hist[0][d] = 0;
      if (warp == 0 && ONE) {
        // The digit, from the top, that holds the need-th largest: eight of them a lane.
        const int low = kDigits - 8 - 8 * lane;
        const int4 x = *reinterpret_cast<const int4*>(hist + low), y = *reinterpret_cast<const int4*>(hist + low + 4);
        const int out_of = lane == 0 ? held_counted<ONE>(a.sinks + a.recent, prefix, pass) : 0;
        const int c[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w - out_of};
        int all = 0;
#pragma unroll
        for (int d = 0; d < 8; d++) all += c[d];
        const int upto = scan_up(all);
        if (lane == __ffs(__ballot_sync(0xffffffffu, upto >= need)) - 1) {
          int left = need - (upto - all), digit = low + 7;  // after the digits above this lane's
#pragma unroll
          for (int d = 7; d > 0; d--)
            if (digit == low + d && c[d] < left) left -= c[d], digit--;
          s_digit = digit, s_left = left, s_rest = hist[digit] - (digit == low + 7 ? out_of : 0) - left;
        }
      } else if (warp == 0) {
        // The group of digits, then the digit, two of them a lane.
        int c = 0;
#pragma unroll
        for (int p = 0; p < kMaxCluster; p++)
          if (p < parts) c += cluster.map_shared_rank(s_coarse[pass], p)[31 - lane];
        int upto = scan_up(c);
        int src = __ffs(__ballot_sync(0xffffffffu, upto >= need)) - 1;
        const int left = need - __shfl_sync(0xffffffffu, upto - c, src);
        const int top = (31 - src) * kGroup + kGroup - 2 - 2 * lane;  // this lane's lower digit
        int2 both = make_int2(0, 0);
#pragma unroll
        for (int p = 0; p < kMaxCluster; p++)
          if (p < parts) {
            const int2 v = *reinterpret_cast<const int2*>(cluster.map_shared_rank(hist, p) + top);
            both.x += v.x, both.y += v.y;
          }
        upto = scan_up(both.x + both.y);
        src = __ffs(__ballot_sync(0xffffffffu, upto >= left)) - 1;
        if (lane == src) {
          const int rest = left - (upto - both.x - both.y);  // after the digits above this lane's
          const bool upper = both.y >= rest;
          s_digit = upper ? top + 1 : top;
          s_left = upper ? rest : rest - both.y;
          s_rest = upper ? both.y - rest : both.x - (rest - both.y);
        }
      }
      __syncthreads();
      prefix |= (uint32_t)s_digit << shift, need = s_left;
      // All that share the prefix are kept: no more digits are needed.
      if (s_rest == 0 && prefix != 0) prefix -= 1, need = 0;
    }
    // Above `prefix`: kept; equal to it: the first `need`.  A kept slot's place
    // is the number of sure ones before it and of ties before it, up to `need`.
    int sure = 0, tie = 0;
#pragma unroll 4
    for (int r = 0; r < rounds; r++) {
      const uint32_t o = order_at(r);
      sure += __popc(__ballot_sync(0xffffffffu, o > prefix)), tie += __popc(__ballot_sync(0xffffffffu, o == prefix));
    }
    if (lane == 0) s_sure[warp] = sure, s_tie[warp] = tie;
    __syncthreads();
    if (warp == 0) {
      const int a1 = lane < kSelectWarps ? s_sure[lane] : 0, b1 = lane < kSelectWarps ? s_tie[lane] : 0;
      const int a0 = scan_up(a1), b0 = scan_up(b1);
      if (lane < kSelectWarps) s_sure[lane] = a0 - a1, s_tie[lane] = b0 - b1;
      if (lane == 31) s_sure[kSelectWarps] = a0, s_tie[kSelectWarps] = b0;
    }
    sync();
    sure = s_sure[warp], tie = s_tie[warp];
    for (int p = 0; p < part; p++) {
      sure += cluster.map_shared_rank(s_sure, p)[kSelectWarps];
      tie += cluster.map_shared_rank(s_tie, p)[kSelectWarps];
    }
    const unsigned below = (1u << lane) - 1;
#pragma unroll 4
    for (int r = 0; r < rounds; r++) {
      const uint32_t o = order_at(r);
      const unsigned sures = __ballot_sync(0xffffffffu, o > prefix), ties = __ballot_sync(0xffffffffu, o == prefix);
      const int tie_rank = tie + __popc(ties & below);
      if (o > prefix || (o == prefix && tie_rank < need))
        out[sure + __popc(sures & below) + min(tie_rank, need)] = (uint32_t)(slice + mine + r * 32);
      sure += __popc(sures), tie += __popc(ties);
    }
  }
  if (!ONE) cluster.sync();  // no CTA leaves while others read its shared memory
}

// Moves `rows` kept tokens of a pair: K, V and weight rows in 16-byte pieces
// (`pieces` a row; e / pieces = e · by_pieces >> 32).
constexpr int kMoveThreads = 256, kMoveRows = 64;
__global__ void __launch_bounds__(kMoveThreads)
    k_paged_move(const __grid_constant__ PagedEvictArgs a, int pieces, uint32_t by_pieces, int rows) {
  __shared__ uint32_t s_from[kMoveRows], s_to[kMoveRows];
  const int h = blockIdx.y, i = blockIdx.z, j0 = blockIdx.x * rows;
  const int count = min(min((int)a.from.lens[i], a.keep) - j0, rows);
  dependency_wait();
  if (count <= 0) return;
  if (threadIdx.x < count) {
    const int j = j0 + threadIdx.x;
    // No word of `kept` leads outside the sequence, whoever wrote it.
    const uint32_t old = min(a.kept[((size_t)i * a.key_heads + h) * a.keep + j], a.from.lens[i] - 1);
    const uint32_t from = (uint32_t)pool_row(a.from, i, (int)old, h, a.key_heads);
    const uint32_t to = (uint32_t)pool_row(a.to, i, j, h, a.key_heads);
    s_from[threadIdx.x] = from, s_to[threadIdx.x] = to;
    a.weights[to] = a.weights[from];
  }
  __syncthreads();
  const uint4 *ks = static_cast<const uint4*>(a.k), *vs = static_cast<const uint4*>(a.v);
  uint4 *kd = static_cast<uint4*>(a.k), *vd = static_cast<uint4*>(a.v);
  const int total = count * pieces;
  constexpr int kAtOnce = 4;
  for (int e0 = threadIdx.x; e0 < total; e0 += kMoveThreads * kAtOnce) {
    uint4 kw[kAtOnce], vw[kAtOnce];
    size_t to[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; u++) {
      const uint32_t e = min(e0 + u * kMoveThreads, total - 1);
      const uint32_t r = pieces == 1 ? e : __umulhi(e, by_pieces), c = e - r * pieces;
      const size_t from = (size_t)s_from[r] * pieces + c;
      to[u] = (size_t)s_to[r] * pieces + c;
      kw[u] = ks[from], vw[u] = vs[from];
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; u++)
      if (e0 + u * kMoveThreads < total) kd[to[u]] = kw[u], vd[to[u]] = vw[u];
  }
}

}  // namespace

void paged_cache_prepare() {
  const int bytes = kSelectKeys * (int)sizeof(uint32_t);
  for (auto k : {k_paged_select<false, false>, k_paged_select<false, true>, k_paged_select<true, false>,
                 k_paged_select<true, true>})
    SLM_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
}

void table_put(uint32_t* words, const uint32_t* at, const uint32_t* value, int n, cudaStream_t st) {
  Words w;
  std::memcpy(w.at, at, n * sizeof(uint32_t));
  std::memcpy(w.value, value, n * sizeof(uint32_t));
  k_table_put<<<1, 256, 0, st>>>(words, w, n);
  SLM_LAUNCHED("k_table_put");
}

void paged_store(const PagedStoreArgs& a, cudaStream_t st) {
  const bool vec = (((uintptr_t)a.ks | (uintptr_t)a.vs) & 15) == 0 && a.ldk % 4 == 0 && a.ldv % 4 == 0;
  const size_t ctas = ((size_t)a.count * a.m + kStoreThreads / 32 - 1) / (kStoreThreads / 32);
  const unsigned grid = (unsigned)std::min<size_t>(ctas, 148 * 64);
  launch_after(a.bf16 ? (vec ? k_paged_store<true, true> : k_paged_store<true, false>)
                      : (vec ? k_paged_store<false, true> : k_paged_store<false, false>),
               dim3(grid), kStoreThreads, 0, st, a);
}

void paged_evict(const PagedEvictArgs& a, cudaStream_t st) {
  // As many CTAs a pair as fill the GPU (four an SM; 93 us for 16 ragged
  // sequences of up to 32768 against 98 with two), two slots at least a thread.
  const size_t pairs = (size_t)a.from.n * a.key_heads;
  int parts = 1;
  while (parts < kMaxCluster && pairs * parts * 2 <= 148 * 4 && a.longest > 2 * kSelect * parts) parts *= 2;
  const int rounds = std::max(1, (a.longest + parts * kSelect - 1) / (parts * kSelect));
  const bool fits = rounds * kSelect <= kSelectKeys;
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)parts, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3((unsigned)(pairs * parts)), c.blockDim = dim3(kSelect), c.stream = st;
  c.dynamicSmemBytes = std::min(rounds * kSelect, kSelectKeys) * sizeof(uint32_t), c.attrs = at, c.numAttrs = 2;
  auto select = parts == 1 ? (fits ? k_paged_select<true, true> : k_paged_select<false, true>)
                           : (fits ? k_paged_select<true, false> : k_paged_select<false, false>);
  SLM_CUDA(cudaLaunchKernelEx(&c, select, a));
  const int most = std::min(a.keep, a.longest);
  if (most == 0) return;
  // e / pieces = e · by >> 32 for e < 64 · 64 (one piece: not used).
  const int pieces = a.dh * (a.bf16 ? 2 : 4) / 16, rows = std::min(kMoveRows, std::max(8, 2048 / pieces));
  const uint32_t by = (uint32_t)((((uint64_t)1 << 32) + pieces - 1) / pieces);
  launch_after(k_paged_move, dim3(cdiv(most, rows), a.key_heads, a.from.n), kMoveThreads, 0, st, a, pieces, by, rows);
}

}  // namespace slm
