// Storing tokens into the pages of a paged cache, evicting tokens from it, and
// updates of its tables (checked on the host, paged.cpp).
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <cstring>

#include "common.cuh"
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
// Evict, first part: which slots are kept.  A cluster of CTAs per pair (key
// head, sequence), each CTA a contiguous slice of its slots with their weights
// in shared memory, so memory is read once.  The lowest kept weight is found
// digit by digit from the top (11, 11, 10 bits of an order-preserving integer):
// every CTA counts its slice, the cluster's counts are added through
// distributed shared memory, and the digit that holds the last kept weight is
// the next prefix.  Latency bounds it (five cluster barriers).
// ---------------------------------------------------------------------------
constexpr int kSelect = 1024, kDigits = 2048, kMaxCluster = 8;
constexpr int kSelectKeys = 40 * 1024;  // slots of a slice that shared memory holds; longer ones are read again

// Order of the weights as unsigned integers: NaN lowest, the two zeros equal.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0;
  const uint32_t b = __float_as_uint(w + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__global__ void __launch_bounds__(kSelect) k_paged_select(const __grid_constant__ PagedEvictArgs a, int room) {
  extern __shared__ uint32_t s_order[];
  __shared__ int s_hist[3][kDigits], s_warp[32], s_digit, s_left, s_sure[33], s_tie[33];
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = cluster.num_blocks(), part = cluster.block_rank();
  const int pair = blockIdx.x / parts, h = pair % a.key_heads, i = pair / a.key_heads;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int n = (int)a.from.lens[i];
  uint32_t* out = a.kept + ((size_t)i * a.key_heads + h) * a.keep;
  dependents_launch();
  if (n <= a.keep) {  // all kept; uniform in the cluster
    for (int j = part * kSelect + t; j < a.keep; j += parts * kSelect) out[j] = j < n ? (uint32_t)j : 0xffffffffu;
    return;
  }
  for (int d = t; d < 3 * kDigits; d += kSelect) (&s_hist[0][0])[d] = 0;
  // A warp's slots lie together: 32 · rounds of them from first_slot on.
  const int rounds = (n + parts * kSelect - 1) / (parts * kSelect);
  const int slice = part * rounds * kSelect, mine = warp * rounds * 32;
  const int lo = a.sinks, hi = n - a.recent;  // the slots that compete
  auto order_at = [&](int j) -> uint32_t {    // j: in the slice
    if (j < room) return s_order[j];
    return order_of(a.weights[pool_row(a.from, i, slice + j, h, a.key_heads)]);
  };
  __syncthreads();
#pragma unroll 4
  for (int r = 0; r < rounds; r++) {
    const int j = mine + r * 32 + lane, s = slice + j;
    uint32_t o = 0;
    if (s < n) o = order_of(a.weights[pool_row(a.from, i, s, h, a.key_heads)]);
    if (j < room) s_order[j] = o;
    if (s >= lo && s < hi) atomicAdd(&s_hist[0][o >> 21], 1);
  }
  uint32_t prefix = 0;
  int need = a.keep - a.sinks - a.recent;  // how many of them are kept
#pragma unroll
  for (int pass = 0; pass < 3; pass++) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, digits = pass == 2 ? 1024 : 2048;
    if (pass > 0) {
#pragma unroll 4
      for (int r = 0; r < rounds; r++) {
        const int j = mine + r * 32 + lane, s = slice + j;
        if (s < lo || s >= hi) continue;
        const uint32_t o = order_at(j);
        if (o >> (shift + (pass == 2 ? 10 : 11)) == prefix >> (shift + (pass == 2 ? 10 : 11)))
          atomicAdd(&s_hist[pass][(o >> shift) & (digits - 1)], 1);
      }
    }
    cluster.sync();
    // Thread t: the cluster's counts of digits top - 2t and the one below, from the top.
    const int d1 = kDigits - 1 - 2 * t, d0 = d1 - 1;
    int c1 = 0, c0 = 0;
    for (int p = 0; p < parts; p++) {
      const int* from = cluster.map_shared_rank(s_hist[pass], p);
      c1 += from[d1], c0 += from[d0];
    }
    int upto = c1 + c0;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, x);
      if (lane >= x) upto += v;
    }
    if (lane == 31) s_warp[warp] = upto;
    __syncthreads();
    if (warp == 0) {
      int v = s_warp[lane];
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, x);
        if (lane >= x) v += u;
      }
      s_warp[lane] = v;
    }
    __syncthreads();
    const int above = upto - (c1 + c0) + (warp ? s_warp[warp - 1] : 0);  // counts of higher digits
    // The digit that holds the need-th largest (need 0: above all, the top digit's upper end).
    if (above < need && above + c1 + c0 >= need) {
      const bool first = above + c1 >= need;
      s_digit = first ? d1 : d0;
      s_left = need - above - (first ? 0 : c1);
    }
    if (need == 0 && t == 0) s_digit = digits - 1, s_left = 0;
    __syncthreads();
    prefix |= (uint32_t)s_digit << shift, need = s_left;
  }
  // Above `prefix`: kept; equal to it: the first `need`.  A kept slot's place is
  // the number of sure ones before it and of ties before it, up to `need`.
  int sure = 0, tie = 0;
#pragma unroll 4
  for (int r = 0; r < rounds; r++) {
    const int j = mine + r * 32 + lane, s = slice + j;
    bool is_sure = s < n && (s < lo || s >= hi), is_tie = false;
    if (s >= lo && s < hi) {
      const uint32_t o = order_at(j);
      is_sure = o > prefix, is_tie = o == prefix;
    }
    sure += __popc(__ballot_sync(0xffffffffu, is_sure)), tie += __popc(__ballot_sync(0xffffffffu, is_tie));
  }
  if (lane == 0) s_sure[warp] = sure, s_tie[warp] = tie;
  __syncthreads();
  if (warp == 0) {
    int a0 = s_sure[lane], b0 = s_tie[lane];
    const int a1 = a0, b1 = b0;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, a0, x), v = __shfl_up_sync(0xffffffffu, b0, x);
      if (lane >= x) a0 += u, b0 += v;
    }
    s_sure[lane] = a0 - a1, s_tie[lane] = b0 - b1;
    if (lane == 31) s_sure[32] = a0, s_tie[32] = b0;
  }
  cluster.sync();
  sure = s_sure[warp], tie = s_tie[warp];
  for (int p = 0; p < part; p++) {
    sure += cluster.map_shared_rank(s_sure, p)[32];
    tie += cluster.map_shared_rank(s_tie, p)[32];
  }
  const unsigned below = (1u << lane) - 1;
  for (int r = 0; r < rounds; r++) {
    const int j = mine + r * 32 + lane, s = slice + j;
    bool is_sure = s < n && (s < lo || s >= hi), is_tie = false;
    if (s >= lo && s < hi) {
      const uint32_t o = order_at(j);
      is_sure = o > prefix, is_tie = o == prefix;
    }
    const unsigned sures = __ballot_sync(0xffffffffu, is_sure), ties = __ballot_sync(0xffffffffu, is_tie);
    const int tie_rank = tie + __popc(ties & below);
    if (is_sure || (is_tie && tie_rank < need))
      out[sure + __popc(sures & below) + min(tie_rank, need)] = (uint32_t)s;
    sure += __popc(sures), tie += __popc(ties);
  }
  cluster.sync();  // no CTA leaves while others read its shared memory
}

// ---------------------------------------------------------------------------
// Evict, second part: the kept tokens' K, V and weight rows.  Bytes bound it.
// A CTA moves up to kMoveRows tokens of one pair in 16-byte pieces.
// ---------------------------------------------------------------------------
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
    const uint32_t old = a.kept[((size_t)i * a.key_heads + h) * a.keep + j];
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
      const uint32_t r = __umulhi(e, by_pieces), c = e - r * pieces;
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
  SLM_CUDA(cudaFuncSetAttribute(k_paged_select, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                kSelectKeys * (int)sizeof(uint32_t)));
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
  if (a.bf16)
    (vec ? k_paged_store<true, true> : k_paged_store<true, false>)<<<grid, kStoreThreads, 0, st>>>(a);
  else
    (vec ? k_paged_store<false, true> : k_paged_store<false, false>)<<<grid, kStoreThreads, 0, st>>>(a);
  SLM_LAUNCHED("k_paged_store");
}

void paged_evict(const PagedEvictArgs& a, cudaStream_t st) {
  // As many CTAs a pair as fill the GPU twice, with a slot at least a thread.
  const size_t pairs = (size_t)a.from.n * a.key_heads;
  int parts = 1;
  while (parts < kMaxCluster && pairs * parts * 2 <= 148 * 2 && a.longest > kSelect * parts) parts *= 2;
  const int rounds = (a.longest + parts * kSelect - 1) / (parts * kSelect);
  const int room = std::min(std::max(rounds, 1) * kSelect, kSelectKeys);
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)parts, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3((unsigned)(pairs * parts)), c.blockDim = dim3(kSelect), c.stream = st;
  c.dynamicSmemBytes = room * sizeof(uint32_t), c.attrs = &at, c.numAttrs = 1;
  SLM_CUDA(cudaLaunchKernelEx(&c, k_paged_select, a, room));
  // 16-byte pieces of a row; e / pieces = e · by >> 32 for e < 64 · 64.
  const int pieces = a.dh * (a.bf16 ? 2 : 4) / 16;
  const uint32_t by = (uint32_t)((((uint64_t)1 << 32) + pieces - 1) / pieces);
  const int rows = std::min(kMoveRows, std::max(8, 2048 / pieces));
  const int most = std::min(a.keep, a.longest);
  if (most == 0) return;
  launch_after(k_paged_move, dim3(cdiv(most, rows), a.key_heads, a.from.n), kMoveThreads, st, a, pieces, by, rows);
}

}  // namespace slm
