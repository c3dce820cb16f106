// Storing tokens into the pages of a paged cache, evicting tokens from it, and
// updates of its tables (checked on the host, paged.cpp).
#include <cuda_bf16.h>

#include <cstring>

#include "common.cuh"
#include "paged.cuh"

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

// One warp per (token, key head): grid-stride over them.
template <bool BF16>
__global__ void k_paged_store(PagedStoreArgs a) {
  const int lane = threadIdx.x & 31;
  const long long total = (long long)a.count * a.m * a.key_heads;
  for (long long w = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); w < total;
       w += (long long)gridDim.x * (blockDim.x >> 5)) {
    const int h = (int)(w % a.key_heads);
    const long long tok = w / a.key_heads;
    const int i = a.first + (int)(tok / a.m), j = (int)(tok % a.m);
    const int s = (int)((long long)a.t.lens[i] - a.m + j);
    if (s < 0) continue;
    const size_t row = pool_row(a.t, i, s, h, a.key_heads);
    const float* ks = a.ks + tok * a.ldk + (size_t)h * a.dh;
    const float* vs = a.vs + tok * a.ldv + (size_t)h * a.dh;
    for (int d = lane; d < a.dh; d += 32) {
      if (BF16) {
        static_cast<__nv_bfloat16*>(a.k)[row * a.dh + d] = __float2bfloat16_rn(ks[d]);
        static_cast<__nv_bfloat16*>(a.v)[row * a.dh + d] = __float2bfloat16_rn(vs[d]);
      } else {
        static_cast<float*>(a.k)[row * a.dh + d] = ks[d];
        static_cast<float*>(a.v)[row * a.dh + d] = vs[d];
      }
    }
    if (a.weights && lane == 0) a.weights[row] = 0.0f;
  }
}

// Order of the weights as unsigned integers: NaN lowest, the two zeros equal.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0;
  const uint32_t b = __float_as_uint(w + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int kSelect = 1024;

// Exclusive prefix of a 0/1 flag over the CTA, and its total.
__device__ int block_rank(bool flag, int* total) {
  __shared__ int part[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned votes = __ballot_sync(0xffffffffu, flag);
  __syncthreads();
  if (lane == 0) part[warp] = __popc(votes);
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kSelect / 32; w++) {
    if (w < warp) before += part[w];
    all += part[w];
  }
  *total = all;
  return before + __popc(votes & ((1u << lane) - 1));
}

// One CTA per (key head, sequence): the kept slots in order.  The threshold is
// found digit by digit (8 bits a pass over the weights), then one ordered pass
// writes the slots above it and the first of those equal to it.
__global__ void __launch_bounds__(kSelect) k_paged_select(PagedEvictArgs a) {
  __shared__ int hist[256];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int h = blockIdx.x, i = blockIdx.y, t = threadIdx.x;
  const int n = (int)a.from.lens[i];
  uint32_t* out = a.kept + ((size_t)i * a.key_heads + h) * a.keep;
  if (n <= a.keep) {
    for (int j = t; j < a.keep; j += kSelect) out[j] = j < n ? (uint32_t)j : 0xffffffffu;
    return;
  }
  const int lo = a.sinks, hi = n - a.recent;  // the slots that compete
  uint32_t prefix = 0;
  int need = a.keep - a.sinks - a.recent;  // how many of them are kept
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (t < 256) hist[t] = 0;
    __syncthreads();
    for (int s = lo + t; s < hi; s += kSelect) {
      const uint32_t o = order_of(a.weights[pool_row(a.from, i, s, h, a.key_heads)]);
      if (shift == 24 || (o >> (shift + 8)) == prefix >> (shift + 8)) atomicAdd(&hist[(o >> shift) & 255], 1);
    }
    __syncthreads();
    if (t == 0) {
      int d = 255, left = need;
      while (d > 0 && hist[d] < left) left -= hist[d--];
      s_prefix = prefix | (uint32_t)d << shift;
      s_need = left;
    }
    __syncthreads();
    prefix = s_prefix, need = s_need;
  }
  // Above the threshold `prefix`: all; equal to it: the first `need`.
  int kept = 0, equal = 0;
  for (int base = 0; base < n; base += kSelect) {
    const int s = base + t;
    bool keep = s < n && (s < lo || s >= hi), tie = false;
    if (s >= lo && s < hi) {
      const uint32_t o = order_of(a.weights[pool_row(a.from, i, s, h, a.key_heads)]);
      keep = o > prefix;
      tie = o == prefix;
    }
    int ties, taken;
    const int before = block_rank(tie, &ties);
    keep |= tie && equal + before < need;
    const int at = block_rank(keep, &taken);
    if (keep) out[kept + at] = (uint32_t)s;
    kept += taken, equal += ties;
  }
}

// One warp per kept token: its K, V and weight rows.
__global__ void k_paged_move(PagedEvictArgs a, int row_words) {
  const int lane = threadIdx.x & 31;
  const long long total = (long long)a.from.n * a.key_heads * a.keep;
  for (long long w = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); w < total;
       w += (long long)gridDim.x * (blockDim.x >> 5)) {
    const uint32_t old = a.kept[w];
    if (old == 0xffffffffu) continue;
    const int j = (int)(w % a.keep);
    const long long pair = w / a.keep;
    const int h = (int)(pair % a.key_heads), i = (int)(pair / a.key_heads);
    const size_t src = pool_row(a.from, i, (int)old, h, a.key_heads), dst = pool_row(a.to, i, j, h, a.key_heads);
    uint32_t *k = static_cast<uint32_t*>(a.k), *v = static_cast<uint32_t*>(a.v);
    for (int d = lane; d < row_words; d += 32) {
      k[dst * row_words + d] = k[src * row_words + d];
      v[dst * row_words + d] = v[src * row_words + d];
    }
    if (lane == 0) a.weights[dst] = a.weights[src];
  }
}

}  // namespace

void table_put(uint32_t* words, const uint32_t* at, const uint32_t* value, int n, cudaStream_t st) {
  Words w;
  std::memcpy(w.at, at, n * sizeof(uint32_t));
  std::memcpy(w.value, value, n * sizeof(uint32_t));
  k_table_put<<<1, 256, 0, st>>>(words, w, n);
  SLM_LAUNCHED("k_table_put");
}

void paged_store(const PagedStoreArgs& a, cudaStream_t st) {
  const size_t warps = (size_t)a.count * a.m * a.key_heads;
  const unsigned grid = (unsigned)(warps / 8 + 1 < 148 * 8 ? warps / 8 + 1 : 148 * 8);
  if (a.bf16)
    k_paged_store<true><<<grid, 256, 0, st>>>(a);
  else
    k_paged_store<false><<<grid, 256, 0, st>>>(a);
  SLM_LAUNCHED("k_paged_store");
}

void paged_evict(const PagedEvictArgs& a, cudaStream_t st) {
  k_paged_select<<<dim3(a.key_heads, a.from.n), kSelect, 0, st>>>(a);
  SLM_LAUNCHED("k_paged_select");
  k_paged_move<<<148 * 8, 256, 0, st>>>(a, a.dh * (a.bf16 ? 2 : 4) / 4);
  SLM_LAUNCHED("k_paged_move");
}

}  // namespace slm
