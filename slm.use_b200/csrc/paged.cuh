// Paged key-value caches: what the host side (paged.cpp) hands the kernels.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "common.cuh"

namespace slm {

// The paged kernels begin while the one before them in the stream still runs
// (launch_after): what follows `dependency_wait` sees all that it wrote.  Every
// thread block waits, so a kernel is done only after the one before it; and all
// but the second kernels of a call wait before they let the next one begin, so
// a second kernel may read what older kernels wrote (the table) at once.
__device__ __forceinline__ void dependents_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launches a kernel that begins while the one before it still runs.
template <class... P, class... A>
inline void launch_after(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = grid, c.blockDim = dim3(threads), c.dynamicSmemBytes = smem, c.stream = st, c.attrs = &at, c.numAttrs = 1;
  SLM_CUDA(cudaLaunchKernelEx(&c, kernel, P(args)...));
}


// A table on the device and the pool's geometry.  Row s of sequence i, key
// head h is row (ids[i·per + s / page] · key_heads + h) · page + s % page of
// the pool's K, V ([rows][dh]) and weights ([rows]).
struct PagedTable {
  const uint32_t* lens = nullptr;
  const uint32_t* ids = nullptr;
  int n = 0, per = 0;
  uint32_t page = 0;
  // page_of(s) = s / page for s < 2^30: s · mul >> shift with mul =
  // ⌈2^(30+k) / page⌉, k = ⌈log2 page⌉ (mul · page - 2^(30+k) < 2^k, so the
  // quotient's error stays below 1 / page).
  uint32_t mul = 0, shift = 0;
  void set_page(uint32_t p) {
    uint32_t k = 0;
    while ((1u << k) < p) k++;
    page = p, shift = 30 + k;
    mul = (uint32_t)((((uint64_t)1 << shift) + p - 1) / p);
  }
  __host__ __device__ uint32_t page_of(uint32_t s) const { return (uint32_t)((uint64_t)s * mul >> shift); }
};

struct PagedStoreArgs {
  PagedTable t;
  int first, count, m, key_heads, dh;
  bool bf16;
  const float *ks, *vs;
  long long ldk, ldv;
  void *k, *v;
  float* weights;  // or null
};
void paged_store(const PagedStoreArgs& a, cudaStream_t st);

struct PagedAttendArgs {
  PagedTable t;
  const uint32_t* host_lens;  // the lengths the launch is shaped by (the table's)
  int heads, key_heads, dh;
  long long reach;  // 0: all
  float scale;
  bool bf16;
  const float* q;
  long long ldq;
  const void *k, *v;
  float* weights;  // or null
  float* y;
  float* scratch;  // paged_attend_scratch(a) floats, 16-byte aligned
};
// Shared-memory limits of the kernels, once per device.
void paged_prepare();
size_t paged_attend_scratch(const PagedAttendArgs& a);
void paged_attend(const PagedAttendArgs& a, cudaStream_t st);

struct PagedEvictArgs {
  PagedTable from, to;
  int key_heads, dh;
  bool bf16;
  int keep, sinks, recent;
  int longest;  // the longest sequence's tokens
  void *k, *v;
  float* weights;
  uint32_t* kept;  // [n][key_heads][keep]
};
void paged_cache_prepare();  // as paged_prepare
void paged_evict(const PagedEvictArgs& a, cudaStream_t st);

// words[at[j]] = value[j] for j < n (≤ kPutWords): table updates, by value in
// the launch parameters, so nothing on the host has to outlive the call.
constexpr int kPutWords = 480;
void table_put(uint32_t* words, const uint32_t* at, const uint32_t* value, int n, cudaStream_t st);

}  // namespace slm
