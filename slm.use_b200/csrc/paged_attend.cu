// Attention of one new token per sequence over a paged key-value cache.
//
//   p_s = exp(x_s - max x) / Σ exp(x - max x),  x_s = scale · q·k_s,  y = Σ p_s v_s
//
// over the visible slots, in one pass: a running maximum m, the sum l of
// exp(x - m) and the sum of exp(x - m) v, all f32, rescaled when m rises.
#include <cuda_bf16.h>

#include "common.cuh"
#include "paged.cuh"

namespace slm {

namespace {

constexpr int kWarps = 8, kMaxDh = 256;

template <bool BF16>
__device__ __forceinline__ float value_at(const void* p, size_t at) {
  return BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]) : static_cast<const float*>(p)[at];
}

// One CTA per (query head, sequence), a warp per slot.
template <bool BF16>
__global__ void __launch_bounds__(kWarps * 32) k_paged_attend(PagedAttendArgs a, float* score, float* stat) {
  __shared__ float acc_s[kWarps][kMaxDh], m_s[kWarps], l_s[kWarps];
  const int h = blockIdx.x, i = blockIdx.y, kh = h / (a.heads / a.key_heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = (int)a.t.lens[i], lo = a.reach && n > a.reach ? (int)(n - a.reach) : 0;
  const float* q = a.q + i * a.ldq + (size_t)h * a.dh;
  const size_t cap = (size_t)a.t.per * a.t.page;
  float qr[kMaxDh / 32], acc[kMaxDh / 32], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int j = 0; j < kMaxDh / 32; j++) qr[j] = lane + 32 * j < a.dh ? q[lane + 32 * j] : 0.0f, acc[j] = 0.0f;
  for (int s = lo + warp; s < n; s += kWarps) {
    const size_t row =
        ((size_t)a.t.ids[(size_t)i * a.t.per + s / a.t.page] * a.key_heads + kh) * a.t.page + s % a.t.page;
    float x = 0.0f;
#pragma unroll
    for (int j = 0; j < kMaxDh / 32; j++)
      if (lane + 32 * j < a.dh) x = fmaf(qr[j], value_at<BF16>(a.k, row * a.dh + lane + 32 * j), x);
    x = warp_sum(x) * a.scale;
    if (score && lane == 0) score[((size_t)i * a.heads + h) * cap + s] = x;
    const float top = fmaxf(m, x), keep = expf(m - top), p = expf(x - top);
    m = top, l = l * keep + p;
#pragma unroll
    for (int j = 0; j < kMaxDh / 32; j++)
      if (lane + 32 * j < a.dh) acc[j] = acc[j] * keep + p * value_at<BF16>(a.v, row * a.dh + lane + 32 * j);
  }
  if (lane == 0) m_s[warp] = m, l_s[warp] = l;
#pragma unroll
  for (int j = 0; j < kMaxDh / 32; j++) acc_s[warp][lane + 32 * j] = acc[j];
  __syncthreads();
  float top = -INFINITY, total = 0.0f;
  for (int w = 0; w < kWarps; w++) top = fmaxf(top, m_s[w]);
  for (int w = 0; w < kWarps; w++) total += l_s[w] > 0.0f ? l_s[w] * expf(m_s[w] - top) : 0.0f;
  for (int d = threadIdx.x; d < a.dh; d += kWarps * 32) {
    float y = 0.0f;
    for (int w = 0; w < kWarps; w++) y += l_s[w] > 0.0f ? acc_s[w][d] * expf(m_s[w] - top) : 0.0f;
    a.y[((size_t)i * a.heads + h) * a.dh + d] = n > 0 ? y / total : 0.0f;
  }
  if (stat && threadIdx.x == 0) {
    stat[2 * ((size_t)i * a.heads + h)] = top;
    stat[2 * ((size_t)i * a.heads + h) + 1] = total;
  }
}

// weight[s] += Σ_h p_s over the key head's query heads; a CTA per (key head, sequence).
__global__ void k_paged_weights(PagedAttendArgs a, const float* score, const float* stat) {
  const int kh = blockIdx.x, i = blockIdx.y, group = a.heads / a.key_heads;
  const int n = (int)a.t.lens[i], lo = a.reach && n > a.reach ? (int)(n - a.reach) : 0;
  const size_t cap = (size_t)a.t.per * a.t.page;
  for (int s = lo + threadIdx.x; s < n; s += blockDim.x) {
    float sum = 0.0f;
    for (int g = 0; g < group; g++) {
      const size_t head = (size_t)i * a.heads + kh * group + g;
      sum += expf(score[head * cap + s] - stat[2 * head]) / stat[2 * head + 1];
    }
    a.weights[((size_t)a.t.ids[(size_t)i * a.t.per + s / a.t.page] * a.key_heads + kh) * a.t.page + s % a.t.page] +=
        sum;
  }
}

}  // namespace

size_t paged_attend_scratch(const PagedAttendArgs& a) {
  const size_t heads = (size_t)a.t.n * a.heads;
  return a.weights ? heads * ((size_t)a.t.per * a.t.page + 2) : 1;
}

void paged_attend(const PagedAttendArgs& a, cudaStream_t st) {
  const size_t heads = (size_t)a.t.n * a.heads;
  float* score = a.weights ? a.scratch + 2 * heads : nullptr;
  float* stat = a.weights ? a.scratch : nullptr;
  const dim3 grid(a.heads, a.t.n);
  if (a.bf16)
    k_paged_attend<true><<<grid, kWarps * 32, 0, st>>>(a, score, stat);
  else
    k_paged_attend<false><<<grid, kWarps * 32, 0, st>>>(a, score, stat);
  SLM_LAUNCHED("k_paged_attend");
  if (a.weights) {
    k_paged_weights<<<dim3(a.key_heads, a.t.n), 256, 0, st>>>(a, score, stat);
    SLM_LAUNCHED("k_paged_weights");
  }
}

}  // namespace slm
