// Top-k selection of key positions by score: per row the K largest of its
// first len scores, ties to the lower position, written in ascending order of
// position with -1 behind them: the index list of the attention
// (golden.py:28-66 stops at the first -1).  A score of -inf is never
// selected; NaN ranks above +inf and -0 equals +0.
//
// A score becomes an unsigned key of the same order.  One block per row finds
// the K-th largest key by four passes of 8 bits, then writes the positions
// above it and the first ties by a scan over the row.

#include <cuda_runtime.h>
#include <stdint.h>

#include "sas.h"

namespace {

constexpr int kThreads = 512;
constexpr uint32_t kNegInf = 0x007fffffu;  // key of -inf

__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kThreads)
    topk_kernel(const float* __restrict__ scores, int64_t stride, const int32_t* __restrict__ lengths,
                int n_cols, int K, int32_t* __restrict__ out) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t sh_prefix, sh_need, sh_total;
  __shared__ int warp_gt[kThreads / 32], warp_eq[kThreads / 32];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* x = scores + (size_t)row * stride;
  int32_t* o = out + (size_t)row * K;
  int n = n_cols;
  if (lengths != nullptr) n = max(0, min(n, lengths[row]));
  // Digits of the threshold key, from the top.
  uint32_t prefix = 0, need = K;
  bool all = false;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
    if (tid == 0) sh_total = 0;
    __syncthreads();
    const uint32_t high = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    for (int i = tid; i < n; i += kThreads) {
      const uint32_t k = key_of(x[i]);
      if (k > kNegInf && (k & high) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t above = 0;
      int d = 255;
      for (; d >= 0; --d) {
        if (above + hist[d] >= need) break;
        above += hist[d];
      }
      sh_total = d < 0;
      sh_prefix = prefix | ((uint32_t)max(d, 0) << shift);
      sh_need = need - above;
    }
    __syncthreads();
    if (sh_total) {  // fewer than K selectable scores: take them all
      all = true;
      break;
    }
    prefix = sh_prefix;
    need = sh_need;
    __syncthreads();
  }
  int done = 0, ties = 0;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int i = i0 + tid;
    const uint32_t k = i < n ? key_of(x[i]) : 0u;
    const bool gt = all ? k > kNegInf : k > prefix;
    const bool eq = !all && i < n && k == prefix;
    const uint32_t mg = __ballot_sync(0xffffffffu, gt), me = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) {
      warp_gt[warp] = __popc(mg);
      warp_eq[warp] = __popc(me);
    }
    __syncthreads();
    int g = done, e = ties;
    for (int w = 0; w < warp; ++w) {
      g += warp_gt[w];
      e += warp_eq[w];
    }
    const uint32_t below = (1u << lane) - 1u;
    e += __popc(me & below);
    g += __popc(mg & below);
    // Position in the output: those above before it plus the ties taken.
    const int at = g + min(e, (int)need);
    if (gt) o[all ? g : at] = i;
    if (eq && e < (int)need) o[at] = i;
    for (int w = 0; w < kThreads / 32; ++w) {
      done += warp_gt[w];
      ties += warp_eq[w];
    }
    __syncthreads();
  }
  const int filled = all ? done : K;
  for (int i = filled + tid; i < K; i += kThreads) o[i] = -1;
}

}  // namespace

extern "C" int sas_topk_select(const float* scores, int64_t score_stride, const int32_t* lengths,
                               int32_t rows, int32_t num_keys, int32_t topk, int32_t* indices,
                               void* stream_ptr) {
  if (rows < 0 || num_keys < 0 || topk < 1 || score_stride < num_keys) return SAS_ERR_INVALID;
  if (rows == 0) return SAS_OK;
  if (!indices || (num_keys > 0 && !scores)) return SAS_ERR_INVALID;
  topk_kernel<<<rows, kThreads, 0, reinterpret_cast<cudaStream_t>(stream_ptr)>>>(
      scores, score_stride, lengths, num_keys, topk, indices);
  return cudaGetLastError() == cudaSuccess ? SAS_OK : SAS_ERR_CUDA;
}
