// Index scores: how much each query token wants each key of its sequence, by
// a cheap product with narrow index keys,
//
//   score[t, j] = sum_h w[t, h] * relu(q[t, h, :] . k[j, :])     j < len(t)
//   score[t, j] = -inf                                          j >= len(t)
//
// with k[j] row j of the sequence's paged index-key cache and len(t) the
// causal threshold of the compressed positions, floor((kv - q_len + s + 1) /
// ratio) (golden.py:48-62), so that the top scores are the positions the
// attention may be given.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "sas.h"
#include "sas_internal.h"

namespace {

constexpr int kKeys = 128;

__device__ __forceinline__ void note_error(int32_t* err, int site, int detail, int extra) {
  if (err != nullptr && atomicCAS(err, 0, SAS_ERR_DEVICE) == 0) {
    err[1] = site;
    err[2] = detail;
    err[3] = extra;
  }
}

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

// Batch and keys seen of flat token t (batch -1: of no sequence).
__device__ void token_of(const SasIndexParams& p, int t, int* batch, int* len) {
  int b, s, q_len;
  if (p.max_q_len > 0) {
    b = t / p.max_q_len;
    s = t - b * p.max_q_len;
    q_len = p.cu_seqlens_q ? p.cu_seqlens_q[b + 1] - p.cu_seqlens_q[b] : p.max_q_len;
  } else {
    int lo = 0, hi = p.batch;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.cu_seqlens_q[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    s = t - p.cu_seqlens_q[b];
    q_len = b < p.batch ? p.cu_seqlens_q[b + 1] - p.cu_seqlens_q[b] : 0;
  }
  *batch = -1;
  *len = 0;
  if (b >= p.batch || s < 0 || s >= q_len) return;
  const int64_t n = sas::floordiv((int64_t)p.kv_len[b] - q_len + s + 1, p.cmp_ratio);
  *batch = b;
  *len = n < 0 ? 0 : n > p.num_keys ? p.num_keys : (int)n;
}

template <typename T>
__global__ void __launch_bounds__(kKeys) index_scores_kernel(SasIndexParams p) {
  extern __shared__ float qs[];  // [H, D] then w [H]
  const int t = p.first_token + blockIdx.y;
  int b, len;
  token_of(p, t, &b, &len);
  if (p.lengths != nullptr && blockIdx.x == 0 && threadIdx.x == 0) p.lengths[blockIdx.y] = len;
  const int j = blockIdx.x * kKeys + threadIdx.x;
  const int H = p.num_heads, D = p.head_dim;
  float score = -CUDART_INF_F;
  if ((int)blockIdx.x * kKeys < len) {
    const T* q = static_cast<const T*>(p.q) + (size_t)t * H * D;
    for (int i = threadIdx.x; i < H * D; i += kKeys) qs[i] = to_float(q[i]);
    for (int i = threadIdx.x; i < H; i += kKeys) qs[H * D + i] = p.weights[(size_t)t * H + i];
    __syncthreads();
    if (j < len) {
      const int lb = j / p.block_size;
      const int blk = lb < p.table_len ? p.block_table[(size_t)b * p.table_len + lb] : -1;
      if (blk >= p.num_blocks) note_error(p.err, 53, blk, b);
      if (blk >= 0 && blk < p.num_blocks) {
        const T* k = static_cast<const T*>(p.key_pool) +
                     ((size_t)blk * p.block_size + (j - lb * p.block_size)) * D;
        score = 0.0f;
        for (int h = 0; h < H; ++h) {
          float dot = 0.0f;
          for (int d = 0; d < D; ++d) dot += qs[h * D + d] * to_float(k[d]);
          score += qs[H * D + h] * (dot > 0.0f || dot != dot ? dot : 0.0f);
        }
      }
    }
  }
  if (j < p.num_keys && (j < len || p.fill))
    p.scores[(size_t)blockIdx.y * p.score_stride + j] = score;
}

}  // namespace

extern "C" int sas_index_scores(const SasIndexParams* params, void* stream_ptr) {
  if (!params) return SAS_ERR_INVALID;
  const SasIndexParams& p = *params;
  if (p.batch < 1 || p.total_tokens < 0 || p.max_q_len < 0 || p.num_keys < 0 ||
      p.block_size < 1 || p.num_blocks < 0 || p.table_len < 0 || p.cmp_ratio < 1 ||
      p.score_stride < p.num_keys || p.first_token < 0 || p.num_tokens < 0 ||
      (int64_t)p.first_token + p.num_tokens > p.total_tokens)
    return SAS_ERR_INVALID;
  if (p.dtype != SAS_DTYPE_BF16 && p.dtype != SAS_DTYPE_FP16) return SAS_ERR_UNSUPPORTED;
  if (p.num_heads < 1 || p.num_heads > SAS_MAX_INDEX_HEADS || p.head_dim < 8 ||
      p.head_dim % 8 != 0 || p.head_dim > SAS_MAX_INDEX_DIM ||
      (int64_t)p.num_blocks * p.block_size > INT32_MAX)
    return SAS_ERR_UNSUPPORTED;
  if (p.max_q_len > 0 && (int64_t)p.max_q_len * p.batch != p.total_tokens) return SAS_ERR_INVALID;
  if (p.num_tokens == 0 || (p.num_keys == 0 && !p.lengths)) return SAS_OK;
  if (!p.q || !p.weights || !p.key_pool || !p.block_table || !p.kv_len || !p.scores ||
      (p.max_q_len == 0 && !p.cu_seqlens_q))
    return SAS_ERR_INVALID;
  if (((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.key_pool)) & 15) != 0)
    return SAS_ERR_INVALID;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  const int keys = p.num_keys > 0 ? p.num_keys : 1;
  const dim3 grid((keys + kKeys - 1) / kKeys, p.num_tokens);
  const size_t smem = (size_t)p.num_heads * (p.head_dim + 1) * sizeof(float);
  auto* kernel = p.dtype == SAS_DTYPE_BF16 ? index_scores_kernel<__nv_bfloat16>
                                           : index_scores_kernel<__half>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
      cudaSuccess)
    return SAS_ERR_CUDA;
  kernel<<<grid, kKeys, smem, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? SAS_OK : SAS_ERR_CUDA;
}
