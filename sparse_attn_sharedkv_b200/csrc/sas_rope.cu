// Norm and rotation of attention rows: the query heads before the attention
// (sas_norm_rope) and the key rows on their way into a paged cache
// (sas_kv_append_norm_rope).
//
// One row x[0 .. D) becomes
//   y[c] = x[c] * rsqrt(mean(x[0 .. n)^2) + eps) * w[c]     c < n (norm_dim)
//   y[c] = x[c]                                             c >= n
// and the last `rope` columns of y are then rotated by the angles of the
// row's position: pairs (2 i, 2 i + 1) interleaved or (i, i + rope / 2) by
// halves, with (cos, sin) from tables [positions, rope / 2]; `inverse` turns
// the other way.  Statistics and products are fp32, rounded once at the end.
//
// HBM-bound: every row is read once and written once, as 16-byte vectors.  A
// group of G lanes (8, 16 or 32 by the row's width) holds whole rows in
// registers, so the mean square is a shuffle reduction inside the group and
// no shared memory is used.  With many rows a group takes four heads of a
// token at a time: their loads are in flight together, and the position, the
// angles and the weights are read once for the four.  The partner of a column
// rotated by halves is in another lane and is read a second time (an L1 hit).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "sas.h"

namespace {

constexpr int kThreads = 256;

struct RowArgs {
  const float* cosv;
  const float* sinv;
  const void* weight;
  int32_t table_rows, half, dim, norm_dim;
  float eps, inv_n, sign;
  bool weight_f32, interleaved;
};

template <bool kBf16>
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 p;
    if constexpr (kBf16)
      p = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
    else
      p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}

template <bool kBf16>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kBf16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p));
  const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
  f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

// Eight weights of a row's columns c .. c + 7.
template <bool kBf16>
__device__ __forceinline__ void load_weight(const RowArgs& a, int c, float (&w)[8]) {
  if (a.weight_f32)
    load8(static_cast<const float*>(a.weight) + c, w);
  else
    unpack8<kBf16>(
        __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.weight) + c)), w);
}

// `rows` <= R rows at src (src_stride elements apart) transformed into dst by
// a group of G lanes (lane `gl`), V vectors of 8 columns each.  `pos`: the
// rows' rotation position, checked by the caller.  src == dst is allowed:
// every load is before the group's synchronisation, every store behind it.
// Columns past norm_dim keep a factor of one; at most one of a lane's vectors
// is rotated (rope_dim <= 8 G).
template <int G, int V, int R, bool kBf16>
__device__ __forceinline__ void transform_rows(const RowArgs& a, const uint16_t* src,
                                               int64_t src_stride, uint16_t* dst,
                                               int64_t dst_stride, int rows, int64_t pos, int gl,
                                               uint32_t mask) {
  const int rot0 = a.dim - 2 * a.half;
  uint4 raw[R][V];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * G + gl) * 8;
      raw[r][v] = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows && c < a.dim)
        raw[r][v] = *reinterpret_cast<const uint4*>(src + r * src_stride + c);
    }
  // The lane's rotated vector: columns rc .. rc + 7, -1 without one; by
  // halves its partner is at columns pc.
  int rc = -1, pc = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (v * G + gl) * 8;
    if (a.half > 0 && c >= rot0 && c < a.dim) rc = c;
  }
  float4 cs[2], sn[2];
  uint4 part[R];
  const bool low = rc - rot0 < a.half;
  if (rc >= 0) {
    const int rel = rc - rot0;
    if (a.interleaved) {
      const size_t o = (size_t)pos * a.half + (rel >> 1);
      cs[0] = __ldg(reinterpret_cast<const float4*>(a.cosv + o));
      sn[0] = __ldg(reinterpret_cast<const float4*>(a.sinv + o));
    } else {
      pc = low ? rc + a.half : rc - a.half;
      const size_t o = (size_t)pos * a.half + (low ? rel : rel - a.half);
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r < rows) part[r] = *reinterpret_cast<const uint4*>(src + r * src_stride + pc);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        cs[i] = __ldg(reinterpret_cast<const float4*>(a.cosv + o) + i);
        sn[i] = __ldg(reinterpret_cast<const float4*>(a.sinv + o) + i);
      }
    }
  }
  float scale[R];
#pragma unroll
  for (int r = 0; r < R; ++r) scale[r] = 1.0f;
  if (a.norm_dim > 0) {
    float sum[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      sum[r] = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if ((v * G + gl) * 8 < a.norm_dim) {
          float f[8];
          unpack8<kBf16>(raw[r][v], f);
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[r] += f[i] * f[i];
        }
      }
    }
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1)
#pragma unroll
      for (int r = 0; r < R; ++r) sum[r] += __shfl_xor_sync(mask, sum[r], o);
#pragma unroll
    for (int r = 0; r < R; ++r) scale[r] = rsqrtf(sum[r] * a.inv_n + a.eps);
  }
  __syncwarp(mask);
  // The rows stay packed: unpacked again below rather than kept as floats.
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int v = 0; v < V; ++v)
      asm volatile("" : "+r"(raw[r][v].x), "+r"(raw[r][v].y), "+r"(raw[r][v].z), "+r"(raw[r][v].w));
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (v * G + gl) * 8;
    if (c >= a.dim) continue;
    const bool normed = c < a.norm_dim, rotated = c == rc;
    float w[8], wp[8];
    const bool weighted = normed && a.weight != nullptr;
    if (weighted) load_weight<kBf16>(a, c, w);
    const bool partner = rotated && !a.interleaved;
    const bool p_weighted = partner && pc < a.norm_dim && a.weight != nullptr;
    if (p_weighted) load_weight<kBf16>(a, pc, wp);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r >= rows) continue;
      float f[8];
      unpack8<kBf16>(raw[r][v], f);
      if (normed) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= scale[r];
      }
      if (weighted) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= w[i];
      }
      if (rotated) {
        if (a.interleaved) {
          const float co[4] = {cs[0].x, cs[0].y, cs[0].z, cs[0].w};
          const float si[4] = {sn[0].x, sn[0].y, sn[0].z, sn[0].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float s = a.sign * si[i], x0 = f[2 * i], x1 = f[2 * i + 1];
            f[2 * i] = x0 * co[i] - x1 * s;
            f[2 * i + 1] = x1 * co[i] + x0 * s;
          }
        } else {
          const float sg = low ? -a.sign : a.sign;
          float p[8];
          unpack8<kBf16>(part[r], p);
          if (pc < a.norm_dim) {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] *= scale[r];
          }
          if (p_weighted) {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] *= wp[i];
          }
          const float co[8] = {cs[0].x, cs[0].y, cs[0].z, cs[0].w,
                               cs[1].x, cs[1].y, cs[1].z, cs[1].w};
          const float si[8] = {sn[0].x, sn[0].y, sn[0].z, sn[0].w,
                               sn[1].x, sn[1].y, sn[1].z, sn[1].w};
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = f[i] * co[i] + p[i] * (sg * si[i]);
        }
      }
      *reinterpret_cast<uint4*>(dst + r * dst_stride + c) = pack8<kBf16>(f);
    }
  }
}

__device__ __forceinline__ void note_error(int32_t* err, int site, int detail, int extra) {
  if (err != nullptr && atomicCAS(err, 0, SAS_ERR_DEVICE) == 0) {
    err[1] = site;
    err[2] = detail;
    err[3] = extra;
  }
}

struct HeadArgs {
  const uint16_t* x;
  uint16_t* out;
  const void* positions;
  int32_t* err;
  int64_t x_t, x_h, o_t, o_h;
  int32_t heads;
  int32_t chunks;  // of R heads a token
  int32_t tasks;   // tokens * chunks
  bool pos64;
};

// Blocks an SM: registers for the rows in flight, 128 a thread for four rows of
// up to 768 columns, 64 for one.
template <int G, int V, int R, bool kBf16>
__global__ void __launch_bounds__(kThreads, R == 1 ? 4 : V < 4 ? 2 : 1) norm_rope_kernel(RowArgs a, HeadArgs h) {
  const int64_t task = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
  if (task >= h.tasks) return;
  const int gl = threadIdx.x & (G - 1);
  const uint32_t mask = G == 32 ? 0xffffffffu : ((1u << G) - 1u) << (threadIdx.x & 31 & ~(G - 1));
  const int t = (int)task / h.chunks, head = ((int)task - t * h.chunks) * R;
  const int rows = min(R, h.heads - head);
  int64_t pos = 0;
  uint16_t* dst = h.out + t * h.o_t + head * h.o_h;
  if (a.half > 0) {
    pos = h.pos64 ? __ldg(static_cast<const long long*>(h.positions) + t)
                  : (long long)__ldg(static_cast<const int32_t*>(h.positions) + t);
    if (pos < 0 || pos >= a.table_rows) {
      if (gl == 0) note_error(h.err, 52, t, head);
      for (int r = 0; r < rows; ++r)
        for (int c = gl * 8; c < a.dim; c += G * 8)
          *reinterpret_cast<uint4*>(dst + r * h.o_h + c) = make_uint4(0u, 0u, 0u, 0u);
      return;
    }
  }
  transform_rows<G, V, R, kBf16>(a, h.x + t * h.x_t + head * h.x_h, h.x_h, dst, h.o_h, rows, pos,
                                 gl, mask);
}

struct AppendArgs {
  uint16_t* pool;
  const uint16_t* rows;
  const int32_t* table;
  const int32_t* cu;
  const int32_t* start;
  int32_t* err;
  int32_t num_blocks, block_size, table_len, batch, total, ratio;
};

template <int G, int V, bool kBf16>
__global__ void __launch_bounds__(kThreads, 4) append_norm_rope_kernel(RowArgs a, AppendArgs p) {
  const int64_t row64 = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
  if (row64 >= p.total) return;
  const int row = (int)row64;
  const int gl = threadIdx.x & (G - 1);
  const int shift = threadIdx.x & 31 & ~(G - 1);
  const uint32_t mask = G == 32 ? 0xffffffffu : ((1u << G) - 1u) << shift;
  // The row's batch: the last b with cu[b] <= row, G probes a step.
  int lo = 0, hi = p.batch;
  while (lo < hi) {
    const int step = (hi - lo + G) / G;
    const int at = lo + gl * step;
    const bool le = at <= hi && __ldg(p.cu + at) <= row;
    const int n = __popc(__ballot_sync(mask, le));
    if (n == 0) break;
    lo += (n - 1) * step;
    hi = min(hi, lo + step - 1);
  }
  const int first = __ldg(p.cu + lo);
  // Rows before the first or behind the last sequence belong to none.
  if (lo >= p.batch || row < first) return;
  const int64_t pos = (int64_t)__ldg(p.start + lo) + (row - first);
  const int64_t lb = pos >= 0 ? pos / p.block_size : -1;
  const int blk =
      (lb >= 0 && lb < p.table_len) ? __ldg(p.table + (size_t)lo * p.table_len + lb) : -1;
  if (blk < 0 || blk >= p.num_blocks) {
    if (gl == 0) note_error(p.err, 50, row, lo);
    return;
  }
  const int64_t rot = pos * p.ratio;
  if (a.half > 0 && rot >= a.table_rows) {
    if (gl == 0) note_error(p.err, 51, row, lo);
    return;
  }
  transform_rows<G, V, 1, kBf16>(
      a, p.rows + (size_t)row * a.dim, 0,
      p.pool + ((size_t)blk * p.block_size + (size_t)(pos - lb * p.block_size)) * a.dim, 0, 1, rot,
      gl, mask);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int row_args(const SasRowTransform* tr, RowArgs* a) {
  if (tr->dtype != SAS_DTYPE_BF16 && tr->dtype != SAS_DTYPE_FP16) return SAS_ERR_UNSUPPORTED;
  if (tr->head_dim < 8 || tr->head_dim % 8 != 0) return SAS_ERR_INVALID;
  if (tr->head_dim > SAS_MAX_ROW_DIM) return SAS_ERR_UNSUPPORTED;
  if (tr->norm_dim < 0 || tr->norm_dim > tr->head_dim || tr->norm_dim % 8 != 0)
    return SAS_ERR_INVALID;
  if (tr->rope_dim < 0 || tr->rope_dim > tr->head_dim || tr->rope_dim % 16 != 0)
    return SAS_ERR_INVALID;
  if (tr->rope_dim > SAS_MAX_ROPE_DIM) return SAS_ERR_UNSUPPORTED;
  if (tr->norm_dim > 0 && !(tr->eps >= 0.0f)) return SAS_ERR_INVALID;
  if (tr->rope_dim > 0 &&
      (!tr->cos || !tr->sin || !aligned16(tr->cos) || !aligned16(tr->sin) || tr->table_rows < 0))
    return SAS_ERR_INVALID;
  if (tr->norm_weight != nullptr) {
    if (!aligned16(tr->norm_weight)) return SAS_ERR_INVALID;
    if (tr->weight_dtype != SAS_DTYPE_F32 && tr->weight_dtype != tr->dtype)
      return SAS_ERR_UNSUPPORTED;
  }
  *a = RowArgs{tr->cos,
               tr->sin,
               tr->norm_weight,
               tr->table_rows,
               tr->rope_dim / 2,
               tr->head_dim,
               tr->norm_dim,
               tr->eps,
               tr->norm_dim > 0 ? 1.0f / (float)tr->norm_dim : 0.0f,
               tr->inverse ? -1.0f : 1.0f,
               tr->weight_dtype == SAS_DTYPE_F32,
               tr->interleaved != 0};
  return SAS_OK;
}

// Launches kernel<G, V, ..., bf16> over `tasks` groups, with the group and
// the vectors a lane that hold a row of `dim` columns: the smallest G whose
// lanes hold it at one vector each, else whole warps at up to 4 vectors.
#define SAS_ROW_LAUNCH(G, KERNEL_BF16, KERNEL_FP16, ...)                                  \
  do {                                                                                    \
    const unsigned blocks = (unsigned)((tasks + kThreads / (G)-1) / (kThreads / (G)));    \
    if (bf16)                                                                             \
      KERNEL_BF16<<<blocks, kThreads, 0, stream>>>(__VA_ARGS__);                          \
    else                                                                                  \
      KERNEL_FP16<<<blocks, kThreads, 0, stream>>>(__VA_ARGS__);                          \
  } while (0)

template <int R>
void launch_heads(const RowArgs& a, const HeadArgs& h, bool bf16, cudaStream_t stream) {
  const int64_t tasks = h.tasks;
#define SAS_HEADS(G, V) \
  SAS_ROW_LAUNCH(G, (norm_rope_kernel<G, V, R, true>), (norm_rope_kernel<G, V, R, false>), a, h)
  if (a.dim <= 64) SAS_HEADS(8, 1);
  else if (a.dim <= 128) SAS_HEADS(16, 1);
  else if (a.dim <= 256) SAS_HEADS(32, 1);
  else if (a.dim <= 512) SAS_HEADS(32, 2);
  else if (a.dim <= 768) SAS_HEADS(32, 3);
  else SAS_HEADS(32, 4);
#undef SAS_HEADS
}

void launch_append(const RowArgs& a, const AppendArgs& p, bool bf16, cudaStream_t stream) {
  const int64_t tasks = p.total;
#define SAS_APPEND(G, V)                                                                    \
  SAS_ROW_LAUNCH(G, (append_norm_rope_kernel<G, V, true>), (append_norm_rope_kernel<G, V, false>), \
                 a, p)
  if (a.dim <= 64) SAS_APPEND(8, 1);
  else if (a.dim <= 128) SAS_APPEND(16, 1);
  else if (a.dim <= 256) SAS_APPEND(32, 1);
  else if (a.dim <= 512) SAS_APPEND(32, 2);
  else if (a.dim <= 768) SAS_APPEND(32, 3);
  else SAS_APPEND(32, 4);
#undef SAS_APPEND
}

}  // namespace

extern "C" int sas_norm_rope(const SasRowTransform* tr, const void* x, int64_t x_stride_token,
                             int64_t x_stride_head, void* out, int64_t out_stride_token,
                             int64_t out_stride_head, int32_t tokens, int32_t heads,
                             const void* positions, int32_t positions_i64, int32_t* err,
                             void* stream_ptr) {
  if (!tr || tokens < 0 || heads < 0) return SAS_ERR_INVALID;
  RowArgs a;
  const int rc = row_args(tr, &a);
  if (rc != SAS_OK) return rc;
  const int64_t rows = (int64_t)tokens * heads;
  if (rows == 0) return SAS_OK;
  if (rows > INT32_MAX) return SAS_ERR_UNSUPPORTED;
  if (!x || !out || (a.half > 0 && !positions)) return SAS_ERR_INVALID;
  if (!aligned16(x) || !aligned16(out) || (x_stride_token | x_stride_head | out_stride_token |
                                           out_stride_head) % 8 != 0)
    return SAS_ERR_INVALID;
  // Four heads a group where that still leaves every SM sixteen warps or more;
  // fewer rows are spread one a group for the shortest time.
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return SAS_ERR_CUDA;
  const int per = heads >= 4 && rows / 4 >= 16 * (int64_t)sms ? 4 : 1;
  const int chunks = (heads + per - 1) / per;
  const HeadArgs h{static_cast<const uint16_t*>(x), static_cast<uint16_t*>(out), positions, err,
                   x_stride_token, x_stride_head, out_stride_token, out_stride_head, heads, chunks,
                   tokens * chunks, positions_i64 != 0};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  const bool bf16 = tr->dtype == SAS_DTYPE_BF16;
  if (per == 4)
    launch_heads<4>(a, h, bf16, stream);
  else
    launch_heads<1>(a, h, bf16, stream);
  return cudaGetLastError() == cudaSuccess ? SAS_OK : SAS_ERR_CUDA;
}

extern "C" int sas_kv_append_norm_rope(const SasRowTransform* tr, void* pool, int32_t num_blocks,
                                       int32_t block_size, const int32_t* block_table,
                                       int32_t table_len, const void* new_rows,
                                       const int32_t* cu_new, const int32_t* start_pos,
                                       int32_t batch, int32_t total_new, int32_t cmp_ratio,
                                       int32_t* err, void* stream_ptr) {
  if (!tr || total_new < 0 || batch <= 0 || block_size <= 0 || num_blocks < 0 || table_len < 0 ||
      cmp_ratio < 1)
    return SAS_ERR_INVALID;
  RowArgs a;
  const int rc = row_args(tr, &a);
  if (rc != SAS_OK) return rc;
  if (total_new == 0) return SAS_OK;
  if (!pool || !block_table || !new_rows || !cu_new || !start_pos) return SAS_ERR_INVALID;
  if (!aligned16(pool) || !aligned16(new_rows)) return SAS_ERR_INVALID;
  const AppendArgs p{static_cast<uint16_t*>(pool), static_cast<const uint16_t*>(new_rows),
                     block_table, cu_new, start_pos, err, num_blocks, block_size, table_len, batch,
                     total_new, cmp_ratio};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  launch_append(a, p, tr->dtype == SAS_DTYPE_BF16, stream);
  return cudaGetLastError() == cudaSuccess ? SAS_OK : SAS_ERR_CUDA;
}
