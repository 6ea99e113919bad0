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
// HBM-bound: every row is read once and written once, as 16-byte vectors.
// Eight lanes hold a whole row in registers, V vectors each (9 of them for 576
// columns, with no lane idle), four rows a warp: all of a row's loads are in
// flight together, the mean square takes three shuffles, and what a row costs
// besides (its token, position and address) is shared by four.  The rotated
// columns are taken apart from the others, a lane with both columns of its
// pairs, so no lane needs another's.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "sas.h"
#include "sas_kernels.h"

namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 8;  // of a row

struct RowArgs {
  const float* cosv;
  const float* sinv;
  const void* weight;
  int32_t table_rows, half, dim, norm_dim;
  float eps, inv_n, sign;
  bool weight_f32, interleaved;
};

// Pairs of fp32 in one 64-bit register: one instruction multiplies or adds both.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Eight columns as four pairs.
struct Eight {
  uint64_t p[4];
};

template <bool kBf16>
__device__ __forceinline__ Eight unpack8(const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  Eight e;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kBf16) {
      e.p[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      e.p[i] = pair(f.x, f.y);
    }
  }
  return e;
}

template <bool kBf16>
__device__ __forceinline__ uint4 pack8(const Eight& e) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpair(e.p[i]);
    if constexpr (kBf16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(f.x, f.y);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Weights of a row's columns c .. c + 7 < norm_dim.
template <bool kBf16>
__device__ __forceinline__ Eight load_weight(const RowArgs& a, int c) {
  if (!a.weight_f32)
    return unpack8<kBf16>(
        __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.weight) + c)));
  const float4* w = reinterpret_cast<const float4*>(static_cast<const float*>(a.weight) + c);
  const float4 x = __ldg(w), y = __ldg(w + 1);
  return Eight{{pair(x.x, x.y), pair(x.z, x.w), pair(y.x, y.y), pair(y.z, y.w)}};
}

// Where a row's weights come from: none, the argument, or its floats in shared
// memory.
enum Weights { kNone, kGlobal, kShared };

// Columns c .. c + 7 normed and weighted.
template <bool kBf16, Weights kW>
__device__ __forceinline__ Eight norm8(const RowArgs& a, const uint4& raw, float scale, int c,
                                       const float* sw) {
  Eight e = unpack8<kBf16>(raw);
  if (c < a.norm_dim) {
    const uint64_t k = pair(scale, scale);
#pragma unroll
    for (int i = 0; i < 4; ++i) e.p[i] = mul2(e.p[i], k);
    if constexpr (kW != kNone) {
      Eight w;
      if constexpr (kW == kShared) {
        const float4 x = *reinterpret_cast<const float4*>(sw + c);
        const float4 y = *reinterpret_cast<const float4*>(sw + c + 4);
        w = Eight{{pair(x.x, x.y), pair(x.z, x.w), pair(y.x, y.y), pair(y.z, y.w)}};
      } else {
        w = load_weight<kBf16>(a, c);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) e.p[i] = mul2(e.p[i], w.p[i]);
    }
  }
  return e;
}

// Rotated columns of one lane: eight neighbouring ones (interleaved), or eight
// of the first half and their partners of the second.
struct Turn {
  int c;  // first column, -1 for none
  uint4 x, y;
  float4 cs[2], sn[2];
};

template <bool kInter>
__device__ __forceinline__ Turn load_turn(const RowArgs& a, const uint16_t* src, int64_t pos,
                                          int i) {
  const int rot0 = a.dim - 2 * a.half;
  Turn t;
  t.c = 8 * i < (kInter ? 2 * a.half : a.half) ? rot0 + 8 * i : -1;
  if (t.c >= 0) {
    const size_t o = (size_t)pos * a.half + (kInter ? 4 * i : 8 * i);
    const float4* cp = reinterpret_cast<const float4*>(a.cosv + o);
    const float4* sp = reinterpret_cast<const float4*>(a.sinv + o);
    t.x = *reinterpret_cast<const uint4*>(src + t.c);
    t.cs[0] = __ldg(cp);
    t.sn[0] = __ldg(sp);
    if (!kInter) {
      t.y = *reinterpret_cast<const uint4*>(src + t.c + a.half);
      t.cs[1] = __ldg(cp + 1);
      t.sn[1] = __ldg(sp + 1);
    }
  }
  return t;
}

template <bool kBf16, Weights kW, bool kInter>
__device__ __forceinline__ void store_turn(const RowArgs& a, const Turn& t, uint16_t* dst,
                                           float scale, const float* sw) {
  if (t.c < 0) return;
  Eight e = norm8<kBf16, kW>(a, t.x, scale, t.c, sw);
  if constexpr (kInter) {
    const float co[4] = {t.cs[0].x, t.cs[0].y, t.cs[0].z, t.cs[0].w};
    const float si[4] = {t.sn[0].x, t.sn[0].y, t.sn[0].z, t.sn[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpair(e.p[i]);
      const float s = a.sign * si[i];
      e.p[i] = pair(f.x * co[i] - f.y * s, f.y * co[i] + f.x * s);
    }
  } else {
    Eight q = norm8<kBf16, kW>(a, t.y, scale, t.c + a.half, sw);
    const uint64_t co[4] = {pair(t.cs[0].x, t.cs[0].y), pair(t.cs[0].z, t.cs[0].w),
                            pair(t.cs[1].x, t.cs[1].y), pair(t.cs[1].z, t.cs[1].w)};
    const float si[8] = {t.sn[0].x, t.sn[0].y, t.sn[0].z, t.sn[0].w,
                         t.sn[1].x, t.sn[1].y, t.sn[1].z, t.sn[1].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float s0 = a.sign * si[2 * i], s1 = a.sign * si[2 * i + 1];
      const uint64_t lo = fma2(e.p[i], co[i], mul2(q.p[i], pair(-s0, -s1)));
      q.p[i] = fma2(q.p[i], co[i], mul2(e.p[i], pair(s0, s1)));
      e.p[i] = lo;
    }
    *reinterpret_cast<uint4*>(dst + t.c + a.half) = pack8<kBf16>(q);
  }
  *reinterpret_cast<uint4*>(dst + t.c) = pack8<kBf16>(e);
}

// Columns of the row at `src` that lane `gl` norms or passes on.
template <int V>
__device__ __forceinline__ void load_row(const RowArgs& a, const uint16_t* src, int gl,
                                         uint4 (&raw)[V]) {
  const int read = max(a.dim - 2 * a.half, a.norm_dim);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (v * kLanes + gl) * 8;
    raw[v] = make_uint4(0u, 0u, 0u, 0u);
    if (c < read) raw[v] = *reinterpret_cast<const uint4*>(src + c);
  }
}

// The row at `src`, of which load_row gave `raw`, transformed into `dst` by
// kLanes lanes (lane `gl`), V vectors of 8 columns each.  `pos`: the row's
// rotation position, checked by the caller.  src == dst is allowed: what a
// lane stores, no other lane reads, but for the norm's pass, which the lanes'
// reduction ends.
template <int V, bool kBf16, Weights kW, bool kInter>
__device__ __forceinline__ void transform_row(const RowArgs& a, uint4 (&raw)[V],
                                              const uint16_t* src, uint16_t* dst, int64_t pos,
                                              int gl, uint32_t mask, const float* sw) {
  const int straight = a.dim - 2 * a.half;  // columns before the rotated ones
  Turn t;
  t.c = -1;
  if (a.half > 0) t = load_turn<kInter>(a, src, pos, gl);
  float scale = 1.0f;
  if (a.norm_dim > 0) {
    uint64_t sum2 = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if ((v * kLanes + gl) * 8 < a.norm_dim) {
        const Eight e = unpack8<kBf16>(raw[v]);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum2 = fma2(e.p[i], e.p[i], sum2);
      }
    }
    const float2 f = unpair(sum2);
    float sum = f.x + f.y;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
    scale = rsqrtf(sum * a.inv_n + a.eps);
  }
  __syncwarp(mask);
  // The row stays packed: unpacked again below rather than kept as floats.
#pragma unroll
  for (int v = 0; v < V; ++v)
    asm volatile("" : "+r"(raw[v].x), "+r"(raw[v].y), "+r"(raw[v].z), "+r"(raw[v].w));
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (v * kLanes + gl) * 8;
    if (c < straight)
      *reinterpret_cast<uint4*>(dst + c) =
          pack8<kBf16>(norm8<kBf16, kW>(a, raw[v], scale, c, sw));
  }
  store_turn<kBf16, kW, kInter>(a, t, dst, scale, sw);
  for (int i = gl + kLanes; 4 * i < a.half; i += kLanes)
    store_turn<kBf16, kW, kInter>(a, load_turn<kInter>(a, src, pos, i), dst, scale, sw);
}

__device__ __forceinline__ void note_error(int32_t* err, int site, int detail, int extra) {
  if (err != nullptr && atomicCAS(err, 0, SAS_ERR_DEVICE) == 0) {
    err[1] = site;
    err[2] = detail;
    err[3] = extra;
  }
}

// Lanes of this thread's row.
__device__ __forceinline__ uint32_t row_mask() {
  return ((1u << kLanes) - 1u) << (threadIdx.x & 31 & ~(kLanes - 1));
}

struct HeadArgs {
  const uint16_t* x;
  uint16_t* out;
  const void* positions;
  int32_t* err;
  int64_t x_t, x_h, o_t, o_h;
  int32_t heads;
  int32_t rows;
  bool pos64;
};

// Blocks an SM: two, or where rows of up to 256 columns leave room, as many as
// were fastest.  8192 x 64 rows of 128 columns, all normed and 64 rotated, take 61
// us with four, 96 us with two, 67 us with five; by halves, which hold both columns'
// vectors, 81 us with three, 102 us with two, 87 us with four.  (The bytes need 41
// us.  By halves these instances spill 4 to 16 bytes, and the ones that read the
// weights from global memory, for few rows, 16 to 48.)
__host__ __device__ constexpr int blocks_per_sm(int v, bool interleaved) {
  return v > 4 ? 2 : interleaved ? 4 : 3;
}

// Persistent where there are more rows than the blocks that fit: of 576 columns
// 16 warps an SM with 4 rows each in flight (74 KB), weights in shared memory.  On
// 8192 x 128 rows of 576 columns this takes 382 us in a loop over the same rows (6.3
// TB/s, 97 % of the measured copy rate) and 400 us where the rows change from call to
// call; a block for every 32 rows 467 us, with the weights read from global memory a
// row.
template <int V, bool kBf16, Weights kW, bool kInter>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(V, kInter))
    norm_rope_kernel(RowArgs a, HeadArgs h) {
  __shared__ alignas(16) float sw[kW == kShared ? SAS_MAX_ROW_DIM : 4];
  if constexpr (kW == kShared) {
    for (int c = threadIdx.x * 8; c < a.norm_dim; c += kThreads * 8) {
      const Eight w = load_weight<kBf16>(a, c);
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<float2*>(sw + c + 2 * i) = unpair(w.p[i]);
    }
    __syncthreads();
  }
  const int gl = threadIdx.x & (kLanes - 1);
  const int64_t step = (int64_t)gridDim.x * (kThreads / kLanes);
  for (int64_t row = (int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
       row < h.rows; row += step) {
    const int t = (int)row / h.heads, head = (int)row - t * h.heads;
    const uint16_t* src = h.x + t * h.x_t + head * h.x_h;
    uint4 raw[V];
    load_row<V>(a, src, gl, raw);
    uint16_t* dst = h.out + t * h.o_t + head * h.o_h;
    int64_t pos = 0;
    if (a.half > 0) {
      pos = h.pos64 ? __ldg(static_cast<const long long*>(h.positions) + t)
                    : (long long)__ldg(static_cast<const int32_t*>(h.positions) + t);
      if (pos < 0 || pos >= a.table_rows) {
        if (gl == 0) note_error(h.err, 52, t, head);
        for (int c = gl * 8; c < a.dim; c += kLanes * 8)
          *reinterpret_cast<uint4*>(dst + c) = make_uint4(0u, 0u, 0u, 0u);
        continue;
      }
    }
    transform_row<V, kBf16, kW, kInter>(a, raw, src, dst, pos, gl, row_mask(), sw);
  }
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

// One row for each eight lanes.  Few rows are a chain of latencies (the search's
// probes, the page, the row): the row itself is asked for first.  8 x 4096 rows
// of 576 columns take 25 us (18 us with the rows in L2), twice what their bytes
// need: this launch goes through 3.5 rounds of such chains, and every row reads
// its weights from global memory.
template <int V, bool kBf16, Weights kW, bool kInter>
__global__ void __launch_bounds__(kThreads, 2)
    append_norm_rope_kernel(RowArgs a, AppendArgs p) {
  const int64_t row64 = (int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  if (row64 >= p.total) return;
  const int row = (int)row64;
  const int gl = threadIdx.x & (kLanes - 1);
  const uint32_t mask = row_mask();
  // The row is on its way while its place is looked up.
  const uint16_t* src = p.rows + (size_t)row * a.dim;
  uint4 raw[V];
  load_row<V>(a, src, gl, raw);
  // The row's batch: the last b with cu[b] <= row, kLanes probes a step; the
  // probes bring cu[b] and the batch's start along.
  int lo = 0, hi = p.batch, first = 0, start = 0;
  while (true) {
    const int step = (hi - lo + kLanes) / kLanes;
    const int at = lo + gl * step;
    const int cu = at <= hi ? __ldg(p.cu + at) : 0;
    const int st = at <= hi && at < p.batch ? __ldg(p.start + at) : 0;
    const int n = __popc(__ballot_sync(mask, at <= hi && cu <= row));
    if (n == 0) return;  // before the first sequence
    first = __shfl_sync(mask, cu, n - 1, kLanes);
    start = __shfl_sync(mask, st, n - 1, kLanes);
    lo += (n - 1) * step;
    if (step == 1) break;
    hi = min(hi, lo + step - 1);
  }
  // Rows behind the last sequence belong to none.
  if (lo >= p.batch) return;
  const int64_t pos = (int64_t)start + (row - first);
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
  transform_row<V, kBf16, kW, kInter>(
      a, raw, src,
      p.pool + ((size_t)blk * p.block_size + (size_t)(pos - lb * p.block_size)) * a.dim, rot, gl,
      mask, nullptr);
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

// Calls LAUNCH(V, bf16, weights) with the vectors a lane that hold a row.
#define SAS_ROW_TYPES(V, LAUNCH)                                          \
  do {                                                                    \
    const bool weighted = a.weight != nullptr && a.norm_dim > 0;          \
    if (bf16 && weighted) LAUNCH(V, true, kGlobal);                       \
    else if (bf16) LAUNCH(V, true, kNone);                                \
    else if (weighted) LAUNCH(V, false, kGlobal);                         \
    else LAUNCH(V, false, kNone);                                         \
  } while (0)
#define SAS_ROW_DISPATCH(LAUNCH)                                          \
  do {                                                                    \
    if (a.dim <= 64) SAS_ROW_TYPES(1, LAUNCH);                            \
    else if (a.dim <= 128) SAS_ROW_TYPES(2, LAUNCH);                      \
    else if (a.dim <= 256) SAS_ROW_TYPES(4, LAUNCH);                      \
    else if (a.dim <= 512) SAS_ROW_TYPES(8, LAUNCH);                      \
    else if (a.dim <= 576) SAS_ROW_TYPES(9, LAUNCH);                      \
    else SAS_ROW_TYPES(16, LAUNCH);                                       \
  } while (0)

unsigned blocks_of(int64_t rows) {
  return (unsigned)((rows + kThreads / kLanes - 1) / (kThreads / kLanes));
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
  const HeadArgs h{static_cast<const uint16_t*>(x), static_cast<uint16_t*>(out), positions, err,
                   x_stride_token, x_stride_head, out_stride_token, out_stride_head, heads,
                   (int32_t)rows, positions_i64 != 0};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  const bool bf16 = tr->dtype == SAS_DTYPE_BF16;
  int dev = 0;
  const int sms = sas::current_device_sms(&dev);
  if (sms <= 0) return SAS_ERR_CUDA;
  const unsigned blocks = blocks_of(rows);
#define SAS_HEADS_OF(V, B, W, I)                                           \
  do {                                                                     \
    const unsigned full = (unsigned)(blocks_per_sm(V, I) * sms);           \
    if (blocks > full)                                                     \
      norm_rope_kernel<V, B, (W) == kGlobal ? kShared : (W), I>            \
          <<<full, kThreads, 0, stream>>>(a, h);                           \
    else                                                                   \
      norm_rope_kernel<V, B, W, I><<<blocks, kThreads, 0, stream>>>(a, h); \
  } while (0)
#define SAS_HEADS(V, B, W)                          \
  do {                                              \
    if (a.interleaved) SAS_HEADS_OF(V, B, W, true); \
    else SAS_HEADS_OF(V, B, W, false);              \
  } while (0)
  SAS_ROW_DISPATCH(SAS_HEADS);
#undef SAS_HEADS_OF
#undef SAS_HEADS
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
  const bool bf16 = tr->dtype == SAS_DTYPE_BF16;
  const unsigned blocks = blocks_of(total_new);
#define SAS_APPEND(V, B, W)                                                            \
  do {                                                                                 \
    if (a.interleaved)                                                                 \
      append_norm_rope_kernel<V, B, W, true><<<blocks, kThreads, 0, stream>>>(a, p);   \
    else                                                                               \
      append_norm_rope_kernel<V, B, W, false><<<blocks, kThreads, 0, stream>>>(a, p);  \
  } while (0)
  SAS_ROW_DISPATCH(SAS_APPEND);
#undef SAS_APPEND
  return cudaGetLastError() == cudaSuccess ? SAS_OK : SAS_ERR_CUDA;
}
