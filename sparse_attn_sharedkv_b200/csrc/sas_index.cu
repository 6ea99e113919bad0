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
//
// Work.  A group is up to 256 / Hp consecutive tokens of one sequence (Hp:
// the heads, padded to 16, 32, 64 or 128), so that the (token, head) pairs of
// a group are the N <= 256 columns of one tcgen05.mma; its M = 128 rows are a
// tile of 128 keys.  With keys in the rows, a thread of the epilogue owns one
// key and sums over heads along its own TMEM lane, without exchanging
// anything; the weights of its columns stay in registers over all the key
// tiles of a group.  An item is a group and a span of its key tiles; a
// persistent block per SM takes every gridDim-th item.  Tiles that no token of
// the group sees are filled with -inf without loads.
//
// Warp roles (384 threads, one block per SM):
//   0      keys: page lookup of a tile, TMA into a ring of stages (boxes of a
//          page's rows where the page size allows, tile::gather4 else)
//   1      MMA issue (one lane), accumulators alternating between two halves
//          of TMEM
//   2      queries of the next item into the other of two buffers; TMEM
//   4-11   epilogue: warpgroup g takes columns 128 g .. 128 g + 127 of each
//          accumulator: relu, weight, sum over heads, mask, store
//
// Every wait is bounded (~2 s): on timeout the thread records an error and
// raises the block's abort flag, on which every role leaves its loop.

#include <math_constants.h>

#include "sas_dev.cuh"

namespace sas {
namespace {

constexpr int kIxThreads = 384;
constexpr int kIxKeys = 128;           // keys of a tile (M)
constexpr int kIxCols = 256;           // (token, head) columns of a group (N)
constexpr int kIxHalf = kIxCols / 2;   // columns of an epilogue warpgroup
constexpr int kIxMaxStages = 8;
constexpr int kIxBits = 16;            // tiles whose page bits are kept
constexpr int kIxQChunk = kIxCols * 128;   // 64 dims of a group's columns
constexpr int kIxKChunk = kIxKeys * 128;   // 64 dims of a key tile
constexpr int kIxSmem = 232448;            // the per-block opt-in maximum

// Registers of the loading and issuing warpgroup and of an epilogue one: 88 +
// 2 x 208 = 3 x 168, the launch's share of 384 threads.
constexpr int kIxRegsLoad = 88, kIxRegsEpi = 208;

struct IxCtl {
  uint64_t q_full[2], q_empty[2];
  uint64_t k_full[kIxMaxStages], k_empty[kIxMaxStages];
  // Two arrivals: the issuing thread (for the page bits it has seen written)
  // and the commit of the tile's MMAs.
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  volatile int abort;
  // Byte i of a tile: bit r set when key 4 i + r has a page.  The slot of
  // tile n is written again for tile n + kIxBits, after the MMAs of tile n +
  // kIxBits - stages, whose accumulator the epilogue released behind tile
  // n + kIxBits - stages - 3 >= n.
  uint8_t bits[kIxBits][32];
};
static_assert(kIxBits >= kIxMaxStages + 3, "page bits are kept long enough");

struct IxArgs {
  SasIndexParams p;
  int32_t hp, tq;              // padded heads, tokens of a group
  int32_t groups;              // groups of the call (some may be empty)
  int32_t tiles, span_tiles, spans;
  int32_t box_rows;            // rows of a key box, 0: tile::gather4
  int32_t no_row;              // row past the pool: reads as zeros
  int32_t chunks, stages;
};

// Group g: tokens tok0 .. tok0 + live of the call (relative to first_token),
// of sequence `batch` (p.batch: of none), whose tokens start at `start`.
struct IxGroup {
  int tok0, live, batch, start, q_len, kv;
};

__device__ __forceinline__ int ix_start(const SasIndexParams& p, int b) {
  if (p.max_q_len > 0) return b * p.max_q_len;
  return __ldg(p.cu_seqlens_q + b);
}

// Start of sequence b's tokens inside the call's range.
__device__ __forceinline__ int ix_local(const SasIndexParams& p, int b) {
  return min(max(ix_start(p, b) - p.first_token, 0), p.num_tokens);
}

// Sequence b owns the groups from (local(b) + b (tq - 1)) / tq on: at least
// ceil(tokens / tq) of them, without a scan over the lengths before it.  The
// tokens behind the last sequence are those of a sequence p.batch.  Called by
// whole warps: 32 probes a step.
__device__ __forceinline__ IxGroup ix_group(const IxArgs& a, int g, int lane) {
  const SasIndexParams& p = a.p;
  auto first = [&](int b) { return (int)(((int64_t)ix_local(p, b) + (int64_t)b * (a.tq - 1)) / a.tq); };
  int lo = 0, hi = p.batch;
  while (lo < hi) {
    const int step = (hi - lo + 32) / 32;
    const int at = lo + lane * step;
    const int n = __popc(__ballot_sync(0xffffffffu, at <= hi && first(at) <= g));
    if (n == 0) break;
    lo += (n - 1) * step;
    hi = min(hi, lo + step - 1);
  }
  IxGroup r;
  r.batch = lo;
  r.start = lo < p.batch || p.max_q_len == 0 ? ix_start(p, lo) : p.total_tokens;
  const int begin = ix_local(p, lo);
  const int end = lo < p.batch ? ix_local(p, lo + 1) : p.num_tokens;
  const int64_t t0 = (int64_t)begin + (int64_t)(g - first(lo)) * a.tq;
  r.tok0 = (int)(t0 < end ? t0 : end);
  r.live = g < first(lo) ? 0 : max(0, min(a.tq, end - r.tok0));
  r.q_len = 0;
  r.kv = 0;
  if (lo < p.batch) {
    r.q_len = p.cu_seqlens_q ? __ldg(p.cu_seqlens_q + lo + 1) - __ldg(p.cu_seqlens_q + lo)
                             : p.max_q_len;
    r.kv = __ldg(p.kv_len + lo);
  }
  return r;
}

// Keys that token `i` of the group sees.
__device__ __forceinline__ int ix_len(const SasIndexParams& p, const IxGroup& g, int i) {
  const int s = p.first_token + g.tok0 + i - g.start;
  if (i >= g.live || g.batch >= p.batch || s < 0 || s >= g.q_len) return 0;
  const int64_t n = floordiv((int64_t)g.kv - g.q_len + s + 1, p.cmp_ratio);
  return n < 0 ? 0 : n > p.num_keys ? p.num_keys : (int)n;
}

// Item: a group and its key tiles [t0, t1), computed up to tc, filled behind.
struct IxItem {
  IxGroup g;
  int len;   // of token `lane`
  int most;  // the longest of the group
  int t0, t1, tc;
};

__device__ __forceinline__ IxItem ix_item(const IxArgs& a, int item, int lane) {
  IxItem r;
  const int gi = item / a.spans;
  r.g = ix_group(a, gi, lane);
  r.len = ix_len(a.p, r.g, lane);
  r.most = __reduce_max_sync(0xffffffffu, r.len);
  r.t0 = (item - gi * a.spans) * a.span_tiles;
  r.t1 = min(r.t0 + a.span_tiles, a.tiles);
  r.tc = max(r.t0, min(r.t1, (r.most + kIxKeys - 1) / kIxKeys));
  return r;
}

__device__ __forceinline__ void ix_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                            int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// relu that keeps NaN.
__device__ __forceinline__ float relu_nan(uint32_t bits) {
  float y;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(__uint_as_float(bits)));
  return y;
}

// Wait for copies or MMAs already issued, abort or not; bounded.
__device__ __forceinline__ void ix_settle(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try_wait(smem_addr(bar), parity) && clock64() - t0 < kWaitCycles) {
  }
}

// Row in the pool of logical key position `pos`, no_row without a page or
// where no token of the group looks.
__device__ __forceinline__ int ix_row(const IxArgs& a, int batch, int pos, int most) {
  const SasIndexParams& p = a.p;
  const int lb = pos / p.block_size;
  if (pos >= most || lb >= p.table_len) return a.no_row;
  const int blk = __ldg(p.block_table + (size_t)batch * p.table_len + lb);
  if (blk >= p.num_blocks) record_error(p.err, SAS_ERR_DEVICE, 53, blk);
  if (blk < 0 || blk >= p.num_blocks) return a.no_row;
  return blk * p.block_size + (pos - lb * p.block_size);
}

template <int kHp>
__device__ __forceinline__ void ix_epilogue(const IxArgs& a, IxCtl& ctl, uint32_t tmem, int items) {
  const SasIndexParams& p = a.p;
  constexpr int kTok = kIxHalf / kHp;  // tokens of a warpgroup
  const int tid = threadIdx.x - 128, wg = tid >> 7, lane = tid & 31;
  const int row = tid & 127;
  const uint32_t base = tmem + ((uint32_t)(row & ~31) << 16) + (uint32_t)(wg * kIxHalf);
  float w[kIxHalf];
#pragma unroll
  for (int i = 0; i < kIxHalf; ++i) w[i] = 0.0f;
  int n = 0;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    if (ctl.abort) break;
    const IxItem it = ix_item(a, item, lane);
    const int tok0 = it.g.tok0 + wg * kTok;           // first token of the warpgroup
    const int live = min(kTok, it.g.live - wg * kTok);  // its tokens, may be <= 0
    if (it.t0 == 0 && p.lengths != nullptr && tid < it.g.live) p.lengths[it.g.tok0 + tid] = it.len;
    if (it.tc > it.t0) {
#pragma unroll
      for (int i = 0; i < kIxHalf; ++i) {
        const int t = i / kHp, h = i % kHp;
        w[i] = t < live && h < p.num_heads
                   ? __ldg(p.weights + (size_t)(p.first_token + tok0 + t) * p.num_heads + h)
                   : 0.0f;
      }
    }
    float* out = p.scores + (size_t)max(tok0, 0) * p.score_stride;
    bool ok = true;
    for (int t = it.t0; t < it.tc; ++t, ++n) {
      const int b = n & 1;
      if (!__all_sync(0xffffffffu, wait_bar(&ctl, &ctl.acc_full[b], (uint32_t)(n >> 1) & 1, p.err, 73))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int key = t * kIxKeys + row;
      const bool paged = (ctl.bits[n % kIxBits][row >> 2] >> (row & 3)) & 1;
      const uint32_t acc = base + (uint32_t)(b * kIxCols);
      uint32_t v[2][16];
      if (live > 0) tmem_ld16(acc, v[0]);
      float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
      for (int c = 0; c < kIxHalf / 16; ++c) {
        constexpr int kPieces = kHp / 16;  // 16-column pieces of a token
        const int tok = c / kPieces;
        if (tok < live) {
          tmem_wait_ld();
          if (c + 1 < kIxHalf / 16 && (c + 1) / kPieces < live) tmem_ld16(acc + 16u * (c + 1), v[(c + 1) & 1]);
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            s0 = fmaf(w[16 * c + i], relu_nan(v[c & 1][i]), s0);
            s1 = fmaf(w[16 * c + i + 1], relu_nan(v[c & 1][i + 1]), s1);
          }
          if ((c + 1) % kPieces == 0) {
            const int len = __shfl_sync(0xffffffffu, it.len, wg * kTok + tok);
            if (key < len || (p.fill && key < p.num_keys))
              out[(size_t)tok * p.score_stride + key] =
                  key < len && paged ? s0 + s1 : -CUDART_INF_F;
            s0 = s1 = 0.0f;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&ctl.acc_empty[b]));
    }
    if (!ok) break;
    // Columns of the item that no token of the group sees.
    const int c0 = it.tc * kIxKeys, c1 = min(it.t1 * kIxKeys, p.num_keys);
    if (p.fill && c0 < c1) {
      const bool vec = ((reinterpret_cast<uintptr_t>(p.scores) & 15) | (p.score_stride & 3)) == 0;
      for (int t = 0; t < it.g.live; ++t) {
        float* o = p.scores + (size_t)(it.g.tok0 + t) * p.score_stride;
        if (vec) {
          const float4 none = make_float4(-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F);
          for (int c = c0 + 4 * tid; c + 4 <= c1; c += 1024) *reinterpret_cast<float4*>(o + c) = none;
          if (tid < (c1 & 3)) o[(c1 & ~3) + tid] = -CUDART_INF_F;
        } else {
          for (int c = c0 + tid; c < c1; c += 256) o[c] = -CUDART_INF_F;
        }
      }
    }
  }
}

template <bool kBf16, int kHp>
__global__ void __launch_bounds__(kIxThreads, 1)
    index_scores_kernel(const __grid_constant__ IxArgs a, const __grid_constant__ CUtensorMap tm_q,
                        const __grid_constant__ CUtensorMap tm_k) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const SasIndexParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q_bytes = a.chunks * kIxQChunk, stage_bytes = a.chunks * kIxKChunk;
  const uint32_t sQ = smem_addr(smem), sK = sQ + 2u * q_bytes;
  IxCtl& ctl = *reinterpret_cast<IxCtl*>(smem + 2 * q_bytes + a.stages * stage_bytes);
  const int items = a.groups * a.spans;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&ctl.q_full[i]), 1);
      mbar_init(smem_addr(&ctl.q_empty[i]), 1);
      mbar_init(smem_addr(&ctl.acc_full[i]), 2);
      mbar_init(smem_addr(&ctl.acc_empty[i]), 8);
    }
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(smem_addr(&ctl.k_full[i]), 1);
      mbar_init(smem_addr(&ctl.k_empty[i]), 1);
    }
    mbar_init(smem_addr(&ctl.drain), 1);
    ctl.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(&ctl.tmem_base)),
                 "r"(2 * kIxCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl.tmem_base;

  if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kIxRegsEpi));
    ix_epilogue<kHp>(a, ctl, tmem, items);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIxRegsLoad));
    if (warp == 0) {
      // Keys.
      int n = 0;
      bool ok = true;
      for (int item = blockIdx.x; ok && item < items && !ctl.abort; item += gridDim.x) {
        const IxItem it = ix_item(a, item, lane);
        for (int t = it.t0; t < it.tc; ++t, ++n) {
          const int s = n % a.stages;
          const uint32_t stage = sK + (uint32_t)(s * stage_bytes);
          const uint32_t bar = smem_addr(&ctl.k_full[s]);
          int rows[4];
          if (a.box_rows > 0) {
            const int boxes = kIxKeys / a.box_rows;
            rows[0] = lane < boxes
                          ? ix_row(a, it.g.batch, t * kIxKeys + lane * a.box_rows, it.most)
                          : a.no_row;
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              rows[r] = ix_row(a, it.g.batch, t * kIxKeys + 4 * lane + r, it.most);
          }
          if (!__all_sync(0xffffffffu, wait_bar(&ctl, &ctl.k_empty[s],
                                                (uint32_t)((n / a.stages) & 1) ^ 1, p.err, 70))) {
            ok = false;
            break;
          }
          uint32_t bits = 0;
          if (a.box_rows > 0) {
            const uint32_t mapped = __ballot_sync(0xffffffffu, rows[0] != a.no_row);
            bits = (mapped >> (4 * lane / a.box_rows)) & 1 ? 15u : 0u;
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) bits |= (rows[r] != a.no_row ? 1u : 0u) << r;
          }
          ctl.bits[n % kIxBits][lane] = (uint8_t)bits;
          __syncwarp();
          if (lane == 0) mbar_expect_tx(bar, (uint32_t)stage_bytes);
          __syncwarp();
          for (int c = 0; c < a.chunks; ++c) {
            const uint32_t dst = stage + (uint32_t)(c * kIxKChunk);
            if (a.box_rows == 0)
              tma_gather4(dst + (uint32_t)lane * 512u, &tm_k, c * 64, rows[0], rows[1], rows[2],
                          rows[3], bar);
            else if (lane < kIxKeys / a.box_rows)
              tma_load_2d(dst + (uint32_t)(lane * a.box_rows) * 128u, &tm_k, c * 64, rows[0], bar);
          }
        }
      }
      // Nothing may land after the block has gone: the last loads of each stage.
      for (int k = max(0, n - a.stages); k < n; ++k)
        ix_settle(&ctl.k_full[k % a.stages], (uint32_t)((k / a.stages) & 1));
    } else if (warp == 1) {
      // MMA.
      int n = 0, m = 0;
      bool ok = true;
      const int steps = (p.head_dim + 15) / 16;
      for (int item = blockIdx.x; ok && item < items && !ctl.abort; item += gridDim.x) {
        const IxItem it = ix_item(a, item, lane);
        if (it.tc == it.t0) continue;
        if (lane == 0) {
          const int qb = m & 1;
          const uint32_t idesc = instr_desc(kIxKeys, it.g.live * kHp, kBf16, false, false);
          const uint64_t dq = smem_desc(sQ + (uint32_t)(qb * q_bytes), 16, 1024);
          ok = wait_bar(&ctl, &ctl.q_full[qb], (uint32_t)(m >> 1) & 1, p.err, 74);
          for (int t = it.t0; ok && t < it.tc; ++t, ++n) {
            const int s = n % a.stages, b = n & 1;
            ok = wait_bar(&ctl, &ctl.k_full[s], (uint32_t)((n / a.stages) & 1), p.err, 75) &&
                 wait_bar(&ctl, &ctl.acc_empty[b], (uint32_t)((n >> 1) & 1) ^ 1, p.err, 76);
            if (!ok) break;
            tc_fence_after();
            const uint64_t dk = smem_desc(sK + (uint32_t)(s * stage_bytes), 16, 1024);
            for (int k = 0; k < steps; ++k) {
              const uint32_t in = (uint32_t)(k & 3) * 32u;
              ix_mma(tmem + (uint32_t)(b * kIxCols), dk + ((in + (uint32_t)(k >> 2) * kIxKChunk) >> 4),
                     dq + ((in + (uint32_t)(k >> 2) * kIxQChunk) >> 4), idesc, k > 0);
            }
            tc_commit(smem_addr(&ctl.k_empty[s]));
            mbar_arrive(smem_addr(&ctl.acc_full[b]));
            tc_commit(smem_addr(&ctl.acc_full[b]));
          }
          tc_commit(smem_addr(&ctl.q_empty[qb]));
        }
        n = __shfl_sync(0xffffffffu, n, 0);
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        ++m;
      }
      if (lane == 0) {  // every MMA has read its operands before the block goes
        tc_commit(smem_addr(&ctl.drain));
        ix_settle(&ctl.drain, 0u);
      }
    } else if (warp == 2) {
      // Queries.
      int m = 0;
      bool ok = true;
      for (int item = blockIdx.x; ok && item < items && !ctl.abort; item += gridDim.x) {
        const IxItem it = ix_item(a, item, lane);
        if (it.tc == it.t0) continue;
        const int qb = m & 1;
        if (!__all_sync(0xffffffffu, wait_bar(&ctl, &ctl.q_empty[qb], (uint32_t)((m >> 1) & 1) ^ 1,
                                              p.err, 72))) {
          ok = false;
          break;
        }
        const uint32_t bar = smem_addr(&ctl.q_full[qb]);
        if (lane == 0) mbar_expect_tx(bar, (uint32_t)(it.g.live * a.chunks * kHp * 128));
        __syncwarp();
        for (int i = lane; i < it.g.live * a.chunks; i += 32) {
          const int c = i / it.g.live, t = i - c * it.g.live;
          tma_load_3d(sQ + (uint32_t)(qb * q_bytes + c * kIxQChunk + t * kHp * 128), &tm_q, c * 64, 0,
                      p.first_token + it.g.tok0 + t, bar);
        }
        ++m;
      }
      for (int k = max(0, m - 2); k < m; ++k)
        ix_settle(&ctl.q_full[k & 1], (uint32_t)(k >> 1) & 1);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(2 * kIxCols)
                 : "memory");
  }
}

PFN_cuTensorMapEncodeTiled_v12000 ix_encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  return fn;
}

// Map over 16-bit rows [rows, mid, cols] with boxes of 64 columns, box_mid
// rows of the middle axis.
bool ix_map(CUtensorMap* m, const void* base, uint64_t cols, uint64_t mid, uint64_t rows,
            uint32_t box_mid, bool three) {
  auto fn = ix_encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[3] = {cols, mid, rows};
  cuuint64_t strides[2] = {cols * 2, cols * mid * 2};
  cuuint32_t box[3] = {64, box_mid, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, three ? 3 : 2, const_cast<void*>(base), dims,
            strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool kBf16, int kHp>
int ix_launch(const IxArgs& a, int grid, const CUtensorMap& q, const CUtensorMap& k,
              cudaStream_t stream) {
  // Per device: set on every call (a host call of well under a microsecond).
  if (cudaFuncSetAttribute(index_scores_kernel<kBf16, kHp>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize, kIxSmem) != cudaSuccess)
    return SAS_ERR_CUDA;
  index_scores_kernel<kBf16, kHp><<<grid, kIxThreads, kIxSmem, stream>>>(a, q, k);
  return cudaGetLastError() == cudaSuccess ? SAS_OK : SAS_ERR_CUDA;
}

}  // namespace
}  // namespace sas

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
      (int64_t)p.num_blocks * p.block_size > INT32_MAX - 1 ||
      p.num_keys > INT32_MAX - 1024)
    return SAS_ERR_UNSUPPORTED;
  if (p.max_q_len > 0 && (int64_t)p.max_q_len * p.batch != p.total_tokens) return SAS_ERR_INVALID;
  if (p.num_tokens == 0 || (p.num_keys == 0 && !p.lengths)) return SAS_OK;
  if (!p.q || !p.weights || !p.key_pool || !p.block_table || !p.kv_len || !p.scores ||
      (p.max_q_len == 0 && !p.cu_seqlens_q))
    return SAS_ERR_INVALID;
  if (((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.key_pool)) & 15) != 0)
    return SAS_ERR_INVALID;
  using namespace sas;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return SAS_ERR_CUDA;

  IxArgs a{};
  a.p = p;
  a.hp = p.num_heads <= 16 ? 16 : p.num_heads <= 32 ? 32 : p.num_heads <= 64 ? 64 : 128;
  a.tq = kIxCols / a.hp;
  const int64_t groups =
      ((int64_t)p.num_tokens + ((int64_t)p.batch + 1) * (a.tq - 1)) / a.tq;
  a.tiles = (p.num_keys + kIxKeys - 1) / kIxKeys;
  // Spans: short enough for about 16 items a block, so that blocks end
  // together; whole rows where the groups alone are that many.
  const int64_t total = groups * (a.tiles > 0 ? a.tiles : 1);
  const int64_t span = (total + 16 * sms - 1) / (16 * sms);
  a.span_tiles = (int)(span < 1 ? 1 : span > a.tiles ? (a.tiles > 0 ? a.tiles : 1) : span);
  a.spans = a.tiles > 0 ? (a.tiles + a.span_tiles - 1) / a.span_tiles : 1;
  if (groups * a.spans > INT32_MAX - 4096) return SAS_ERR_UNSUPPORTED;
  a.groups = (int)groups;
  a.no_row = p.num_blocks * p.block_size;
  a.chunks = p.head_dim > 64 ? 2 : 1;
  a.stages = (kIxSmem - (int)sizeof(IxCtl) - 2 * a.chunks * kIxQChunk) / (a.chunks * kIxKChunk);
  if (a.stages > kIxMaxStages) a.stages = kIxMaxStages;
  // Box of key rows: the largest power of two up to 128 that divides the page
  // (a box then never leaves its page); pages that 8 does not divide are
  // gathered row by row.
  int box = 128;
  while (box >= 8 && p.block_size % box != 0) box >>= 1;
  a.box_rows = box >= 8 ? box : 0;

  alignas(64) CUtensorMap tm_q, tm_k;
  const uint64_t D = (uint64_t)p.head_dim, H = (uint64_t)p.num_heads, T = (uint64_t)p.total_tokens;
  if (!ix_map(&tm_q, p.q, D, H, T, (uint32_t)a.hp, true)) return SAS_ERR_CUDA;
  if (a.no_row > 0) {
    if (!ix_map(&tm_k, p.key_pool, D, (uint64_t)a.no_row, 1, a.box_rows > 0 ? a.box_rows : 1, false))
      return SAS_ERR_CUDA;
  } else {
    // An empty pool: every page is unmapped, and the row past it has to read
    // as zeros, as the row past the queries does.
    if (T * H > INT32_MAX - 1) return SAS_ERR_UNSUPPORTED;
    a.no_row = (int)(T * H);
    if (!ix_map(&tm_k, p.q, D, T * H, 1, a.box_rows > 0 ? a.box_rows : 1, false))
      return SAS_ERR_CUDA;
  }
  const int64_t items = (int64_t)a.groups * a.spans;
  const int grid = (int)(items < sms ? items : sms);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
#define SAS_IX(HP)                                                                      \
  (p.dtype == SAS_DTYPE_BF16 ? ix_launch<true, HP>(a, grid, tm_q, tm_k, stream)         \
                             : ix_launch<false, HP>(a, grid, tm_q, tm_k, stream))
  return a.hp == 16 ? SAS_IX(16) : a.hp == 32 ? SAS_IX(32) : a.hp == 64 ? SAS_IX(64) : SAS_IX(128);
#undef SAS_IX
}
