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
// a group are up to 256 columns, in two halves of whole tokens; the rows are a
// tile of 256 keys, 128 in each CTA of a pair, and a half is one
// tcgen05.mma.cta_group::2 of M = 256, N = 128 a step of 16 dims.  With keys in
// the rows, a thread of the epilogue owns one key and sums over heads along
// its own TMEM lane, without exchanging anything; the weights of its half's
// columns stay in registers over all the key tiles of a group.  The pair
// halves what the queries take of each SM's shared memory, which leaves room
// for five key stages beside two query buffers.  Each half has two
// accumulators of its own, so that the two epilogue warpgroups do not wait for
// each other.  An item is a group and a span of its key tiles; a persistent
// pair takes every num_pairs-th item.  Tiles that no token of the group sees
// are filled with -inf without loads.
//
// Bounds.  With few tokens a sequence the keys are read once each from HBM: 256
// tokens of 64 heads against 32768 keys of 128 dims take 350 us, 6.2 TB/s of
// keys and scores.  With many tokens the products: 8 x 4096 causal tokens of 64
// heads take 1120 us in a run of such calls (1090 to 1250 us from device to
// device), of which the products alone need 680 us at the burst rate of bf16 and
// 840 us at the sustained one.  An MMA of a half takes 64 cycles alone and about
// 100 beside the epilogue, with no unit saturated (tensor 58 %, ALU 50 %, issue
// slots 51 %): whether the tiles wait for the epilogue's TMEM reads or for its
// arithmetic has not been told apart.
//
// Warp roles in each CTA (384 threads, one CTA per SM):
//   0, 3   keys, every other tile each: page lookup, TMA into a ring of stages
//          (boxes of a page's rows where the page size allows, tile::gather4
//          else)
//   1      CTA 0: MMA issue (one elected lane)
//   2      items: the group of the next item, its queries into the other of
//          two buffers, its weights; the -inf fill; TMEM
//   4-11   epilogue: warpgroup g takes half g: relu, weight, sum over heads,
//          mask, store
//
// TMA loads of both CTAs complete on the leader's barriers; the leader's
// commits arrive in both CTAs; CTA 1's epilogue releases accumulators on the
// leader's barrier.  Every wait is bounded (~2 s): on timeout the thread
// records an error and raises its CTA's abort flag, on which every role leaves
// its loop; both CTAs meet at the final cluster barriers.

#include <math_constants.h>
#include <stddef.h>

#include <atomic>

#include "sas_dev.cuh"

namespace sas {
namespace {

constexpr int kIxThreads = 384;
constexpr int kIxKeys = 128;               // keys of a CTA's tile
constexpr int kIxTile = 2 * kIxKeys;       // keys of the pair's tile (M)
constexpr int kIxCols = 256;               // (token, head) columns of a group (N)
constexpr int kIxHalf = kIxCols / 2;       // columns of half a group
constexpr int kIxTokens = kIxCols / 16;    // tokens of a group at most
constexpr int kIxMaxStages = 8;
constexpr int kIxBits = 16;                // tiles whose page bits are kept
constexpr int kIxItems = 4;                // items described ahead
constexpr int kIxQHalf = kIxHalf / 2 * 128;  // 64 dims of a CTA's columns of one half
constexpr int kIxQChunk = 2 * kIxQHalf;
constexpr int kIxKChunk = kIxKeys * 128;   // 64 dims of a CTA's key tile
constexpr int kIxSmem = 232448;            // the per-block opt-in maximum

// Registers of the loading and issuing warpgroup and of an epilogue one: 88 +
// 2 x 208 = 3 x 168, the launch's share of 384 threads.  (Of the instances only that of
// 128 heads, all of them there, spills: 20 bytes.)
constexpr int kIxRegsLoad = 88, kIxRegsEpi = 208;

// An item as its roles need it: tokens tok0 .. tok0 + live (relative to the
// call's first), of sequence `batch`; key tiles [t0, tc) are computed.
struct IxInfo {
  int tok0, live, batch, most, t0, tc, unused[2];
  int len[kIxTokens];  // keys that each token sees
};

struct IxCtl {
  uint64_t q_full[2], q_empty[2];  // full: leader, one arrival per CTA and the bytes of both
  uint64_t k_full[kIxMaxStages], k_empty[kIxMaxStages];
  // [half][buffer]; empty: leader, the half's epilogue warps of both CTAs.
  uint64_t acc_full[2][2], acc_empty[2][2];
  uint64_t item_full[kIxItems], item_empty[kIxItems];
  uint64_t w_full, w_empty;
  uint64_t bits_full[kIxBits];
  uint64_t drain;
  uint32_t tmem_base;
  volatile int abort;
  uint8_t issued[kIxMaxStages];  // 1 + parity of the stage's last load, 0 before the first
  // Bit r of byte i of a tile: key 8 i + r has a page.  The slot of tile n is
  // written again for tile n + kIxBits, after the MMAs of tile n + kIxBits -
  // stages, whose accumulators the epilogue released behind tile n + kIxBits -
  // stages - 3 >= n (a half without tokens in an item has released all of its
  // before that item's first MMA).
  uint8_t bits[kIxBits][16];
  IxInfo items[kIxItems];
  alignas(16) float w[kIxCols];  // read as 16-byte vectors
};
static_assert(offsetof(IxCtl, w) % 16 == 0 && alignof(IxCtl) == 16, "vector reads of w");
static_assert(kIxBits >= kIxMaxStages + 3, "page bits are kept long enough");

// Shared memory: two query buffers, the key stages, control.
template <int kChunks>
struct IxSmem {
  static constexpr int kQ = kChunks * kIxQChunk;
  static constexpr int kFit = (kIxSmem - (int)sizeof(IxCtl) - 2 * kQ) / (kChunks * kIxKChunk);
  static constexpr int kStages = kFit < kIxMaxStages ? kFit : kIxMaxStages;
  static constexpr int kCtl = 2 * kQ + kStages * kChunks * kIxKChunk;
};
static_assert(IxSmem<1>::kCtl % 16 == 0 && IxSmem<2>::kCtl % 16 == 0, "control block alignment");
static_assert(IxSmem<2>::kStages == 5, "five stages of 128 keys by 128 dims fit");

struct IxArgs {
  SasIndexParams p;
  int32_t tq_shift;            // log2 of the tokens of a group
  int32_t groups;              // groups of the call (some may be empty)
  int32_t tiles, span_tiles, spans;
  int32_t box_shift;           // log2 of the rows of a key box, 0: tile::gather4
  int32_t no_row;              // row past the pool: reads as zeros
  uint32_t idesc;              // MMA instruction without its N
};

__device__ __forceinline__ int ix_start(const SasIndexParams& p, int b) {
  if (p.max_q_len > 0) return b * p.max_q_len;
  return __ldg(p.cu_seqlens_q + b);
}

// Start of sequence b's tokens inside the call's range.
__device__ __forceinline__ int ix_local(const SasIndexParams& p, int b) {
  return min(max(ix_start(p, b) - p.first_token, 0), p.num_tokens);
}

// Item `item` by a whole warp, lane i with the length of token i in *len.
// Sequence b owns the groups from (local(b) + b (tq - 1)) / tq on: at least
// ceil(tokens / tq) of them, without a scan over the lengths before it; the
// group's sequence is searched with 32 probes a step.  Items are in the order of
// their spans first: a pair's items are then spread over the groups in every
// span.  (Groups first, an even number of spans gave half of the pairs all the
// late spans, which causal tokens mostly do not see: 4096 of them with 64 heads
// took 230 us against 146.)  The tokens behind the
// last sequence are those of a sequence p.batch that sees no key; those before the
// first are in no group (ix_items fills their rows).
__device__ __forceinline__ IxInfo ix_item(const IxArgs& a, int item, int lane, int* t1) {
  const SasIndexParams& p = a.p;
  const int tq = 1 << a.tq_shift;
  const int span = item / a.groups, g = item - span * a.groups;
  auto first = [&](int b) {
    return (int)(((int64_t)ix_local(p, b) + (int64_t)b * (tq - 1)) >> a.tq_shift);
  };
  int lo = 0, hi = p.batch;
  while (lo < hi) {
    const int step = (hi - lo + 32) / 32;
    const int at = lo + lane * step;
    const int n = __popc(__ballot_sync(0xffffffffu, at <= hi && first(at) <= g));
    if (n == 0) break;
    lo += (n - 1) * step;
    hi = min(hi, lo + step - 1);
  }
  const int begin = ix_local(p, lo), f = first(lo);
  const int end = lo < p.batch ? ix_local(p, lo + 1) : p.num_tokens;
  const int64_t tok = (int64_t)begin + (int64_t)(g - f) * tq;
  IxInfo r;
  r.batch = lo;
  r.tok0 = (int)(tok < end ? tok : end);
  r.live = g < f ? 0 : max(0, min(tq, end - r.tok0));
  r.len[0] = 0;
  if (lo < p.batch && lane < r.live) {
    const int start = ix_start(p, lo);
    const int q_len =
        p.cu_seqlens_q ? __ldg(p.cu_seqlens_q + lo + 1) - __ldg(p.cu_seqlens_q + lo) : p.max_q_len;
    const int s = p.first_token + r.tok0 + lane - start;
    if (s >= 0 && s < q_len) {
      const int64_t n = floordiv((int64_t)__ldg(p.kv_len + lo) - q_len + s + 1, p.cmp_ratio);
      r.len[0] = n < 0 ? 0 : n > p.num_keys ? p.num_keys : (int)n;
    }
  }
  r.most = __reduce_max_sync(0xffffffffu, r.len[0]);
  r.t0 = span * a.span_tiles;
  *t1 = min(r.t0 + a.span_tiles, a.tiles);
  r.tc = max(r.t0, min(*t1, (r.most + kIxTile - 1) / kIxTile));
  return r;
}

__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, int x,
                                                 int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::"
      "bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// relu that keeps NaN.
__device__ __forceinline__ float relu_nan(float x) {
  float y;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(x));
  return y;
}

// One lane of a converged warp: the code behind it runs once, and the compiler
// keeps the descriptors of the MMAs there in uniform registers (behind lane ==
// 0 it copies them lane by lane: 120 cycles an MMA against 30).
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok));
  return ok != 0;
}

// Pairs of fp32 in one 64-bit register, for the packed FMA.
__device__ __forceinline__ uint64_t pack_f32(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}

__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ float sum_f32(uint64_t a) {
  float x, y;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a));
  return x + y;
}

// Wait for copies or MMAs already issued, abort or not; bounded.
__device__ __forceinline__ void ix_settle(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try_wait(smem_addr(bar), parity) && clock64() - t0 < kWaitCycles) {
  }
}

// Wait by a whole warp.
__device__ __forceinline__ bool ix_wait(IxCtl& ctl, uint64_t* bar, int parity, int32_t* err,
                                        int site) {
  return __all_sync(0xffffffffu, wait_bar(&ctl, bar, (uint32_t)parity, err, site));
}

// The next item of a role's warp; it may be overwritten once the warp has
// arrived on its item_empty.
__device__ __forceinline__ const IxInfo* ix_next(IxCtl& ctl, int i, int32_t* err, int site) {
  const int slot = i % kIxItems;
  if (!ix_wait(ctl, &ctl.item_full[slot], (i / kIxItems) & 1, err, site)) return nullptr;
  return &ctl.items[slot];
}

__device__ __forceinline__ void ix_done(IxCtl& ctl, int i, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(smem_addr(&ctl.item_empty[i % kIxItems]));
}

// Pages of logical key positions that advance by a fixed step: one division
// at the start.
struct IxPage {
  int lb, off;  // page of the table, row inside it
  __device__ __forceinline__ void start(const SasIndexParams& p, int pos) {
    lb = pos / p.block_size;
    off = pos - lb * p.block_size;
  }
  __device__ __forceinline__ void advance(const SasIndexParams& p, int pages, int rows) {
    lb += pages;
    off += rows;
    if (off >= p.block_size) {
      off -= p.block_size;
      ++lb;
    }
  }
  // Page id as the table has it (-1 past the table).
  __device__ __forceinline__ int id(const SasIndexParams& p, const int32_t* table) const {
    return lb < p.table_len ? __ldg(table + lb) : -1;
  }
};

// Row in the pool of a key of sequence `batch`, no_row without a page.
__device__ __forceinline__ int ix_row(const IxArgs& a, int id, int off, int batch) {
  if (id >= a.p.num_blocks) record_error(a.p.err, SAS_ERR_DEVICE, 53, id, batch);
  return id < 0 || id >= a.p.num_blocks ? a.no_row : id * a.p.block_size + off;
}

// Keys of the tiles n % 2 == half of the pair's tiles, n counted over its
// items: page ids are read two tiles ahead of their use, behind the wait for
// a stage.
template <int kChunks>
__device__ __forceinline__ void ix_keys(const IxArgs& a, IxCtl& ctl, uint32_t sK, int count,
                                        const CUtensorMap* tm_k, int half, int rank, int lane) {
  constexpr int kStages = IxSmem<kChunks>::kStages;
  const SasIndexParams& p = a.p;
  const bool gather = a.box_shift == 0;
  const int boxes = gather ? 32 : kIxKeys >> a.box_shift;
  const int step = gather ? 4 : 1 << a.box_shift;  // rows of a lane
  const int my_box = a.box_shift > 0 ? (8 * (lane & 15)) >> a.box_shift : 0;
  const int adv_pages = 2 * kIxTile / p.block_size, adv_rows = 2 * kIxTile % p.block_size;
  const uint32_t full0 = peer_addr(smem_addr(&ctl.k_full[0]), 0);
  int n = 0;               // tiles before the item's first
  int s = half, ph = 1;    // stage and parity of the warp's next tile
  for (int i = 0; i < count; ++i) {
    const IxInfo* info = ix_next(ctl, i, p.err, 69);
    if (info == nullptr) return;
    const int t0 = info->t0, tc = info->tc, most = info->most, batch = info->batch;
    const int32_t* table = p.block_table + (size_t)batch * p.table_len;
    ix_done(ctl, i, lane);
    if (tc == t0) continue;
    int t = t0 + ((n ^ half) & 1);
    int pos = t * kIxTile + rank * kIxKeys + lane * step;
    IxPage pg;
    pg.start(p, pos);
    int id[4];
    auto read_ids = [&](int tile) {
      if (!gather) {
        id[0] = lane < boxes && tile < tc && pos < most ? pg.id(p, table) : -1;
      } else {
        IxPage q = pg;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          id[r] = tile < tc && pos + r < most ? q.id(p, table) : -1;
          q.advance(p, 0, 1);
        }
      }
    };
    read_ids(t);
    for (; t < tc; t += 2) {
      const uint32_t stage = sK + (uint32_t)(s * kChunks * kIxKChunk);
      const uint32_t bar = full0 + 8u * (uint32_t)s;
      const int slot = (n + t - t0) % kIxBits;
      if (!ix_wait(ctl, &ctl.k_empty[s], ph, p.err, 70)) return;
      int rows[4];
      if (!gather) {
        rows[0] = ix_row(a, id[0], pg.off, batch);
        const uint32_t mapped = __ballot_sync(0xffffffffu, rows[0] != a.no_row);
        if (lane < 16) ctl.bits[slot][lane] = (mapped >> my_box) & 1 ? 255 : 0;
      } else {
        IxPage q = pg;
        uint32_t four = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          rows[r] = ix_row(a, id[r], q.off, batch);
          four |= (rows[r] != a.no_row ? 1u : 0u) << r;
          q.advance(p, 0, 1);
        }
        const uint32_t next = __shfl_down_sync(0xffffffffu, four, 1);
        if ((lane & 1) == 0) ctl.bits[slot][lane >> 1] = (uint8_t)(four | next << 4);
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(smem_addr(&ctl.bits_full[slot]));
        ctl.issued[s] = (uint8_t)(1 + (ph ^ 1));
        arrive_tx_cluster(bar, (uint32_t)(kChunks * kIxKChunk), false);
      }
      __syncwarp();
      if (lane < boxes) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const uint32_t dst = stage + (uint32_t)(c * kIxKChunk + lane * step * 128);
          if (gather)
            tma_gather4_pair(dst, tm_k, c * 64, rows[0], rows[1], rows[2], rows[3], bar);
          else
            tma_load_2d_pair(dst, tm_k, c * 64, rows[0], bar);
        }
      }
      s += 2;
      if (s >= kStages) {
        s -= kStages;
        ph ^= 1;
      }
      pos += 2 * kIxTile;
      pg.advance(p, adv_pages, adv_rows);
      read_ids(t + 2);
    }
    n += tc - t0;
  }
}

template <int kHp, bool kPadded>
__device__ __forceinline__ void ix_epilogue(const IxArgs& a, IxCtl& ctl, uint32_t tmem, int count,
                                            int rank) {
  const SasIndexParams& p = a.p;
  constexpr int kTok = kIxHalf / kHp;  // tokens of a warpgroup
  const int tid = threadIdx.x - 128, wg = tid >> 7, lane = tid & 31;
  const int row = tid & 127;
  const uint32_t base = tmem + ((uint32_t)(row & ~31) << 16) + (uint32_t)(wg * 2 * kIxHalf);
  const uint32_t empty0 = peer_addr(smem_addr(&ctl.acc_empty[wg][0]), 0);
  uint64_t w[kIxHalf / 2];
#pragma unroll
  for (int i = 0; i < kIxHalf / 2; ++i) w[i] = 0;
  // The least of a product and its column's limit: the product where the limit
  // is NaN, 0 or less (also for NaN) where it is 0, in the piece of 16 columns in
  // which the heads end.
  float limit[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) limit[k] = k < p.num_heads % 16 ? CUDART_NAN_F : 0.0f;
  int n = 0, u = 0, m = 0;  // tiles of the pair, of this half, items with tiles
  for (int i = 0; i < count; ++i) {
    const IxInfo* info = ix_next(ctl, i, p.err, 73);
    if (info == nullptr) return;
    const int t0 = info->t0, tc = info->tc;
    const int tok0 = info->tok0 + wg * kTok;           // first token of the warpgroup
    const int live = min(kTok, info->live - wg * kTok);  // its tokens, may be <= 0
    int len[kTok];
#pragma unroll
    for (int t = 0; t < kTok; ++t) len[t] = info->len[wg * kTok + t];
    ix_done(ctl, i, lane);
    if (tc == t0) continue;
    if (!ix_wait(ctl, &ctl.w_full, m & 1, p.err, 79)) return;
#pragma unroll
    for (int c = 0; c < kIxHalf / 4; ++c) {
      const float4 v = *reinterpret_cast<const float4*>(&ctl.w[wg * kIxHalf + 4 * c]);
      w[2 * c] = pack_f32(v.x, v.y);
      w[2 * c + 1] = pack_f32(v.z, v.w);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_addr(&ctl.w_empty));
    ++m;
    if (live <= 0) {
      n += tc - t0;
      continue;
    }
    float* out = p.scores + (size_t)tok0 * p.score_stride;
    for (int t = t0; t < tc; ++t, ++n, ++u) {
      const int b = u & 1, slot = n % kIxBits;
      if (!ix_wait(ctl, &ctl.acc_full[wg][b], (u >> 1) & 1, p.err, 80) ||
          !ix_wait(ctl, &ctl.bits_full[slot], (n / kIxBits) & 1, p.err, 81))
        return;
      tc_fence_after();
      const int key = t * kIxTile + rank * kIxKeys + row;
      const bool paged = (ctl.bits[slot][row >> 3] >> (row & 7)) & 1;
      const uint32_t acc = base + (uint32_t)(b * kIxHalf);
      uint32_t v[2][16];
      tmem_ld16(acc, v[0]);
      uint64_t s0 = 0, s1 = 0;
#pragma unroll
      for (int c = 0; c < kIxHalf / 16; ++c) {
        constexpr int kPieces = kHp / 16;  // 16-column pieces of a token
        const int tok = c / kPieces;
        if (tok < live) {
          tmem_wait_ld();
          if (c + 1 < kIxHalf / 16 && (c + 1) / kPieces < live) {
            tmem_ld16(acc + 16u * (c + 1), v[(c + 1) & 1]);
          } else {  // all read: the accumulator is free
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_remote(empty0 + 8u * (uint32_t)b);
          }
          // Columns of padded heads stay out of the sum: their products are zero,
          // but NaN with a key of infinities.  They are in the upper half of a
          // token's columns, for which alone there are branches.  (Without the
          // template argument they cost heads that fill the tile 20 %: 1046 ->
          // 1240 us for 8 x 4096 tokens of 64 heads.  4096 tokens of 48 heads take 138
          // us, 149 with branches in both halves and a select for each column, and
          // 134 with 64 heads; 24 heads 110, 115 and, with 32, 87 us.)
          const bool upper = kPadded && 16 * (c % kPieces) + 16 > kHp / 2;
          const int heads = upper ? p.num_heads - 16 * (c % kPieces) : 16;  // of this piece
          if (heads > 0) {
            const bool ends = upper && heads < 16;
            auto add = [&](bool cut) {
#pragma unroll
              for (int k = 0; k < 16; k += 4) {
                float x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  x[j] = __uint_as_float(v[c & 1][k + j]);
                  if (cut) x[j] = fminf(x[j], limit[k + j]);
                  x[j] = relu_nan(x[j]);
                }
                s0 = fma2(w[8 * c + k / 2], pack_f32(x[0], x[1]), s0);
                s1 = fma2(w[8 * c + k / 2 + 1], pack_f32(x[2], x[3]), s1);
              }
            };
            if (ends)
              add(true);
            else
              add(false);
          }
          if ((c + 1) % kPieces == 0) {
            if (key < len[tok] || (p.fill && key < p.num_keys))
              out[(size_t)tok * p.score_stride + key] =
                  key < len[tok] && paged ? sum_f32(s0) + sum_f32(s1) : -CUDART_INF_F;
            s0 = s1 = 0;
          }
        }
      }
    }
  }
}

// Items, their queries and weights, and the fills.
template <int kChunks, int kHp>
__device__ __forceinline__ void ix_items(const IxArgs& a, IxCtl& ctl, uint32_t sQ, int count,
                                         int pair, int pairs, const CUtensorMap* tm_q, int rank,
                                         int lane) {
  const SasIndexParams& p = a.p;
  const uint32_t full0 = peer_addr(smem_addr(&ctl.q_full[0]), 0);
  const bool vec = ((reinterpret_cast<uintptr_t>(p.scores) & 15) | (p.score_stride & 3)) == 0;
  int m = 0;
  for (int i = 0; i < count; ++i) {
    int t1;
    const IxInfo r = ix_item(a, pair + i * pairs, lane, &t1);
    const bool busy = r.tc > r.t0;
    float w[kIxCols / 32];
    if (busy) {
#pragma unroll
      for (int k = 0; k < kIxCols / 32; ++k) {
        const int c = 32 * k + lane, t = c / kHp, h = c % kHp;
        w[k] = t < r.live && h < p.num_heads
                   ? __ldg(p.weights + (size_t)(p.first_token + r.tok0 + t) * p.num_heads + h)
                   : 0.0f;
      }
    }
    const int slot = i % kIxItems;
    if (!ix_wait(ctl, &ctl.item_empty[slot], ((i / kIxItems) & 1) ^ 1, p.err, 68)) break;
    IxInfo& o = ctl.items[slot];
    if (lane == 0) {
      o.tok0 = r.tok0;
      o.live = r.live;
      o.batch = r.batch;
      o.most = r.most;
      o.t0 = r.t0;
      o.tc = r.tc;
    }
    if (lane < kIxTokens) o.len[lane] = r.len[0];
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_addr(&ctl.item_full[slot]));
    if (rank == 0 && r.t0 == 0 && p.lengths != nullptr && lane < r.live)
      p.lengths[r.tok0 + lane] = r.len[0];
    if (busy) {
      const int qb = m & 1;
      if (!ix_wait(ctl, &ctl.q_empty[qb], ((m >> 1) & 1) ^ 1, p.err, 72)) break;
      // Half g holds the tokens g kTok ..; of its columns each CTA holds half,
      // in units of half a token's heads.
      constexpr int kTok = kIxHalf / kHp, kUnit = kHp / 2;
      const uint32_t bar = full0 + 8u * (uint32_t)qb;
      if (lane == 0) arrive_tx_cluster(bar, (uint32_t)(r.live * kChunks * kUnit * 128), false);
      __syncwarp();
      const int g = lane / kTok, u = lane % kTok;  // unit u of half g
      const int tokens = min(kTok, r.live - g * kTok);
      if (g < 2 && u < tokens) {
        const int unit = rank * tokens + u;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          tma_load_3d_pair(sQ + (uint32_t)(qb * IxSmem<kChunks>::kQ + c * kIxQChunk +
                                           g * kIxQHalf + u * kUnit * 128),
                           tm_q, c * 64, (unit & 1) * kUnit,
                           p.first_token + r.tok0 + g * kTok + (unit >> 1), bar);
      }
      if (!ix_wait(ctl, &ctl.w_empty, (m & 1) ^ 1, p.err, 78)) break;
#pragma unroll
      for (int k = 0; k < kIxCols / 32; ++k) ctl.w[32 * k + lane] = w[k];
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&ctl.w_full));
      ++m;
    }
    // Columns of the item that no token of the group sees: 32-lane pieces
    // alternate between the CTAs.
    const int c0 = r.tc * kIxTile, c1 = min(t1 * kIxTile, p.num_keys);
    if (p.fill && c0 < c1) {
      const float4 none = make_float4(-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F);
      const int first = 32 * rank + lane;
      for (int t = 0; t < r.live; ++t) {
        float* o2 = p.scores + (size_t)(r.tok0 + t) * p.score_stride;
        if (vec) {
          for (int c = c0 + 4 * first; c + 4 <= c1; c += 256)
            *reinterpret_cast<float4*>(o2 + c) = none;
          if (first < (c1 & 3)) o2[(c1 & ~3) + first] = -CUDART_INF_F;
        } else {
          for (int c = c0 + first; c < c1; c += 64) o2[c] = -CUDART_INF_F;
        }
      }
    }
  }
  // The tokens before the first sequence, of which no group has any, see no key.
  const int lost = ix_local(p, 0);
  for (int t = 2 * pair + rank; t < lost; t += 2 * pairs) {
    if (p.lengths != nullptr && lane == 0) p.lengths[t] = 0;
    if (p.fill)
      for (int c = lane; c < p.num_keys; c += 32)
        p.scores[(size_t)t * p.score_stride + c] = -CUDART_INF_F;
  }
  // The leader's barriers count the queries of both CTAs.
  if (rank == 0)
    for (int k = max(0, m - 2); k < m; ++k) ix_settle(&ctl.q_full[k & 1], (uint32_t)(k >> 1) & 1);
}

template <int kChunks, int kHp>
__device__ __forceinline__ void ix_issue(const IxArgs& a, IxCtl& ctl, uint32_t sQ, uint32_t sK,
                                         uint32_t tmem, int count, int rank, int lane) {
  using L = IxSmem<kChunks>;
  const SasIndexParams& p = a.p;
  constexpr int kTok = kIxHalf / kHp;
  int s = 0, ph = 0;        // key stage and the parity awaited
  int units[2] = {0, 0};    // accumulators filled of each half
  int m = 0;
  const int steps = (p.head_dim + 15) / 16;
  for (int i = 0; i < count; ++i) {
    const IxInfo* info = ix_next(ctl, i, p.err, 67);
    if (info == nullptr) break;
    const int t0 = __shfl_sync(0xffffffffu, info->t0, 0);
    const int tc = __shfl_sync(0xffffffffu, info->tc, 0);
    const int live = __shfl_sync(0xffffffffu, info->live, 0);
    ix_done(ctl, i, lane);
    if (rank != 0 || tc == t0) continue;
    const int halves = live > kTok ? 2 : 1;
    bool ok = true;
    // A half that this item leaves out is done with the items before: its
    // epilogue still reads the page bits of their tiles.
    if (halves == 1)
      for (int u = max(0, units[1] - 2); ok && u < units[1]; ++u)
        ok = ix_wait(ctl, &ctl.acc_empty[1][u & 1], (u >> 1) & 1, p.err, 77);
    const int qb = m & 1;
    ++m;
    const uint64_t dq0 = smem_desc(sQ + (uint32_t)(qb * L::kQ), 16, 1024);
    ok = ok && ix_wait(ctl, &ctl.q_full[qb], ((m - 1) >> 1) & 1, p.err, 74);
    for (int t = t0; ok && t < tc; ++t) {
      ok = ix_wait(ctl, &ctl.k_full[s], ph, p.err, 75);
      const uint64_t dk = smem_desc(sK + (uint32_t)(s * kChunks * kIxKChunk), 16, 1024);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if (!ok || g >= halves) break;
        const int b = units[g] & 1;
        ok = ix_wait(ctl, &ctl.acc_empty[g][b], ((units[g] >> 1) & 1) ^ 1, p.err, 76);
        if (!ok) break;
        tc_fence_after();
        const uint32_t cols = (uint32_t)(min(kTok, live - g * kTok) * kHp);
        const uint32_t idesc = a.idesc | (cols >> 3) << 17;
        const uint64_t dq = dq0 + (uint64_t)(g * kIxQHalf >> 4);
        const uint32_t acc = tmem + (uint32_t)((2 * g + b) * kIxHalf);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4 * kChunks; ++k) {
            const uint32_t in = (uint32_t)(k & 3) * 32u, ch = (uint32_t)(k >> 2);
            if (k < steps)
              mma2(acc, dk + ((in + ch * kIxKChunk) >> 4), dq + ((in + ch * kIxQChunk) >> 4),
                   idesc, k > 0);
          }
          commit_both(smem_addr(&ctl.acc_full[g][b]));
          if (g + 1 == halves) commit_both(smem_addr(&ctl.k_empty[s]));
        }
        __syncwarp();
        ++units[g];
      }
      if (++s == L::kStages) {
        s = 0;
        ph ^= 1;
      }
    }
    if (!ok) break;
    if (elect_one()) commit_both(smem_addr(&ctl.q_empty[qb]));
    __syncwarp();
  }
  // Every MMA has read its operands before either CTA goes.
  if (rank == 0) {
    if (elect_one()) commit_both(smem_addr(&ctl.drain));
    __syncwarp();
    ix_settle(&ctl.drain, 0u);
  }
}

template <int kChunks, int kHp, bool kPadded>
__global__ void __launch_bounds__(kIxThreads, 1) __cluster_dims__(2, 1, 1)
    index_scores_kernel(const __grid_constant__ IxArgs a, const __grid_constant__ CUtensorMap tm_q,
                        const __grid_constant__ CUtensorMap tm_k) {
  using L = IxSmem<kChunks>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const uint32_t sQ = smem_addr(smem), sK = sQ + 2u * L::kQ;
  IxCtl& ctl = *reinterpret_cast<IxCtl*>(smem + L::kCtl);
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int items = a.groups * a.spans;
  const int count = pair < items ? (items - pair + pairs - 1) / pairs : 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&ctl.q_full[i]), 2);
      mbar_init(smem_addr(&ctl.q_empty[i]), 1);
      for (int b = 0; b < 2; ++b) {
        mbar_init(smem_addr(&ctl.acc_full[i][b]), 1);
        mbar_init(smem_addr(&ctl.acc_empty[i][b]), 8);
      }
    }
    for (int i = 0; i < kIxMaxStages; ++i) {
      mbar_init(smem_addr(&ctl.k_full[i]), 2);
      mbar_init(smem_addr(&ctl.k_empty[i]), 1);
      ctl.issued[i] = 0;
    }
    for (int i = 0; i < kIxItems; ++i) {
      mbar_init(smem_addr(&ctl.item_full[i]), 1);
      mbar_init(smem_addr(&ctl.item_empty[i]), 11);  // warps 0, 1, 3 and the epilogue
    }
    for (int i = 0; i < kIxBits; ++i) mbar_init(smem_addr(&ctl.bits_full[i]), 1);
    mbar_init(smem_addr(&ctl.w_full), 1);
    mbar_init(smem_addr(&ctl.w_empty), 8);
    mbar_init(smem_addr(&ctl.drain), 1);
    ctl.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(&ctl.tmem_base)),
                 "r"(2 * kIxCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers are initialised before any remote arrival
  tc_fence_after();
  const uint32_t tmem = ctl.tmem_base;

  if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kIxRegsEpi));
    ix_epilogue<kHp, kPadded>(a, ctl, tmem, count, rank);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIxRegsLoad));
    if (warp == 1)
      ix_issue<kChunks, kHp>(a, ctl, sQ, sK, tmem, count, rank, lane);
    else if (warp == 2)
      ix_items<kChunks, kHp>(a, ctl, sQ, count, pair, pairs, &tm_q, rank, lane);
    else
      ix_keys<kChunks>(a, ctl, sK, count, &tm_k, warp == 3, rank, lane);
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  // Nothing may land after the pair has gone: loads that no MMA waited for
  // after an abort complete on the leader's barriers.
  if (rank == 0 && threadIdx.x == 0)
    for (int i = 0; i < L::kStages; ++i)
      if (ctl.issued[i] != 0) ix_settle(&ctl.k_full[i], ctl.issued[i] - 1u);
  __syncthreads();
  cluster_sync_all();
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
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

template <int kChunks, int kHp, bool kPadded>
int ix_launch(const IxArgs& a, int grid, int dev, const CUtensorMap& q, const CUtensorMap& k,
              cudaStream_t stream) {
  static std::atomic<bool> configured[kMaxDevices];
  if (!configured[dev].load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(index_scores_kernel<kChunks, kHp, kPadded>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, kIxSmem) != cudaSuccess)
      return SAS_ERR_CUDA;
    configured[dev].store(true, std::memory_order_relaxed);
  }
  index_scores_kernel<kChunks, kHp, kPadded><<<grid, kIxThreads, kIxSmem, stream>>>(a, q, k);
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
  if (!p.q || !p.weights || !p.kv_len || (p.num_keys > 0 && !p.scores) ||
      (p.num_blocks > 0 && !p.key_pool) || (p.table_len > 0 && !p.block_table) ||
      (p.max_q_len == 0 && !p.cu_seqlens_q))
    return SAS_ERR_INVALID;
  if (((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.key_pool)) & 15) != 0)
    return SAS_ERR_INVALID;
  using namespace sas;
  int dev = 0;
  const int sms = current_device_sms(&dev);
  if (sms <= 0) return SAS_ERR_CUDA;

  IxArgs a{};
  a.p = p;
  const int hp = p.num_heads <= 16 ? 16 : p.num_heads <= 32 ? 32 : p.num_heads <= 64 ? 64 : 128;
  const int tq = kIxCols / hp;
  while ((1 << a.tq_shift) < tq) ++a.tq_shift;
  const int64_t groups = ((int64_t)p.num_tokens + ((int64_t)p.batch + 1) * (tq - 1)) / tq;
  a.tiles = (p.num_keys + kIxTile - 1) / kIxTile;
  // Spans: the pairs end together where each has the same number of items of the
  // same length, an item costs about a tile besides its own (its queries and
  // weights), and causal tokens want a few items a pair.  So: of 4 to 16 items a
  // pair, those with the fewest tiles for the pair that has most.  64 tokens
  // against 65536 keys: 172 us with 17 items, 182 with 7, 190 with 5; 8 tokens
  // against 20000: 16 us with 3, 23 with 9; 1024 causal tokens 21 us with 4, 34
  // with 14.
  const int pairs = sms > 1 ? sms / 2 : 1;
  int64_t best = INT64_MAX;
  a.spans = a.span_tiles = 1;
  for (int n = 4; n <= 16 && a.tiles > 0; ++n) {
    const int64_t most = (int64_t)n * pairs / groups;
    const int spans = (int)(most < 1 ? 1 : most > a.tiles ? a.tiles : most);
    const int tiles = (a.tiles + spans - 1) / spans;
    const int64_t cost = (groups * spans + pairs - 1) / pairs * (tiles + 1);
    if (cost >= best) continue;
    best = cost;
    a.span_tiles = tiles;
    a.spans = (a.tiles + tiles - 1) / tiles;
  }
  if (groups * a.spans > INT32_MAX - 4096) return SAS_ERR_UNSUPPORTED;
  a.groups = (int)groups;
  a.no_row = p.num_blocks * p.block_size;
  a.idesc = instr_desc(kIxTile, 0, p.dtype == SAS_DTYPE_BF16, false, false);
  // Box of key rows: the largest power of two up to 128 that divides the page
  // (a box then never leaves its page); pages that 8 does not divide are
  // gathered row by row.  (256 tokens against 32768 keys of 128 dims, one CTA a
  // tile: boxes of 64 rows 436 us, of 16 456 us, of 8 514 us, gathered 770 us.)
  int box = 128;
  while (box >= 8 && p.block_size % box != 0) box >>= 1;
  if (box >= 8)
    while ((1 << a.box_shift) < box) ++a.box_shift;
  else
    box = 1;

  alignas(64) CUtensorMap tm_q, tm_k;
  const uint64_t D = (uint64_t)p.head_dim, H = (uint64_t)p.num_heads, T = (uint64_t)p.total_tokens;
  if (!ix_map(&tm_q, p.q, D, H, T, (uint32_t)hp / 2, true)) return SAS_ERR_CUDA;
  if (a.no_row > 0) {
    if (!ix_map(&tm_k, p.key_pool, D, (uint64_t)a.no_row, 1, (uint32_t)box, false))
      return SAS_ERR_CUDA;
  } else {
    // An empty pool: every page is unmapped, and the row past it has to read
    // as zeros, as the row past the queries does.
    if (T * H > INT32_MAX - 1) return SAS_ERR_UNSUPPORTED;
    a.no_row = (int)(T * H);
    if (!ix_map(&tm_k, p.q, D, T * H, 1, (uint32_t)box, false))
      return SAS_ERR_CUDA;
  }
  const int64_t items = (int64_t)a.groups * a.spans;
  const int grid = 2 * (int)(items < pairs ? items : pairs);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
#define SAS_IX_HP(C, HP)                                              \
  (p.num_heads < HP ? ix_launch<C, HP, true>(a, grid, dev, tm_q, tm_k, stream) \
                    : ix_launch<C, HP, false>(a, grid, dev, tm_q, tm_k, stream))
#define SAS_IX(C)               \
  (hp == 16   ? SAS_IX_HP(C, 16) \
   : hp == 32 ? SAS_IX_HP(C, 32) \
   : hp == 64 ? SAS_IX_HP(C, 64) \
              : SAS_IX_HP(C, 128))
  return p.head_dim > 64 ? SAS_IX(2) : SAS_IX(1);
#undef SAS_IX
#undef SAS_IX_HP
}
