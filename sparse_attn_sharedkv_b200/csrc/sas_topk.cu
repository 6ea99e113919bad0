// Top-k selection of key positions by score: per row the K largest of its
// first len scores, ties to the lower position, written in ascending order of
// position with -1 behind them: the index list of the attention
// (golden.py:28-66 stops at the first -1).  A score of -inf is never
// selected; NaN ranks above +inf and -0 equals +0.
//
// A row is read once and stays in the registers of a block, 16 or 32 scores a
// thread, or of a cluster of up to 8 blocks (262144 scores) that exchange a few values through
// distributed shared memory.  Rows of finite scores (the ordinary case):
//
//   1. the least and the greatest score; a row of at most K is all selected;
//   2. a histogram of 1024 bins linear in the scores, over which near-normal
//      scores spread (a bin then holds a few, and the shared-memory atomics
//      seldom meet); the bin in which the K-th largest lies.  The bin is the
//      low bits of a float near 2^23, so no conversion is needed;
//   3. scores in higher bins are selected, those of the border bin listed (if
//      they are more than 512, those of one bin of a second histogram inside
//      of it);
//   4. up to 32 listed are ranked by (score, position) by the threads that hold
//      them; among more, a histogram inside of the bin again, and the list's
//      winners are marked for the threads that hold them;
//   5. the selected positions are counted and written.
//
// Scores of -inf are left out of all of this.  Any other row (+inf, NaN, a single
// value, more left than the lists hold) is read again as unsigned keys of the same
// order: histograms linear in the keys divide the range of the border keys by at
// least 512 a round until 128 or a single key are left; equal keys are taken by a
// count over their positions.
//
// Each warp of a block holds neighbouring positions, 32 a round: loads are
// coalesced for any row alignment, the count of the selected positions before
// a warp's is one number, a ballot counts those of a round, and its selected
// lanes write neighbouring words.
//
// The floor is one read of the scores and one write of the positions; what
// bounds many rows is the issue of instructions (70 % of the slots; about 60 a
// score of a lane) with the latency of the phases.  32768 causal rows of up to
// 4096, K 2048: 172 us (82 us of memory); 4000 rows of 16384 to 32768: 230 us; 64
// rows of 8192 to 32768: 12 us.

#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "sas.h"
#include "sas_kernels.h"

namespace {

constexpr int kBins = 1024;
constexpr int kCand = 512;                 // border scores listed
constexpr int kList = 128;                 // keys ranked by as many threads
constexpr int kDirect = 32;                // entries ranked by the threads that list them
constexpr uint32_t kNegInf = 0x007fffffu;  // key of -inf
constexpr uint32_t kPosInf = 0xff800000u;  // key of +inf

__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// A score's key and its position as one number: greater is selected first.
__device__ __forceinline__ uint64_t entry_of(uint32_t key, uint32_t pos) {
  return (uint64_t)key << 32 | (uint32_t)~pos;
}

__device__ __forceinline__ float score_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

// Address of `p` (own shared memory) in block `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_smem(const void* p, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(r)
               : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t peer_load(const void* p, int rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer_smem(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void peer_store(void* p, int rank, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_smem(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ uint64_t peer_load64(const void* p, int rank) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(peer_smem(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void peer_store64(void* p, int rank, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(peer_smem(p, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t peer_add(void* p, int rank, uint32_t v) {
  uint32_t old;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;"
               : "=r"(old)
               : "r"(peer_smem(p, rank)), "r"(v)
               : "memory");
  return old;
}

// Barriers of a cluster here are not `.aligned` ones: loops over a lane's own scores
// or entries end right before them.
template <int C>
__device__ __forceinline__ void row_sync() {
  if constexpr (C == 1)
    __syncthreads();
  else
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// A block's shared memory may be written by its peers once it runs: every block of
// a cluster arrives when it starts and waits before it first reaches for another's,
// the loads of the scores in between.
template <int C>
__device__ __forceinline__ void peers_arrive() {
  if constexpr (C > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
}
template <int C>
__device__ __forceinline__ void peers_wait() {
  if constexpr (C > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// Shared memory of a block.
template <int T, int C>
struct TopkShared {
  alignas(16) uint32_t hist[kBins];  // from the top bin down
  uint32_t wmin[T / 32], wmax[T / 32], wcnt[T / 32], wsum[T / 32];
  uint32_t rmin[C], rmax[C], rcnt[C], rtot[C];  // one entry per block of the cluster
  uint32_t bin, above, inside;                  // found in the histogram, bin from the top
  uint32_t listed, ranked;
  alignas(16) uint64_t list[kCand];        // of the cluster, in block 0
  alignas(16) uint64_t mine[C > 1 ? kCand : 2];  // own copy
  uint64_t entry[kList];
  uint32_t taken[T];  // listed scores of each thread that are selected
  uint64_t threshold;
};

// One more entry of the row's list.
template <int T, int C>
__device__ __forceinline__ void add_entry(TopkShared<T, C>& s, uint64_t e) {
  if constexpr (C == 1) {
    s.list[atomicAdd(&s.listed, 1u)] = e;
  } else {
    peer_store64(&s.list[peer_add(&s.listed, 0, 1u)], 0, e);
  }
}

// Positions of a block: `len` from `begin` on, `seg` for each warp.
struct Places {
  int begin, len, seg, last;  // the warps' rounds are 0 .. last

  __device__ __forceinline__ Places(int begin_, int end, int threads)
      : begin(begin_), len(end - begin_), last(max(0, (end - begin_ - 1) / threads)) {
    seg = (last + 1) * 32;
  }
  // Rounds in which the thread holds a position, and the position.
  __device__ __forceinline__ int rounds() const {
    const int rest = len - (int)(threadIdx.x >> 5) * seg - (int)(threadIdx.x & 31);
    return max(0, min(last + 1, (rest + 31) >> 5));
  }
  __device__ __forceinline__ int at(int i) const {
    return begin + (int)(threadIdx.x >> 5) * seg + i * 32 + (int)(threadIdx.x & 31);
  }
};

// Least and greatest of the keys (kmin, kmax) and the sum of n over the row's
// threads.
template <int T, int C>
__device__ __forceinline__ void row_reduce(TopkShared<T, C>& s, int rank, uint32_t& kmin,
                                           uint32_t& kmax, uint32_t& n) {
  constexpr int W = T / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  kmin = __reduce_min_sync(0xffffffffu, kmin);
  kmax = __reduce_max_sync(0xffffffffu, kmax);
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0) {
    s.wmin[warp] = kmin;
    s.wmax[warp] = kmax;
    s.wcnt[warp] = n;
  }
  __syncthreads();
  kmin = __reduce_min_sync(0xffffffffu, lane < W ? s.wmin[lane] : 0xffffffffu);
  kmax = __reduce_max_sync(0xffffffffu, lane < W ? s.wmax[lane] : 0u);
  n = __reduce_add_sync(0xffffffffu, lane < W ? s.wcnt[lane] : 0u);
  if constexpr (C > 1) {
    if (warp == 0 && lane < C) {
      peer_store(&s.rmin[rank], lane, kmin);
      peer_store(&s.rmax[rank], lane, kmax);
      peer_store(&s.rcnt[rank], lane, n);
    }
    row_sync<C>();
    kmin = __reduce_min_sync(0xffffffffu, lane < C ? s.rmin[lane] : 0xffffffffu);
    kmax = __reduce_max_sync(0xffffffffu, lane < C ? s.rmax[lane] : 0u);
    n = __reduce_add_sync(0xffffffffu, lane < C ? s.rcnt[lane] : 0u);
  }
}

template <int T, int C>
__device__ __forceinline__ void clear_histogram(TopkShared<T, C>& s) {
  uint4* h = reinterpret_cast<uint4*>(s.hist);
  for (int i = threadIdx.x; i < kBins / 4; i += T) h[i] = make_uint4(0u, 0u, 0u, 0u);
}

// The bin of the histograms (of all the row's blocks) in which the need-th
// largest lies: into s.bin, with the count above it and the one inside.
// Starts and ends with a barrier of the row / the block.
// kAlone: the histogram of this block alone.
template <int T, int C, bool kAlone = C == 1>
__device__ __forceinline__ void find_bin(TopkShared<T, C>& s, uint32_t need) {
  constexpr int W = T / 32, kOwn = kBins / T;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  row_sync<kAlone ? 1 : C>();
  uint32_t h[kOwn], sum = 0;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int b = tid * kOwn + i;
    h[i] = 0;
    if constexpr (kAlone) {
      h[i] = s.hist[b];
    } else {
#pragma unroll
      for (int r = 0; r < C; ++r) h[i] += peer_load(&s.hist[b], r);
    }
    sum += h[i];
  }
  uint32_t incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) s.wsum[warp] = incl;
  __syncthreads();
  uint32_t before = __reduce_add_sync(0xffffffffu, lane < W && lane < warp ? s.wsum[lane] : 0u);
  before += incl - sum;
  if (before < need && need <= before + sum) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      if (before < need && need <= before + h[i]) {
        s.bin = (uint32_t)(tid * kOwn + i);
        s.above = before;
        s.inside = h[i];
      }
      before += h[i];
    }
  }
  __syncthreads();
}

// Sum of the threads' counts over the row's warps and blocks before this warp.
template <int T, int C>
__device__ __forceinline__ uint32_t count_before(TopkShared<T, C>& s, int rank, uint32_t count) {
  constexpr int W = T / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t own = __reduce_add_sync(0xffffffffu, count);
  if (lane == 0) s.wsum[warp] = own;
  __syncthreads();
  const uint32_t other = lane < W ? s.wsum[lane] : 0u;
  uint32_t base = __reduce_add_sync(0xffffffffu, lane < warp ? other : 0u);
  if constexpr (C > 1) {
    const uint32_t total = __reduce_add_sync(0xffffffffu, other);
    if (warp == 0 && lane < C) peer_store(&s.rtot[rank], lane, total);
    row_sync<C>();
    base += __reduce_add_sync(0xffffffffu, lane < rank ? s.rtot[lane] : 0u);
  }
  return base;
}

// Bins linear in the scores for keys of -inf < score < +inf between the keys kmin
// and kmax, +inf and NaN above.  A range whose scale is not finite (it overflows,
// is subnormal or a single value) puts every finite score into the last bin.
struct LinearBins {
  float low, scale;

  __device__ __forceinline__ LinearBins(uint32_t kmin, uint32_t kmax) : low(score_of(kmin)) {
    scale = kmin <= kmax ? __fdividef(kBins - 0.5f, score_of(kmax) - low) : 0.0f;
    if (!(scale < CUDART_INF_F)) scale = 0.0f;
  }
  __device__ __forceinline__ int operator()(uint32_t k) const {
    if (k >= kPosInf) return 0;
    // An infinite difference times a scale of zero is NaN, which max takes to 0.
    return kBins - 1 - (int)fminf(fmaxf((score_of(k) - low) * scale, 0.0f), (float)(kBins - 1));
  }
};

// The need-th greatest entry of the row's list of `inside` <= kList entries, in
// every thread.
template <int T, int C>
__device__ __forceinline__ uint64_t list_threshold(TopkShared<T, C>& s, uint32_t inside,
                                                   uint32_t need) {
  const int tid = threadIdx.x;
  row_sync<C>();
  const uint64_t* list = s.list;
  if constexpr (C > 1) {
    if (tid < (int)inside) s.mine[tid] = peer_load64(&s.list[tid], 0);
    __syncthreads();
    list = s.mine;
  }
  if (tid < (int)inside) {
    const uint64_t e = list[tid];
    uint32_t r = 0;
    for (int j = 0; j < (int)inside; ++j) r += list[j] > e ? 1u : 0u;
    if (r + 1 == need) s.threshold = e;
  }
  __syncthreads();
  return s.threshold;
}

// Selection flags of any row, by keys.  Shared memory is in use up to here by
// no thread of the row.
template <int T, int C, int P>
__device__ __noinline__ uint32_t select_general(TopkShared<T, C>& s, const float* x, Places pl,
                                                int rank, int K, uint32_t* selectable) {
  const int tid = threadIdx.x, rounds = pl.rounds();
  uint32_t key[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    key[i] = i < rounds ? key_of(__ldg(x + pl.at(i))) : 0u;
  }
  clear_histogram<T, C>(s);

  uint32_t kmin = 0xffffffffu, kmax = 0, able = 0;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    if (key[i] > kNegInf) {
      ++able;
      if (key[i] < kPosInf) {
        kmin = min(kmin, key[i]);
        kmax = max(kmax, key[i]);
      }
    }
  }
  row_reduce<T, C>(s, rank, kmin, kmax, able);

  uint32_t sel = 0;  // bit i: key[i] is selected
  if (able <= (uint32_t)K) {
#pragma unroll
    for (int i = 0; i < P; ++i) sel |= (key[i] > kNegInf ? 1u : 0u) << i;
  } else {
    const LinearBins bin_of(kmin, kmax);
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (key[i] > kNegInf) atomicAdd(&s.hist[bin_of(key[i])], 1u);
    uint32_t need = (uint32_t)K;
    find_bin<T, C>(s, need);
    uint32_t cand = 0;
    int bin = (int)s.bin;
    need -= s.above;
    uint32_t inside = s.inside;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if (key[i] > kNegInf) {
        const int b = bin_of(key[i]);
        sel |= (b < bin ? 1u : 0u) << i;
        cand |= (b == bin ? 1u : 0u) << i;
      }
    }
    bool equal = false;
    while (inside > need && inside > kList) {
      kmin = 0xffffffffu;
      kmax = 0;
      uint32_t none = 0;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        if (cand >> i & 1) {
          kmin = min(kmin, key[i]);
          kmax = max(kmax, key[i]);
        }
      }
      row_reduce<T, C>(s, rank, kmin, kmax, none);
      if (kmin == kmax) {
        equal = true;
        break;
      }
      // Every block of the row has read the histograms: its last barrier was
      // behind them.
      clear_histogram<T, C>(s);
      __syncthreads();
      const int shift = max(0, 22 - __clz(kmax - kmin));  // range >> shift below 1024
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (cand >> i & 1) atomicAdd(&s.hist[kBins - 1 - (int)((key[i] - kmin) >> shift)], 1u);
      find_bin<T, C>(s, need);
      bin = (int)s.bin;
      need -= s.above;
      inside = s.inside;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        if (cand >> i & 1) {
          const int b = kBins - 1 - (int)((key[i] - kmin) >> shift);
          sel |= (b < bin ? 1u : 0u) << i;
          if (b != bin) cand &= ~(1u << i);
        }
      }
    }
    if (inside == need) {
      sel |= cand;
    } else if (equal) {
      // The first `need` of the equal keys by position.
      uint32_t base = count_before<T, C>(s, rank, __popc(cand));
      const uint32_t below = (1u << (tid & 31)) - 1u;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const uint32_t on = __ballot_sync(0xffffffffu, cand >> i & 1);
        if (cand >> i & 1) sel |= (base + __popc(on & below) < need ? 1u : 0u) << i;
        base += __popc(on);
      }
      row_sync<C>();  // before the counts are written again
    } else {
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (cand >> i & 1) add_entry<T, C>(s, entry_of(key[i], (uint32_t)pl.at(i)));
      const uint64_t threshold = list_threshold<T, C>(s, inside, need);
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (cand >> i & 1)
          sel |= (entry_of(key[i], (uint32_t)pl.at(i)) >= threshold ? 1u : 0u) << i;
    }
  }

  *selectable = able;
  return sel;
}

// redux over the warp, NaN if any is.
__device__ __forceinline__ float warp_min(float v) {
  float r;
  asm("redux.sync.min.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Rounds a thread: 32 make the barriers and scans of a row cheaper by half, 16
// make its phases shorter (launcher).  1024 threads an SM, 64 registers each:
// 30000 rows of 1500 to 2048, K 512, take 138 us so, 174 us with 2048 threads of
// 32 registers, some of them spilled.  (Of the instances of one block a row, that of
// 128 threads and 32 rounds spills 8 bytes; the way by keys, with 32 rounds, 52 to 96.)
template <int T, int C, int P>
__global__ void __launch_bounds__(T, C == 1 ? 1024 / T : 1) __cluster_dims__(C, 1, 1)
    topk_kernel(const float* __restrict__ scores, int64_t stride,
                const int32_t* __restrict__ lengths, int rows, int ahead, int n_cols, int K,
                int32_t* __restrict__ out) {
  constexpr int W = T / 32;
  constexpr int kStep = 4;  // rounds between looks at the last one
  constexpr float kShift = 8388608.0f;         // 2^23: integers are its low bits
  constexpr uint32_t kShiftBits = 0x4b000000u;
  __shared__ TopkShared<T, C> s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = C == 1 ? 0 : (int)(blockIdx.x % C);
  const int64_t row = blockIdx.x / C;
  const float* x = scores + row * stride;
  int32_t* o = out + row * K;
  int n = n_cols;
  if (lengths != nullptr) n = max(0, min(n, __ldg(lengths + row)));
  if (n == 0) {  // the whole row's blocks alike
    for (int i = rank * T + tid; i < K; i += C * T) o[i] = -1;
    return;
  }
  peers_arrive<C>();
  const int part = (n + C - 1) / C;  // of the block
  const int begin = min(n, rank * part), end = min(n, begin + part);
  const Places pl(begin, end, T);
  const int rounds = pl.rounds(), last = pl.last;

  // Empty places hold the row's first score, which changes no extremum.
  const float first = __ldg(x);
  float v[P];
  float low = first, high = first;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    if (i % kStep == 0 && i > last) break;
    v[i] = i < rounds ? __ldg(x + pl.at(i)) : first;
  }
  // The row that a later block will take comes into L2 meanwhile.
  if (C == 1 && row + ahead < rows) {
    int m = n_cols;
    if (lengths != nullptr) m = min(m, __ldg(lengths + row + ahead));
    const float* y = x + ahead * stride;
    for (int c = tid * 32; c < m; c += T * 32)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(y + c));
  }
  const bool short_row = n <= K;
  if (short_row) {
    // Every score is selected, unless one of them turns out to be -inf: the
    // positions are on their way before the scores are here.
    for (int i = begin + tid; i < end; i += T) o[i] = i;
    for (int i = n + rank * T + tid; i < K; i += C * T) o[i] = -1;
  } else {
    clear_histogram<T, C>(s);
    if (tid < kDirect + 4) s.list[tid] = 0;
    if (tid == 0) s.listed = 0;
  }
#pragma unroll
  for (int i = 0; i < P; ++i) {
    if (i % kStep == 0 && i > last) break;
    low = min_nan(low, v[i]);
    high = max_nan(high, v[i]);
  }
  if (C == 1 && short_row && !__syncthreads_or(!(low > -CUDART_INF_F))) return;
  low = warp_min(low);
  high = warp_max(high);
  if (lane == 0) {
    s.wmin[warp] = __float_as_uint(low);
    s.wmax[warp] = __float_as_uint(high);
  }
  __syncthreads();
  low = warp_min(__uint_as_float(s.wmin[lane % W]));
  high = warp_max(__uint_as_float(s.wmax[lane % W]));
  if constexpr (C > 1) {
    peers_wait<C>();
    if (warp == 0 && lane < C) {
      peer_store(&s.rmin[rank], lane, __float_as_uint(low));
      peer_store(&s.rmax[rank], lane, __float_as_uint(high));
    }
    row_sync<C>();
    low = warp_min(__uint_as_float(s.rmin[lane % C]));
    high = warp_max(__uint_as_float(s.rmax[lane % C]));
  }

  uint32_t sel = 0, able = (uint32_t)n;  // bit i of sel: v[i] is selected
  uint32_t valid = rounds < 32 ? (1u << rounds) - 1u : 0xffffffffu;  // bits of scores that count
  bool general = true;
  if (short_row && low > -CUDART_INF_F) return;
  // Scores of -inf (there is no NaN then) do not count: the extremes again without
  // them.  4096 rows of 16384, a third of them masked: 168 us, as keys 314 us,
  // without a mask 135 us.
  if (low == -CUDART_INF_F) {
    uint32_t kmin = 0xffffffffu, kmax = 0;
    able = 0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if (i % kStep == 0 && i > last) break;
      const bool on = i < rounds && v[i] > -CUDART_INF_F;
      sel |= (on ? 1u : 0u) << i;
      kmin = min(kmin, on ? key_of(v[i]) : 0xffffffffu);
    }
    valid = sel;
    able = __popc(sel);
    row_sync<C>();  // the extremes have been read
    row_reduce<T, C>(s, rank, kmin, kmax, able);
    low = score_of(kmin);
    general = able > (uint32_t)K;
  }
  const float scale = __fdividef((float)(kBins - 2), high - low);
  if (general && low > -CUDART_INF_F && high < CUDART_INF_F && scale > 0.0f &&
      scale < CUDART_INF_F) {
    sel = 0;
    uint32_t need = (uint32_t)K;
    // 2^23 plus the bin of a score, rounded: non-decreasing in the score.
    auto place = [&](float a) { return fmaf(a - low, scale, kShift); };
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if (i % kStep == 0 && i > last) break;
      if (valid >> i & 1)
        atomicAdd(&s.hist[kShiftBits + (kBins - 1) - __float_as_uint(place(v[i]))], 1u);
    }
    find_bin<T, C>(s, need);
    const float bin = kShift + (float)(kBins - 1 - (int)s.bin);
    need -= s.above;
    uint32_t inside = s.inside;
    // A histogram inside of the bin: bin - 0.5 .. bin + 0.5 of the first, cut
    // to 1024 bins, is non-decreasing in the score again.
    const float edge = bin - kShift - 0.5f;
    auto place2 = [&](float a) {
      const float u = fmaf(a - low, scale, -edge);
      return fminf(fmaxf(u * (float)kBins, 0.0f), (float)(kBins - 1)) + kShift;
    };
    float bin2 = kShift;
    const bool twice = inside > need && inside > kCand;
    if (twice) {
      row_sync<C>();  // every block has read the first histogram
      clear_histogram<T, C>(s);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < P; ++i) {
        if (i % kStep == 0 && i > last) break;
        if (i < rounds && place(v[i]) == bin)
          atomicAdd(&s.hist[kShiftBits + (kBins - 1) - __float_as_uint(place2(v[i]))], 1u);
      }
      find_bin<T, C>(s, need);
      bin2 = kShift + (float)(kBins - 1 - (int)s.bin);
      need -= s.above;
      inside = s.inside;
    }
    if (inside == need || inside <= kCand) {
      const bool all = inside == need;
      uint32_t cand = 0;  // of the border
      float border = 0.0f;  // the score of its highest bit
#pragma unroll
      for (int i = 0; i < P; ++i) {
        if (i % kStep == 0 && i > last) break;
        const float t = place(v[i]);
        sel |= (t > bin ? 1u : 0u) << i;
        cand |= (t == bin ? 1u : 0u) << i;
        if (t == bin) border = v[i];
      }
      const int kept = (cand & ~valid) != 0 ? -1 : 31 - __clz(cand);  // the bit `border` belongs to
      sel &= valid;
      cand &= valid;
      auto score_at = [&](int i) { return i == kept ? border : __ldg(x + pl.at(i)); };
      uint32_t mine = 0;  // listed of this thread
      if (twice || !all) {
        // Few of the border a thread, most often one.
        for (uint32_t rest = cand; rest != 0;) {
          const int i = 31 - __clz(rest);
          rest ^= 1u << i;
          const float a = score_at(i);
          if (twice) {
            const float d = place2(a) - bin2;
            if (d > 0.0f || (all && d == 0.0f)) sel |= 1u << i;
            if (d != 0.0f || all) continue;
          }
          mine |= 1u << i;
          add_entry<T, C>(s, entry_of(key_of(a), (uint32_t)pl.at(i)));
        }
      } else {
        sel |= cand;
      }
      general = false;
      if (!all) {
        row_sync<C>();
        const uint64_t* list = s.list;
        if constexpr (C > 1) {
          for (int i = tid; i < min((int)inside + 3, kCand); i += T)
            s.mine[i] = peer_load64(&s.list[i], 0);
          list = s.mine;
        }
        if (inside <= kDirect) {
          // Each thread ranks its own entries, four at a time against the list
          // (zeros behind it).
          if constexpr (C > 1) __syncthreads();
          for (uint32_t rest = mine; rest != 0;) {
            const int i = 31 - __clz(rest);
            rest ^= 1u << i;
            const uint64_t e = entry_of(key_of(score_at(i)), (uint32_t)pl.at(i));
            uint32_t r = 0;
            for (int j = 0; j < (int)inside; j += 4) {
              const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(list + j);
              const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(list + j + 2);
              r += (a.x > e ? 1u : 0u) + (a.y > e ? 1u : 0u) + (b.x > e ? 1u : 0u) +
                   (b.y > e ? 1u : 0u);
            }
            if (r < need) sel |= 1u << i;
          }
        } else {
          // What the list's entries are told apart by: their bin inside of the
          // border bin (or of bin2), then (score, position).
          const float edge3 = twice ? bin2 - kShift - 0.5f : 0.0f;
          auto place3 = [&](float a) {
            const float u = fmaf(a - low, scale, -edge) * (float)kBins;
            const float w = twice ? (u - edge3) * (float)kBins : u;
            return fminf(fmaxf(w, 0.0f), (float)(kBins - 1)) + kShift;
          };
          clear_histogram<T, C>(s);
          s.taken[tid] = 0;
          if (tid == 0) s.ranked = 0;
          __syncthreads();
          for (int i = tid; i < (int)inside; i += T)
            atomicAdd(&s.hist[kShiftBits + (kBins - 1) -
                              __float_as_uint(place3(score_of((uint32_t)(list[i] >> 32))))],
                      1u);
          find_bin<T, C, true>(s, need);
          const float bin3 = kShift + (float)(kBins - 1 - (int)s.bin);
          need -= s.above;
          const uint32_t left = s.inside;
          if (left > kList) {
            general = true;  // the same in every block of the row
          } else {
            auto take = [&](uint32_t p) {
              if ((int)p < begin || (int)p >= end) return;
              const int q = (int)p - begin, w = q / pl.seg, r = q - w * pl.seg;
              atomicOr(&s.taken[w * 32 + (r & 31)], 1u << (r >> 5));
            };
            for (int i = tid; i < (int)inside; i += T) {
              const float d = place3(score_of((uint32_t)(list[i] >> 32))) - bin3;
              if (d > 0.0f)
                take(~(uint32_t)list[i]);
              else if (d == 0.0f)
                s.entry[atomicAdd(&s.ranked, 1u)] = list[i];
            }
            __syncthreads();
            if (tid < (int)left) {
              const uint64_t e = s.entry[tid];
              uint32_t r = 0;
              for (int j = 0; j < (int)left; ++j) r += s.entry[j] > e ? 1u : 0u;
              if (r < need) take(~(uint32_t)e);
            }
            __syncthreads();
            sel |= s.taken[tid];
          }
        }
      }
    }
  }
  if (general) {
    row_sync<C>();
    if (tid == 0) s.listed = 0;
    sel = select_general<T, C, P>(s, x, pl, rank, K, &able);
  }

  uint32_t base = count_before<T, C>(s, rank, __popc(sel));
  const uint32_t below = (1u << lane) - 1u;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    if (i % kStep == 0 && i > last) break;
    uint32_t on;  // written out, for one predicate and no branch
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b32 c;\n\t.reg .b64 a;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "vote.sync.ballot.b32 %0, p, 0xffffffff;\n\t"
        "and.b32 c, %0, %2;\n\tpopc.b32 c, c;\n\tadd.u32 c, c, %3;\n\t"
        "mad.wide.u32 a, c, 4, %4;\n\t"
        "@p st.global.u32 [a], %5;\n\t}"
        : "=&r"(on)
        : "r"(sel & (1u << i)), "r"(below), "r"(base), "l"(o), "r"(pl.at(i))
        : "memory");
    base += __popc(on);
  }
  const uint32_t filled = min(able, (uint32_t)K);
  for (uint32_t i = filled + rank * T + tid; i < (uint32_t)K; i += C * T) o[i] = -1;
  if constexpr (C > 1) row_sync<C>();  // no block leaves while another reads its shared memory
}

// Rows longer than the registers of a cluster: a cluster of eight blocks reads its
// row again for each step (from L2, after the first).  The border is a range of
// keys that histograms narrow, first linear in the scores, then in the keys, and
// the selected scores are the entries (key, position) from a threshold on.
// One row of 1000000, K 2048, takes 100 us, 32 of them 300 us; 300 rows of 300000
// 730 us.  (One block a row and four passes of 8 bits: 1020, 1660 and 930 us.)
constexpr int kLongThreads = 1024, kLongBlocks = 8;

__global__ void __launch_bounds__(kLongThreads, 1) __cluster_dims__(kLongBlocks, 1, 1)
    topk_long_kernel(const float* __restrict__ scores, int64_t stride,
                     const int32_t* __restrict__ lengths, int n_cols, int K,
                     int32_t* __restrict__ out) {
  constexpr int T = kLongThreads, C = kLongBlocks;
  __shared__ TopkShared<T, C> s;
  const int tid = threadIdx.x, lane = tid & 31, rank = (int)(blockIdx.x % C);
  const int64_t row = blockIdx.x / C;
  const float* x = scores + row * stride;
  int32_t* o = out + row * K;
  int n = n_cols;
  if (lengths != nullptr) n = max(0, min(n, __ldg(lengths + row)));
  if (n == 0) {  // the whole row's blocks alike
    for (int i = rank * T + tid; i < K; i += C * T) o[i] = -1;
    return;
  }
  peers_arrive<C>();
  const int part = (int)(((int64_t)n + C - 1) / C);
  const int begin = (int)min((int64_t)n, (int64_t)rank * part);
  const Places pl(begin, min(n - begin, part) + begin, T);
  const int rounds = pl.rounds();
  // Eight rounds from `i` on, -inf behind the thread's last: loads first.
  auto load = [&](int i, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = i + j < rounds ? __ldg(x + pl.at(i + j)) : -CUDART_INF_F;
  };
  auto each = [&](auto f) {
    for (int i = 0; i < rounds; i += 8) {
      float v[8];
      load(i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) f(key_of(v[j]), pl.at(i + j));
    }
  };

  clear_histogram<T, C>(s);
  if (tid == 0) s.listed = 0;
  uint32_t kmin = 0xffffffffu, kmax = 0, able = 0;
  each([&](uint32_t k, int) {
    able += k > kNegInf ? 1u : 0u;
    if (k > kNegInf && k < kPosInf) {
      kmin = min(kmin, k);
      kmax = max(kmax, k);
    }
  });
  uint32_t row_able = able;
  peers_wait<C>();
  row_reduce<T, C>(s, rank, kmin, kmax, row_able);

  uint64_t threshold = (uint64_t)(kNegInf + 1) << 32;  // entries from it on are selected
  uint32_t count = able;                               // selected ones of the thread
  if (row_able > (uint32_t)K) {
    uint32_t need = (uint32_t)K;
    const LinearBins bin_of(kmin, kmax);
    each([&](uint32_t k, int) {
      if (k > kNegInf) atomicAdd(&s.hist[bin_of(k)], 1u);
    });
    find_bin<T, C>(s, need);
    const int bin = (int)s.bin;
    need -= s.above;
    uint32_t inside = s.inside, none = 0;
    count = 0;
    if (inside <= kList) {
      each([&](uint32_t k, int p) {
        if (k <= kNegInf) return;
        const int b = bin_of(k);
        count += b < bin ? 1u : 0u;
        if (b == bin) add_entry<T, C>(s, entry_of(k, (uint32_t)p));
      });
      threshold = list_threshold<T, C>(s, inside, need);
    } else {
      // The border's keys: its bin is a range of them.
      uint32_t from = 0xffffffffu, to = 0;
      each([&](uint32_t k, int) {
        if (k > kNegInf && bin_of(k) == bin) {
          from = min(from, k);
          to = max(to, k);
        }
      });
      row_reduce<T, C>(s, rank, from, to, none);
      while (inside > need && inside > kList && from < to) {
        // Every block has read the histograms: the barrier of row_reduce or the
        // one below was behind them.
        clear_histogram<T, C>(s);
        __syncthreads();
        const int shift = max(0, 22 - __clz(to - from));  // range >> shift below 1024
        each([&](uint32_t k, int) {
          if (k >= from && k <= to) atomicAdd(&s.hist[kBins - 1 - (int)((k - from) >> shift)], 1u);
        });
        find_bin<T, C>(s, need);
        need -= s.above;
        inside = s.inside;
        from += (uint32_t)(kBins - 1 - (int)s.bin) << shift;
        to = from + min(to - from, (1u << shift) - 1u);
        row_sync<C>();
      }
      const bool list = inside <= kList, all = inside == need;
      uint32_t equal = 0;
      each([&](uint32_t k, int p) {
        count += k > to ? 1u : 0u;
        if (k >= from && k <= to) {
          ++equal;
          if (list) add_entry<T, C>(s, entry_of(k, (uint32_t)p));
        }
      });
      if (list) {
        threshold = list_threshold<T, C>(s, inside, need);
      } else if (all) {
        threshold = (uint64_t)from << 32;
        count += equal;
      } else {
        // Equal keys: the warp that holds the need-th of them looks for it.
        uint32_t base = count_before<T, C>(s, rank, equal);
        const uint32_t own = __reduce_add_sync(0xffffffffu, equal);
        if (lane == 0) count += base < need ? min(own, need - base) : 0u;
        if (base < need && need <= base + own) {
          for (int i = 0; i <= pl.last; ++i) {
            const bool here = i < rounds && key_of(__ldg(x + pl.at(i))) == from;
            const uint32_t on = __ballot_sync(0xffffffffu, here);
            if (here && base + __popc(on & ((1u << lane) - 1u)) + 1 == need)
              for (int r = 0; r < C; ++r)
                peer_store64(&s.threshold, r, entry_of(from, (uint32_t)pl.at(i)));
            base += __popc(on);
          }
        }
        row_sync<C>();
        threshold = s.threshold;
      }
    }
    if (inside <= kList) {
      // The listed ones of the warp's positions.
      const int first = pl.begin + (tid >> 5) * pl.seg;
      const int end = min(first + pl.seg, pl.begin + pl.len);
      for (int i = lane; i < (int)inside; i += 32) {
        const uint64_t e = s.mine[i];
        const int p = (int)~(uint32_t)e;
        count += e >= threshold && p >= first && p < end ? 1u : 0u;
      }
    }
  }

  uint32_t base = count_before<T, C>(s, rank, count);
  for (int i = 0; i <= pl.last; i += 8) {
    float v[8];
    load(i, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool here = entry_of(key_of(v[j]), (uint32_t)pl.at(i + j)) >= threshold;
      const uint32_t on = __ballot_sync(0xffffffffu, here);
      if (here) o[base + __popc(on & ((1u << lane) - 1u))] = pl.at(i + j);
      base += __popc(on);
    }
  }
  const uint32_t filled = min(row_able, (uint32_t)K);
  for (uint32_t i = filled + rank * T + tid; i < (uint32_t)K; i += C * T) o[i] = -1;
  row_sync<C>();  // no block leaves while another reads its shared memory
}

}  // namespace

extern "C" int sas_topk_select(const float* scores, int64_t score_stride, const int32_t* lengths,
                               int32_t rows, int32_t num_keys, int32_t topk, int32_t* indices,
                               void* stream_ptr) {
  if (rows < 0 || num_keys < 0 || topk < 1 || score_stride < num_keys) return SAS_ERR_INVALID;
  if (rows == 0) return SAS_OK;
  if (!indices || (num_keys > 0 && !scores)) return SAS_ERR_INVALID;
  // Positions and outputs are stepped through by up to a cluster's threads.
  if (rows > INT32_MAX / 8 || topk > SAS_MAX_TOPK || num_keys > INT32_MAX - 65536)
    return SAS_ERR_UNSUPPORTED;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  // The smallest block whose registers hold the row, or a cluster of as few of
  // the largest as it takes (a cluster's barriers and remote reads cost more
  // than a block's longer phases: 256 rows of 32768 take 23 us in blocks of 1024
  // threads and 63 us in clusters of four of 512) unless the rows are so few
  // that the clusters fit the SMs side by side (16 rows 10.3 against 12.3 us).  Rows
  // of up to 16384 take 32 scores a thread where there are many of them: 4000 rows of
  // 4096 to 8192 62 us (73 us with 16 a thread), 32768 of up to 4096 178 (197), but 8
  // rows of 4096 10.3 us (8.2); about 300 to 600 rows take the same time either way.
#define SAS_TOPK(T, C, P)                                     \
  topk_kernel<T, C, P><<<(unsigned)rows * C, T, 0, stream>>>( \
      scores, score_stride, lengths, rows, sms * (1024 / T), num_keys, topk, indices)
  int dev = 0;
  const int sms = sas::current_device_sms(&dev);
  if (sms <= 0) return SAS_ERR_CUDA;
  const bool few = (int64_t)rows * 4 <= sms;
  const bool many = rows > 2 * sms;
  if (num_keys <= 16 * 128) SAS_TOPK(128, 1, 16);
  else if (num_keys <= 32 * 128 && many) SAS_TOPK(128, 1, 32);
  else if (num_keys <= 16 * 256) SAS_TOPK(256, 1, 16);
  else if (num_keys <= 32 * 256 && many) SAS_TOPK(256, 1, 32);
  else if (num_keys <= 16 * 512) SAS_TOPK(512, 1, 16);
  else if (num_keys <= 32 * 512 && many) SAS_TOPK(512, 1, 32);
  else if (num_keys <= 16 * 1024) SAS_TOPK(1024, 1, 16);
  else if (num_keys <= 32 * 1024 && few) SAS_TOPK(512, 4, 16);
  else if (num_keys <= 32 * 1024) SAS_TOPK(1024, 1, 32);
  else if (num_keys <= 32 * 1024 * 2) SAS_TOPK(1024, 2, 32);
  else if (num_keys <= 32 * 1024 * 4) SAS_TOPK(1024, 4, 32);
  else if (num_keys <= 32 * 1024 * 8) SAS_TOPK(1024, 8, 32);
  else
    topk_long_kernel<<<(unsigned)rows * kLongBlocks, kLongThreads, 0, stream>>>(
        scores, score_stride, lengths, num_keys, topk, indices);
#undef SAS_TOPK
  return cudaGetLastError() == cudaSuccess ? SAS_OK : SAS_ERR_CUDA;
}
