// token_logprobs.cu -- log probabilities of given tokens under a row of logits,
// the row's entropy and its likeliest tokens, and their gradient.
//
//   forward    m = max x, s = sum e^{x - m};  lse = m + ln s,
//              lp = (x_t - m) - ln s          (t: the row's target),
//              H  = ln s - (1/s) sum e^{x - m} (x - m),
//              the k largest x_j as log probabilities and ids, ordered by value
//              and, among equals, by index.
//   backward   dx_j = g_lp [j = t] + p_j (g_lse - g_lp - g_H (ln p_j + H)),
//              p_j = e^{x_j - lse}.
//
// A logit of -inf is a token that cannot come: p = 0, and nothing added to H or
// the gradient.  A row of which nothing is left has lse = lp = -inf, H = 0 and
// no gradient.  A NaN or +inf in a row makes its results NaN.  A negative
// target is padding (lp = 0, no gradient through lp); a target past the last
// column gives NaN and reads nothing.
#include <type_traits>

#include "row_ops.cuh"

namespace mcke_sm100 {
namespace {

constexpr int kThreads = 256;    // of the backward pass
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// 16 bytes of a row: kPer elements.  A row is taken in vectors counted from the
// 16-byte boundary at or below its first element, so rows of any length and start
// are read in whole aligned vectors; only the first and the last of a row can be
// partial, and those are read element by element.
template <class T>
struct Vec {
  static constexpr int kPer = 16 / sizeof(T);
};
template <class T>
__device__ __forceinline__ int vec_shift(const T* row) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}
// Plain loads: the backward pass may overwrite the row in place.
__device__ __forceinline__ uint4 ld_vec(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
__device__ __forceinline__ void unpack(const uint4& q, F2 (&v)[2], const float*) {
  v[0] = f2(__uint_as_float(q.x), __uint_as_float(q.y));
  v[1] = f2(__uint_as_float(q.z), __uint_as_float(q.w));
}
__device__ __forceinline__ void unpack(const uint4& q, F2 (&v)[4], const uint16_t*) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = f2(bf16_lo(w[j]), bf16_hi(w[j]));
}
// Vector of a row that starts at element `first`; -inf where the row has no element.
template <class T>
__device__ __forceinline__ uint4 ld_row(const T* row, int64_t first, int64_t cols) {
  constexpr int kPer = Vec<T>::kPer;
  if (first >= 0 && first + kPer <= cols) return ld_vec(row + first);
  uint32_t w[4];
  constexpr int kPerWord = kPer / 4;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    w[j] = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
#pragma unroll
    for (int h = 0; h < kPerWord; ++h) {
      const int64_t c = first + j * kPerWord + h;
      if (c < 0 || c >= cols) continue;
      if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(row[c]);
      else w[j] = (w[j] & (h ? 0x0000ffffu : 0xffff0000u)) | (static_cast<uint32_t>(row[c]) << (16 * h));
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Maxima that keep a NaN, as the sums they belong to do.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float vec_max(const uint4& q, const float*) {
  return max_nan(max_nan(__uint_as_float(q.x), __uint_as_float(q.y)), max_nan(__uint_as_float(q.z), __uint_as_float(q.w)));
}
__device__ __forceinline__ float vec_max(const uint4& q, const uint16_t*) {
  const uint32_t m = max_nan_bf16x2(max_nan_bf16x2(q.x, q.y), max_nan_bf16x2(q.z, q.w));
  return max_nan(bf16_lo(m), bf16_hi(m));
}
__device__ __forceinline__ float exp2_fast(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}

__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// Running statistics of a part of a row: its maximum m, s = sum 2^t and
// w = sum 2^t t with t = (x - m) log2 e, so that the maximum itself counts exactly
// 1 and 0.  Where there is nothing but -inf, m = -inf and s = w = 0.
struct Stats {
  float m, s, w;
};
// What a maximum of -inf is replaced by, so that x - m is -inf and not NaN.
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }
// The sums of `a` on the scale of a maximum m >= a.m.
__device__ __forceinline__ Stats rescale(const Stats& a, float m) {
  if (m == a.m || a.m == -INFINITY) return Stats{m, a.s, a.w};
  const float t = (a.m - m) * kLog2E;
  const float f = exp2_fast(t);
  // a maximum so far above that nothing is left: f = 0, and t may be -inf
  return Stats{m, a.s * f, f == 0.0f ? 0.0f : f * fmaf(a.s, t, a.w)};
}
__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
  const float m = max_nan(a.m, b.m);
  const Stats p = rescale(a, m), q = rescale(b, m);
  return Stats{m, p.s + q.s, p.w + q.w};
}

// Order of the alternatives: larger value first (NaN above all, -0 equal to
// +0), then lower index.  Never 0, which stands for "none", nor all ones.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return (v != v) ? 0xfffffffeu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ uint64_t full_key(float v, uint32_t index) {
  return (static_cast<uint64_t>(order_key(v)) << 32) | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ int64_t key_index(uint64_t key) {
  return static_cast<uint32_t>(~static_cast<uint32_t>(key));
}
// Dynamic shared memory of one row's search, in 8-byte words (an even number): the keys
// of the chunks of MCKE_TOP_MAX runs, where a run is more than one chunk, and the
// maxima of max_chunks chunks.
struct TopScratch {
  int run_keys, words;
  __host__ __device__ TopScratch(int max_chunks, int threads) {
    const int run = (max_chunks + threads - 1) / threads;
    run_keys = run > 1 ? MCKE_TOP_MAX * run : 0;
    words = run_keys + (max_chunks + 3) / 4 * 2;
  }
};

struct ForwardArgs {
  int64_t stride, cols;
  const int64_t* targets;
  float* logprobs;
  float* lse;
  float* entropy;
  float* top_logprobs;
  int64_t* top_ids;
  int top_k;
};

__device__ __forceinline__ uint32_t cluster_block() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_blocks() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t address_in_block(const void* p, uint32_t block) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(r)
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(block));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

constexpr int kMaxCluster = 8;
constexpr int kLoads = 4;  // vectors of a thread in flight
template <class T>
constexpr int64_t kWarpCols = 32 * kLoads * 4 * Vec<T>::kPer;  // four rounds of a warp

// For the entropy 2^t t has to stay finite.  Next to a maximum in (kMaxAbove, kMaxBelow)
// it is enough to raise the elements below kLow (-inf among them) to it, two bf16 at a
// time: 2^t is 0 for them, and t = (kLow - m) log2 e is finite.  Otherwise t itself
// is kept from falling below -200, long after 2^t is 0.
constexpr float kLow = -5e37f, kMaxAbove = -1e37f, kMaxBelow = 1e38f;
__device__ __forceinline__ void raise_low(uint4& q, const float*) {
  q.x = __float_as_uint(max_nan(__uint_as_float(q.x), kLow));
  q.y = __float_as_uint(max_nan(__uint_as_float(q.y), kLow));
  q.z = __float_as_uint(max_nan(__uint_as_float(q.z), kLow));
  q.w = __float_as_uint(max_nan(__uint_as_float(q.w), kLow));
}
__device__ __forceinline__ void raise_low(uint4& q, const uint16_t*) {
  constexpr uint32_t kLowPair = 0xfe16fe16u;  // -4.98e37 twice
  q.x = max_nan_bf16x2(q.x, kLowPair);
  q.y = max_nan_bf16x2(q.y, kLowPair);
  q.z = max_nan_bf16x2(q.z, kLowPair);
  q.w = max_nan_bf16x2(q.w, kLowPair);
}

// Shared memory of one row's search for its likeliest elements.
template <int kRowWarps>
struct TopSpace {
  static constexpr int kThreads = 32 * kRowWarps;
  alignas(16) uint64_t keys[kThreads];  // a key to each of the row's threads
  alignas(16) uint64_t best[MCKE_TOP_MAX];
  int count[kRowWarps];                 // of each warp's 32 keys, those in use
};

// The k largest of n different keys in shared memory, into best[0 .. k) in order, zeros
// behind them if there are fewer: each thread counts the keys above its own.  keys
// is 16-byte aligned, and keys[n] = 0 where n is odd.  By the `threads` threads of a
// row; `sync` is their barrier.
template <class Sync>
__device__ __forceinline__ void k_largest(const uint64_t* keys, int n, uint64_t* best, int k, int t, int threads,
                                          Sync&& sync) {
  if (t < k) best[t] = 0;
  sync();
  const ulonglong2* pairs = reinterpret_cast<const ulonglong2*>(keys);
  for (int i = t; i < n; i += threads) {
    const uint64_t mine = keys[i];
    int above = 0;
#pragma unroll 8
    for (int j = 0; 2 * j < n; ++j) {
      const ulonglong2 p = pairs[j];
      above += (p.x > mine) + (p.y > mine);
    }
    if (above < k) best[above] = mine;
  }
  sync();
}

// One warp's choice of the k largest chunk maxima, one after the other, into best: for
// small k cheaper than counting ranks, though the other warps wait for it (8192 x 32768
// bf16, k = 5: 118 us against 129; 1024 x 131072, k = 20: 82 us against 68).  A row
// that has one warp counts in any case (8192 x 2000 f32, k = 8: 26.6 us against 24.6).
constexpr int kFewTop = 8;
__device__ __forceinline__ void pick_chunks(const float* chunk_max, int chunks, int k, uint64_t* best) {
  constexpr int kHeld = 4;  // keys of a lane that stay in registers
  const int lane = threadIdx.x & 31;
  auto key_of = [&](int i) { return lane + 32 * i < chunks ? full_key(chunk_max[lane + 32 * i], lane + 32 * i) : 0; };
  uint64_t held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held[i] = key_of(i);
  uint64_t last = ~uint64_t{0};
  for (int i = 0; i < k && i < chunks; ++i) {
    uint64_t key = 0;
#pragma unroll
    for (int h = 0; h < kHeld; ++h)
      if (held[h] < last && held[h] > key) key = held[h];
    for (int h = kHeld; 32 * h < chunks; ++h) {
      const uint64_t e = key_of(h);
      if (e < last && e > key) key = e;
    }
    const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(key >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(key >> 32) == hi ? static_cast<uint32_t>(key) : 0u);
    last = (static_cast<uint64_t>(hi) << 32) | lo;
    if (lane == 0) best[i] = last;
  }
}

// The k likeliest of a block's part of the row, into space.best in order.
//
// Every warp load is a chunk of 32 vectors whose maximum the first pass left in
// chunk_max (chunk c of the part is entry c).  Ordered by maximum and, among
// equals, by position, the k best chunks hold the k best elements: an element of
// any other chunk has the k chunks' maxima before it.  In the same way the k best
// runs of `run` chunks hold the k best chunks; a run to a thread, so that ranks come
// from counting.  Only the k chunks are read again.  Their elements that the k-th
// maximum does not rule out, a few more than k, are left in 32 places of their
// warp and ranked; a warp that equal values give more than that keeps its k best in
// its lanes instead.  Where there are hardly more chunks than k their k-th maximum rules out
// little, and all of them are read again, twice: first for each thread's own maximum, whose
// k-th rules out more (1200 rows, k = 20: 2500 f32, 20 chunks, 19.1 us against 30.4; 5888
// bf16, 23 chunks, 23.2 against 20.0).  The border holds for k = 20 only: with fewer
// alternatives threads' maxima win at more chunks than it says (8000 x 4000 bf16, k = 13,
// 16 chunks of one warp, 48.6 us against the 62 taken; 1200 x 1400 f32, k = 9, 11 chunks, 10.9
// against 14).
template <class T, int kRowWarps, class Sync>
__device__ __forceinline__ void top_of_part(const T* row, int64_t cols, int64_t first_vec, int shift,
                                            const float* chunk_max, uint64_t* run_keys, int chunks, int k,
                                            TopSpace<kRowWarps>& space, Sync&& sync) {
  constexpr int kPer = Vec<T>::kPer, kThreads = TopSpace<kRowWarps>::kThreads;
  constexpr int kBatch = 2;  // chunks of a warp in flight
  const int lane = threadIdx.x & 31, warp = kRowWarps == 1 ? 0 : threadIdx.x >> 5;
  const int t = kRowWarps == 1 ? lane : threadIdx.x;
  uint64_t key = 0;
  const bool few = chunks <= k + k / 8;
  if (few) {
    float m = -INFINITY;
    for (int c = warp; c < chunks; c += kRowWarps)
      m = max_nan(m, vec_max(ld_row(row, (first_vec + static_cast<int64_t>(c) * 32 + lane) * kPer - shift, cols), row));
    space.keys[t] = full_key(m, t);
    k_largest(space.keys, kThreads, space.best, k, t, kThreads, sync);
  } else if (kRowWarps > 1 && k <= kFewTop) {
    if (warp == 0) pick_chunks(chunk_max, chunks, k, space.best);
    sync();
  } else {
    const int run = (chunks + kThreads - 1) / kThreads, runs = (chunks + run - 1) / run;
    for (int c = t * run; c < min((t + 1) * run, chunks); ++c) key = max(key, full_key(chunk_max[c], c));
    space.keys[t] = key;
    k_largest(space.keys, runs, space.best, k, t, kThreads, sync);
    if (run > 1) {
      // the chunks of those runs
      const int n = min(k, runs) * run;
      for (int i = t; i < n + (n & 1); i += kThreads) {
        const int c = i < n ? static_cast<int>(key_index(space.best[i / run])) / run * run + i % run : chunks;
        run_keys[i] = c < chunks ? full_key(chunk_max[c], c) : 0;
      }
      sync();
      k_largest(run_keys, n, space.best, k, t, kThreads, sync);
    }
  }
  const int n = few ? chunks : k;
  const float threshold = key_value(static_cast<uint32_t>(space.best[k - 1] >> 32));
  // f(lanes whose element counts, the element's value, its index), for this warp's chunks
  auto for_candidates = [&](auto&& f) {
    for (int i0 = warp; i0 < n; i0 += kRowWarps * kBatch) {
      uint4 q[kBatch];
      int64_t first[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (i0 + u * kRowWarps >= n) break;
        const int64_t c = few ? i0 + u * kRowWarps : key_index(space.best[i0 + u * kRowWarps]);
        first[u] = (first_vec + c * 32 + lane) * kPer - shift;
        q[u] = ld_row(row, first[u], cols);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (i0 + u * kRowWarps >= n) break;
        // elements lo .. hi of the vector are the row's
        const int lo = static_cast<int>(max(-first[u], int64_t{0}));
        const int hi = static_cast<int>(min(cols - first[u], static_cast<int64_t>(kPer)));
        F2 v[kPer / 2];
        unpack(q[u], v, row);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const float x = j % 2 ? split(v[j / 2]).y : split(v[j / 2]).x;
          // not below: a NaN is above all
          const unsigned lanes = __ballot_sync(0xffffffffu, !(x < threshold) && j >= lo && j < hi);
          if (lanes) f(lanes, x, static_cast<uint32_t>(first[u] + j));
        }
      }
    }
  };
  uint64_t* const mine = space.keys + 32 * warp;
  int found = 0;
  for_candidates([&](unsigned lanes, float x, uint32_t index) {
    const int at = found + __popc(lanes & ((1u << lane) - 1u));
    if ((lanes >> lane & 1u) && at < 32) mine[at] = full_key(x, index);
    found += __popc(lanes);
  });
  if (found > 32) {
    uint64_t listed = 0;  // lane l: this warp's l-th best
    for_candidates([&](unsigned lanes, float x, uint32_t index) {
      const uint64_t own = full_key(x, index);
      // of equal values the first come first: most do not reach the list
      const uint64_t last = __shfl_sync(0xffffffffu, listed, k - 1);
      unsigned todo = __ballot_sync(0xffffffffu, (lanes >> lane & 1u) && own > last);
      while (todo) {
        const int from = __ffs(todo) - 1;
        todo &= todo - 1;
        const uint64_t add = __shfl_sync(0xffffffffu, own, from);
        const int at = __popc(__ballot_sync(0xffffffffu, listed > add));
        const uint64_t up = __shfl_up_sync(0xffffffffu, listed, 1);
        if (lane == at) listed = add;
        else if (lane > at) listed = up;
      }
    });
    mine[lane] = lane < k ? listed : 0;
    found = k;
  } else if (lane >= found) {
    mine[lane] = 0;
  }
  if (lane == 0) space.count[warp] = found;
  sync();
  if (t < k) space.best[t] = 0;
  sync();
  if (lane < found) {
    key = mine[lane];
    int above = 0;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      const ulonglong2* pairs = reinterpret_cast<const ulonglong2*>(space.keys + 32 * w);
#pragma unroll 4
      for (int j = 0; 2 * j < space.count[w]; ++j) {
        const ulonglong2 p = pairs[j];
        above += (p.x > key) + (p.y > key);
      }
    }
    if (above < k) space.best[above] = key;
  }
  sync();
}

// kRowWarps > 1: a row to each cluster of 1, 2, 4 or 8 blocks of so many warps, each block
// with a run of the row's chunks; the blocks' results are joined in the first
// block's shared memory, in order.  kRowWarps = 1: a row to each warp, four to a block.
//
// One read of the row: a warp has kLoads chunks in flight, takes their maximum, and
// adds up the sums on its scale.  f32 is bound by HBM (4096 x 32768 80 us, 6.7 TB/s, 1.02 of
// the copy rate: reads alone), bf16 by issue, the exponential unit 65% busy (8192 x
// 32768 88.9 us, 6.04 TB/s, 0.92; 103 us in seconds of such calls, at the 1.65 GHz that the power
// limit leaves of 1.965); with alternatives by a row's end, in which most warps
// wait (the same rows with five 118 us).  One row of 131072: 10 us, of which 2 read it.
template <int kRowWarps>
constexpr int kBlockWarps = kRowWarps == 1 ? 4 : kRowWarps;

template <class T, int kRowWarps, bool kEntropy, bool kTop>
__global__ void __launch_bounds__(32 * kBlockWarps<kRowWarps>)
    token_logprobs_kernel(const T* __restrict__ x, const ForwardArgs a, int64_t rows, int max_chunks) {
  pdl_entry();
  constexpr int kPer = Vec<T>::kPer, kPairs = kPer / 2;
  constexpr int kWarps = kBlockWarps<kRowWarps>, kRows = kWarps / kRowWarps;
  extern __shared__ __align__(16) uint64_t top_scratch[];  // [kRows]: the runs' chunks, the chunks' maxima
  __shared__ Stats warp_stats[kWarps];
  __shared__ Stats part_stats[kRowWarps == 1 ? 1 : kMaxCluster];
  __shared__ __align__(16) uint64_t part_best[kTop && kRowWarps > 1 ? kMaxCluster * MCKE_TOP_MAX : 1];
  __shared__ TopSpace<kTop ? kRowWarps : 1> top_space[kTop ? kRows : 1];
  const int lane = threadIdx.x & 31, warp = kRowWarps == 1 ? 0 : threadIdx.x >> 5;
  const int slot = kRowWarps == 1 ? threadIdx.x >> 5 : 0;
  const uint32_t blocks = kRowWarps == 1 ? 1 : cluster_blocks(), block = kRowWarps == 1 ? 0 : cluster_block();
  const int64_t row = kRowWarps == 1 ? static_cast<int64_t>(blockIdx.x) * kRows + slot : blockIdx.x / blocks;
  if (kRowWarps == 1 && row >= rows) return;
  auto sync = [] {
    if constexpr (kRowWarps == 1) __syncwarp();
    else __syncthreads();
  };
  const TopScratch scratch(max_chunks, 32 * kRowWarps);
  uint64_t* const run_keys = top_scratch + slot * scratch.words;
  float* const chunk_max = reinterpret_cast<float*>(run_keys + scratch.run_keys);
  const T* xr = x + row * a.stride;
  const int shift = vec_shift(xr);
  const int64_t vecs = (a.cols + shift + kPer - 1) / kPer;
  const int64_t all_chunks = (vecs + 31) / 32;
  const int64_t chunk0 = all_chunks * block / blocks, chunk1 = all_chunks * (block + 1) / blocks;
  const int chunks = static_cast<int>(chunk1 - chunk0);

  // chunks inner0 .. inner1 of the part hold no vector that the row's ends cut
  const int inner0 = chunk0 == 0 && shift > 0 ? 1 : 0;
  const int inner1 = static_cast<int>(min((a.cols + shift) / (32 * kPer), chunk1) - chunk0);
  const T* const inner = xr + (chunk0 * 32 + lane) * kPer - shift;

  Stats st{-INFINITY, 0.0f, 0.0f};  // m is the warp's, the sums are the lane's
  for (int c = warp; c < chunks; c += kRowWarps * kLoads) {
    uint4 q[kLoads];
    if (c >= inner0 && c + (kLoads - 1) * kRowWarps < inner1) {
      const T* p = inner + static_cast<int64_t>(c) * (32 * kPer);
#pragma unroll
      for (int u = 0; u < kLoads; ++u) q[u] = ld_vec(p + u * kRowWarps * (32 * kPer));
    } else {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int64_t v = (chunk0 + c + u * kRowWarps) * 32 + lane;
        const int64_t first = c + u * kRowWarps < chunks ? v * kPer - shift : a.cols;  // past the row: -inf
        q[u] = ld_row(xr, first, a.cols);
      }
    }
    float m;
    if constexpr (kTop) {
      m = st.m;
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const float mu = warp_max_nan(vec_max(q[u], xr));
        if (lane == 0 && c + u * kRowWarps < chunks) chunk_max[c + u * kRowWarps] = mu;
        m = max_nan(m, mu);
      }
    } else {
      m = vec_max(q[0], xr);
#pragma unroll
      for (int u = 1; u < kLoads; ++u) m = max_nan(m, vec_max(q[u], xr));
      m = max_nan(st.m, warp_max_nan(m));
    }
    st = rescale(st, m);
    F2 s2 = f2(0.0f), w2 = f2(0.0f);
    const F2 scale = f2(kLog2E), minus_m = f2(-finite_max(m));
    auto add_up = [&](auto raise) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        if constexpr (kEntropy && decltype(raise)::value) raise_low(q[u], xr);
        F2 v[kPairs];
        unpack(q[u], v, xr);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          F2 tt = mul2(add2(v[j], minus_m), scale);
          float2 t = split(tt);
          if constexpr (kEntropy && !decltype(raise)::value) {
            t.x = max_nan(t.x, -200.0f);
            t.y = max_nan(t.y, -200.0f);
            tt = f2(t.x, t.y);
          }
          const F2 e = f2(exp2_fast(t.x), exp2_fast(t.y));
          s2 = add2(s2, e);
          if constexpr (kEntropy) w2 = fma2(e, tt, w2);
        }
      }
    };
    if (!kEntropy || (m > kMaxAbove && m < kMaxBelow)) add_up(std::true_type{});
    else add_up(std::false_type{});
    st.s += sum2(s2);
    if constexpr (kEntropy) st.w += sum2(w2);
  }
  st.s = warp_all_sum(st.s);
  if constexpr (kEntropy) st.w = warp_all_sum(st.w);
  if constexpr (kRowWarps > 1) {
    if (lane == 0) warp_stats[warp] = st;
  }
  sync();
  if constexpr (kTop)
    top_of_part<T, kRowWarps>(xr, a.cols, chunk0 * 32, shift, chunk_max, run_keys, chunks, a.top_k, top_space[slot],
                              sync);
  const uint64_t* best = top_space[slot].best;
  if constexpr (kRowWarps > 1) {
    // eight statistics, a lane to each: the same bits in every lane
    auto join_lanes = [&](Stats s8) {
#pragma unroll
      for (int o = 4; o > 0; o >>= 1)
        s8 = join(s8, Stats{__shfl_xor_sync(0xffffffffu, s8.m, o), __shfl_xor_sync(0xffffffffu, s8.s, o),
                            __shfl_xor_sync(0xffffffffu, s8.w, o)});
      return s8;
    };
    static_assert(kWarps <= 8 && kMaxCluster <= 8, "eight lanes");
    const Stats nothing{-INFINITY, 0.0f, 0.0f};
    if (warp == 0) st = join_lanes((lane & 7) < kWarps ? warp_stats[lane & 7] : nothing);
    if (blocks > 1) {
      cluster_barrier();  // every block of the cluster runs: its shared memory may be written
      if (threadIdx.x < 3) {
        const float v = threadIdx.x == 0 ? st.m : threadIdx.x == 1 ? st.s : st.w;
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(address_in_block(&part_stats[block], 0) + 4 * threadIdx.x),
                     "f"(v)
                     : "memory");
      }
      if (kTop && threadIdx.x < a.top_k)
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(
                         address_in_block(&part_best[block * a.top_k + threadIdx.x], 0)),
                     "l"(best[threadIdx.x])
                     : "memory");
      cluster_barrier();
      if (block > 0) return;
      // blocks * top_k is even
      if constexpr (kTop)
        k_largest(part_best, static_cast<int>(blocks) * a.top_k, top_space[slot].best, a.top_k, threadIdx.x,
                  32 * kWarps, sync);
    }
    if (warp > 0) return;
    if (blocks > 1)
      st = join_lanes((lane & 7) < static_cast<int>(blocks) ? part_stats[lane & 7] : nothing);
  }
  // a row of which nothing is left (with a NaN or +inf in it, m or s is not so)
  const bool none = st.m == -INFINITY;
  const float ln_s = logf(st.s);
  auto logprob = [&](float v) { return none ? -INFINITY : (v - st.m) - ln_s; };
  if (lane == 0) {
    if (a.lse) a.lse[row] = none ? -INFINITY : st.m + ln_s;
    if (kEntropy && a.entropy) a.entropy[row] = none ? 0.0f : ln_s - kLn2 * (st.w / st.s);
    if (a.logprobs) {
      const int64_t t = a.targets[row];
      a.logprobs[row] = t < 0 ? 0.0f : t >= a.cols ? NAN : logprob(ld_val(xr + t));
    }
  }
  if (kTop && lane < a.top_k) {
    a.top_ids[row * a.top_k + lane] = key_index(best[lane]);
    a.top_logprobs[row * a.top_k + lane] = logprob(key_value(static_cast<uint32_t>(best[lane] >> 32)));
  }
}

struct Grads {
  const float* lse;
  const int64_t* targets;
  const float* logprobs;
  const float* entropy;
  const float* grad_entropy;
  const float* grad_lse;
};

// dx may be x itself: a vector is read before it is written, by the same thread.
// `threads` threads of a block (a power of two) take a part of a row, kVecs vectors
// each; kSame: dx has the row's offset from a 16-byte boundary, so whole vectors
// are stored.
// A p below float's smallest normal number, 2^-126, is 0.
// f32 is bound by HBM (2048 x 32768 80 us, 1.02 of the copy rate), bf16 by issue, 77% of
// the slots (4096 x 50257 with the entropy's gradient 136 us, 6.04 TB/s, 0.92; 154 us in
// seconds of such calls, at 1.63 GHz under the power limit).  Six blocks an SM leave 40
// registers, of which the bf16 instances spill 12 to 40 bytes.  A check for whole blocks of
// vectors costs more in registers than it saves (144 us).
constexpr int kVecs = 4;
template <class T, bool kEntropy, bool kSame>
__global__ void __launch_bounds__(kThreads, 6)
    token_logprobs_backward_kernel(const T* x, int64_t stride, T* dx, int64_t dx_stride, int64_t rows, int64_t cols,
                                   int parts, int threads, Grads g) {
  pdl_entry();
  constexpr int kPer = Vec<T>::kPer, kPairs = kPer / 2;
  const int t0 = threadIdx.x & (threads - 1);
  // a block to a part of a row, or (parts == 1) several rows to a block
  const int64_t row = parts > 1 ? blockIdx.x / static_cast<unsigned>(parts)
                                : static_cast<int64_t>(blockIdx.x) * (kThreads / threads) + threadIdx.x / threads;
  const int part = parts > 1 ? static_cast<int>(blockIdx.x % static_cast<unsigned>(parts)) : 0;
  if (row >= rows) return;
  const T* xr = x + row * stride;
  T* dxr = dx + row * dx_stride;
  const int shift = vec_shift(xr);
  int64_t first[kVecs];
  uint4 q[kVecs];
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    first[u] = (static_cast<int64_t>(part * kVecs + u) * threads + t0) * kPer - shift;
    q[u] = ld_row(xr, min(first[u], cols), cols);
  }
  const float lse = g.lse[row];
  const int64_t t = g.logprobs ? g.targets[row] : -1;
  const float g_lp = t < 0 ? 0.0f : t >= cols ? NAN : g.logprobs[row];
  const float a0 = (g.grad_lse ? g.grad_lse[row] : 0.0f) - g_lp;
  const float g_h = kEntropy ? g.grad_entropy[row] : 0.0f;
  // dx = p (a - g_h (q + H)) = p (b - g_h q) besides the target's own term
  const F2 b = f2(kEntropy ? a0 - g_h * g.entropy[row] : a0), minus_gh = f2(-g_h);
  const bool none = lse == -INFINITY;
  const F2 minus_lse = f2(none ? 0.0f : -lse), scale = f2(kLog2E);
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    if (first[u] >= cols) continue;
    F2 v[kPairs];
    unpack(q[u], v, xr);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      float2 d = split(add2(v[j], minus_lse));
      if constexpr (kEntropy) {
        // p is 0 long before -150; q itself has to stay finite for p q
        d.x = max_nan(d.x, -150.0f);
        d.y = max_nan(d.y, -150.0f);
      }
      const F2 dd = f2(d.x, d.y);
      const float2 e = split(mul2(dd, scale));
      const F2 p = f2(exp2_fast(e.x), exp2_fast(e.y));
      v[j] = mul2(p, kEntropy ? fma2(dd, minus_gh, b) : b);
    }
    const int64_t hit = t - first[u];
    if (hit >= 0 && hit < kPer && !none) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) v[j] = add2(v[j], f2(hit == 2 * j ? g_lp : 0.0f, hit == 2 * j + 1 ? g_lp : 0.0f));
    }
    const bool whole = kSame && first[u] >= 0 && first[u] + kPer <= cols;
    if constexpr (sizeof(T) == 4) {
      const float2 lo = split(v[0]), hi = split(v[1]);
      if (whole) {
        st_stream_f4(dxr + first[u], make_float4(lo.x, lo.y, hi.x, hi.y));
        continue;
      }
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = split(v[j]);
        w[j] = pack_bf16x2(f.x, f.y);
      }
      if (whole) {
        st_stream_u4(dxr + first[u], make_uint4(w[0], w[1], w[2], w[3]));
        continue;
      }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int64_t c = first[u] + j;
      if (c >= 0 && c < cols) st_val(dxr + c, j % 2 ? split(v[j / 2]).y : split(v[j / 2]).x);
    }
  }
}

// Blocks that share a row: 1, 2, 4 or 8, whichever takes the least time in rounds of
// loads when the blocks run in waves over the device, with kTail rounds for what
// a block does besides its loads.  With few rows that spreads a row over eight
// blocks; with many it keeps the last wave from running half empty.  The waves are counted
// at the 40 registers of the kernels without alternatives; those with alternatives have 48 to
// 64 and fit 32 to 40 warps an SM, not 48.
template <class T, int kRowWarps, bool kTop>
int row_blocks(int64_t rows, int64_t cols) {
  constexpr int64_t kRound = 32 * kRowWarps * kLoads * Vec<T>::kPer, kTail = kTop ? 4 : 2;
  constexpr int64_t kResident = 148 * (48 / kRowWarps);
  const int64_t rounds = (cols + kRound - 1) / kRound;
  int best = 1;
  int64_t best_time = 0;
  for (int n = 1; n <= kMaxCluster && n <= rounds; n *= 2) {
    const int64_t time = ((rows * n + kResident - 1) / kResident) * ((rounds + n - 1) / n + kTail);
    if (n == 1 || time < best_time) {
      best = n;
      best_time = time;
    }
  }
  return best;
}
// A row to a warp where a block would have few rounds of loads for it, up to 32 KB, if there
// are rows enough for every SM's warps, the more the longer they are.  us, a warp against a
// block: bf16 8000 x 5000 18.2, 39.5; 3000 x 8000 15.7, 15.5; 8000 x 16000 48.0, 53.1; 8192 x
// 32768 98, 89; 1300 x 8000 9.9, 8.4; f32 8000 x 5000 28.4, 43.5; 1300 x 5000 10.5, 10.6; 8000
// x 16000 87, 78.  More than a few alternatives keep a warp long, and only narrow
// rows make up for it (4000 x 12000 bf16, k = 20: 58, 50).
template <class T>
bool warp_rows(int64_t rows, int64_t cols, int top_k) {
  if (rows < 148 * 8) return false;
  if (top_k > kFewTop) return cols <= kWarpCols<T>;
  return cols <= 32768 / static_cast<int64_t>(sizeof(T)) && cols <= rows * (sizeof(T) == 2 ? 5 : 4);
}

template <class T, int kRowWarps, bool kTop>
void launch_forward(const T* x, const ForwardArgs& a, int64_t rows, cudaStream_t s) {
  const int blocks = kRowWarps == 1 ? 1 : row_blocks<T, kRowWarps, kTop>(rows, a.cols);
  // the chunk maxima of the largest part, whatever the row's shift
  const int64_t chunks = ((a.cols + Vec<T>::kPer - 1) / Vec<T>::kPer + 1 + 31) / 32;
  const int max_chunks = kTop ? static_cast<int>((chunks + blocks - 1) / blocks + 1) : 0;
  constexpr int kRows = kBlockWarps<kRowWarps> / kRowWarps;
  const std::size_t smem = kTop ? static_cast<std::size_t>(TopScratch(max_chunks, 32 * kRowWarps).words) * kRows * 8 : 0;
  auto kernel = a.entropy ? token_logprobs_kernel<T, kRowWarps, true, kTop> : token_logprobs_kernel<T, kRowWarps, false, kTop>;
  if (smem > 32 * 1024) allow_shared_memory(reinterpret_cast<const void*>(kernel), smem);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(static_cast<unsigned>((rows + kRows - 1) / kRows * blocks));
  cfg.blockDim = dim3(32 * kBlockWarps<kRowWarps>);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(blocks);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.numAttrs = 1;
  if (pdl_enabled()) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  cudaLaunchKernelEx(&cfg, kernel, x, a, rows, max_chunks);  // errors are left for check_launch()
}

// With alternatives a row's end is long, and blocks of four warps leave more of them on
// an SM to cover it (8192 x 32768 bf16 with five: 118 us against 145 with eight, 64 x
// 131072 with eight: 12.2 against 12.9) unless the rows do not fill the device in
// either form (one row of 131072 with twenty: 11.8 us against 10.0); without, blocks of eight
// are the faster (89 us against 94).
template <class T>
void launch_forward(const T* x, const ForwardArgs& a, int64_t rows, cudaStream_t s) {
  const bool narrow = warp_rows<T>(rows, a.cols, a.top_k);
  if (a.top_k == 0) narrow ? launch_forward<T, 1, false>(x, a, rows, s) : launch_forward<T, 8, false>(x, a, rows, s);
  else if (narrow) launch_forward<T, 1, true>(x, a, rows, s);
  else if (rows * kMaxCluster <= 148) launch_forward<T, 8, true>(x, a, rows, s);
  else launch_forward<T, 4, true>(x, a, rows, s);
}

template <class T>
int launch_backward(const char* who, const T* x, int64_t stride, T* dx, int64_t dx_stride, int64_t rows, int64_t cols,
                    const Grads& g, cudaStream_t s) {
  constexpr int kPer = Vec<T>::kPer;
  const int64_t vecs = (cols + kPer - 1 + kPer - 1) / kPer;  // whatever the row's shift
  int threads = 32;
  while (threads < kThreads && threads * kVecs < vecs) threads *= 2;
  const int64_t parts = (vecs + threads * kVecs - 1) / (threads * kVecs);
  const int64_t blocks = (rows * parts + kThreads / threads - 1) / (kThreads / threads);
  if (blocks > 2147483647LL) return fail(MCKE_INVALID_ARGUMENT, "%s: too many elements for one launch", who);
  const bool same = (reinterpret_cast<std::uintptr_t>(x) - reinterpret_cast<std::uintptr_t>(dx)) % 16 == 0 &&
                    (rows == 1 || (stride - dx_stride) % kPer == 0);
  auto kernel = g.grad_entropy ? (same ? token_logprobs_backward_kernel<T, true, true>
                                       : token_logprobs_backward_kernel<T, true, false>)
                               : (same ? token_logprobs_backward_kernel<T, false, true>
                                       : token_logprobs_backward_kernel<T, false, false>);
  launch_async(kernel, static_cast<unsigned>(blocks), kThreads, 0, s, x, stride, dx, dx_stride, rows, cols,
               static_cast<int>(parts), threads, g);
  return MCKE_OK;
}

}  // namespace
}  // namespace mcke_sm100

using namespace mcke_sm100;

extern "C" int mcke_sm100_token_logprobs(const void* logits, int64_t stride, int64_t rows, int64_t cols, int dtype,
                                         const int64_t* targets, float* logprobs, float* lse, float* entropy,
                                         int top_k, float* top_logprobs, int64_t* top_ids, mcke_stream_t stream) {
  static const char* who = "mcke_sm100_token_logprobs";
  clear_error();
  MCKE_RETURN_IF(check_dtype(who, dtype));
  if (rows < 0 || cols < 0) return fail(MCKE_INVALID_ARGUMENT, "%s: negative extent", who);
  if (top_k < 0 || top_k > MCKE_TOP_MAX)
    return fail(MCKE_INVALID_ARGUMENT, "%s: top_k must be 0 .. %d", who, MCKE_TOP_MAX);
  if (rows == 0) return MCKE_OK;
  if (cols == 0) return fail(MCKE_INVALID_ARGUMENT, "%s: rows of no columns have no distribution", who);
  if (rows > kMaxRows || cols > 2147483647LL)
    return fail(MCKE_INVALID_ARGUMENT, "%s: extent exceeds INT32_MAX (rows: 65536 less)", who);
  if (top_k > cols) return fail(MCKE_INVALID_ARGUMENT, "%s: top_k %d of %lld columns", who, top_k, static_cast<long long>(cols));
  if (top_k > 0 && cols > MCKE_TOP_COLS_MAX)
    return fail(MCKE_INVALID_ARGUMENT, "%s: top_k of more than %d columns", who, MCKE_TOP_COLS_MAX);
  if (!logits || (logprobs && !targets) || (top_k > 0 && (!top_logprobs || !top_ids)))
    return fail(MCKE_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!logprobs && !lse && !entropy && top_k == 0) return MCKE_OK;
  MCKE_RETURN_IF(check_stride(who, "logits", stride, rows, cols, false));
  const std::size_t e = dtype_bytes(dtype);
  MCKE_RETURN_IF(check_aligned(who, {{"logits", logits, e}, {"targets", targets, 8}, {"logprobs", logprobs, 4},
                                     {"lse", lse, 4}, {"entropy", entropy, 4},
                                     {"top_logprobs", top_logprobs, 4}, {"top_ids", top_ids, 8}}));
  const RowSpan outs[] = {span_of("logprobs", logprobs, rows * 4), span_of("lse", lse, rows * 4),
                          span_of("entropy", entropy, rows * 4),
                          span_of("top_logprobs", top_k > 0 ? top_logprobs : nullptr, rows * top_k * 4),
                          span_of("top_ids", top_k > 0 ? top_ids : nullptr, rows * top_k * 8)};
  const RowSpan ins[] = {span_of("logits", logits, rows, cols, stride, e), span_of("targets", targets, rows * 8)};
  MCKE_RETURN_IF(check_overlaps(who, outs, ins));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const ForwardArgs a = {stride, cols, targets, logprobs, lse, entropy, top_logprobs, top_ids, top_k};
  if (dtype == MCKE_DTYPE_BF16) launch_forward(static_cast<const uint16_t*>(logits), a, rows, s);
  else launch_forward(static_cast<const float*>(logits), a, rows, s);
  return check_launch(who);
}

extern "C" int mcke_sm100_token_logprobs_backward(const void* logits, int64_t stride, int64_t rows, int64_t cols,
                                                  int dtype, const float* lse, const int64_t* targets,
                                                  const float* grad_logprobs, const float* entropy,
                                                  const float* grad_entropy, const float* grad_lse, void* dlogits,
                                                  int64_t dlogits_stride, mcke_stream_t stream) {
  static const char* who = "mcke_sm100_token_logprobs_backward";
  clear_error();
  MCKE_RETURN_IF(check_dtype(who, dtype));
  if (rows < 0 || cols < 0) return fail(MCKE_INVALID_ARGUMENT, "%s: negative extent", who);
  if (rows == 0 || cols == 0) return MCKE_OK;
  if (rows > kMaxRows || cols > 2147483647LL)
    return fail(MCKE_INVALID_ARGUMENT, "%s: extent exceeds INT32_MAX (rows: 65536 less)", who);
  if (!logits || !lse || !dlogits || (grad_logprobs && !targets) || (grad_entropy && !entropy))
    return fail(MCKE_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!grad_logprobs && !grad_entropy && !grad_lse)
    return fail(MCKE_INVALID_ARGUMENT, "%s: no gradient is given", who);
  MCKE_RETURN_IF(check_stride(who, "logits", stride, rows, cols, false));
  MCKE_RETURN_IF(check_stride(who, "dlogits", dlogits_stride, rows, cols, true));
  const std::size_t e = dtype_bytes(dtype);
  MCKE_RETURN_IF(check_aligned(who, {{"logits", logits, e}, {"dlogits", dlogits, e}, {"lse", lse, 4},
                                     {"targets", targets, 8}, {"grad_logprobs", grad_logprobs, 4},
                                     {"entropy", entropy, 4}, {"grad_entropy", grad_entropy, 4},
                                     {"grad_lse", grad_lse, 4}}));
  const bool in_place = dlogits == logits && (rows == 1 || dlogits_stride == stride);
  const RowSpan outs[] = {span_of("dlogits", dlogits, rows, cols, dlogits_stride, e)};
  const RowSpan ins[] = {span_of("logits", in_place ? nullptr : logits, rows, cols, stride, e),
                         span_of("lse", lse, rows * 4),
                         span_of("targets", grad_logprobs ? targets : nullptr, rows * 8),
                         span_of("grad_logprobs", grad_logprobs, rows * 4),
                         span_of("entropy", grad_entropy ? entropy : nullptr, rows * 4),
                         span_of("grad_entropy", grad_entropy, rows * 4),
                         span_of("grad_lse", grad_lse, rows * 4)};
  MCKE_RETURN_IF(check_overlaps(who, outs, ins));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const Grads g = {lse, targets, grad_logprobs, entropy, grad_entropy, grad_lse};
  if (dtype == MCKE_DTYPE_BF16)
    MCKE_RETURN_IF(launch_backward(who, static_cast<const uint16_t*>(logits), stride, static_cast<uint16_t*>(dlogits),
                                   dlogits_stride, rows, cols, g, s));
  else
    MCKE_RETURN_IF(launch_backward(who, static_cast<const float*>(logits), stride, static_cast<float*>(dlogits),
                                   dlogits_stride, rows, cols, g, s));
  return check_launch(who);
}
