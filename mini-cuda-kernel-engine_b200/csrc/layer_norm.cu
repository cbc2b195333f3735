// layer_norm.cu -- layer norm over the last dim, forward and backward.
//
//   forward    mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps),
//              y = (x - mu) r w + b;  mu and r are kept for the backward pass.
//   backward   xh = (x - mu) r, g = dy w,
//              dx = r (g - mean(g) - xh mean(g xh)),
//              dw = sum over rows of dy xh,  db = sum over rows of dy.
//
// Statistics and sums are float whatever the tensors' type; y and dx are rounded
// once.  The variance is the mean of the squared deviations from the row's
// mean, not a difference of two large sums.
#include <map>
#include <mutex>
#include <new>
#include <type_traits>
#include <utility>

#include "row_ops.cuh"

namespace mcke_sm100 {
namespace {

// One persistent block on each SM of a B200, a constant so that results do not
// depend on the device.
constexpr int64_t kStreamBlocks = 148;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// A thread's unit of a row: 16 bytes of it.
template <class T>
struct Unit;
template <>
struct Unit<float> {
  static constexpr int kPer = 4;
  static __device__ __forceinline__ uint4 load(const float* p) { return ld_stream_u4(p); }
  static __device__ __forceinline__ void pairs(const uint4& q, F2 (&v)[2]) {
    v[0] = f2(__uint_as_float(q.x), __uint_as_float(q.y));
    v[1] = f2(__uint_as_float(q.z), __uint_as_float(q.w));
  }
  static __device__ __forceinline__ void store_pairs(float* p, const F2 (&v)[2]) {
    const float2 a = split(v[0]), b = split(v[1]);
    st_stream_f4(p, make_float4(a.x, a.y, b.x, b.y));
  }
};
template <>
struct Unit<uint16_t> {
  static constexpr int kPer = 8;
  static __device__ __forceinline__ uint4 load(const uint16_t* p) { return ld_stream_u4(p); }
  static __device__ __forceinline__ void pairs(const uint4& q, F2 (&v)[4]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = f2(bf16_lo(w[j]), bf16_hi(w[j]));
  }
  static __device__ __forceinline__ void store_pairs(uint16_t* p, const F2 (&v)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = split(v[j]);
      w[j] = pack_bf16x2(a.x, a.y);
    }
    st_stream_u4(p, make_uint4(w[0], w[1], w[2], w[3]));
  }
};
__device__ __forceinline__ uint4 no_unit() { return make_uint4(0u, 0u, 0u, 0u); }

// kPer consecutive floats of a parameter vector (`other` where there is none).
template <int kPer>
__device__ __forceinline__ void load_param(const float* p, int c, float other, float (&v)[kPer]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = other;
  } else {
#pragma unroll
    for (int j = 0; j < kPer; j += 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(p + c + j));
      v[j] = f.x;
      v[j + 1] = f.y;
      v[j + 2] = f.z;
      v[j + 3] = f.w;
    }
  }
}

// Blocks of a row kernel that are to fit an SM: its registers are held to that, or the
// compiler keeps a row's parameters in flight and leaves no room for other rows.
template <class T, int kUnits, int kRowWarps>
struct RowBlocks {
  static constexpr int kThreadsPer = kRowWarps == 1 ? kThreads : 32 * kRowWarps;
  static constexpr int kRegs = Unit<T>::kPer * kUnits + 36;  // the row as floats, and the rest
  static constexpr int kMin = 65536 / (kThreadsPer * kRegs) < 1 ? 1 : 65536 / (kThreadsPer * kRegs);
};

struct ForwardArgs {
  const void* x;
  int64_t x_stride;
  const float* weight;
  const float* bias;
  void* y;
  int64_t y_stride;
  float* mean;
  float* rstd;
  int rows, cols;
  float eps;
};

// kPer consecutive values of a parameter vector, in pairs.
template <int kPer>
__device__ __forceinline__ void load_param_pairs(const float* p, int c, float other, F2 (&v)[kPer / 2]) {
  float f[kPer];
  load_param<kPer>(p, c, other, f);
#pragma unroll
  for (int j = 0; j < kPer / 2; ++j) v[j] = f2(f[2 * j], f[2 * j + 1]);
}

// A row in the registers of kRowWarps warps, kUnits units a thread (a warp per row: eight
// rows a block, no barrier; else a block per row): x is read once and y
// written once.  kFull: the row fills the threads' units, and none needs a check.
// Bound by HBM for f32: 16384 x 2048 in 42.3 us (6.35 TB/s, 0.97 of the copy rate).
template <class T, int kUnits, int kRowWarps, bool kFull>
__global__ void __launch_bounds__(kRowWarps == 1 ? kThreads : 32 * kRowWarps, RowBlocks<T, kUnits, kRowWarps>::kMin)
    layer_norm_kernel(const ForwardArgs a) {
  pdl_entry();
  using U = Unit<T>;
  constexpr int kPer = U::kPer, kPairs = kPer / 2;
  __shared__ float red[2][kRowWarps];
  const int t = kRowWarps == 1 ? threadIdx.x & 31 : threadIdx.x;
  const int row = kRowWarps == 1 ? blockIdx.x * kWarps + (threadIdx.x >> 5) : blockIdx.x;
  if (kRowWarps == 1 && row >= a.rows) return;
  const T* xr = static_cast<const T*>(a.x) + row * a.x_stride + t * kPer;
  T* yr = static_cast<T*>(a.y) + row * a.y_stride + t * kPer;
  constexpr int kStep = 32 * kRowWarps * kPer;
  auto live = [&](int i) { return kFull || i * kStep + t * kPer < a.cols; };
  uint4 q[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) q[i] = live(i) ? U::load(xr + i * kStep) : no_unit();
  F2 s2 = f2(0.0f);
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    F2 v[kPairs];
    U::pairs(q[i], v);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) s2 = add2(s2, v[j]);
  }
  const float n = static_cast<float>(a.cols), inv_n = 1.0f / n;
  const float s = kRowWarps == 1 ? warp_all_sum(sum2(s2)) : block_all_sum<kRowWarps>(sum2(s2), red[0]);
  const float mu = div_by(s, n, inv_n);
  const F2 minus_mu = f2(-mu);
  F2 d2 = f2(0.0f);
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    if (!live(i)) continue;
    F2 v[kPairs];
    U::pairs(q[i], v);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      v[j] = add2(v[j], minus_mu);
      d2 = fma2(v[j], v[j], d2);
    }
  }
  const float var = kRowWarps == 1 ? warp_all_sum(sum2(d2)) : block_all_sum<kRowWarps>(sum2(d2), red[1]);
  const float r = rsqrtf(div_by(var, n, inv_n) + a.eps);
  if (t == 0) {
    if (a.mean) a.mean[row] = mu;
    if (a.rstd) a.rstd[row] = r;
  }
  const F2 rr = f2(r);
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    if (!live(i)) continue;
    F2 v[kPairs], w[kPairs], b[kPairs];
    U::pairs(q[i], v);
    load_param_pairs<kPer>(a.weight, i * kStep + t * kPer, 1.0f, w);
    load_param_pairs<kPer>(a.bias, i * kStep + t * kPer, 0.0f, b);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) v[j] = fma2(mul2(add2(v[j], minus_mu), rr), w[j], b[j]);
    U::store_pairs(yr + i * kStep, v);
  }
}

// Rows that are not whole 16-byte units from a 16-byte boundary on: a block per row,
// consecutive threads on consecutive elements, kPairs pairs of elements (of columns
// c and c + kThr) to a thread.  The row fills all pairs but the last.
template <class T, int kPairs, int kThr>
__global__ void __launch_bounds__(kThr) layer_norm_elements_kernel(const ForwardArgs a) {
  pdl_entry();
  __shared__ float red[2][kThr / 32];
  const int row = blockIdx.x;
  const T* xr = static_cast<const T*>(a.x) + row * a.x_stride + threadIdx.x;
  T* yr = static_cast<T*>(a.y) + row * a.y_stride + threadIdx.x;
  const int left = a.cols - 2 * (kPairs - 1) * kThr - static_cast<int>(threadIdx.x);  // the last pair's: > 0, > kThr
  auto lo_live = [&](int i) { return i + 1 < kPairs || left > 0; };
  auto hi_live = [&](int i) { return i + 1 < kPairs || left > kThr; };
  F2 v[kPairs];
#pragma unroll
  for (int i = 0; i < kPairs; ++i)
    v[i] = f2(lo_live(i) ? ld_val(xr + 2 * i * kThr) : 0.0f, hi_live(i) ? ld_val(xr + (2 * i + 1) * kThr) : 0.0f);
  F2 s2 = v[0];
#pragma unroll
  for (int i = 1; i < kPairs; ++i) s2 = add2(s2, v[i]);
  const float n = static_cast<float>(a.cols), inv_n = 1.0f / n;
  const float mu = div_by(block_all_sum<kThr / 32>(sum2(s2), red[0]), n, inv_n);
  const F2 minus_mu = f2(-mu);
  F2 d2 = f2(0.0f);
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    v[i] = add2(v[i], minus_mu);
    const float2 d = split(v[i]);
    const F2 counted = i + 1 < kPairs ? v[i] : f2(lo_live(i) ? d.x : 0.0f, hi_live(i) ? d.y : 0.0f);
    d2 = fma2(counted, counted, d2);
  }
  const float r = rsqrtf(div_by(block_all_sum<kThr / 32>(sum2(d2), red[1]), n, inv_n) + a.eps);
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[row] = mu;
    if (a.rstd) a.rstd[row] = r;
  }
  const F2 rr = f2(r);
  auto finish = [&](auto weight, auto bias) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const int c = 2 * i * kThr + threadIdx.x;
      const F2 w = f2(lo_live(i) ? weight(c) : 0.0f, hi_live(i) ? weight(c + kThr) : 0.0f);
      const F2 b = f2(lo_live(i) ? bias(c) : 0.0f, hi_live(i) ? bias(c + kThr) : 0.0f);
      const float2 y = split(fma2(mul2(v[i], rr), w, b));
      if (lo_live(i)) st_val(yr + 2 * i * kThr, y.x);
      if (hi_live(i)) st_val(yr + (2 * i + 1) * kThr, y.y);
    }
  };
  auto w_at = [&](int c) { return __ldg(a.weight + c); };
  auto b_at = [&](int c) { return __ldg(a.bias + c); };
  auto one = [](int) { return 1.0f; };
  auto zero = [](int) { return 0.0f; };
  if (a.weight && a.bias) finish(w_at, b_at);
  else if (a.weight) finish(w_at, zero);
  else if (a.bias) finish(one, b_at);
  else finish(one, zero);
}

// ---- rows streamed through shared memory ----------------------------------------
//
// A persistent block per SM of kGroups groups of kWarps warps; a group works on a
// row at a time and a thread on the same kUnits 16-byte units of every row, so
// the parameters (and the backward pass's column sums) stay in its registers.
// Rows come through a ring of kStages in shared memory filled by asynchronous
// copies: a thread copies only what it will read itself, so the ring needs no
// barrier, and rows ahead are in flight while a row is worked on.
template <class T, int kUnits, int kWarps, int kGroups, int kStages, int kOperands>
struct Stream {
  static constexpr int kTpg = 32 * kWarps;
  static constexpr int kThreads = kTpg * kGroups;
  static constexpr std::size_t kSmem = static_cast<std::size_t>(kStages) * kOperands * kUnits * kThreads * 16;
  static_assert(kGroups <= 15, "a named barrier per group, besides the block's");
};

__device__ __forceinline__ void copy_unit_async(const uint4* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// Sums kN values over the warp; value i is left in lanes i * 32 / kN on.  The values
// part ways on the first exchanges (of four, 16 lanes go on with two each, then 8
// lanes with one), so four cost six shuffles.
template <int kN>
__device__ __forceinline__ float warp_sums(const float (&v)[kN]) {
  const int lane = threadIdx.x & 31;
  const bool up = lane & 16;
  float a;
  if constexpr (kN == 4) {
    const bool right = lane & 8;
    a = (up ? v[2] : v[0]) + __shfl_xor_sync(0xffffffffu, up ? v[0] : v[2], 16);
    const float b = (up ? v[3] : v[1]) + __shfl_xor_sync(0xffffffffu, up ? v[1] : v[3], 16);
    a = (right ? b : a) + __shfl_xor_sync(0xffffffffu, right ? a : b, 8);
  } else {
    a = (up ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, up ? v[0] : v[1], 16);
  }
#pragma unroll
  for (int o = 16 / kN; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  return a;
}

// Sums of four values over a group of kW warps at once: the same bits in every
// thread.  Behind the group's barrier eight lanes per value add the warps' sums
// up.  The two halves take turns, so a thread that still reads one is never
// overtaken (the next write to it comes behind the other half's barrier).
template <int kW>
struct GroupSums {
  static constexpr int kPerLane = (kW + 7) / 8;
  float part[2][4][8 * kPerLane];
};
template <int kW>
__device__ __forceinline__ void group_all_sum(float (&v)[4], GroupSums<kW>& red, int& parity, int group) {
  const int lane = threadIdx.x & 31;
  float a = warp_sums(v);
  if constexpr (kW > 1) {
    float(*r)[8 * GroupSums<kW>::kPerLane] = red.part[parity];
    parity ^= 1;
    if ((lane & 7) == 0) r[lane >> 3][(threadIdx.x >> 5) % kW] = a;
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(32 * kW) : "memory");
    const int at = (lane & 7) * GroupSums<kW>::kPerLane;
    const float* mine = r[lane >> 3] + at;
    a = 0.0f;
#pragma unroll
    for (int i = 0; i < GroupSums<kW>::kPerLane; ++i)
      if (at + i < kW) a += mine[i];
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __shfl_sync(0xffffffffu, a, 8 * i);
}

// Two rows at a time, 16 elements of each to a thread; the sums of the next two
// rows and the squared deviations of the current two are reduced together, so
// two rows cost one barrier and six shuffles although each variance is taken
// about its row's exact mean.  bf16 rows have half the bytes to cover the same
// instructions: 8192 x 4096 bf16 took 48 us with a row to a block and the parameters
// from L1, 29.5 with one row at a time here, 22.4 with two (5.99 TB/s, 0.92 of the copy
// rate); 32768 x 1024 20.6 us (1.00).
template <class T, int kW, int kGroups, int kStages, bool kFull>
__global__ void __launch_bounds__(32 * kW * kGroups, 1) layer_norm_stream_kernel(const ForwardArgs a) {
  pdl_entry();
  using U = Unit<T>;
  constexpr int kPer = U::kPer, kPairs = kPer / 2, kUnits = 16 / kPer;
  using S = Stream<T, kUnits, kW, kGroups, kStages, 2>;
  extern __shared__ __align__(128) uint4 ring[];
  __shared__ GroupSums<kW> red[kGroups];
  constexpr int kTpr = S::kTpg;
  const int group = threadIdx.x / S::kTpg, t = threadIdx.x % S::kTpg;
  auto live = [&](int i) { return kFull || (i * kTpr + t) * kPer < a.cols; };
  uint4* const mine = ring + threadIdx.x;
  // rows 2 p and 2 p + 1 of pair p = blockIdx.x + gridDim.x * (group + kGroups * j)
  const int step = 2 * gridDim.x * kGroups;
  int row = 2 * (blockIdx.x + gridDim.x * group);
  int ahead_row = row;
  const T* ahead = static_cast<const T*>(a.x) + ahead_row * a.x_stride + t * kPer;
  auto fetch = [&](int stage) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (ahead_row + k < a.rows) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i)
          if (live(i))
            copy_unit_async(mine + ((stage * 2 + k) * kUnits + i) * S::kThreads, ahead + k * a.x_stride + i * kTpr * kPer);
      }
    }
    copies_commit();
    ahead += step * a.x_stride;
    ahead_row += step;
  };
  // this thread's units of row r (that has arrived), and their sum
  auto take = [&](int r, int stage, int k, uint4 (&q)[kUnits]) {
    F2 s = f2(0.0f);
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      q[i] = r < a.rows && live(i) ? mine[((stage * 2 + k) * kUnits + i) * S::kThreads] : no_unit();
      F2 v[kPairs];
      U::pairs(q[i], v);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) s = add2(s, v[j]);
    }
    return sum2(s);
  };
#pragma unroll
  for (int k = 0; k < kStages - 1; ++k) fetch(k);
  F2 w[kUnits][kPairs], b[kUnits][kPairs];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    load_param_pairs<kPer>(live(i) ? a.weight : nullptr, (i * kTpr + t) * kPer, 1.0f, w[i]);
    load_param_pairs<kPer>(live(i) ? a.bias : nullptr, (i * kTpr + t) * kPer, 0.0f, b[i]);
  }
  const float n = static_cast<float>(a.cols), inv_n = 1.0f / n;
  int parity = 0, stage = 0;
  uint4 q[2][kUnits];
  float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f}, mu[2];
  copies_wait<kStages - 2>();
#pragma unroll
  for (int k = 0; k < 2; ++k) sums[k] = take(row + k, 0, k, q[k]);
  group_all_sum(sums, red[group], parity, group);
#pragma unroll
  for (int k = 0; k < 2; ++k) mu[k] = div_by(sums[k], n, inv_n);
  T* yr = static_cast<T*>(a.y) + row * a.y_stride + t * kPer;
  for (; row < a.rows; row += step) {
    fetch(stage == 0 ? kStages - 1 : stage - 1);
    stage = stage + 1 == kStages ? 0 : stage + 1;
    copies_wait<kStages - 2>();
    uint4 next[2][kUnits];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      sums[k] = take(row + step + k, stage, k, next[k]);
      F2 d2 = f2(0.0f);
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const F2 minus_mu = f2(live(i) ? -mu[k] : 0.0f);  // a deviation of 0 past the row's end
        F2 v[kPairs];
        U::pairs(q[k][i], v);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const F2 d = add2(v[j], minus_mu);
          d2 = fma2(d, d, d2);
        }
      }
      sums[2 + k] = sum2(d2);
    }
    group_all_sum(sums, red[group], parity, group);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (row + k >= a.rows) break;
      const float r = rsqrtf(div_by(sums[2 + k], n, inv_n) + a.eps);
      if (t == 0) {
        if (a.mean) a.mean[row + k] = mu[k];
        if (a.rstd) a.rstd[row + k] = r;
      }
      const F2 rr = f2(r), minus_mu = f2(-mu[k]);
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        F2 v[kPairs];
        U::pairs(q[k][i], v);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) v[j] = fma2(mul2(add2(v[j], minus_mu), rr), w[i][j], b[i][j]);
        if (live(i)) U::store_pairs(yr + k * a.y_stride + i * kTpr * kPer, v);
      }
    }
    yr += step * a.y_stride;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      mu[k] = div_by(sums[k], n, inv_n);
#pragma unroll
      for (int i = 0; i < kUnits; ++i) q[k][i] = next[k][i];
    }
  }
  copies_wait<0>();
}

__device__ __forceinline__ uint32_t block_in_cluster() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- sums that are posted and collected -----------------------------------------
//
// A sum over a row's warps comes in two parts: a warp posts its share and goes on
// with other rows while the others' arrive, and collects the sum later.  Each warp
// leaves its share in the shared memory of every block of the cluster and arrives on
// that block's barrier; behind it eight lanes per value add the shares up.
// Four places take turns.  A warp posts row j + 4 behind its collection of row
// j + 2, which every warp posted behind its collection of row j: nobody still
// reads the place of row j.
constexpr int kPlaces = 4;
constexpr unsigned long long kWaitNs = 2000000000ull;
__device__ uint32_t g_layer_norm_watchdog;

template <int kN, int kW, int kCluster>
struct PostedSums {
  static_assert(kN == 2 || kN == 4, "values");
  static constexpr int kEntries = kW * kCluster;  // shares per value
  static constexpr int kPerLane = (kEntries + 7) / 8;
  float share[kPlaces][kN][8 * kPerLane];
  uint64_t arrived[kPlaces];
  volatile int gave_up;  // a wait has run out: the later ones do not wait
};

__device__ __forceinline__ uint32_t shared_address(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint32_t in_block(uint32_t address, uint32_t block) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(address), "r"(block));
  return r;
}

// By one thread, before any warp of the cluster posts.
template <int kN, int kW, int kCluster>
__device__ __forceinline__ void init_sums(PostedSums<kN, kW, kCluster>& p) {
  p.gave_up = 0;
  for (int k = 0; k < kPlaces; ++k)
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_address(&p.arrived[k])), "r"(kW) : "memory");
}

// Posts a warp's shares of kN values to place k.
template <int kN, int kW, int kCluster>
__device__ __forceinline__ void post_sums(const float (&v)[kN], PostedSums<kN, kW, kCluster>& p, int k) {
  constexpr int kLanes = 32 / kN;
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % kW;
  const float a = warp_sums(v);
  const uint32_t bar = shared_address(&p.arrived[k]);
  if constexpr (kCluster == 1) {
    if (lane % kLanes == 0) p.share[k][lane / kLanes][warp] = a;
    __syncwarp();
    if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
  } else {
    // the first kCluster lanes of each value store it into those blocks; the stores
    // complete on the barrier there
    const uint32_t to = lane % kLanes;
    if (to < kCluster) {
      const uint32_t at = shared_address(&p.share[k][lane / kLanes][block_in_cluster() * kW + warp]);
      asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(in_block(at, to)),
                   "r"(__float_as_uint(a)), "r"(in_block(bar, to))
                   : "memory");
    }
    // this block's warps arrive; the first of them says how many bytes are to come
    if (lane == 0) {
      if (warp == 0)
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar),
                     "n"(kN * 4 * PostedSums<kN, kW, kCluster>::kEntries)
                     : "memory");
      else
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
    }
  }
}

__device__ __forceinline__ bool try_phase(uint32_t bar, uint32_t phase) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(phase)
      : "memory");
  return done != 0;
}

// Waits, kLimitNs at most: a wait that runs out is recorded and passed, as are all later
// ones of the group, whose sums are then incomplete.
template <unsigned long long kLimitNs>
__device__ __noinline__ void wait_phase(uint32_t bar, uint32_t phase, volatile int* gave_up) {
  unsigned long long t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  while (!*gave_up && !try_phase(bar, phase)) {
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    if (t - t0 > kLimitNs) {
      *gave_up = 1;
      atomicCAS(&g_layer_norm_watchdog, 0u, 1u);
    }
  }
}

// Waits until every share of place k is there, and returns the sums: the
// same bits in every thread.
template <unsigned long long kLimitNs = kWaitNs, int kN, int kW, int kCluster>
__device__ __forceinline__ void collect_sums(float (&v)[kN], PostedSums<kN, kW, kCluster>& p, int k, uint32_t phase) {
  const uint32_t bar = shared_address(&p.arrived[k]);
  if (!try_phase(bar, phase)) wait_phase<kLimitNs>(bar, phase, &p.gave_up);
  using P = PostedSums<kN, kW, kCluster>;
  const int lane = threadIdx.x & 31, at = (lane & 7) * P::kPerLane;
  const float* mine = p.share[k][(lane >> 3) % kN] + at;
  float a = 0.0f;
#pragma unroll
  for (int i = 0; i < P::kPerLane; ++i)
    if (at + i < P::kEntries) a += mine[i];
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
#pragma unroll
  for (int i = 0; i < kN; ++i) v[i] = __shfl_sync(0xffffffffu, a, 8 * i);
}

// Self-test of the wait: of a group's two warps one posts and the other does not.  The first
// wait runs out after 20 ms and is recorded; the second could not end either and is passed.
__global__ void __launch_bounds__(64) layer_norm_selftest_kernel() {
  pdl_entry();
  __shared__ PostedSums<2, 2, 1> posted;
  if (threadIdx.x == 0) init_sums(posted);
  __syncthreads();
  if (threadIdx.x >= 32) return;
  for (int k = 0; k < 2; ++k) {
    float v[2] = {0.0f, 0.0f};
    post_sums(v, posted, k);
    collect_sums<20000000ull>(v, posted, k, 0);
  }
}

// Rows over the blocks of a cluster.  The statistics take two exchanges, the mean's and
// that of the squared deviations about it, and both ride in one post: turn p collects
// what turn p - 1 posted (the means of rows p, the variances of rows p - 1), posts the
// sums of rows p + 1 and the squared deviations of rows p, and writes rows p - 1 while
// they arrive.  "Rows p" are kRows rows; each is read from the ring in three turns
// running; kElems elements to a thread.  4096 x 16384 bf16 43.6 us (6.16 TB/s, 0.94 of the
// copy rate); for rows that one block holds the kernel above is the faster (8192 x 4096:
// 22.4 us against 24.4).
template <class T, int kElems, int kW, int kCluster, int kRows, int kStages, bool kFull>
__global__ void __launch_bounds__(32 * kW, 1) layer_norm_cluster_kernel(const ForwardArgs a) {
  pdl_entry();
  using U = Unit<T>;
  constexpr int kPer = U::kPer, kPairs = kPer / 2, kUnits = kElems / kPer;
  using S = Stream<T, kUnits, kW, 1, kStages, kRows>;
  extern __shared__ __align__(128) uint4 ring[];
  __shared__ PostedSums<2 * kRows, kW, kCluster> posted;
  constexpr int kTpr = S::kTpg * kCluster;  // the row's threads of all blocks
  const int t = threadIdx.x + static_cast<int>(block_in_cluster()) * S::kTpg;
  auto live = [&](int i) { return kFull || (i * kTpr + t) * kPer < a.cols; };
  const int clusters = gridDim.x / kCluster, cluster = blockIdx.x / kCluster;
  const int step = kRows * clusters;
  int row = kRows * cluster;
  if (threadIdx.x == 0) init_sums(posted);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  cluster_barrier();  // every block of it runs, its barriers in place, before one posts into another
  int ahead_row = row;
  const T* ahead = static_cast<const T*>(a.x) + row * a.x_stride + t * kPer;
  constexpr int kStage = kRows * kUnits * S::kThreads;  // units of a stage
  auto slot = [&](uint4* stage, int k, int i) { return stage + (k * kUnits + i) * S::kThreads; };
  uint4* const first_stage = ring + threadIdx.x;
  uint4* const end_stage = first_stage + kStages * kStage;
  auto after = [&](uint4* stage) { return stage + kStage == end_stage ? first_stage : stage + kStage; };
  uint4 *ahead_stage = first_stage, *next_stage = first_stage, *stage = first_stage, *last_stage = first_stage;
  auto fetch = [&]() {
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (ahead_row + k < a.rows) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i)
          if (live(i)) copy_unit_async(slot(ahead_stage, k, i), ahead + k * a.x_stride + i * kTpr * kPer);
      }
    }
    copies_commit();
    ahead += step * a.x_stride;
    ahead_row += step;
    ahead_stage = after(ahead_stage);
  };
#pragma unroll
  for (int k = 0; k < kStages - 2; ++k) fetch();
  F2 w[kUnits][kPairs], b[kUnits][kPairs];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    load_param_pairs<kPer>(live(i) ? a.weight : nullptr, (i * kTpr + t) * kPer, 1.0f, w[i]);
    load_param_pairs<kPer>(live(i) ? a.bias : nullptr, (i * kTpr + t) * kPer, 0.0f, b[i]);
  }
  const float n = static_cast<float>(a.cols), inv_n = 1.0f / n;
  T* yr = static_cast<T*>(a.y) + row * a.y_stride + t * kPer;
  float mu[kRows], last_mu[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) mu[k] = 0.0f;
  row -= step;
  // turns p = -1 (it posts the first sums) to one past the last rows
  for (int turn = 0; row < a.rows + step; ++turn, row += step) {
    float c[2 * kRows];
#pragma unroll
    for (int i = 0; i < 2 * kRows; ++i) c[i] = 0.0f;
    if (turn > 0) {
      collect_sums(c, posted, (turn - 1) % kPlaces, static_cast<uint32_t>((turn - 1) / kPlaces) & 1u);
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        last_mu[k] = mu[k];
        mu[k] = div_by(c[k], n, inv_n);
      }
    }
    if (turn > 0) fetch();
    copies_wait<kStages - 3>();
    if (row < a.rows) {
      float sums[2 * kRows];
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        F2 s = f2(0.0f), d2 = f2(0.0f);
        if (row + step + k < a.rows) {
#pragma unroll
          for (int i = 0; i < kUnits; ++i) {
            F2 v[kPairs];
            U::pairs(live(i) ? *slot(next_stage, k, i) : no_unit(), v);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) s = add2(s, v[j]);
          }
        }
        if (turn > 0 && row + k < a.rows) {
#pragma unroll
          for (int i = 0; i < kUnits; ++i) {
            const F2 minus_mu = f2(live(i) ? -mu[k] : 0.0f);  // a deviation of 0 past the row's end
            F2 v[kPairs];
            U::pairs(live(i) ? *slot(stage, k, i) : no_unit(), v);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
              const F2 d = add2(v[j], minus_mu);
              d2 = fma2(d, d, d2);
            }
          }
        }
        sums[k] = sum2(s);
        sums[kRows + k] = sum2(d2);
      }
      post_sums(sums, posted, turn % kPlaces);
    }
    if (turn > 1) {
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const int done = row - step + k;
        if (kRows > 1 && done >= a.rows) break;
        const float r = rsqrtf(div_by(c[kRows + k], n, inv_n) + a.eps);
        if (t == 0) {
          if (a.mean) a.mean[done] = last_mu[k];
          if (a.rstd) a.rstd[done] = r;
        }
        const F2 rr = f2(r), minus_mu = f2(-last_mu[k]);
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          F2 v[kPairs];
          U::pairs(live(i) ? *slot(last_stage, k, i) : no_unit(), v);
#pragma unroll
          for (int j = 0; j < kPairs; ++j) v[j] = fma2(mul2(add2(v[j], minus_mu), rr), w[i][j], b[i][j]);
          if (live(i)) U::store_pairs(yr + k * a.y_stride + i * kTpr * kPer, v);
        }
      }
      yr += step * a.y_stride;
    }
    last_stage = stage;
    stage = next_stage;
    next_stage = after(next_stage);
  }
  copies_wait<0>();
  cluster_barrier();  // no block leaves while another's post may be on its way to it
}

struct BackwardArgs {
  const void* dy;
  int64_t dy_stride;
  const void* x;
  int64_t x_stride;
  const float* weight;
  const float* mean;
  const float* rstd;
  void* dx;
  int64_t dx_stride;
  float* part;  // [slabs][dw, db][cols], or null: no parameter gradients are wanted
  int rows, cols;
};

// Adds the groups' column sums, kN pairs of dw and db to a thread, to the first group's, in
// group order.  cell: (kGroups - 1) * 2 kN * kTpg pairs of shared memory that the whole
// block is done with.  False for the other groups' threads.
template <int kGroups, int kTpg, int kN>
__device__ __forceinline__ bool join_groups(F2* cell, int group, F2* dw, F2* db) {
  if constexpr (kGroups > 1) {
    cell += threadIdx.x % kTpg;  // [group - 1][dw, db][pair][thread]
    __syncthreads();
    if (group > 0) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        cell[((group - 1) * 2 * kN + i) * kTpg] = dw[i];
        cell[((group - 1) * 2 * kN + kN + i) * kTpg] = db[i];
      }
    }
    __syncthreads();
    if (group > 0) return false;
    for (int g = 0; g < kGroups - 1; ++g) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        dw[i] = add2(dw[i], cell[(g * 2 * kN + i) * kTpg]);
        db[i] = add2(db[i], cell[(g * 2 * kN + kN + i) * kTpg]);
      }
    }
  }
  return true;
}

// What x - mu is multiplied by in dx: -r^2 c2, where c2 is r times `c`, the mean of dy w
// (x - mu).  A row whose squared deviations are past float's range has r = 0 and takes no
// part, though `c` may be infinite.
__device__ __forceinline__ float dx_scale(float r, float c) { return r == 0.0f ? 0.0f : -r * r * (r * c); }

// dx, and the column sums of each slab (the rows of one cluster), in one read of dy
// and x: a thread adds up its 16 columns in registers over all its rows, the
// block's groups are added in shared memory at the end.  Each turn of the loop
// posts the sums of kRows rows and writes dx of the rows of the turn before, whose
// units are read a second time from the ring.
//
// f32 is bound by HBM (16384 x 2048 64 us, 0.96 of the copy rate), bf16 by what is issued
// for its elements: 8192 x 4096 51 us with a barrier a row, 44 with the sums posted, 36.5
// with two rows a turn, 35.4 (5.69 TB/s, 0.87) with the ring on 128 bytes.  24 warps
// instead of 16 spill (49 us).  4096 x 16384 over pairs of blocks 69.7 us (0.89).
template <class T, int kW, int kGroups, int kCluster, int kRows, int kStages, bool kFull>
__global__ void __launch_bounds__(32 * kW * kGroups, 1) layer_norm_backward_kernel(const BackwardArgs a) {
  pdl_entry();
  using U = Unit<T>;
  constexpr int kPer = U::kPer, kPairs = kPer / 2, kUnits = 16 / kPer;
  using S = Stream<T, kUnits, kW, kGroups, kStages, 2 * kRows>;
  extern __shared__ __align__(128) uint4 ring[];
  __shared__ PostedSums<2 * kRows, kW, kCluster> posted[kGroups];
  constexpr int kTpr = S::kTpg * kCluster;
  const int group = threadIdx.x / S::kTpg;
  const int t = threadIdx.x % S::kTpg + (kCluster > 1 ? static_cast<int>(block_in_cluster()) * S::kTpg : 0);
  auto live = [&](int i) { return kFull || (i * kTpr + t) * kPer < a.cols; };
  // rows kRows p .. of the turn's p = cluster + clusters * (group + kGroups * turn)
  const int clusters = gridDim.x / kCluster, cluster = blockIdx.x / kCluster;
  const int step = kRows * clusters * kGroups;
  int row = kRows * (cluster + clusters * group);
  if (threadIdx.x % S::kTpg == 0) init_sums(posted[group]);
  if constexpr (kCluster > 1) {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    cluster_barrier();  // every block of it runs, its barriers in place, before one posts into another
  } else {
    __syncthreads();
  }
  int ahead_row = row;
  const T* dy_ahead = static_cast<const T*>(a.dy) + row * a.dy_stride + t * kPer;
  const T* x_ahead = static_cast<const T*>(a.x) + row * a.x_stride + t * kPer;
  constexpr int kStage = 2 * kRows * kUnits * S::kThreads;  // units of a stage
  auto slot = [&](uint4* stage, int k, int operand, int i) {
    return stage + ((k * 2 + operand) * kUnits + i) * S::kThreads;
  };
  uint4* const first_stage = ring + threadIdx.x;
  uint4* const end_stage = first_stage + kStages * kStage;
  auto after = [&](uint4* stage) { return stage + kStage == end_stage ? first_stage : stage + kStage; };
  uint4 *stage = first_stage, *last_stage = first_stage, *ahead_stage = first_stage;
  auto fetch = [&]() {
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (ahead_row + k < a.rows) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          if (live(i)) {
            copy_unit_async(slot(ahead_stage, k, 0, i), dy_ahead + k * a.dy_stride + i * kTpr * kPer);
            copy_unit_async(slot(ahead_stage, k, 1, i), x_ahead + k * a.x_stride + i * kTpr * kPer);
          }
        }
      }
    }
    copies_commit();
    dy_ahead += step * a.dy_stride;
    x_ahead += step * a.x_stride;
    ahead_row += step;
    ahead_stage = after(ahead_stage);
  };
#pragma unroll
  for (int k = 0; k < kStages - 2; ++k) fetch();
  F2 w[kUnits][kPairs], dw[kUnits][kPairs], db[kUnits][kPairs];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    load_param_pairs<kPer>(live(i) ? a.weight : nullptr, (i * kTpr + t) * kPer, 1.0f, w[i]);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) dw[i][j] = db[i][j] = f2(0.0f);
  }
  const float n = static_cast<float>(a.cols), inv_n = 1.0f / n;
  T* dxr = static_cast<T*>(a.dx) + row * a.dx_stride + t * kPer;
  // the statistics of this turn's rows, of the last turn's and of the next one's
  float mu[kRows], r[kRows], last_mu[kRows], last_r[kRows], next_mu[kRows], next_r[kRows];
  auto stats = [&](int first, float (&m)[kRows], float (&s)[kRows]) {
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      m[k] = first + k < a.rows ? __ldg(a.mean + first + k) : 0.0f;
      s[k] = first + k < a.rows ? __ldg(a.rstd + first + k) : 0.0f;
    }
  };
  stats(row, mu, r);
  // one turn past the last rows: what is posted is collected a turn later
  for (int turn = 0; row < a.rows + step; ++turn, row += step) {
    stats(row + step, next_mu, next_r);
    fetch();
    copies_wait<kStages - 2>();
    if (row < a.rows) {
      float sums[2 * kRows];
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const F2 minus_mu = f2(-mu[k]), rr = f2(r[k]);
        F2 s1 = f2(0.0f), s2 = f2(0.0f);
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          // past the row's end, and in a row that is not there, dy = 0 adds nothing; no branch
          // around a unit's work (1600 x 20000 bf16: 47.6 us, with one 50.0)
          const bool there = live(i) && (kRows == 1 || row + k < a.rows);
          F2 d[kPairs], v[kPairs];
          U::pairs(there ? *slot(stage, k, 0, i) : no_unit(), d);
          U::pairs(there ? *slot(stage, k, 1, i) : no_unit(), v);
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            const F2 dev = add2(v[j], minus_mu), p = mul2(d[j], dev);
            db[i][j] = add2(db[i][j], d[j]);
            dw[i][j] = fma2(p, rr, dw[i][j]);
            s1 = fma2(d[j], w[i][j], s1);
            s2 = fma2(p, w[i][j], s2);
          }
        }
        sums[2 * k] = sum2(s1);
        sums[2 * k + 1] = sum2(s2);
      }
      post_sums(sums, posted[group], turn % kPlaces);
    }
    if (turn > 0) {
      float c[2 * kRows];
      collect_sums(c, posted[group], (turn - 1) % kPlaces, static_cast<uint32_t>((turn - 1) / kPlaces) & 1u);
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        if (kRows > 1 && row - step + k >= a.rows) break;
        // dx = r dy w - r c1 - (x - mu) r^2 c2
        const F2 minus_mu = f2(-last_mu[k]), rr = f2(last_r[k]);
        const F2 k1 = f2(-last_r[k] * div_by(c[2 * k], n, inv_n));
        const F2 k2 = f2(dx_scale(last_r[k], div_by(c[2 * k + 1], n, inv_n)));
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          F2 d[kPairs], v[kPairs];
          U::pairs(live(i) ? *slot(last_stage, k, 0, i) : no_unit(), d);
          U::pairs(live(i) ? *slot(last_stage, k, 1, i) : no_unit(), v);
#pragma unroll
          for (int j = 0; j < kPairs; ++j)
            v[j] = fma2(add2(v[j], minus_mu), k2, fma2(mul2(d[j], w[i][j]), rr, k1));
          if (live(i)) U::store_pairs(dxr + k * a.dx_stride + i * kTpr * kPer, v);
        }
      }
      dxr += step * a.dx_stride;
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      last_mu[k] = mu[k];
      last_r[k] = r[k];
      mu[k] = next_mu[k];
      r[k] = next_r[k];
    }
    last_stage = stage;
    stage = after(stage);
  }
  copies_wait<0>();
  if constexpr (kCluster > 1) cluster_barrier();  // no block leaves while another's post may be on its way to it
  if (!a.part) return;
  static_assert(2 * kUnits * kPairs * 8 <= static_cast<int>(S::kSmem / S::kThreads), "the ring holds the groups' sums");
  if (!join_groups<kGroups, S::kTpg, kUnits * kPairs>(reinterpret_cast<F2*>(ring), group, &dw[0][0], &db[0][0])) return;
  float* const out = a.part + static_cast<int64_t>(cluster) * 2 * a.cols + t * kPer;
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    if (!live(i)) continue;
#pragma unroll
    for (int j = 0; j < kPairs; j += 2) {
      const float2 a0 = split(dw[i][j]), a1 = split(dw[i][j + 1]), b0 = split(db[i][j]), b1 = split(db[i][j + 1]);
      *reinterpret_cast<float4*>(out + i * kTpr * kPer + 2 * j) = make_float4(a0.x, a0.y, a1.x, a1.y);
      *reinterpret_cast<float4*>(out + a.cols + i * kTpr * kPer + 2 * j) = make_float4(b0.x, b0.y, b1.x, b1.y);
    }
  }
}

// 16 elements of a thread, one behind the other, as units.
__device__ __forceinline__ void pack_units(const float (&e)[16], uint4 (&q)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    q[i] = make_uint4(__float_as_uint(e[4 * i]), __float_as_uint(e[4 * i + 1]), __float_as_uint(e[4 * i + 2]),
                      __float_as_uint(e[4 * i + 3]));
}
__device__ __forceinline__ void pack_units(const uint16_t (&e)[16], uint4 (&q)[2]) {
  auto word = [&](int j) { return static_cast<uint32_t>(e[2 * j]) | static_cast<uint32_t>(e[2 * j + 1]) << 16; };
#pragma unroll
  for (int i = 0; i < 2; ++i) q[i] = make_uint4(word(4 * i), word(4 * i + 1), word(4 * i + 2), word(4 * i + 3));
}

// The same for rows that are not whole 16-byte units: consecutive threads have consecutive
// elements, 16 of them each, in pairs (of columns c and c + kTpr).  Elements of the row
// after next come into registers (two bytes are less than an asynchronous copy
// moves) and go to the ring, of the last row, this one and the next, a turn later, as
// units: a thread reads only its own.  Bound by the element-wide accesses: 8192 x 4097
// bf16 85 us (2.37 TB/s, 0.36 of the copy rate; 98 with elements in the ring, 142 with a pass
// each for dx and for the sums), 5003 x 1537 f32 26 us (0.54); over clusters 2000 x 20001 bf16
// 119 us, the two passes 195.  Some instances spill, the f32 one over four blocks most (60
// bytes stored, 104 loaded), the others 8 and less.
template <class T, int kW, int kGroups, int kCluster>
__global__ void __launch_bounds__(32 * kW * kGroups, 1) layer_norm_backward_elements_kernel(const BackwardArgs a) {
  pdl_entry();
  using U = Unit<T>;
  constexpr int kPer = U::kPer, kUnits = 16 / kPer, kPairs = 8, kStages = 3;
  constexpr int kTpg = 32 * kW, kThr = kTpg * kGroups, kTpr = kTpg * kCluster;
  extern __shared__ __align__(128) uint4 ring[];  // [stage][dy, x][unit][thread]
  __shared__ PostedSums<2, kW, kCluster> posted[kGroups];
  static_assert(kGroups == 1 || kCluster == 1, "a block of a cluster is one group");
  const int group = threadIdx.x / kTpg;
  const int t = threadIdx.x % kTpg + (kCluster > 1 ? static_cast<int>(block_in_cluster()) * kTpg : 0);
  auto col = [&](int e) { return e * kTpr + t; };
  const int clusters = gridDim.x / kCluster, cluster = blockIdx.x / kCluster;
  const int step = clusters * kGroups;
  int row = cluster + clusters * group;
  if (threadIdx.x % kTpg == 0) init_sums(posted[group]);
  if constexpr (kCluster > 1) {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    cluster_barrier();  // every block of it runs, its barriers in place, before one posts into another
  } else {
    __syncthreads();
  }
  uint4* const units = ring + threadIdx.x;
  auto unit = [&](int stage, int operand, int i) { return units + ((stage * 2 + operand) * kUnits + i) * kThr; };
  T dyr[16], xr[16];
  auto load = [&](int64_t r) {
    if (r >= a.rows) return;
    const T* dy = static_cast<const T*>(a.dy) + r * a.dy_stride;
    const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      dyr[e] = col(e) < a.cols ? __ldg(dy + col(e)) : T(0);
      xr[e] = col(e) < a.cols ? __ldg(x + col(e)) : T(0);
    }
  };
  auto store = [&](int stage) {
    uint4 q[2][kUnits];
    pack_units(dyr, q[0]);
    pack_units(xr, q[1]);
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      *unit(stage, 0, i) = q[0][i];
      *unit(stage, 1, i) = q[1][i];
    }
  };
  // f(first pair, dy, x) over this thread's units of a stage
  auto for_units = [&](int stage, auto&& f) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      F2 d[kPer / 2], v[kPer / 2];
      U::pairs(*unit(stage, 0, i), d);
      U::pairs(*unit(stage, 1, i), v);
      f(i * (kPer / 2), d, v);
    }
  };
#pragma unroll
  for (int e = 0; e < 16; ++e) dyr[e] = xr[e] = T(0);
  load(row);
  F2 w[kPairs], dw[kPairs], db[kPairs];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const int lo = col(2 * i), hi = col(2 * i + 1);
    w[i] = f2(a.weight && lo < a.cols ? __ldg(a.weight + lo) : 1.0f, a.weight && hi < a.cols ? __ldg(a.weight + hi) : 1.0f);
    dw[i] = db[i] = f2(0.0f);
  }
  store(0);
  load(static_cast<int64_t>(row) + step);
  const float n = static_cast<float>(a.cols), inv_n = 1.0f / n;
  auto mean_of = [&](int r) { return r < a.rows ? __ldg(a.mean + r) : 0.0f; };
  auto rstd_of = [&](int r) { return r < a.rows ? __ldg(a.rstd + r) : 0.0f; };
  float mu = mean_of(row), r = rstd_of(row), last_mu = 0.0f, last_r = 0.0f;
  int stage = 0, last_stage = 0;
  for (int turn = 0; row < a.rows + step; ++turn, row += step) {
    const float next_mu = mean_of(row + step), next_r = rstd_of(row + step);
    if (row < a.rows) {
      const F2 minus_mu = f2(-mu), rr = f2(r);
      F2 s1 = f2(0.0f), s2 = f2(0.0f);
      for_units(stage, [&](int i, const auto& d, const auto& v) {
#pragma unroll
        for (int j = 0; j < kPer / 2; ++j) {
          // columns past the row have dy = 0 and add nothing
          const F2 p = mul2(d[j], add2(v[j], minus_mu));
          db[i + j] = add2(db[i + j], d[j]);
          dw[i + j] = fma2(p, rr, dw[i + j]);
          s1 = fma2(d[j], w[i + j], s1);
          s2 = fma2(p, w[i + j], s2);
        }
      });
      const float sums[2] = {sum2(s1), sum2(s2)};
      post_sums(sums, posted[group], turn % kPlaces);
    }
    const int next_stage = stage + 1 == kStages ? 0 : stage + 1;
    if (turn > 0) {
      float c[2];
      collect_sums(c, posted[group], (turn - 1) % kPlaces, static_cast<uint32_t>((turn - 1) / kPlaces) & 1u);
      const F2 minus_mu = f2(-last_mu), rr = f2(last_r);
      const F2 k1 = f2(-last_r * div_by(c[0], n, inv_n));
      const F2 k2 = f2(dx_scale(last_r, div_by(c[1], n, inv_n)));
      T* dx = static_cast<T*>(a.dx) + static_cast<int64_t>(row - step) * a.dx_stride;
      for_units(last_stage, [&](int i, const auto& d, const auto& v) {
#pragma unroll
        for (int j = 0; j < kPer / 2; ++j) {
          const float2 g = split(fma2(add2(v[j], minus_mu), k2, fma2(mul2(d[j], w[i + j]), rr, k1)));
          if (col(2 * (i + j)) < a.cols) st_val(dx + col(2 * (i + j)), g.x);
          if (col(2 * (i + j) + 1) < a.cols) st_val(dx + col(2 * (i + j) + 1), g.y);
        }
      });
    }
    store(next_stage);
    load(static_cast<int64_t>(row) + 2 * step);
    last_mu = mu;
    last_r = r;
    mu = next_mu;
    r = next_r;
    last_stage = stage;
    stage = next_stage;
  }
  if constexpr (kCluster > 1) cluster_barrier();  // no block leaves while another's post may be on its way to it
  if (!a.part) return;
  if (!join_groups<kGroups, kTpg, kPairs>(reinterpret_cast<F2*>(ring), group, dw, db)) return;
  float* const out = a.part + static_cast<int64_t>(cluster) * 2 * a.cols;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const float2 x = split(dw[i]), b = split(db[i]);
    if (col(2 * i) < a.cols) {
      out[col(2 * i)] = x.x;
      out[a.cols + col(2 * i)] = b.x;
    }
    if (col(2 * i + 1) < a.cols) {
      out[col(2 * i + 1)] = x.y;
      out[a.cols + col(2 * i + 1)] = b.y;
    }
  }
}

// Sums over a row of any length by a block, kN of them at once: terms(c, t) gives column c's.
// A thread adds four columns' terms in float, pair by pair and while the next four are
// loaded, and the fours in double, so that the error does not grow with the row: one float
// sum a thread gave a constant row of 1.1 a mean off by 7e-4 at 2^24 columns, whose square
// stands beside eps.  A warp's threads are joined in double as well, its sum is rounded, and
// the warps are joined in float.
// (1600 x 40000 bf16: forward 123.7 us, with one float sum 120.1; backward 323 and 335.)
template <int kN, class F>
__device__ __forceinline__ void long_sums(int64_t cols, float (*red)[kWarps], float (&total)[kN], F&& terms) {
  double s[kN] = {};
  float last[4][kN] = {};
  auto add_last = [&] {
#pragma unroll
    for (int i = 0; i < kN; ++i) s[i] += static_cast<double>((last[0][i] + last[1][i]) + (last[2][i] + last[3][i]));
  };
  int64_t c = threadIdx.x;
  for (; c + 3 * kThreads < cols; c += 4 * kThreads) {
    float t[4][kN];
#pragma unroll
    for (int u = 0; u < 4; ++u) terms(c + u * kThreads, t[u]);
    add_last();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int i = 0; i < kN; ++i) last[u][i] = t[u][i];
    }
  }
  add_last();
  float rest[kN] = {};  // of three columns at most
  for (; c < cols; c += kThreads) {
    float t[kN];
    terms(c, t);
#pragma unroll
    for (int i = 0; i < kN; ++i) rest[i] += t[i];
  }
#pragma unroll
  for (int i = 0; i < kN; ++i) s[i] += static_cast<double>(rest[i]);
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    s[i] = warp_all_sum(s[i]);
    if ((threadIdx.x & 31) == 0) red[i][threadIdx.x >> 5] = static_cast<float>(s[i]);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    total[i] = red[i][0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) total[i] += red[i][w];
  }
}

// Rows of any length: one block per row, three reads of it (the second and third from L2).
template <class T>
__global__ void __launch_bounds__(kThreads)
    layer_norm_row_kernel(const T* __restrict__ x, int64_t x_stride, const float* __restrict__ weight,
                          const float* __restrict__ bias, T* __restrict__ y, int64_t y_stride,
                          float* __restrict__ mean, float* __restrict__ rstd, int64_t cols, float eps) {
  pdl_entry();
  __shared__ float red[2][kWarps];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * x_stride;
  T* yr = y + row * y_stride;
  float sum[1];
  long_sums(cols, red, sum, [&](int64_t c, float (&t)[1]) { t[0] = ld_val(xr + c); });
  const float mu = sum[0] / static_cast<float>(cols);
  long_sums(cols, red + 1, sum, [&](int64_t c, float (&t)[1]) {
    const float d = ld_val(xr + c) - mu;
    t[0] = d * d;
  });
  const float r = 1.0f / sqrtf(sum[0] / static_cast<float>(cols) + eps);
  if (threadIdx.x == 0) {
    if (mean) mean[row] = mu;
    if (rstd) rstd[row] = r;
  }
  for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
    float v = (ld_val(xr + c) - mu) * r;
    if (weight) v *= weight[c];
    if (bias) v += bias[c];
    st_val(yr + c, v);
  }
}

// One block per row: the two means, then dx.
template <class T>
__global__ void __launch_bounds__(kThreads)
    layer_norm_dx_kernel(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride,
                         const float* __restrict__ weight, const float* __restrict__ mean,
                         const float* __restrict__ rstd, T* __restrict__ dx, int64_t dx_stride, int64_t cols) {
  pdl_entry();
  __shared__ float red[2][kWarps];
  const int64_t row = blockIdx.x;
  const T* dyr = dy + row * dy_stride;
  const T* xr = x + row * x_stride;
  T* dxr = dx + row * dx_stride;
  const float mu = mean[row], r = rstd[row];
  float sums[2];
  long_sums(cols, red, sums, [&](int64_t c, float (&t)[2]) {
    t[0] = ld_val(dyr + c) * (weight ? weight[c] : 1.0f);
    t[1] = t[0] * ((ld_val(xr + c) - mu) * r);
  });
  const float c1 = sums[0] / static_cast<float>(cols), c2 = sums[1] / static_cast<float>(cols);
  for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
    const float g = ld_val(dyr + c) * (weight ? weight[c] : 1.0f);
    st_val(dxr + c, r * (g - c1 - (ld_val(xr + c) - mu) * r * c2));
  }
}

// Column sums of one slab of rows (blockIdx.y of gridDim.y), a thread per
// column, into part[slab][0 = dw, 1 = db][cols].
template <class T>
__global__ void __launch_bounds__(kThreads)
    layer_norm_columns_kernel(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride,
                              const float* __restrict__ mean, const float* __restrict__ rstd,
                              float* __restrict__ part, int64_t rows, int64_t cols) {
  pdl_entry();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= cols) return;
  const int64_t r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = r0; row < r1; ++row) {
    const float d = ld_val(dy + row * dy_stride + c);
    dw += d * ((ld_val(x + row * x_stride + c) - mean[row]) * rstd[row]);
    db += d;
  }
  part[(2 * static_cast<int64_t>(blockIdx.y)) * cols + c] = dw;
  part[(2 * static_cast<int64_t>(blockIdx.y) + 1) * cols + c] = db;
}

// dw and db from the slabs' partial sums [slabs][2 cols]; zeros for no slab.  A block
// folds 32 kPer columns: warp w adds slabs w, w + 32, ... in order, all of them in flight
// at once, then the warps' sums are added in a fixed tree.  kPer = 4, for wide rows:
// fewer blocks than fit at once (4096 x 16384 bf16, both kernels: 71.5 us with 1, 69.7 with 4).
constexpr int kFoldWarps = 32;
template <int kPer>
__global__ void __launch_bounds__(32 * kFoldWarps)
    layer_norm_fold_kernel(const float* __restrict__ part, int slabs, float* __restrict__ dweight,
                           float* __restrict__ dbias, int cols) {
  pdl_entry();
  __shared__ float red[kPer][kFoldWarps][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t width = 2 * static_cast<int64_t>(cols);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * 32 * kPer, c = first + lane * kPer;
  float s[kPer] = {};
  if (c < width) {
#pragma unroll
    for (int k = 0; k < (kStreamBlocks + kFoldWarps - 1) / kFoldWarps; ++k) {
      if (warp + k * kFoldWarps >= slabs) break;
      const float* p = part + (warp + k * kFoldWarps) * width + c;
      if constexpr (kPer == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        s[0] += v.x;
        s[1] += v.y;
        s[2] += v.z;
        s[3] += v.w;
      } else {
        s[0] += *p;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) red[j][warp][lane] = s[j];
  __syncthreads();
  // warp w sums up columns kPer w and on, a lane per warp's share
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const float sum = warp_all_sum(red[j][lane][warp]);
    const int64_t mine = first + warp * kPer + j;
    if (lane > 0 || mine >= width) continue;
    if (mine < cols) {
      if (dweight) dweight[mine] = sum;
    } else if (dbias) {
      dbias[mine - cols] = sum;
    }
  }
}

// Whether every row of these tensors is a whole number of 16-byte units from a
// 16-byte boundary on.
bool whole_units(std::initializer_list<const void*> tensors, std::initializer_list<int64_t> strides, int64_t rows,
                 int64_t cols, std::size_t elem) {
  const int64_t per = 16 / static_cast<int64_t>(elem);
  bool ok = cols % per == 0;
  for (const void* p : tensors) ok = ok && aligned(p, 16);
  for (int64_t st : strides) ok = ok && (rows <= 1 || st % per == 0);
  return ok;
}

// Rows up to which a launch is bound by one row's latency, not by bandwidth: a
// row is then spread over as many threads as it has units.
constexpr int64_t kFewRows = 4 * 148;

// Slabs of rows whose column sums are kept apart: the same on any GPU, as is the kernel that
// extents, strides and alignment choose, and so is every bit of dw and db.
int64_t column_slabs(int64_t rows) { return rows < kStreamBlocks ? rows : kStreamBlocks; }

// Calls f with the smallest of the unit counts kUnits, 2 kUnits .. kMax that holds n
// units over `threads` threads, and with whether they are filled.
template <int kMax, int kUnits = 1, class F>
void with_units(int64_t n, int64_t threads, F&& f) {
  if constexpr (kUnits < kMax) {
    if (n > kUnits * threads) return with_units<kMax, 2 * kUnits>(n, threads, f);
  }
  if (n == kUnits * threads) f(std::integral_constant<int, kUnits>{}, std::true_type{});
  else f(std::integral_constant<int, kUnits>{}, std::false_type{});
}
// Calls f with n, of 1 .. kMax.
template <int kMax, int kN = 1, class F>
void with_count(int64_t n, F&& f) {
  if constexpr (kN < kMax) {
    if (n > kN) return with_count<kMax, kN + 1>(n, f);
  }
  f(std::integral_constant<int, kN>{});
}

// Launches a persistent kernel of one block per SM, in clusters of kCluster: as many
// clusters as there are items, kStreamBlocks blocks at most.  Returns the clusters.
template <int kCluster, class A>
int64_t launch_stream(void (*kernel)(const A), const A& a, int64_t items, int threads, std::size_t smem, cudaStream_t s) {
  allow_shared_memory(reinterpret_cast<const void*>(kernel), smem);  // a launch that lacks it fails
  // 33 clusters of four fit a B200 (its 148 SMs come in groups that four does not
  // divide), 74 of two
  constexpr int64_t kMost = kCluster == 4 ? 32 : kStreamBlocks / kCluster;
  const int64_t clusters = items < kMost ? items : kMost;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * kCluster));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  if (kCluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = kCluster;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (pdl_enabled()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  cudaLaunchKernelEx(&cfg, kernel, a);  // errors are left for check_launch()
  return clusters;
}

// Calls f(warps, blocks) with the smallest group, of 1 .. 16 warps in each of 1, 2 or 4
// blocks, whose threads hold a row of `cols` <= kStreamCols at 16 elements each.
constexpr int64_t kStreamCols = 4 * 8192;
template <class F>
void with_group(int64_t cols, F&& f) {
  using std::integral_constant;
  const int64_t warps = (cols + 511) / 512;
  const integral_constant<int, 1> one;
  if (warps <= 1) f(one, one);
  else if (warps <= 2) f(integral_constant<int, 2>{}, one);
  else if (warps <= 3) f(integral_constant<int, 3>{}, one);
  else if (warps <= 4) f(integral_constant<int, 4>{}, one);
  else if (warps <= 6) f(integral_constant<int, 6>{}, one);
  else if (warps <= 8) f(integral_constant<int, 8>{}, one);
  else if (warps <= 12) f(integral_constant<int, 12>{}, one);
  else if (warps <= 16) f(integral_constant<int, 16>{}, one);
  else if (warps <= 24) f(integral_constant<int, 12>{}, integral_constant<int, 2>{});
  else if (warps <= 32) f(integral_constant<int, 16>{}, integral_constant<int, 2>{});
  else if (warps <= 48) f(integral_constant<int, 12>{}, integral_constant<int, 4>{});
  else f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
}

template <class T>
void launch_forward_stream(const ForwardArgs& a, cudaStream_t s) {
  using std::integral_constant;
  constexpr int kUnits = 16 / Unit<T>::kPer;
  with_group(a.cols, [&](auto warps, auto blocks) {
    constexpr int kW = decltype(warps)::value, kC = decltype(blocks)::value;
    const int64_t pairs = (a.rows + 1) / 2;
    if constexpr (kC > 1) {
      constexpr int kRows = sizeof(T) == 2 ? 2 : 1;
      auto over = [&](auto elems, auto w, auto c, auto stages) {
        constexpr int kElems = decltype(elems)::value, kWc = decltype(w)::value, kCc = decltype(c)::value;
        constexpr int kStages = decltype(stages)::value;
        using S = Stream<T, kElems / Unit<T>::kPer, kWc, 1, kStages, kRows>;
        launch_stream<kCc>(a.cols == 32 * kElems * kWc * kCc
                               ? layer_norm_cluster_kernel<T, kElems, kWc, kCc, kRows, kStages, true>
                               : layer_norm_cluster_kernel<T, kElems, kWc, kCc, kRows, kStages, false>,
                           a, kRows == 2 ? pairs : a.rows, S::kThreads, S::kSmem, s);
      };
      // 16384 .. 24576 columns: 24 elements to a thread of two blocks, not 16 of four, of which
      // fewer fit (1600 x 20000 bf16 26.7 us against 40.5, f32 42.5 against 52.9)
      if constexpr (kC == 4 && kW == 12)
        over(integral_constant<int, 24>{}, integral_constant<int, 16>{}, integral_constant<int, 2>{},
             integral_constant<int, 4>{});
      else
        over(integral_constant<int, 16>{}, warps, blocks, integral_constant<int, 5>{});
    } else if constexpr (sizeof(T) == 2) {
      constexpr int kGroups = kW == 1 ? 15 : 16 / kW, kStages = 3;
      using S = Stream<T, kUnits, kW, kGroups, kStages, 2>;
      launch_stream<1>(a.cols == 512 * kW ? layer_norm_stream_kernel<T, kW, kGroups, kStages, true>
                            : layer_norm_stream_kernel<T, kW, kGroups, kStages, false>,
                       a, pairs, S::kThreads, S::kSmem, s);
    }
  });
}

// Which kernel, with kernel times of both sides (us):
//   whole units, few rows   a row to 1, 4 or 16 warps, one unit to a thread where it fits:
//                           1000 x 1024 f32 2.5, streamed 3.1; of more than 2048 units
//                           streamed: 400 x 17408 bf16 10.2, a row to 16 warps 12.5
//   f32 up to 8192 columns  a row to 1, 2 or 4 warps: 16384 x 2048 42.3, streamed 47.9
//   bf16, and wider f32     streamed: 8192 x 4096 bf16 22.4, a row to a warp 37.5; over
//                           clusters: 4096 x 16384 bf16 43.6, a row to a block 99
//   the rest up to 16384    element by element: 8192 x 4097 bf16 46, three reads 94 (1600 x
//                           17409 with 1024 threads: bf16 54, f32 66, three reads 49, 76)
//   wider still             three reads
template <class T>
void launch_forward(const ForwardArgs& a, bool whole, cudaStream_t s) {
  using std::integral_constant;
  constexpr int kPer = Unit<T>::kPer;
  const unsigned rows = static_cast<unsigned>(a.rows);
  const bool few = a.rows <= kFewRows;
  const int64_t n = a.cols / kPer;  // units
  // a row's kW warps hold it at kMin to kMax units a thread
  auto row_kernel = [&](auto w, auto min, auto max) {
    constexpr int kW = decltype(w)::value;
    with_units<decltype(max)::value, decltype(min)::value>(n, 32 * kW, [&](auto units, auto full) {
      launch_async(layer_norm_kernel<T, decltype(units)::value, kW, decltype(full)::value>,
                   kW == 1 ? (rows + kWarps - 1) / kWarps : rows, kW == 1 ? kThreads : 32 * kW, 0, s, a);
    });
  };
  auto elements = [&](auto thr, auto max) {
    constexpr int kThr = decltype(thr)::value;
    with_count<decltype(max)::value>((a.cols + 2 * kThr - 1) / (2 * kThr), [&](auto pairs) {
      launch_async(layer_norm_elements_kernel<T, decltype(pairs)::value, kThr>, rows, kThr, 0, s, a);
    });
  };
  if (!whole && a.cols <= (few ? 512 : 4096)) {
    elements(integral_constant<int, 128>{}, integral_constant<int, 16>{});
  } else if (!whole && a.cols <= 16384) {
    elements(integral_constant<int, 512>{}, integral_constant<int, 16>{});
  } else if (whole && few && n <= 32) {
    row_kernel(integral_constant<int, 1>{}, integral_constant<int, 1>{}, integral_constant<int, 1>{});
  } else if (whole && few && n <= 128) {
    row_kernel(integral_constant<int, 4>{}, integral_constant<int, 1>{}, integral_constant<int, 1>{});
  } else if (whole && ((!few && sizeof(T) == 2) || n > 2048) && a.cols <= kStreamCols) {
    launch_forward_stream<T>(a, s);
  } else if (whole && sizeof(T) == 4 && !few && n <= 512) {
    if constexpr (sizeof(T) == 4)
      row_kernel(integral_constant<int, 1>{}, integral_constant<int, 1>{}, integral_constant<int, 16>{});
  } else if (whole && sizeof(T) == 4 && !few && n <= 1024) {
    if constexpr (sizeof(T) == 4)
      row_kernel(integral_constant<int, 2>{}, integral_constant<int, 16>{}, integral_constant<int, 16>{});
  } else if (whole && sizeof(T) == 4 && !few && n <= 2048) {
    if constexpr (sizeof(T) == 4)
      row_kernel(integral_constant<int, 4>{}, integral_constant<int, 16>{}, integral_constant<int, 16>{});
  } else if (whole && n <= 2048) {
    row_kernel(integral_constant<int, 16>{}, integral_constant<int, 1>{}, integral_constant<int, 4>{});
  } else {
    launch_async(layer_norm_row_kernel<T>, rows, kThreads, 0, s, static_cast<const T*>(a.x), a.x_stride, a.weight,
                 a.bias, static_cast<T*>(a.y), a.y_stride, a.mean, a.rstd, static_cast<int64_t>(a.cols), a.eps);
  }
}

// Returns the number of slabs of partial sums that were written.
template <class T>
int64_t launch_backward_stream(const BackwardArgs& a, cudaStream_t s) {
  // two bf16 rows a turn halve what a turn costs besides their elements; two f32 rows
  // would not leave the ring three stages
  constexpr int kRows = sizeof(T) == 2 ? 2 : 1, kStages = 3;
  int64_t slabs = 0;
  with_group(a.cols, [&](auto warps, auto blocks) {
    constexpr int kW = decltype(warps)::value, kC = decltype(blocks)::value;
    constexpr int kGroups = kW == 1 ? 15 : 16 / kW;
    using S = Stream<T, 16 / Unit<T>::kPer, kW, kGroups, kStages, 2 * kRows>;
    const int64_t items = (a.rows + kRows - 1) / kRows;
    if (a.cols == 512 * kW * kC)
      slabs = launch_stream<kC>(layer_norm_backward_kernel<T, kW, kGroups, kC, kRows, kStages, true>, a, items,
                                S::kThreads, S::kSmem, s);
    else
      slabs = launch_stream<kC>(layer_norm_backward_kernel<T, kW, kGroups, kC, kRows, kStages, false>, a, items,
                                S::kThreads, S::kSmem, s);
  });
  return slabs;
}

template <class T>
void launch_backward(const BackwardArgs& a, bool whole, float* dweight, float* dbias, cudaStream_t s) {
  const T* dy = static_cast<const T*>(a.dy);
  const T* x = static_cast<const T*>(a.x);
  int64_t slabs = 0;
  if (a.rows > 0 && whole && a.cols <= kStreamCols) {
    slabs = launch_backward_stream<T>(a, s);
  } else if (a.rows > 0 && a.cols <= kStreamCols) {
    with_group(a.cols, [&](auto warps, auto blocks) {
      constexpr int kW = decltype(warps)::value, kC = decltype(blocks)::value;
      constexpr int kGroups = kC > 1 ? 1 : kW == 1 ? 15 : 16 / kW;
      // the ring, or at the end the groups' sums
      constexpr std::size_t kRing = 3 * 2 * 16 * 32 * kW * kGroups * sizeof(T);
      constexpr std::size_t kSums = static_cast<std::size_t>(kGroups - 1) * 32 * 32 * kW * sizeof(float);
      slabs = launch_stream<kC>(layer_norm_backward_elements_kernel<T, kW, kGroups, kC>, a, a.rows, 32 * kW * kGroups,
                                kRing > kSums ? kRing : kSums, s);
    });
  } else if (a.rows > 0) {
    launch_async(layer_norm_dx_kernel<T>, static_cast<unsigned>(a.rows), kThreads, 0, s, dy, a.dy_stride, x, a.x_stride,
                 a.weight, a.mean, a.rstd, static_cast<T*>(a.dx), a.dx_stride, static_cast<int64_t>(a.cols));
    if (a.part) {
      slabs = column_slabs(a.rows);
      launch_async(layer_norm_columns_kernel<T>,
                   dim3(static_cast<unsigned>((a.cols + kThreads - 1) / kThreads), static_cast<unsigned>(slabs)),
                   kThreads, 0, s, dy, a.dy_stride, x, a.x_stride, a.mean, a.rstd, a.part, static_cast<int64_t>(a.rows),
                   static_cast<int64_t>(a.cols));
    }
  }
  if (!dweight && !dbias) return;
  const int64_t width = 2 * static_cast<int64_t>(a.cols);
  if (a.cols >= 8192 && width % 4 == 0)
    launch_async(layer_norm_fold_kernel<4>, static_cast<unsigned>((width + 127) / 128), 32 * kFoldWarps, 0, s,
                 static_cast<const float*>(a.part), static_cast<int>(slabs), dweight, dbias, a.cols);
  else
    launch_async(layer_norm_fold_kernel<1>, static_cast<unsigned>((width + 31) / 32), 32 * kFoldWarps, 0, s,
                 static_cast<const float*>(a.part), static_cast<int>(slabs), dweight, dbias, a.cols);
}

}  // namespace
}  // namespace mcke_sm100

namespace mcke_sm100 {
bool allow_shared_memory(const void* kernel, std::size_t bytes) {
  static std::mutex mu;
  static std::map<std::pair<const void*, int>, std::size_t> done;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  std::lock_guard<std::mutex> lk(mu);
  try {
    std::size_t& most = done[{kernel, dev}];
    if (bytes <= most) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) != cudaSuccess)
      return false;
    most = bytes;
    return true;
  } catch (const std::bad_alloc&) {  // no room to remember it
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) ==
           cudaSuccess;
  }
}

// Reads and clears the word that an expired wait of either pass sets.
int read_layer_norm_watchdog(uint32_t* site) {
  uint32_t v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_layer_norm_watchdog, sizeof(v));
  if (e != cudaSuccess) return fail(MCKE_CUDA_ERROR, "watchdog read: %s", cudaGetErrorString(e));
  if (v != 0) {
    const uint32_t zero = 0;
    e = cudaMemcpyToSymbol(g_layer_norm_watchdog, &zero, sizeof(zero));
    if (e != cudaSuccess) return fail(MCKE_CUDA_ERROR, "watchdog clear: %s", cudaGetErrorString(e));
  }
  *site = v;
  return MCKE_OK;
}
}  // namespace mcke_sm100

using namespace mcke_sm100;

extern "C" int mcke_sm100_layer_norm_watchdog_selftest(mcke_stream_t stream) {
  clear_error();
  launch_async(layer_norm_selftest_kernel, 1, 64, 0, reinterpret_cast<cudaStream_t>(stream));
  return check_launch("mcke_sm100_layer_norm_watchdog_selftest");
}

extern "C" int mcke_sm100_layer_norm(const void* x, int64_t x_stride, const float* weight, const float* bias, void* y,
                                     int64_t y_stride, float* mean, float* rstd, int64_t rows, int64_t cols, float eps,
                                     int dtype, mcke_stream_t stream) {
  static const char* who = "mcke_sm100_layer_norm";
  clear_error();
  MCKE_RETURN_IF(check_dtype(who, dtype));
  if (rows < 0 || cols < 0) return fail(MCKE_INVALID_ARGUMENT, "%s: negative extent", who);
  if (!(eps >= 0.0f) || std::isinf(eps)) return fail(MCKE_INVALID_ARGUMENT, "%s: eps must be finite and >= 0", who);
  if (rows > 0 && cols == 0 && (mean || rstd))
    return fail(MCKE_INVALID_ARGUMENT, "%s: rows of no columns have no statistics", who);
  if (rows == 0 || cols == 0) return MCKE_OK;
  if (!x || !y) return fail(MCKE_INVALID_ARGUMENT, "%s: null pointer", who);
  if (rows > kMaxRows || cols > 2147483647LL)
    return fail(MCKE_INVALID_ARGUMENT, "%s: extent exceeds INT32_MAX (rows: 65536 less)", who);
  MCKE_RETURN_IF(check_stride(who, "x", x_stride, rows, cols, false));
  MCKE_RETURN_IF(check_stride(who, "y", y_stride, rows, cols, true));
  const std::size_t e = dtype_bytes(dtype);
  MCKE_RETURN_IF(check_aligned(
      who, {{"x", x, e}, {"y", y, e}, {"weight", weight, 4}, {"bias", bias, 4}, {"mean", mean, 4}, {"rstd", rstd, 4}}));
  const RowSpan outs[] = {span_of("y", y, rows, cols, y_stride, e), span_of("mean", mean, rows * 4),
                          span_of("rstd", rstd, rows * 4)};
  const RowSpan ins[] = {span_of("x", x, rows, cols, x_stride, e), span_of("weight", weight, cols * 4),
                         span_of("bias", bias, cols * 4)};
  MCKE_RETURN_IF(check_overlaps(who, outs, ins));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const ForwardArgs a = {x, x_stride, weight, bias, y, y_stride, mean, rstd, static_cast<int>(rows),
                         static_cast<int>(cols), eps};
  const bool whole = whole_units({x, y}, {x_stride, y_stride}, rows, cols, e) && aligned(weight, 16) && aligned(bias, 16);
  if (dtype == MCKE_DTYPE_BF16) launch_forward<uint16_t>(a, whole, s);
  else launch_forward<float>(a, whole, s);
  return check_launch(who);
}

extern "C" size_t mcke_sm100_layer_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return static_cast<size_t>(column_slabs(rows)) * 2 * static_cast<size_t>(cols) * sizeof(float);
}

extern "C" int mcke_sm100_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride,
                                              const float* weight, const float* mean, const float* rstd, void* dx,
                                              int64_t dx_stride, float* dweight, float* dbias, int64_t rows,
                                              int64_t cols, int dtype, void* workspace, size_t workspace_bytes,
                                              mcke_stream_t stream) {
  static const char* who = "mcke_sm100_layer_norm_backward";
  clear_error();
  MCKE_RETURN_IF(check_dtype(who, dtype));
  if (rows < 0 || cols < 0) return fail(MCKE_INVALID_ARGUMENT, "%s: negative extent", who);
  if (cols == 0) return MCKE_OK;
  if (rows > kMaxRows || cols > 2147483647LL)
    return fail(MCKE_INVALID_ARGUMENT, "%s: extent exceeds INT32_MAX (rows: 65536 less)", who);
  if (rows > 0 && (!dy || !x || !mean || !rstd || !dx)) return fail(MCKE_INVALID_ARGUMENT, "%s: null pointer", who);
  MCKE_RETURN_IF(check_stride(who, "dy", dy_stride, rows, cols, false));
  MCKE_RETURN_IF(check_stride(who, "x", x_stride, rows, cols, false));
  MCKE_RETURN_IF(check_stride(who, "dx", dx_stride, rows, cols, true));
  const std::size_t e = dtype_bytes(dtype);
  MCKE_RETURN_IF(check_aligned(who, {{"dy", dy, e}, {"x", x, e}, {"dx", dx, e}, {"weight", weight, 4}, {"mean", mean, 4},
                                     {"rstd", rstd, 4}, {"dweight", dweight, 4}, {"dbias", dbias, 4}}));
  const bool params = dweight || dbias;
  const size_t need = params ? mcke_sm100_layer_norm_backward_workspace_bytes(rows, cols) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(MCKE_INVALID_ARGUMENT,
                "%s: needs %zu bytes of 16-byte aligned workspace (got %zu); query "
                "mcke_sm100_layer_norm_backward_workspace_bytes() first",
                who, need, workspace ? workspace_bytes : static_cast<size_t>(0));
  const RowSpan outs[] = {span_of("dx", dx, rows, cols, dx_stride, e), span_of("dweight", dweight, cols * 4),
                          span_of("dbias", dbias, cols * 4),
                          span_of("workspace", workspace, static_cast<int64_t>(need))};
  const RowSpan ins[] = {span_of("dy", dy, rows, cols, dy_stride, e), span_of("x", x, rows, cols, x_stride, e),
                         span_of("weight", weight, cols * 4), span_of("mean", mean, rows * 4),
                         span_of("rstd", rstd, rows * 4)};
  MCKE_RETURN_IF(check_overlaps(who, outs, ins));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const BackwardArgs a = {dy, dy_stride, x, x_stride, weight, mean, rstd, dx, dx_stride,
                          params ? static_cast<float*>(workspace) : nullptr, static_cast<int>(rows),
                          static_cast<int>(cols)};
  const bool whole = whole_units({dy, x, dx}, {dy_stride, x_stride, dx_stride}, rows, cols, e) && aligned(weight, 16);
  if (dtype == MCKE_DTYPE_BF16) launch_backward<uint16_t>(a, whole, dweight, dbias, s);
  else launch_backward<float>(a, whole, dweight, dbias, s);
  return check_launch(who);
}
