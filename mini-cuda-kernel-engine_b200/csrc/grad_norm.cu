// grad_norm.cu -- the global L2 norm of a list of tensors, and clipping by it.
//
//   n = sqrt(sum over tensors and elements of x^2),
//   c = min(1, max_norm / (n + 1e-6)),   out = c x.
//
// The list's table (pointers, lengths, types) travels in the launch's
// parameters, so a call copies nothing to the device and a captured CUDA graph
// holds all it needs.  Every tensor is cut into chunks of 2048 16-byte vectors
// (counted from the 16-byte boundary at or below its first element, so a tensor
// may start anywhere), the chunks of all tensors are numbered through, and the
// blocks take them in turn: short tensors cost no launch and no block of their own,
// and the blocks move through memory side by side.
//
// Squares are added in double: the sum neither loses small gradients next to
// large ones nor leaves float's range where the norm itself does not.  The
// blocks' sums go to the workspace and are folded in block order, of a short list by
// every block of the scaling kernel (one launch less: ten tensors of up to 1000 floats
// 5.0 us against 5.8), of one that fills the grid, more than 14 MB, by a kernel of one block
// (f32 that needs no clipping: 18 MB 8.8 us against 8.6, 43 MB 12.8 against 13.0, 103 MB 23.3
// against 25.3; clipped the two are within 1%).  The grid follows from the tensors alone
// (lengths, types, where they start), so the norm has the same bits on any GPU.
//
// Bound by HBM: beyond what L2 keeps the tensors are read twice and written once.
// 1.04 GB of bf16 in 60 tensors: the norm 173 us (6.0 TB/s, 0.92 of the copy rate), clipping
// 306 us (6.8 TB/s: what the norm read last is still in L2).
#include <algorithm>
#include <new>
#include <vector>

#include "row_ops.cuh"

namespace mcke_sm100 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kChunkVecs = 2048;  // 32 KB
constexpr int kUnroll = kChunkVecs / kThreads;
// Blocks of the two passes at most.  The squares: what is resident at once, three to
// an SM with two chunks each in flight (1.04 GB of bf16: 173 us, 191 us with five blocks of
// 16 KB chunks, 227 us with six, which are more than fit).  Scaling: many short blocks,
// so that none of a few long ones is the last (the same list: 306 us, 333 us with
// six to an SM that stay).
constexpr int64_t kMaxBlocks = 3 * 148;
constexpr int64_t kClipBlocks = 64 * 148;
constexpr float kNormEps = 1e-6f;

struct Entry {
  const char* data;
  char* out;
  int64_t numel;
  uint32_t first_chunk;
  uint16_t bf16, out_bf16;
};
constexpr int kMaxEntries = 1000;  // 32,000 bytes of the 32,764 that a launch's parameters hold
// Capacities of the parameter table, 64 and kMaxEntries; a launch takes the smaller if it
// fits (60 tensors of up to 100,000 floats: 5.0 us against 5.4 with the larger).
template <int kCap>
struct Table {
  Entry e[kCap];
  uint32_t chunks;
  int count;
};

// Where the launch's coefficient comes from: the blocks' sums of squares
// (count of them), or a norm that the caller has.
struct NormSource {
  const double* sums;
  int count;
  const float* given;
  float* norm;  // written by block 0, may be null
  float max_norm;
};

// The tensor that holds chunk c: tensor i if it is still that one, else by bisection.
template <int kCap>
__device__ __forceinline__ int find_entry(const Table<kCap>& t, uint32_t c, int i) {
  const uint32_t end = i + 1 < t.count ? t.e[i + 1].first_chunk : t.chunks;
  if (c >= t.e[i].first_chunk && c < end) return i;
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first_chunk <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// 16-byte vectors of a tensor are counted from the boundary at or below its first
// element, which is element -shift of that count.
template <class T>
struct Vec {
  static constexpr int kPer = 16 / sizeof(T);
  static __device__ __forceinline__ int shift(const char* data) {
    return static_cast<int>((reinterpret_cast<uintptr_t>(data) & 15) / sizeof(T));
  }
};

// Plain loads: in place, another element of the tensor may be written by this grid.
__device__ __forceinline__ uint4 ld_u4(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
// The vector that starts at element `first`; zeros where the tensor has no element.
template <class T>
__device__ __forceinline__ uint4 ld_part(const T* data, int64_t first, int64_t numel) {
  constexpr int kPer = Vec<T>::kPer, kPerWord = kPer / 4;
  if (first >= 0 && first + kPer <= numel) return ld_u4(data + first);
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (first + j < 0 || first + j >= numel) continue;
    if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(data[first + j]);
    else w[j / kPerWord] |= static_cast<uint32_t>(data[first + j]) << (16 * (j % kPerWord));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// This thread's kUnroll vectors of a chunk.
template <class T>
__device__ __forceinline__ void ld_chunk(const Entry& e, uint32_t c, uint4 (&q)[kUnroll]) {
  constexpr int kPer = Vec<T>::kPer;
  const T* data = reinterpret_cast<const T*>(e.data);
  const int64_t first = (static_cast<int64_t>(c - e.first_chunk) * kChunkVecs + threadIdx.x) * kPer - Vec<T>::shift(e.data);
  if (first >= 0 && first + ((kUnroll - 1) * kThreads + 1) * kPer <= e.numel) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) q[u] = ld_u4(data + first + u * kThreads * kPer);
  } else {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) q[u] = ld_part(data, first + u * kThreads * kPer, e.numel);
  }
}

// x 2^-896 as a double, from the bits of |x| moved to a double's places: exact for every
// finite float, and without the conversion unit, which the bf16 stream would keep 63%
// busy at three quarters of the copy rate.  An infinity or a NaN becomes a
// finite value of 2^-768 and up.
__device__ __forceinline__ double scaled_abs(uint32_t bits) {
  return __hiloint2double(static_cast<int>((bits & 0x7fffffffu) >> 3), static_cast<int>(bits << 29));
}
constexpr double kUnscale = 0x1p896;
__device__ __forceinline__ double add_square(uint32_t bits, double s) {
  const double x = scaled_abs(bits) * kUnscale;
  return fma(x, x, s);
}
__device__ __forceinline__ double add_squares(const uint4 (&q)[kUnroll], bool bf16, double s) {
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t w[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (bf16) s = add_square(w[j] << 16, s);
      s = add_square(bf16 ? w[j] & 0xffff0000u : w[j], s);
    }
  }
  return s;
}
__device__ __forceinline__ bool any_nan(const uint4 (&q)[kUnroll], bool bf16) {
  bool nan = false;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t w[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float hi = __uint_as_float(bf16 ? w[j] & 0xffff0000u : w[j]), lo = __uint_as_float(bf16 ? w[j] << 16 : 0u);
      nan = nan || hi != hi || lo != lo;
    }
  }
  return nan;
}

// The squares of a block's chunks, the next chunk's loads in flight while one is added
// up.  A sum of 2^256 and more may have had a NaN or an infinity for a finite value:
// the norm is then infinite in float, unless the block, looking again, finds a NaN.
template <int kCap>
__global__ void __launch_bounds__(kThreads)
    grad_squares_kernel(const __grid_constant__ Table<kCap> t, double* __restrict__ sums) {
  pdl_entry();
  __shared__ double red[kWarps];
  int i = 0;
  auto load = [&](uint32_t c, uint4 (&q)[kUnroll]) {
    i = find_entry(t, c, i);
    const Entry& e = t.e[i];
    if (e.bf16) ld_chunk<uint16_t>(e, c, q);
    else ld_chunk<float>(e, c, q);
    return e.bf16 != 0;
  };
  double s = 0.0;
  if (blockIdx.x < t.chunks) {
    uint4 q[kUnroll], next[kUnroll];
    bool bf16 = load(blockIdx.x, q);
    for (uint32_t c = blockIdx.x;;) {
      c += gridDim.x;
      bool next_bf16 = false;
      if (c < t.chunks) next_bf16 = load(c, next);
      s = bf16 ? add_squares(q, true, s) : add_squares(q, false, s);
      if (c >= t.chunks) break;
      bf16 = next_bf16;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) q[u] = next[u];
    }
  }
  s = block_all_sum<kWarps>(s, red);
  if (s >= 0x1p256) {
    bool nan = false;
    for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
      uint4 q[kUnroll];
      const bool bf16 = load(c, q);
      nan = nan || any_nan(q, bf16);
    }
    s = __syncthreads_or(nan) ? static_cast<double>(NAN) : static_cast<double>(INFINITY);
  }
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// The norm from the blocks' sums, the same bits in every thread and block.
__device__ __forceinline__ float fold_norm(const double* sums, int count, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += kThreads) s += sums[i];
  return static_cast<float>(sqrt(block_all_sum<kWarps>(s, red)));
}

__global__ void __launch_bounds__(kThreads) grad_norm_fold_kernel(const double* __restrict__ sums, int count,
                                                                  float* __restrict__ norm) {
  pdl_entry();
  __shared__ double red[kWarps];
  const float n = fold_norm(sums, count, red);
  if (threadIdx.x == 0) *norm = n;
}

__device__ __forceinline__ void store_vec(float* out, int64_t first, int64_t numel, const float* v, int per,
                                          bool whole) {
  if (whole && first >= 0 && first + per <= numel) {
    for (int j = 0; j < per; j += 4)
      *reinterpret_cast<float4*>(out + first + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    return;
  }
  for (int j = 0; j < per; ++j)
    if (first + j >= 0 && first + j < numel) out[first + j] = v[j];
}
__device__ __forceinline__ void store_vec(uint16_t* out, int64_t first, int64_t numel, const float* v, int per,
                                          bool whole) {
  if (whole && first >= 0 && first + per <= numel) {
    *reinterpret_cast<uint4*>(out + first) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                                        pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    return;
  }
  for (int j = 0; j < per; ++j)
    if (first + j >= 0 && first + j < numel) out[first + j] = to_bf16(v[j]);
}

// out = coef * data over one chunk.  Vectors start on 16-byte boundaries of
// `data`; those of `out` are whole where it has the same offset to a boundary.
template <class T, class U>
__device__ __forceinline__ void chunk_scale(const Entry& e, uint32_t c, float coef) {
  constexpr int kPer = Vec<T>::kPer;
  U* out = reinterpret_cast<U*>(e.out);
  const int shift = Vec<T>::shift(e.data);
  const int64_t first = (static_cast<int64_t>(c - e.first_chunk) * kChunkVecs + threadIdx.x) * kPer - shift;
  const bool whole = ((reinterpret_cast<uintptr_t>(e.out) - shift * sizeof(U)) & 15) == 0;
  uint4 q[kUnroll];
  ld_chunk<T>(e, c, q);
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t w[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
    float v[kPer];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        v[j] = coef * __uint_as_float(w[j]);
      } else {
        v[2 * j] = coef * bf16_lo(w[j]);
        v[2 * j + 1] = coef * bf16_hi(w[j]);
      }
    }
    store_vec(out, first + u * kThreads * kPer, e.numel, v, kPer, whole);
  }
}

template <int kCap>
__global__ void __launch_bounds__(kThreads)
    grad_clip_kernel(const __grid_constant__ Table<kCap> t, NormSource src) {
  pdl_entry();
  __shared__ double red[kWarps];
  const float n = src.given ? *src.given : fold_norm(src.sums, src.count, red);
  if (src.norm && blockIdx.x == 0 && threadIdx.x == 0) *src.norm = n;
  // a NaN norm stays NaN (fminf would return 1)
  const float ratio = src.max_norm / (n + kNormEps);
  const float coef = ratio > 1.0f ? 1.0f : ratio;
  // the last chunks first: the norm's pass has left them in L2
  int i = 0;
  for (uint32_t n = blockIdx.x; n < t.chunks; n += gridDim.x) {
    const uint32_t c = t.chunks - 1 - n;
    i = find_entry(t, c, i);
    const Entry& e = t.e[i];
    if (coef == 1.0f && e.out == e.data) continue;  // 1 x is x: nothing to write
    if (!e.bf16) chunk_scale<float, float>(e, c, coef);
    else if (e.out_bf16) chunk_scale<uint16_t, uint16_t>(e, c, coef);
    else chunk_scale<uint16_t, float>(e, c, coef);
  }
}

// ---- host -------------------------------------------------------------------------

int64_t chunks_of(const mcke_grad& g) {
  const int64_t size = static_cast<int64_t>(dtype_bytes(g.dtype));
  const int64_t shift = static_cast<int64_t>(reinterpret_cast<std::uintptr_t>(g.data) & 15) / size;
  const int64_t per = 16 / size;
  const int64_t vecs = (g.numel + shift + per - 1) / per;
  return (vecs + kChunkVecs - 1) / kChunkVecs;
}

int64_t blocks_of(int64_t chunks, int64_t most) { return chunks < 1 ? 1 : chunks < most ? chunks : most; }

// One launch's share of the list: grads [begin, end), tensors of no element left out.
template <int kCap>
void fill(Table<kCap>& t, const mcke_grad* g, int begin, int end) {
  int64_t at = 0;
  t.count = 0;
  for (int i = begin; i < end; ++i) {
    if (g[i].numel == 0) continue;
    t.e[t.count++] = Entry{static_cast<const char*>(g[i].data), static_cast<char*>(g[i].out), g[i].numel,
                           static_cast<uint32_t>(at), static_cast<uint16_t>(g[i].dtype == MCKE_DTYPE_BF16),
                           static_cast<uint16_t>(g[i].out_dtype == MCKE_DTYPE_BF16)};
    at += chunks_of(g[i]);
  }
  t.chunks = static_cast<uint32_t>(at);
}

template <int kCap>
int64_t launch_squares(const mcke_grad* g, int begin, int end, double* sums, cudaStream_t s) {
  Table<kCap> t;
  fill(t, g, begin, end);
  const int64_t blocks = blocks_of(t.chunks, kMaxBlocks);
  launch_async(grad_squares_kernel<kCap>, static_cast<unsigned>(blocks), kThreads, 0, s, t, sums);
  return blocks;
}
template <int kCap>
void launch_clip(const mcke_grad* g, int begin, int end, const NormSource& src, cudaStream_t s) {
  Table<kCap> t;
  fill(t, g, begin, end);
  launch_async(grad_clip_kernel<kCap>, static_cast<unsigned>(blocks_of(t.chunks, kClipBlocks)), kThreads, 0, s, t, src);
}

// Sums of squares of the whole list; returns how many sums were written.
int all_squares(const mcke_grad* g, int count, double* sums, cudaStream_t s) {
  int64_t at = 0;
  for (int b = 0; b < count; b += kMaxEntries) {
    const int e = std::min(count, b + kMaxEntries);
    if (e - b <= 64) at += launch_squares<64>(g, b, e, sums + at, s);
    else at += launch_squares<kMaxEntries>(g, b, e, sums + at, s);
  }
  return static_cast<int>(at);
}
void all_clip(const mcke_grad* g, int count, NormSource src, cudaStream_t s) {
  for (int b = 0; b == 0 || b < count; b += kMaxEntries) {
    const int e = std::min(count, b + kMaxEntries);
    if (e - b <= 64) launch_clip<64>(g, b, e, src, s);
    else launch_clip<kMaxEntries>(g, b, e, src, s);
    src.norm = nullptr;
  }
}

size_t workspace_bytes_of(int count) {
  const size_t launches = count <= 0 ? 1 : (static_cast<size_t>(count) + kMaxEntries - 1) / kMaxEntries;
  return launches * kMaxBlocks * sizeof(double);
}

struct Interval {
  std::uintptr_t begin, end;
  int index;  // of the tensor, or -1 (norm), -2 (workspace)
  bool out;
};
const char* what(const Interval& v) { return v.index == -1 ? "norm" : v.index == -2 ? "workspace" : "tensor"; }

// Checks the list.  Outputs share no byte with one another nor with another
// tensor's data; data may be listed twice where nothing is written.
int check_list(const char* who, const mcke_grad* g, int count, bool writes, const void* norm, bool norm_out,
               const void* ws, size_t ws_bytes) {
  if (count < 0) return fail(MCKE_INVALID_ARGUMENT, "%s: negative count", who);
  if (count > 0 && !g) return fail(MCKE_INVALID_ARGUMENT, "%s: null list", who);
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    if (g[i].numel < 0) return fail(MCKE_INVALID_ARGUMENT, "%s: tensor %d has a negative extent", who, i);
    MCKE_RETURN_IF(check_dtype(who, g[i].dtype));
    if (writes) MCKE_RETURN_IF(check_dtype(who, g[i].out_dtype));
    if (writes && g[i].out_dtype != g[i].dtype && g[i].out_dtype != MCKE_DTYPE_F32)
      return fail(MCKE_INVALID_ARGUMENT, "%s: tensor %d: an f32 gradient is not clipped into bf16", who, i);
    if (g[i].numel == 0) continue;
    if (g[i].numel > (int64_t{1} << 40)) return fail(MCKE_INVALID_ARGUMENT, "%s: tensor %d is too large", who, i);
    if (!g[i].data || (writes && !g[i].out)) return fail(MCKE_INVALID_ARGUMENT, "%s: tensor %d: null pointer", who, i);
    if (!aligned(g[i].data, dtype_bytes(g[i].dtype)) || (writes && !aligned(g[i].out, dtype_bytes(g[i].out_dtype))))
      return fail(MCKE_INVALID_ARGUMENT, "%s: tensor %d is not element-aligned", who, i);
    chunks += chunks_of(g[i]);
    if (chunks > 2147483647LL) return fail(MCKE_INVALID_ARGUMENT, "%s: the list holds too many elements", who);
  }
  if (!aligned(norm, 4)) return fail(MCKE_INVALID_ARGUMENT, "%s: norm is not element-aligned", who);
  try {
    std::vector<Interval> v;
    v.reserve(2 * static_cast<size_t>(count) + 2);
    auto add = [&](const void* p, int64_t bytes, int index, bool out) {
      const auto b = reinterpret_cast<std::uintptr_t>(p);
      if (p && bytes > 0) v.push_back(Interval{b, b + static_cast<std::uintptr_t>(bytes), index, out});
    };
    for (int i = 0; i < count; ++i) {
      const int64_t bytes = g[i].numel * static_cast<int64_t>(dtype_bytes(g[i].dtype));
      const bool in_place = writes && g[i].out == g[i].data && g[i].out_dtype == g[i].dtype;
      if (!in_place) add(g[i].data, bytes, i, false);
      if (writes) add(g[i].out, g[i].numel * static_cast<int64_t>(dtype_bytes(g[i].out_dtype)), i, true);
    }
    add(norm, 4, -1, norm_out);
    add(ws, static_cast<int64_t>(ws_bytes), -2, true);
    std::sort(v.begin(), v.end(), [](const Interval& a, const Interval& b) { return a.begin < b.begin; });
    // in order of begin: the furthest end so far, of all intervals and of the outputs
    const Interval* any = nullptr;
    const Interval* out = nullptr;
    for (const Interval& x : v) {
      const Interval* hit = x.out ? (any && any->end > x.begin ? any : nullptr)
                                  : (out && out->end > x.begin ? out : nullptr);
      if (hit)
        return fail(MCKE_INVALID_ARGUMENT, "%s: %s %d overlaps %s %d, one of them an output", who, what(x), x.index,
                    what(*hit), hit->index);
      if (!any || x.end > any->end) any = &x;
      if (x.out && (!out || x.end > out->end)) out = &x;
    }
  } catch (const std::bad_alloc&) {
    return fail(MCKE_OUT_OF_MEMORY, "%s: no host memory for the list's check", who);
  }
  return MCKE_OK;
}

int check_workspace(const char* who, int count, const void* workspace, size_t workspace_bytes) {
  const size_t need = workspace_bytes_of(count);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
    return fail(MCKE_INVALID_ARGUMENT,
                "%s: needs %zu bytes of 16-byte aligned workspace (got %zu); query "
                "mcke_sm100_grad_norm_workspace_bytes() first",
                who, need, workspace ? workspace_bytes : static_cast<size_t>(0));
  return MCKE_OK;
}

int check_max_norm(const char* who, float max_norm) {
  if (!(max_norm >= 0.0f) || std::isinf(max_norm))
    return fail(MCKE_INVALID_ARGUMENT, "%s: max_norm must be finite and >= 0", who);
  return MCKE_OK;
}

}  // namespace
}  // namespace mcke_sm100

using namespace mcke_sm100;

extern "C" size_t mcke_sm100_grad_norm_workspace_bytes(int count) { return workspace_bytes_of(count); }

extern "C" int mcke_sm100_grad_norm(const mcke_grad* grads, int count, float* norm, void* workspace,
                                    size_t workspace_bytes, mcke_stream_t stream) {
  static const char* who = "mcke_sm100_grad_norm";
  clear_error();
  if (!norm) return fail(MCKE_INVALID_ARGUMENT, "%s: null norm", who);
  MCKE_RETURN_IF(check_workspace(who, count, workspace, workspace_bytes));
  MCKE_RETURN_IF(check_list(who, grads, count, false, norm, true, workspace, workspace_bytes_of(count)));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  double* sums = static_cast<double*>(workspace);
  const int n = all_squares(grads, count, sums, s);
  launch_async(grad_norm_fold_kernel, 1, kThreads, 0, s, static_cast<const double*>(sums), n, norm);
  return check_launch(who);
}

extern "C" int mcke_sm100_clip_grads(const mcke_grad* grads, int count, float max_norm, const float* norm,
                                     mcke_stream_t stream) {
  static const char* who = "mcke_sm100_clip_grads";
  clear_error();
  if (!norm) return fail(MCKE_INVALID_ARGUMENT, "%s: null norm", who);
  MCKE_RETURN_IF(check_max_norm(who, max_norm));
  MCKE_RETURN_IF(check_list(who, grads, count, true, norm, false, nullptr, 0));
  if (count == 0) return MCKE_OK;
  all_clip(grads, count, NormSource{nullptr, 0, norm, nullptr, max_norm}, reinterpret_cast<cudaStream_t>(stream));
  return check_launch(who);
}

extern "C" int mcke_sm100_clip_grad_norm(const mcke_grad* grads, int count, float max_norm, float* norm,
                                         void* workspace, size_t workspace_bytes, mcke_stream_t stream) {
  static const char* who = "mcke_sm100_clip_grad_norm";
  clear_error();
  if (!norm) return fail(MCKE_INVALID_ARGUMENT, "%s: null norm", who);
  MCKE_RETURN_IF(check_max_norm(who, max_norm));
  MCKE_RETURN_IF(check_workspace(who, count, workspace, workspace_bytes));
  MCKE_RETURN_IF(check_list(who, grads, count, true, norm, true, workspace, workspace_bytes_of(count)));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  double* sums = static_cast<double*>(workspace);
  const int n = all_squares(grads, count, sums, s);
  if (n < kMaxBlocks) {
    all_clip(grads, count, NormSource{sums, n, nullptr, norm, max_norm}, s);
  } else {
    // a full grid, so many blocks of the scaling: folded once for all of them
    launch_async(grad_norm_fold_kernel, 1, kThreads, 0, s, static_cast<const double*>(sums), n, norm);
    all_clip(grads, count, NormSource{nullptr, 0, norm, nullptr, max_norm}, s);
  }
  return check_launch(who);
}
