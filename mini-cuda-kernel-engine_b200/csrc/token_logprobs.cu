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
#include "row_ops.cuh"

namespace mcke_sm100 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// Order of the alternatives: larger value first (NaN above all, -0 equal to
// +0), then lower index.  Never 0, so 0 stands for "none".
__device__ __forceinline__ uint64_t order_key(float v, int64_t index) {
  uint32_t u = __float_as_uint(v + 0.0f);
  u = (v != v) ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return (static_cast<uint64_t>(u) << 32) | static_cast<uint32_t>(~static_cast<uint32_t>(index));
}

__device__ __forceinline__ uint64_t warp_all_max(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  return v;
}
__device__ __forceinline__ float warp_all_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// `red` as for block_all_sum.
template <class V>
__device__ __forceinline__ V block_all_max(V v, V* red) {
  v = warp_all_max(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  V t = red[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) t = red[w] > t ? red[w] : t;
  return t;
}

struct ForwardOut {
  float* logprobs;
  float* lse;
  float* entropy;
  float* top_logprobs;
  int64_t* top_ids;
  int top_k;
};

// One block per row: the maximum, the sums, then one pass per alternative.
template <class T>
__global__ void __launch_bounds__(kThreads)
    token_logprobs_row_kernel(const T* __restrict__ x, int64_t stride, int64_t cols,
                              const int64_t* __restrict__ targets, ForwardOut out) {
  pdl_entry();
  __shared__ float red[3][kWarps];
  __shared__ uint64_t red_key[2][kWarps];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * stride;
  float m = -INFINITY;
  for (int64_t c = threadIdx.x; c < cols; c += kThreads) m = fmaxf(m, ld_val(xr + c));
  m = block_all_max(m, red[0]);
  const bool none = m == -INFINITY;
  float s = 0.0f, w = 0.0f;
  for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
    const float v = ld_val(xr + c);
    if (v == -INFINITY) continue;
    const float d = v - m, e = expf(d);
    s += e;
    w += e > 0.0f ? e * d : 0.0f;  // e^d d -> 0
  }
  s = block_all_sum<kWarps>(s, red[1]);
  w = block_all_sum<kWarps>(w, red[2]);
  const float ln_s = logf(s);
  if (threadIdx.x == 0) {
    if (out.lse) out.lse[row] = none ? (s != s ? s : m) : m + ln_s;
    if (out.entropy) out.entropy[row] = none ? (s != s ? s : 0.0f) : ln_s - w / s;
    if (out.logprobs) {
      const int64_t t = targets[row];
      float lp = 0.0f;
      if (t >= cols) lp = NAN;
      else if (t >= 0) lp = none ? (s != s ? s : m) : (ld_val(xr + t) - m) - ln_s;
      out.logprobs[row] = lp;
    }
  }
  uint64_t last = ~uint64_t{0};
  for (int k = 0; k < out.top_k; ++k) {
    uint64_t best = 0;
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
      const uint64_t key = order_key(ld_val(xr + c), c);
      if (key < last && key > best) best = key;
    }
    last = block_all_max(best, red_key[k & 1]);
    if (threadIdx.x == 0) {
      const int64_t id = static_cast<uint32_t>(~static_cast<uint32_t>(last));
      out.top_ids[row * out.top_k + k] = id;
      out.top_logprobs[row * out.top_k + k] = none ? (s != s ? s : m) : (ld_val(xr + id) - m) - ln_s;
    }
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

// dx may be x itself: an element is read before it is written, by the same thread.
template <class T>
__global__ void __launch_bounds__(kThreads)
    token_logprobs_backward_kernel(const T* x, int64_t stride, T* dx, int64_t dx_stride, int64_t cols, Grads g) {
  pdl_entry();
  const int64_t row = blockIdx.x;
  const T* xr = x + row * stride;
  T* dxr = dx + row * dx_stride;
  const float lse = g.lse[row];
  const int64_t t = g.logprobs ? g.targets[row] : -1;
  const float g_lp = t < 0 ? 0.0f : t >= cols ? NAN : g.logprobs[row];
  const float g_h = g.grad_entropy ? g.grad_entropy[row] : 0.0f;
  const float h = g.grad_entropy ? g.entropy[row] : 0.0f;
  const float a = (g.grad_lse ? g.grad_lse[row] : 0.0f) - g_lp;
  for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
    float d = 0.0f;
    if (lse != -INFINITY) {
      const float q = ld_val(xr + c) - lse;
      const float p = expf(q);
      d = (c == t ? g_lp : 0.0f) + (p == 0.0f ? 0.0f : p * (a - g_h * (q + h)));
      if (p == 0.0f && a != a) d = a;  // a bad target's NaN reaches every element
    }
    st_val(dxr + c, d);
  }
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
  if (rows > 2147483647LL || cols > 2147483647LL)
    return fail(MCKE_INVALID_ARGUMENT, "%s: extent exceeds INT32_MAX", who);
  if (top_k > cols) return fail(MCKE_INVALID_ARGUMENT, "%s: top_k %d of %lld columns", who, top_k, static_cast<long long>(cols));
  if (!logits || (logprobs && !targets) || (top_k > 0 && (!top_logprobs || !top_ids)))
    return fail(MCKE_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!logprobs && !lse && !entropy && top_k == 0) return MCKE_OK;
  MCKE_RETURN_IF(check_stride(who, "logits", stride, rows, cols, false));
  const std::size_t e = dtype_bytes(dtype);
  if (!aligned(logits, e)) return fail(MCKE_INVALID_ARGUMENT, "%s: logits is not element-aligned", who);
  const RowSpan outs[] = {span_of("logprobs", logprobs, rows * 4), span_of("lse", lse, rows * 4),
                          span_of("entropy", entropy, rows * 4),
                          span_of("top_logprobs", top_k > 0 ? top_logprobs : nullptr, rows * top_k * 4),
                          span_of("top_ids", top_k > 0 ? top_ids : nullptr, rows * top_k * 8)};
  const RowSpan ins[] = {span_of("logits", logits, rows, cols, stride, e), span_of("targets", targets, rows * 8)};
  MCKE_RETURN_IF(check_overlaps(who, outs, ins));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const ForwardOut out = {logprobs, lse, entropy, top_logprobs, top_ids, top_k};
  if (dtype == MCKE_DTYPE_BF16)
    launch_async(token_logprobs_row_kernel<uint16_t>, static_cast<unsigned>(rows), kThreads, 0, s,
                 static_cast<const uint16_t*>(logits), stride, cols, targets, out);
  else
    launch_async(token_logprobs_row_kernel<float>, static_cast<unsigned>(rows), kThreads, 0, s,
                 static_cast<const float*>(logits), stride, cols, targets, out);
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
  if (rows > 2147483647LL || cols > 2147483647LL)
    return fail(MCKE_INVALID_ARGUMENT, "%s: extent exceeds INT32_MAX", who);
  if (!logits || !lse || !dlogits || (grad_logprobs && !targets) || (grad_entropy && !entropy))
    return fail(MCKE_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!grad_logprobs && !grad_entropy && !grad_lse)
    return fail(MCKE_INVALID_ARGUMENT, "%s: no gradient is given", who);
  MCKE_RETURN_IF(check_stride(who, "logits", stride, rows, cols, false));
  MCKE_RETURN_IF(check_stride(who, "dlogits", dlogits_stride, rows, cols, true));
  const std::size_t e = dtype_bytes(dtype);
  if (!aligned(logits, e) || !aligned(dlogits, e))
    return fail(MCKE_INVALID_ARGUMENT, "%s: logits or dlogits is not element-aligned", who);
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
    launch_async(token_logprobs_backward_kernel<uint16_t>, static_cast<unsigned>(rows), kThreads, 0, s,
                 static_cast<const uint16_t*>(logits), stride, static_cast<uint16_t*>(dlogits), dlogits_stride, cols,
                 g);
  else
    launch_async(token_logprobs_backward_kernel<float>, static_cast<unsigned>(rows), kThreads, 0, s,
                 static_cast<const float*>(logits), stride, static_cast<float*>(dlogits), dlogits_stride, cols, g);
  return check_launch(who);
}
