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
#include "row_ops.cuh"

namespace mcke_sm100 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// One block per row, three reads of it.
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
  float s = 0.0f;
  for (int64_t c = threadIdx.x; c < cols; c += kThreads) s += ld_val(xr + c);
  const float mu = block_all_sum<kWarps>(s, red[0]) / static_cast<float>(cols);
  float q = 0.0f;
  for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
    const float d = ld_val(xr + c) - mu;
    q += d * d;
  }
  const float r = 1.0f / sqrtf(block_all_sum<kWarps>(q, red[1]) / static_cast<float>(cols) + eps);
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
  float s1 = 0.0f, s2 = 0.0f;
  for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
    const float g = ld_val(dyr + c) * (weight ? weight[c] : 1.0f);
    s1 += g;
    s2 += g * ((ld_val(xr + c) - mu) * r);
  }
  const float c1 = block_all_sum<kWarps>(s1, red[0]) / static_cast<float>(cols);
  const float c2 = block_all_sum<kWarps>(s2, red[1]) / static_cast<float>(cols);
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

// dw and db from the slabs' partial sums, in slab order; zeros for no slab.
__global__ void __launch_bounds__(kThreads)
    layer_norm_fold_kernel(const float* __restrict__ part, int slabs, float* __restrict__ dweight,
                           float* __restrict__ dbias, int64_t cols) {
  pdl_entry();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= cols) return;
  float dw = 0.0f, db = 0.0f;
  for (int s = 0; s < slabs; ++s) {
    dw += part[(2 * static_cast<int64_t>(s)) * cols + c];
    db += part[(2 * static_cast<int64_t>(s) + 1) * cols + c];
  }
  if (dweight) dweight[c] = dw;
  if (dbias) dbias[c] = db;
}

// Slabs of rows whose column sums are kept apart.  From the extents alone, so
// the order of the sums, and every bit of dw and db, is the same on any GPU.
int64_t column_slabs(int64_t rows) { return rows < 148 ? rows : 148; }

template <class T>
void launch_forward(const void* x, int64_t x_stride, const float* weight, const float* bias, void* y, int64_t y_stride,
                    float* mean, float* rstd, int64_t rows, int64_t cols, float eps, cudaStream_t s) {
  launch_async(layer_norm_row_kernel<T>, static_cast<unsigned>(rows), kThreads, 0, s, static_cast<const T*>(x),
               x_stride, weight, bias, static_cast<T*>(y), y_stride, mean, rstd, cols, eps);
}

template <class T>
void launch_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const float* weight,
                     const float* mean, const float* rstd, void* dx, int64_t dx_stride, float* dweight, float* dbias,
                     int64_t rows, int64_t cols, float* part, cudaStream_t s) {
  const T* dyt = static_cast<const T*>(dy);
  const T* xt = static_cast<const T*>(x);
  const unsigned blocks = static_cast<unsigned>((cols + kThreads - 1) / kThreads);
  const int64_t slabs = column_slabs(rows);
  if (rows > 0)
    launch_async(layer_norm_dx_kernel<T>, static_cast<unsigned>(rows), kThreads, 0, s, dyt, dy_stride, xt, x_stride,
                 weight, mean, rstd, static_cast<T*>(dx), dx_stride, cols);
  if (!dweight && !dbias) return;
  if (rows > 0)
    launch_async(layer_norm_columns_kernel<T>, dim3(blocks, static_cast<unsigned>(slabs)), kThreads, 0, s, dyt,
                 dy_stride, xt, x_stride, mean, rstd, part, rows, cols);
  launch_async(layer_norm_fold_kernel, blocks, kThreads, 0, s, static_cast<const float*>(part),
               static_cast<int>(slabs), dweight, dbias, cols);
}

}  // namespace
}  // namespace mcke_sm100

using namespace mcke_sm100;

extern "C" int mcke_sm100_layer_norm(const void* x, int64_t x_stride, const float* weight, const float* bias, void* y,
                                     int64_t y_stride, float* mean, float* rstd, int64_t rows, int64_t cols, float eps,
                                     int dtype, mcke_stream_t stream) {
  static const char* who = "mcke_sm100_layer_norm";
  clear_error();
  MCKE_RETURN_IF(check_dtype(who, dtype));
  if (rows < 0 || cols < 0) return fail(MCKE_INVALID_ARGUMENT, "%s: negative extent", who);
  if (!(eps >= 0.0f) || std::isinf(eps)) return fail(MCKE_INVALID_ARGUMENT, "%s: eps must be finite and >= 0", who);
  if (rows == 0 || cols == 0) return MCKE_OK;
  if (!x || !y) return fail(MCKE_INVALID_ARGUMENT, "%s: null pointer", who);
  if (rows > 2147483647LL || cols > 2147483647LL)
    return fail(MCKE_INVALID_ARGUMENT, "%s: extent exceeds INT32_MAX", who);
  MCKE_RETURN_IF(check_stride(who, "x", x_stride, rows, cols, false));
  MCKE_RETURN_IF(check_stride(who, "y", y_stride, rows, cols, true));
  const std::size_t e = dtype_bytes(dtype);
  if (!aligned(x, e) || !aligned(y, e)) return fail(MCKE_INVALID_ARGUMENT, "%s: x or y is not element-aligned", who);
  const RowSpan outs[] = {span_of("y", y, rows, cols, y_stride, e), span_of("mean", mean, rows * 4),
                          span_of("rstd", rstd, rows * 4)};
  const RowSpan ins[] = {span_of("x", x, rows, cols, x_stride, e), span_of("weight", weight, cols * 4),
                         span_of("bias", bias, cols * 4)};
  MCKE_RETURN_IF(check_overlaps(who, outs, ins));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == MCKE_DTYPE_BF16)
    launch_forward<uint16_t>(x, x_stride, weight, bias, y, y_stride, mean, rstd, rows, cols, eps, s);
  else
    launch_forward<float>(x, x_stride, weight, bias, y, y_stride, mean, rstd, rows, cols, eps, s);
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
  if (rows > 2147483647LL || cols > 2147483647LL)
    return fail(MCKE_INVALID_ARGUMENT, "%s: extent exceeds INT32_MAX", who);
  if (rows > 0 && (!dy || !x || !mean || !rstd || !dx)) return fail(MCKE_INVALID_ARGUMENT, "%s: null pointer", who);
  MCKE_RETURN_IF(check_stride(who, "dy", dy_stride, rows, cols, false));
  MCKE_RETURN_IF(check_stride(who, "x", x_stride, rows, cols, false));
  MCKE_RETURN_IF(check_stride(who, "dx", dx_stride, rows, cols, true));
  const std::size_t e = dtype_bytes(dtype);
  if (!aligned(dy, e) || !aligned(x, e) || !aligned(dx, e))
    return fail(MCKE_INVALID_ARGUMENT, "%s: dy, x or dx is not element-aligned", who);
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
  float* part = static_cast<float*>(workspace);
  if (dtype == MCKE_DTYPE_BF16)
    launch_backward<uint16_t>(dy, dy_stride, x, x_stride, weight, mean, rstd, dx, dx_stride, dweight, dbias, rows,
                              cols, part, s);
  else
    launch_backward<float>(dy, dy_stride, x, x_stride, weight, mean, rstd, dx, dx_stride, dweight, dbias, rows, cols,
                           part, s);
  return check_launch(who);
}
