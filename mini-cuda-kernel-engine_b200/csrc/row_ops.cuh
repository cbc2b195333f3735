// row_ops.cuh -- what the operators over rows of f32 or bf16 tensors share:
// element access, warp and block sums, and the argument checks of their entry
// points (row strides, overlap of outputs with inputs).
#pragma once

#include <cfloat>
#include <cmath>
#include <initializer_list>

#include "mcke_common.cuh"

namespace mcke_sm100 {

// ---- host: argument checks ------------------------------------------------------

inline std::size_t dtype_bytes(int dtype) { return dtype == MCKE_DTYPE_BF16 ? 2 : 4; }

// A block of rows: `rows` runs of `row_bytes` bytes, `pitch` bytes apart.
struct RowSpan {
  const char* name;
  const void* p;
  int64_t rows, row_bytes, pitch;
};
inline RowSpan span_of(const char* name, const void* p, int64_t rows, int64_t cols, int64_t stride, std::size_t elem) {
  return RowSpan{name, p, rows, cols * static_cast<int64_t>(elem), stride * static_cast<int64_t>(elem)};
}
inline RowSpan span_of(const char* name, const void* p, int64_t bytes) { return RowSpan{name, p, 1, bytes, bytes}; }

// Whether two blocks share a byte.  Blocks of one pitch that lie in disjoint
// column windows of the same buffer do not.
inline bool spans_overlap(const RowSpan& a, const RowSpan& b) {
  if (!a.p || !b.p || a.rows <= 0 || b.rows <= 0 || a.row_bytes <= 0 || b.row_bytes <= 0) return false;
  const auto a0 = reinterpret_cast<std::uintptr_t>(a.p), b0 = reinterpret_cast<std::uintptr_t>(b.p);
  const std::uintptr_t a1 = a0 + static_cast<std::uintptr_t>((a.rows - 1) * a.pitch + a.row_bytes);
  const std::uintptr_t b1 = b0 + static_cast<std::uintptr_t>((b.rows - 1) * b.pitch + b.row_bytes);
  if (a1 <= b0 || b1 <= a0) return false;
  if (a.rows > 1 && b.rows > 1 && a.pitch == b.pitch && a.pitch > 0) {
    const std::uintptr_t pitch = static_cast<std::uintptr_t>(a.pitch);
    const std::uintptr_t off = a0 <= b0 ? (b0 - a0) % pitch : (pitch - (a0 - b0) % pitch) % pitch;
    // b's window starts `off` bytes after a's: behind a's end, and its end before a's next row
    if (off >= static_cast<std::uintptr_t>(a.row_bytes) && off + static_cast<std::uintptr_t>(b.row_bytes) <= pitch)
      return false;
  }
  return true;
}

// Every output against every input and every other output.
template <int NOut, int NIn>
inline int check_overlaps(const char* who, const RowSpan (&out)[NOut], const RowSpan (&in)[NIn]) {
  for (int i = 0; i < NOut; ++i) {
    for (int j = 0; j < NIn; ++j)
      if (spans_overlap(out[i], in[j]))
        return fail(MCKE_INVALID_ARGUMENT, "%s: %s overlaps %s", who, out[i].name, in[j].name);
    for (int j = 0; j < i; ++j)
      if (spans_overlap(out[i], out[j]))
        return fail(MCKE_INVALID_ARGUMENT, "%s: %s overlaps %s", who, out[i].name, out[j].name);
  }
  return MCKE_OK;
}

inline int check_dtype(const char* who, int dtype) {
  if (dtype != MCKE_DTYPE_F32 && dtype != MCKE_DTYPE_BF16)
    return fail(MCKE_INVALID_ARGUMENT, "%s: unknown dtype %d", who, dtype);
  return MCKE_OK;
}

// Rows of an input may repeat or overlap (stride 0: one row read `rows` times);
// rows of an output may not.
inline int check_stride(const char* who, const char* name, int64_t stride, int64_t rows, int64_t cols, bool output) {
  if (rows > 1 && (stride < 0 || (output && stride < cols)))
    return fail(MCKE_INVALID_ARGUMENT, "%s: %s has row stride %lld for %lld columns", who, name,
                static_cast<long long>(stride), static_cast<long long>(cols));
  if (rows > 1 && stride > (int64_t{1} << 40) / rows)
    return fail(MCKE_INVALID_ARGUMENT, "%s: %s spans more than 2^40 elements", who, name);
  return MCKE_OK;
}

// Rows of one launch: row numbers plus a step over all blocks stay below 2^31.
constexpr int64_t kMaxRows = 2147483647LL - (1 << 16);

// Vectors of 4- or 8-byte elements, null allowed.
struct Aligned {
  const char* name;
  const void* p;
  std::size_t bytes;
};
inline int check_aligned(const char* who, std::initializer_list<Aligned> list) {
  for (const Aligned& v : list)
    if (v.p && !aligned(v.p, v.bytes)) return fail(MCKE_INVALID_ARGUMENT, "%s: %s is not element-aligned", who, v.name);
  return MCKE_OK;
}

// Lets a kernel use `bytes` of dynamic shared memory on the current device; one call
// to the runtime per kernel and device.
bool allow_shared_memory(const void* kernel, std::size_t bytes);

// ---- device: elements ---------------------------------------------------------------

// T is float, or uint16_t for raw bfloat16 patterns.
__device__ __forceinline__ float ld_val(const float* p) { return *p; }
__device__ __forceinline__ float ld_val(const uint16_t* p) { return from_bf16(*p); }
__device__ __forceinline__ void st_val(float* p, float v) { *p = v; }
__device__ __forceinline__ void st_val(uint16_t* p, float v) { *p = to_bf16(v); }

// Two floats in a 64-bit register: one instruction adds, multiplies or fuses both
// (sm_100's f32x2 forms; each half rounds as its scalar form does).
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 f2(float both) { return f2(both, both); }
__device__ __forceinline__ float2 split(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float sum2(F2 a) {
  const float2 s = split(a);
  return s.x + s.y;
}

// s / n for a row length n whose reciprocal is at hand: the product, and
// Markstein's correction of it by the remainder.  Of an infinite q the remainder is a
// NaN, of which fmaxf makes a finite number, and q stays as it is.
__device__ __forceinline__ float div_by(float s, float n, float inv_n) {
  const float q = s * inv_n;
  return fmaf(fmaxf(fmaf(-q, n, s), -FLT_MAX), inv_n, q);
}

// ---- device: sums --------------------------------------------------------------------

template <class V>
__device__ __forceinline__ V warp_all_sum(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the block's `kWarps` warps, the same bits in every thread.  `red`:
// kWarps values of shared memory that no thread still reads.
template <int kWarps, class V>
__device__ __forceinline__ V block_all_sum(V v, V* red) {
  v = warp_all_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  V t = red[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) t += red[w];
  return t;
}

}  // namespace mcke_sm100
