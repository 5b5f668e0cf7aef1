// Shared by the quantized K/V cache's kernels (kv_cache.cu, kv_attend.cu):
// how a call's rows are addressed, and element types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "qmk_device.cuh"
#include "qwen_megakernel.h"

namespace qkv {

constexpr int kGroup = QMK_KV_GROUP;

// Device copy of QmkKvRows with the cache's limits.
struct Rows {
  const int *start, *row_offsets, *seq;
  int rows, segments, max_rows, num_seqs, max_seq_len;
};

// Rows [r0, r0 + n) of segment b; n is clamped so that no device data can
// lead outside the call's row tensors.
__device__ __forceinline__ void segment_rows(const Rows &R, int b, int &r0, int &n) {
  if (R.row_offsets == nullptr) {
    r0 = b;
    n = 1;
    return;
  }
  r0 = min(max(R.row_offsets[b], 0), R.rows);
  n = max(min(max(R.row_offsets[b + 1], 0), R.rows) - r0, 0);
}

__device__ __forceinline__ int segment_seq(const Rows &R, int b) { return R.seq ? R.seq[b] : b; }

// Sequence and position of row r: 1 ok, 0 no segment holds the row, -1 out of
// range.  The segment is the last one that starts at or before r.
__device__ __forceinline__ int locate_row(const Rows &R, int r, int &seq, int &pos) {
  int b = r, i = 0;
  if (R.row_offsets) {
    int lo = 0, hi = R.segments;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (R.row_offsets[mid] <= r) lo = mid;
      else hi = mid;
    }
    b = lo;
    i = r - max(R.row_offsets[b], 0);
    if (i < 0 || r >= R.row_offsets[b + 1]) return 0;
    if (i >= R.max_rows) return -1;
  }
  seq = segment_seq(R, b);
  const int start = R.start[b];
  if (seq < 0 || seq >= R.num_seqs || start < 0 || start >= R.max_seq_len || i >= R.max_seq_len - start) return -1;
  pos = start + i;
  return 1;
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// N consecutive elements, N * sizeof(T) a multiple of 16 bytes: as 16-byte
// accesses where `aligned` (the base and every stride allow it), else singly.
template <typename T, int N>
__device__ __forceinline__ void load_n(const T *p, bool aligned, float (&x)[N]) {
  constexpr int kPer = 16 / sizeof(T);
  if (aligned) {
#pragma unroll
    for (int i = 0; i < N; i += kPer) {
      const uint4 w = __ldg(reinterpret_cast<const uint4 *>(p + i));
      const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
      for (int k = 0; k < kPer; ++k) x[i + k] = to_float(e[k]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_float(p[i]);
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_n(T *p, bool aligned, const float (&x)[N]) {
  constexpr int kPer = 16 / sizeof(T);
  if (aligned) {
#pragma unroll
    for (int i = 0; i < N; i += kPer) {
      uint4 w;
      T *e = reinterpret_cast<T *>(&w);
#pragma unroll
      for (int k = 0; k < kPer; ++k) e[k] = from_float<T>(x[i + k]);
      *reinterpret_cast<uint4 *>(p + i) = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = from_float<T>(x[i]);
  }
}

inline size_t dtype_size(int dtype) { return dtype == QMK_FP32 ? 4 : 2; }

// Host-side checks shared by the entry points (kv_cache.cu): QMK_OK or an
// error recorded for qmk_get_last_error().
int check_cache(const char *who, const QmkKvCache *c);
int check_rows(const char *who, const QmkKvCache *c, const QmkKvRows *r);
int check_tensor(const char *who, const char *name, const QmkKvTensor *t);
int fail(int code, const char *fmt, ...);
Rows device_rows(const QmkKvCache *c, const QmkKvRows *r);
bool vector_aligned(const QmkKvTensor *t);

}  // namespace qkv
