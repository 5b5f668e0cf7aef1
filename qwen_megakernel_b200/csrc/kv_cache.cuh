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
  }
  if (i >= R.max_rows) return -1;
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

// ------------------------------------------------------------ quantization
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// x / s, correctly rounded for what is asked here, from r ~ 1 / s: one Newton
// step on the quotient with its exact remainder (Markstein's division).  Its
// error before the last rounding is below 2^-44 of the quotient, so a quotient
// that fp32 holds (the border of two codes, or of two bf16 scales, among them)
// comes out exactly, and one that lies off a border is not rounded onto it: x
// and s have 24 and 8 bits, the nearest such quotient is more than half a step
// of fp32 away.  Both within 2^-100 .. 2^126.
__device__ __forceinline__ float divide(float x, float s, float r) {
  const float q = x * r;
  return fmaf(fmaf(-q, s, x), r, q);
}

// N values of a group to codes, packed; any scale, any value.
template <int BITS, int N>
__device__ __forceinline__ void codes_any(const float (&x)[N], float s, unsigned (&word)[(N * BITS + 31) / 32]) {
  constexpr float kTop = BITS == 4 ? 7.f : 127.f, kOffset = BITS == 4 ? 8.f : 128.f;
#pragma unroll
  for (int i = 0; i < (N * BITS + 31) / 32; ++i) word[i] = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float c = 0.f;
    if (s != 0.f && x[i] == x[i]) c = fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -kTop), kTop);
    word[i * BITS / 32] |= (unsigned)(int)(c + kOffset) << (i * BITS % 32);
  }
}

// Codes (packed from the low bits) and scale of a thread's N values; the 32 / N
// neighbouring lanes of a group agree.  All lanes of the warp call it; what a
// lane without values (!live) gets means nothing.
template <int BITS, int N>
__device__ __forceinline__ __nv_bfloat16 quantize(const float (&x)[N], unsigned (&word)[(N * BITS + 31) / 32],
                                                  unsigned *status, bool live = true) {
  constexpr float kTop = BITS == 4 ? 7.f : 127.f;
  unsigned top = 0;  // bits of the largest magnitude, infinities and NaN above all
#pragma unroll
  for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = 1; o < kGroup / N; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  // largest magnitude within 2^-90 .. 2^126: scale and quotients are ordinary numbers
  const bool easy = !live || (top >= 0x12800000u && top < 0x7e800000u);
  if (__all_sync(0xffffffffu, easy)) {
    const __nv_bfloat16 sb = __float2bfloat16_rn(divide(__uint_as_float(top), kTop, 1.f / kTop));
    const float s = __bfloat162float(sb), r = fast_rcp(s);
    // x / s + 1.5 2^23 + offset holds the code, rounded to even, in its low
    // bits; in a word's sum the patterns above the codes add up to a constant
    constexpr float kMagic = 12582912.f + (BITS == 4 ? 8.f : 128.f);
    constexpr int kPer = N < 32 / BITS ? N : 32 / BITS;
    unsigned above = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) above += 0x4b400000u << (BITS * i);
#pragma unroll
    for (int w = 0; w < (N * BITS + 31) / 32; ++w) {
      unsigned sum = 0u - above;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        sum += __float_as_uint(divide(x[kPer * w + i], s, r) + kMagic) * (1u << (BITS * i));
      word[w] = sum;
    }
    return sb;
  }
  unsigned fin = 0;  // largest finite magnitude
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const unsigned u = __float_as_uint(x[i]) & 0x7fffffffu;
    fin = max(fin, u < 0x7f800000u ? u : 0u);
  }
#pragma unroll
  for (int o = 1; o < kGroup / N; o <<= 1) fin = max(fin, __shfl_xor_sync(0xffffffffu, fin, o));
  if (live && top >= 0x7f800000u && status) atomicOr(status, QMK_KV_NONFINITE);
  const __nv_bfloat16 sb = __float2bfloat16_rn(__fdiv_rn(__uint_as_float(fin), kTop));
  codes_any<BITS, N>(x, __bfloat162float(sb), word);
  return sb;
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
