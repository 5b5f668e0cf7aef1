// Quantized K/V cache: rows quantized as they are written, and read back
// (qmk_kv_write, qmk_kv_read; the format is in include/qwen_megakernel.h).
//
// Both are one pass over the data, bound by the row tensors' bytes (bf16: 256
// of a row and head's 328).  A thread owns 8 consecutive dimensions of one
// head (16 bytes of bf16, one 32-bit word of 4-bit codes) in a few rows, K and
// V alike, with all its loads issued first; 4 neighbouring lanes hold a group
// of 32, so the group's largest magnitude is two shuffles.  A CTA looks its
// rows' sequences and positions up once, in shared memory.
//
// Measured, 32,368 rows of 8 x 128 bf16, 4 bits: written and read back in 86 us,
// 51 and 35 us (170 MB each, 3.3 and 4.8 TB/s).  The write runs 15 instructions
// a value (the exact quotient 4 of them) at half the issue rate, the loads'
// latency the rest: 4 CTAs an SM of 64 registers 86 us, 3 of 70 92, one row a
// thread in flight 95, four 102.  With the row looked up by every thread and a
// correctly rounded division a value the pair took 161 us.

#include <algorithm>
#include <cstdarg>
#include <cstdio>

#include "kv_cache.cuh"

int qmk_internal_set_error(int code, const char *msg);
int qmk_internal_clear_error();

namespace qkv {

int fail(int code, const char *fmt, ...) {
  char msg[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  return qmk_internal_set_error(code, msg);
}

int check_cache(const char *who, const QmkKvCache *c) {
  if (!c) return fail(QMK_ERR_ARGS, "%s: null cache", who);
  if (!c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales)
    return fail(QMK_ERR_ARGS, "%s: null cache pointer", who);
  if (c->bits != 4 && c->bits != 8) return fail(QMK_ERR_ARGS, "%s: bits=%d is not 4 or 8", who, c->bits);
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(QMK_ERR_ARGS, "%s: head_dim=%d is not 64 or 128", who, c->head_dim);
  if (c->num_seqs < 1 || c->num_kv_heads < 1)
    return fail(QMK_ERR_ARGS, "%s: num_seqs=%d num_kv_heads=%d", who, c->num_seqs, c->num_kv_heads);
  if (c->max_seq_len < 1 || c->capacity < c->max_seq_len || c->capacity % QMK_KV_CAPACITY_STEP)
    return fail(QMK_ERR_ARGS, "%s: capacity=%d must be a multiple of %d and >= max_seq_len=%d >= 1", who, c->capacity,
                QMK_KV_CAPACITY_STEP, c->max_seq_len);
  const long long rows = (long long)c->num_kv_heads * c->capacity;
  if (c->num_seqs > 1 && (c->code_seq_stride < rows * (c->head_dim * c->bits / 8) ||
                          c->scale_seq_stride < rows * (c->head_dim / kGroup)))
    return fail(QMK_ERR_ARGS, "%s: sequence strides smaller than one sequence's cache", who);
  if (c->num_seqs > 1 && (c->code_seq_stride % 16 || c->scale_seq_stride % 8))
    return fail(QMK_ERR_ARGS, "%s: sequence strides are not multiples of 16 bytes", who);
  if ((reinterpret_cast<uintptr_t>(c->k_codes) | reinterpret_cast<uintptr_t>(c->v_codes) |
       reinterpret_cast<uintptr_t>(c->k_scales) | reinterpret_cast<uintptr_t>(c->v_scales)) % 16)
    return fail(QMK_ERR_ARGS, "%s: cache not 16-byte aligned", who);
  return QMK_OK;
}

int check_rows(const char *who, const QmkKvCache *c, const QmkKvRows *r) {
  if (!r) return fail(QMK_ERR_ARGS, "%s: null rows", who);
  if (r->rows < 0 || r->segments < 0 || r->max_rows < 0)
    return fail(QMK_ERR_ARGS, "%s: rows=%d segments=%d max_rows=%d", who, r->rows, r->segments, r->max_rows);
  if (r->rows == 0 || r->segments == 0) return QMK_OK;
  if (!r->start) return fail(QMK_ERR_ARGS, "%s: null start", who);
  if (!r->row_offsets && r->segments != r->rows)
    return fail(QMK_ERR_ARGS, "%s: %d segments for %d rows need row_offsets", who, r->segments, r->rows);
  if (r->max_rows > c->capacity) return fail(QMK_ERR_ARGS, "%s: max_rows=%d exceeds the cache", who, r->max_rows);
  return QMK_OK;
}

int check_tensor(const char *who, const char *name, const QmkKvTensor *t) {
  if (!t || !t->data) return fail(QMK_ERR_ARGS, "%s: null %s", who, name);
  if (t->dtype != QMK_BF16 && t->dtype != QMK_FP16 && t->dtype != QMK_FP32)
    return fail(QMK_ERR_ARGS, "%s: %s has dtype %d", who, name, t->dtype);
  if (reinterpret_cast<uintptr_t>(t->data) % dtype_size(t->dtype))
    return fail(QMK_ERR_ARGS, "%s: %s is not aligned to its elements", who, name);
  return QMK_OK;
}

Rows device_rows(const QmkKvCache *c, const QmkKvRows *r) {
  return Rows{r->start, r->row_offsets, r->seq, r->rows, r->segments, r->max_rows, c->num_seqs, c->max_seq_len};
}

bool vector_aligned(const QmkKvTensor *t) {
  const long long per = 16 / (long long)dtype_size(t->dtype);
  return reinterpret_cast<uintptr_t>(t->data) % 16 == 0 && t->row_stride % per == 0 && t->head_stride % per == 0;
}

// One of K and V: codes, scales and the row tensor.
template <typename T>
struct Side {
  uint8_t *codes;
  __nv_bfloat16 *scales;
  T *x;
  long long row_stride, head_stride;
};

template <typename T>
struct Args {
  Side<T> side[2];  // K, V
  Rows rows;
  long long code_seq_stride, scale_seq_stride;
  int heads, capacity, rows_per_cta;
  unsigned *status;
};

constexpr int kThreads = 256;
constexpr int kMaxRowsPerCta = 64;
constexpr int kBatch = 2;  // rows of a thread in flight

// Where the CTA's rows lie, looked up once: offsets of their sequence and
// position (the head's come on top), -1 where no segment holds the row, -2
// where it is out of range.
struct RowTable {
  long long code[kMaxRowsPerCta];
  long long scale[kMaxRowsPerCta];
};

template <typename T, int BITS, int D>
__device__ __forceinline__ int fill_rows(RowTable &t, const Args<T> &a, int row0) {
  const int n = min(a.rows_per_cta, a.rows.rows - row0);
  if ((int)threadIdx.x < n) {
    int seq = 0, pos = 0;
    const int ok = locate_row(a.rows, row0 + threadIdx.x, seq, pos);
    if (ok < 0 && a.status) atomicOr(a.status, QMK_KV_BAD_ROW);
    t.code[threadIdx.x] = ok > 0 ? seq * a.code_seq_stride + (long long)pos * (D * BITS / 8) : ok - 1;
    t.scale[threadIdx.x] = seq * a.scale_seq_stride + (long long)pos * (D / kGroup);
  }
  __syncthreads();
  return n;
}

// 8 elements as they lie in memory; single loads unless VEC.
template <typename T, bool VEC>
struct Raw {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) reinterpret_cast<T *>(w)[i] = p[i];
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float(reinterpret_cast<const T *>(w)[i]);
  }
};

template <typename T, int BITS, int D, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) write_kernel(const __grid_constant__ Args<T> a) {
  __shared__ RowTable tab;
  qmk::pdl_wait();  // rows and cache may be touched by the previous kernel
  qmk::pdl_trigger();
  constexpr int kChunks = D / 8;
  const int row0 = blockIdx.x * a.rows_per_cta;
  const int n = fill_rows<T, BITS, D>(tab, a, row0);
  const int cols = a.heads * kChunks;                               // (head, chunk) pairs, a multiple of 8
  const int width = min(cols, kThreads), lines = kThreads / width;  // threads a row, rows at once
  const int line = threadIdx.x / width;
  // (all lanes of a warp run the same trips, for the shuffles: those without a value idle along)
  for (int base = 0; base < cols; base += width) {
    const int c0 = base + threadIdx.x - line * width;
    const int head = c0 / kChunks, chunk = c0 % kChunks;
    const bool in = line < lines && c0 < cols;
    const T *src[2];
    uint8_t *codes[2];
    __nv_bfloat16 *scales[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const Side<T> &sd = a.side[i];
      src[i] = sd.x + (size_t)row0 * (size_t)sd.row_stride + (size_t)head * (size_t)sd.head_stride + 8 * chunk;
      codes[i] = sd.codes + (size_t)head * (size_t)a.capacity * (D * BITS / 8) + BITS * chunk;
      scales[i] = sd.scales + (size_t)head * (size_t)a.capacity * (D / kGroup) + (chunk >> 2);
    }
    for (int r0 = 0; r0 < n; r0 += kBatch * lines) {
      Raw<T, VEC> raw[kBatch][2];
      bool ok[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int r = r0 + k * lines + line;
        ok[k] = in && r < n && tab.code[r] >= 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          raw[k][i].zero();
          if (ok[k]) raw[k][i].load(src[i] + (size_t)r * (size_t)a.side[i].row_stride);
        }
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x[8];
          unsigned word[BITS / 4];
          raw[k][i].get(x);
          const __nv_bfloat16 sb = quantize<BITS, 8>(x, word, a.status, ok[k]);
          if (ok[k]) {
            const int r = r0 + k * lines + line;
            uint8_t *dst = codes[i] + tab.code[r];
            if constexpr (BITS == 4) *reinterpret_cast<unsigned *>(dst) = word[0];
            else *reinterpret_cast<uint2 *>(dst) = make_uint2(word[0], word[1]);
            if ((chunk & 3) == 0) scales[i][tab.scale[r]] = sb;
          }
        }
    }
  }
}

template <typename T, int BITS, int D, bool VEC>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ Args<T> a) {
  __shared__ RowTable tab;
  qmk::pdl_wait();  // the cache is written by the previous kernel
  qmk::pdl_trigger();
  constexpr int kChunks = D / 8;
  const int row0 = blockIdx.x * a.rows_per_cta;
  const int n = fill_rows<T, BITS, D>(tab, a, row0);
  const int cols = a.heads * kChunks;
  const int width = min(cols, kThreads), lines = kThreads / width;
  const int line = threadIdx.x / width;
  if (line >= lines) return;
  for (int c0 = threadIdx.x - line * width; c0 < cols; c0 += width) {
    const int head = c0 / kChunks, chunk = c0 % kChunks;
    const uint8_t *codes[2];
    const __nv_bfloat16 *scales[2];
    T *dst[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const Side<T> &sd = a.side[i];
      dst[i] = sd.x + (size_t)row0 * (size_t)sd.row_stride + (size_t)head * (size_t)sd.head_stride + 8 * chunk;
      codes[i] = sd.codes + (size_t)head * (size_t)a.capacity * (D * BITS / 8) + BITS * chunk;
      scales[i] = sd.scales + (size_t)head * (size_t)a.capacity * (D / kGroup) + (chunk >> 2);
    }
    for (int r0 = line; r0 < n; r0 += kBatch * lines) {
      unsigned word[kBatch][2][BITS / 4];
      float s[kBatch][2];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int r = r0 + k * lines;
        const bool ok = r < n && tab.code[r] >= 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // a row out of range reads as zeros: the scale is 0
          s[k][i] = 0.f;
#pragma unroll
          for (int e = 0; e < BITS / 4; ++e) word[k][i][e] = 0u;
          if (ok) {
            s[k][i] = __bfloat162float(scales[i][tab.scale[r]]);
            if constexpr (BITS == 4) {
              word[k][i][0] = *reinterpret_cast<const unsigned *>(codes[i] + tab.code[r]);
            } else {
              const uint2 w = *reinterpret_cast<const uint2 *>(codes[i] + tab.code[r]);
              word[k][i][0] = w.x;
              word[k][i][1] = w.y;
            }
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int r = r0 + k * lines;
        if (r >= n || tab.code[r] == -1) continue;  // (-1: no segment holds the row)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int u = (int)((word[k][i][e * BITS / 32] >> (e * BITS % 32)) & ((1u << BITS) - 1u));
            x[e] = s[k][i] * (float)(u - (1 << (BITS - 1)));  // exact: 8 + 7 significant bits
          }
          store_n<T, 8>(dst[i] + (size_t)r * (size_t)a.side[i].row_stride, VEC, x);
        }
      }
    }
  }
}

template <typename T, bool WRITE, int BITS, int D>
void (*pick(bool vec))(const Args<T>) {
  if constexpr (WRITE) return vec ? write_kernel<T, BITS, D, true> : write_kernel<T, BITS, D, false>;
  else return vec ? read_kernel<T, BITS, D, true> : read_kernel<T, BITS, D, false>;
}

template <typename T, bool WRITE>
int launch(const QmkKvCache *c, const QmkKvRows *r, const QmkKvTensor *k, const QmkKvTensor *v, unsigned *status,
           cudaStream_t stream) {
  Args<T> a;
  const QmkKvTensor *t[2] = {k, v};
  void *codes[2] = {c->k_codes, c->v_codes}, *scales[2] = {c->k_scales, c->v_scales};
  for (int i = 0; i < 2; ++i)
    a.side[i] = Side<T>{static_cast<uint8_t *>(codes[i]), static_cast<__nv_bfloat16 *>(scales[i]),
                        static_cast<T *>(t[i]->data), t[i]->row_stride, t[i]->head_stride};
  a.rows = device_rows(c, r);
  a.code_seq_stride = c->code_seq_stride;
  a.scale_seq_stride = c->scale_seq_stride;
  a.heads = c->num_kv_heads;
  a.capacity = c->capacity;
  a.status = status;
  // rows a CTA: enough for its threads' batches, fewer while that leaves SMs without work
  const int width = std::min(c->num_kv_heads * (c->head_dim / 8), kThreads);
  const int batch = kBatch * (kThreads / width);
  int per = std::min(kMaxRowsPerCta, 4 * batch);
  while (per > 1 && (r->rows + per - 1) / per < 4 * 148) per = (per + 1) / 2;
  a.rows_per_cta = per;
  const int blocks = (r->rows + per - 1) / per;
  const bool vec = vector_aligned(k) && vector_aligned(v);
  void (*kernel)(const Args<T>) =
      c->head_dim == 128 ? (c->bits == 4 ? pick<T, WRITE, 4, 128>(vec) : pick<T, WRITE, 8, 128>(vec))
                         : (c->bits == 4 ? pick<T, WRITE, 4, 64>(vec) : pick<T, WRITE, 8, 64>(vec));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) return fail(QMK_ERR_CUDA, "qmk_kv launch: %s", cudaGetErrorString(e));
  return QMK_OK;
}

template <bool WRITE>
int run(const char *who, const QmkKvCache *c, const QmkKvRows *r, const QmkKvTensor *k, const QmkKvTensor *v,
        unsigned *status, cudaStream_t stream) {
  qmk_internal_clear_error();
  int rc = check_cache(who, c);
  if (rc == QMK_OK) rc = check_rows(who, c, r);
  if (rc == QMK_OK && (r->rows == 0 || r->segments == 0)) return QMK_OK;
  if (rc == QMK_OK) rc = check_tensor(who, "k", k);
  if (rc == QMK_OK) rc = check_tensor(who, "v", v);
  if (rc != QMK_OK) return rc;
  if (k->dtype != v->dtype) return fail(QMK_ERR_ARGS, "%s: k and v have different types", who);
  if (k->dtype == QMK_BF16) return launch<__nv_bfloat16, WRITE>(c, r, k, v, status, stream);
  if (k->dtype == QMK_FP16) return launch<__half, WRITE>(c, r, k, v, status, stream);
  return launch<float, WRITE>(c, r, k, v, status, stream);
}

}  // namespace qkv

extern "C" int qmk_kv_write(const QmkKvCache *cache, const QmkKvRows *rows, const QmkKvTensor *k,
                            const QmkKvTensor *v, unsigned int *status, cudaStream_t stream) {
  return qkv::run<true>("qmk_kv_write", cache, rows, k, v, status, stream);
}

extern "C" int qmk_kv_read(const QmkKvCache *cache, const QmkKvRows *rows, const QmkKvTensor *k,
                           const QmkKvTensor *v, unsigned int *status, cudaStream_t stream) {
  return qkv::run<false>("qmk_kv_read", cache, rows, k, v, status, stream);
}
