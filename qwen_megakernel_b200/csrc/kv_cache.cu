// Quantized K/V cache: rows quantized as they are written, and read back
// (qmk_kv_write, qmk_kv_read; the format is in include/qwen_megakernel.h).
//
// Both are one pass over the data: a thread owns 8 consecutive dimensions of
// one row and head (16 bytes of bf16, one 32-bit word of 4-bit codes), 4
// neighbouring lanes one group of 32, so the group's largest magnitude is two
// shuffles and every access is a full, coalesced vector.

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
  bool aligned;
};

template <typename T>
struct Args {
  Side<T> side[2];  // K, V
  Rows rows;
  long long code_seq_stride, scale_seq_stride;
  int heads, capacity;
  unsigned *status;
};

constexpr int kThreads = 256;

// rint(x / s) for |x| <= s * (127 + 1/2), s a normal bf16: exact, with one
// reciprocal for the group.  r = rint(x * (1 / s)) can miss only at a
// border between two codes; d = x - r s has no rounding error (r s has at
// most 15 significant bits; for r != 0 x and r s are within a factor 2 of
// each other), so the comparison of |d| with s / 2 decides, ties to even.
__device__ __forceinline__ float code_of(float x, float s, float inv, float half) {
  float r = rintf(x * inv);
  const float d = fmaf(-r, s, x), ad = fabsf(d);
  if (ad > half || (ad == half && (static_cast<int>(r) & 1))) r += copysignf(1.f, d);
  return r;
}

template <typename T, int BITS, int D>
__global__ void __launch_bounds__(kThreads) write_kernel(const __grid_constant__ Args<T> a) {
  qmk::pdl_wait();  // rows and cache may be touched by the previous kernel
  qmk::pdl_trigger();
  constexpr int kChunks = D / 8;
  constexpr float kTop = BITS == 4 ? 7.f : 127.f;
  const Side<T> &sd = a.side[blockIdx.y];
  const long long unit = ((long long)blockIdx.x * kThreads + threadIdx.x) / kChunks;  // (row, head)
  const int chunk = threadIdx.x % kChunks;
  const long long row = unit / a.heads;
  const int head = (int)(unit - row * a.heads);
  int seq = 0, pos = 0, ok = 0;
  if (row < a.rows.rows) ok = locate_row(a.rows, (int)row, seq, pos);
  if (ok < 0 && chunk == 0 && head == 0 && a.status) atomicOr(a.status, QMK_KV_BAD_ROW);
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (ok > 0)
    load_n<T, 8>(sd.x + (size_t)row * (size_t)sd.row_stride + (size_t)head * (size_t)sd.head_stride + 8 * chunk,
                 sd.aligned, x);
  float top = 0.f;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float m = fabsf(x[i]);
    const bool fin = m < INFINITY;  // false for NaN too
    odd |= !fin;
    top = fin ? fmaxf(top, m) : top;
  }
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  if (odd && a.status) atomicOr(a.status, QMK_KV_NONFINITE);
  if (ok <= 0) return;
  const __nv_bfloat16 sb = __float2bfloat16_rn(__fdiv_rn(top, kTop));
  const float s = __bfloat162float(sb);
  unsigned word[BITS / 4] = {};
  constexpr float kOffset = BITS == 4 ? 8.f : 128.f;
  // The reciprocal needs s well inside the normal range (2^-100 .. 2^126).
  const bool normal = s > 7.9e-31f && s < 8e37f;
  const float inv = __frcp_rn(s), half = 0.5f * s;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float c;
    if (s == 0.f) {
      c = 0.f;
    } else if (!(fabsf(x[i]) < INFINITY)) {
      c = (x[i] != x[i]) ? 0.f : copysignf(kTop, x[i]);
    } else {
      c = normal ? code_of(x[i], s, inv, half) : rintf(__fdiv_rn(x[i], s));
      c = fminf(fmaxf(c, -kTop), kTop);  // beyond only where s is rounded coarsely (subnormal)
    }
    const unsigned u = (unsigned)(int)(c + kOffset);
    word[i * BITS / 32] |= u << (i * BITS % 32);
  }
  const size_t at = (size_t)head * (size_t)a.capacity + (size_t)pos;
  uint8_t *dst = sd.codes + (size_t)seq * (size_t)a.code_seq_stride + at * (D * BITS / 8) + chunk * BITS;
  if constexpr (BITS == 4) *reinterpret_cast<unsigned *>(dst) = word[0];
  else *reinterpret_cast<uint2 *>(dst) = make_uint2(word[0], word[1]);
  if ((chunk & 3) == 0)
    sd.scales[(size_t)seq * (size_t)a.scale_seq_stride + at * (D / kGroup) + (chunk >> 2)] = sb;
}

template <typename T, int BITS, int D>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ Args<T> a) {
  qmk::pdl_wait();  // the cache is written by the previous kernel
  qmk::pdl_trigger();
  constexpr int kChunks = D / 8;
  const Side<T> &sd = a.side[blockIdx.y];
  const long long unit = ((long long)blockIdx.x * kThreads + threadIdx.x) / kChunks;
  const int chunk = threadIdx.x % kChunks;
  const long long row = unit / a.heads;
  const int head = (int)(unit - row * a.heads);
  if (row >= a.rows.rows) return;
  int seq = 0, pos = 0;
  const int ok = locate_row(a.rows, (int)row, seq, pos);
  if (ok == 0) return;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (ok > 0) {
    const size_t at = (size_t)head * (size_t)a.capacity + (size_t)pos;
    const uint8_t *src = sd.codes + (size_t)seq * (size_t)a.code_seq_stride + at * (D * BITS / 8) + chunk * BITS;
    const float s =
        __bfloat162float(sd.scales[(size_t)seq * (size_t)a.scale_seq_stride + at * (D / kGroup) + (chunk >> 2)]);
    unsigned word[BITS / 4];
    if constexpr (BITS == 4) {
      word[0] = *reinterpret_cast<const unsigned *>(src);
    } else {
      const uint2 w = *reinterpret_cast<const uint2 *>(src);
      word[0] = w.x;
      word[1] = w.y;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int u = (int)((word[i * BITS / 32] >> (i * BITS % 32)) & ((1u << BITS) - 1u));
      x[i] = s * (float)(u - (1 << (BITS - 1)));
    }
  } else if (chunk == 0 && head == 0 && a.status) {
    atomicOr(a.status, QMK_KV_BAD_ROW);
  }
  store_n<T, 8>(sd.x + (size_t)row * (size_t)sd.row_stride + (size_t)head * (size_t)sd.head_stride + 8 * chunk,
                sd.aligned, x);
}

template <typename T, bool WRITE>
int launch(const QmkKvCache *c, const QmkKvRows *r, const QmkKvTensor *k, const QmkKvTensor *v, unsigned *status,
           cudaStream_t stream) {
  Args<T> a;
  const QmkKvTensor *t[2] = {k, v};
  void *codes[2] = {c->k_codes, c->v_codes}, *scales[2] = {c->k_scales, c->v_scales};
  for (int i = 0; i < 2; ++i)
    a.side[i] = Side<T>{static_cast<uint8_t *>(codes[i]), static_cast<__nv_bfloat16 *>(scales[i]),
                        static_cast<T *>(t[i]->data), t[i]->row_stride, t[i]->head_stride, vector_aligned(t[i])};
  a.rows = device_rows(c, r);
  a.code_seq_stride = c->code_seq_stride;
  a.scale_seq_stride = c->scale_seq_stride;
  a.heads = c->num_kv_heads;
  a.capacity = c->capacity;
  a.status = status;
  const long long threads = (long long)r->rows * c->num_kv_heads * (c->head_dim / 8);
  const long long blocks = (threads + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffLL) return fail(QMK_ERR_ARGS, "qmk_kv: too many rows");
  void (*kernel)(const Args<T>) = nullptr;
  if (c->head_dim == 128) {
    if (c->bits == 4) kernel = WRITE ? write_kernel<T, 4, 128> : read_kernel<T, 4, 128>;
    else kernel = WRITE ? write_kernel<T, 8, 128> : read_kernel<T, 8, 128>;
  } else {
    if (c->bits == 4) kernel = WRITE ? write_kernel<T, 4, 64> : read_kernel<T, 4, 64>;
    else kernel = WRITE ? write_kernel<T, 8, 64> : read_kernel<T, 8, 64>;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, 2);
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
