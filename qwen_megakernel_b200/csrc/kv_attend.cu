// Causal attention over the quantized K/V cache (qmk_kv_attend; the cache
// format is in include/qwen_megakernel.h).
//
// One CTA takes one (row, q head): its 4 warps take positions 4i + w, a lane
// D / 32 dimensions, with a running maximum and sum of the softmax per warp;
// the warps' states meet in shared memory.

#include "kv_cache.cuh"

int qmk_internal_set_error(int code, const char *msg);
int qmk_internal_clear_error();

namespace qkv {

struct AttendArgs {
  const uint8_t *k_codes, *v_codes;
  const __nv_bfloat16 *k_scales, *v_scales;
  long long code_seq_stride, scale_seq_stride;
  int capacity, heads, ratio;
  Rows rows;
  const void *q;
  void *out;
  long long q_row, q_head, o_row, o_head;
  float scale_log2;
  unsigned *status;
};

template <typename T, int BITS, int D>
__global__ void __launch_bounds__(128) attend_kernel(const __grid_constant__ AttendArgs a) {
  qmk::pdl_wait();
  qmk::pdl_trigger();
  constexpr int kPer = D / 32;
  __shared__ float sm[4], sl[4], so[4][D];
  const int r = blockIdx.x, hq = blockIdx.y, h = hq / a.ratio;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int seq = 0, pos = 0;
  const int ok = locate_row(a.rows, r, seq, pos);
  if (ok == 0) return;
  if (ok < 0) {
    if (threadIdx.x == 0 && a.status) atomicOr(a.status, QMK_KV_BAD_ROW);
    pos = -1;
    seq = 0;
  }
  const T *q = static_cast<const T *>(a.q) + (size_t)r * (size_t)a.q_row + (size_t)hq * (size_t)a.q_head;
  float qf[kPer], o[kPer];
  for (int i = 0; i < kPer; ++i) {
    qf[i] = to_float(q[kPer * lane + i]) * a.scale_log2;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const size_t row0 = (size_t)h * (size_t)a.capacity;
  const uint8_t *kc = a.k_codes + (size_t)seq * (size_t)a.code_seq_stride;
  const uint8_t *vc = a.v_codes + (size_t)seq * (size_t)a.code_seq_stride;
  const __nv_bfloat16 *ks = a.k_scales + (size_t)seq * (size_t)a.scale_seq_stride;
  const __nv_bfloat16 *vs = a.v_scales + (size_t)seq * (size_t)a.scale_seq_stride;
  auto value = [&](const uint8_t *codes, const __nv_bfloat16 *scales, size_t row, int d) {
    const float s = __bfloat162float(scales[row * (D / kGroup) + d / kGroup]);
    const uint8_t *c = codes + row * (D * BITS / 8);
    const int u = BITS == 4 ? (c[d >> 1] >> (4 * (d & 1))) & 15 : c[d];
    return s * (float)(u - (1 << (BITS - 1)));
  };
  for (int j = warp; j <= pos; j += 4) {
    float s = 0.f;
    for (int i = 0; i < kPer; ++i) s += qf[i] * value(kc, ks, row0 + j, kPer * lane + i);
    s = qmk::warp_sum(s);
    const float mn = fmaxf(m, s), corr = exp2f(m - mn), p = exp2f(s - mn);
    l = l * corr + p;
    m = mn;
    for (int i = 0; i < kPer; ++i) o[i] = o[i] * corr + p * value(vc, vs, row0 + j, kPer * lane + i);
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  for (int i = 0; i < kPer; ++i) so[warp][kPer * lane + i] = o[i];
  __syncthreads();
  if (threadIdx.x < D) {
    float M = -INFINITY, L = 0.f, v = 0.f;
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sm[w]);
    for (int w = 0; w < 4; ++w) {
      const float f = sm[w] == -INFINITY ? 0.f : exp2f(sm[w] - M);
      L += sl[w] * f;
      v += so[w][threadIdx.x] * f;
    }
    static_cast<T *>(a.out)[(size_t)r * (size_t)a.o_row + (size_t)hq * (size_t)a.o_head + threadIdx.x] =
        from_float<T>(pos < 0 ? 0.f : v / L);
  }
}

template <typename T>
int launch_attend(const QmkKvCache *c, const AttendArgs &a, int q_heads, cudaStream_t stream) {
  const dim3 grid((unsigned)a.rows.rows, (unsigned)q_heads);
  if (c->head_dim == 128) {
    if (c->bits == 4) attend_kernel<T, 4, 128><<<grid, 128, 0, stream>>>(a);
    else attend_kernel<T, 8, 128><<<grid, 128, 0, stream>>>(a);
  } else {
    if (c->bits == 4) attend_kernel<T, 4, 64><<<grid, 128, 0, stream>>>(a);
    else attend_kernel<T, 8, 64><<<grid, 128, 0, stream>>>(a);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(QMK_ERR_CUDA, "qmk_kv_attend launch: %s", cudaGetErrorString(e));
  return QMK_OK;
}

}  // namespace qkv

namespace qkv {

int check_attend(const char *who, const QmkKvCache *c, const QmkKvRows *r, int num_q_heads, int dtype) {
  int rc = check_cache(who, c);
  if (rc == QMK_OK) rc = check_rows(who, c, r);
  if (rc != QMK_OK) return rc;
  if (num_q_heads < 1 || num_q_heads % c->num_kv_heads || num_q_heads / c->num_kv_heads > QMK_KV_MAX_RATIO)
    return fail(QMK_ERR_ARGS, "%s: num_q_heads=%d is not 1 .. %d times num_kv_heads=%d", who, num_q_heads,
                QMK_KV_MAX_RATIO, c->num_kv_heads);
  if (dtype != QMK_BF16 && dtype != QMK_FP16 && dtype != QMK_FP32)
    return fail(QMK_ERR_ARGS, "%s: dtype %d", who, dtype);
  return QMK_OK;
}

size_t workspace_need(const QmkKvCache *, const QmkKvRows *, int, int) { return 256; }

}  // namespace qkv

extern "C" size_t qmk_kv_attend_workspace_bytes(const QmkKvCache *cache, const QmkKvRows *rows, int num_q_heads,
                                                int dtype) {
  qmk_internal_clear_error();
  if (qkv::check_attend("qmk_kv_attend_workspace_bytes", cache, rows, num_q_heads, dtype) != QMK_OK) return 0;
  return qkv::workspace_need(cache, rows, num_q_heads, dtype);
}

extern "C" int qmk_kv_attend(const QmkKvCache *cache, const QmkKvRows *rows, const QmkKvTensor *q, int num_q_heads,
                             const QmkKvTensor *out, float scale, void *workspace, size_t workspace_bytes,
                             unsigned int *status, cudaStream_t stream) {
  using namespace qkv;
  const char *who = "qmk_kv_attend";
  qmk_internal_clear_error();
  int rc = check_attend(who, cache, rows, num_q_heads, q ? q->dtype : QMK_BF16);
  if (rc != QMK_OK) return rc;
  if (rows->rows == 0 || rows->segments == 0) return QMK_OK;
  rc = check_tensor(who, "q", q);
  if (rc == QMK_OK) rc = check_tensor(who, "out", out);
  if (rc != QMK_OK) return rc;
  if (q->dtype != out->dtype) return fail(QMK_ERR_ARGS, "%s: out has another type than q", who);
  const size_t need = workspace_need(cache, rows, num_q_heads, q->dtype);
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(QMK_ERR_WORKSPACE, "%s: workspace needs %zu bytes, 256-byte aligned", who, need);
  AttendArgs a{static_cast<const uint8_t *>(cache->k_codes), static_cast<const uint8_t *>(cache->v_codes),
               static_cast<const __nv_bfloat16 *>(cache->k_scales), static_cast<const __nv_bfloat16 *>(cache->v_scales),
               cache->code_seq_stride, cache->scale_seq_stride, cache->capacity, cache->num_kv_heads,
               num_q_heads / cache->num_kv_heads, device_rows(cache, rows), q->data, out->data, q->row_stride,
               q->head_stride, out->row_stride, out->head_stride, scale * 1.4426950408889634f, status};
  if (q->dtype == QMK_BF16) return launch_attend<__nv_bfloat16>(cache, a, num_q_heads, stream);
  if (q->dtype == QMK_FP16) return launch_attend<__half>(cache, a, num_q_heads, stream);
  return launch_attend<float>(cache, a, num_q_heads, stream);
}
