// Causal attention over the quantized K/V cache (qmk_kv_attend; the cache
// format is in include/qwen_megakernel.h).
//
// Mathematics.  A held value is s c: c the code, s the scale of its position
// and group g of 32 dimensions.  So
//   q . k_j = sum_g s_jg (sum_{d in g} q_d c_jd),   out_d = sum_j (p_j s_jg) c_jd:
// the products on the tensor cores take the CODES, as fp16, and the scales
// are applied to the fp32 partial sums (scores) or to p (values).  Decoding
// is exact: a code's bits under the exponent of 1024 are the fp16 number 1024
// + u (or 1024 + 16 u for the nibbles that lie four bits higher), u the stored
// code, and one fp16 FMA takes the offset off: 9 instructions for 8 nibbles.
// (The bits alone, as the fp16 subnormal u 2^-24, would need 5, but the tensor
// cores align products by the exponent of a subnormal operand's format, not
// of its value, and drop what lies 2^-14 below one code.)
//
// Precision: q is scaled per row by a power of two into fp16's range; bf16
// and fp16 queries lose nothing by it (elements 2^-24 below the row's
// largest aside).  p s keeps to fp16's range by taking the running maximum
// of score + e, 2^e the power of two of a tile's largest scale; it is
// rounded to fp16 (2^-11 of a term); fp32 queries are split into an fp16
// pair hi + lo on two columns of the same product, as is p s (2^-22).
// Scores, maxima, sums and outputs are fp32.

#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "kv_attend.cuh"

int qmk_internal_clear_error();

namespace qkv {

constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------- instructions
__device__ __forceinline__ void mma_f16(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                        unsigned b1, float c0, float c1, float c2, float c3) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma_acc(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                        unsigned b1) {
  mma_f16(d, a0, a1, a2, a3, b0, b1, d[0], d[1], d[2], d[3]);
}
__device__ __forceinline__ void ldmatrix4(unsigned (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(unsigned (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ unsigned transpose8(unsigned x) {
  unsigned y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ bool wait_copy(uint64_t *bar, unsigned parity) {
  uint64_t t0 = 0;
  for (unsigned it = 0;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 63u) == 63u) {
      const uint64_t now = global_timer_ns();
      if (t0 == 0) t0 = now;
      else if (now - t0 > kWaitNs) return false;
    }
  }
}

// ------------------------------------------------------------------- kernel
// Every warp is a worker of its own: it walks its range of the tile list with
// a private ring of tiles (codes by TMA, as 128-byte lines under the 128-byte
// swizzle, which leaves 8 positions of a 16-byte column free of bank conflicts
// for ldmatrix; scales by 1-D bulk copies) and a running maximum, sum and
// output in registers; warps never wait for one another.  Score product: M =
// 16 positions, N = 8 columns (query rows x heads; hi and lo apart for fp32),
// K = 16 dimensions.  Output product: M = 16 dimensions, N = the same columns,
// K = 16 positions, the code words transposed by ldmatrix, p transposed in
// registers.
//
// What bounds it: 64 sequences of 8k (601.6 MB) take 137 us, 4.4 TB/s or 0.68 of
// the measured copy rate.  16 positions of a K/V head are 2.3 KB, 100 cycles of
// an SM at that rate, and 353 warp instructions, 88 issue cycles: 144 decode,
// the rest the scales, the softmax and p.  The issue ports are busy 62 % of the
// time, the integer pipe (half rate, where decoding's masks go) 53 %.  Tiles of
// 64 positions and 12 warps of 168 registers were the best of those tried: 32
// positions 150 us, 16 warps of 128 registers 156, code rolled up over the 16
// positions 148.  A short call costs about 7 us (the plan 2, the first copies
// and queries 2, a cold first tile 1) and its merge 3.
// p is held 2^14 times too large: p s < 2^15 fits fp16, and so do its small values
constexpr float kShift = 14.f;

template <typename T, int BITS, int D, int NT>
struct Shape {
  static constexpr bool kSplit = sizeof(T) == 4;
  static constexpr int kSlots = NT * (kSplit ? 4 : 8);  // (row, head) pairs of an item
  static constexpr int kGroups = D / kGroup;
  static constexpr int kRowBytes = D * BITS / 8;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kTile = kRowBytes == 128 ? 32 : 64;  // positions
  static constexpr int kCodeBytes = kTile * kRowBytes;
  static constexpr int kScaleBytes = kTile * kGroups * 2;
  static constexpr int kTxBytes = 2 * (kCodeBytes + kScaleBytes);
  static constexpr int kStageBytes = (kTxBytes + 1023) / 1024 * 1024;
  static constexpr int kWarps = NT == 1 ? 12 : 8;
  static constexpr int kStages = std::min(6, 222 * 1024 / (kWarps * kStageBytes));
  static constexpr int kSmem = 1024 + kWarps * kStages * (kStageBytes + 8);
  static_assert(kStages >= 2 && kSmem <= 226 * 1024, "ring");
};

template <typename T, int BITS, int D, int NT>
__global__ void __launch_bounds__(32 * Shape<T, BITS, D, NT>::kWarps, 1)
    attend_kernel(const __grid_constant__ AttendArgs a) {
  using S = Shape<T, BITS, D, NT>;
  constexpr int G = S::kGroups, SL = S::kSlots, W = S::kWarps;
  constexpr bool SPLIT = S::kSplit;
  constexpr int NS = SPLIT ? 1 : 2;  // slots of a lane's two columns
  constexpr int kSteps = D / 16;     // K steps of the score product
  constexpr int kTile = S::kTile;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
  uint8_t *ring = smem + warp * S::kStages * S::kStageBytes;
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + W * S::kStages * S::kStageBytes) + warp * S::kStages;
  if (lane == 0) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  int rb, hb, head_blocks;
  block_shape(SL, a.ratio, rb, hb, head_blocks);
  pdl_wait();  // cache, queries and rows may be written by the previous kernel
  pdl_trigger();

  // ---- this warp's range: with few tiles, one each to the first warps of all CTAs
  const long long me = (long long)warp * gridDim.x + blockIdx.x;
  Range rg = find_range<kTile, 32 * W>(a.rows, rb, a.heads * head_blocks, (long long)gridDim.x * W, me);
  int *desc = a.desc + me * kDescWords;
  if (lane == 0) desc[0] = 0;
  if (rg.u0 >= rg.u1) return;
  Segment sg = load_segment<kTile>(a.rows, rg.b, rb);

  const Decode dec(BITS);
  const uint64_t pol = l2_policy_evict_first();
  // this lane's ldmatrix address within 16 positions (position lane % 16, chunk lane / 16)
  constexpr int kPerLine = 128 / S::kRowBytes;
  const int lr = lane & 15;
  const uint32_t frag = (lr / kPerLine) * 128 +
                        ((((lr % kPerLine) * S::kChunks + (lane >> 4)) ^ ((lr / kPerLine) & 7)) << 4);
  unsigned issued = 0, used = 0;  // ring positions
  bool dead = false;              // a wait ran out

  while (rg.u0 < rg.u1 && !dead) {
    const Item it = next_item<kTile>(a.rows, rg, sg, rb, hb, head_blocks, a.heads);
    const int h = it.h, head0 = it.head0, row0 = it.row0, nrows = it.nrows, ok_rows = it.ok_rows, len = it.len;
    const int t_lo = it.t_lo, nt = len > 0 ? it.t_hi - t_lo : 0;  // tiles to read
    const size_t sc_at =
        (size_t)(len ? sg.seq : 0) * (size_t)a.scale_seq_stride + (size_t)h * (size_t)a.capacity * G;
    auto issue = [&](int i) {  // the i-th tile of the item (lane 0)
      const int st = issued % S::kStages, pos = (t_lo + i) * kTile;
      uint8_t *dst = ring + st * S::kStageBytes;
      mbar_arrive_expect_tx(&full[st], S::kTxBytes);
      tma_load_4d(dst, &a.k_map, 0, pos / kPerLine, h, sg.seq, &full[st]);
      tma_load_4d(dst + S::kCodeBytes, &a.v_map, 0, pos / kPerLine, h, sg.seq, &full[st]);
      bulk_g2s(dst + 2 * S::kCodeBytes, a.k_scales + sc_at + (size_t)pos * G, S::kScaleBytes, &full[st], pol);
      bulk_g2s(dst + 2 * S::kCodeBytes + S::kScaleBytes, a.v_scales + sc_at + (size_t)pos * G, S::kScaleBytes,
               &full[st], pol);
    };
    for (int i = 0; i < min(nt, S::kStages); ++i) {
      if (lane == 0) issue(i);
      ++issued;
    }

    // ---- queries: the B operand of the score product, column n = gid
    unsigned qb[NT][kSteps][2];
    float cmul[NT][NS];  // score factor of this lane's slots
    int lim[NT][NS];     // positions that the slot's row sees
    auto slot_stored = [&](int slot) {
      return slot < rb * hb && slot / hb < nrows && head0 + slot % hb < a.ratio;
    };
    auto slot_limit = [&](int slot) {
      const int i = slot / hb;
      if (i >= nrows || slot >= rb * hb) return len;  // no row: never stored
      return i < ok_rows ? sg.start + row0 + i + 1 : 0;
    };
    auto slot_offset = [&](int slot, long long row_stride, long long head_stride) {
      return (size_t)(sg.r0 + row0 + slot / hb) * (size_t)row_stride +
             (size_t)(h * a.ratio + head0 + slot % hb) * (size_t)head_stride;
    };
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int slot = SPLIT ? 4 * t + (gid >> 1) : 8 * t + gid;
      const bool lo_half = SPLIT && (gid & 1);
      float x[kSteps][4];
      float top = 0.f;
      const T *qp = static_cast<const T *>(a.q) + slot_offset(slot, a.q_row, a.q_head);
      const bool have = slot_stored(slot) && slot / hb < ok_rows;
      if constexpr (BITS == 4) {
        // word tig of group g: dimensions 32 g + 8 tig + (0 .. 7)
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          if (have) load_n<T, 8>(qp + 32 * g + 8 * tig, a.q_aligned, y);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            x[2 * g + i][0] = y[2 * i];
            x[2 * g + i][1] = y[2 * i + 4];
            x[2 * g + i][2] = y[2 * i + 1];
            x[2 * g + i][3] = y[2 * i + 5];
          }
        }
      } else {
        // word tig of 16-byte chunk c: dimensions 16 c + 4 tig + (0 .. 3)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          float y[4] = {0.f, 0.f, 0.f, 0.f};
          if (have) {
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = to_float(qp[16 * s + 4 * tig + i]);
          }
          x[s][0] = y[0];
          x[s][1] = y[2];
          x[s][2] = y[1];
          x[s][3] = y[3];
        }
      }
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(x[s][i]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // scale the row so that its largest element lies in [2^12, 2^13)
      const int fe = min(254, 266 - (int)((__float_as_uint(top) >> 23) & 255u));
      // (with the softmax scale's sign, so that the factor of the products is > 0)
      const float f = copysignf(__uint_as_float((unsigned)fe << 23), a.scale_log2);
      const float finv = __uint_as_float((unsigned)(254 - fe) << 23);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[i] = x[s][i] * f;
          if (lo_half) y[i] -= f16_round(y[i]);
        }
        qb[t][s][0] = pack_f16(y[0], y[1]);
        qb[t][s][1] = pack_f16(y[2], y[3]);
      }
      // column n's factor sits in lanes 4 n ..; the accumulators hold columns 2 tig, 2 tig + 1
      const float cm = fmaxf(fabsf(a.scale_log2) * finv, 1e-37f);
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        cmul[t][i] = __shfl_sync(0xffffffffu, cm, 8 * tig + 4 * i);
        lim[t][i] = slot_limit(SPLIT ? 4 * t + tig : 8 * t + 2 * tig + i);
      }
    }
    const int seen_by_all = it.seen_by_all();
    float m[NT][NS], l[NT][NS];
    float acc[NT][G][2][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        m[t][i] = -INFINITY;
        l[t][i] = 0.f;
      }
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][g][0][i] = acc[t][g][1][i] = 0.f;
    }

    for (int i = 0; i < nt; ++i) {
      const int st = used % S::kStages;
      if (!__all_sync(0xffffffffu, wait_copy(&full[st], (used / S::kStages) & 1))) {
        dead = true;
        break;
      }
      ++used;
      const int pos0 = (t_lo + i) * kTile;
      uint8_t *stage = ring + st * S::kStageBytes;
      if (pos0 + kTile > len) {
        // the scales of positions that no row sees may hold anything: zero
        for (int p = (len - pos0) * G + lane; p < kTile * G; p += 32) {
          reinterpret_cast<__nv_bfloat16 *>(stage + 2 * S::kCodeBytes)[p] = __float2bfloat16_rn(0.f);
          reinterpret_cast<__nv_bfloat16 *>(stage + 2 * S::kCodeBytes + S::kScaleBytes)[p] = __float2bfloat16_rn(0.f);
        }
        fence_proxy_async_smem();  // before a later copy into this stage
        __syncwarp();
      }
#pragma unroll 1
      for (int half = 0; half < kTile / 32; ++half) {  // 32 positions
        const int p0 = 32 * half;
        const uint32_t kb = smem_addr(stage) + p0 * S::kRowBytes, vb = kb + S::kCodeBytes;
        const uint8_t *ksc = stage + 2 * S::kCodeBytes + (p0 + gid) * (G * 2), *vsc = ksc + S::kScaleBytes;
        // products q . k over the factor cmul: [16 positions][tile][row gid, gid + 8][slot]; then p
        float x[2][NT][2][NS];
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
          float sc[2][G];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint8_t *p = ksc + (16 * sub + 8 * r) * (G * 2);
            if constexpr (G == 4) {
              const uint2 w = *reinterpret_cast<const uint2 *>(p);
              sc[r][0] = bf_lo(w.x), sc[r][1] = bf_hi(w.x), sc[r][2] = bf_lo(w.y), sc[r][3] = bf_hi(w.y);
            } else {
              const unsigned w = *reinterpret_cast<const unsigned *>(p);
              sc[r][0] = bf_lo(w), sc[r][1] = bf_hi(w);
            }
          }
          float s[NT][4];
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[t][k] = 0.f;
#pragma unroll
          for (int c2 = 0; c2 < S::kChunks; c2 += 2) {
            unsigned w[4];  // chunk c2: rows gid, gid + 8; chunk c2 + 1: the same
            ldmatrix4(w, (kb + 16 * sub * S::kRowBytes + frag) ^ ((c2 ^ (kPerLine == 4 ? 4 * (sub & 1) : 0)) << 4));
            if constexpr (BITS == 4) {
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const int g = c2 + k;
                unsigned ha[4], hs[4];  // rows gid, gid + 8
                dec.nibbles(w[2 * k], ha);
                dec.nibbles(w[2 * k + 1], hs);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                  float cc[4];
                  mma_f16(cc, ha[0], hs[0], ha[1], hs[1], qb[t][2 * g][0], qb[t][2 * g][1], 0.f, 0.f, 0.f, 0.f);
                  mma_acc(cc, ha[2], hs[2], ha[3], hs[3], qb[t][2 * g + 1][0], qb[t][2 * g + 1][1]);
#pragma unroll
                  for (int e = 0; e < 4; ++e) s[t][e] = fmaf(sc[e >> 1][g], cc[e], s[t][e]);
                }
              }
            } else {
              const int g = c2 / 2;
              unsigned hd[4][2];
#pragma unroll
              for (int k = 0; k < 4; ++k) dec.bytes(w[k], hd[k]);
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                float cc[4];
                mma_f16(cc, hd[0][0], hd[1][0], hd[0][1], hd[1][1], qb[t][c2][0], qb[t][c2][1], 0.f, 0.f, 0.f, 0.f);
                mma_acc(cc, hd[2][0], hd[3][0], hd[2][1], hd[3][1], qb[t][c2 + 1][0], qb[t][c2 + 1][1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][e] = fmaf(sc[e >> 1][g], cc[e], s[t][e]);
              }
            }
          }
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              if constexpr (SPLIT) {
                x[sub][t][r][0] = s[t][2 * r] + s[t][2 * r + 1];
              } else {
                x[sub][t][r][0] = s[t][2 * r];
                x[sub][t][r][1] = s[t][2 * r + 1];
              }
            }
        }
        if (pos0 + p0 + 32 > seen_by_all) {
#pragma unroll
          for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int k = 0; k < NS; ++k)
                  if (pos0 + p0 + 16 * sub + 8 * r + gid >= lim[t][k]) x[sub][t][r][k] = -INFINITY;
        }
        // V scales of this lane's positions, and the exponent of the largest
        uint2 vw[2][2];
        unsigned vmax = 0;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint8_t *p = vsc + (16 * sub + 8 * r) * (G * 2);
            if constexpr (G == 4) vw[sub][r] = *reinterpret_cast<const uint2 *>(p);
            else vw[sub][r] = make_uint2(*reinterpret_cast<const unsigned *>(p), 0u);
            vmax = max_u16x2(vmax, max_u16x2(vw[sub][r].x, vw[sub][r].y));
          }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) vmax = max_u16x2(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
        // 2^40 either way: beyond it p s leaves fp16's range or p leaves fp32's
        const int ve = min(max((int)(max(vmax & 0xffffu, vmax >> 16) >> 7), 127 - 40), 127 + 40);
        const float vexp = (float)(ve - 127);
        float corr[NT][NS];
        bool moved = false;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            float mx = fmaxf(fmaxf(x[0][t][0][i], x[0][t][1][i]), fmaxf(x[1][t][0][i], x[1][t][1][i]));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            // m: running maximum of score + e; -inf: nothing seen yet
            const float mn = fmaxf(m[t][i], fmaf(mx, cmul[t][i], vexp));
            const float ref = mn == -INFINITY ? 0.f : mn;
            corr[t][i] = fast_exp2(m[t][i] - ref);
            moved |= mn != m[t][i];
            m[t][i] = mn;
            float sum = 0.f;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                x[sub][t][r][i] = fast_exp2(fmaf(x[sub][t][r][i], cmul[t][i], kShift - ref));
                sum += x[sub][t][r][i];
              }
            l[t][i] = fmaf(l[t][i], corr[t][i], sum);
          }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float cr = corr[t][NS == 1 ? 0 : (e & 1)];
                acc[t][g][0][e] *= cr;
                acc[t][g][1][e] *= cr;
              }
        }
        // outputs
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
          float sv[2][4];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            sv[r][0] = bf_lo(vw[sub][r].x);
            sv[r][1] = bf_hi(vw[sub][r].x);
            sv[r][2] = bf_lo(vw[sub][r].y);
            sv[r][3] = bf_hi(vw[sub][r].y);
          }
          auto p_frag = [&](int t, int g, unsigned (&pb)[2]) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float y0 = x[sub][t][r][0] * sv[r][g];
              const float y1 = SPLIT ? y0 - f16_round(y0) : x[sub][t][r][NS - 1] * sv[r][g];
              pb[r] = transpose8(pack_f16(y0, y1));
            }
          };
#pragma unroll
          for (int c2 = 0; c2 < S::kChunks; c2 += 2) {
            unsigned w[4];  // chunk c2: positions 0-7, 8-15; chunk c2 + 1: the same
            ldmatrix4_trans(w,
                            (vb + 16 * sub * S::kRowBytes + frag) ^ ((c2 ^ (kPerLine == 4 ? 4 * (sub & 1) : 0)) << 4));
            if constexpr (BITS == 4) {
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const int g = c2 + k;
                unsigned ha[4], hs[4];  // positions 0-7, 8-15
                dec.nibbles(w[2 * k], ha);
                dec.nibbles(w[2 * k + 1], hs);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                  unsigned pb[2];
                  p_frag(t, g, pb);
                  mma_acc(acc[t][g][0], ha[0], ha[1], hs[0], hs[1], pb[0], pb[1]);
                  mma_acc(acc[t][g][1], ha[2], ha[3], hs[2], hs[3], pb[0], pb[1]);
                }
              }
            } else {
              const int g = c2 / 2;
              unsigned hd[4][2];
#pragma unroll
              for (int k = 0; k < 4; ++k) dec.bytes(w[k], hd[k]);
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                unsigned pb[2];
                p_frag(t, g, pb);
                mma_acc(acc[t][g][0], hd[0][0], hd[0][1], hd[1][0], hd[1][1], pb[0], pb[1]);
                mma_acc(acc[t][g][1], hd[2][0], hd[2][1], hd[3][0], hd[3][1], pb[0], pb[1]);
              }
            }
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      if (i + S::kStages < nt) {
        if (lane == 0) issue(i + S::kStages);
        ++issued;
      }
    }

    // ---- the item's rows, or the part of them that this range holds
    const bool whole = it.whole(), head_part = t_lo == 0;
    if (lane == 0) {
      if (!whole && head_part) describe_cut(desc, it, sg, rg, me, a.ratio, hb);
      if (ok_rows < nrows && a.status) atomicOr(a.status, QMK_KV_BAD_ROW);
    }
    float *part = a.parts + (size_t)(me * 2 + (head_part ? 0 : 1)) * SL * (D + 4);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], o);
        const int slot = SPLIT ? 4 * t + tig : 8 * t + 2 * tig + i;
        if (!slot_stored(slot)) continue;
        const float inv = whole ? (l[t][i] == 0.f ? 0.f : 1.f / l[t][i]) : 1.f;  // 0: the row sees nothing
        float *dst = part + slot * (D + 4);
        T *o = static_cast<T *>(a.out) + slot_offset(slot, a.o_row, a.o_head);
        if (!whole && gid == 0) *reinterpret_cast<float2 *>(dst + D) = make_float2(m[t][i], l[t][i]);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            // 4 bits: dimensions 32 g + 4 gid + 2 k + (0, 1); 8 bits: 32 g + 16 k + 2 gid + (0, 1)
            const int d = 32 * g + (BITS == 4 ? 4 * gid + 2 * k : 16 * k + 2 * gid);
            const float *v = acc[t][g][k];
            const float y0 = (SPLIT ? v[0] + v[1] : v[i]) * inv, y1 = (SPLIT ? v[2] + v[3] : v[2 + i]) * inv;
            if (whole) {
              o[d] = from_float<T>(y0);
              o[d + 1] = from_float<T>(y1);
            } else {
              *reinterpret_cast<float2 *>(dst + d) = make_float2(y0, y1);
            }
          }
      }
    }
  }
  if (dead && lane == 0) {
    if (a.status) atomicOr(a.status, QMK_KV_TIMEOUT);
    // copies in flight must land before this shared memory goes away
    bool drained = true;
    for (; used != issued; ++used) drained &= wait_copy(&full[used % S::kStages], (used / S::kStages) & 1);
    if (!drained && a.status) atomicOr(a.status, QMK_KV_COPIES_PENDING);
  }
}

// Joins the parts of items that were cut: CTA x takes the items whose first
// tile is in the range of one of its workers and that go on in the next
// ranges, grid y shares their rows.  A warp takes an output row, or several
// share one (few rows mean many parts, 222 a row for one stream of 32k);
// kMergeBatch parts are loaded at a time.  What it takes is latency: of the
// descriptor, of a round of parts, of the warps' sums.
constexpr int kMergeWarps = 8, kMergeBatch = 4;

template <typename T, int D>
__global__ void __launch_bounds__(32 * kMergeWarps, 4) merge_kernel(const int *__restrict__ desc,
                                                                    const float *__restrict__ parts, int workers,
                                                                    int slots, void *out, long long o_row,
                                                                    long long o_head) {
  pdl_wait();  // the parts are written by the attention kernel
  pdl_trigger();
  __shared__ float s_ml[kMergeWarps][2];
  __shared__ float s_o[kMergeWarps][D];
  constexpr int kPer = D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the CTA's workers, a lane each (the host keeps them to 32); neighbours, for
  // heads of long items lie a regular distance apart
  const int per = (workers + gridDim.x - 1) / gridDim.x, mine = blockIdx.x * per + lane;
  const int np_mine = lane < per && mine < workers ? __ldcg(desc + (size_t)mine * kDescWords) : 0;
  for (unsigned todo = __ballot_sync(0xffffffffu, np_mine > 0); todo; todo &= todo - 1) {
    const int src = __ffs(todo) - 1, c = blockIdx.x * per + src;
    const int np = __shfl_sync(0xffffffffu, np_mine, src);
    const int *dd = desc + (size_t)c * kDescWords;
    const int4 d4 = __ldcg(reinterpret_cast<const int4 *>(dd + 4));
    const int row0 = d4.x, nrows = d4.y, head0 = d4.z, nheads = d4.w & 0xffff, hb = d4.w >> 16, n = nrows * nheads;
    // rows [v_lo, v_hi) of this CTA; `share` warps a row
    const int each = (n + gridDim.y - 1) / gridDim.y, v_lo = blockIdx.y * each, v_hi = min(n, v_lo + each);
    const int share = each >= kMergeWarps ? 1 : kMergeWarps / each, at_once = kMergeWarps / share;
    for (int v0 = v_lo; v0 < v_hi; v0 += at_once) {
      const int v = v0 + warp / share, first = warp % share;
      const bool live = v < v_hi && warp < share * at_once;
      const int i = live ? v / nheads : 0, j = live ? v % nheads : 0;
      // part k: worker c + k's, the head part first
      const float *p0 = parts + ((size_t)c * 2 * slots + i * hb + j) * (D + 4) + kPer * lane;
      const size_t step = (size_t)2 * slots * (D + 4), tail = (size_t)slots * (D + 4);
      float M = -INFINITY, L = 0.f, y[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) y[e] = 0.f;
      for (int k0 = first; live && k0 < np; k0 += kMergeBatch * share) {
        float2 ml[kMergeBatch];
        float x[kMergeBatch][kPer];
#pragma unroll
        for (int q = 0; q < kMergeBatch; ++q) {
          // (the last part again rather than a branch round each load)
          const int k = min(k0 + q * share, np - 1);
          const float *p = p0 + k * step + (k == 0 ? 0 : tail);
          ml[q] = __ldcg(reinterpret_cast<const float2 *>(p - kPer * lane + D));
          if constexpr (kPer == 4) *reinterpret_cast<float4 *>(x[q]) = __ldcg(reinterpret_cast<const float4 *>(p));
          else *reinterpret_cast<float2 *>(x[q]) = __ldcg(reinterpret_cast<const float2 *>(p));
        }
        float mn = M;
#pragma unroll
        for (int q = 0; q < kMergeBatch; ++q) mn = fmaxf(mn, ml[q].x);
        const float ref = mn == -INFINITY ? 0.f : mn, corr = fast_exp2(M - ref);
        M = mn;
        L *= corr;
#pragma unroll
        for (int e = 0; e < kPer; ++e) y[e] *= corr;
#pragma unroll
        for (int q = 0; q < kMergeBatch; ++q) {
          // (0 times a NaN state: NaN)
          const float w = fast_exp2(ml[q].x - ref) * (k0 + q * share < np ? 1.f : 0.f);
          L = fmaf(w, ml[q].y, L);
#pragma unroll
          for (int e = 0; e < kPer; ++e) y[e] = fmaf(w, x[q][e], y[e]);
        }
      }
      if (share > 1) {
        __syncthreads();  // the last row's sums have been read
        if (lane == 0) {
          s_ml[warp][0] = M;
          s_ml[warp][1] = L;
        }
#pragma unroll
        for (int e = 0; e < kPer; ++e) s_o[warp][kPer * lane + e] = y[e];
        __syncthreads();
        if (live && first == 0) {
          float mn = M;
          for (int w = 1; w < share; ++w) mn = fmaxf(mn, s_ml[warp + w][0]);
          const float ref = mn == -INFINITY ? 0.f : mn, corr = fast_exp2(M - ref);
          L *= corr;
#pragma unroll
          for (int e = 0; e < kPer; ++e) y[e] *= corr;
          for (int w = 1; w < share; ++w) {
            const float f = fast_exp2(s_ml[warp + w][0] - ref);
            L = fmaf(f, s_ml[warp + w][1], L);
#pragma unroll
            for (int e = 0; e < kPer; ++e) y[e] = fmaf(f, s_o[warp + w][kPer * lane + e], y[e]);
          }
        }
      }
      if (live && first == 0) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        T *o = static_cast<T *>(out) + (size_t)(row0 + i) * (size_t)o_row + (size_t)(head0 + j) * (size_t)o_head;
#pragma unroll
        for (int e = 0; e < kPer; ++e) o[kPer * lane + e] = from_float<T>(y[e] * inv);
      }
    }
  }
}

// ---------------------------------------------------------------- host side
constexpr int kMaxDevices = 64;
constexpr int kMaxSms = 160;
constexpr int kMaxWorkers = 12 * kMaxSms;
constexpr size_t kDescBytes = ((size_t)kMaxWorkers * kDescWords * 4 + 255) / 256 * 256;

std::mutex g_mutex;

int encode_codes(CUtensorMap *m, const QmkKvCache *c, void *codes, int tile) {
  static PFN_cuTensorMapEncodeTiled_v12000 enc = nullptr;
  {
    std::lock_guard<std::mutex> lock(g_mutex);
    if (!enc) {
      void *fn = nullptr;
      cudaDriverEntryPointQueryResult r;
      const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &r);
      if (e != cudaSuccess || r != cudaDriverEntryPointSuccess || !fn)
        return fail(QMK_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
      enc = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    }
  }
  // rows of 32, 64 or 128 bytes as lines of 128, boxes of `tile` positions
  const cuuint64_t row = (cuuint64_t)c->head_dim * c->bits / 8, head = row * c->capacity;
  const cuuint64_t seq = c->num_seqs > 1 ? (cuuint64_t)c->code_seq_stride : head * c->num_kv_heads;
  const cuuint64_t dims[4] = {128, head / 128, (cuuint64_t)c->num_kv_heads, (cuuint64_t)c->num_seqs};
  const cuuint64_t strides[3] = {128, head, seq};
  const cuuint32_t box[4] = {128, (cuuint32_t)(tile * row / 128), 1, 1}, one[4] = {1, 1, 1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, codes, dims, strides, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(QMK_ERR_ARGS, "cuTensorMapEncodeTiled rejected the cache");
  return QMK_OK;
}

template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, int block, size_t smem, cudaStream_t stream,
                       const Args &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Slots an item holds: one N = 8 tile, or two where the segments' rows and
// heads fill more than two (an item of two decodes the cache once for both, but
// its warps need 255 registers, 8 to an SM).  Measured, us with one / two tiles
// an item, 4 bits x 128, 2 q heads a K/V head, 4000 positions:
//   1 sequence    10 columns 18.3 / 25.6   16: 19.0 / 26.0   32: 24.1 / 27.7
//   16 sequences  10 columns 45.1 / 44.3   16: 46.0 / 46.1   32: 81.5 / 69.8
int tiles_n(int dtype, int max_rows, int ratio) {
  return (long long)max_rows * ratio > (dtype == QMK_FP32 ? 8 : 16) ? 2 : 1;
}
int slots_of(int dtype, int nt) { return nt * (dtype == QMK_FP32 ? 4 : 8); }

// Where the tcgen05 kernel takes over: its lines come in 128s and cost the same
// however few are used, the warps' kernel decodes the cache again for every 16
// columns.  Measured as above, us of the warps' / the tcgen05 kernel:
//   1 sequence    32 columns 27.7 / 30.1   64: 28.3 / 31.2   128: 38.9 / 32.0
//   16 sequences  32 columns 69.8 / 106    64: 119 / 107     128: 217 / 106
bool use_tc(int dtype, int max_rows, int ratio) { return dtype != QMK_FP32 && (long long)max_rows * ratio >= 64; }

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

size_t workspace_need(const QmkKvCache *c, const QmkKvRows *r, int num_q_heads, int dtype) {
  const int ratio = num_q_heads / c->num_kv_heads;
  const bool tc = use_tc(dtype, r->max_rows, ratio);
  const int slots = tc ? kTcLines : slots_of(dtype, tiles_n(dtype, r->max_rows, ratio));
  const size_t parts = (size_t)(tc ? kMaxSms : kMaxWorkers) * 2 * slots * (c->head_dim + 4) * 4;
  return kDescBytes + (parts + 255) / 256 * 256;
}

// Nothing is cut where no sequence can be longer than a tile.
template <typename T, int D>
cudaError_t launch_merge(const AttendArgs &a, int tile, int workers, int slots, int sms, cudaStream_t stream) {
  if (a.rows.max_seq_len <= tile) return cudaSuccess;
  const int grid = std::max((workers + 31) / 32, std::min(workers, 3 * sms));
  return launch_pdl(merge_kernel<T, D>, dim3(grid, slots > 16 ? 16 : 2), 32 * kMergeWarps, 0, stream,
                    (const int *)a.desc, (const float *)a.parts, workers, slots, a.out, a.o_row, a.o_head);
}

template <typename T, int BITS, int D, int NT>
int launch_attend(AttendArgs &a, int sms, int dev, cudaStream_t stream) {
  using S = Shape<T, BITS, D, NT>;
  static bool ready[kMaxDevices] = {};
  {
    std::lock_guard<std::mutex> lock(g_mutex);
    if (!ready[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(attend_kernel<T, BITS, D, NT>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
      if (e != cudaSuccess) return fail(QMK_ERR_CUDA, "qmk_kv_attend shared memory: %s", cudaGetErrorString(e));
      ready[dev] = true;
    }
  }
  cudaError_t e = launch_pdl(attend_kernel<T, BITS, D, NT>, dim3(sms), 32 * S::kWarps, S::kSmem, stream, a);
  if (e == cudaSuccess) e = launch_merge<T, D>(a, S::kTile, sms * S::kWarps, S::kSlots, sms, stream);
  if (e != cudaSuccess) return fail(QMK_ERR_CUDA, "qmk_kv_attend launch: %s", cudaGetErrorString(e));
  return QMK_OK;
}

template <typename T>
int launch_tc_attend(const QmkKvCache *c, AttendArgs &a, int dtype, int sms, int dev, cudaStream_t stream) {
  cudaError_t e = attend_tc(a, dtype, c->bits, c->head_dim, sms, dev, stream);
  if (e == cudaSuccess)
    e = c->head_dim == 128 ? launch_merge<T, 128>(a, 128, sms, kTcLines, sms, stream)
                           : launch_merge<T, 64>(a, 128, sms, kTcLines, sms, stream);
  if (e != cudaSuccess) return fail(QMK_ERR_CUDA, "qmk_kv_attend launch: %s", cudaGetErrorString(e));
  return QMK_OK;
}

template <typename T, int BITS, int D>
int pick_tiles(AttendArgs &a, int nt, int sms, int dev, cudaStream_t stream) {
  return nt == 1 ? launch_attend<T, BITS, D, 1>(a, sms, dev, stream) : launch_attend<T, BITS, D, 2>(a, sms, dev, stream);
}

template <typename T>
int pick_format(const QmkKvCache *c, AttendArgs &a, int nt, int sms, int dev, cudaStream_t stream) {
  if (c->head_dim == 128)
    return c->bits == 4 ? pick_tiles<T, 4, 128>(a, nt, sms, dev, stream) : pick_tiles<T, 8, 128>(a, nt, sms, dev, stream);
  return c->bits == 4 ? pick_tiles<T, 4, 64>(a, nt, sms, dev, stream) : pick_tiles<T, 8, 64>(a, nt, sms, dev, stream);
}

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
  if (!(fabsf(scale) < INFINITY)) return fail(QMK_ERR_ARGS, "%s: scale is not finite", who);
  const size_t need = workspace_need(cache, rows, num_q_heads, q->dtype);
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(QMK_ERR_WORKSPACE, "%s: workspace needs %zu bytes, 256-byte aligned", who, need);
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev < 0 || dev >= kMaxDevices)) e = cudaErrorInvalidDevice;
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return fail(QMK_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  sms = std::min(sms, kMaxSms);
  AttendArgs a;
  const bool tc = use_tc(q->dtype, rows->max_rows, num_q_heads / cache->num_kv_heads);
  const int tile = tc ? 128 : cache->head_dim * cache->bits == 1024 ? 32 : 64;  // Shape::kTile
  rc = encode_codes(&a.k_map, cache, cache->k_codes, tile);
  if (rc == QMK_OK) rc = encode_codes(&a.v_map, cache, cache->v_codes, tile);
  if (rc != QMK_OK) return rc;
  a.k_scales = static_cast<const __nv_bfloat16 *>(cache->k_scales);
  a.v_scales = static_cast<const __nv_bfloat16 *>(cache->v_scales);
  a.scale_seq_stride = cache->scale_seq_stride;
  a.capacity = cache->capacity;
  a.heads = cache->num_kv_heads;
  a.ratio = num_q_heads / cache->num_kv_heads;
  a.rows = device_rows(cache, rows);
  a.q = q->data;
  a.out = out->data;
  a.q_row = q->row_stride;
  a.q_head = q->head_stride;
  a.o_row = out->row_stride;
  a.o_head = out->head_stride;
  a.q_aligned = vector_aligned(q);
  a.o_aligned = vector_aligned(out);
  a.scale_log2 = scale * kLog2e;
  a.desc = static_cast<int *>(workspace);
  a.parts = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + kDescBytes);
  a.status = status;
  if (tc)
    return q->dtype == QMK_BF16 ? launch_tc_attend<__nv_bfloat16>(cache, a, QMK_BF16, sms, dev, stream)
                                : launch_tc_attend<__half>(cache, a, QMK_FP16, sms, dev, stream);
  const int nt = tiles_n(q->dtype, rows->max_rows, a.ratio);
  if (q->dtype == QMK_BF16) return pick_format<__nv_bfloat16>(cache, a, nt, sms, dev, stream);
  if (q->dtype == QMK_FP16) return pick_format<__half>(cache, a, nt, sms, dev, stream);
  return pick_format<float>(cache, a, nt, sms, dev, stream);
}
