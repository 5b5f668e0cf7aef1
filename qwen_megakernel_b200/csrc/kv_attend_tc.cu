// Causal attention over the quantized K/V cache for many query rows (prompts,
// chunks of prompts): tcgen05 tiles.  The same operator as kv_attend.cu's
// kernel (qmk_kv_attend picks), for bf16 and fp16 queries.
//
// An item is 128 query lines (rows x the q heads of one K/V head) against
// tiles of 128 positions.  Per tile: codes and scales arrive by TMA; eight
// warps decode K and V to fp16 in shared memory, s c 2^-E with E the exponent
// of the tile's largest scale, which is exact for 4-bit codes (8 + 3
// significant bits) and rounds 8-bit ones to 11 bits; S = Q K^T (128 x 128,
// fp32 in TMEM); four warps, a thread a line, take the softmax and write P as
// fp16 to TMEM; O += P V with P as the TMEM operand and V in its natural
// layout (dimensions contiguous: an MN-major operand).  Queries are scaled per
// line by a power of two (exact), P by 2^7 so that small probabilities keep
// fp16's precision.  The running reference R of a line's exponents moves only
// when its maximum grows past R + 8 (P < 2^15 then), so O is rescaled rarely.
// Dimensions are held in the order that decoding leaves them in, in Q, K and
// V alike, and put back when O is stored.
//
// Work division, parts and their merge are those of kv_attend.cu, a CTA being
// one worker.  Warps: 0 TMA, 1 MMA issue, 2-5 softmax and output, 6-9 decode
// K, 10-13 decode V; S, P and the decoded tiles are double-buffered, so the
// products of one tile overlap the softmax of another and the decoding of a
// third.  Every wait is bounded (QMK_KV_TIMEOUT).

#include <algorithm>
#include <mutex>

#include "kv_attend.cuh"

namespace qkv {

namespace {

constexpr int kLines = 128;    // query lines of an item (MMA M)
constexpr int kPos = 128;      // positions of a tile
constexpr int kTcThreads = 448;
constexpr float kTcShift = 7.f;   // P is held 2^7 times too large
constexpr float kTcSlack = 8.f;   // R follows a line's maximum when it is 2^8 behind
constexpr uint32_t kColS = 0, kColO = 256, kColP = 384;  // TMEM columns: S 2 x 128, O 128, P 2 x 64

template <int BITS, int D>
struct TcShape {
  static constexpr int kRowBytes = D * BITS / 8;
  static constexpr int kGroups = D / kGroup;
  static constexpr int kCodeBytes = kPos * kRowBytes;
  static constexpr int kScaleBytes = kPos * kGroups * 2;
  static constexpr int kRawBytes = kCodeBytes + kScaleBytes;           // of K or V
  static constexpr int kRawStages = kRowBytes == 128 ? 1 : 2;
  static constexpr int kTileBytes = kPos * D * 2;                      // fp16, two halves of 64 dimensions (one)
  static constexpr int kQ = 0, kK = kLines * D * 2, kV = kK + 2 * kTileBytes, kRaw = kV + 2 * kTileBytes;
  static constexpr int kRawSlot = (kRawBytes + 1023) / 1024 * 1024;
  static constexpr int kBars = kRaw + 2 * kRawStages * kRawSlot;
  static constexpr int kSmem = 1024 + kBars + 512;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

struct TcBars {
  uint64_t raw_full[2][2], raw_empty[2][2];    // [K, V][stage]
  uint64_t tile_full[2][2], k_empty[2];        // decoded [K, V][buffer]; K read by the MMA
  uint64_t s_full[2], s_empty[2];
  uint64_t p_full[2], pv[2];                   // pv: P V of a tile done: V, P and O are free to touch
  uint64_t q_full, exps[4], drain;
  float exp_k[4], exp_v[4];                    // 2^E of K and E of V, of tile t in slot t % 4
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(TcBars) <= 512, "barrier area");

__device__ __forceinline__ void mma_ts_warp(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// MN-major operand under the 128-byte swizzle: 64 elements of N in a 128-byte
// row, 8 rows of K in a 1024-byte atom; `lbo` bytes between atoms along N,
// 1024 along K.
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// Bounded wait of a whole warp; false on timeout (which aborts the CTA) or abort.
__device__ __forceinline__ bool wait_warp(uint64_t *bar, unsigned parity, volatile int *abort) {
  bool ok = false;
  uint64_t t0 = 0;
  for (unsigned it = 0;; ++it) {
    if (mbar_try_wait(bar, parity)) {
      ok = true;
      break;
    }
    if ((it & 63u) == 63u) {
      if (*abort) break;
      const uint64_t now = global_timer_ns();
      if (t0 == 0) {
        t0 = now;
      } else if (now - t0 > kWaitNs) {
        *abort = 1;
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// Element `slot` of 8 stored dimensions is dimension order(slot): what the
// decoding of a word's halves leaves.
template <int BITS>
__host__ __device__ constexpr int order(int slot) {
  return BITS == 4 ? (slot >> 1) + 4 * (slot & 1) : (slot & 4) + ((slot >> 1) & 1) + 2 * (slot & 1);
}

template <typename T, int BITS, int D>
__global__ void __launch_bounds__(kTcThreads, 1) attend_tc_kernel(const __grid_constant__ AttendArgs a) {
  using S = TcShape<BITS, D>;
  constexpr int G = S::kGroups, RS = S::kRawStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcBars &B = *reinterpret_cast<TcBars *>(smem + S::kBars);
  volatile int *abort = &B.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      for (int j = 0; j < 2; ++j) {
        mbar_init(&B.raw_full[i][j], 1);
        mbar_init(&B.raw_empty[i][j], 4);
        mbar_init(&B.tile_full[i][j], 4);
      }
      mbar_init(&B.k_empty[i], 1);
      mbar_init(&B.s_full[i], 1);
      mbar_init(&B.s_empty[i], 4);
      mbar_init(&B.p_full[i], 4);
      mbar_init(&B.pv[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&B.exps[i], 2);
    mbar_init(&B.q_full, 4);
    mbar_init(&B.drain, 1);
    fence_mbar_init();
    B.abort = 0;
  }
  if (warp == 0) tmem_alloc(&B.tmem, 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = B.tmem;
  int rb, hb, head_blocks;
  block_shape(kLines, a.ratio, rb, hb, head_blocks);
  pdl_wait();  // cache, queries and rows may be written by the previous kernel
  pdl_trigger();
  const long long me = blockIdx.x;
  Range rg = find_range<kPos, kTcThreads>(a.rows, rb, a.heads * head_blocks, gridDim.x, me);
  int *desc = a.desc + me * kDescWords;
  if (tid == 0) desc[0] = 0;
  Segment sg = load_segment<kPos>(a.rows, rg.b, rb);
  unsigned t = 0;  // tiles of this CTA so far
  auto items = [&](auto &&body) {  // every role walks the same items
    while (rg.u0 < rg.u1) {
      const Item it = next_item<kPos>(a.rows, rg, sg, rb, hb, head_blocks, a.heads);
      const int nt = it.len > 0 ? it.t_hi - it.t_lo : 0;
      if (!body(it, nt)) return;
    }
  };

  if (warp == 0) {
    // ---- codes and scales, K and V rings
    if (lane == 0) {
      const uint64_t pol = l2_policy_evict_last();  // the blocks of a segment read the same tiles
      unsigned sent[2] = {0, 0};
      items([&](const Item &it, int nt) {
        const size_t sc = (size_t)sg.seq * (size_t)a.scale_seq_stride + (size_t)it.h * (size_t)a.capacity * G;
        for (int i = 0; i < nt; ++i) {
          const int pos = (it.t_lo + i) * kPos;
#pragma unroll
          for (int side = 0; side < 2; ++side) {
            const unsigned n = sent[side]++;
            const int st = n % RS;
            if (n >= RS) {
              uint64_t t0 = 0;
              while (!mbar_try_wait(&B.raw_empty[side][st], (n / RS - 1) & 1)) {
                if (*abort) {
                  --sent[side];
                  return false;
                }
                const uint64_t now = global_timer_ns();
                if (t0 == 0) t0 = now;
                if (now - t0 > kWaitNs) *abort = 1;
              }
            }
            uint8_t *dst = smem + S::kRaw + (side * RS + st) * S::kRawSlot;
            mbar_arrive_expect_tx(&B.raw_full[side][st], S::kRawBytes);
            tma_load_4d(dst, side ? &a.v_map : &a.k_map, 0, pos * S::kRowBytes / 128, it.h, sg.seq,
                        &B.raw_full[side][st]);
            bulk_g2s(dst + S::kCodeBytes, (side ? a.v_scales : a.k_scales) + sc + (size_t)pos * G, S::kScaleBytes,
                     &B.raw_full[side][st], pol);
          }
        }
        return true;
      });
      // copies in flight must land before this shared memory goes away
      bool drained = true;
      for (int side = 0; side < 2; ++side)
        for (unsigned i = sent[side] > RS ? sent[side] - RS : 0; i < sent[side]; ++i) {
          const uint64_t t0 = global_timer_ns();
          while (!mbar_try_wait(&B.raw_full[side][i % RS], (i / RS) & 1))
            if (global_timer_ns() - t0 > kWaitNs) {
              drained = false;
              break;
            }
        }
      if (!drained && a.status) atomicOr(a.status, QMK_KV_COPIES_PENDING);
    }
  } else if (warp == 1) {
    // ---- MMA issue: QK of tile i + 1 before PV of tile i
    constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(kLines >> 4) << 24);  // fp16 x fp16 -> fp32, M = 128
    constexpr uint32_t kIdescS = kIdesc | ((uint32_t)(kPos >> 3) << 17);
    constexpr uint32_t kIdescO = kIdesc | (1u << 16) | ((uint32_t)(D >> 3) << 17);  // V: MN-major
    const uint32_t q0 = smem_addr(smem + S::kQ);
    auto scores = [&](unsigned g) {
      const int b = g & 1;
      if (!wait_warp(&B.tile_full[0][b], (g >> 1) & 1, abort)) return false;
      if (g >= 2 && !wait_warp(&B.s_empty[b], ((g >> 1) - 1) & 1, abort)) return false;
      tc_fence_after_sync();
      const uint32_t k0 = smem_addr(smem + S::kK + b * S::kTileBytes);
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        const uint32_t half = (s / 4) * (kPos * 128), in = (s % 4) * 32;
        tc_mma_bf16_warp(tmem + kColS + 128 * b, smem_desc_sw128(q0 + half + in, 1024u),
                         smem_desc_sw128(k0 + half + in, 1024u), kIdescS, s > 0);
      }
      tc_commit_warp(&B.k_empty[b]);
      tc_commit_warp(&B.s_full[b]);
      return true;
    };
    auto outputs = [&](unsigned g, bool first) {
      const int b = g & 1;
      if (!wait_warp(&B.tile_full[1][b], (g >> 1) & 1, abort)) return false;
      if (!wait_warp(&B.p_full[b], (g >> 1) & 1, abort)) return false;
      tc_fence_after_sync();
      const uint32_t v0 = smem_addr(smem + S::kV + b * S::kTileBytes);
#pragma unroll
      for (int s = 0; s < kPos / 16; ++s)
        mma_ts_warp(tmem + kColO, tmem + kColP + 64 * b + 8 * s, desc_mn(v0 + s * 2048, kPos * 128), kIdescO,
                    !first || s > 0);
      tc_commit_warp(&B.pv[b]);
      return true;
    };
    unsigned item = 0;
    items([&](const Item &, int nt) {
      if (nt == 0) return true;
      if (!wait_warp(&B.q_full, item++ & 1, abort)) return false;
      if (!scores(t)) return false;
      for (int i = 0; i < nt; ++i) {
        if (i + 1 < nt && !scores(t + i + 1)) return false;
        if (!outputs(t + i, i == 0)) return false;
      }
      t += nt;
      return true;
    });
    tc_commit_warp(&B.drain);  // completes once every MMA issued above has
  } else if (warp < 6) {
    // ---- softmax and output: a thread a line
    const int line = 32 * (warp & 3) + lane;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const int i_row = line / hb, j_head = line % hb;
    items([&](const Item &it, int nt) {
      const bool stored = line < rb * hb && i_row < it.nrows;
      const bool have = stored && i_row < it.ok_rows;
      const size_t row = sg.r0 + it.row0 + i_row, head = it.h * a.ratio + it.head0 + j_head;
      const int lim = have ? sg.start + it.row0 + i_row + 1 : 0;
      float cm = 0.f;
      if (nt > 0) {
        // the line's query into shared memory (the previous item's products have read theirs: S was waited for)
        const T *q = static_cast<const T *>(a.q) + row * (size_t)a.q_row + head * (size_t)a.q_head;
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          if (have) load_n<T, 8>(q + 8 * c, a.q_aligned, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
        }
        // scaled so that its largest element lies in [2^12, 2^13), with the softmax scale's sign
        const int fe = min(254, 266 - (int)((__float_as_uint(top) >> 23) & 255u));
        const float f = copysignf(__uint_as_float((unsigned)fe << 23), a.scale_log2);
        cm = fmaxf(fabsf(a.scale_log2) * __uint_as_float((unsigned)(254 - fe) << 23), 1e-37f);
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          if (have) load_n<T, 8>(q + 8 * c, a.q_aligned, x);
          const uint4 w = make_uint4(pack_f16(x[order<BITS>(0)] * f, x[order<BITS>(1)] * f),
                                     pack_f16(x[order<BITS>(2)] * f, x[order<BITS>(3)] * f),
                                     pack_f16(x[order<BITS>(4)] * f, x[order<BITS>(5)] * f),
                                     pack_f16(x[order<BITS>(6)] * f, x[order<BITS>(7)] * f));
          *reinterpret_cast<uint4 *>(smem + S::kQ + (c / 8) * (kLines * 128) + line * 128 +
                                     (((c & 7) ^ (line & 7)) << 4)) = w;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.q_full);
      }
      float R = -INFINITY, l = 0.f;
      for (int i = 0; i < nt; ++i) {
        const unsigned g = t + i;
        const int b = g & 1, pos0 = (it.t_lo + i) * kPos;
        if (!wait_warp(&B.exps[g & 3], (g >> 2) & 1, abort)) return false;
        const float ck = cm * B.exp_k[g & 3], ev = B.exp_v[g & 3];
        if (!wait_warp(&B.s_full[b], (g >> 1) & 1, abort)) return false;
        tc_fence_after_sync();
        const uint32_t s_at = tmem + lanes + kColS + 128 * b;
        const bool all = pos0 + kPos <= it.seen_by_all();
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < kPos; c += 32) {
          uint32_t r[32];
          tmem_ld32(s_at + c, r);
          if (all) {
#pragma unroll
            for (int e = 0; e < 32; ++e) mx = fmaxf(mx, __uint_as_float(r[e]));
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) mx = fmaxf(mx, pos0 + c + e < lim ? __uint_as_float(r[e]) : -INFINITY);
          }
        }
        const float m = fmaf(mx, ck, ev);  // of score + E
        float f = 1.f;
        if (m > R + kTcSlack) {  // (R = -inf at first)
          f = fast_exp2(R - m);
          R = m;
        }
        if (i > 0 && __any_sync(0xffffffffu, f != 1.f)) {
          if (!wait_warp(&B.pv[(g - 1) & 1], ((g - 1) >> 1) & 1, abort)) return false;
          tc_fence_after_sync();
#pragma unroll
          for (int c = 0; c < D; c += 16) {
            uint32_t r[16];
            tmem_ld16(tmem + lanes + kColO + c, r);
#pragma unroll
            for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * f);
            tmem_st16(tmem + lanes + kColO + c, r);
          }
          tmem_st_wait();
        }
        // P of tile g - 2 has been read
        if (g >= 2 && !wait_warp(&B.pv[b], ((g >> 1) - 1) & 1, abort)) return false;
        const float add = ev + kTcShift - (R == -INFINITY ? 0.f : R);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < kPos; c += 32) {
          uint32_t r[32], p[16];
          tmem_ld32(s_at + c, r);
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float y0 = fast_exp2(fmaf(__uint_as_float(r[e]), ck, add));
            float y1 = fast_exp2(fmaf(__uint_as_float(r[e + 1]), ck, add));
            if (!all) {
              y0 = pos0 + c + e < lim ? y0 : 0.f;
              y1 = pos0 + c + e + 1 < lim ? y1 : 0.f;
            }
            sum += y0 + y1;
            p[e / 2] = pack_f16(y0, y1);
          }
          tmem_st16(tmem + lanes + kColP + 64 * b + c / 2, p);
        }
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&B.s_empty[b]);
          mbar_arrive(&B.p_full[b]);
        }
        l = fmaf(l, f, sum * fast_exp2(-ev));
      }
      // ---- the line's output, or the part of it that this range holds
      if (nt > 0) {
        const unsigned g = t + nt - 1;
        if (!wait_warp(&B.pv[g & 1], (g >> 1) & 1, abort)) return false;
        tc_fence_after_sync();
      }
      t += nt;
      const bool whole = it.whole(), head_part = it.t_lo == 0;
      if (tid == 64) {
        if (!whole && head_part) describe_cut(desc, it, sg, rg, me, a.ratio, hb);
        if (it.ok_rows < it.nrows && a.status) atomicOr(a.status, QMK_KV_BAD_ROW);
      }
      const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;  // 0: the line sees nothing
      float *part = a.parts + ((size_t)(me * 2 + (head_part ? 0 : 1)) * kLines + line) * (D + 4);
      T *o = static_cast<T *>(a.out) + row * (size_t)a.o_row + head * (size_t)a.o_head;
      if (stored && !whole) *reinterpret_cast<float2 *>(part + D) = make_float2(R, l);
#pragma unroll
      for (int c = 0; c < D; c += 16) {
        uint32_t r[16];
        if (nt > 0) {
          tmem_ld16(tmem + lanes + kColO + c, r);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) r[e] = 0u;
        }
#pragma unroll
        for (int h8 = 0; h8 < 16; h8 += 8) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[order<BITS>(e)] = __uint_as_float(r[h8 + e]) * inv;
          if (!stored) continue;
          if (whole) {
            store_n<T, 8>(o + c + h8, a.o_aligned, y);
          } else {
            *reinterpret_cast<float4 *>(part + c + h8) = make_float4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<float4 *>(part + c + h8 + 4) = make_float4(y[4], y[5], y[6], y[7]);
          }
        }
      }
      tc_fence_before_sync();  // O has been read: the next item's first P V may overwrite it
      return true;
    });
  } else {
    // ---- decode: a thread a position, warps 6-9 K, 10-13 V
    const int side = warp >= 10, p = (warp - (side ? 10 : 6)) * 32 + lane;
    const Decode dec(BITS);
    items([&](const Item &it, int nt) {
      for (int i = 0; i < nt; ++i) {
        const unsigned g = t + i;
        const int b = g & 1, st = g % RS, live = it.len - (it.t_lo + i) * kPos;  // positions that some row sees
        if (!wait_warp(&B.raw_full[side][st], (g / RS) & 1, abort)) return false;
        const uint8_t *raw = smem + S::kRaw + (side * RS + st) * S::kRawSlot;
        const uint8_t *scales = raw + S::kCodeBytes;
        // the exponent of the tile's largest scale; what lies past the last position may hold anything
        unsigned big = 0;
#pragma unroll
        for (int k = 0; k < kPos / 32; ++k) {
          const int pp = 32 * k + lane;
          uint2 w;
          if constexpr (G == 4) w = *reinterpret_cast<const uint2 *>(scales + pp * 8);
          else w = make_uint2(*reinterpret_cast<const unsigned *>(scales + pp * 4), 0u);
          if (pp < live) big = max_u16x2(big, max_u16x2(w.x, w.y));
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) big = max_u16x2(big, __shfl_xor_sync(0xffffffffu, big, o));
        // (V's as in kv_attend.cu; K's only has to keep 2^-E within fp32)
        const int bound = side ? 40 : 100;
        const int e = min(max((int)(max(big & 0xffffu, big >> 16) >> 7), 127 - bound), 127 + bound);
        const float down = p < live ? __uint_as_float((unsigned)(254 - e) << 23) : 0.f;
        unsigned sc[G];
        {
          uint2 w;
          if constexpr (G == 4) w = *reinterpret_cast<const uint2 *>(scales + p * 8);
          else w = make_uint2(*reinterpret_cast<const unsigned *>(scales + p * 4), 0u);
          if (p >= live) w = make_uint2(0u, 0u);
          const float s[4] = {bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y)};
#pragma unroll
          for (int k = 0; k < G; ++k) sc[k] = pack_f16(s[k] * down, s[k] * down);
        }
        // (tile g - 2 has been read)
        if (g >= 2 && !wait_warp(side ? &B.pv[b] : &B.k_empty[b], ((g >> 1) - 1) & 1, abort)) return false;
        uint8_t *tile = smem + (side ? S::kV : S::kK) + b * S::kTileBytes;
        constexpr int kPerLine = 128 / S::kRowBytes;
        const uint8_t *src = raw + (p / kPerLine) * 128;
        const int src_swz = (p / kPerLine) & 7;
#pragma unroll
        for (int c = 0; c < S::kRowBytes / 16; ++c) {
          const uint4 w = *reinterpret_cast<const uint4 *>(
              src + ((((p % kPerLine) * (S::kRowBytes / 16) + c) ^ src_swz) << 4));
          const unsigned ww[4] = {w.x, w.y, w.z, w.w};
          constexpr int kOut = 16 / BITS;  // 16-byte chunks of fp16 per 16 bytes of codes
#pragma unroll
          for (int k = 0; k < kOut; ++k) {
            const int oc = c * kOut + k;  // dimensions 8 oc ..
            const unsigned s2 = sc[oc / 4];
            unsigned h[4];
            if constexpr (BITS == 4) {
              dec.nibbles(ww[k], h);
            } else {
              unsigned h0[2], h1[2];
              dec.bytes(ww[2 * k], h0);
              dec.bytes(ww[2 * k + 1], h1);
              h[0] = h0[0], h[1] = h0[1], h[2] = h1[0], h[3] = h1[1];
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(h[x]) : "r"(h[x]), "r"(s2));
            *reinterpret_cast<uint4 *>(tile + (oc / 8) * (kPos * 128) + p * 128 + (((oc & 7) ^ (p & 7)) << 4)) =
                make_uint4(h[0], h[1], h[2], h[3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (warp == 6) B.exp_k[g & 3] = __uint_as_float((unsigned)e << 23);
          if (warp == 10) B.exp_v[g & 3] = (float)(e - 127);
          if (warp == 6 || warp == 10) mbar_arrive(&B.exps[g & 3]);
          mbar_arrive(&B.raw_empty[side][st]);
          mbar_arrive(&B.tile_full[side][b]);
        }
      }
      t += nt;
      return true;
    });
  }
  // Every MMA the issuer started must finish before TMEM is freed (bounded).
  if (warp == 1 && lane == 0) {
    const uint64_t t0 = global_timer_ns();
    while (!mbar_try_wait(&B.drain, 0))
      if (global_timer_ns() - t0 > kWaitNs) break;
  }
  if (warp == 2 && lane == 0 && *abort && a.status) atomicOr(a.status, QMK_KV_TIMEOUT);
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

constexpr int kMaxDevices = 64;

template <typename T, int BITS, int D>
cudaError_t launch_tc(const AttendArgs &a, int grid, int dev, cudaStream_t stream) {
  static std::mutex mutex;
  static bool ready[kMaxDevices] = {};
  {
    std::lock_guard<std::mutex> lock(mutex);
    if (!ready[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(attend_tc_kernel<T, BITS, D>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, TcShape<BITS, D>::kSmem);
      if (e != cudaSuccess) return e;
      ready[dev] = true;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = TcShape<BITS, D>::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attend_tc_kernel<T, BITS, D>, a);
}

template <typename T>
cudaError_t launch_tc_format(const AttendArgs &a, int bits, int head_dim, int grid, int dev, cudaStream_t stream) {
  if (head_dim == 128)
    return bits == 4 ? launch_tc<T, 4, 128>(a, grid, dev, stream) : launch_tc<T, 8, 128>(a, grid, dev, stream);
  return bits == 4 ? launch_tc<T, 4, 64>(a, grid, dev, stream) : launch_tc<T, 8, 64>(a, grid, dev, stream);
}

}  // namespace

cudaError_t attend_tc(const AttendArgs &a, int dtype, int bits, int head_dim, int grid, int dev, cudaStream_t stream) {
  return dtype == QMK_BF16 ? launch_tc_format<__nv_bfloat16>(a, bits, head_dim, grid, dev, stream)
                           : launch_tc_format<__half>(a, bits, head_dim, grid, dev, stream);
}

}  // namespace qkv
