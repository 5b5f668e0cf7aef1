// Causal attention over the quantized K/V cache for many query rows (prompts,
// chunks of prompts): tcgen05 tiles.  The same operator as kv_attend.cu's
// kernel (qmk_kv_attend picks), for bf16 and fp16 queries.
//
// An item is 256 query lines (rows x the q heads of one K/V head), two MMA
// tiles A and B of 128, against tiles of 128 positions.  Per tile of positions:
// codes and scales arrive by TMA; eight warps decode K and V to fp16 in shared
// memory, s c 2^-E with E the exponent of the tile's largest scale, which is
// exact for 4-bit codes (8 + 3 significant bits) and rounds 8-bit ones to 11
// bits; S = Q K^T (128 x 128, fp32 in TMEM) for A and B; two times four warps,
// a thread a line, take the softmax and write P as fp16 over S; O += P V with
// P as the TMEM operand and V in its natural layout (dimensions contiguous: an
// MN-major operand).  Queries are scaled per line by a power of two (exact), P
// by 2^7 so that small probabilities keep fp16's precision.  The running
// reference R of a line's exponents moves only when its maximum grows past R +
// 8 (P < 2^15 then), so O is rescaled rarely.  Dimensions are held in the
// order that decoding leaves them in, in Q, K and V alike, and put back when O
// is stored.
//
// A pair of line tiles needs 4 x 512 cycles of the tensor cores, 2048 of the
// special-function units for its exponentials and about 11,600 warp
// instructions (2,900 cycles of four issue ports); while A's softmax runs, B's
// products do, and the other way round, and decoding is shared by both.  It
// takes about 5k: what bounds it is the chain of one line tile, scores -> 2.5k
// cycles of softmax by one warp a scheduler -> P stored -> P V.  Measured, 1023
// rows at the end of an 8k prompt (4 bits x 128, 16 q and 8 K/V heads): 118 us,
// 64.4 GFLOP, 546 TFLOP/s, the tensor pipe active 32 % of the time; the same
// with one line tile of 128 a CTA, S and P double-buffered, 212 us.  A fresh
// prompt of 1024 tokens takes 50 us, most of it what an item costs whatever its
// length (plan, queries, output, parts and their merge: about 20 us).
//
// Work division, parts and their merge are those of kv_attend.cu, a CTA being
// one worker.  Warps: 0 TMA, 1 MMA issue, 4-11 softmax and output of A and B,
// 12-15 decode K, 16-19 decode V.  Every wait is bounded (QMK_KV_TIMEOUT).

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "kv_attend.cuh"

namespace qkv {

namespace {

constexpr int kHalf = 128;     // query lines of an MMA tile
constexpr int kLines = kTcLines;  // of an item
constexpr int kPos = 128;      // positions of a tile
constexpr int kTcThreads = 640;
// Registers a thread: 640 x 96 at the launch, 64 + 2 x 128 + 2 x 80 = 5 x 96 after the roles part.
constexpr int kRegsIssue = 64, kRegsSoftmax = 128, kRegsDecode = 80;
static_assert(kRegsIssue + 2 * kRegsSoftmax + 2 * kRegsDecode <= 5 * 96, "more than the launch holds");
constexpr float kTcShift = 7.f;   // P is held 2^7 times too large
constexpr float kTcSlack = 8.f;   // R follows a line's maximum when it is 2^8 behind
constexpr uint32_t kColS = 0, kColO = 256;  // TMEM columns: S (then P, 64 columns) and O of A and B, 128 each

template <int BITS, int D>
struct TcShape {
  static constexpr int kRowBytes = D * BITS / 8;
  static constexpr int kGroups = D / kGroup;
  static constexpr int kCodeBytes = kPos * kRowBytes;
  static constexpr int kScaleBytes = kPos * kGroups * 2;
  static constexpr int kRawBytes = kCodeBytes + kScaleBytes;           // of K or V
  static constexpr int kRawSlots = 3;                                  // K, V, K, V, ... take turns
  // Two places of decoded K where they fit (8 bits x 128: 34 KB of raw slots
  // more): with one, decoding waits for B's scores and A's next for decoding
  // (a tile 6.4k cycles).
  static constexpr int kKBufs = kRowBytes == 128 ? 1 : 2;
  static constexpr int kTileBytes = kPos * D * 2;                      // fp16, two halves of 64 dimensions (one)
  static constexpr int kQ = 0, kK = kLines * D * 2, kV = kK + kKBufs * kTileBytes, kRaw = kV + 2 * kTileBytes;
  static constexpr int kRawSlot = (kRawBytes + 1023) / 1024 * 1024;
  static constexpr int kBars = kRaw + kRawSlots * kRawSlot;
  static constexpr int kSmem = 1024 + kBars + 512;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

struct TcBars {
  uint64_t raw_full[4], raw_empty[4];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];  // decoded tiles; empty: read by the MMAs
  uint64_t s_full[2], p_full[2], pv[2];             // of A and B; pv: P V of a tile done
  // queries in place, of A and B apart: where B has no lines its warps wait for
  // nothing and may be items ahead, so an arrival of theirs must not count for A
  uint64_t q_full[2], drain;
  float exp_k[4], exp_v[4];  // 2^E of K and E of V, of tile t in slot t % 4
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(TcBars) <= 512, "barrier area");

// The K steps of a tile's product, issued by one elected lane of a converged
// warp in one go (an election an MMA cost 70 cycles each, the issuer was what
// the softmax waited for).  Descriptors advance by 16-byte units: 32 bytes a
// step within 64 dimensions of Q and K, 16 positions (2048 bytes) of V; P by 8
// TMEM columns.
#define QKV_MMA(A, AS, B, BS) "@e tcgen05.mma.cta_group::1.kind::f16 [%0], " A ", b, %3, p;\n\t" AS BS
template <int STEPS>
__device__ __forceinline__ void mma_scores(uint32_t d, uint64_t q, uint64_t k, uint32_t idesc) {
  static_assert(STEPS == 4 || STEPS == 8, "64 or 128 dimensions");
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 a, b;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "mov.b64 a, %1;\n\tmov.b64 b, %2;\n\t"
      "setp.ne.b32 p, 0, 0;\n\t"
      QKV_MMA("a", "add.s64 a, a, 2;\n\t", "b", "add.s64 b, b, 2;\n\t")
      "setp.eq.b32 p, 0, 0;\n\t"
      QKV_MMA("a", "add.s64 a, a, 2;\n\t", "b", "add.s64 b, b, 2;\n\t")
      QKV_MMA("a", "add.s64 a, a, 2;\n\t", "b", "add.s64 b, b, 2;\n\t")
      QKV_MMA("a", "", "b", "")
      "}" ::"r"(d), "l"(q), "l"(k), "r"(idesc)
      : "memory");
  if constexpr (STEPS == 8)  // the second 64 dimensions
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 a, b;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "mov.b64 a, %1;\n\tmov.b64 b, %2;\n\t"
        "setp.eq.b32 p, 0, 0;\n\t"
        QKV_MMA("a", "add.s64 a, a, 2;\n\t", "b", "add.s64 b, b, 2;\n\t")
        QKV_MMA("a", "add.s64 a, a, 2;\n\t", "b", "add.s64 b, b, 2;\n\t")
        QKV_MMA("a", "add.s64 a, a, 2;\n\t", "b", "add.s64 b, b, 2;\n\t")
        QKV_MMA("a", "", "b", "")
        "}" ::"r"(d), "l"(q + (kHalf * 128 >> 4)), "l"(k + (kPos * 128 >> 4)), "r"(idesc)
        : "memory");
}
__device__ __forceinline__ void mma_outputs(uint32_t d, uint32_t p_cols, uint64_t v, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 a;\n\t.reg .b64 b;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "mov.b32 a, %1;\n\tmov.b64 b, %2;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      QKV_MMA("[a]", "add.s32 a, a, 8;\n\t", "b", "add.s64 b, b, 128;\n\t")
      "setp.eq.b32 p, 0, 0;\n\t"
      QKV_MMA("[a]", "add.s32 a, a, 8;\n\t", "b", "add.s64 b, b, 128;\n\t")
      QKV_MMA("[a]", "add.s32 a, a, 8;\n\t", "b", "add.s64 b, b, 128;\n\t")
      QKV_MMA("[a]", "add.s32 a, a, 8;\n\t", "b", "add.s64 b, b, 128;\n\t")
      QKV_MMA("[a]", "add.s32 a, a, 8;\n\t", "b", "add.s64 b, b, 128;\n\t")
      QKV_MMA("[a]", "add.s32 a, a, 8;\n\t", "b", "add.s64 b, b, 128;\n\t")
      QKV_MMA("[a]", "add.s32 a, a, 8;\n\t", "b", "add.s64 b, b, 128;\n\t")
      QKV_MMA("[a]", "", "b", "")
      "}" ::"r"(d), "r"(p_cols), "l"(v), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
#undef QKV_MMA
// TMEM loads that are waited for apart (tmem_ld_wait), so that one can be in
// flight while the last one's values are used.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {  // r cannot be used before
  asm volatile(
      "tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
        "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
        "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
        "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
      :
      : "memory");
}
// (a x + b, a y + b) and (x + u, y + v), two fp32 operations an instruction
__device__ __forceinline__ void fma2(float &x, float &y, float a, float b) {
  asm("{\n\t.reg .b64 p, q, r;\n\t"
      "mov.b64 p, {%0, %1};\n\t"
      "mov.b64 q, {%2, %2};\n\t"
      "mov.b64 r, {%3, %3};\n\t"
      "fma.rn.f32x2 p, p, q, r;\n\t"
      "mov.b64 {%0, %1}, p;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ void add2(float &x, float &y, float u, float v) {
  asm("{\n\t.reg .b64 p, q;\n\t"
      "mov.b64 p, {%0, %1};\n\t"
      "mov.b64 q, {%2, %3};\n\t"
      "add.rn.f32x2 p, p, q;\n\t"
      "mov.b64 {%0, %1}, p;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(u), "f"(v));
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

// 16 bytes to shared memory (completed by cp.async.wait_all), zeros where !ok.
template <typename T>
__device__ __forceinline__ void copy8(uint8_t *dst, const T *src, bool ok, bool aligned) {
  if (aligned) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(ok ? 16 : 0)
                 : "memory");
  } else {
    T *d = reinterpret_cast<T *>(dst);
#pragma unroll 1
    for (int e = 0; e < 8; ++e) d[e] = ok ? src[e] : from_float<T>(0.f);
  }
}
// 8 elements of shared memory
template <typename T>
__device__ __forceinline__ void load_row8(const T *p, float (&y)[8]) {
  const uint4 w = *reinterpret_cast<const uint4 *>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = to_float(reinterpret_cast<const T *>(&w)[e]);
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
  constexpr int G = S::kGroups, RS = S::kRawSlots, KB = S::kKBufs;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcBars &B = *reinterpret_cast<TcBars *>(smem + S::kBars);
  volatile int *abort = &B.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < RS; ++i) {
      mbar_init(&B.raw_full[i], 1);
      mbar_init(&B.raw_empty[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&B.k_full[i], 4);
      mbar_init(&B.k_empty[i], 1);
      mbar_init(&B.v_full[i], 4);
      mbar_init(&B.v_empty[i], 1);
      mbar_init(&B.s_full[i], 2);  // the MMAs' commit, and the issuer itself: it passes the exponents on
      mbar_init(&B.p_full[i], 4);
      mbar_init(&B.pv[i], 1);
      mbar_init(&B.q_full[i], 4);
    }
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

  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
  if (warp == 0) {
    // ---- codes and scales, K and V rings
    if (lane == 0) {
      const uint64_t pol = l2_policy_evict_last();  // the blocks of a segment read the same tiles
      unsigned sent = 0;
      items([&](const Item &it, int nt) {
        const size_t sc = (size_t)sg.seq * (size_t)a.scale_seq_stride + (size_t)it.h * (size_t)a.capacity * G;
        for (int i = 0; i < 2 * nt; ++i) {
          const int side = i & 1, pos = (it.t_lo + i / 2) * kPos, st = sent % RS;
          if (sent >= RS) {
            uint64_t t0 = 0;
            while (!mbar_try_wait(&B.raw_empty[st], (sent / RS - 1) & 1)) {
              if (*abort) return false;
              const uint64_t now = global_timer_ns();
              if (t0 == 0) t0 = now;
              if (now - t0 > kWaitNs) *abort = 1;
            }
          }
          uint8_t *dst = smem + S::kRaw + st * S::kRawSlot;
          mbar_arrive_expect_tx(&B.raw_full[st], S::kRawBytes);
          tma_load_4d(dst, side ? &a.v_map : &a.k_map, 0, pos / (128 / S::kRowBytes), it.h, sg.seq, &B.raw_full[st]);
          bulk_g2s(dst + S::kCodeBytes, (side ? a.v_scales : a.k_scales) + sc + (size_t)pos * G, S::kScaleBytes,
                   &B.raw_full[st], pol);
          ++sent;
        }
        return true;
      });
      // copies in flight must land before this shared memory goes away
      bool drained = true;
      for (unsigned i = sent > RS ? sent - RS : 0; i < sent; ++i) {
        const uint64_t t0 = global_timer_ns();
        while (!mbar_try_wait(&B.raw_full[i % RS], (i / RS) & 1))
          if (global_timer_ns() - t0 > kWaitNs) {
            drained = false;
            break;
          }
      }
      if (!drained && a.status) atomicOr(a.status, QMK_KV_COPIES_PENDING);
    }
  } else if (warp == 1) {
    // ---- MMA issue, per tile: P V of A, the next scores of A, then B's alike
    constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(kHalf >> 4) << 24);  // fp16 x fp16 -> fp32, M = 128
    constexpr uint32_t kIdescS = kIdesc | ((uint32_t)(kPos >> 3) << 17);
    constexpr uint32_t kIdescO = kIdesc | (1u << 16) | ((uint32_t)(D >> 3) << 17);  // V: MN-major
    // S of line tile x (MMAs run in the order of issue: what P V of the tile before reads of P comes first)
    auto scores = [&](int x, unsigned g, bool last) {
      const uint32_t k0 = smem_addr(smem + S::kK + (g % KB) * S::kTileBytes);
      const uint32_t q0 = smem_addr(smem + S::kQ) + x * (kHalf * D * 2);
      mma_scores<D / 16>(tmem + kColS + 128 * x, smem_desc_sw128(q0, 1024u), smem_desc_sw128(k0, 1024u), kIdescS);
      tc_commit_warp(&B.s_full[x]);
      if (last) tc_commit_warp(&B.k_empty[g % KB]);
      if (lane == 0) mbar_arrive(&B.s_full[x]);
    };
    unsigned n_p[2] = {0, 0};
    auto outputs = [&](int x, unsigned g, bool first, bool last) {
      if (!wait_warp(&B.p_full[x], n_p[x]++ & 1, abort)) return false;
      tc_fence_after_sync();
      const uint32_t v0 = smem_addr(smem + S::kV + (g & 1) * S::kTileBytes);
      static_assert(kPos == 128, "8 steps");
      mma_outputs(tmem + kColO + 128 * x, tmem + kColS + 128 * x, desc_mn(v0, kPos * 128), kIdescO, !first);
      tc_commit_warp(&B.pv[x]);
      if (last) tc_commit_warp(&B.v_empty[g & 1]);
      return true;
    };
    // K and V of tile g decoded: V too, since the scores' barrier passes both exponents on
    auto tiles_ready = [&](unsigned g) {
      if (!wait_warp(&B.k_full[g % KB], (g / KB) & 1, abort)) return false;
      if (!wait_warp(&B.v_full[g & 1], (g >> 1) & 1, abort)) return false;
      tc_fence_after_sync();
      return true;
    };
    unsigned n_q[2] = {0, 0};
    items([&](const Item &it, int nt) {
      if (nt == 0) return true;
      const bool two = it.nrows * hb > kHalf;
      if (!wait_warp(&B.q_full[0], n_q[0]++ & 1, abort)) return false;
      if (two && !wait_warp(&B.q_full[1], n_q[1]++ & 1, abort)) return false;
      if (!tiles_ready(t)) return false;
      scores(0, t, !two);
      if (two) scores(1, t, true);
      for (int i = 0; i < nt; ++i) {
        const unsigned g = t + i;
        const bool more = i + 1 < nt;
        // (decoded long before A's P as a rule: waited for here, off A's way)
        if (more && !tiles_ready(g + 1)) return false;
        if (!outputs(0, g, i == 0, !two)) return false;
        if (more) scores(0, g + 1, !two);
        if (two) {
          if (!outputs(1, g, i == 0, true)) return false;
          if (more) scores(1, g + 1, true);
        }
      }
      t += nt;
      return true;
    });
    tc_commit_warp(&B.drain);  // completes once every MMA issued above has
  } else if (warp < 4) {
    // (completes the first four warps, whose registers move together)
  } else if (warp < 12) {
    // ---- softmax and output: a thread a line, warps 4-7 A, 8-11 B
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int x = warp >= 8, line = kHalf * x + 32 * (warp & 3) + lane;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, s_at = tmem + lanes + kColS + 128 * x,
                   o_at = tmem + lanes + kColO + 128 * x;
    const int i_row = line / hb, j_head = line % hb;
    unsigned n_s = 0;  // tiles of this line tile so far
    constexpr int kCh = D / 8, kLoad = 32 / kCh, kIter = 32 / kLoad;  // 16-byte pieces of a row, rows a warp load
    uint8_t *q_at = smem + S::kQ + x * (kHalf * D * 2);
    items([&](const Item &it, int nt) {
      const bool idle = x == 1 && it.nrows * hb <= kHalf;  // no lines: no products either
      const bool stored = line < rb * hb && i_row < it.nrows;
      const bool have = stored && i_row < it.ok_rows;
      const size_t row = sg.r0 + it.row0 + i_row, head = it.h * a.ratio + it.head0 + j_head;
      const int lim = have ? sg.start + it.row0 + i_row + 1 : 0;
      float cm = 0.f;
      if (nt > 0 && !idle) {
        // The warp's 32 queries into shared memory (the previous item's products
        // have read theirs: S was waited for): first as they are, whole rows at
        // a time, then each lane converts its line in place.
#pragma unroll 1
        for (int k = 0; k < kIter; ++k) {
          const int src = k * kLoad + lane / kCh, c = lane % kCh, to = 32 * (warp & 3) + src;
          const long long at =
              __shfl_sync(0xffffffffu, have ? (long long)(row * (size_t)a.q_row + head * (size_t)a.q_head) : -1ll, src);
          uint8_t *dst = q_at + (c / 8) * (kHalf * 128) + to * 128 + (((c & 7) ^ (to & 7)) << 4);
          copy8(dst, static_cast<const T *>(a.q) + (at < 0 ? 0 : at + 8 * c), at >= 0, a.q_aligned);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        uint8_t *mine = q_at + (line & 127) * 128;
        float top = 0.f;
#pragma unroll 1
        for (int c = 0; c < kCh; ++c) {
          float y[8];
          load_row8(reinterpret_cast<const T *>(mine + (c / 8) * (kHalf * 128) + (((c & 7) ^ (line & 7)) << 4)), y);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(y[e]));
        }
        // scaled so that its largest element lies in [2^12, 2^13), with the softmax scale's sign
        const int fe = min(254, 266 - (int)((__float_as_uint(top) >> 23) & 255u));
        const float f = copysignf(__uint_as_float((unsigned)fe << 23), a.scale_log2);
        cm = fmaxf(fabsf(a.scale_log2) * __uint_as_float((unsigned)(254 - fe) << 23), 1e-37f);
#pragma unroll 1
        for (int c = 0; c < kCh; ++c) {
          uint8_t *at = mine + (c / 8) * (kHalf * 128) + (((c & 7) ^ (line & 7)) << 4);
          float y[8];
          load_row8(reinterpret_cast<const T *>(at), y);
          *reinterpret_cast<uint4 *>(at) = make_uint4(pack_f16(y[order<BITS>(0)] * f, y[order<BITS>(1)] * f),
                                                      pack_f16(y[order<BITS>(2)] * f, y[order<BITS>(3)] * f),
                                                      pack_f16(y[order<BITS>(4)] * f, y[order<BITS>(5)] * f),
                                                      pack_f16(y[order<BITS>(6)] * f, y[order<BITS>(7)] * f));
        }
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (nt > 0 && !idle && lane == 0) mbar_arrive(&B.q_full[x]);
      float R = -INFINITY, l = 0.f;
      for (int i = 0; i < (idle ? 0 : nt); ++i, ++n_s) {
        const unsigned g = t + i;
        const int pos0 = (it.t_lo + i) * kPos;
        if (!wait_warp(&B.s_full[x], n_s & 1, abort)) return false;
        tc_fence_after_sync();
        const float ck = fmaxf(cm * B.exp_k[g & 3], 1.2e-38f), ev = B.exp_v[g & 3];  // (> 0: -inf stays -inf)
        const bool all = pos0 + kPos <= it.seen_by_all();
        float mx, f = 1.f, sum0, sum1;
        uint32_t p[kPos / 2];
        // One pass over S: P against the reference R, kept in registers so that
        // S stays until R is known to do, and the maximum on the way.
        auto pass = [&](auto masked) {
          const float add = ev + kTcShift - (R == -INFINITY ? 0.f : R);
          mx = -INFINITY;
          sum0 = sum1 = 0.f;
#pragma unroll
          for (int c = 0; c < kPos; c += 32) {
            uint32_t r[32];
            tmem_ld32_async(s_at + c, r);
            tmem_ld_wait(r);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              if constexpr (decltype(masked)::value) {
                if (pos0 + c + e >= lim) r[e] = 0xff800000u;  // -inf
                if (pos0 + c + e + 1 >= lim) r[e + 1] = 0xff800000u;
              }
              float y0 = __uint_as_float(r[e]), y1 = __uint_as_float(r[e + 1]);
              mx = fmaxf(mx, fmaxf(y0, y1));
              fma2(y0, y1, ck, add);
              y0 = fast_exp2(y0);
              y1 = fast_exp2(y1);
              add2(sum0, sum1, y0, y1);
              p[(c + e) / 2] = pack_f16(y0, y1);
            }
          }
        };
        if (i == 0) {  // the first maximum by itself
          float m0 = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < kPos; c += 32) {
            uint32_t r[32];
            tmem_ld32_async(s_at + c, r);
            tmem_ld_wait(r);
#pragma unroll
            for (int e = 0; e < 32; ++e) m0 = fmaxf(m0, pos0 + c + e < lim ? __uint_as_float(r[e]) : -INFINITY);
          }
          R = fmaf(m0, ck, ev);
        }
#pragma unroll 1
        for (;;) {
          if (all) pass(std::false_type{});
          else pass(std::true_type{});
          const float m = fmaf(mx, ck, ev);  // of score + E
          const bool behind = m > R + kTcSlack;
          if (!__any_sync(0xffffffffu, behind)) break;
          // rare: the reference moves, O with it (i > 0: at i = 0 R is the maximum)
          if (behind) {
            f = fast_exp2(R - m);
            R = m;
          }
          if (!wait_warp(&B.pv[x], (n_s - 1) & 1, abort)) return false;
          tc_fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t r[16];
            tmem_ld16(o_at + c, r);
#pragma unroll
            for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * f);
            tmem_st16(o_at + c, r);
          }
        }
#pragma unroll
        for (int c = 0; c < kPos / 2; c += 16) {  // over S's first columns
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = p[c + e];
          tmem_st16(s_at + c, w);
        }
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.p_full[x]);
        l = fmaf(l, f, (sum0 + sum1) * fast_exp2(-ev));
      }
      // ---- the line's output, or the part of it that this range holds
      if (nt > 0 && !idle) {
        if (!wait_warp(&B.pv[x], (n_s - 1) & 1, abort)) return false;
        tc_fence_after_sync();
      }
      t += nt;
      const bool whole = it.whole(), head_part = it.t_lo == 0;
      if (tid == 128) {
        if (!whole && head_part) describe_cut(desc, it, sg, rg, me, a.ratio, hb);
        if (it.ok_rows < it.nrows && a.status) atomicOr(a.status, QMK_KV_BAD_ROW);
      }
      const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;  // 0: the line sees nothing
      // Through the warp's place of the query tile (read: the last tile's S was
      // waited for), so that rows leave in whole lines: a row of T at once, or a
      // part's fp32 row in two turns.
      const long long row_at =
          stored ? (whole ? (long long)(row * (size_t)a.o_row + head * (size_t)a.o_head)
                          : (long long)((me * 2 + (head_part ? 0 : 1)) * kLines + line) * (D + 4))
                 : -1ll;
      if (stored && !whole) *reinterpret_cast<float2 *>(a.parts + row_at + D) = make_float2(R, l);
#pragma unroll 1
      for (int turn = 0; turn < (whole ? 1 : 2); ++turn) {
        const int to = 32 * (warp & 3) + lane;
#pragma unroll 1
        for (int c = 0; c < (whole ? D : D / 2); c += 16) {
          uint32_t r[16];
          if (nt > 0 && !idle) {
            tmem_ld16(o_at + turn * (D / 2) + c, r);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) r[e] = 0u;
          }
#pragma unroll
          for (int h8 = 0; h8 < 16; h8 += 8) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[order<BITS>(e)] = __uint_as_float(r[h8 + e]) * inv;
            auto put = [&](int piece, uint4 w) {
              *reinterpret_cast<uint4 *>(q_at + (piece / 8) * (kHalf * 128) + to * 128 +
                                         (((piece & 7) ^ (to & 7)) << 4)) = w;
            };
            if (whole) {
              uint4 w;
              T *t8 = reinterpret_cast<T *>(&w);
#pragma unroll
              for (int e = 0; e < 8; ++e) t8[e] = from_float<T>(y[e]);
              put((c + h8) / 8, w);
            } else {
              const uint32_t *u = reinterpret_cast<const uint32_t *>(y);
              put((c + h8) / 4, make_uint4(u[0], u[1], u[2], u[3]));
              put((c + h8) / 4 + 1, make_uint4(u[4], u[5], u[6], u[7]));
            }
          }
        }
        __syncwarp();
#pragma unroll 4
        for (int k = 0; k < kIter; ++k) {
          const int src = k * kLoad + lane / kCh, piece = lane % kCh, from = 32 * (warp & 3) + src;
          const uint4 w = *reinterpret_cast<const uint4 *>(q_at + (piece / 8) * (kHalf * 128) + from * 128 +
                                                           (((piece & 7) ^ (from & 7)) << 4));
          const long long at = __shfl_sync(0xffffffffu, row_at, src);
          if (at < 0) continue;
          if (!whole) {
            *reinterpret_cast<uint4 *>(a.parts + at + turn * (D / 2) + 4 * piece) = w;
          } else if (a.o_aligned) {
            *reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + at + 8 * piece) = w;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              static_cast<T *>(a.out)[at + 8 * piece + e] = reinterpret_cast<const T *>(&w)[e];
          }
        }
        __syncwarp();
      }
      tc_fence_before_sync();  // O has been read: the next item's first P V may overwrite it
      return true;
    });
  } else {
    // ---- decode: a thread a position, warps 12-15 K, 16-19 V
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsDecode));
    const int side = warp >= 16, p = (warp - (side ? 16 : 12)) * 32 + lane;
    const Decode dec(BITS);
    items([&](const Item &it, int nt) {
      for (int i = 0; i < nt; ++i) {
        const unsigned g = t + i;
        const unsigned n = 2 * g + side;  // K, V, K, V, ... through the slots
        const int b = g & 1, st = n % RS, live = it.len - (it.t_lo + i) * kPos;  // positions that some row sees
        if (!wait_warp(&B.raw_full[st], (n / RS) & 1, abort)) return false;
        const uint8_t *raw = smem + S::kRaw + st * S::kRawSlot;
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
        // the tile's place has been read: K's by the scores of g - KB, V's by the outputs of g - 2
        if (side ? g >= 2 && !wait_warp(&B.v_empty[b], ((g >> 1) - 1) & 1, abort)
                 : g >= KB && !wait_warp(&B.k_empty[g % KB], (g / KB - 1) & 1, abort))
          return false;
        uint8_t *tile = smem + (side ? S::kV + b * S::kTileBytes : S::kK + (g % KB) * S::kTileBytes);
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
          if (warp == 12) B.exp_k[g & 3] = __uint_as_float((unsigned)e << 23);
          if (warp == 16) B.exp_v[g & 3] = (float)(e - 127);
          mbar_arrive(&B.raw_empty[st]);
          mbar_arrive(side ? &B.v_full[b] : &B.k_full[g % KB]);
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
  if (tid == 64 && *abort && a.status) atomicOr(a.status, QMK_KV_TIMEOUT);
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
