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
// largest aside).  p s is scaled per tile by the power of two e of the
// tile's largest scale, with the running maximum taken of score + e, and
// rounded to fp16 (2^-11 of a term); fp32 queries are split into an fp16
// pair hi + lo on two columns of the same product, as is p s (2^-22).
// Scores, maxima, sums and outputs are fp32.

#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

#include "kv_cache.cuh"

int qmk_internal_set_error(int code, const char *msg);
int qmk_internal_clear_error();

namespace qkv {

using namespace qmk;

constexpr unsigned long long kWaitNs = 1000000000ull;  // bound on one copy wait
constexpr float kLog2e = 1.4426950408889634f;

struct AttendArgs {
  CUtensorMap k_map, v_map;  // codes: dims {row bytes, capacity, heads, sequences}
  const __nv_bfloat16 *k_scales, *v_scales;
  long long scale_seq_stride;
  int capacity, heads, ratio;
  Rows rows;
  const void *q;
  void *out;
  long long q_row, q_head, o_row, o_head;
  bool q_aligned;
  float scale_log2;  // softmax scale * log2(e)
  int *desc;         // workspace: per CTA 2 part descriptors of kDescWords
  float *parts;      // workspace: per CTA 2 x slots x (D + 2)
  unsigned *status;
};

// ------------------------------------------------------------- work division
// The query rows of one segment and K/V head are cut into blocks of RB rows
// by HB of the K/V head's q heads; a block and its positions [0, len), in
// tiles, are an item.  All items' tiles in order (segment, K/V head, head
// block, row block) form one list that is dealt to the CTAs in equal
// contiguous ranges, so ragged lengths and few items both load every SM; an
// item cut by a range border leaves parts that merge_kernel joins.
struct Segment {
  int r0, n;      // rows
  int ok_rows;    // the first ok_rows of them are in range
  int start, seq;
  int blocks;     // row blocks
  int ok_blocks;  // those that hold a row in range
  long long units;       // tiles of one (K/V head, head block)
};

// sum of floor((a i + b) / m) over i < n, by the Euclidean exchange of a and m
__device__ inline long long floor_sum(long long n, unsigned m, unsigned a, unsigned b) {
  long long sum = 0;
  unsigned k = (unsigned)n;
  while (k > 0) {
    if (a >= m) {
      sum += (long long)(k - 1) * k / 2 * (a / m);
      a %= m;
    }
    if (b >= m) {
      sum += (long long)k * (b / m);
      b %= m;
    }
    const unsigned long long y = (unsigned long long)a * k + b;
    if (y < m) break;
    const unsigned nk = (unsigned)(y / m);
    b = (unsigned)(y % m);
    k = nk;
    const unsigned t = m;
    m = a;
    a = t;
  }
  return sum;
}

// Tiles of row blocks [0, cb) of a segment, cb <= s.blocks.
template <int TILE>
__device__ inline long long block_prefix(const Segment &s, int rb, int cb) {
  long long u = 0;
  const int whole = min(cb, s.ok_blocks - 1);  // the last block in range may be cut
  if (whole > 0) u = floor_sum(whole, TILE, rb, s.start + rb + TILE - 1);
  if (cb >= s.ok_blocks && s.ok_blocks > 0) u += (s.start + s.ok_rows + TILE - 1) / TILE;
  return u + max(0, cb - s.ok_blocks);  // a block out of range: one empty tile
}

template <int TILE>
__device__ inline Segment load_segment(const Rows &R, int b, int rb) {
  Segment s;
  segment_rows(R, b, s.r0, s.n);
  s.seq = segment_seq(R, b);
  s.start = R.start[b];
  const bool ok = s.seq >= 0 && s.seq < R.num_seqs && s.start >= 0 && s.start < R.max_seq_len;
  s.ok_rows = ok ? min(s.n, min(R.max_rows, R.max_seq_len - s.start)) : 0;
  s.blocks = (s.n + rb - 1) / rb;
  s.ok_blocks = (s.ok_rows + rb - 1) / rb;
  s.units = block_prefix<TILE>(s, rb, s.blocks);
  return s;
}

constexpr int kDescWords = 8;

// ------------------------------------------------------------- instructions
__device__ __forceinline__ void mma_f16(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                        unsigned b1, float c0, float c1, float c2, float c3) {
  asm volatile(
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
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned *>(&h);
}
__device__ __forceinline__ unsigned hadd2(unsigned x, unsigned c) {
  unsigned y;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(c));
  return y;
}
__device__ __forceinline__ unsigned hfma2(unsigned x, unsigned m, unsigned c) {
  unsigned y;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(x), "r"(m), "r"(c));
  return y;
}
// The fp16 values u - 8 of nibbles (0, 4), (1, 5), (2, 6), (3, 7) of w.
__device__ __forceinline__ void decode4(unsigned w, unsigned (&h)[4]) {
  const unsigned v = w >> 8;
  h[0] = hadd2((w & 0x000f000fu) | 0x64006400u, 0xe408e408u);               // - 1032
  h[1] = hfma2((w & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd480d480u);  // / 16 - 72
  h[2] = hadd2((v & 0x000f000fu) | 0x64006400u, 0xe408e408u);
  h[3] = hfma2((v & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd480d480u);
}
// The fp16 values u - 128 of bytes (0, 2) and (1, 3) of w.
__device__ __forceinline__ void decode8(unsigned w, unsigned (&h)[2]) {
  h[0] = hadd2(__byte_perm(w, 0x64646464u, 0x4240), 0xe480e480u);  // - 1152
  h[1] = hadd2(__byte_perm(w, 0x64646464u, 0x4341), 0xe480e480u);
}
__device__ __forceinline__ float f16_round(float x) { return __half2float(__float2half_rn(x)); }

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, int x, int y, int z, int w,
                                            uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar))
      : "memory");
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
// A CTA is 4 warps that share an item; warp w takes its tiles w, w + 4, ...
// of 32 positions through a ring of its own (codes by TMA with the swizzle
// that makes 8 rows of a 16-byte column free of bank conflicts for ldmatrix,
// scales by 1-D bulk copies), with its own running maximum, sum and output:
// no barrier between warps inside an item.  Score product: M = 16 positions,
// N = 8 columns (query rows x heads; hi and lo apart for fp32), K = 16
// dimensions.  Output product: M = 16 dimensions, N = the same columns,
// K = 16 positions, the code words transposed by ldmatrix.
constexpr int kWarps = 4;
constexpr int kTile = 32;
constexpr float kShift = 14.f;  // p is held 2^14 times too large: p s < 2^15 fits fp16, and its small values do too

template <typename T, int BITS, int D, int NT>
struct Shape {
  static constexpr bool kSplit = sizeof(T) == 4;
  static constexpr int kPerTile = kSplit ? 4 : 8;
  static constexpr int kSlots = NT * kPerTile;  // (row, head) pairs of an item
  static constexpr int kGroups = D / kGroup;
  static constexpr int kRowBytes = D * BITS / 8;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kCodeBytes = kTile * kRowBytes;
  static constexpr int kScaleBytes = kTile * kGroups * 2;
  static constexpr int kTxBytes = 2 * (kCodeBytes + kScaleBytes);
  static constexpr int kStageBytes = (kTxBytes + 1023) / 1024 * 1024;
  static constexpr int kCtas = NT == 1 && kRowBytes < 128 ? 3 : 2;  // per SM
  static constexpr int kStages = std::min(6, (224 * 1024 / kCtas - 2048 - kWarps * kSlots * (D + 2) * 4) / (kWarps * kStageBytes));
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kSmem = 1024 + kRing + kWarps * kSlots * (D + 2) * 4 + kWarps * kStages * 8;
  static_assert(kStages >= 2, "ring too small");
};

// Tiles per (head block) row block: rows and q heads that share kSlots slots.
__host__ __device__ inline void block_shape(int slots, int ratio, int &rb, int &hb, int &head_blocks) {
  hb = min(ratio, slots);
  rb = max(1, slots / ratio);
  head_blocks = (ratio + hb - 1) / hb;
}

template <typename T, int BITS, int D, int NT>
__global__ void __launch_bounds__(32 * kWarps, Shape<T, BITS, D, NT>::kCtas)
    attend_kernel(const __grid_constant__ AttendArgs a) {
  using S = Shape<T, BITS, D, NT>;
  constexpr int G = S::kGroups, SL = S::kSlots;
  constexpr bool SPLIT = S::kSplit;
  constexpr int kSteps = D / 16;  // K steps of the score product
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float *buf = reinterpret_cast<float *>(smem + S::kRing);  // [warp][slot][D + 2]
  uint64_t *bars = reinterpret_cast<uint64_t *>(buf + kWarps * SL * (D + 2));
  __shared__ long long s_scan[kWarps];
  __shared__ long long s_at;  // tiles before the first segment of this CTA's range
  __shared__ int s_seg;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
  uint8_t *ring = smem + warp * S::kStages * S::kStageBytes;
  uint64_t *full = bars + warp * S::kStages;
  if (lane == 0) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  int rb, hb, head_blocks;
  block_shape(SL, a.ratio, rb, hb, head_blocks);
  const int per_seg = a.heads * head_blocks;
  pdl_wait();  // cache, queries and rows may be written by the previous kernel
  pdl_trigger();

  // ---- this CTA's range of the list of tiles
  const int each = (a.rows.segments + 32 * kWarps - 1) / (32 * kWarps);
  const int b_lo = min(tid * each, a.rows.segments), b_hi = min(b_lo + each, a.rows.segments);
  long long mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += load_segment<kTile>(a.rows, b, rb).units * per_seg;
  long long before = mine;  // inclusive prefix over the threads
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += x;
  }
  if (lane == 31) s_scan[warp] = before;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += s_scan[w];
    total += s_scan[w];
  }
  before -= mine;
  // every CTA with work has a tile for each warp
  const long long ctas = min((long long)gridDim.x, max(1ll, (total + kWarps - 1) / kWarps));
  const long long c = blockIdx.x;
  const long long u0 = c < ctas ? c * total / ctas : 0, u1 = c < ctas ? (c + 1) * total / ctas : 0;
  int *desc = a.desc + (size_t)c * 2 * kDescWords;
  if (tid == 0) desc[0] = desc[kDescWords] = 0;
  if (u0 >= u1) return;
  if (before <= u0 && u0 < before + mine) {
    long long at = before;
    for (int b = b_lo; b < b_hi; ++b) {
      const long long n = load_segment<kTile>(a.rows, b, rb).units * per_seg;
      if (u0 < at + n) {
        s_seg = b;
        s_at = at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  int b = s_seg;
  long long seg_at = s_at;
  Segment sg = load_segment<kTile>(a.rows, b, rb);
  long long u = u0;
  unsigned issued = 0, used = 0;  // ring positions of this warp
  bool dead = false;              // a wait ran out

  while (u < u1) {
    while (u >= seg_at + sg.units * per_seg) {
      seg_at += sg.units * per_seg;
      sg = load_segment<kTile>(a.rows, ++b, rb);
    }
    // item: K/V head h, head block, row block cb, tiles [t_lo, t_hi) of its `tiles`
    const long long in_seg = u - seg_at;
    const int hh = (int)(in_seg / sg.units), h = hh / head_blocks, head0 = (hh - h * head_blocks) * hb;
    const long long in_head = in_seg - (long long)hh * sg.units;
    int lo = 0, hi = sg.blocks;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (block_prefix<kTile>(sg, rb, mid) <= in_head) lo = mid;
      else hi = mid;
    }
    const int cb = lo, row0 = cb * rb;
    const int ok_rows = max(0, min(rb, sg.ok_rows - row0));  // rows of this block in range
    const int nrows = min(rb, sg.n - row0);
    const int len = ok_rows > 0 ? sg.start + row0 + ok_rows : 0;
    const int tiles = max(1, (len + kTile - 1) / kTile);
    const long long item_u0 = seg_at + (long long)hh * sg.units + block_prefix<kTile>(sg, rb, cb);
    const int t_lo = (int)(u - item_u0), t_hi = (int)min((long long)tiles, u1 - item_u0);
    u = item_u0 + t_hi;
    const int nt = len > 0 ? t_hi - t_lo : 0;                    // tiles to read
    const int my = nt > warp ? (nt - warp + kWarps - 1) / kWarps : 0;  // of this warp
    const size_t srow = ((size_t)h * (size_t)a.capacity);
    const __nv_bfloat16 *ks_g = a.k_scales + (size_t)(len ? sg.seq : 0) * (size_t)a.scale_seq_stride + srow * G;
    const __nv_bfloat16 *vs_g = a.v_scales + (size_t)(len ? sg.seq : 0) * (size_t)a.scale_seq_stride + srow * G;
    auto issue = [&](int i) {  // the warp's i-th tile of the item (lane 0)
      const int st = issued % S::kStages, pos = (t_lo + warp + i * kWarps) * kTile;
      uint8_t *dst = ring + st * S::kStageBytes;
      mbar_arrive_expect_tx(&full[st], S::kTxBytes);
      tma_load_4d(dst, &a.k_map, 0, pos, h, sg.seq, &full[st]);
      tma_load_4d(dst + S::kCodeBytes, &a.v_map, 0, pos, h, sg.seq, &full[st]);
      const uint64_t pol = l2_policy_evict_first();
      bulk_g2s(dst + 2 * S::kCodeBytes, ks_g + (size_t)pos * G, S::kScaleBytes, &full[st], pol);
      bulk_g2s(dst + 2 * S::kCodeBytes + S::kScaleBytes, vs_g + (size_t)pos * G, S::kScaleBytes, &full[st], pol);
    };
    int ahead = dead ? 0 : min(my, S::kStages);
    for (int i = 0; i < ahead; ++i) {
      if (lane == 0) issue(i);
      ++issued;
    }

    // ---- queries: the B operand of the score product, column n = gid
    unsigned qb[NT][kSteps][2];
    float cmul[NT][2];  // score factor of columns 2 tig, 2 tig + 1
    int lim[NT][2];                     // positions that the slot's row sees
    auto slot_row = [&](int slot) { return slot / hb; };
    auto slot_limit = [&](int slot) {
      const int i = slot_row(slot);
      if (i >= nrows || slot >= rb * hb) return len;  // no row: never masked, never stored
      return i < ok_rows ? sg.start + row0 + i + 1 : 0;
    };
    auto slot_stored = [&](int slot) {
      return slot < rb * hb && slot_row(slot) < nrows && head0 + slot % hb < a.ratio;
    };
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int slot = SPLIT ? 4 * t + (gid >> 1) : 8 * t + gid;
      const bool lo_half = SPLIT && (gid & 1);
      float x[kSteps][4];
      float top = 0.f;
      const T *qp = static_cast<const T *>(a.q) + (size_t)(sg.r0 + row0 + slot_row(slot)) * (size_t)a.q_row +
                    (size_t)(h * a.ratio + head0 + slot % hb) * (size_t)a.q_head;
      const bool have = slot_stored(slot) && slot_row(slot) < ok_rows;
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
      const float f = __uint_as_float((unsigned)fe << 23), finv = __uint_as_float((unsigned)(254 - fe) << 23);
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
      const float cm = a.scale_log2 * finv;
      cmul[t][0] = __shfl_sync(0xffffffffu, cm, 8 * tig);
      cmul[t][1] = __shfl_sync(0xffffffffu, cm, 8 * tig + 4);
      lim[t][0] = slot_limit(SPLIT ? 4 * t + tig : 8 * t + 2 * tig);
      lim[t][1] = SPLIT ? lim[t][0] : slot_limit(8 * t + 2 * tig + 1);
    }
    // positions below this are seen by every row of the block
    const int seen_by_all = ok_rows == nrows ? len - ok_rows + 1 : 0;

    constexpr int NS = SPLIT ? 1 : 2;  // slots of a lane's two columns
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

    auto tile_step = [&](int pos0, const uint8_t *st, auto masked) {
      constexpr bool MASK = decltype(masked)::value;
      const uint32_t kb = smem_addr(st), vb = kb + S::kCodeBytes;
      const uint8_t *ksc = st + 2 * S::kCodeBytes, *vsc = ksc + S::kScaleBytes;
      // row of this lane's ldmatrix address within 16 positions, and its swizzle
      const int lr = lane & 15, lc = lane >> 4;
      const int swz = S::kRowBytes == 128 ? (lr & 7) : S::kRowBytes == 64 ? ((lr >> 1) & 3) : ((lr >> 2) & 1);
      float x[2][NT][2][NS];  // score [16 positions][tile][row gid, gid + 8][slot]
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        float sc[2][G];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint8_t *p = ksc + (16 * sub + 8 * r + gid) * (G * 2);
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
          for (int i = 0; i < 4; ++i) s[t][i] = 0.f;
#pragma unroll
        for (int c2 = 0; c2 < S::kChunks; c2 += 2) {
          unsigned w[4];  // chunk c2: rows gid, gid + 8; chunk c2 + 1: the same
          ldmatrix4(w, kb + (16 * sub + lr) * S::kRowBytes + (((c2 + lc) ^ swz) << 4));
          if constexpr (BITS == 4) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int g = c2 + k;
              unsigned ha[4], hs[4];  // rows gid, gid + 8
              decode4(w[2 * k], ha);
              decode4(w[2 * k + 1], hs);
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                float cc[4];
                mma_f16(cc, ha[0], hs[0], ha[1], hs[1], qb[t][2 * g][0], qb[t][2 * g][1], 0.f, 0.f, 0.f, 0.f);
                mma_acc(cc, ha[2], hs[2], ha[3], hs[3], qb[t][2 * g + 1][0], qb[t][2 * g + 1][1]);
                s[t][0] = fmaf(sc[0][g], cc[0], s[t][0]);
                s[t][1] = fmaf(sc[0][g], cc[1], s[t][1]);
                s[t][2] = fmaf(sc[1][g], cc[2], s[t][2]);
                s[t][3] = fmaf(sc[1][g], cc[3], s[t][3]);
              }
            }
          } else {
            const int g = c2 / 2;
            unsigned h[4][2];
#pragma unroll
            for (int k = 0; k < 4; ++k) decode8(w[k], h[k]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              float cc[4];
              mma_f16(cc, h[0][0], h[1][0], h[0][1], h[1][1], qb[t][c2][0], qb[t][c2][1], 0.f, 0.f, 0.f, 0.f);
              mma_acc(cc, h[2][0], h[3][0], h[2][1], h[3][1], qb[t][c2 + 1][0], qb[t][c2 + 1][1]);
              s[t][0] = fmaf(sc[0][g], cc[0], s[t][0]);
              s[t][1] = fmaf(sc[0][g], cc[1], s[t][1]);
              s[t][2] = fmaf(sc[1][g], cc[2], s[t][2]);
              s[t][3] = fmaf(sc[1][g], cc[3], s[t][3]);
            }
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if constexpr (SPLIT) {
              x[sub][t][r][0] = (s[t][2 * r] + s[t][2 * r + 1]) * cmul[t][0];
            } else {
              x[sub][t][r][0] = s[t][2 * r] * cmul[t][0];
              x[sub][t][r][1] = s[t][2 * r + 1] * cmul[t][1];
            }
          }
      }
      // V scales of this lane's 4 positions, and the exponent of the tile's largest
      uint2 vw[2][2];
      unsigned vmax = 0;
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = 16 * sub + 8 * r + gid;
          if constexpr (G == 4) vw[sub][r] = *reinterpret_cast<const uint2 *>(vsc + row * 8);
          else vw[sub][r] = make_uint2(*reinterpret_cast<const unsigned *>(vsc + row * 4), 0u);
          if (MASK && pos0 + row >= len) vw[sub][r] = make_uint2(0u, 0u);
          vmax = __vmaxu2(vmax, __vmaxu2(vw[sub][r].x, vw[sub][r].y));
        }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) vmax = __vmaxu2(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
      // 2^40 either way: beyond it p s leaves fp16's range or the sum of p underflows
      const int ve = min(max((int)(max(vmax & 0xffffu, vmax >> 16) >> 7), 127 - 40), 127 + 40);
      const float vinv = __uint_as_float((unsigned)(254 - ve) << 23), vexp = (float)(ve - 127);
      float corr[NT][NS];
      bool moved = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          float mx = m[t][i];
#pragma unroll
          for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float &y = x[sub][t][r][i];
              y += vexp;
              if (MASK && pos0 + 16 * sub + 8 * r + gid >= lim[t][i]) y = -INFINITY;
              mx = fmaxf(mx, y);
            }
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          const float ref = (mx == -INFINITY ? 0.f : mx) - kShift;  // (-inf: nothing seen yet)
          corr[t][i] = fast_exp2(m[t][i] - (ref + kShift));
          moved |= mx != m[t][i];
          m[t][i] = mx;
          float sum = 0.f;
#pragma unroll
          for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              x[sub][t][r][i] = fast_exp2(x[sub][t][r][i] - ref);
              sum += x[sub][t][r][i];
            }
          l[t][i] = l[t][i] * corr[t][i] + sum * vinv;
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float cr = corr[t][NS == 1 ? 0 : (i & 1)];
              acc[t][g][0][i] *= cr;
              acc[t][g][1][i] *= cr;
            }
      }
      // outputs
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        float sv[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          sv[r][0] = bf_lo(vw[sub][r].x) * vinv;
          sv[r][1] = bf_hi(vw[sub][r].x) * vinv;
          sv[r][2] = bf_lo(vw[sub][r].y) * vinv;
          sv[r][3] = bf_hi(vw[sub][r].y) * vinv;
        }
        auto p_frag = [&](int t, int g, unsigned (&pb)[2]) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float y0 = x[sub][t][r][0] * sv[r][g], y1;
            if (MASK && x[sub][t][r][0] == 0.f) y0 = 0.f;  // whatever the scale holds
            if constexpr (SPLIT) {
              y1 = y0 - f16_round(y0);
            } else {
              y1 = x[sub][t][r][1] * sv[r][g];
              if (MASK && x[sub][t][r][1] == 0.f) y1 = 0.f;
            }
            pb[r] = transpose8(pack_f16(y0, y1));
          }
        };
#pragma unroll
        for (int c2 = 0; c2 < S::kChunks; c2 += 2) {
          unsigned w[4];  // chunk c2: positions 0-7, 8-15; chunk c2 + 1: the same
          // lanes 0-15 address the positions of chunk c2, lanes 16-31 of c2 + 1
          ldmatrix4_trans(w, vb + (16 * sub + lr) * S::kRowBytes + (((c2 + lc) ^ swz) << 4));
          if constexpr (BITS == 4) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int g = c2 + k;
              unsigned ha[4], hs[4];  // positions 0-7, 8-15
              decode4(w[2 * k], ha);
              decode4(w[2 * k + 1], hs);
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
            unsigned h[4][2];
#pragma unroll
            for (int k = 0; k < 4; ++k) decode8(w[k], h[k]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              unsigned pb[2];
              p_frag(t, g, pb);
              mma_acc(acc[t][g][0], h[0][0], h[0][1], h[1][0], h[1][1], pb[0], pb[1]);
              mma_acc(acc[t][g][1], h[2][0], h[2][1], h[3][0], h[3][1], pb[0], pb[1]);
            }
          }
        }
      }
    };

    for (int i = 0; i < my && !dead; ++i) {
      const int st = used % S::kStages;
      if (!__all_sync(0xffffffffu, wait_copy(&full[st], (used / S::kStages) & 1))) {
        dead = true;
        break;
      }
      ++used;
      const int pos0 = (t_lo + warp + i * kWarps) * kTile;
      const uint8_t *stage = ring + st * S::kStageBytes;
      if (pos0 + kTile <= seen_by_all) tile_step(pos0, stage, std::false_type{});
      else tile_step(pos0, stage, std::true_type{});
      __syncwarp();  // every lane has read the stage
      if (i + S::kStages < my) {
        if (lane == 0) issue(i + S::kStages);
        ++issued;
      }
    }

    // ---- the warp's state to shared memory: per slot m, l, outputs
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], o);
        const int slot = SPLIT ? 4 * t + tig : 8 * t + 2 * tig + i;
        float *dst = buf + (warp * SL + slot) * (D + 2);
        if (gid == 0) *reinterpret_cast<float2 *>(dst + D) = make_float2(m[t][i], l[t][i]);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float y[2][2];  // [product][row gid, gid + 8]
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float *v = &acc[t][g][k][2 * r];
              y[k][r] = SPLIT ? v[0] + v[1] : v[i];
            }
          if constexpr (BITS == 4) {  // dimensions 32 g + 4 gid + 2 k + r
            *reinterpret_cast<float2 *>(dst + 32 * g + 4 * gid) = make_float2(y[0][0], y[0][1]);
            *reinterpret_cast<float2 *>(dst + 32 * g + 4 * gid + 2) = make_float2(y[1][0], y[1][1]);
          } else {  // dimensions 32 g + 16 k + 2 gid + r
            *reinterpret_cast<float2 *>(dst + 32 * g + 2 * gid) = make_float2(y[0][0], y[0][1]);
            *reinterpret_cast<float2 *>(dst + 32 * g + 16 + 2 * gid) = make_float2(y[1][0], y[1][1]);
          }
        }
      }
    }
    if (dead && lane == 0) {
      if (a.status) atomicOr(a.status, QMK_KV_TIMEOUT);
      // copies in flight must land before this shared memory is reused
      bool drained = true;
      for (; used != issued; ++used) drained &= wait_copy(&full[used % S::kStages], (used / S::kStages) & 1);
      if (!drained && a.status) atomicOr(a.status, QMK_KV_COPIES_PENDING);
    }
    if (dead) used = issued;
    __syncthreads();
    // ---- the warps' states joined; slot by slot, a warp a slot
    const bool whole = t_lo == 0 && t_hi == tiles, head_part = t_lo == 0;
    if (!whole && tid == 0) {
      int *dd = desc + (head_part ? kDescWords : 0);
      dd[0] = 1;
      dd[1] = sg.r0 + row0;
      dd[2] = nrows;
      dd[3] = h * a.ratio + head0;
      dd[4] = min(hb, a.ratio - head0);
      // parts: this CTA's and those of the CTAs up to the one with the item's last tile
      dd[5] = (int)(((item_u0 + tiles) * ctas - 1) / total - c) + 1;
    }
    if (ok_rows < nrows && tid == 0 && a.status) atomicOr(a.status, QMK_KV_BAD_ROW);
    float *part = a.parts + ((size_t)c * 2 + (head_part ? 1 : 0)) * SL * (D + 2);
    for (int slot = warp; slot < SL; slot += kWarps) {
      if (!slot_stored(slot)) continue;
      float M = -INFINITY, L = 0.f;
      float w[kWarps];
#pragma unroll
      for (int k = 0; k < kWarps; ++k) M = fmaxf(M, buf[(k * SL + slot) * (D + 2) + D]);
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float mk = buf[(k * SL + slot) * (D + 2) + D];
        w[k] = mk == -INFINITY ? 0.f : fast_exp2(mk - M);
        L += w[k] * buf[(k * SL + slot) * (D + 2) + D + 1];
      }
      const float inv = whole ? (M == -INFINITY ? 0.f : 1.f / L) : 1.f;
      constexpr int kPer = D / 32;
      float y[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        y[e] = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) y[e] += w[k] * buf[(k * SL + slot) * (D + 2) + 32 * e + lane];
      }
      if (whole) {
        T *o = static_cast<T *>(a.out) + (size_t)(sg.r0 + row0 + slot_row(slot)) * (size_t)a.o_row +
               (size_t)(h * a.ratio + head0 + slot % hb) * (size_t)a.o_head;
#pragma unroll
        for (int e = 0; e < kPer; ++e) o[32 * e + lane] = from_float<T>(y[e] * inv);
      } else {
        float *p = part + slot * (D + 2);
#pragma unroll
        for (int e = 0; e < kPer; ++e) p[32 * e + lane] = y[e];
        if (lane == 0) *reinterpret_cast<float2 *>(p + D) = make_float2(M, L);
      }
    }
    __syncthreads();  // buf is free again
  }
}

// Joins the parts of items that were cut: CTA c takes the item whose first
// tile is in range c and that goes on in the next ranges; warp by slot.
template <typename T, int D>
__global__ void __launch_bounds__(128) merge_kernel(const int *__restrict__ desc, const float *__restrict__ parts,
                                                    int slots, int hb, void *out, long long o_row, long long o_head) {
  pdl_wait();  // the parts are written by attend_kernel
  pdl_trigger();
  const int c = blockIdx.x;
  const int *dd = desc + (size_t)c * 2 * kDescWords + kDescWords;
  if (dd[0] == 0) return;
  const int row0 = dd[1], nrows = dd[2], head0 = dd[3], nheads = dd[4], np = dd[5];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t stride = (size_t)slots * (D + 2);
  constexpr int kPer = D / 32;
  for (int slot = warp; slot < slots; slot += 4) {
    const int i = slot / hb, j = slot % hb;
    if (i >= nrows || j >= nheads) continue;
    // part k: CTA c + k's, the head part first
    auto at = [&](int k) { return parts + ((size_t)(c + k) * 2 + (k == 0 ? 1 : 0)) * stride + (size_t)slot * (D + 2); };
    float M = -INFINITY;
    for (int k = lane; k < np; k += 32) M = fmaxf(M, at(k)[D]);
    M = warp_max(M);
    float L = 0.f, y[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) y[e] = 0.f;
    for (int k0 = 0; k0 < np; k0 += 32) {
      float w = 0.f, lw = 0.f;
      if (k0 + lane < np) {
        const float2 ml = *reinterpret_cast<const float2 *>(at(k0 + lane) + D);
        w = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - M);
        lw = w * ml.y;
      }
      L += warp_sum(lw);
      const int n = min(32, np - k0);
#pragma unroll 8
      for (int k = 0; k < n; ++k) {
        const float wk = __shfl_sync(0xffffffffu, w, k);
        const float *p = at(k0 + k);
#pragma unroll
        for (int e = 0; e < kPer; ++e) y[e] += wk * p[32 * e + lane];
      }
    }
    const float inv = M == -INFINITY ? 0.f : 1.f / L;
    T *o = static_cast<T *>(out) + (size_t)(row0 + i) * (size_t)o_row + (size_t)(head0 + j) * (size_t)o_head;
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[32 * e + lane] = from_float<T>(y[e] * inv);
  }
}

// ---------------------------------------------------------------- host side
constexpr int kMaxDevices = 64;
constexpr int kMaxSms = 160;
constexpr int kMaxCtas = 3 * kMaxSms;
constexpr size_t kDescBytes = ((size_t)kMaxCtas * 2 * kDescWords * 4 + 255) / 256 * 256;

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
  const cuuint64_t row = (cuuint64_t)c->head_dim * c->bits / 8, head = row * c->capacity;
  const cuuint64_t seq = c->num_seqs > 1 ? (cuuint64_t)c->code_seq_stride : head * c->num_kv_heads;
  const cuuint64_t dims[4] = {row, (cuuint64_t)c->capacity, (cuuint64_t)c->num_kv_heads, (cuuint64_t)c->num_seqs};
  const cuuint64_t strides[3] = {row, head, seq};
  const cuuint32_t box[4] = {(cuuint32_t)row, (cuuint32_t)tile, 1, 1}, one[4] = {1, 1, 1, 1};
  const CUtensorMapSwizzle sw = row == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                                : row == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                            : CU_TENSOR_MAP_SWIZZLE_32B;
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, codes, dims, strides, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, sw, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(QMK_ERR_ARGS, "cuTensorMapEncodeTiled rejected the cache");
  return QMK_OK;
}

template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kernel)(KArgs...), int grid, int block, size_t smem, cudaStream_t stream,
                       const Args &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
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
// heads fill more than one.
int tiles_n(int dtype, int max_rows, int ratio) {
  return (long long)max_rows * ratio > (dtype == QMK_FP32 ? 4 : 8) ? 2 : 1;
}
int slots_of(int dtype, int nt) { return nt * (dtype == QMK_FP32 ? 4 : 8); }

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
  const int slots = slots_of(dtype, tiles_n(dtype, r->max_rows, num_q_heads / c->num_kv_heads));
  const size_t parts = (size_t)kMaxCtas * 2 * slots * (c->head_dim + 2) * 4;
  return kDescBytes + (parts + 255) / 256 * 256;
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
  const int grid = std::min(sms * S::kCtas, kMaxCtas);
  int rb, hb, head_blocks;
  block_shape(S::kSlots, a.ratio, rb, hb, head_blocks);
  cudaError_t e = launch_pdl(attend_kernel<T, BITS, D, NT>, grid, 32 * kWarps, S::kSmem, stream, a);
  if (e == cudaSuccess)
    e = launch_pdl(merge_kernel<T, D>, grid, 128, 0, stream, (const int *)a.desc, (const float *)a.parts,
                   (int)S::kSlots, hb, a.out, a.o_row, a.o_head);
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
  const size_t need = workspace_need(cache, rows, num_q_heads, q->dtype);
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(QMK_ERR_WORKSPACE, "%s: workspace needs %zu bytes, 256-byte aligned", who, need);
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev < 0 || dev >= kMaxDevices)) e = cudaErrorInvalidDevice;
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return fail(QMK_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  AttendArgs a;
  rc = encode_codes(&a.k_map, cache, cache->k_codes, kTile);
  if (rc == QMK_OK) rc = encode_codes(&a.v_map, cache, cache->v_codes, kTile);
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
  a.scale_log2 = scale * kLog2e;
  a.desc = static_cast<int *>(workspace);
  a.parts = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + kDescBytes);
  a.status = status;
  const int nt = tiles_n(q->dtype, rows->max_rows, a.ratio);
  if (q->dtype == QMK_BF16) return pick_format<__nv_bfloat16>(cache, a, nt, sms, dev, stream);
  if (q->dtype == QMK_FP16) return pick_format<__half>(cache, a, nt, sms, dev, stream);
  return pick_format<float>(cache, a, nt, sms, dev, stream);
}
