// Shared by the two attention kernels over the quantized K/V cache
// (kv_attend.cu: warps on mma.sync, few query rows; kv_attend_tc.cu: tcgen05
// tiles, prompts): arguments, division of the work, decoding.
#pragma once

#include <cuda.h>

#include "kv_cache.cuh"

namespace qkv {

using namespace qmk;

constexpr int kTcLines = 256;  // query lines of an item of kv_attend_tc.cu
constexpr unsigned long long kWaitNs = 1000000000ull;  // bound on one wait

struct AttendArgs {
  CUtensorMap k_map, v_map;  // codes: dims {128 bytes, 128-byte lines, heads, sequences}
  const __nv_bfloat16 *k_scales, *v_scales;
  long long scale_seq_stride;
  int capacity, heads, ratio;
  Rows rows;
  const void *q;
  void *out;
  long long q_row, q_head, o_row, o_head;
  bool q_aligned, o_aligned;
  float scale_log2;  // softmax scale * log2(e)
  int *desc;         // workspace: per worker a descriptor of kDescWords
  float *parts;      // workspace: per worker 2 x slots x (D + 4)
  unsigned *status;
};

// ------------------------------------------------------------- work division
// The query rows of one segment and K/V head are cut into blocks of rb rows
// by hb of the K/V head's q heads; a block and its positions [0, len), in
// tiles, are an item.  All items' tiles in order (segment, K/V head, head
// block, row block) form one list that is dealt to the workers (warps) in
// equal contiguous ranges, so ragged lengths, few items and many all load
// every SM alike; an item cut by a range border leaves parts that
// merge_kernel joins, in order.
struct Segment {
  int r0, n;      // rows
  int ok_rows;    // the first ok_rows of them are in range
  int start, seq;
  int blocks;     // row blocks
  int ok_blocks;  // those that hold a row in range
  long long units;       // tiles of one (K/V head, head block)
};

// a / b of values that are rarely past 32 bits (a 64-bit division is ten times a 32-bit one)
__device__ __forceinline__ long long quotient(long long a, long long b) {
  if (((a | b) >> 32) == 0) return (unsigned)a / (unsigned)b;
  return a / b;
}

// sum of floor((a i + b) / M) over i < k, by the Euclidean exchange of a and
// the divisor; the first step by itself, for M is a power of two.
template <unsigned M>
__device__ inline long long floor_sum(unsigned k, unsigned a, unsigned b) {
  if (k == 0) return 0;
  long long sum = (long long)(k - 1) * k / 2 * (a / M) + (long long)k * (b / M);
  unsigned m = M;
  a %= M;
  b %= M;
  while (a > 0) {
    const unsigned y = a * k + b;  // (a, b < M <= 2^7: below 2^32 for k < 2^24 row blocks)
    if (y < m) break;
    k = y / m;
    b = y % m;
    const unsigned t = m;
    m = a;
    a = t % m;
    sum += (long long)(k - 1) * k / 2 * (t / m) + (long long)k * (b / m);
    b %= m;
  }
  return sum;
}

// Tiles of row blocks [0, cb) of a segment, cb <= s.blocks.
template <int TILE>
__device__ inline long long block_prefix(const Segment &s, int rb, int cb) {
  long long u = 0;
  const int whole = min(cb, s.ok_blocks - 1);  // the last block in range may be cut
  if (whole > 0) u = floor_sum<TILE>(whole, rb, s.start + rb + TILE - 1);
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

constexpr int kDescWords = 8;  // a worker's descriptor of the item it cut, see merge_kernel

// Rows and q heads that share an item's slots.
__host__ __device__ inline void block_shape(int slots, int ratio, int &rb, int &hb, int &head_blocks) {
  hb = min(ratio, slots);
  rb = max(1, slots / ratio);
  head_blocks = (ratio + hb - 1) / hb;
}

// One worker's range of the list of tiles.
struct Range {
  long long u0, u1;          // tiles [u0, u1) of
  long long total, workers;  // all, dealt to so many
  int b;                     // a segment at or before u0's, and
  long long seg_at;          // the tiles before it
};

// Called by all THREADS threads of a CTA; thread t counts the segments [t
// each, (t + 1) each).  `me` of at most `most` workers (uniform in a warp).
template <int TILE, int THREADS>
__device__ inline Range find_range(const Rows &R, int rb, int per_seg, long long most, long long me) {
  constexpr int W = THREADS / 32;
  __shared__ long long s_before[THREADS], s_scan[W];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int each = (R.segments + THREADS - 1) / THREADS;
  long long mine = 0;
  for (int b = tid * each; b < min((tid + 1) * each, R.segments); ++b)
    mine += load_segment<TILE>(R, b, rb).units * per_seg;
  long long before = mine;  // inclusive prefix over the warp's threads
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += x;
  }
  if (lane == 31) s_scan[warp] = before;
  s_before[tid] = before - mine;
  __syncthreads();
  Range r;
  r.total = 0;
  long long base = 0;  // tiles counted by earlier warps
  for (int w = 0; w < W; ++w) {
    const long long x = s_scan[w];
    r.total += x;
    if (w < warp) base += x;
  }
  s_before[tid] += base;
  __syncthreads();
  r.workers = max(1ll, min(most, r.total));
  r.u0 = me < r.workers ? quotient(me * r.total, r.workers) : 0;
  r.u1 = me < r.workers ? quotient((me + 1) * r.total, r.workers) : 0;
  // the last thread whose count starts at or before u0 (equal starts are
  // segments without rows; threads past the last segment start at `total`)
  int at = 0;
  for (int i = lane; i < THREADS; i += 32) at += s_before[i] <= r.u0;
  at = max(0, __reduce_add_sync(0xffffffffu, at) - 1);
  r.b = min(at * each, R.segments - 1);  // (past it only where there are no tiles at all)
  r.seg_at = s_before[at];
  return r;
}

// An item's part that lies in a worker's range.
struct Item {
  int h, head0;         // K/V head, first q head (of the K/V head's)
  int row0;             // first row of the segment
  int nrows, ok_rows;   // rows, and how many of them are in range
  int len;              // positions that some row sees
  int tiles;            // of the whole item
  int t_lo, t_hi;       // of this part
  long long u0;         // the item's first tile in the list
  __device__ __forceinline__ bool whole() const { return t_lo == 0 && t_hi == tiles; }
  // positions below this are seen by every row
  __device__ __forceinline__ int seen_by_all() const { return ok_rows == nrows ? len - ok_rows + 1 : 0; }
};

// The item at tile r.u0 < r.u1, which moves past it; s: segment r.b.
template <int TILE>
__device__ inline Item next_item(const Rows &R, Range &r, Segment &s, int rb, int hb, int head_blocks, int heads) {
  const int per_seg = heads * head_blocks;
  while (r.u0 >= r.seg_at + s.units * per_seg) {
    r.seg_at += s.units * per_seg;
    s = load_segment<TILE>(R, ++r.b, rb);
  }
  Item it;
  const long long in_seg = r.u0 - r.seg_at;
  const int hh = (int)quotient(in_seg, s.units);
  it.h = hh / head_blocks;
  it.head0 = (hh - it.h * head_blocks) * hb;
  const long long in_head = in_seg - (long long)hh * s.units;
  int cb = 0;
  for (int hi = s.blocks; hi - cb > 1;) {
    const int mid = (cb + hi) >> 1;
    if (block_prefix<TILE>(s, rb, mid) <= in_head) cb = mid;
    else hi = mid;
  }
  it.row0 = cb * rb;
  it.ok_rows = max(0, min(rb, s.ok_rows - it.row0));
  it.nrows = min(rb, s.n - it.row0);
  it.len = it.ok_rows > 0 ? s.start + it.row0 + it.ok_rows : 0;
  it.tiles = max(1, (it.len + TILE - 1) / TILE);
  it.u0 = r.seg_at + (long long)hh * s.units + block_prefix<TILE>(s, rb, cb);
  it.t_lo = (int)(r.u0 - it.u0);
  it.t_hi = (int)min((long long)it.tiles, r.u1 - it.u0);
  r.u0 = it.u0 + it.t_hi;
  return it;
}

// Tells merge_kernel about an item whose head part worker `me` holds.
__device__ __forceinline__ void describe_cut(int *desc, const Item &it, const Segment &s, const Range &r, long long me,
                                             int ratio, int hb) {
  // parts: this worker's and those up to the worker with the item's last tile
  desc[0] = (int)(quotient((it.u0 + it.tiles) * r.workers - 1, r.total) - me) + 1;
  desc[4] = s.r0 + it.row0;
  desc[5] = it.nrows;
  desc[6] = it.h * ratio + it.head0;
  desc[7] = min(hb, ratio - it.head0) | hb << 16;
}

// ------------------------------------------------------------- instructions
__device__ __forceinline__ unsigned max_u16x2(unsigned a, unsigned b) {
  unsigned y;
  asm("max.u16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
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
// Constants of the decoding, kept in registers: an instruction takes one
// immediate operand, and these are second ones.
struct Decode {
  unsigned exp, off;
  __device__ __forceinline__ explicit Decode(int bits) {
    asm volatile("mov.b32 %0, %1;" : "=r"(exp) : "r"(bits == 4 ? 0x64006400u : 0x64646464u));
    asm volatile("mov.b32 %0, %1;" : "=r"(off) : "r"(0xd480d480u));  // -72
  }
  template <unsigned MASK>
  __device__ __forceinline__ unsigned take(unsigned w) const {  // (w & MASK) | exp
    unsigned y;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(y) : "r"(w), "n"(MASK), "r"(exp));
    return y;
  }
  // The fp16 values u - 8 of nibbles (0, 4), (1, 5), (2, 6), (3, 7) of w.
  __device__ __forceinline__ void nibbles(unsigned w, unsigned (&h)[4]) const {
    const unsigned v = w >> 8;
    h[0] = hadd2(take<0x000f000fu>(w), 0xe408e408u);        // 1024 + u - 1032
    h[1] = hfma2(take<0x00f000f0u>(w), 0x2c002c00u, off);  // (1024 + 16 u) / 16 - 72
    h[2] = hadd2(take<0x000f000fu>(v), 0xe408e408u);
    h[3] = hfma2(take<0x00f000f0u>(v), 0x2c002c00u, off);
  }
  // The fp16 values u - 128 of bytes (0, 2) and (1, 3) of w.
  __device__ __forceinline__ void bytes(unsigned w, unsigned (&h)[2]) const {
    h[0] = hadd2(__byte_perm(w, exp, 0x4240), 0xe480e480u);  // 1024 + u - 1152
    h[1] = hadd2(__byte_perm(w, exp, 0x4341), 0xe480e480u);
  }
};
__device__ __forceinline__ float f16_round(float x) { return __half2float(__float2half_rn(x)); }

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, int x, int y, int z, int w,
                                            uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar))
      : "memory");
}

// Host: kv_attend.cu.
int check_attend(const char *who, const QmkKvCache *c, const QmkKvRows *r, int num_q_heads, int dtype);
// kv_attend_tc.cu: dtype QMK_BF16 or QMK_FP16; parts of kTcLines slots a worker (CTA).
cudaError_t attend_tc(const AttendArgs &a, int dtype, int bits, int head_dim, int grid, int dev, cudaStream_t stream);

}  // namespace qkv
