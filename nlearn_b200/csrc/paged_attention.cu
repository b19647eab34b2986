// paged_attention.cu — attention of one new token per sequence over a paged
// key-value cache (the decode step of a ragged batch).
//
//   o[b, h] = sum_{j < len_b} p_j v_j / sum_j p_j,  p_j = exp(scale q[b, h] . k_j)
//   lse[b, h] = ln sum_j exp(scale q . k_j)
//
// Key j of sequence b lies in page table[b, j / P], row j % P, of kv head
// h / group (group = Hq / Hk query heads share one kv head).  Keys and values
// are bf16, or e4m3 with one f32 scale per kv head.  No reference counterpart:
// nlearn recomputes the whole sequence for every token (nlearn/model.py:417-447).
//
// Bound: HBM.  Every cached element is used once per query head of its group,
// 2 FLOP per element and head, so the kernel is built to keep loads in flight
// and to spend few instructions on a byte:
//   * a warp works on tiles of 16 or 32 keys (8 KB, 4 KB for the shortest rows), gathered row by row with 16-byte
//     cp.async (any page size, any strides) into a ring of tiles of its own: no
//     block barrier between tiles, and the ring is filled across the ends of
//     sequences, so a new sequence finds its first tiles on the way;
//   * both products are m16n8k16 with the group's heads as the 8 columns:
//     s^T = k q^T takes the key tile as its 16 rows, o^T += v^T p^T the value
//     tile.  A tcgen05 tile needs 64 or 128 rows of keys in one piece of shared
//     memory and its result back from TMEM for the softmax, for 8 columns of
//     work; mma.sync takes a warp's own tile, and the tensor pipe is idle most
//     of the time either way;
//   * the running maximum moves only when a score passes it by 2^8 (the sums
//     hold that in f32), so the cross-lane maximum and the rescaling of o are
//     rare.
// p is split into two 16-bit terms (p = hi + lo) for the second product: the
// tensor pipe has room and the output then keeps the accuracy of f32
// probabilities.  In bf16 the two are off by 2^-16 at most.  With an e4m3 cache
// both products run in f16: e4m3 values are exact in f16, q is scaled by a power
// of two per head (exact), and p, kept below 2^15, is off by 2^-22, or by the
// 2^-25 of f16's smallest step where the largest p is at least 2^7.  (One f16 term moved 9 % of the outputs of 64
// sequences of up to 4097 by a bf16 step; the second takes 53.4 us there as without it, 51.9 us in
// place of 49.6 for 32 of up to 8192 with 64/4 heads of 128, 25.9 in place of 24.4 with 16/4 heads of 64.)
//
// Two ways of dividing the work, both with lengths read on the device only:
//   * flat: the work of all sequences and heads is one list of units of 64 or 128
//     keys (four warps, one tile each), cut into equal ranges, one per CTA, so any mix of
//     lengths balances.  The cut ends leave partials (max, sum, o) that
//     join_kernel merges in the order of the cache;
//   * clustered, where the table allows at most 2048 keys a CTA: a cluster of up to 8 CTAs
//     per (sequence, head) merges over distributed shared memory: one launch,
//     no prefix sums.
// Neither depends on the order in which CTAs finish.  Measured (B200, share of the 6.56 TB/s of a copy):
// 48 sequences of up to 8192, 32/8 heads of 128, token-major: 128 us, 96 %; one of
// 131072: 85 us, 96 %; 64 of up to 4097 on an e4m3 cache: 53 us, 78 % (the run's
// start and end, and the join, are the rest: between them a unit takes what its bytes do);
// 32 of up to 512, 8 heads of 64: 7.5 us, one of 512: 4.5 us (the chain of loads: length, page, tile).
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <math.h>
#include <stdint.h>

#include "host_common.h"
#include "sm100.cuh"

namespace nl {
namespace pa {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kGroup = 16;                // keys of one product (its rows); a page lookup of whole pages
constexpr int kHeads = 8;                 // query heads of one product (its columns)
constexpr int kMaxTiles = 2;              // products of 8 heads a CTA keeps: groups of up to 16 read the keys once
constexpr int kMaxCluster = 8;
// Keys of a CTA up to which a call is clustered.  A flat call costs about 5 us
// more (prefix sums, join) and balances sequences of different lengths: 32 sequences, 8 heads of 64, clustered /
// flat, all of 2048: 25.1 / 29.9 us, of up to 2048: 18.0 / 21.8; of up to 8192 (4096 a CTA): 58.0 / 57.2.
constexpr int kMaxShare = 2048;
// Where the clusters leave most of the card idle (less than a third of its CTAs), what the flat mode gains by
// taking all of it counts for more: one sequence, 8 heads of 64, of 4096: 8.4 / 10.2 us, of 8192: 12.6 / 10.1;
// four of them fill 43 %, of 8192: 17.1 / 19.2.
constexpr int kMaxShareFew = 512;
constexpr int kJoinThreads = 256;
constexpr int kJoinCtas = 4;              // resident join blocks of an SM (registers)
// Starting and ending a run costs a CTA as much as one unit of work with a bf16 cache, two with
// an e4m3 one (a fit of the CTAs' times on ragged batches, d 128: 1.34 us a unit
// and 1.14 to 1.38 us a run; 1.39 us and 3.2 to 3.7 us), so it is counted as that.
template <bool FP8>
constexpr int kOver = FP8 ? 2 : 1;
constexpr float kNoRef = -3.402823466e38f;  // before the first score: any finite one is above it
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.f;             // log2 of how far p may grow before the maximum moves
constexpr uint32_t kNoRow = 0xffffffffu;

enum : int { kErrPos = 3, kErrPage = 4 };  // device error word

struct Params {
  const __nv_bfloat16* q;
  long long q_b, q_h;               // elements
  uint8_t* k;                       // caches: bytes
  uint8_t* v;
  uint32_t page16, tok16;           // page and token strides, 16-byte units
  long long head_bytes;
  const int* table;
  long long table_ld;
  const int* lens;
  const __nv_bfloat16* k_new;       // may be null
  const __nv_bfloat16* v_new;
  long long n_b, n_h;
  const float* k_scale;             // [Hk], e4m3 only
  const float* v_scale;
  __nv_bfloat16* o;
  long long o_b, o_h;
  float* lse;                       // may be null, [B, Hq]
  long long lse_b;
  float* part_o;                    // [2 * ctas][rows][HD]
  float2* part_ml;                  // [2 * ctas][rows]
  int4* desc;                       // what the join's blocks join: [segments] or [ctas]
  int by_seg;
  int B, Hq, Hk, group, mtiles, rows;  // rows: query heads of one CTA's product, at most 16
  int page, page_shift, max_blocks, n_pages;
  float scale_log2;
  int* err;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 8x8 transpose of 16-bit elements across the warp
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two e4m3 values (low 16 bits of x) as f16x2; exact
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t x) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(x)));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ int cap_of(const Params& p) { return p.max_blocks * p.page; }
__device__ __forceinline__ int clamp_len(const Params& p, int b) {
  const int n = p.lens[b], cap = cap_of(p);
  return n < 0 ? 0 : (n > cap ? cap : n);
}
template <int UNIT>
__device__ __forceinline__ int units_of(int len) {
  return (len + UNIT - 1) / UNIT;
}
// Length of one (sequence, head tile) in the flat list: its units, after OVER for its start and its end.
template <int UNIT, int OVER>
__device__ __forceinline__ int weight_of(int len) {
  return len > 0 ? units_of<UNIT>(len) + OVER : 0;
}

// First unit of CTA i of n over U units.
__device__ __forceinline__ int cut(int i, int U, int n) {
  return static_cast<int>(static_cast<long long>(i) * U / n);
}

// A run: units [c0, c1) of one sequence and one segment of its heads (a tile of
// query heads, or four of them, one per warp).
struct Run {
  int b, seg, len, nu, c0, c1;
};
// Walks a CTA's range of the flat list, run by run (a run is not empty).
template <int UNIT, int OVER>
struct Walk {
  int segs;      // segments of a sequence
  int u, u1;     // next unit, end of the range
  int b, base;   // sequence of unit u (or an earlier one), units before it
  __device__ __forceinline__ bool next(const Params& p, Run& r) {
    while (u < u1) {
      int len = 0, w = 0;
      for (; b < p.B; ++b) {
        len = clamp_len(p, b);
        w = weight_of<UNIT, OVER>(len);
        if (u - base < w * segs) break;
        base += w * segs;
      }
      if (b >= p.B) return false;  // (lengths that changed under the call)
      const int local = u - base;
      r.b = b;
      r.len = len;
      r.nu = w - OVER;
      r.seg = local / w;
      const int c = local - r.seg * w, n = min(w - c, u1 - u);
      r.c0 = max(0, c - OVER);
      r.c1 = max(0, c + n - OVER);
      u += n;
      if (r.c1 > r.c0) return true;
    }
    return false;
  }
};

template <int HD, bool FP8>
struct Shape {
  static constexpr int RB = HD * (FP8 ? 1 : 2);  // bytes of a key row
  static constexpr int NG = RB >= 128 ? 1 : 2;   // groups of 16 keys a warp takes at a time
  static constexpr int TILE = kGroup * NG;       // keys of a tile
  static constexpr int CPR = RB / 16;            // 16-byte chunks of a row
  static constexpr int RPI = 32 / CPR;           // rows one copy instruction of a warp covers
  static constexpr int NI = kGroup / RPI;        // copy instructions of a group
  static constexpr int GB = kGroup * RB;         // bytes of a group
  static constexpr int TB = NG * GB;             // bytes of a tile
  static constexpr int SB = 2 * TB;              // K and V tiles of a stage
  static constexpr int KS = HD / 16;             // k steps of k q^T; row tiles of v^T p^T
  static constexpr int STAGES = 3;
  static constexpr int MT = RB == 256 ? 4 : 2;   // row tiles joined at a time (shared memory)
  static constexpr int RING = kWarps * STAGES * SB;
  static constexpr int SMEM = RING + kWarps * MT * 4 * 32 * 4;
  // Byte offset of chunk c of row r.  Chunks are permuted inside 128 bytes so
  // that the eight rows of an ldmatrix hit different banks.
  __device__ static __forceinline__ uint32_t at(int r, int c) {
    if constexpr (RB >= 128) return r * RB + ((c ^ (r & 7)) << 4);
    return (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ ((r >> 1) & 3)) << 4);  // two 64-byte rows a line
  }
};

// Resident CTAs an SM is meant to hold (shared memory allows them; caps registers).
template <int HD, bool FP8, int NH>
constexpr int min_ctas() {
  return Shape<HD, FP8>::SMEM > 64 * 1024 ? 2 : (NH == 2 ? 3 : 4);
}

// MODE: how the four warps and the CTAs share the work (kClustered: see the top).
enum : int { kByKeys = 0, kByHeads = 1, kClustered = 2 };

template <int HD, bool FP8, int NH, int MODE>
__global__ void __launch_bounds__(kThreads, min_ctas<HD, FP8, NH>()) decode_kernel(const Params p) {
  using S = Shape<HD, FP8>;
  constexpr bool CLUSTER = MODE == kClustered, HEADS = MODE == kByHeads;
  constexpr int UNIT = HEADS ? S::TILE : S::TILE * kWarps;  // keys of one unit of work
  constexpr int OVER = kOver<FP8>;
  // p = 2^(y - ref) with ref the running maximum less kUp: below 2^15, in f16's range, with the slack
  constexpr float kUp = FP8 ? 7.f : 0.f;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_m[kWarps][kHeads * NH], s_l[kWarps][kHeads * NH];
  __shared__ uint32_t s_valid[kWarps][S::STAGES];  // keys of a tile that take part
  __shared__ int s_scan[kWarps];
  __shared__ int s_start[2];
  __shared__ float2 s_ml[kHeads * NH];  // clustered: this CTA's (max, sum)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  // Flat, the next grid (the join) is let in when a CTA is done, not here: its CTAs
  // would take the place of this grid's on some SMs and stay there, waiting (128
  // sequences of 2048, 8 heads of 64: 108 -> 92 us).
  if constexpr (MODE == kClustered) griddep_sync();
  else griddep_wait();

  const int segs = p.Hk * p.mtiles / (HEADS ? kWarps : 1);  // of a sequence
  int U = 0, ctas = 0, rank = 0, csize = 1, ustep = 1;
  const int cta = blockIdx.x;
  Walk<UNIT, OVER> walk;  // of the copies
  Run first = {};      // of the products
  Walk<UNIT, OVER> cwalk;
  bool live;
  if constexpr (CLUSTER) {
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(csize));
    rank = cluster_ctarank();
    const int seg = cta / csize;
    first.b = seg / segs;
    first.seg = seg - first.b * segs;
    first.len = clamp_len(p, first.b);
    first.nu = units_of<UNIT>(first.len);
    // heads of 64 and short tables: a CTA takes every csize-th unit, so that its first one does not
    // depend on the length and the page of it is looked up beside that (1 of 512, 8 heads: 4.8 -> 4.6 us;
    // of 2048, 8 units a CTA: 6.5 -> 6.1, both with the join in one piece); else shares are in one piece
    // (32/8 heads of 128: 5.5 us, every csize-th unit 5.7)
    if (HD == 64 && cap_of(p) <= 2 * csize * UNIT) {
      ustep = csize;
      first.c0 = rank;
      first.c1 = first.nu;
    } else {
      first.c0 = rank * first.nu / csize;
      first.c1 = (rank + 1) * first.nu / csize;
    }
    live = first.c1 > first.c0;
    if (seg == 0 && rank == 0)
      for (int b = tid; b < p.B; b += kThreads)
        if ((p.lens[b] < 0 || p.lens[b] > cap_of(p)) && p.err) atomicExch(p.err, kErrPos);
  } else {
    // length of the flat list, and where this CTA's range begins
    const int per = (p.B + kThreads - 1) / kThreads;
    const int sb0 = min(tid * per, p.B), sb1 = min(sb0 + per, p.B);
    int mine = 0;
    for (int b = sb0; b < sb1; ++b) {
      const int n = p.lens[b];
      if (cta == 0 && (n < 0 || n > cap_of(p)) && p.err) atomicExch(p.err, kErrPos);
      mine += weight_of<UNIT, OVER>(clamp_len(p, b));
    }
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    int before = inc - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s_scan[w];
      total += s_scan[w];
    }
    U = total * segs;
    ctas = min(U, static_cast<int>(gridDim.x));
    // sequences with no key: zeros (the sum over nothing), lse = -inf
    for (int b = cta; b < p.B; b += gridDim.x) {
      if (clamp_len(p, b) > 0) continue;
      for (int i = tid; i < p.Hq * HD; i += kThreads)
        p.o[b * p.o_b + (i / HD) * p.o_h + i % HD] = __float2bfloat16_rn(0.f);
      if (p.lse)
        for (int i = tid; i < p.Hq; i += kThreads) p.lse[b * p.lse_b + i] = -INFINITY;
      if (p.by_seg)
        for (int i = tid; i < segs; i += kThreads) p.desc[b * segs + i] = make_int4(-1, 0, 0, 0);
    }
    if (cta >= ctas) {
      if (tid == 0 && !p.by_seg) p.desc[cta] = make_int4(-1, 0, 0, 0);
      return;
    }
    const int u0 = cut(cta, U, ctas), x = u0 / segs;
    if (x >= before && x < before + mine) {
      int b = sb0, pre = before;
      for (; b < sb1; ++b) {
        const int n = weight_of<UNIT, OVER>(clamp_len(p, b));
        if (x < pre + n) break;
        pre += n;
      }
      s_start[0] = b;
      s_start[1] = pre;
    }
    __syncthreads();
    walk.u = u0;
    walk.u1 = cut(cta + 1, U, ctas);
    walk.b = s_start[0];
    walk.base = s_start[1] * segs;
    walk.segs = segs;
    live = walk.next(p, first);
    cwalk = walk;
  }

  // tile of query heads (kv head * mtiles + its part of the group) of a segment, for this warp
  auto tile_of = [&](const Run& r) { return HEADS ? r.seg * kWarps + warp : r.seg; };
  const int warp_key = HEADS ? 0 : warp * S::TILE;  // where in a unit this warp's tile is

  // ---- copies: the ring is filled STAGES - 1 tiles ahead, run after run
  uint8_t* ring = smem + warp * (S::STAGES * S::SB);
  const uint32_t ring_s = smem_u32(ring);
  const int my_row = lane / S::CPR, my_chunk = lane % S::CPR;
  const uint32_t my_dst = S::at(my_row, my_chunk);
  const bool whole = p.page % kGroup == 0;  // a group of 16 keys lies in one page
  const size_t v_minus_k = static_cast<size_t>(p.v - p.k);
  const size_t step = static_cast<size_t>(p.tok16) * (16 * S::RPI);  // bytes between a lane's rows
  bool bad_page = false;
  bool more = live;         // tiles left to copy
  Run in = first;           // run being copied
  int unit = first.c0;      // its next unit
  int in_stage = 0;
  // Page of the next tile's groups (of key lane % 16, if groups are not whole).  Ordinary loads: the kernel before
  // may write the table while this one is already resident, so it is not read-only for this kernel's life.
  int pg[S::NG];
  auto block_of = [&](int pos) { return p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page; };
  auto look_up = [&]() {
    const int pos = unit * UNIT + warp_key + (whole ? 0 : (lane & 15));
    const int* row = p.table + in.b * p.table_ld;
#pragma unroll
    for (int j = 0; j < S::NG; ++j)
      pg[j] = (more && pos + j * kGroup < in.len) ? row[block_of(pos + j * kGroup)] : 0;
  };
  // key of this lane in the shared tile: i-th row of a group, relative to my_dst (my_row < RPI)
  auto row_dst = [&](int i) -> uint32_t {
    // at(my_row + i RPI, c): the row's part of the permutation splits into my_row's and i's bits
    if constexpr (S::RB >= 128) return i * S::RPI * S::RB + (my_dst ^ (((i * S::RPI) & 7) << 4));
    return i * S::RPI * S::RB + my_dst;  // 64-byte rows: 8 rows an instruction, same permutation
  };
  if (HD == 64 && ustep > 1) {
    // (the table has an entry for every position below cap)
    const int pos = unit * UNIT + warp_key + (whole ? 0 : (lane & 15));
    const int* row = p.table + in.b * p.table_ld;
#pragma unroll
    for (int j = 0; j < S::NG; ++j) {
      const int at = pos + j * kGroup;
      const int page = at < cap_of(p) ? row[block_of(at)] : 0;
      pg[j] = more && at < in.len ? page : 0;
    }
  } else {
    look_up();
  }
  auto copy_tile = [&]() {
    if (more) {
      const int hm = tile_of(in), h = hm / p.mtiles;
      const int k0 = unit * UNIT + warp_key;
      const int left = in.len - k0;  // keys of the tile that exist
      const uint8_t* kb = p.k + (h * p.head_bytes + my_chunk * 16);
      uint32_t mask = 0;
#pragma unroll
      for (int j = 0; j < S::NG; ++j) {
        const int pos0 = k0 + j * kGroup;
        const uint32_t dst = ring_s + in_stage * S::SB + j * S::GB;
        const int lj = left - j * kGroup;
        const bool in_cache = pg[j] >= 0 && pg[j] < p.n_pages;
        const bool append = p.k_new != nullptr && lj > 0 && lj <= kGroup;  // the last key is here
        if (whole && in_cache && lj >= kGroup && !append) {
          // sixteen keys of one page: rows at equal steps
          mask |= 0xffffu << (16 * j);
          const uint32_t off =
              static_cast<uint32_t>(pg[j]) * p.page16 +
              static_cast<uint32_t>(pos0 - block_of(pos0) * p.page + my_row) * p.tok16;
          const uint8_t* src = kb + static_cast<size_t>(off) * 16;
#pragma unroll
          for (int i = 0; i < S::NI; ++i) {
            cp_async16(dst + row_dst(i), src, 16u);
            cp_async16(dst + S::TB + row_dst(i), src + v_minus_k, 16u);
            src += step;
          }
          continue;
        }
        // row by row: the end of a sequence, a group over several pages, a bad page, the new token
        const int pos = pos0 + (whole ? 0 : (lane & 15));
        const bool here = pos < in.len;
        if (here && !in_cache) bad_page = true;
        const uint32_t off = static_cast<uint32_t>(pg[j]) * p.page16 +
                             static_cast<uint32_t>(pos - block_of(pos) * p.page) * p.tok16;
        uint32_t ok;
        if (whole) ok = !in_cache || lj <= 0 ? 0u : (lj >= kGroup ? 0xffffu : (1u << lj) - 1);
        else ok = __ballot_sync(0xffffffffu, here && in_cache) & 0xffffu;
        mask |= ok << (16 * j);
        const int arow = append && (ok >> (lj - 1) & 1) && p.lens[in.b] <= cap_of(p) ? lj - 1 : -1;
#pragma unroll
        for (int i = 0; i < S::NI; ++i) {
          const int r = i * S::RPI + my_row;
          const uint32_t o = whole ? off + r * p.tok16 : __shfl_sync(0xffffffffu, off, r);
          const bool use = ok >> r & 1;
          const uint8_t* src = kb + (use ? static_cast<size_t>(o) * 16 : 0);
          if (r != arow) {
            cp_async16(dst + row_dst(i), src, use ? 16u : 0u);  // rows that do not exist become zeros
            cp_async16(dst + S::TB + row_dst(i), src + v_minus_k, use ? 16u : 0u);
            continue;
          }
          // the new token: from k_new, v_new into the tile, and into its slot
          const long long nb = in.b * p.n_b + h * p.n_h + my_chunk * (FP8 ? 16 : 8);
#pragma unroll
          for (int which = 0; which < 2; ++which) {
            const __nv_bfloat16* x = (which ? p.v_new : p.k_new) + nb;
            uint4 val;
            if constexpr (!FP8) {
              val = *reinterpret_cast<const uint4*>(x);
            } else {
              const float* scp = which ? p.v_scale : p.k_scale;
              const float sc = scp ? scp[h] : 1.f;
              uint8_t* ob = reinterpret_cast<uint8_t*>(&val);
#pragma unroll
              for (int e = 0; e < 16; ++e)
                ob[e] = __nv_cvt_float_to_fp8(__bfloat162float(x[e]) / sc, __NV_SATFINITE, __NV_E4M3);
            }
            *reinterpret_cast<uint4*>(ring + in_stage * S::SB + which * S::TB + j * S::GB + row_dst(i)) = val;
            if (hm == h * p.mtiles)
              *reinterpret_cast<uint4*>(const_cast<uint8_t*>(src) + (which ? v_minus_k : 0)) = val;
          }
        }
      }
      if (lane == 0) s_valid[warp][in_stage] = mask;
      if constexpr (CLUSTER) {
        unit += HD == 64 ? ustep : 1;
        more = unit < in.c1;
      } else if (++unit == in.c1) {
        more = walk.next(p, in);
        unit = in.c0;
      }
      look_up();
    }
    in_stage = in_stage + 1 == S::STAGES ? 0 : in_stage + 1;
    cp_commit();  // an empty group past the end keeps the count
  };

  // ---- q of a run: column g of tile n is query head row0 + 8 n + g; zero past the group
  uint32_t qf[NH][S::KS][2];
  float sl[NH][2];  // factor of the scores of columns 2 t4, 2 t4 + 1
  auto load_q = [&](const Run& r) {
    const int hm = tile_of(r), h = hm / p.mtiles, mt = hm - h * p.mtiles;
    const int have = min(p.rows, p.group - mt * p.rows);
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      const bool in_group = n * kHeads + g < have;
      const __nv_bfloat16* qr = p.q + r.b * p.q_b + (h * p.group + mt * p.rows + n * kHeads + g) * p.q_h;
#pragma unroll
      for (int ks = 0; ks < S::KS; ++ks) {
        if constexpr (!FP8) {
          qf[n][ks][0] = in_group ? *reinterpret_cast<const uint32_t*>(qr + ks * 16 + t4 * 2) : 0u;
          qf[n][ks][1] = in_group ? *reinterpret_cast<const uint32_t*>(qr + ks * 16 + t4 * 2 + 8) : 0u;
        } else {
          // the k index of a product may run over the 16 dims in any fixed order:
          // lane t4 takes dims 4 t4 .. 4 t4 + 3, the four e4m3 bytes it gets of a key row
          const uint2 x = in_group ? *reinterpret_cast<const uint2*>(qr + ks * 16 + t4 * 4) : make_uint2(0, 0);
          qf[n][ks][0] = x.x;
          qf[n][ks][1] = x.y;
        }
      }
    }
  };
  auto scale_q = [&](const Run& r) {
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      if constexpr (!FP8) {
        sl[n][0] = sl[n][1] = p.scale_log2;
      } else {
        float m = 0.f;
#pragma unroll
        for (int ks = 0; ks < S::KS; ++ks)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            m = fmaxf(m, fmaxf(fabsf(bf16_lo(qf[n][ks][e])), fabsf(bf16_hi(qf[n][ks][e]))));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        // 2^e takes the head's largest |q| to [2^14, 2^15): exponent of m from its bits
        // (m is a bf16 value; below 2^-100 it is scaled by 2^114 at most)
        const int ex = max(static_cast<int>(__float_as_uint(m) >> 23), 27) - 127;
        const float up = m < INFINITY ? __uint_as_float(static_cast<uint32_t>(min(14 - ex, 127) + 127) << 23) : 1.f;
#pragma unroll
        for (int ks = 0; ks < S::KS; ++ks)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            qf[n][ks][e] = pack_f16x2(bf16_lo(qf[n][ks][e]) * up, bf16_hi(qf[n][ks][e]) * up);
        const float ksc = p.k_scale ? p.k_scale[tile_of(r) / p.mtiles] : 1.f;
        const float down = p.scale_log2 * ksc / up;
        sl[n][0] = __shfl_sync(0xffffffffu, down, 8 * t4);      // column 2 t4 is lane 4 (2 t4)'s
        sl[n][1] = __shfl_sync(0xffffffffu, down, 8 * t4 + 4);
      }
    }
  };

  if (live) load_q(first);
#pragma unroll
  for (int s = 0; s < S::STAGES - 1; ++s) copy_tile();

  int4 my_desc = make_int4(-1, 0, 0, 0);
  Run r = first;
  int stage = 0;
  while (live || CLUSTER) {
    if (live) scale_q(r);
    float acc[NH][S::KS][4];
    // columns 2 t4, 2 t4 + 1: reference of the exponents (base 2; p = 2^(y - ref)), this lane's share of the sum
    float ref[NH][2], l[NH][2];
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      ref[n][0] = ref[n][1] = kNoRef;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < S::KS; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
    }

    for (int c = r.c0; c < r.c1; c += CLUSTER && HD == 64 ? ustep : 1) {
      cp_wait<S::STAGES - 2>();
      __syncwarp();
      copy_tile();
      const uint32_t kt = ring_s + stage * S::SB, vt = kt + S::TB;
      const uint32_t valid = s_valid[warp][stage];
      stage = stage + 1 == S::STAGES ? 0 : stage + 1;
      if (valid == 0) continue;

      // ---- scores: rows (keys) g, g + 8 of a group; columns (heads) 2 t4, 2 t4 + 1
      float y[S::NG][NH][4];
#pragma unroll
      for (int j = 0; j < S::NG; ++j) {
#pragma unroll
        for (int n = 0; n < NH; ++n) y[j][n][0] = y[j][n][1] = y[j][n][2] = y[j][n][3] = 0.f;
        if constexpr (!FP8) {
#pragma unroll
          for (int ks = 0; ks < S::KS; ++ks) {
            uint32_t a[4];
            ldsm4(a, kt + j * S::GB + S::at(lane & 15, 2 * ks + (lane >> 4)));
#pragma unroll
            for (int n = 0; n < NH; ++n) mma16816<false>(y[j][n], a, qf[n][ks][0], qf[n][ks][1]);
          }
        } else {
#pragma unroll
          for (int kk = 0; kk < S::KS / 2; ++kk) {  // 32 dims
            uint32_t x[4];
            ldsm4(x, kt + j * S::GB + S::at(lane & 15, 2 * kk + (lane >> 4)));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t a[4] = {e4m3x2_f16x2(x[2 * e]), e4m3x2_f16x2(x[2 * e + 1]),
                                     e4m3x2_f16x2(x[2 * e] >> 16), e4m3x2_f16x2(x[2 * e + 1] >> 16)};
#pragma unroll
              for (int n = 0; n < NH; ++n) mma16816<true>(y[j][n], a, qf[n][2 * kk + e][0], qf[n][2 * kk + e][1]);
            }
          }
        }
      }
      bool grow = false;
#pragma unroll
      for (int j = 0; j < S::NG; ++j)
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) y[j][n][e] *= sl[n][e & 1];
      if (valid != (S::NG == 2 ? 0xffffffffu : 0xffffu)) {
#pragma unroll
        for (int j = 0; j < S::NG; ++j)
#pragma unroll
          for (int n = 0; n < NH; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!(valid >> (16 * j + g + 8 * (e >> 1)) & 1)) y[j][n][e] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < S::NG; ++j)
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) grow = grow || y[j][n][e] > ref[n][e & 1] + (kSlack + kUp);
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = kNoRef;
#pragma unroll
            for (int j = 0; j < S::NG; ++j) x = fmaxf(x, fmaxf(y[j][n][e], y[j][n][2 + e]));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            x = fmaxf(x - kUp, ref[n][e]);
            const float f = ex2_approx(ref[n][e] - x);
            ref[n][e] = x;
            l[n][e] *= f;
#pragma unroll
            for (int i = 0; i < S::KS; ++i) {
              acc[n][i][e] *= f;
              acc[n][i][2 + e] *= f;
            }
          }
      }
#pragma unroll
      for (int j = 0; j < S::NG; ++j) {
        uint32_t ph[NH][2], pl[NH][2];  // p^T as the second product's columns; its low part
#pragma unroll
        for (int n = 0; n < NH; ++n) {
          float pr[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            pr[e] = ex2_approx(y[j][n][e] - ref[n][e & 1]);
            l[n][e & 1] += pr[e];
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if constexpr (FP8) {
              const uint32_t hi = pack_f16x2(pr[2 * e], pr[2 * e + 1]);
              const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
              ph[n][e] = transpose8(hi);
              pl[n][e] = transpose8(pack_f16x2(pr[2 * e] - h.x, pr[2 * e + 1] - h.y));
            } else {
              const uint32_t hi = pack_bf16x2(pr[2 * e], pr[2 * e + 1]);
              ph[n][e] = transpose8(hi);
              pl[n][e] = transpose8(pack_bf16x2(pr[2 * e] - bf16_lo(hi), pr[2 * e + 1] - bf16_hi(hi)));
            }
          }
        }
        // ---- o^T += v^T p^T
        if constexpr (!FP8) {
#pragma unroll
          for (int i = 0; i < S::KS; ++i) {
            uint32_t a[4];
            ldsm4_t(a, vt + j * S::GB + S::at((lane & 7) + ((lane >> 4) << 3), 2 * i + ((lane >> 3) & 1)));
#pragma unroll
            for (int n = 0; n < NH; ++n) {
              mma16816<false>(acc[n][i], a, ph[n][0], ph[n][1]);
              mma16816<false>(acc[n][i], a, pl[n][0], pl[n][1]);
            }
          }
        } else {
          // a transposed 8x8 of 16-bit units holds, per key, two neighbouring dims:
          // rows g of a tile are the even dims of 16, rows g + 8 the odd ones
#pragma unroll
          for (int ii = 0; ii < S::KS / 2; ++ii) {
            uint32_t x[4];
            ldsm4_t(x, vt + j * S::GB + S::at(lane & 15, 2 * ii + (lane >> 4)));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t lo = __byte_perm(x[2 * e], 0, 0x3120), hi = __byte_perm(x[2 * e + 1], 0, 0x3120);
              const uint32_t a[4] = {e4m3x2_f16x2(lo), e4m3x2_f16x2(lo >> 16), e4m3x2_f16x2(hi),
                                     e4m3x2_f16x2(hi >> 16)};
#pragma unroll
              for (int n = 0; n < NH; ++n) {
                mma16816<true>(acc[n][2 * ii + e], a, ph[n][0], ph[n][1]);
                mma16816<true>(acc[n][2 * ii + e], a, pl[n][0], pl[n][1]);
              }
            }
          }
        }
      }
    }

    // ---- the next run's q is on its way while this run's four warps are joined
    Run nr = r;
    bool again = false;
    if constexpr (!CLUSTER) {
      again = cwalk.next(p, nr);
      if (again) load_q(nr);
    }
    const int hm = tile_of(r), h = hm / p.mtiles, mt = hm - h * p.mtiles;
    const int row0 = h * p.group + mt * p.rows, nrows = min(p.rows, p.group - mt * p.rows);
    const bool begins = r.c0 == 0, ends = r.c1 == r.nu;
    const int slot = 2 * cta + (begins ? 1 : 0);  // a run that began in an earlier CTA goes to slot 0
    if constexpr (!CLUSTER)
      if (begins) {
        const int end = cut(cta + 1, U, ctas) - r.c1 + r.nu;  // unit after this segment's last (if it goes on)
        if (!ends) my_desc = make_int4(r.b, r.seg, static_cast<int>((static_cast<long long>(end) * ctas - 1) / U), cta);
        if (p.by_seg && tid == 0) p.desc[r.b * segs + r.seg] = my_desc;
      }
    const float vsc = (FP8 && p.v_scale) ? p.v_scale[h] : 1.f;
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], o);
    if constexpr (HEADS) {
      // ---- this warp's head is whole in its registers
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int col = n * kHeads + 2 * t4 + e;
          if (col >= nrows) continue;
          const float L = l[n][e];
          if (begins && ends) {
            const float inv = L == 0.f ? 0.f : vsc / L;  // (L is 0 only where every key was left out: o is 0 too)
            __nv_bfloat16* out = p.o + r.b * p.o_b + (row0 + col) * p.o_h;
#pragma unroll
            for (int i = 0; i < S::KS; ++i)
#pragma unroll
              for (int f = 0; f < 2; ++f)
                out[i * 16 + (FP8 ? 2 * g + f : g + 8 * f)] = __float2bfloat16_rn(acc[n][i][2 * f + e] * inv);
            if (g == 0 && p.lse)
              p.lse[r.b * p.lse_b + row0 + col] = L == 0.f ? -INFINITY : (ref[n][e] + log2f(L)) * kLn2;
          } else {
            const long long at = (static_cast<long long>(slot) * kWarps + warp) * p.rows + col;
#pragma unroll
            for (int i = 0; i < S::KS; ++i)
#pragma unroll
              for (int f = 0; f < 2; ++f)
                p.part_o[at * HD + i * 16 + (FP8 ? 2 * g + f : g + 8 * f)] = acc[n][i][2 * f + e];
            if (g == 0) p.part_ml[at] = make_float2(ref[n][e], L);
          }
        }
    } else {
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (g == 0) {
            s_m[warp][n * kHeads + 2 * t4 + e] = ref[n][e];
            s_l[warp][n * kHeads + 2 * t4 + e] = l[n][e];
          }
      // clustered, a short o is joined at once, over the ring, which is idle by then
      constexpr int MT = CLUSTER && HD == 64 ? S::KS : S::MT;
      static_assert(!CLUSTER || kHeads * NH * HD * 4 + kWarps * MT * 4 * 32 * 4 <= S::SMEM, "join");
      float* scratch = reinterpret_cast<float*>(smem + (CLUSTER ? kHeads * NH * HD * 4 : S::RING));
      float* part = reinterpret_cast<float*>(smem);  // clustered: [rows][HD] over the ring, which is idle by then
      if constexpr (CLUSTER) {
        cp_wait<0>();
        __syncthreads();
      }
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        // warp w sums element w of every accumulator: column 2 t4 + (w & 1), row g or g + 8
        const int col = n * kHeads + 2 * t4 + (warp & 1);
        float f[kWarps], M = -INFINITY, L = 0.f;
#pragma unroll
        for (int i0 = 0; i0 < S::KS; i0 += MT) {
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) scratch[((warp * MT + i) * 4 + e) * 32 + lane] = acc[n][i0 + i][e];
          __syncthreads();
          if (i0 == 0) {
#pragma unroll
            for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w][col]);
            const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
              f[w] = ex2_approx(s_m[w][col] - ref);
              L += f[w] * s_l[w][col];
            }
          }
          if (col < nrows) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              float O = 0.f;
#pragma unroll
              for (int w = 0; w < kWarps; ++w) O += f[w] * scratch[((w * MT + i) * 4 + warp) * 32 + lane];
              const int d = (i0 + i) * 16 + (FP8 ? 2 * g + (warp >> 1) : g + 8 * (warp >> 1));
              if constexpr (CLUSTER) {
                part[col * HD + d] = O;
                if (d == 0) s_ml[col] = make_float2(M, L);
              } else if (begins && ends) {
                p.o[r.b * p.o_b + (row0 + col) * p.o_h + d] = __float2bfloat16_rn(L == 0.f ? 0.f : O / L * vsc);
                if (d == 0 && p.lse)
                  p.lse[r.b * p.lse_b + row0 + col] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
              } else {
                p.part_o[(static_cast<long long>(slot) * p.rows + col) * HD + d] = O;
                if (d == 0) p.part_ml[static_cast<long long>(slot) * p.rows + col] = make_float2(M, L);
              }
            }
          }
          if (!CLUSTER || n + 1 < NH || i0 + MT < S::KS) __syncthreads();  // scratch is written again (s_m after a run)
        }
      }
      if constexpr (CLUSTER) {
        // ---- every CTA of the cluster joins its share of the elements
        cluster_sync();
        for (int i = rank * kThreads + tid; i < nrows * HD; i += csize * kThreads) {
          const int col = i / HD, d = i - col * HD;
          float M = -INFINITY, L = 0.f, O = 0.f;
          float cm[kMaxCluster];
#pragma unroll
          for (int k = 0; k < kMaxCluster; ++k) {
            cm[k] = k < csize ? ld_cluster(mapa_shared(smem_u32(&s_ml[col]), k)) : -INFINITY;
            M = fmaxf(M, cm[k]);
          }
          const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
          for (int k = 0; k < kMaxCluster; ++k)
            if (k < csize) {
              const float f = ex2_approx(cm[k] - ref);
              L += f * ld_cluster(mapa_shared(smem_u32(&s_ml[col].y), k));
              O += f * ld_cluster(mapa_shared(smem_u32(part + i), k));
            }
          p.o[r.b * p.o_b + (row0 + col) * p.o_h + d] = __float2bfloat16_rn(L == 0.f ? 0.f : O / L * vsc);
          if (d == 0 && p.lse)
            p.lse[r.b * p.lse_b + row0 + col] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
        }
        cluster_sync();  // no CTA leaves while another reads its shared memory
        break;
      }
    }
    r = nr;
    live = again;
  }
  if constexpr (!CLUSTER) {
    griddep_launch();
    if (tid == 0 && !p.by_seg) p.desc[cta] = my_desc;
  }
  if (bad_page && p.err) atomicExch(p.err, kErrPage);
}

// Joins the partials of each segment that more than one CTA worked on: a block for each segment, or,
// where there are more segments than CTAs, for the one that began in a CTA's range and went on past its end.  A group of
// lanes covers one row (query head) with 16 bytes each; the groups of a row take
// every `per_row`-th partial, with a running maximum of their own, so that a
// partial's sum and its values are loaded together, and are added up in a
// fixed order.  grid.y splits the rows.
template <int HD, bool FP8>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Params p, const int tiles) {
  constexpr int LPR = HD / 4;                     // lanes (of float4) that cover a row
  constexpr int GR = kJoinThreads / LPR;          // groups of lanes
  __shared__ float4 s_o[GR][LPR];
  __shared__ float2 s_ml[GR];
  griddep_sync();
  const int4 d = p.desc[blockIdx.x];
  if (d.x < 0) return;
  const int b = d.x, j = d.w, n = d.z - j + 1;  // CTAs j .. d.z
  const int seg_rows = tiles * p.rows;            // `tiles` tiles of query heads lie in a segment
  const int li = threadIdx.x % LPR, gi = threadIdx.x / LPR;
  const int rows = (seg_rows - blockIdx.y + gridDim.y - 1) / static_cast<int>(gridDim.y);  // of this block
  if (rows <= 0) return;
  const int per_row = max(1, GR / rows);
  for (int i0 = 0; i0 < rows; i0 += GR / per_row) {
    const int i = i0 + gi / per_row, sub = gi % per_row;
    const int r = blockIdx.y + i * gridDim.y;
    const int hm = d.y * tiles + r / p.rows, h = hm / p.mtiles, mt = hm - h * p.mtiles;
    const int row = mt * p.rows + r % p.rows;  // in the group of kv head h (the last tile may be short)
    const bool on = i < rows && gi / per_row < GR / per_row && row < p.group;
    float M = -INFINITY, L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    if (on) {
#pragma unroll 4
      for (int k = sub; k < n; k += per_row) {
        // partial k of this segment: slot 2 j + 1, then slot 0 of the CTAs that follow
        const long long at = (k == 0 ? 2LL * j + 1 : 2LL * (j + k)) * seg_rows + r;
        const float2 ml = p.part_ml[at];
        const float4 x = reinterpret_cast<const float4*>(p.part_o + at * HD)[li];
        const float m = fmaxf(M, ml.x), ref = m == -INFINITY ? 0.f : m;
        const float f = ex2_approx(M - ref), e = ex2_approx(ml.x - ref);
        M = m;
        L = f * L + e * ml.y;
        O.x = f * O.x + e * x.x;
        O.y = f * O.y + e * x.y;
        O.z = f * O.z + e * x.z;
        O.w = f * O.w + e * x.w;
      }
    }
    s_o[gi][li] = O;
    if (li == 0) s_ml[gi] = make_float2(M, L);
    __syncthreads();
    if (on && sub == 0) {
      for (int k = 1; k < per_row; ++k) M = fmaxf(M, s_ml[gi + k].x);
      const float ref = M == -INFINITY ? 0.f : M;
      const float f = ex2_approx(s_ml[gi].x - ref);
      L *= f;
      O = make_float4(O.x * f, O.y * f, O.z * f, O.w * f);
      for (int k = 1; k < per_row; ++k) {
        const float e = ex2_approx(s_ml[gi + k].x - ref);
        const float4 x = s_o[gi + k][li];
        L += e * s_ml[gi + k].y;
        O.x += e * x.x;
        O.y += e * x.y;
        O.z += e * x.z;
        O.w += e * x.w;
      }
      const float vsc = (FP8 && p.v_scale) ? p.v_scale[h] : 1.f;
      const float inv = L == 0.f ? 0.f : vsc / L;  // (L is 0 only where every key was left out: O is 0 too)
      __nv_bfloat16* out = p.o + b * p.o_b + (h * p.group + row) * p.o_h + li * 4;
      out[0] = __float2bfloat16_rn(O.x * inv);
      out[1] = __float2bfloat16_rn(O.y * inv);
      out[2] = __float2bfloat16_rn(O.z * inv);
      out[3] = __float2bfloat16_rn(O.w * inv);
      if (li == 0 && p.lse)
        p.lse[b * p.lse_b + h * p.group + row] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
    }
    __syncthreads();
  }
}

// Resident CTAs of an SM, asked once per device (0: the query failed).
template <int HD, bool FP8, int NH>
int ctas_per_sm() {
  constexpr int kMaxDev = 64;
  constexpr int smem = Shape<HD, FP8>::SMEM;
  static int known[kMaxDev] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return 0;
  if (known[dev] == 0) {
    int least = INT32_MAX;
    void (*const kerns[3])(const Params) = {decode_kernel<HD, FP8, NH, 0>, decode_kernel<HD, FP8, NH, 1>,
                                            decode_kernel<HD, FP8, NH, 2>};
    for (auto kern : kerns) {
      int k = 0;
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
          cudaOccupancyMaxActiveBlocksPerMultiprocessor(&k, kern, kThreads, smem) != cudaSuccess)
        return 0;
      if (k < least) least = k;
    }
    known[dev] = least;
  }
  return known[dev];
}

// How a call is launched.
struct Plan {
  int mode, grid, cluster;
  int tiles() const { return mode == kByHeads ? kWarps : 1; }  // tiles of query heads in a segment
  bool by_seg(long long segs) const { return segs <= grid; }   // the join: a block per segment, or per CTA
  int descs(long long segs) const { return by_seg(segs) ? static_cast<int>(segs) : grid; }
};

template <int HD, bool FP8, int NH>
Plan plan_of(int B, int heads, int rows, int max_blocks, int page) {
  const int occ = ctas_per_sm<HD, FP8, NH>();
  if (occ <= 0) return {0, 0, 0};
  const long long card = static_cast<long long>(sm_count()) * occ;
  const long long segs = static_cast<long long>(B) * heads;
  const long long cap = static_cast<long long>(max_blocks) * page;
  constexpr int unit = Shape<HD, FP8>::TILE * kWarps;
  const long long units = (cap + unit - 1) / unit;  // of a full table row
  int c = 1;
  while (c < kMaxCluster && 2 * c <= units && segs * 2 * c <= card) c *= 2;
  const int share = 3 * segs * c >= card ? kMaxShare : kMaxShareFew;
  if (cap <= share * c && segs * c <= INT32_MAX) return {kClustered, static_cast<int>(segs * c), c};
  // The four warps of a CTA on four heads (nothing to join at a run's end, four
  // times the rows of partials at a CTA's; token-major rows of neighbouring heads are read
  // together) or on one head: by heads where partials are small (at most two query heads
  // share a kv head, and 32 (sequence, head) pairs share the CTAs) or few (sequences end
  // often: at least half as many pairs as CTAs).  By heads / by keys: 200 sequences of up to 4096, 8 heads of 64,
  // token-major: 136 / 165 us, e4m3: 80 / 143; 32 of up to 8192: 52.0 / 57.9; 1 of 8192: 13.5 / 10.1; 48
  // of up to 8192, 32/8 heads of 128: 130.0 / 129.3; but 1 of 131072: 94.3 / 85.7, and 32
  // of up to 8192, 64/4 heads of 128: 84.1 / 59.0.
  // (A unit is as many bytes either way, so there are as many of them.)
  const int mode = heads % kWarps == 0 && NH == 1 && ((rows <= 2 && segs >= 32) || 2 * segs >= card) ? kByHeads : kByKeys;
  return {mode, static_cast<int>(segs * units < card ? segs * units : card), 0};
}

template <int HD, bool FP8, int NH>
int launch(Params& p, const Plan& plan, cudaStream_t stream) {
  constexpr int smem = Shape<HD, FP8>::SMEM;
  const dim3 grid(plan.grid), block(kThreads);
  if (plan.mode == kClustered) {
    launch_kernel(decode_kernel<HD, FP8, NH, kClustered>, grid, block, smem, stream, plan.cluster, p);
    return launch_status();
  }
  if (plan.mode == kByHeads) launch_kernel(decode_kernel<HD, FP8, NH, kByHeads>, grid, block, smem, stream, 1, p);
  else launch_kernel(decode_kernel<HD, FP8, NH, kByKeys>, grid, block, smem, stream, 1, p);
  const int st = launch_status();
  if (st != NL_OK) return st;
  // Rows of a segment are split over as many blocks as an SM holds at once: the fewer rows a block has, the more of
  // a row's partials are loaded at the same time (64 sequences of up to 4097 on an e4m3 cache: 53.1 us, as many again
  // 55.1, a block per CTA for all rows 55.5; 48 of up to 8192: 128.5, 130.3, 130.6).
  const long long segs = static_cast<long long>(p.B) * p.Hk * p.mtiles / plan.tiles();
  const int rows = plan.tiles() * p.rows, blocks = plan.descs(segs);
  const int split = kJoinCtas * sm_count() / blocks;
  launch_kernel(join_kernel<HD, FP8>, dim3(blocks, split < 1 ? 1 : (split < rows ? split : rows)), dim3(kJoinThreads),
                0, stream, 1, p, plan.tiles());
  return launch_status();
}

// Calls f<HD, FP8, NH>() of a shape that was checked.
template <typename F>
auto dispatch(int d, bool fp8, int rows, F f) {
  const bool two = rows > kHeads;
  if (d == 64)
    return fp8 ? (two ? f.template operator()<64, true, 2>() : f.template operator()<64, true, 1>())
               : (two ? f.template operator()<64, false, 2>() : f.template operator()<64, false, 1>());
  return fp8 ? (two ? f.template operator()<128, true, 2>() : f.template operator()<128, true, 1>())
             : (two ? f.template operator()<128, false, 2>() : f.template operator()<128, false, 1>());
}
struct PlanCall {
  int B, heads, rows, max_blocks, page;
  template <int HD, bool FP8, int NH>
  Plan operator()() const { return plan_of<HD, FP8, NH>(B, heads, rows, max_blocks, page); }
};
struct LaunchCall {
  Params& p;
  const Plan& plan;
  cudaStream_t stream;
  template <int HD, bool FP8, int NH>
  int operator()() const { return launch<HD, FP8, NH>(p, plan, stream); }
};

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
// Workspace of a flat call: partials and descriptors (a clustered call needs none).
size_t workspace(const Plan& plan, int rows, int d, size_t* ml, size_t* desc) {
  if (plan.mode == kClustered) return 0;
  rows *= plan.tiles();
  size_t n = align256(static_cast<size_t>(2) * plan.grid * rows * d * sizeof(float));
  if (ml) *ml = n;
  n += align256(static_cast<size_t>(2) * plan.grid * rows * sizeof(float2));
  if (desc) *desc = n;
  return n + align256(static_cast<size_t>(plan.grid) * sizeof(int4));
}
// Query heads of one CTA's product (the group in equal parts of at most 16) and the parts of a group.
void split_group(int group, int* rows, int* mtiles) {
  *mtiles = (group + kHeads * kMaxTiles - 1) / (kHeads * kMaxTiles);
  *rows = (group + *mtiles - 1) / *mtiles;
}
bool shape_ok(int B, int Hq, int Hk, int d, int page, int max_blocks) {
  if (B <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || (d != 64 && d != 128) || page <= 0 || max_blocks <= 0) return false;
  int rows, mtiles;
  split_group(Hq / Hk, &rows, &mtiles);
  const long long cap = static_cast<long long>(max_blocks) * page;
  // unit counts of a call are 32-bit
  return cap <= INT32_MAX - 256 &&
         static_cast<double>(B) * Hk * mtiles * static_cast<double>((cap + 63) / 64 + kOver<true> + 1) <= INT32_MAX;
}

}  // namespace pa
}  // namespace nl

using namespace nl;

extern "C" size_t nl_paged_attention_workspace_bytes(int B, int Hq, int Hk, int d, int page_size, int max_blocks,
                                                     int cache_dtype) {
  if (!pa::shape_ok(B, Hq, Hk, d, page_size, max_blocks)) return 0;
  int rows, mtiles;
  pa::split_group(Hq / Hk, &rows, &mtiles);
  const pa::Plan plan =
      pa::dispatch(d, cache_dtype == NL_E4M3, rows, pa::PlanCall{B, Hk * mtiles, rows, max_blocks, page_size});
  return pa::workspace(plan, rows, d, nullptr, nullptr);
}

extern "C" int nl_paged_attention(const nl_paged_attention_args* args, cudaStream_t stream) {
  if (!args) return NL_ERR_SHAPE;
  const nl_paged_attention_args& a = *args;
  const int B = a.B, Hq = a.Hq, Hk = a.Hk, d = a.d, page_size = a.page_size, max_blocks = a.max_blocks;
  const int n_pages = a.n_pages, cache_dtype = a.cache_dtype;
  const long long page_stride = a.page_stride, head_stride = a.head_stride, tok_stride = a.tok_stride;
  if (!pa::shape_ok(B, Hq, Hk, d, page_size, max_blocks) || n_pages <= 0 || a.table_ld < max_blocks)
    return NL_ERR_SHAPE;
  if (cache_dtype != NL_BF16 && cache_dtype != NL_E4M3) return NL_ERR_DTYPE;
  if (!a.q || !a.k_cache || !a.v_cache || !a.block_table || !a.lens || !a.o ||
      (a.k_new != nullptr) != (a.v_new != nullptr))
    return NL_ERR_SHAPE;
  if (page_stride <= 0 || tok_stride <= 0 || head_stride < 0 || a.q_b < 0 || a.q_h < 0 || a.n_b < 0 || a.n_h < 0)
    return NL_ERR_SHAPE;
  const int el = cache_dtype == NL_E4M3 ? 1 : 2;
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k_cache) |
                         reinterpret_cast<uintptr_t>(a.v_cache) | reinterpret_cast<uintptr_t>(a.k_new) |
                         reinterpret_cast<uintptr_t>(a.v_new);
  if ((ptrs & 15) || ((a.q_b | a.q_h | a.n_b | a.n_h) & 7) || ((page_stride | head_stride | tok_stride) * el & 15) ||
      (reinterpret_cast<uintptr_t>(a.workspace) & 255))
    return NL_ERR_ALIGN;
  // rows are addressed inside one head by 32-bit offsets of 16 bytes: 64 GB of each cache
  if (page_stride > (1LL << 36) || tok_stride > (1LL << 36)) return NL_ERR_TOO_LARGE;
  const double extent = (n_pages - 1.) * (page_stride * el / 16) + (page_size - 1.) * (tok_stride * el / 16);
  if (extent >= UINT32_MAX) return NL_ERR_TOO_LARGE;
  pa::Params p;
  p.group = Hq / Hk;
  pa::split_group(p.group, &p.rows, &p.mtiles);
  const pa::Plan plan =
      pa::dispatch(d, cache_dtype == NL_E4M3, p.rows, pa::PlanCall{B, Hk * p.mtiles, p.rows, max_blocks, page_size});
  if (plan.grid <= 0) return NL_ERR_CUDA;
  size_t ml = 0, desc = 0;
  const size_t need = pa::workspace(plan, p.rows, d, &ml, &desc);
  if (need > 0 && (!a.workspace || a.ws_bytes < need)) return NL_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float2*>(ws + ml);
  p.desc = reinterpret_cast<int4*>(ws + desc);
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.q_b = a.q_b;
  p.q_h = a.q_h;
  p.k = static_cast<uint8_t*>(a.k_cache);
  p.v = static_cast<uint8_t*>(a.v_cache);
  p.page16 = static_cast<uint32_t>(page_stride * el / 16);
  p.tok16 = static_cast<uint32_t>(tok_stride * el / 16);
  p.head_bytes = head_stride * el;
  p.table = a.block_table;
  p.table_ld = a.table_ld;
  p.lens = a.lens;
  p.k_new = static_cast<const __nv_bfloat16*>(a.k_new);
  p.v_new = static_cast<const __nv_bfloat16*>(a.v_new);
  p.n_b = a.n_b;
  p.n_h = a.n_h;
  p.k_scale = cache_dtype == NL_E4M3 ? a.k_scale : nullptr;
  p.v_scale = cache_dtype == NL_E4M3 ? a.v_scale : nullptr;
  p.o = static_cast<__nv_bfloat16*>(a.o);
  p.o_b = a.o_b;
  p.o_h = a.o_h;
  p.lse = a.lse;
  p.lse_b = a.lse_b;
  p.B = B;
  p.by_seg = plan.by_seg(static_cast<long long>(B) * Hk * p.mtiles / plan.tiles());
  p.Hq = Hq;
  p.Hk = Hk;
  p.page = page_size;
  p.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
  p.max_blocks = max_blocks;
  p.n_pages = n_pages;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.err = device_error_word();
  return pa::dispatch(d, cache_dtype == NL_E4M3, p.rows, pa::LaunchCall{p, plan, stream});
}
