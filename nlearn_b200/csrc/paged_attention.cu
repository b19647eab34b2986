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
// 2 FLOP per element and head, so the kernel is built to keep loads in flight:
//   * a warp works on tiles of 16 keys, gathered row by row with 16-byte
//     cp.async (any page size, any strides) into a ring of tiles of its own:
//     no block barrier between tiles, only the warp's own wait;
//   * the group's query heads are the 16 rows of m16n8k16 products (q k^T, then
//     p v with the running maximum and sum in registers): with at most 16 rows
//     a 128-row tcgen05 tile would be mostly padding, and the keys would have
//     to be transposed through TMEM; mma.sync takes them straight from the tile;
//   * the work of all sequences and heads is one flat list of units of 64 keys
//     (four warps, one tile each), cut into equal ranges, one per CTA: lengths
//     are read on the device, so ragged batches balance without the host.  A
//     range's cut ends leave partials (max, sum, o) that join_kernel merges in
//     the order of the cache, so results do not depend on timing.
// p is split into two bf16 terms (p = hi + lo, error 2^-17) for the second
// product: the tensor pipe is idle anyway and the output then keeps the accuracy of
// f32 probabilities.  With an e4m3 cache both products run in f16: e4m3 values
// are exact in f16, q is scaled by a power of two per row (exact), and p, kept
// in [0, 2^15], is rounded to f16's 11 bits, a quarter of the bf16 output's step.
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
constexpr int kTile = 16;                 // keys a warp takes at a time
constexpr int kUnit = kTile * kWarps;     // keys of one unit of work
constexpr int kStages = 3;                // tiles in a warp's ring
constexpr int kRows = 16;                 // query heads of one product
constexpr int kJoinThreads = 256;
constexpr float kLn2 = 0.6931471805599453f;
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
  int4* desc;                       // [ctas]
  int B, Hq, Hk, group, mtiles, rows;  // rows = min(group, 16): rows kept of a product
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
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(x), __NV_E4M3);
  return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

__device__ __forceinline__ int clamp_len(const Params& p, int b) {
  const int cap = p.max_blocks * p.page;
  const int n = p.lens[b];
  return n < 0 ? 0 : (n > cap ? cap : n);
}
__device__ __forceinline__ int units_of(int len) { return (len + kUnit - 1) / kUnit; }

// Range of CTA i of n over U units: [i U / n, (i + 1) U / n).
__device__ __forceinline__ long long cut(long long i, long long U, long long n) { return i * U / n; }

// State of one warp's pass over a run of units of one (sequence, kv head).
template <int HD, bool FP8>
struct Warp {
  static constexpr int EL = FP8 ? 1 : 2;
  static constexpr int RB = HD * EL;             // bytes of a key row
  static constexpr int CPR = RB / 16;            // 16-byte chunks of a row
  static constexpr int RPI = 32 / CPR;           // rows a warp's copy instruction covers
  static constexpr int NI = kTile / RPI;         // copy instructions of a tile
  static constexpr int TB = kTile * RB;          // bytes of a tile
  static constexpr int SB = 2 * TB;              // K and V tiles of a stage
  static constexpr int KS = HD / 16;             // k steps of q k^T
  static constexpr int NT = HD / 8;              // n tiles of p v

  // byte offset of 16-byte chunk c of row r: chunks are permuted inside groups
  // of eight rows so that the eight rows of an ldmatrix hit different banks
  __device__ static __forceinline__ uint32_t at(int r, int c) {
    if constexpr (RB >= 128) return r * RB + ((c ^ (r & 7)) << 4);
    // 64-byte rows: two rows share 128 bytes
    return (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ ((r >> 1) & 3)) << 4);
  }
};

template <int HD, bool FP8>
__global__ void __launch_bounds__(kThreads) decode_kernel(const Params p) {
  using W = Warp<HD, FP8>;
  constexpr int OS = HD + 8;  // row pitch of the warps' o in shared memory (floats)
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
  __shared__ uint32_t s_valid[kWarps][kStages];
  __shared__ int s_scan[kWarps + 1];
  __shared__ int s_start[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  griddep_sync();

  // ---- units of all sequences: where this CTA's range begins
  const int per = (p.B + kThreads - 1) / kThreads;
  const int sb0 = min(tid * per, p.B), sb1 = min(sb0 + per, p.B);
  int mine = 0;
  for (int b = sb0; b < sb1; ++b) {
    const int n = p.lens[b];
    if (blockIdx.x == 0 && (n < 0 || n > p.max_blocks * p.page) && p.err) atomicExch(p.err, kErrPos);
    mine += units_of(clamp_len(p, b));
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
  const int heads = p.Hk * p.mtiles;
  const long long U = static_cast<long long>(total) * heads;
  const long long ctas = U < gridDim.x ? U : gridDim.x;
  const long long cta = blockIdx.x;

  // sequences with no key: zeros (the sum over nothing), lse = -inf
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    if (clamp_len(p, b) > 0) continue;
    for (int i = tid; i < p.Hq * HD; i += kThreads)
      p.o[b * p.o_b + (i / HD) * p.o_h + i % HD] = __float2bfloat16_rn(0.f);
    if (p.lse)
      for (int i = tid; i < p.Hq; i += kThreads) p.lse[b * p.lse_b + i] = -INFINITY;
  }
  if (cta >= ctas) {
    if (tid == 0) p.desc[cta] = make_int4(-1, 0, 0, 0);
    return;
  }
  const long long u0 = cut(cta, U, ctas), u1 = cut(cta + 1, U, ctas);
  {
    const int x = static_cast<int>(u0 / heads);
    if (x >= before && x < before + mine) {
      int b = sb0, pre = before;
      for (; b < sb1; ++b) {
        const int n = units_of(clamp_len(p, b));
        if (x < pre + n) break;
        pre += n;
      }
      s_start[0] = b;
      s_start[1] = pre;
    }
  }
  __syncthreads();
  int b = s_start[0];
  long long base = static_cast<long long>(s_start[1]) * heads;
  int4 my_desc = make_int4(-1, 0, 0, 0);

  uint8_t* ring = smem + warp * (kStages * W::SB);
  const uint32_t ring_s = smem_u32(ring);
  float* my_o = reinterpret_cast<float*>(ring);
  bool bad_page = false;

  for (long long u = u0; u < u1;) {
    const int len = clamp_len(p, b);
    const int nu = units_of(len);
    const long long local = u - base;
    if (local >= static_cast<long long>(nu) * heads) {
      base += static_cast<long long>(nu) * heads;
      ++b;
      continue;
    }
    const int hm = static_cast<int>(local / nu);
    const int c0 = static_cast<int>(local % nu);
    const int c1 = static_cast<int>(min(static_cast<long long>(nu), c0 + (u1 - u)));
    const int h = hm / p.mtiles, mt = hm % p.mtiles;
    const int row0 = h * p.group + mt * kRows;          // first query head of this product
    const int nrows = min(kRows, p.group - mt * kRows);

    // ---- tile copies
    const uint8_t* kb = p.k + h * p.head_bytes;
    const uint8_t* vb = p.v + h * p.head_bytes;
    const int* trow = p.table + b * p.table_ld;
    const int cpr_row = lane / W::CPR, cpr_c = lane % W::CPR;
    const bool append = p.k_new != nullptr && len > 0 && p.lens[b] <= p.max_blocks * p.page;
    const int ntiles = c1 - c0;
    auto pos_of = [&](int it) { return (c0 + it) * kUnit + warp * kTile + (lane & 15); };
    auto block_of = [&](int pos) { return p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page; };
    auto page_at = [&](int it) {
      const int pos = pos_of(it);
      return (it < ntiles && pos < len) ? __ldg(trow + block_of(pos)) : 0;
    };
    int pg = page_at(0);
    auto issue = [&](int it) {
      if (it < ntiles) {
        const int pos = pos_of(it);
        const bool in = pos < len;
        const bool ok = in && pg >= 0 && pg < p.n_pages;
        if (in && !ok) bad_page = true;
        const uint32_t off =
            ok ? static_cast<uint32_t>(pg) * p.page16 + static_cast<uint32_t>(pos - block_of(pos) * p.page) * p.tok16
               : kNoRow;
        const uint32_t mask = __ballot_sync(0xffffffffu, ok) & 0xffffu;
        const int stage = it % kStages;
        if (lane == 0) s_valid[warp][stage] = mask;
        const uint32_t dst = ring_s + stage * W::SB;
        const int arow = append ? len - 1 - (c0 + it) * kUnit - warp * kTile : -1;  // row of the new token, if here
        const bool here = arow >= 0 && arow < kTile && (mask >> arow & 1);
#pragma unroll
        for (int i = 0; i < W::NI; ++i) {
          const int r = i * W::RPI + cpr_row;
          const uint32_t o = __shfl_sync(0xffffffffu, off, r);
          const uint32_t sz = o == kNoRow ? 0u : 16u;
          const size_t src = o == kNoRow ? 0 : static_cast<size_t>(o) * 16 + cpr_c * 16;
          const uint32_t d = dst + W::at(r, cpr_c);
          if (here && r == arow) {
            const long long nb = b * p.n_b + h * p.n_h;
            if constexpr (!FP8) {
              const uint4 nk = reinterpret_cast<const uint4*>(p.k_new + nb)[cpr_c];
              const uint4 nv = reinterpret_cast<const uint4*>(p.v_new + nb)[cpr_c];
              *reinterpret_cast<uint4*>(ring + stage * W::SB + W::at(r, cpr_c)) = nk;
              *reinterpret_cast<uint4*>(ring + stage * W::SB + W::TB + W::at(r, cpr_c)) = nv;
              if (mt == 0) {
                *reinterpret_cast<uint4*>(const_cast<uint8_t*>(kb) + src) = nk;
                *reinterpret_cast<uint4*>(const_cast<uint8_t*>(vb) + src) = nv;
              }
            } else {
#pragma unroll
              for (int which = 0; which < 2; ++which) {
                const float sc = which ? (p.v_scale ? p.v_scale[h] : 1.f) : (p.k_scale ? p.k_scale[h] : 1.f);
                const __nv_bfloat16* x = (which ? p.v_new : p.k_new) + nb + cpr_c * 16;
                uint4 out;
                uint8_t* ob = reinterpret_cast<uint8_t*>(&out);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                  ob[e] = __nv_cvt_float_to_fp8(__bfloat162float(x[e]) / sc, __NV_SATFINITE, __NV_E4M3);
                *reinterpret_cast<uint4*>(ring + stage * W::SB + which * W::TB + W::at(r, cpr_c)) = out;
                if (mt == 0) *reinterpret_cast<uint4*>(const_cast<uint8_t*>(which ? vb : kb) + src) = out;
              }
            }
          } else {
            cp_async16(d, kb + src, sz);
            cp_async16(d + W::TB, vb + src, sz);
          }
        }
        pg = page_at(it + 1);
      }
      cp_commit();  // an empty group past the end keeps the count
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) issue(s);

    // ---- q of this product: 16 rows, rows past the group are zero
    uint32_t qf[W::KS][4];
    float sl0 = p.scale_log2, sl1 = p.scale_log2;  // per-row factor of the scores (rows g, g + 8)
    {
      const __nv_bfloat16* q0 = p.q + b * p.q_b + static_cast<long long>(row0 + g) * p.q_h;
      const __nv_bfloat16* q1 = q0 + 8 * p.q_h;
      const bool r0 = g < nrows, r1 = g + 8 < nrows;
      if constexpr (!FP8) {
#pragma unroll
        for (int ks = 0; ks < W::KS; ++ks) {
          const int d = ks * 16 + t4 * 2;
          qf[ks][0] = r0 ? *reinterpret_cast<const uint32_t*>(q0 + d) : 0u;
          qf[ks][1] = r1 ? *reinterpret_cast<const uint32_t*>(q1 + d) : 0u;
          qf[ks][2] = r0 ? *reinterpret_cast<const uint32_t*>(q0 + d + 8) : 0u;
          qf[ks][3] = r1 ? *reinterpret_cast<const uint32_t*>(q1 + d + 8) : 0u;
        }
      } else {
        // the k index of a product is any fixed order of the 16 dims: lane t4
        // takes dims 4 t4 .. 4 t4 + 3, the four e4m3 bytes it gets of a key row
        float m0 = 0.f, m1 = 0.f;
#pragma unroll
        for (int ks = 0; ks < W::KS; ++ks) {
          const int d = ks * 16 + t4 * 4;
          const uint2 x0 = r0 ? *reinterpret_cast<const uint2*>(q0 + d) : make_uint2(0, 0);
          const uint2 x1 = r1 ? *reinterpret_cast<const uint2*>(q1 + d) : make_uint2(0, 0);
          qf[ks][0] = x0.x;
          qf[ks][1] = x1.x;
          qf[ks][2] = x0.y;
          qf[ks][3] = x1.y;
          m0 = fmaxf(m0, fmaxf(fmaxf(fabsf(bf16_lo(x0.x)), fabsf(bf16_hi(x0.x))),
                               fmaxf(fabsf(bf16_lo(x0.y)), fabsf(bf16_hi(x0.y)))));
          m1 = fmaxf(m1, fmaxf(fmaxf(fabsf(bf16_lo(x1.x)), fabsf(bf16_hi(x1.x))),
                               fmaxf(fabsf(bf16_lo(x1.y)), fabsf(bf16_hi(x1.y)))));
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
          m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
        }
        // largest |q| of the row to [2^14, 2^15): a power of two, exact
        auto pow2_to = [](float m) {
          int e = 0;
          if (m > 0.f && m < INFINITY) frexpf(m, &e);  // m = f 2^e, f in [0.5, 1)
          return 15 - e;
        };
        const int e0 = pow2_to(m0), e1 = pow2_to(m1);
#pragma unroll
        for (int ks = 0; ks < W::KS; ++ks) {
          qf[ks][0] = pack_f16x2(ldexpf(bf16_lo(qf[ks][0]), e0), ldexpf(bf16_hi(qf[ks][0]), e0));
          qf[ks][1] = pack_f16x2(ldexpf(bf16_lo(qf[ks][1]), e1), ldexpf(bf16_hi(qf[ks][1]), e1));
          qf[ks][2] = pack_f16x2(ldexpf(bf16_lo(qf[ks][2]), e0), ldexpf(bf16_hi(qf[ks][2]), e0));
          qf[ks][3] = pack_f16x2(ldexpf(bf16_lo(qf[ks][3]), e1), ldexpf(bf16_hi(qf[ks][3]), e1));
        }
        const float ksc = p.k_scale ? p.k_scale[h] : 1.f;
        sl0 = ldexpf(p.scale_log2 * ksc, -e0);
        sl1 = ldexpf(p.scale_log2 * ksc, -e1);
      }
    }

    float acc[W::NT][4];
#pragma unroll
    for (int n = 0; n < W::NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;  // base-2 running max; this lane's share of the sum
    constexpr float kUp = FP8 ? 15.f : 0.f;                    // p is kept as 2^(y - m + kUp)

    for (int it = 0; it < ntiles; ++it) {
      cp_wait<kStages - 2>();
      __syncwarp();
      issue(it + kStages - 1);
      const int stage = it % kStages;
      const uint32_t valid = s_valid[warp][stage];
      if (valid == 0) continue;
      const uint32_t kt = ring_s + stage * W::SB, vt = kt + W::TB;

      // ---- scores: two n tiles of 8 keys
      float s[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      const int kr = (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;
      if constexpr (!FP8) {
#pragma unroll
        for (int ks = 0; ks < W::KS; ++ks) {
          uint32_t kf[4];
          ldsm4(kf, kt + W::at(kr, 2 * ks + kc));
          mma16816<false>(s[0], qf[ks], kf[0], kf[1]);
          mma16816<false>(s[1], qf[ks], kf[2], kf[3]);
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < W::KS / 2; ++kk) {  // 32 dims
          uint32_t kf[4];
          ldsm4(kf, kt + W::at(kr, 2 * kk + kc));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mma16816<true>(s[0], qf[2 * kk + e], e4m3x2_f16x2(kf[e] & 0xffff), e4m3x2_f16x2(kf[e] >> 16));
            mma16816<true>(s[1], qf[2 * kk + e], e4m3x2_f16x2(kf[2 + e] & 0xffff), e4m3x2_f16x2(kf[2 + e] >> 16));
          }
        }
      }
      // ---- running maximum and sum (base 2)
      float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const bool ok = valid >> (n * 8 + t4 * 2 + e) & 1;
          s[n][e] = ok ? s[n][e] * sl0 : -INFINITY;
          s[n][2 + e] = ok ? s[n][2 + e] * sl1 : -INFINITY;
          x0 = fmaxf(x0, s[n][e]);
          x1 = fmaxf(x1, s[n][2 + e]);
        }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, o));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, o));
      }
      if (__any_sync(0xffffffffu, x0 > m0 || x1 > m1)) {
        const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
        const float f0 = n0 == -INFINITY ? 1.f : ex2_approx(m0 - n0), f1 = n1 == -INFINITY ? 1.f : ex2_approx(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int n = 0; n < W::NT; ++n) {
          acc[n][0] *= f0;
          acc[n][1] *= f0;
          acc[n][2] *= f1;
          acc[n][3] *= f1;
        }
      }
      const float r0 = (m0 == -INFINITY ? 0.f : m0) - kUp, r1 = (m1 == -INFINITY ? 0.f : m1) - kUp;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[n][e] = ex2_approx(s[n][e] - r0);
          s[n][2 + e] = ex2_approx(s[n][2 + e] - r1);
          l0 += s[n][e];
          l1 += s[n][2 + e];
        }
      // ---- o += p v
      const int vr = (lane & 7) + (((lane >> 3) & 1) << 3), vc = lane >> 4;
      if constexpr (!FP8) {
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t hi = pack_bf16x2(s[n][2 * e], s[n][2 * e + 1]);
            ph[2 * n + e] = hi;
            pl[2 * n + e] = pack_bf16x2(s[n][2 * e] - bf16_lo(hi), s[n][2 * e + 1] - bf16_hi(hi));
          }
#pragma unroll
        for (int dd = 0; dd < HD / 16; ++dd) {
          uint32_t vf[4];
          ldsm4_t(vf, vt + W::at(vr, 2 * dd + vc));
          mma16816<false>(acc[2 * dd], ph, vf[0], vf[1]);
          mma16816<false>(acc[2 * dd + 1], ph, vf[2], vf[3]);
          mma16816<false>(acc[2 * dd], pl, vf[0], vf[1]);
          mma16816<false>(acc[2 * dd + 1], pl, vf[2], vf[3]);
        }
      } else {
        uint32_t ph[4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) ph[2 * n + e] = pack_f16x2(s[n][2 * e], s[n][2 * e + 1]);
        // a transposed 8x8 of 16-bit units holds, per key, two neighbouring
        // dims: n tile 2 dd takes the even dims of 16, tile 2 dd + 1 the odd ones
#pragma unroll
        for (int d2 = 0; d2 < HD / 32; ++d2) {
          uint32_t vf[4];
          ldsm4_t(vf, vt + W::at(vr, 2 * d2 + vc));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t a = __byte_perm(vf[2 * e], 0, 0x3120), c = __byte_perm(vf[2 * e + 1], 0, 0x3120);
            mma16816<true>(acc[4 * d2 + 2 * e], ph, e4m3x2_f16x2(a & 0xffff), e4m3x2_f16x2(c & 0xffff));
            mma16816<true>(acc[4 * d2 + 2 * e + 1], ph, e4m3x2_f16x2(a >> 16), e4m3x2_f16x2(c >> 16));
          }
        }
      }
    }
    cp_wait<0>();
    __syncwarp();

    // ---- the four warps' (max, sum, o) of this run, joined in shared memory
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, o);
      l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    }
    if (t4 == 0) {
      s_m[warp][g] = m0;
      s_m[warp][g + 8] = m1;
      s_l[warp][g] = l0;
      s_l[warp][g + 8] = l1;
    }
#pragma unroll
    for (int n = 0; n < W::NT; ++n) {
      if constexpr (!FP8) {
        if (g < nrows) *reinterpret_cast<float2*>(my_o + g * OS + n * 8 + t4 * 2) = make_float2(acc[n][0], acc[n][1]);
        if (g + 8 < nrows)
          *reinterpret_cast<float2*>(my_o + (g + 8) * OS + n * 8 + t4 * 2) = make_float2(acc[n][2], acc[n][3]);
      } else if ((n & 1) == 0) {
        if (g < nrows)
          *reinterpret_cast<float4*>(my_o + g * OS + n * 8 + t4 * 4) =
              make_float4(acc[n][0], acc[n + 1][0], acc[n][1], acc[n + 1][1]);
        if (g + 8 < nrows)
          *reinterpret_cast<float4*>(my_o + (g + 8) * OS + n * 8 + t4 * 4) =
              make_float4(acc[n][2], acc[n + 1][2], acc[n][3], acc[n + 1][3]);
      }
    }
    __syncthreads();
    const bool first = c0 == 0, last = c1 == nu;
    const int slot = static_cast<int>(2 * cta) + (first ? 1 : 0);  // a run that began earlier goes to slot 0
    if (first && !last) {
      const long long end = u - c0 + nu;  // unit after this (sequence, head)'s last
      my_desc = make_int4(b, hm, static_cast<int>((end * ctas - 1) / U), 0);
    }
    const float vsc = (FP8 && p.v_scale) ? p.v_scale[h] : 1.f;
    for (int i = tid; i < nrows * HD; i += kThreads) {
      const int r = i / HD, d = i % HD;
      float M = s_m[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) M = fmaxf(M, s_m[w][r]);
      const float ref = M == -INFINITY ? 0.f : M;
      float L = 0.f, O = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2_approx(s_m[w][r] - ref);
        L += f * s_l[w][r];
        O += f * reinterpret_cast<const float*>(smem + w * (kStages * W::SB))[r * OS + d];
      }
      if (first && last) {
        p.o[b * p.o_b + (row0 + r) * p.o_h + d] = __float2bfloat16_rn(L == 0.f ? 0.f : O / L * vsc);
        if (d == 0 && p.lse)
          p.lse[b * p.lse_b + row0 + r] = L == 0.f ? -INFINITY : (M + log2f(L) - kUp) * kLn2;
      } else {
        p.part_o[(static_cast<long long>(slot) * p.rows + r) * HD + d] = O;
        if (d == 0) p.part_ml[static_cast<long long>(slot) * p.rows + r] = make_float2(M, L);
      }
    }
    __syncthreads();  // the next run's copies overwrite the warps' o
    u += c1 - c0;
  }
  if (tid == 0) p.desc[cta] = my_desc;
  if (bad_page && p.err) atomicExch(p.err, kErrPage);
}

// Joins the partials of each (sequence, head) that more than one CTA worked on:
// block j does the one that began in CTA j's range and went on past its end,
// in the order of the cache.  grid.y splits its rows.
template <int HD, bool FP8>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Params p) {
  constexpr int LPR = HD / 4;                     // lanes (of float4) that cover a row
  constexpr int GR = kJoinThreads / LPR;          // groups of lanes
  constexpr float kUp = FP8 ? 15.f : 0.f;
  __shared__ float4 s_o[GR][LPR];
  __shared__ float s_ml[GR];
  griddep_sync();
  const int j = blockIdx.x;
  const int4 d = p.desc[j];
  if (d.x < 0) return;
  const int b = d.x, h = d.y / p.mtiles, mt = d.y % p.mtiles, n = d.z - j + 1;
  const int nrows = min(kRows, p.group - mt * kRows);
  const int row0 = h * p.group + mt * kRows;
  const int li = threadIdx.x % LPR, gi = threadIdx.x / LPR;
  // partial i of this segment: slot 2 j + 1, then slot 0 of the CTAs that follow
  auto slot = [&](int i) { return i == 0 ? 2LL * j + 1 : 2LL * (j + i); };
  for (int r = blockIdx.y; r < nrows; r += gridDim.y) {
    float M = -INFINITY;
    for (int i = threadIdx.x % 32; i < n; i += 32) M = fmaxf(M, p.part_ml[slot(i) * p.rows + r].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = gi; i < n; i += GR) {
      const float2 ml = p.part_ml[slot(i) * p.rows + r];
      const float4 x = reinterpret_cast<const float4*>(p.part_o + (slot(i) * p.rows + r) * HD)[li];
      const float f = ex2_approx(ml.x - ref);
      L += f * ml.y;
      O.x += f * x.x;
      O.y += f * x.y;
      O.z += f * x.z;
      O.w += f * x.w;
    }
    __syncthreads();
    s_o[gi][li] = O;
    if (li == 0) s_ml[gi] = L;
    __syncthreads();
    if (gi == 0) {
      for (int i = 1; i < GR; ++i) {
        const float4 x = s_o[i][li];
        O.x += x.x;
        O.y += x.y;
        O.z += x.z;
        O.w += x.w;
        L += s_ml[i];
      }
      const float vsc = (FP8 && p.v_scale) ? p.v_scale[h] : 1.f;
      const float inv = L == 0.f ? 0.f : vsc / L;
      __nv_bfloat16* out = p.o + b * p.o_b + (row0 + r) * p.o_h + li * 4;
      // (L is 0 only where every key was left out: o is then 0 as well)
      out[0] = __float2bfloat16_rn(O.x * inv);
      out[1] = __float2bfloat16_rn(O.y * inv);
      out[2] = __float2bfloat16_rn(O.z * inv);
      out[3] = __float2bfloat16_rn(O.w * inv);
      if (li == 0 && p.lse)
        p.lse[b * p.lse_b + row0 + r] = L == 0.f ? -INFINITY : (M + log2f(L) - kUp) * kLn2;
    }
  }
}

// Resident CTAs of an SM, asked once per device (0: the query failed).
template <int HD, bool FP8>
int ctas_per_sm() {
  constexpr int smem = kWarps * kStages * Warp<HD, FP8>::SB;
  constexpr int kMaxDev = 64;
  static int known[kMaxDev] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return 0;
  if (known[dev] == 0) {
    int k = 0;
    if (cudaFuncSetAttribute(decode_kernel<HD, FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
            cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&k, decode_kernel<HD, FP8>, kThreads, smem) != cudaSuccess)
      return 0;
    known[dev] = k;
  }
  return known[dev];
}

// CTAs of a call: what the card holds at once, or fewer where even full block
// tables have fewer units.
template <int HD, bool FP8>
int grid_of(int B, int Hk, int mtiles, int max_blocks, int page) {
  const int occ = ctas_per_sm<HD, FP8>();
  if (occ <= 0) return 0;
  const long long most = static_cast<long long>(B) * Hk * mtiles *
                         ((static_cast<long long>(max_blocks) * page + kUnit - 1) / kUnit);
  const long long card = static_cast<long long>(sm_count()) * occ;
  return static_cast<int>(most < card ? most : card);
}

template <int HD, bool FP8>
int launch(Params& p, cudaStream_t stream) {
  constexpr int smem = kWarps * kStages * Warp<HD, FP8>::SB;
  const int grid = grid_of<HD, FP8>(p.B, p.Hk, p.mtiles, p.max_blocks, p.page);
  if (grid <= 0) return NL_ERR_CUDA;
  launch_kernel(decode_kernel<HD, FP8>, dim3(grid), dim3(kThreads), smem, stream, 1, p);
  const int st = launch_status();
  if (st != NL_OK || static_cast<long long>(p.max_blocks) * p.page <= kUnit) return st;  // one unit each: no partials
  // few (sequence, head) pairs: many partials each, so their rows are split over blocks too
  const int ysplit = static_cast<long long>(p.B) * p.Hk * p.mtiles <= 16 ? p.rows : 1;
  launch_kernel(join_kernel<HD, FP8>, dim3(grid, ysplit), dim3(kJoinThreads), 0, stream, 1, p);
  return launch_status();
}

}  // namespace pa
}  // namespace nl

using namespace nl;

namespace {
size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
// Workspace for the most CTAs a call can use: partials and descriptors.
size_t paged_ws(int rows, int d, int ctas, size_t* ml, size_t* desc) {
  size_t n = align256(static_cast<size_t>(2) * ctas * rows * d * sizeof(float));
  if (ml) *ml = n;
  n += align256(static_cast<size_t>(2) * ctas * rows * sizeof(float2));
  if (desc) *desc = n;
  return n + align256(static_cast<size_t>(ctas) * sizeof(int4));
}
int paged_grid(int d, int dtype, int B, int Hk, int mtiles, int max_blocks, int page) {
  if (d == 64)
    return dtype == NL_E4M3 ? pa::grid_of<64, true>(B, Hk, mtiles, max_blocks, page)
                            : pa::grid_of<64, false>(B, Hk, mtiles, max_blocks, page);
  return dtype == NL_E4M3 ? pa::grid_of<128, true>(B, Hk, mtiles, max_blocks, page)
                          : pa::grid_of<128, false>(B, Hk, mtiles, max_blocks, page);
}
bool paged_shape_ok(int B, int Hq, int Hk, int d, int page, int max_blocks) {
  return B > 0 && Hq > 0 && Hk > 0 && Hq % Hk == 0 && (d == 64 || d == 128) && page > 0 && max_blocks > 0 &&
         static_cast<long long>(max_blocks) * page <= INT32_MAX - pa::kUnit &&
         B * ((static_cast<long long>(max_blocks) * page + pa::kUnit - 1) / pa::kUnit) <= INT32_MAX;
}
}  // namespace

extern "C" size_t nl_paged_attention_workspace_bytes(int B, int Hq, int Hk, int d, int page_size, int max_blocks,
                                                     int cache_dtype) {
  if (!paged_shape_ok(B, Hq, Hk, d, page_size, max_blocks)) return 0;
  const int group = Hq / Hk, rows = group < pa::kRows ? group : pa::kRows;
  const int grid = paged_grid(d, cache_dtype, B, Hk, (group + pa::kRows - 1) / pa::kRows, max_blocks, page_size);
  return grid <= 0 ? 0 : paged_ws(rows, d, grid, nullptr, nullptr);
}

extern "C" int nl_paged_attention(const void* q, long long q_b, long long q_h, void* k_cache, void* v_cache,
                                  int cache_dtype, long long page_stride, long long head_stride,
                                  long long tok_stride, const int* block_table, long long table_ld, const int* lens,
                                  const void* k_new, const void* v_new, long long n_b, long long n_h,
                                  const float* k_scale, const float* v_scale, float scale, void* o, long long o_b,
                                  long long o_h, float* lse, long long lse_b, void* workspace, size_t ws_bytes, int B,
                                  int Hq, int Hk, int d, int page_size, int max_blocks, int n_pages,
                                  cudaStream_t stream) {
  if (!paged_shape_ok(B, Hq, Hk, d, page_size, max_blocks) || n_pages <= 0 || table_ld < max_blocks)
    return NL_ERR_SHAPE;
  if (cache_dtype != NL_BF16 && cache_dtype != NL_E4M3) return NL_ERR_DTYPE;
  if (!q || !k_cache || !v_cache || !block_table || !lens || !o || (k_new != nullptr) != (v_new != nullptr))
    return NL_ERR_SHAPE;
  if (page_stride <= 0 || tok_stride <= 0 || head_stride < 0 || q_b < 0 || q_h < 0 || n_b < 0 || n_h < 0)
    return NL_ERR_SHAPE;
  const int el = cache_dtype == NL_E4M3 ? 1 : 2;
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) |
                         reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(k_new) |
                         reinterpret_cast<uintptr_t>(v_new);
  if ((ptrs & 15) || ((q_b | q_h | n_b | n_h) & 7) || ((page_stride | head_stride | tok_stride) * el & 15) ||
      (reinterpret_cast<uintptr_t>(workspace) & 255))
    return NL_ERR_ALIGN;
  // rows are addressed inside one head by 32-bit offsets of 16 bytes: 64 GB of each cache
  const long long extent = (n_pages - 1) * (page_stride * el / 16) + (page_size - 1) * (tok_stride * el / 16);
  if (page_stride * el / 16 > UINT32_MAX || tok_stride * el / 16 > UINT32_MAX || extent >= UINT32_MAX)
    return NL_ERR_TOO_LARGE;
  const int group = Hq / Hk;
  pa::Params p;
  p.rows = group < pa::kRows ? group : pa::kRows;
  p.mtiles = (group + pa::kRows - 1) / pa::kRows;
  const int grid = paged_grid(d, cache_dtype, B, Hk, p.mtiles, max_blocks, page_size);
  if (grid <= 0) return NL_ERR_CUDA;
  size_t ml, desc;
  if (!workspace || ws_bytes < paged_ws(p.rows, d, grid, &ml, &desc)) return NL_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float2*>(ws + ml);
  p.desc = reinterpret_cast<int4*>(ws + desc);
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_b = q_b;
  p.q_h = q_h;
  p.k = static_cast<uint8_t*>(k_cache);
  p.v = static_cast<uint8_t*>(v_cache);
  p.page16 = static_cast<uint32_t>(page_stride * el / 16);
  p.tok16 = static_cast<uint32_t>(tok_stride * el / 16);
  p.head_bytes = head_stride * el;
  p.table = block_table;
  p.table_ld = table_ld;
  p.lens = lens;
  p.k_new = static_cast<const __nv_bfloat16*>(k_new);
  p.v_new = static_cast<const __nv_bfloat16*>(v_new);
  p.n_b = n_b;
  p.n_h = n_h;
  p.k_scale = cache_dtype == NL_E4M3 ? k_scale : nullptr;
  p.v_scale = cache_dtype == NL_E4M3 ? v_scale : nullptr;
  p.o = static_cast<__nv_bfloat16*>(o);
  p.o_b = o_b;
  p.o_h = o_h;
  p.lse = lse;
  p.lse_b = lse_b;
  p.B = B;
  p.Hq = Hq;
  p.Hk = Hk;
  p.group = group;
  p.page = page_size;
  p.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
  p.max_blocks = max_blocks;
  p.n_pages = n_pages;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.err = device_error_word();
  if (d == 64) return cache_dtype == NL_E4M3 ? pa::launch<64, true>(p, stream) : pa::launch<64, false>(p, stream);
  return cache_dtype == NL_E4M3 ? pa::launch<128, true>(p, stream) : pa::launch<128, false>(p, stream);
}
