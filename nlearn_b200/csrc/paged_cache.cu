// paged_cache.cu — the bookkeeping of a paged key-value cache: block tables and
// slot maps built from request lengths, and the write of keys and values into
// their slots.  No reference counterpart (nlearn keeps no cache).
//
// update_tables_kernel: one serving step.  With len0 = 0 for rows that ended and
// up(x) = ceil(x / P):
//   freed pages  the up(len) pages of each row that ended go on top of the
//                stack of free pages, row after row;
//   taken pages  row b takes up(len0 + new) - up(len0) pages from the top, at
//                the prefix sum of the rows before it; a row whose pages do not
//                all fit is refused and takes none, and so is every later row
//                that needs pages (the prefix sums only grow);
//   slots        token i of the flat list (rows back to back, by the prefix sum
//                of new) has slot page * P + pos % P.
// All of it is prefix sums over the rows, which every CTA of the one cluster
// makes for itself, so the CTAs share no state but the two sides of the
// cluster barrier: lengths, stack and tables are read before it and rewritten
// after it (the outputs may then be the inputs).
// Bound by latency: one launch, and a chain of five loads (lengths, freed pages, taken
// pages, the slots' pages; each with all of a thread's loads in flight) and
// two prefix sums.  256 rows of one token: 5.9 us; 96 prompts, 109000 slots: 9.9 us
// (8 CTAs; up to 4096 slots one CTA does them without a cluster barrier).
//
// kv_write_kernel: a thread per 16 bytes of a key row and of its value row.
// Bound by HBM: each element is read and written once.
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "host_common.h"
#include "sm100.cuh"

namespace nl {
namespace pc {

constexpr int kThreads = 1024;
constexpr int kMaxRows = 8192;  // rows of a block table: 20 bytes of shared memory each

enum : int { kOk = 0, kNoPages = 1, kTooLong = 2, kNoSlots = 3, kInvalid = 4 };  // status of a row
enum : int { kErrPage = 4 };                                                      // device error word

struct TableParams {
  int* table;
  long long ld;
  const int* lens;
  const int* new_lens;
  const int* done;  // may be null: no row ended
  int* free_pages;
  const int* n_free;
  int* lens_out;
  int* n_free_out;
  int* slots;
  int* positions;
  int* cu;
  int* status;
  int B, max_blocks, page, page_shift, n_pages, tokens;
};

// Exclusive prefix sums of two values per thread over the block, and their
// totals.  Every warp sums the warps' totals for itself: one barrier, and one
// before s_sum may be written again.
struct Two {
  long long a, b;
};
__device__ __forceinline__ Two warp_scan(Two v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, v.a, o), y = __shfl_up_sync(0xffffffffu, v.b, o);
    if (lane >= o) {
      v.a += x;
      v.b += y;
    }
  }
  return v;
}
__device__ __forceinline__ Two block_scan(Two v, Two* s_sum, Two& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const Two inc = warp_scan(v);
  if (lane == 31) s_sum[warp] = inc;
  __syncthreads();
  const Two w = warp_scan(lane < warps ? s_sum[lane] : Two{0, 0});
  total = {__shfl_sync(0xffffffffu, w.a, 31), __shfl_sync(0xffffffffu, w.b, 31)};
  const int prev = warp > 0 ? warp - 1 : 0;
  const long long pa = __shfl_sync(0xffffffffu, w.a, prev), pb = __shfl_sync(0xffffffffu, w.b, prev);
  return {inc.a - v.a + (warp > 0 ? pa : 0), inc.b - v.b + (warp > 0 ? pb : 0)};
}

// A warp copies n entries, dst[i] = src[step i], with four loads of a lane in flight.
__device__ __forceinline__ void move_pages(int* dst, const int* src, int n, int step) {
  for (int i0 = threadIdx.x & 31; i0 < n; i0 += 128) {
    int x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = i0 + 32 * k < n ? __ldcg(src + step * (i0 + 32 * k)) : 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i0 + 32 * k < n) dst[i0 + 32 * k] = x[k];
  }
}

__device__ __forceinline__ int sat(long long x) { return x > INT32_MAX ? INT32_MAX : static_cast<int>(x); }

template <bool CLUSTER>
__global__ void __launch_bounds__(kThreads) update_tables_kernel(const TableParams p) {
  extern __shared__ int4 s_row[];  // {first token, len0 or -1 if refused, first page from the top, pages held}
  int* s_new = reinterpret_cast<int*>(s_row + p.B);  // tokens a row grows by
  __shared__ Two s_sum[3][32];
  __shared__ int s_used;
  const int tid = threadIdx.x, lane = tid & 31, threads = blockDim.x;
  const int rank = blockIdx.x, nctas = gridDim.x;
  if (tid == 0) s_used = 0;
  griddep_sync();

  const int P = p.page;
  const long long cap = static_cast<long long>(p.max_blocks) * P;
  // pages of x tokens, page of position x (x >= 0; sums stay below 2^32)
  auto block_of = [&](unsigned x) {
    return static_cast<int>(p.page_shift >= 0 ? x >> p.page_shift : x / static_cast<unsigned>(P));
  };
  auto up = [&](int x) { return block_of(static_cast<unsigned>(x) + static_cast<unsigned>(P - 1)); };
  const int stack0 = max(0, min(*p.n_free, p.n_pages));
  const int warps = nctas * (threads / 32), gw = rank * (threads / 32) + (tid >> 5);

  // ---- first tokens, and the pages of rows that ended
  long long tok = 0, freed = 0;
  int turn = 0;  // consecutive scans use different sums: one barrier each
  for (int b0 = 0; b0 < p.B; b0 += threads) {
    const int b = b0 + tid;
    int n = 0, back = 0, len = 0;
    if (b < p.B) {
      len = p.lens[b];
      n = p.new_lens[b];
      if (p.done && p.done[b] && len > 0 && len <= cap) back = up(len);
      s_new[b] = n;
      n = max(0, n);
    }
    Two t;
    const Two at = block_scan({n, back}, s_sum[turn], t);
    turn = turn == 2 ? 0 : turn + 1;
    if (b < p.B) {
      s_row[b] = make_int4(sat(tok + at.a), len, sat(freed + at.b), back);
      if (rank == 0) p.cu[b] = sat(tok + at.a);
    }
    tok += t.a;
    freed += t.b;
  }
  if (rank == 0 && tid == 0) p.cu[p.B] = sat(tok);
  if (freed > 0) {  // (the same in every thread)
    __syncthreads();
    // a lane looks at a row, the warp moves its pages; neighbouring rows belong to different warps
    for (int b0 = gw; b0 < p.B; b0 += warps * 32) {
      const int mine = b0 + lane * warps;
      uint32_t m = __ballot_sync(0xffffffffu, mine < p.B && s_row[mine].w > 0);
      for (; m; m &= m - 1) {
        const int b = b0 + (__ffs(m) - 1) * warps;
        const int4 r = s_row[b];
        // (entries past the stack's capacity, which only pages freed twice can make, are dropped)
        const long long at = static_cast<long long>(stack0) + r.z;
        if (at < p.n_pages)
          move_pages(p.free_pages + at, p.table + b * p.ld,
                     static_cast<int>(min(static_cast<long long>(r.w), p.n_pages - at)), 1);
      }
    }
    __syncthreads();
  }
  const int avail = static_cast<int>(min(static_cast<long long>(p.n_pages), stack0 + freed));

  // ---- refusals and the pages each row takes (from the top of the stack)
  long long taken = 0;
  int used = 0;  // pages taken by this thread's rows that were not refused
  for (int b0 = 0; b0 < p.B; b0 += threads) {
    const int b = b0 + tid;
    int st = kOk, len0 = 0, n = 0, take = 0, first = 0;
    if (b < p.B) {
      const int4 r = s_row[b];
      const int len = r.y;
      first = r.x;
      n = s_new[b];
      const bool bad = len < 0 || len > cap;
      len0 = r.w > 0 ? 0 : len;  // (a row that ended with no page had no token)
      if (bad || n < 0) st = kInvalid;
      else if (static_cast<long long>(len0) + n > cap) st = kTooLong;
      else if (n > 0 && static_cast<long long>(first) + n > p.tokens) st = kNoSlots;
      if (st == kOk) take = up(len0 + n) - up(len0);
    }
    Two t;
    const Two off = block_scan({take, 0}, s_sum[turn], t);
    turn = turn == 2 ? 0 : turn + 1;
    if (b < p.B) {
      const long long at = taken + off.a;
      if (take > 0 && at + take > avail) st = kNoPages;
      if (st != kOk) take = 0;
      used += take;
      s_row[b] = make_int4(first, st == kOk ? len0 : -1, sat(at), st == kOk ? up(len0) : 0);
      if (rank == 0) p.status[b] = st;
    }
    taken += t.a;
  }
  if (used) atomicAdd(&s_used, used);
  if constexpr (CLUSTER) cluster_sync();  // stack written, lengths and stack size read by every CTA
  else __syncthreads();

  // ---- the taken pages into the tables, new lengths
  const int* top = p.free_pages + avail - 1;
  for (int b0 = gw; b0 < p.B; b0 += warps * 32) {
    // rows that take one page, as most do in a decode step: a lane each; the others one after the other
    const int mine = b0 + lane * warps;
    int take = 0;
    if (mine < p.B) {
      const int4 r = s_row[mine];
      if (r.y >= 0) take = up(r.y + s_new[mine]) - r.w;
      if (take == 1) p.table[mine * p.ld + r.w] = __ldcg(top - r.z);
    }
    uint32_t m = __ballot_sync(0xffffffffu, take > 1);
    for (; m; m &= m - 1) {
      const int src = __ffs(m) - 1, b = b0 + src * warps, n = __shfl_sync(0xffffffffu, take, src);
      const int4 r = s_row[b];
      move_pages(p.table + b * p.ld + r.w, top - r.z, n, -1);
    }
  }
  if (rank == 0) {
    for (int b = tid; b < p.B; b += threads) {
      const int4 r = s_row[b];
      if (r.y >= 0) {
        p.lens_out[b] = r.y + s_new[b];
      } else {  // refused: a row that ended still gave its pages back
        const int old = p.lens[b];
        p.lens_out[b] = (p.done && p.done[b] && old >= 0 && old <= cap) ? 0 : old;
      }
    }
    if (tid == 0) *p.n_free_out = avail - s_used;
  }

  // ---- slots, four tokens a thread
  const bool vec = ((reinterpret_cast<uintptr_t>(p.slots) | reinterpret_cast<uintptr_t>(p.positions)) & 15) == 0;
  // (unsigned: the last step may pass 2^31)
  for (unsigned t0 = 4 * (rank * threads + tid); t0 < static_cast<unsigned>(p.tokens); t0 += 4 * nctas * threads) {
    const int t = static_cast<int>(t0);
    int slot[4], pos[4];
    int lo = 0;
    if (t < tok) {
      int hi = p.B - 1;  // last row whose first token is not after t
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_row[mid].x <= t) lo = mid;
        else hi = mid - 1;
      }
    }
    int4 r = s_row[lo];
    int next = lo + 1 < p.B ? s_row[lo + 1].x : INT32_MAX;
    const int* entry[4];  // where a token's page stands: all four before the first is read
    int off[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      pos[k] = -1;
      off[k] = 0;
      entry[k] = nullptr;
      if (t + k >= tok || t + k >= p.tokens) continue;
      while (t + k >= next) {
        r = s_row[++lo];
        next = lo + 1 < p.B ? s_row[lo + 1].x : INT32_MAX;
      }
      if (r.y < 0) continue;
      pos[k] = r.y + t + k - r.x;
      const int blk = block_of(pos[k]);
      off[k] = pos[k] - blk * P;
      // (pages already held are not rewritten by this call; the others come off the stack)
      entry[k] = blk < r.w ? p.table + lo * p.ld + blk : top - r.z - (blk - r.w);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) slot[k] = entry[k] ? __ldcg(entry[k]) : -1;
#pragma unroll
    for (int k = 0; k < 4; ++k) slot[k] = slot[k] >= 0 && slot[k] < p.n_pages ? slot[k] * P + off[k] : -1;
    if (vec && t <= p.tokens - 4) {
      *reinterpret_cast<int4*>(p.slots + t) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<int4*>(p.positions + t) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (t + k < p.tokens) {
          p.slots[t + k] = slot[k];
          p.positions[t + k] = pos[k];
        }
    }
  }
}

struct WriteParams {
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  long long n_t, n_h;  // token and head strides (elements)
  uint8_t* kc;
  uint8_t* vc;
  long long page_bytes, head_bytes, tok_bytes;
  const int* slots;
  const float* k_scale;  // [Hk], e4m3 only
  const float* v_scale;
  int T, Hk, cpr, page;
  long long n_slots;
  int* err;
};

template <bool FP8>
__device__ __forceinline__ uint4 convert(const __nv_bfloat16* x, float scale) {
  if constexpr (!FP8) {
    return *reinterpret_cast<const uint4*>(x);
  } else {
    uint4 in[2] = {reinterpret_cast<const uint4*>(x)[0], reinterpret_cast<const uint4*>(x)[1]};
    const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(in);
    uint4 out;
    uint8_t* o = reinterpret_cast<uint8_t*>(&out);
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = __nv_cvt_float_to_fp8(__bfloat162float(e[i]) / scale, __NV_SATFINITE, __NV_E4M3);
    return out;
  }
}

template <bool FP8>
__global__ void __launch_bounds__(256) kv_write_kernel(const WriteParams p) {
  griddep_sync();
  const int per_tok = p.Hk * p.cpr;
  const long long n = static_cast<long long>(p.T) * per_tok;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    const int t = static_cast<int>(i / per_tok), r = static_cast<int>(i - static_cast<long long>(t) * per_tok);
    const int h = r / p.cpr, c = r - h * p.cpr;
    const int slot = p.slots[t];
    if (slot < 0) continue;  // padding
    if (slot >= p.n_slots) {
      if (p.err) atomicExch(p.err, kErrPage);
      continue;
    }
    const int page = slot / p.page, off = slot - page * p.page;
    const long long src = t * p.n_t + h * p.n_h + c * (FP8 ? 16 : 8);
    const long long dst = page * p.page_bytes + h * p.head_bytes + off * p.tok_bytes + c * 16;
    const uint4 kx = convert<FP8>(p.k + src, FP8 && p.k_scale ? p.k_scale[h] : 1.f);
    const uint4 vx = convert<FP8>(p.v + src, FP8 && p.v_scale ? p.v_scale[h] : 1.f);
    *reinterpret_cast<uint4*>(p.kc + dst) = kx;
    *reinterpret_cast<uint4*>(p.vc + dst) = vx;
  }
}

}  // namespace pc
}  // namespace nl

using namespace nl;

extern "C" int nl_update_block_tables(const nl_update_block_tables_args* args, cudaStream_t stream) {
  if (!args) return NL_ERR_SHAPE;
  const nl_update_block_tables_args& a = *args;
  const int B = a.B, n_tokens = a.n_tokens;
  if (B <= 0 || B > pc::kMaxRows || a.max_blocks <= 0 || a.page_size <= 0 || a.n_pages <= 0 || n_tokens < 0 ||
      a.table_ld < a.max_blocks || static_cast<long long>(a.max_blocks) * a.page_size > INT32_MAX ||
      static_cast<long long>(a.n_pages) * a.page_size > INT32_MAX)
    return NL_ERR_SHAPE;
  if (!a.block_table || !a.lens || !a.new_lens || !a.free_pages || !a.n_free || !a.lens_out || !a.n_free_out ||
      !a.cu || !a.status || (n_tokens > 0 && (!a.slots || !a.positions)))
    return NL_ERR_SHAPE;
  pc::TableParams p{a.block_table, a.table_ld, a.lens, a.new_lens, a.done, a.free_pages, a.n_free, a.lens_out,
                    a.n_free_out, a.slots, a.positions, a.cu, a.status, B, a.max_blocks, a.page_size,
                    (a.page_size & (a.page_size - 1)) == 0 ? __builtin_ctz(a.page_size) : -1, a.n_pages, n_tokens};
  const size_t smem = static_cast<size_t>(B) * (sizeof(int4) + sizeof(int));
  // one CTA of half as many threads again as rows or fours of tokens need (the pages of rows that ended are moved
  // a warp to a row: 256 rows of which 3 % end, 256 threads 6.3 us, 384 5.9, 512 6.4); a cluster of 8 for long lists
  const bool wide = n_tokens > 4 * pc::kThreads;
  const int need = B > n_tokens / 4 ? B : n_tokens / 4;
  const int more = (need + need / 2 + 31) / 32 * 32;
  const int threads = wide || more >= pc::kThreads ? pc::kThreads : more <= 128 ? 128 : more;
  auto kern = wide ? pc::update_tables_kernel<true> : pc::update_tables_kernel<false>;
  if (smem > 40 * 1024 &&
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
    return NL_ERR_LAUNCH;
  const int ctas = wide ? 8 : 1;
  launch_kernel(kern, dim3(ctas), dim3(threads), smem, stream, ctas, p);
  return launch_status();
}

extern "C" int nl_paged_kv_write(const nl_paged_kv_write_args* args, cudaStream_t stream) {
  if (!args) return NL_ERR_SHAPE;
  const nl_paged_kv_write_args& a = *args;
  const int T = a.T, Hk = a.Hk, d = a.d, page_size = a.page_size, n_pages = a.n_pages, cache_dtype = a.cache_dtype;
  const long long n_t = a.n_t, n_h = a.n_h;
  const long long page_stride = a.page_stride, head_stride = a.head_stride, tok_stride = a.tok_stride;
  if (T <= 0 || Hk <= 0 || d <= 0 || page_size <= 0 || n_pages <= 0 || !a.k || !a.v || !a.k_cache || !a.v_cache ||
      !a.slots || n_t < 0 || n_h < 0 || page_stride <= 0 || head_stride < 0 || tok_stride <= 0)
    return NL_ERR_SHAPE;
  if (cache_dtype != NL_BF16 && cache_dtype != NL_E4M3) return NL_ERR_DTYPE;
  const bool fp8 = cache_dtype == NL_E4M3;
  const int el = fp8 ? 1 : 2, per = fp8 ? 16 : 8;  // elements of a 16-byte store
  if (d % per || static_cast<long long>(Hk) * (d / per) > INT32_MAX) return NL_ERR_SHAPE;
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                         reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache);
  if ((ptrs & 15) || ((n_t | n_h) & 7) || ((page_stride | head_stride | tok_stride) * el & 15)) return NL_ERR_ALIGN;
  pc::WriteParams p{static_cast<const __nv_bfloat16*>(a.k), static_cast<const __nv_bfloat16*>(a.v), n_t, n_h,
                    static_cast<uint8_t*>(a.k_cache), static_cast<uint8_t*>(a.v_cache), page_stride * el,
                    head_stride * el, tok_stride * el, a.slots, a.k_scale, a.v_scale, T, Hk, d / per, page_size,
                    static_cast<long long>(n_pages) * page_size, device_error_word()};
  const long long n = static_cast<long long>(T) * Hk * (d / per);
  long long blocks = (n + 255) / 256;
  const long long most = static_cast<long long>(sm_count()) * 32;
  if (blocks > most) blocks = most;
  launch_kernel(fp8 ? pc::kv_write_kernel<true> : pc::kv_write_kernel<false>, dim3(static_cast<int>(blocks)),
                dim3(256), 0, stream, 1, p);
  return launch_status();
}
