// logits.cu — what a sampler does to logits before it draws: penalties for
// repeated tokens, additive biases, and a mask of allowed tokens.
//
// Row b, column v, in this order (each part may be absent):
//   x = x > 0 ? x / r : x * r              if v occurs among the row's tokens
//   x = x - f c - a                        if v was generated c > 0 times (tokens after the prompt)
//   x = x + sum of the row's biases of v   (in list order)
//   x = -inf                               if bit v of the row's mask is 0
// No reference counterpart (nlearn/model.py:440-444 samples the raw logits).
//
// Bound: HBM, one read and one write of the logits.  A CTA owns a chunk of one
// row's columns.  The chunk comes into shared memory by asynchronous copies;
// meanwhile the row's tokens that fall into it are counted there (integer
// atomics: the order does not matter), and the first that comes to a column puts
// the column on a list.  The list is then worked off with all lanes busy, on the
// copy in shared memory, and the chunk is written once, with the mask.  (With the
// rules inside a pass over all columns nearly every warp held a named one and
// took the long way; with the list worked off in global memory its scattered
// 2-byte accesses were the longest part: 36 and 27 us for 256 rows of 50257 in
// bf16 with 2048 tokens each; now 17.3.)  In place and without a mask a row with
// few tokens is not copied: only the columns on its list are read and written.
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "host_common.h"
#include "sm100.cuh"

namespace nl {
namespace lg {

// Every chunk of a row looks through all of the row's tokens, so chunks are large; two CTAs to an SM, so that one's
// copies run beside the other's counting (256 rows of 50257 in bf16, 2048 tokens each, threads x CTAs of an SM:
// 512 x 2 17.3 us, 1024 x 1 18.2, 384 x 3 21.5, 256 x 4 21.2, 128 x 8 28.3).
constexpr int kThreads = 512;
constexpr int kCtas = 2;              // resident CTAs of an SM: registers and shared memory are kept for them
constexpr int kList = 128;            // biases of a row that are kept in shared memory
constexpr int kSmem = 111 * 1024;     // dynamic shared memory of a CTA: kCtas of them fit an SM
// In place and without a mask: bytes of the row to a column on the list from which the list is worked off in
// global memory, a sector read and written for each.  In place / through shared memory, 256 rows of 50257, us:
// bf16 with 512 tokens 7.5 / 13.2, 1024 12.9 / 13.6, 2048 20.0 / 14.3; f32 1024 14.6 / 21.3, 2048 22.9 / 22.1.
constexpr int kFew = 96;

// A column's word: how often it was generated, and two flags.
template <typename C>
struct Word {
  static constexpr int BITS = 8 * sizeof(C);
  static constexpr uint32_t kSeen = 1u << (BITS - 1);   // occurs in the prompt
  static constexpr uint32_t kNamed = 1u << (BITS - 2);  // a bias names it
  static constexpr uint32_t kCount = kNamed - 1;
  static constexpr uint32_t kField = kSeen | kNamed | kCount;
};

struct Params {
  const void* x;
  long long ldx;
  void* y;
  long long ldy;
  const int* tokens;  // [B, L] (null: no penalties)
  long long ldt;
  const int* lens;
  const int* prompt_lens;  // null: everything counts as generated
  const float* repetition;
  const float* frequency;
  const float* presence;
  const int* bias_ids;  // [B, n_bias]
  const float* bias;
  long long ldb;
  const uint32_t* mask;  // [R, words]
  long long ldm;
  const int* mask_rows;  // null: row b uses mask row b; < 0: row b has no mask
  int V, L, n_bias, n_masks, chunk, staged;  // staged: there is room for the chunk in shared memory
};

template <typename T>
__device__ __forceinline__ float get(T x);
template <>
__device__ __forceinline__ float get<float>(float x) { return x; }
template <>
__device__ __forceinline__ float get<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T put(float x);
template <>
__device__ __forceinline__ float put<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 put<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// 16 bytes of a row's columns, x[i .. i + VEC).  Pieces are cut where the output is
// 16-byte aligned; an input that is not aligned there is read by 32-bit words,
// shifted together.
template <typename T>
struct Piece {
  static constexpr int VEC = 16 / sizeof(T);
  uint4 w;
  // of n columns that exist, all of the piece's among them
  __device__ __forceinline__ void load(const T* x, int i, int n, bool aligned) {
    if (aligned) {
      w = *reinterpret_cast<const uint4*>(x + i);
      return;
    }
    const uintptr_t a = reinterpret_cast<uintptr_t>(x + i);
    if (i > 0 && i + VEC < n) {  // the words around the piece lie in the row too
      const uint32_t* p = reinterpret_cast<const uint32_t*>(a & ~uintptr_t(3));
      if (sizeof(T) == 4 || (a & 3) == 0) {
        w = make_uint4(p[0], p[1], p[2], p[3]);
      } else {
        const uint32_t w0 = p[0], w1 = p[1], w2 = p[2], w3 = p[3], w4 = p[4];
        w = make_uint4(__funnelshift_r(w0, w1, 16), __funnelshift_r(w1, w2, 16), __funnelshift_r(w2, w3, 16),
                       __funnelshift_r(w3, w4, 16));
      }
      return;
    }
    T e[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) e[k] = x[i + k];
    w = *reinterpret_cast<const uint4*>(e);
  }
  // From shared memory: the piece that begins WORD words and `half` bits into the
  // 16-byte unit at u (WORD < 0: at u; the unit after it can be read too).
  template <int WORD>
  __device__ __forceinline__ void load_shared(const uint4* u, int half) {
    const uint4 lo = u[0];
    if constexpr (WORD < 0) {
      w = lo;
    } else {
      const uint4 hi = u[1];
      const uint32_t v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      if constexpr (sizeof(T) == 4)
        w = make_uint4(v[WORD], v[WORD + 1], v[WORD + 2], v[WORD + 3]);
      else
        w = make_uint4(__funnelshift_r(v[WORD], v[WORD + 1], half), __funnelshift_r(v[WORD + 1], v[WORD + 2], half),
                       __funnelshift_r(v[WORD + 2], v[WORD + 3], half),
                       __funnelshift_r(v[WORD + 3], v[WORD + 4], half));
    }
  }
  // columns whose bit is 0 become -inf
  __device__ __forceinline__ void mask(uint32_t bits) {
    if constexpr (sizeof(T) == 4) {
      if (!(bits & 1)) w.x = 0xff800000u;
      if (!(bits & 2)) w.y = 0xff800000u;
      if (!(bits & 4)) w.z = 0xff800000u;
      if (!(bits & 8)) w.w = 0xff800000u;
    } else {
      uint32_t* u = &w.x;
      const uint32_t both = bits | bits << 15;  // even bits below, odd ones 16 places above them
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // bits 2 k and 2 k + 1 to the tops of the two halves, spread over them
        uint32_t keep;
        asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(keep) : "r"(both << (15 - 2 * k)));
        u[k] = (u[k] & keep) | (0xff80ff80u & ~keep);
      }
    }
  }
};

// Columns before the first 128-byte line of a row that begins at x.
template <typename T>
__device__ __forceinline__ int before_line(const T* x, int n) {
  constexpr int LINE = 128 / sizeof(T);
  return min(n, static_cast<int>(-(reinterpret_cast<uintptr_t>(x) / sizeof(T)) % LINE));
}
template <typename T>
__device__ __forceinline__ int phase_of(const T* x) {  // place in a 16-byte unit
  return static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
}
// Where a chunk of n columns is cut into pieces: from the output's first line on, so that a warp
// writes whole lines.
template <typename T>
struct Cut {
  int first, behind;
  __device__ __forceinline__ Cut(const T* y, int n) {
    constexpr int VEC = Piece<T>::VEC;
    first = before_line(y, n);
    behind = first + (n - first) / VEC * VEC;
  }
  // the i-th column that is in no piece
  __device__ __forceinline__ int rest(int i) const { return i < first ? i : behind + i - first; }
};

// Four of a row's tokens, -1 past the last.
__device__ __forceinline__ int4 four_tokens(const int* t, int i, int len, bool vec) {
  if (vec && i + 4 <= len) return *reinterpret_cast<const int4*>(t + i);
  return make_int4(i < len ? t[i] : -1, i + 1 < len ? t[i + 1] : -1, i + 2 < len ? t[i + 2] : -1,
                   i + 3 < len ? t[i + 3] : -1);
}

// Bit v of row b's mask, as bytes from the chunk's first column on (null: no mask).
__device__ __forceinline__ const uint8_t* mask_of(const Params& p, int b, int c0) {
  if (!p.mask) return nullptr;
  const int r = p.mask_rows ? p.mask_rows[b] : b;
  return r >= 0 && r < p.n_masks ? reinterpret_cast<const uint8_t*>(p.mask + r * p.ldm) + (c0 >> 3) : nullptr;
}

// No rule but the mask: straight through, two pieces ahead.
template <typename T>
__global__ void __launch_bounds__(kThreads, kCtas) mask_kernel(const Params p) {
  constexpr int VEC = Piece<T>::VEC, STEP = kThreads * VEC;
  constexpr uint32_t kAll = (1u << VEC) - 1;
  const int tid = threadIdx.x;
  const int b = blockIdx.y, c0 = blockIdx.x * p.chunk, n = min(p.chunk, p.V - c0);
  griddep_sync();
  const T* x = static_cast<const T*>(p.x) + b * p.ldx + c0;
  T* y = static_cast<T*>(p.y) + b * p.ldy + c0;
  const bool in_place = p.x == p.y;
  const uint8_t* mask = mask_of(p, b, c0);
  if (in_place && !mask) return;
  const Cut<T> cut(y, n);
  const bool aligned = phase_of(x) == phase_of(y);
  // bits i .. i + VEC, all of which exist
  auto bits_of = [&](int i) -> uint32_t {
    if (!mask) return kAll;
    uint32_t bits = mask[i >> 3];
    if ((i & 7) + VEC > 8) bits |= static_cast<uint32_t>(mask[(i >> 3) + 1]) << 8;
    return bits >> (i & 7) & kAll;
  };
  const int rest = cut.rest(tid);
  T single = put<T>(-INFINITY);
  if (rest < n && (!mask || (mask[rest >> 3] >> (rest & 7) & 1))) single = x[rest];
  Piece<T> next[2];
  uint32_t next_bits[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = cut.first + tid * VEC + k * STEP;
    if (i < cut.behind) {
      next[k].load(x, i, n, aligned);
      next_bits[k] = bits_of(i);
    }
  }
#pragma unroll 2
  for (int i = cut.first + tid * VEC; i < cut.behind; i += STEP) {
    Piece<T> cur = next[0];
    const uint32_t bits = next_bits[0];
    next[0] = next[1];
    next_bits[0] = next_bits[1];
    if (i + 2 * STEP < cut.behind) {
      next[1].load(x, i + 2 * STEP, n, aligned);
      next_bits[1] = bits_of(i + 2 * STEP);
    }
    if (bits != kAll) cur.mask(bits);
    if (!in_place || bits != kAll) *reinterpret_cast<uint4*>(y + i) = cur.w;
  }
  if (rest < n) y[rest] = single;
}

template <typename T, typename C>
__global__ void __launch_bounds__(kThreads, kCtas) process_kernel(const Params p) {
  using W = Word<C>;
  constexpr int VEC = Piece<T>::VEC;
  constexpr uint32_t kAll = (1u << VEC) - 1;
  constexpr int STEP = kThreads * VEC;
  constexpr int HEADS = 2;  // groups of four tokens a thread asks for at the start
  extern __shared__ __align__(16) uint8_t smem[];  // words C [chunk], if staged: logits T [chunk + 2 VEC], mask [chunk / 32 + 1]; the list
  uint8_t* s_chunk = smem + p.chunk * sizeof(C);
  uint32_t* s_mask = reinterpret_cast<uint32_t*>(s_chunk + (p.staged ? (p.chunk + 2 * VEC) * sizeof(T) : 0));
  uint16_t* s_list = reinterpret_cast<uint16_t*>(s_mask + (p.staged && p.mask ? p.chunk / 32 + 1 : 0));
  __shared__ __align__(16) int s_ids[kList];  // -1 past the last
  __shared__ __align__(16) float s_add[kList];
  __shared__ int s_n;
  const int tid = threadIdx.x;
  const int b = blockIdx.y, c0 = blockIdx.x * p.chunk, n = min(p.chunk, p.V - c0);
  const bool counts = p.tokens != nullptr, biases = p.n_bias > 0;
  for (int i = tid; i < static_cast<int>(p.chunk * sizeof(C) / 16); i += kThreads)
    reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  if (tid == 0) s_n = 0;
  griddep_sync();
  // ---- what depends on no other load is asked for first
  const T* x = static_cast<const T*>(p.x) + b * p.ldx + c0;
  T* y = static_cast<T*>(p.y) + b * p.ldy + c0;
  const int* t = counts ? p.tokens + b * p.ldt : nullptr;
  const bool vec_t = (reinterpret_cast<uintptr_t>(t) & 15) == 0;
  int4 head[HEADS];
#pragma unroll
  for (int k = 0; k < HEADS; ++k) head[k] = four_tokens(t, 4 * (k * kThreads + tid), counts ? p.L : 0, vec_t);
  const int* ids = p.bias_ids + b * p.ldb;
  const float* add = p.bias + b * p.ldb;
  int my_id = -1, len = 0, prompt = 0;
  float my_add = 0.f, rep = 1.f, freq = 0.f, pres = 0.f;
  if (tid < min(p.n_bias, kList)) my_id = ids[tid], my_add = add[tid];
  if (counts) {
    len = p.lens[b];
    if (p.prompt_lens) prompt = p.prompt_lens[b];
    if (p.repetition) rep = p.repetition[b];
    if (p.frequency) freq = p.frequency[b];
    if (p.presence) pres = p.presence[b];
  }
  const uint8_t* mask = mask_of(p, b, c0);
  len = max(0, min(len, p.L));
  prompt = min(prompt, len);
  const bool few = (static_cast<long long>(len) + p.n_bias) * kFew < static_cast<long long>(p.V) * static_cast<int>(sizeof(T));
  const bool staged = p.staged && !(p.x == p.y && !mask && few);
  const int phase = phase_of(x);
  // the chunk into shared memory, at the same place in a 16-byte unit as it has in memory
  T* s_x = reinterpret_cast<T*>(s_chunk) + phase;
  if (staged) {
    const int lead = before_line(x, n), units = (n - lead) / VEC, done = lead + units * VEC;
    const T* src = x + lead + tid * VEC;
    uint32_t dst = smem_u32(s_x + lead + tid * VEC);
    for (int i = tid; i < units; i += kThreads) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
      src += STEP;
      dst += STEP * sizeof(T);
    }
    if (mask)
      for (int i = tid; i < (n + 31) / 32; i += kThreads)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(s_mask + i)), "l"(mask + 4 * i)
                     : "memory");
    if (tid < lead) s_x[tid] = x[tid];
    if (tid < n - done) s_x[done + tid] = x[done + tid];
  }

  // ---- the columns that tokens and biases name
  auto word_of = [&](unsigned j) { return reinterpret_cast<uint32_t*>(smem) + (sizeof(C) == 2 ? j >> 1 : j); };
  auto shift_of = [&](unsigned j) { return sizeof(C) == 2 ? (j & 1) * 16 : 0; };
  if (tid < kList) s_ids[tid] = my_id, s_add[tid] = my_add;
  __syncthreads();
  if (biases) {
    for (int i = tid; i < p.n_bias; i += kThreads) {
      const unsigned j = static_cast<unsigned>(i < kList ? my_id : ids[i]) - static_cast<unsigned>(c0);
      if (j >= static_cast<unsigned>(n)) continue;
      if ((atomicOr(word_of(j), W::kNamed << shift_of(j)) >> shift_of(j) & W::kField) == 0)
        s_list[atomicAdd(&s_n, 1)] = static_cast<uint16_t>(j);
    }
    __syncthreads();  // a column with a bias is on the list before a token comes to it
  }
  if (counts) {
    // whole warps: the new columns of its 128 tokens get their places on the list with one addition
    auto count4 = [&](const int4& u, int i) {
      const int token[4] = {u.x, u.y, u.z, u.w};
      uint32_t fresh[4];
      int total = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned j = static_cast<unsigned>(token[k]) - static_cast<unsigned>(c0);
        bool is_new = false;
        if (j < static_cast<unsigned>(n) && i + k < len) {
          const uint32_t old = i + k < prompt ? atomicOr(word_of(j), W::kSeen << shift_of(j))
                                              : atomicAdd(word_of(j), 1u << shift_of(j));
          is_new = (old >> shift_of(j) & W::kField) == 0;
        }
        fresh[k] = __ballot_sync(0xffffffffu, is_new);
        total += __popc(fresh[k]);
      }
      if (total == 0) return;
      const int lane = tid & 31;
      int at = lane == 0 ? atomicAdd(&s_n, total) : 0;
      at = __shfl_sync(0xffffffffu, at, 0);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int mine = at + __popc(fresh[k] & ((1u << lane) - 1));
        if (fresh[k] >> lane & 1) s_list[mine] = static_cast<uint16_t>(token[k] - c0);
        at += __popc(fresh[k]);
      }
    };
#pragma unroll
    for (int k = 0; k < HEADS; ++k)
      if (4 * (k * kThreads + (tid & ~31)) < len) count4(head[k], 4 * (k * kThreads + tid));
    for (int i0 = 4 * HEADS * kThreads + 4 * (tid & ~31); i0 < len; i0 += 4 * kThreads) {
      const int i = i0 + 4 * (tid & 31);
      count4(four_tokens(t, i, len, vec_t), i);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();  // counts, list and chunk
  T* to = staged ? s_x : y;
  const int on_list = s_n;
  auto rewrite = [&](unsigned j, float f) {
    const uint32_t w = *word_of(j) >> shift_of(j);
    if (w & (W::kSeen | W::kCount)) {
      f = f > 0.f ? f / rep : f * rep;
      const uint32_t made = w & W::kCount;
      if (made) f = f - freq * static_cast<float>(made) - pres;
    }
    if (w & W::kNamed) {  // its entries of the list, in order
      const int id = c0 + static_cast<int>(j), kept = min(p.n_bias, kList);
#pragma unroll 2
      for (int m = 0; m < kept; m += 4) {
        const int4 at = *reinterpret_cast<const int4*>(s_ids + m);
        const float4 by = *reinterpret_cast<const float4*>(s_add + m);
        if (at.x == id) f += by.x;
        if (at.y == id) f += by.y;
        if (at.z == id) f += by.z;
        if (at.w == id) f += by.w;
      }
      for (int m = kept; m < p.n_bias; ++m)
        if (ids[m] == id) f += add[m];
    }
    to[j] = put<T>(f);  // (rounded once: a masked column is overwritten below)
  };
  if (staged) {
    for (int i = tid; i < on_list; i += kThreads) rewrite(s_list[i], get<T>(s_x[s_list[i]]));
  } else {
    // in place the columns come from HBM: four are asked for before the first is worked on
    for (int i0 = tid; i0 < on_list; i0 += 4 * kThreads) {
      float f[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = get<T>(x[s_list[min(i0 + k * kThreads, on_list - 1)]]);
#pragma unroll 1
      for (int k = 0; k < 4; ++k) {
        if (i0 + k * kThreads < on_list) rewrite(s_list[i0 + k * kThreads], f[0]);
        f[0] = f[1], f[1] = f[2], f[2] = f[3];
      }
    }
  }
  if (!staged) return;
  __syncthreads();
  const Cut<T> cut(y, n);
  const int rest = cut.rest(tid);
  if (rest < n) y[rest] = mask && !(s_mask[rest >> 5] >> (rest & 31) & 1) ? put<T>(-INFINITY) : s_x[rest];
  const int shift = (phase + cut.first) % VEC * static_cast<int>(sizeof(T));
  const uint4* src = reinterpret_cast<const uint4*>(s_chunk) + (phase + cut.first) / VEC + tid;
  uint4* dst = reinterpret_cast<uint4*>(y + cut.first) + tid;
  const int begin = cut.first + tid * VEC;
  const uint32_t* words = s_mask + (begin >> 5);  // (a step is whole words)
  auto write = [&](auto word) {
#pragma unroll 2
    for (int i = begin; i < cut.behind; i += STEP) {
      Piece<T> cur;
      cur.template load_shared<decltype(word)::value>(src, (shift & 2) * 8);
      if (mask) {
        const uint32_t bits = __funnelshift_r(words[0], words[1], begin & 31) & kAll;
        if (bits != kAll) cur.mask(bits);
        words += STEP / 32;
      }
      *dst = cur.w;
      src += kThreads;
      dst += kThreads;
    }
  };
  if (shift == 0) write(std::integral_constant<int, -1>{});
  else if (shift < 4) write(std::integral_constant<int, 0>{});
  else if (shift < 8) write(std::integral_constant<int, 1>{});
  else if (shift < 12) write(std::integral_constant<int, 2>{});
  else write(std::integral_constant<int, 3>{});
}

// Columns of a CTA: a row in as many equal chunks as fill one wave of CTAs, of at most `most` columns.
int chunk_of(int B, int V, int most) {
  int parts = sm_count() * kCtas / B;
  const int least = (V + most - 1) / most, limit = (V + 2047) / 2048;
  if (parts > limit) parts = limit;
  if (parts < least) parts = least;
  return ((V + parts - 1) / parts + 63) / 64 * 64;
}

template <typename T, typename C>
int launch(Params& p, int B, cudaStream_t stream) {
  // a list holds each column once, and no more than there are tokens and biases
  const long long list = static_cast<long long>(p.tokens ? p.L : 0) + p.n_bias;
  p.staged = p.x != p.y || p.mask || list * kFew >= static_cast<long long>(p.V) * static_cast<int>(sizeof(T));
  const double bytes = sizeof(C) + (p.staged ? sizeof(T) + (p.mask ? 0.125 : 0.) : 0.);
  constexpr int tail = 64;
  long long most = static_cast<long long>((kSmem - tail) / (bytes + 2));
  if (list < most) most = static_cast<long long>((kSmem - tail - 2 * list) / bytes);
  p.chunk = chunk_of(B, p.V, static_cast<int>(most / 64 * 64));
  const size_t smem =
      tail + static_cast<size_t>(p.chunk * bytes) + 2 * static_cast<size_t>(list < p.chunk ? list : p.chunk);
  constexpr int kMaxDev = 64;
  static bool ready[kMaxDev] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return NL_ERR_CUDA;
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(process_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
      return NL_ERR_LAUNCH;
    ready[dev] = true;
  }
  launch_kernel(process_kernel<T, C>, dim3((p.V + p.chunk - 1) / p.chunk, B), dim3(kThreads), smem, stream, 1, p);
  return launch_status();
}

template <typename T>
int launch(Params& p, int B, cudaStream_t stream) {
  if (p.tokens || p.n_bias > 0) {
    const bool small = p.L <= static_cast<int>(Word<uint16_t>::kCount);  // no count can overflow
    return small ? launch<T, uint16_t>(p, B, stream) : launch<T, uint32_t>(p, B, stream);
  }
  if (p.x == p.y && !p.mask) return NL_OK;
  p.chunk = chunk_of(B, p.V, 65536);
  launch_kernel(mask_kernel<T>, dim3((p.V + p.chunk - 1) / p.chunk, B), dim3(kThreads), 0, stream, 1, p);
  return launch_status();
}

}  // namespace lg
}  // namespace nl

using namespace nl;

extern "C" int nl_process_logits(const nl_process_logits_args* args, cudaStream_t stream) {
  if (!args) return NL_ERR_SHAPE;
  const nl_process_logits_args& a = *args;
  const int B = a.B, V = a.V, dtype = a.dtype;
  constexpr int kMost = (1 << 30) - 1;  // columns, tokens and biases of a row: indices and counts stay in 32 bits
  if (V > kMost || a.n_bias > kMost || (a.tokens && a.L > kMost)) return NL_ERR_TOO_LARGE;
  if (B <= 0 || B > 65535 || V <= 0 || a.ldx < V || a.ldy < V || !a.logits || !a.out) return NL_ERR_SHAPE;
  if (dtype != NL_F32 && dtype != NL_BF16) return NL_ERR_DTYPE;
  if (a.logits == a.out && B > 1 && a.ldx != a.ldy) return NL_ERR_SHAPE;
  if (a.tokens && (a.L <= 0 || a.ldt < a.L || !a.lens)) return NL_ERR_SHAPE;
  if (a.n_bias < 0 || (a.n_bias > 0 && (!a.bias_ids || !a.bias || a.ldb < a.n_bias))) return NL_ERR_SHAPE;
  if (a.mask && (a.ldm < (V + 31) / 32 || a.n_masks <= 0 || (!a.mask_rows && a.n_masks < B))) return NL_ERR_SHAPE;
  const size_t align = dtype == NL_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.out)) % align) return NL_ERR_ALIGN;
  lg::Params p{a.logits, a.ldx, a.out, a.ldy, a.tokens, a.ldt, a.lens, a.prompt_lens, a.repetition, a.frequency,
               a.presence, a.bias_ids, a.bias, a.ldb, static_cast<const uint32_t*>(a.mask), a.ldm, a.mask_rows, V,
               a.tokens ? a.L : 0, a.n_bias, a.n_masks, 0, 0};
  return dtype == NL_F32 ? lg::launch<float>(p, B, stream) : lg::launch<__nv_bfloat16>(p, B, stream);
}
