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
// row's columns: it counts the row's tokens that fall into the chunk in shared
// memory (integer atomics: the order does not matter), sums the biases the
// same way, and then streams the chunk once.  The row's history is read once
// per chunk, from L2 after the first time.
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <math.h>
#include <stdint.h>

#include "host_common.h"
#include "sm100.cuh"

namespace nl {
namespace lg {

constexpr int kThreads = 256;
constexpr uint32_t kSeen = 0x80000000u;  // a token's count word: occurs in the prompt

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
  int V, L, n_bias, n_masks, chunk;
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

template <typename T>
__global__ void __launch_bounds__(kThreads) process_kernel(const Params p) {
  extern __shared__ uint32_t s_count[];  // [chunk], then (with biases) float [chunk]
  float* s_bias = reinterpret_cast<float*>(s_count + p.chunk);
  const int tid = threadIdx.x;
  const int b = blockIdx.y, c0 = blockIdx.x * p.chunk, n = min(p.chunk, p.V - c0);
  griddep_sync();
  const bool counts = p.tokens != nullptr, biases = p.n_bias > 0;
  float rep = 1.f, freq = 0.f, pres = 0.f;
  if (counts) {
    rep = p.repetition ? p.repetition[b] : 1.f;
    freq = p.frequency ? p.frequency[b] : 0.f;
    pres = p.presence ? p.presence[b] : 0.f;
  }
  if (counts)
    for (int i = tid; i < n; i += kThreads) s_count[i] = 0;
  if (biases)
    for (int i = tid; i < n; i += kThreads) s_bias[i] = 0.f;
  __syncthreads();
  if (counts) {
    const int len = max(0, min(p.lens[b], p.L));
    const int prompt = p.prompt_lens ? max(0, min(p.prompt_lens[b], len)) : 0;
    const int* t = p.tokens + b * p.ldt;
    for (int i = tid; i < len; i += kThreads) {
      const unsigned j = static_cast<unsigned>(t[i]) - static_cast<unsigned>(c0);
      if (j < static_cast<unsigned>(n)) {
        if (i < prompt) atomicOr(s_count + j, kSeen);
        else atomicAdd(s_count + j, 1u);
      }
    }
  }
  if (biases) {
    const int* ids = p.bias_ids + b * p.ldb;
    const float* val = p.bias + b * p.ldb;
    for (int i = tid; i < p.n_bias; i += kThreads) {
      const int id = ids[i];
      const unsigned j = static_cast<unsigned>(id) - static_cast<unsigned>(c0);
      if (j >= static_cast<unsigned>(n)) continue;
      // the first entry of an id sums the later ones, in list order
      bool first = true;
      for (int k = 0; k < i; ++k) first = first && ids[k] != id;
      if (!first) continue;
      float sum = val[i];
      for (int k = i + 1; k < p.n_bias; ++k)
        if (ids[k] == id) sum += val[k];
      s_bias[j] = sum;
    }
  }
  __syncthreads();
  const uint32_t* mask = nullptr;
  if (p.mask) {
    const int r = p.mask_rows ? p.mask_rows[b] : b;
    if (r >= 0 && r < p.n_masks) mask = p.mask + r * p.ldm;
  }
  const T* x = static_cast<const T*>(p.x) + b * p.ldx;
  T* y = static_cast<T*>(p.y) + b * p.ldy;
  for (int i = tid; i < n; i += kThreads) {
    const int v = c0 + i;
    float f = get<T>(x[v]);
    if (counts) {
      const uint32_t c = s_count[i];
      if (c) {
        f = f > 0.f ? f / rep : f * rep;
        const uint32_t made = c & ~kSeen;
        if (made) f = f - freq * static_cast<float>(made) - pres;
      }
    }
    if (biases) f += s_bias[i];
    if (mask && !(mask[v >> 5] >> (v & 31) & 1)) f = -INFINITY;
    y[v] = put<T>(f);
  }
}

}  // namespace lg
}  // namespace nl

using namespace nl;

extern "C" int nl_process_logits(const void* logits, long long ldx, int dtype, void* out, long long ldy,
                                 const int* tokens, long long ldt, const int* lens, const int* prompt_lens, int L,
                                 const float* repetition, const float* frequency, const float* presence,
                                 const int* bias_ids, const float* bias, long long ldb, int n_bias,
                                 const void* mask, long long ldm, int n_masks, const int* mask_rows, int B, int V,
                                 cudaStream_t stream) {
  if (B <= 0 || B > 65535 || V <= 0 || ldx < V || ldy < V || !logits || !out) return NL_ERR_SHAPE;
  if (dtype != NL_F32 && dtype != NL_BF16) return NL_ERR_DTYPE;
  if (tokens && (L <= 0 || ldt < L || !lens)) return NL_ERR_SHAPE;
  if (n_bias < 0 || (n_bias > 0 && (!bias_ids || !bias || ldb < n_bias))) return NL_ERR_SHAPE;
  if (mask && (ldm < (V + 31) / 32 || n_masks <= 0 || (!mask_rows && n_masks < B))) return NL_ERR_SHAPE;
  lg::Params p{logits, ldx,  out,  ldy, tokens, ldt, lens, prompt_lens, repetition, frequency, presence, bias_ids,
               bias,   ldb, static_cast<const uint32_t*>(mask), ldm, mask_rows, V, tokens ? L : 0, n_bias, n_masks, 0};
  p.chunk = 4096;
  const size_t smem = static_cast<size_t>(p.chunk) * (4 + (n_bias > 0 ? 4 : 0));
  const dim3 grid((V + p.chunk - 1) / p.chunk, B);
  if (dtype == NL_F32) launch_kernel(lg::process_kernel<float>, grid, dim3(lg::kThreads), smem, stream, 1, p);
  else launch_kernel(lg::process_kernel<__nv_bfloat16>, grid, dim3(lg::kThreads), smem, stream, 1, p);
  return launch_status();
}
