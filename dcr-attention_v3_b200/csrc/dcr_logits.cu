// dcr_logits.cu — penalties for repeated tokens, a bias and a grammar mask on the logits of a
// decode step, and the greedy token, in one pass over the logits (sm_100a).
//
// For row b, with the token history tokens[b][0 .. n) of which the first `prompt` are the
// prompt, c[t] the number of times t occurs after the prompt and "seen" whether it occurs at
// all, every logit x[t] becomes, in fp32 and in this order,
//   x > 0 ? x / repetition : x * repetition    where t was seen
//   x - c[t] * frequency,  x - presence        where c[t] > 0
//   x + bias[t];  -inf where the mask's bit t is clear
// rounded once to the logits' type; next_token is the lowest index of the largest returned
// value among the allowed tokens (a NaN is the largest), -1 where the mask allows none. A
// negative id in the history is padding. The reference's decode loop takes the plain argmax
// (tests/kernel/test_m1_acceptance.py:198); the rest has no counterpart there.
//
// Kernel 1 counts the history into a workspace table [B][V]; kernel 2, a CTA a row, applies.
#include <math.h>

#include "dcr_common.cuh"
#include "dcr_internal.h"

namespace dcr {

struct LogitsParams {
  const void* x;
  int64_t xsb;
  int V;
  const void* tokens;
  int tok64;
  int64_t tsb;
  int L;
  const int32_t* n_tok;
  const int32_t* n_prompt;
  const float* repetition;
  const float* presence;
  const float* frequency;
  const float* bias;
  int64_t bsb;
  const uint32_t* allowed;
  int64_t asb;
  void* out;
  int64_t osb;
  int64_t* next;
  uint32_t* counts;  // [B][V]: bit 31 seen in the prompt, the rest the count after it
};

__device__ __forceinline__ void logits_span(const LogitsParams& p, int b, int& n, int& prompt) {
  n = p.n_tok != nullptr ? p.n_tok[b] : p.L;
  n = n < 0 ? 0 : n > p.L ? p.L : n;
  prompt = p.n_prompt != nullptr ? p.n_prompt[b] : 0;
}

__global__ void logits_count_kernel(const LogitsParams p) {
  const int b = blockIdx.y;
  int n, prompt;
  logits_span(p, b, n, prompt);
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t t = p.tok64 ? static_cast<const int64_t*>(p.tokens)[b * p.tsb + i]
                            : static_cast<const int32_t*>(p.tokens)[b * p.tsb + i];
  if (t < 0) return;
  if (t >= p.V) {
    raise_status(DCR_ERR_DEVICE_INDEX);
    return;
  }
  uint32_t* c = p.counts + static_cast<int64_t>(b) * p.V + t;
  if (i < prompt) atomicOr(c, 0x80000000u);
  else atomicAdd(c, 1u);
}

// Order of two fp32 values as unsigned keys: -0 equals +0, NaN above all; never 0.
__device__ __forceinline__ uint32_t logit_key(float v) {
  uint32_t u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

template <typename T>
__device__ __forceinline__ float lg_load(const void* p, int64_t i) {
  if constexpr (sizeof(T) == 4)
    return static_cast<const float*>(p)[i];
  else
    return ElemTraits<T>::widen1(static_cast<const uint16_t*>(p)[i]);
}

template <typename T>
__global__ void __launch_bounds__(1024) logits_apply_kernel(const LogitsParams p) {
  __shared__ uint64_t best_s[32];
  const int b = blockIdx.x, tid = threadIdx.x;
  const float r = p.repetition != nullptr ? p.repetition[b] : 1.0f;
  const float pr = p.presence != nullptr ? p.presence[b] : 0.0f;
  const float fr = p.frequency != nullptr ? p.frequency[b] : 0.0f;
  uint64_t best = 0;
  for (int t = tid; t < p.V; t += 1024) {
    float x = lg_load<T>(p.x, b * p.xsb + t);
    const uint32_t c = p.counts != nullptr ? p.counts[static_cast<int64_t>(b) * p.V + t] : 0u;
    if (c != 0u) {
      x = x > 0.0f ? __fdiv_rn(x, r) : __fmul_rn(x, r);
      const uint32_t said = c & 0x7fffffffu;
      if (said != 0u) {
        x = __fsub_rn(x, __fmul_rn(static_cast<float>(said), fr));
        x = __fsub_rn(x, pr);
      }
    }
    if (p.bias != nullptr) x = __fadd_rn(x, p.bias[b * p.bsb + t]);
    const bool ok = p.allowed == nullptr || (p.allowed[b * p.asb + (t >> 5)] >> (t & 31)) & 1u;
    if (!ok) x = -INFINITY;
    T* out = static_cast<T*>(p.out) + b * p.osb;
    ElemTraits<T>::store(out, t, x);
    if (ok) {
      const uint64_t k = (static_cast<uint64_t>(logit_key(lg_load<T>(out, t))) << 32) |
                         (0xffffffffu - static_cast<uint32_t>(t));
      best = k > best ? k : best;
    }
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    const uint64_t y = __shfl_xor_sync(0xffffffffu, best, o);
    best = y > best ? y : best;
  }
  if ((tid & 31) == 0) best_s[tid >> 5] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < 32; ++w) best = best_s[w] > best ? best_s[w] : best;
    p.next[b] = best == 0 ? -1 : static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(best));
  }
}

}  // namespace dcr

using namespace dcr;

extern "C" {

size_t dcr_logits_workspace_bytes(int B, int V, int L) {
  if (B <= 0 || V <= 0 || L < 0) return 0;
  return L > 0 ? sizeof(uint32_t) * static_cast<size_t>(B) * V : 16;
}

int dcr_process_logits(const void* logits, int64_t l_stride_b, int dtype, int B, int V,
                       const void* tokens, int tokens_are_int64, int64_t t_stride_b, int L,
                       const int32_t* token_lengths, const int32_t* prompt_lengths,
                       const float* repetition, const float* presence, const float* frequency,
                       const float* bias, int64_t bias_stride_b, const uint32_t* allowed,
                       int64_t a_stride_b, void* out, int64_t o_stride_b, int64_t* next_token,
                       void* workspace, size_t workspace_bytes, void* stream) {
  if (logits == nullptr || out == nullptr || next_token == nullptr) return DCR_ERR_NULL;
  if (dtype != DCR_DTYPE_BF16 && dtype != DCR_DTYPE_F16 && dtype != DCR_DTYPE_F32)
    return DCR_ERR_DTYPE;
  if (B <= 0 || B > 65535 || V <= 0 || V > 0x7ffffff0 || L < 0) return DCR_ERR_SHAPE;
  if (L > 0 && tokens == nullptr) return DCR_ERR_NULL;
  if (l_stride_b < 0 || t_stride_b < 0 || bias_stride_b < 0 || a_stride_b < 0) return DCR_ERR_SHAPE;
  if (B > 1 && o_stride_b < V) return DCR_ERR_SHAPE;
  if (workspace == nullptr || workspace_bytes < dcr_logits_workspace_bytes(B, V, L))
    return DCR_ERR_WORKSPACE;
  LogitsParams p;
  p.x = logits;
  p.xsb = l_stride_b;
  p.V = V;
  p.tokens = tokens;
  p.tok64 = tokens_are_int64;
  p.tsb = t_stride_b;
  p.L = L;
  p.n_tok = token_lengths;
  p.n_prompt = prompt_lengths;
  p.repetition = repetition;
  p.presence = presence;
  p.frequency = frequency;
  p.bias = bias;
  p.bsb = bias_stride_b;
  p.allowed = allowed;
  p.asb = a_stride_b;
  p.out = out;
  p.osb = o_stride_b;
  p.next = next_token;
  p.counts = L > 0 ? static_cast<uint32_t*>(workspace) : nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (L > 0) {
    if (cudaMemsetAsync(p.counts, 0, sizeof(uint32_t) * static_cast<size_t>(B) * V, s) != cudaSuccess)
      return DCR_ERR_CUDA;
    logits_count_kernel<<<dim3((L + 255) / 256, B), 256, 0, s>>>(p);
    if (cudaGetLastError() != cudaSuccess) return DCR_ERR_CUDA;
  }
  switch (dtype) {
    case DCR_DTYPE_BF16: logits_apply_kernel<__nv_bfloat16><<<B, 1024, 0, s>>>(p); break;
    case DCR_DTYPE_F16: logits_apply_kernel<__half><<<B, 1024, 0, s>>>(p); break;
    default: logits_apply_kernel<float><<<B, 1024, 0, s>>>(p); break;
  }
  return cudaGetLastError() == cudaSuccess ? DCR_OK : DCR_ERR_CUDA;
}

}  // extern "C"
