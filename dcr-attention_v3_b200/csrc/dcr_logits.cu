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
// Bound: the logits, read and written once, with the bias and the mask; for one row, latency.
//
// A cluster of C CTAs takes a row, each a slice of the vocabulary (in chunks that fit the
// shared memory). Per chunk a CTA counts the whole history into a table in shared memory,
// keeping what falls into its chunk (one word a token: bit 31 = occurs, the rest = times after
// the prompt), and streams its logits through it, 16 bytes a thread. Counting from the list is
// cheaper than keeping counts in memory, which would be read at 4 bytes a logit: a history of
// thousands is a few KB, and the C readers of a row find it in L2. The CTAs' best tokens meet
// in CTA 0.
#include <cooperative_groups.h>
#include <math.h>

#include <type_traits>

#include "dcr_common.cuh"
#include "dcr_internal.h"

namespace dcr {

namespace cg = cooperative_groups;

constexpr int kLgThreads = 512;
constexpr int kLgChunk = 24576;  // most logits a chunk's table holds (96 KB: two CTAs an SM)

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
  int chunk;  // logits per table
};

// Signed order of fp32 values: -0 equals +0 and NaN (made canonical by the addition) is above
// all; never INT_MIN.
__device__ __forceinline__ int logit_order(float v) {
  const int s = __float_as_int(__fadd_rn(v, 0.0f));
  return s ^ ((s >> 31) & 0x7fffffff);
}

template <typename T>
__device__ __forceinline__ float lg_round(float v) {
  if constexpr (sizeof(T) == 4)
    return v;
  else if constexpr (std::is_same<T, __half>::value)
    return __half2float(__float2half_rn(v));
  else
    return __bfloat162float(__float2bfloat16_rn(v));
}

// Counts the tokens [from, to) of a history that lie in [t0, t0 + span) of the vocabulary.
template <typename I>
__device__ __forceinline__ void lg_count(const I* tokens, int n, int prompt, int64_t t0, int span,
                                         int V, bool report, uint32_t* table) {
  constexpr int U = 4;
  for (int i0 = threadIdx.x; i0 < n; i0 += kLgThreads * U) {
    int64_t t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kLgThreads;
      t[u] = i < n ? static_cast<int64_t>(__ldg(tokens + i)) : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = t[u] - t0;
      if (t[u] >= V && report) raise_status(DCR_ERR_DEVICE_INDEX);
      if (t[u] < 0 || t[u] >= V || at < 0 || at >= span) continue;
      if (i0 + u * kLgThreads < prompt)
        atomicOr(table + at, 0x80000000u);
      else
        atomicAdd(table + at, 1u);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kLgThreads) logits_kernel(const LogitsParams p) {
  constexpr int N = ElemTraits<T>::kPerChunk;
  extern __shared__ __align__(16) uint32_t table[];
  __shared__ uint64_t best_s[kLgThreads / 32];
  __shared__ uint64_t best_c[8];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // arrives here, waits before the first access to another CTA's shared memory
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  const int b = blockIdx.x / C;
  int n = 0, prompt = 0;
  if (p.L > 0) {
    n = p.n_tok != nullptr ? __ldg(p.n_tok + b) : p.L;
    n = n < 0 ? 0 : n > p.L ? p.L : n;
    prompt = p.n_prompt != nullptr ? __ldg(p.n_prompt + b) : 0;
  }
  const float r = p.repetition != nullptr ? __ldg(p.repetition + b) : 1.0f;
  const float pr = p.presence != nullptr ? __ldg(p.presence + b) : 0.0f;
  const float fr = p.frequency != nullptr ? __ldg(p.frequency + b) : 0.0f;
  const T* x = static_cast<const T*>(p.x) + b * p.xsb;
  T* out = static_cast<T*>(p.out) + b * p.osb;
  const float* bias = p.bias != nullptr ? p.bias + b * p.bsb : nullptr;
  const uint32_t* allowed = p.allowed != nullptr ? p.allowed + b * p.asb : nullptr;
  // vectors lie on 16-byte boundaries of x: the row's first may begin `off` elements early
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  const bool bias16 = (reinterpret_cast<uintptr_t>(bias - off) & 15u) == 0;
  const int vecs = (off + p.V + N - 1) / N;
  const int each = (vecs + C - 1) / C;
  const int v_end = min(vecs, (rank + 1) * each);
  int best = INT_MIN, best_t = -1;
  for (int v0 = rank * each; v0 < v_end; v0 += p.chunk / N) {
    const int v1 = min(v_end, v0 + p.chunk / N);
    if (n > 0) {
      if (v0 > rank * each) __syncthreads();  // the chunk before is done with the table
      for (int i = tid; i < (v1 - v0) * (N / 4); i += kLgThreads)
        reinterpret_cast<uint4*>(table)[i] = make_uint4(0u, 0u, 0u, 0u);
      __syncthreads();
      const int64_t t0 = static_cast<int64_t>(v0) * N - off;
      const bool report = rank == 0 && v0 == 0;
      if (p.tok64)
        lg_count(static_cast<const int64_t*>(p.tokens) + b * p.tsb, n, prompt, t0, (v1 - v0) * N, p.V, report, table);
      else
        lg_count(static_cast<const int32_t*>(p.tokens) + b * p.tsb, n, prompt, t0, (v1 - v0) * N, p.V, report, table);
      __syncthreads();
    }
    for (int v = v0 + tid; v < v1; v += kLgThreads) {
      const int t = v * N - off;  // first token of the vector
      const bool whole = t >= 0 && t + N <= p.V;
      float f[N];
      if (whole) {
        ElemTraits<T>::widen(*reinterpret_cast<const uint4*>(x + t), f);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          float one = 0.0f;
          if (t + e >= 0 && t + e < p.V) {
            if constexpr (sizeof(T) == 4) one = x[t + e];
            else one = ElemTraits<T>::widen1(reinterpret_cast<const uint16_t*>(x)[t + e]);
          }
          f[e] = one;
        }
      }
      uint32_t ok = (1u << N) - 1u;
      if (allowed != nullptr) {
        // bits t .. t + N - 1, which two words may share
        const int lo = t < 0 ? 0 : t, hi = t + N > p.V ? p.V - 1 : t + N - 1;
        const uint32_t wl = __ldg(allowed + (lo >> 5)), wh = __ldg(allowed + (hi >> 5));
        ok = t < 0 ? wl << -t : __funnelshift_r(wl, wh, t & 31);
      }
      if (n > 0) {
        uint32_t c[N];
#pragma unroll
        for (int e = 0; e < N; e += 4) {
          const uint4 q = *reinterpret_cast<const uint4*>(table + (v - v0) * N + e);
          c[e] = q.x;
          c[e + 1] = q.y;
          c[e + 2] = q.z;
          c[e + 3] = q.w;
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
          if (c[e] == 0u) continue;
          f[e] = f[e] > 0.0f ? __fdiv_rn(f[e], r) : __fmul_rn(f[e], r);
          const uint32_t said = c[e] & 0x7fffffffu;
          if (said != 0u)
            f[e] = __fsub_rn(__fsub_rn(f[e], __fmul_rn(static_cast<float>(said), fr)), pr);
        }
      }
      if (bias != nullptr) {
        if (whole && bias16) {
#pragma unroll
          for (int e = 0; e < N; e += 4) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(bias + t + e));
            f[e] = __fadd_rn(f[e], q.x);
            f[e + 1] = __fadd_rn(f[e + 1], q.y);
            f[e + 2] = __fadd_rn(f[e + 2], q.z);
            f[e + 3] = __fadd_rn(f[e + 3], q.w);
          }
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (t + e >= 0 && t + e < p.V) f[e] = __fadd_rn(f[e], __ldg(bias + t + e));
        }
      }
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const bool in = (ok >> e) & 1u;
        f[e] = in ? lg_round<T>(f[e]) : -INFINITY;
        const int k = logit_order(f[e]);
        if (in && k > best && (whole || (t + e >= 0 && t + e < p.V))) {
          best = k;
          best_t = t + e;
        }
      }
      if (whole && same) {
        uint4 q;
        if constexpr (N == 4) {
          q = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                         __float_as_uint(f[3]));
        } else {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
              const __half2 hh = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
              w[i] = *reinterpret_cast<const uint32_t*>(&hh);
            } else {
              const __nv_bfloat162 hh = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
              w[i] = *reinterpret_cast<const uint32_t*>(&hh);
            }
          }
          q = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *reinterpret_cast<uint4*>(out + t) = q;
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (t + e >= 0 && t + e < p.V) ElemTraits<T>::store(out, t + e, f[e]);
      }
    }
  }
  // the lowest index of the largest order: order in the high word, index reversed in the low one
  uint64_t key = best_t < 0 ? 0ull
                            : (static_cast<uint64_t>(static_cast<uint32_t>(best) ^ 0x80000000u) << 32) |
                                  (0xffffffffu - static_cast<uint32_t>(best_t));
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    const uint64_t y = __shfl_xor_sync(0xffffffffu, key, o);
    key = y > key ? y : key;
  }
  if (lane == 0) best_s[warp] = key;
  __syncthreads();
  asm volatile("barrier.cluster.wait;" ::: "memory");
  if (tid == 0) {
    for (int i = 1; i < kLgThreads / 32; ++i) key = best_s[i] > key ? best_s[i] : key;
    *cluster.map_shared_rank(&best_c[rank], 0) = key;
  }
  cluster.sync();
  if (rank == 0 && tid == 0) {
    for (int i = 0; i < C; ++i) key = best_c[i] > key ? best_c[i] : key;
    p.next[b] = key == 0 ? -1 : static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(key));
  }
}

// CTAs per row: a power of two up to 8 while a CTA keeps 2048 logits.
template <typename T>
static int lg_launch(LogitsParams p, int B, cudaStream_t s) {
  int C = 1;
  while (C < 8 && p.V > 2048 * 2 * C) C *= 2;
  const int N = ElemTraits<T>::kPerChunk;
  const int slice = ((p.V + N - 1 + N - 1) / N + C - 1) / C * N;  // a row's longest slice
  p.chunk = slice < kLgChunk ? slice : kLgChunk;
  const size_t smem = p.L > 0 ? sizeof(uint32_t) * p.chunk : 0;
  auto kernel = logits_kernel<T>;
  if (smem > 48 * 1024 &&
      ensure_smem_attr(reinterpret_cast<const void*>(kernel), static_cast<int>(smem)) != cudaSuccess)
    return DCR_ERR_CUDA;
  return launch_cluster(kernel, dim3(static_cast<unsigned>(B) * C), dim3(kLgThreads), smem, s, C, p) ==
                 cudaSuccess
             ? DCR_OK
             : DCR_ERR_CUDA;
}

}  // namespace dcr

using namespace dcr;

extern "C" {

int dcr_process_logits(const void* logits, int64_t l_stride_b, int dtype, int B, int V,
                       const void* tokens, int tokens_are_int64, int64_t t_stride_b, int L,
                       const int32_t* token_lengths, const int32_t* prompt_lengths,
                       const float* repetition, const float* presence, const float* frequency,
                       const float* bias, int64_t bias_stride_b, const uint32_t* allowed,
                       int64_t a_stride_b, void* out, int64_t o_stride_b, int64_t* next_token,
                       void* stream) {
  if (logits == nullptr || out == nullptr || next_token == nullptr) return DCR_ERR_NULL;
  if (dtype != DCR_DTYPE_BF16 && dtype != DCR_DTYPE_F16 && dtype != DCR_DTYPE_F32)
    return DCR_ERR_DTYPE;
  if (B <= 0 || B > (1 << 27) || V <= 0 || V > 0x7fffff00 || L < 0) return DCR_ERR_SHAPE;
  if (L > 0 && tokens == nullptr) return DCR_ERR_NULL;
  if (l_stride_b < 0 || t_stride_b < 0 || bias_stride_b < 0 || a_stride_b < 0) return DCR_ERR_SHAPE;
  if (B > 1 && o_stride_b < V) return DCR_ERR_SHAPE;
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case DCR_DTYPE_BF16: return lg_launch<__nv_bfloat16>(p, B, s);
    case DCR_DTYPE_F16: return lg_launch<__half>(p, B, s);
    default: return lg_launch<float>(p, B, s);
  }
}

}  // extern "C"
