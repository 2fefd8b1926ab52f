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
// A cluster of C CTAs takes a row, each a slice of the vocabulary (in chunks, where the tables
// would not fit the shared memory). Per chunk a CTA marks the history's tokens in a bitmap and
// numbers the marked ones by a prefix sum over the bitmap's words, so that the vocabulary costs
// bits and only distinct tokens take words (place; bit 31 = occurs, the rest = times after the
// prompt). Then the warps part. The side warps finish the marked tokens, whose scattered reads
// are slow; the others stream the logits and pass the marked ones over, unchanged, so that the
// side warps may read them at any time even where the output is the input. The finished ones are
// written at the end. Logits and bias come by cp.async into places of a thread's own in shared
// memory, some 16-byte vectors ahead, the first of them on their way while the history is marked.
// A vector is looked at for the best token only if its maximum reaches the CTA's so far; the
// CTAs' best tokens meet in CTA 0.
//
// Measured (calls back to back on three sets of logits and two outputs in turn): 128 rows of 128256
// fp32 logits, 131 MB: 27.8 us with 16 tokens of history (4.7 TB/s), 39.5 us with 6144 on average;
// a bias adds 3.4 to 4.0 us, a mask 0.4 to 0.8, both with that history 43.1 us (3.2 TB/s). In bf16,
// 66 MB: 20.5 us, 28.7 us with the history, 31.8 with the bias, 42.9 with history, bias and mask:
// there the bias, of twice the logits' bytes, costs 11 to 13 us (0.58 instructions a scheduler's
// cycle, two vectors of 48 bytes in flight a thread). One bf16 row with 1000 tokens of history 8.9
// us, of which 3 us are the history's phases and 3 us the launch and the cluster's barriers. Counts
// of all tokens in shared memory (a slice of 16032 tokens a CTA) took 78 us for the first case with
// bias, mask and history, finishing the marked tokens by all warps before the stream 50.9 us, both
// with one output used again and again (part of it stays in L2), where the kept form takes 39.0.
#include <cooperative_groups.h>
#include <math.h>

#include <type_traits>

#include "dcr_common.cuh"
#include "dcr_internal.h"
#include "dcr_tables.h"

namespace dcr {

namespace cg = cooperative_groups;

constexpr int kLgThreads = 1024;
constexpr int kLgSide = 256;                     // threads beside the stream
constexpr int kLgStream = kLgThreads - kLgSide;
constexpr int kLgHeld = 8;                       // tokens of the history a thread keeps
constexpr int kLgSmem = 226 * 1024;              // bytes a CTA may use

// Vectors a stream thread keeps in flight, and the bytes of their places: 16 of logits and, with
// a bias, 4 per logit.
template <typename T, bool kBias>
struct LgRing {
  static constexpr int N = ElemTraits<T>::kPerChunk;
  static constexpr int kAhead = kBias ? 2 : 4;
  static constexpr int kParts = 1 + (kBias ? N / 4 : 0);  // 16-byte parts of a vector
  static constexpr int kBytes = 16 * kAhead * kParts * kLgStream;
};

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
  int chunk;  // tokens per chunk
  int words;  // 32-token words of a chunk's bitmaps
  int distinct;  // most distinct tokens of a chunk
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

// 4-byte asynchronous global->shared copy.
__device__ __forceinline__ void cp_async_4(void* smem_dst, const void* gsrc) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(smem_dst)), "l"(gsrc) : "memory");
}

// The larger of two values; a NaN is larger than any.
__device__ __forceinline__ float lg_max(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// A history's token i, -1 past the first n.
__device__ __forceinline__ int64_t lg_token(const LogitsParams& p, int b, int i, int n) {
  if (i >= n) return -1;
  return p.tok64 ? static_cast<int64_t>(static_cast<const long long*>(p.tokens)[b * p.tsb + i])
                 : static_cast<int64_t>(static_cast<const int*>(p.tokens)[b * p.tsb + i]);
}

// Its place in the chunk [t0, t0 + span); -1 elsewhere or padding, -2 past the vocabulary.
__device__ __forceinline__ int lg_place(const LogitsParams& p, int64_t t, int64_t t0, int span) {
  const int64_t at = t - t0;
  return t >= p.V ? -2 : t >= 0 && at >= 0 && at < span ? static_cast<int>(at) : -1;
}

// One row's running state and its rule for one logit.
template <typename T>
struct LgRow {
  float r, pr, fr;
  int best, best_t;

  __device__ __forceinline__ float penalise(float f, uint32_t count) const {
    f = f > 0.0f ? __fdiv_rn(f, r) : __fmul_rn(f, r);
    const uint32_t said = count & 0x7fffffffu;
    if (said != 0u) f = __fsub_rn(__fsub_rn(f, __fmul_rn(static_cast<float>(said), fr)), pr);
    return f;
  }
  // The rounded logit of token t (`in`: allowed).
  __device__ __forceinline__ float take(float f, bool in, int t) {
    f = in ? lg_round<T>(f) : -INFINITY;
    see(f, in, t);
    return f;
  }
  __device__ __forceinline__ void see(float f, bool in, int t) {
    const int k = logit_order(f);
    if (in && (k > best || (k == best && t < best_t))) {
      best = k;
      best_t = t;
    }
  }
};

template <typename T, bool kBias>
__global__ void __launch_bounds__(kLgThreads) logits_kernel(const LogitsParams p) {
  using R = LgRing<T, kBias>;
  constexpr int N = R::N;
  extern __shared__ __align__(16) uint8_t lg_smem[];
  uint4* ring = reinterpret_cast<uint4*>(lg_smem);               // [kAhead][kParts][kLgStream]
  uint32_t* mask = reinterpret_cast<uint32_t*>(lg_smem + R::kBytes);  // [words + 2]
  uint32_t* marks = mask + p.words + 2;                          // [words]
  uint32_t* first = marks + p.words;                             // [words] marks before the word
  int* ids = reinterpret_cast<int*>(first + p.words);            // [distinct tokens of a chunk]
  uint32_t* counts = reinterpret_cast<uint32_t*>(ids + p.distinct);
  __shared__ uint64_t best_s[kLgThreads / 32];
  __shared__ uint32_t sums[kLgThreads / 32];
  __shared__ uint64_t best_c[8];
  __shared__ int best_k;  // the largest order so far: a vector below it needs no closer look
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  // arrives here, waits before the first access to another CTA's shared memory
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  const int b = blockIdx.x / C;
  const T* x = static_cast<const T*>(p.x) + b * p.xsb;
  T* out = static_cast<T*>(p.out) + b * p.osb;
  const float* bias = kBias ? p.bias + b * p.bsb : nullptr;
  const uint32_t* allowed = p.allowed != nullptr ? p.allowed + b * p.asb : nullptr;
  // vectors lie on 16-byte boundaries of x: the row's first may begin `off` elements early
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  const bool bias16 = (reinterpret_cast<uintptr_t>(bias - off) & 15u) == 0;
  const int vecs = (off + p.V + N - 1) / N;
  const int each = (vecs + C - 1) / C;
  const int v_end = min(vecs, (rank + 1) * each);
  const bool streams = tid < kLgStream;
  LgRow<T> row;
  row.best = INT_MIN;
  row.best_t = -1;
  if (tid == 0) best_k = INT_MIN;
  int n = 0, prompt = 0;
#pragma unroll 1
  for (int v0 = rank * each; v0 < v_end; v0 += p.chunk / N) {
    const int v1 = min(v_end, v0 + p.chunk / N);
    const int t0 = v0 * N - off;  // the chunk's first token (below 0 in a row's first vector)
    const int span = (v1 - v0) * N;
    // the row's first and last vectors may be partial; va .. vb are whole
    const int va = v0 == 0 && off > 0 ? 1 : v0, vb = v1 == vecs && (off + p.V) % N != 0 ? v1 - 1 : v1;
    int64_t token[kLgHeld];  // on its way while the first vectors are asked for
    if (p.tok64) {
#pragma unroll
      for (int u = 0; u < kLgHeld; ++u) {
        const int i = tid + u * kLgThreads;
        token[u] = i < p.L ? static_cast<int64_t>(static_cast<const long long*>(p.tokens)[b * p.tsb + i]) : -1;
      }
    } else {
#pragma unroll
      for (int u = 0; u < kLgHeld; ++u) {
        const int i = tid + u * kLgThreads;
        token[u] = i < p.L ? static_cast<int64_t>(static_cast<const int*>(p.tokens)[b * p.tsb + i]) : -1;
      }
    }
    if (v0 == rank * each) {
      if (p.L > 0) {
        n = p.n_tok != nullptr ? p.n_tok[b] : p.L;
        n = n < 0 ? 0 : n > p.L ? p.L : n;
        prompt = p.n_prompt != nullptr ? p.n_prompt[b] : 0;
      }
      row.r = p.repetition != nullptr ? p.repetition[b] : 1.0f;
      row.pr = p.presence != nullptr ? p.presence[b] : 0.0f;
      row.fr = p.frequency != nullptr ? p.frequency[b] : 0.0f;
    } else {
      __syncthreads();  // the chunk before is done with the tables
    }
    // the mask's words from that of the chunk's first token on
    const int words = (span + 31) / 32, w0 = max(t0, 0) >> 5;
    if (allowed != nullptr) {
      const int count = min((t0 + span + 31) / 32, (p.V + 31) / 32) - w0;
      for (int j = tid; j < count; j += kLgThreads) cp_async_4(mask + j, allowed + w0 + j);
    }
    cp_async_commit();
    if (p.L > 0) {
      for (int j = tid; j < words; j += kLgThreads) marks[j] = 0u;
      for (int i = tid; i < min(p.L, span); i += kLgThreads) counts[i] = 0u;
    }
    // With a bias on 16-bit logits, whose bytes are twice the logits', the stream begins at
    // another place in every row: rows that share a bias would all read the same part of it at
    // the same time (128 rows of 128256 with mask and history 40.9 instead of 48.9 us; without a
    // bias or in fp32 it costs 2 us and gains nothing).
    constexpr bool kTurn = kBias && N == 8;
    const int rounds = (vb - va + kLgStream - 1) / kLgStream;
    const int begin = kTurn && rounds > 0 ? va + tid + b % rounds * kLgStream : va + tid;
    const int turns = va + tid + rounds * kLgStream;  // past it, back to the first vector
    int ahead = begin, left = rounds;
    auto fetch = [&](int slot) {
      if (ahead < vb && streams && (!kTurn || left > 0)) {
        uint4* dst = ring + slot * (R::kParts * kLgStream) + tid;
        const int t = ahead * N - off;
        cp_async_16(dst, x + t, 16u);
        if constexpr (kBias) {
          if (bias16) {
#pragma unroll
            for (int e = 0; e < N / 4; ++e) cp_async_16(dst + (1 + e) * kLgStream, bias + t + 4 * e, 16u);
          } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
              cp_async_4(reinterpret_cast<uint32_t*>(dst + (1 + e / 4) * kLgStream) + e % 4,
                         reinterpret_cast<const uint32_t*>(bias + t + e));
          }
        }
      }
      cp_async_commit();
      ahead += kLgStream;
      if (kTurn && ahead == turns) ahead = va + tid;
      --left;
    };
#pragma unroll
    for (int i = 0; i < R::kAhead; ++i) fetch(i);
    int total = 0;  // distinct tokens of the history in the chunk
    if (n > 0) {
      int held[kLgHeld];
#pragma unroll
      for (int u = 0; u < kLgHeld; ++u)
        held[u] = tid + u * kLgThreads < n ? lg_place(p, token[u], t0, span) : -1;
      auto each_token = [&](auto&& f) {
#pragma unroll
        for (int u = 0; u < kLgHeld; ++u) f(tid + u * kLgThreads, held[u]);
        for (int i = tid + kLgHeld * kLgThreads; i < n; i += kLgThreads)
          f(i, lg_place(p, lg_token(p, b, i, n), t0, span));
      };
      __syncthreads();
      each_token([&](int, int at) {
        if (at >= 0) atomicOr(marks + (at >> 5), 1u << (at & 31));
        else if (at == -2) raise_status(DCR_ERR_DEVICE_INDEX);
      });
      __syncthreads();
      const int per = (words + kLgThreads - 1) / kLgThreads;
      uint32_t s = 0;
      for (int j = tid * per; j < min(words, (tid + 1) * per); ++j) s += __popc(marks[j]);
      const uint32_t incl = warp_incl_scan(s);
      if (lane == 31) sums[warp] = incl;
      __syncthreads();
      const uint32_t theirs = sums[lane];
      uint32_t before = lane < warp ? theirs : 0u, all = theirs;
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        all += __shfl_xor_sync(0xffffffffu, all, o);
      }
      total = static_cast<int>(all);
      before += incl - s;
      for (int j = tid * per; j < min(words, (tid + 1) * per); ++j) {
        first[j] = before;
        before += __popc(marks[j]);
      }
      __syncthreads();
      each_token([&](int i, int at) {
        if (at < 0) return;
        const int w = at >> 5;
        const int c = first[w] + __popc(marks[w] & ((1u << (at & 31)) - 1u));
        ids[c] = at;
        if (i < prompt) atomicOr(counts + c, 0x80000000u);
        else atomicAdd(counts + c, 1u);
      });
    }
    cp_async_wait<R::kAhead>();  // the mask
    __syncthreads();
    // the N (or 1) mask bits from token t on, the lowest first
    auto allowed_at = [&](int t) {
      if (allowed == nullptr) return 0xffffffffu;
      const int bit = t - 32 * w0;
      return __funnelshift_r(mask[bit >> 5], mask[(bit >> 5) + 1], bit & 31);
    };

    if (!streams) {
      const int side = tid - kLgStream;
      constexpr int kU = 4;
      for (int c0 = side; c0 < total; c0 += kLgSide * kU) {
        float f[kU], bs[kU];
        int at[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const int c = c0 + u * kLgSide;
          at[u] = c < total ? ids[c] : -1;
          if (at[u] < 0) continue;
          const int t = t0 + at[u];
          if constexpr (sizeof(T) == 4) f[u] = __ldcg(reinterpret_cast<const float*>(x) + t);
          else f[u] = ElemTraits<T>::widen1(__ldcg(reinterpret_cast<const unsigned short*>(x) + t));
          bs[u] = kBias ? __ldcg(bias + t) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          if (at[u] < 0) continue;
          const int c = c0 + u * kLgSide, t = t0 + at[u];
          float y = row.penalise(f[u], counts[c]);
          if (kBias) y = __fadd_rn(y, bs[u]);
          counts[c] = __float_as_uint(row.take(y, allowed_at(t) & 1u, t));
        }
      }
    } else {
      int slot = 0, v = begin - kLgStream;
#pragma unroll 1
      for (int i = 0; i < rounds; ++i) {
        v += kLgStream;
        if (kTurn && v == turns) v = va + tid;
        if (!kTurn && v >= vb) break;
        cp_async_wait<R::kAhead - 1>();
        float f[N];
        const uint4* src = ring + slot * (R::kParts * kLgStream) + tid;
        const uint4 raw = src[0];
        ElemTraits<T>::widen(raw, f);
        if constexpr (kBias) {
#pragma unroll
          for (int e = 0; e < N; e += 4) {
            const uint4 q = src[(1 + e / 4) * kLgStream];
            f[e] = __fadd_rn(f[e], __uint_as_float(q.x));
            f[e + 1] = __fadd_rn(f[e + 1], __uint_as_float(q.y));
            f[e + 2] = __fadd_rn(f[e + 2], __uint_as_float(q.z));
            f[e + 3] = __fadd_rn(f[e + 3], __uint_as_float(q.w));
          }
        }
        fetch(slot);  // the thread's own place, which it has just read
        slot = slot + 1 == R::kAhead ? 0 : slot + 1;
        if (kTurn && v >= vb) continue;
        const int place = (v - v0) * N, t = v * N - off;
        const uint32_t marked = n > 0 ? (marks[place >> 5] >> (place & 31)) & ((1u << N) - 1u) : 0u;
        const uint32_t in = allowed_at(t) & ~marked;
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          f[e] = (in >> e) & 1u ? lg_round<T>(f[e]) : -INFINITY;
          top = lg_max(top, f[e]);
        }
        const int k = logit_order(top);
        if (k >= *static_cast<volatile int*>(&best_k)) {
#pragma unroll
          for (int e = 0; e < N; ++e) row.see(f[e], (in >> e) & 1u, t + e);
          if (row.best == k) atomicMax(&best_k, k);
        }
        if (same) {
          uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
              w[i] = (marked >> i) & 1u ? w[i] : __float_as_uint(f[i]);
            } else {
              uint32_t y;
              if constexpr (std::is_same<T, __half>::value) {
                const __half2 hh = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
                y = *reinterpret_cast<const uint32_t*>(&hh);
              } else {
                const __nv_bfloat162 hh = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
                y = *reinterpret_cast<const uint32_t*>(&hh);
              }
              if (marked != 0u) {
                const uint32_t keep = ((marked >> (2 * i)) & 1u ? 0xffffu : 0u) |
                                      ((marked >> (2 * i)) & 2u ? 0xffff0000u : 0u);
                y = (y & ~keep) | (w[i] & keep);
              }
              w[i] = y;
            }
          }
          *reinterpret_cast<uint4*>(out + t) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (!((marked >> e) & 1u)) ElemTraits<T>::store(out, t + e, f[e]);
        }
      }
      cp_async_wait<0>();
    }
    if (warp == 0 && (va > v0 || vb < v1)) {  // the partial vectors: lanes 0.. the first, 16.. the last
      const int v = lane < 16 ? v0 : vb;
      const bool mine = lane % 16 < N && (lane < 16 ? va > v0 : vb < v1 && vb >= va);
      const int place = (v - v0) * N + lane % 16, t = t0 + place;
      if (mine && t >= 0 && t < p.V && !(n > 0 && (marks[place >> 5] >> (place & 31)) & 1u)) {
        float f;
        if constexpr (sizeof(T) == 4) f = x[t];
        else f = ElemTraits<T>::widen1(reinterpret_cast<const uint16_t*>(x)[t]);
        if (kBias) f = __fadd_rn(f, bias[t]);
        ElemTraits<T>::store(out, t, row.take(f, allowed_at(t) & 1u, t));
      }
    }
    if (total > 0) {
      __syncthreads();  // the stream's stores come first
      for (int c = tid; c < total; c += kLgThreads)
        ElemTraits<T>::store(out, t0 + ids[c], __uint_as_float(counts[c]));
    }
  }
  // the lowest index of the largest order: order in the high word, index reversed in the low one
  uint64_t key = row.best_t < 0
                     ? 0ull
                     : (static_cast<uint64_t>(static_cast<uint32_t>(row.best) ^ 0x80000000u) << 32) |
                           (0xffffffffu - static_cast<uint32_t>(row.best_t));
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    const uint64_t y = __shfl_xor_sync(0xffffffffu, key, o);
    key = y > key ? y : key;
  }
  if (lane == 0) best_s[warp] = key;
  __syncthreads();
  asm volatile("barrier.cluster.wait;" ::: "memory");
  if (warp == 0) {
    key = best_s[lane];
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      const uint64_t y = __shfl_xor_sync(0xffffffffu, key, o);
      key = y > key ? y : key;
    }
    if (lane == 0) *cluster.map_shared_rank(&best_c[rank], 0) = key;
  }
  if (C > 1)
    cluster.sync();
  else
    __syncwarp();
  if (rank == 0 && tid == 0) {
    for (int i = 0; i < C; ++i) key = best_c[i] > key ? best_c[i] : key;
    p.next[b] = key == 0 ? -1 : static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(key));
  }
}

// CTAs per row: of 1, 2, 4 and 8 the one whose waves of CTAs take least, with about 4 us and
// 0.6 ns a token of history for a CTA's fixed part and 44 KB/us for its stream (an SM's share of
// the memory).
static int lg_cluster(int B, int V, int L, int bytes) {
  int best = 1;
  double least = 0.0;
  for (int C = 1; C <= 8; C *= 2) {
    const double waves = static_cast<double>((static_cast<int64_t>(B) * C + device_sm_count() - 1) / device_sm_count());
    const double us = waves * (4.0 + 0.0006 * L + 2.0 * bytes * V / (44000.0 * C));
    if (C == 1 || us < least) {
      best = C;
      least = us;
    }
  }
  return best;
}

template <typename T, bool kBias>
static int lg_launch(LogitsParams p, int B, cudaStream_t s) {
  constexpr int N = ElemTraits<T>::kPerChunk;
  const int C = lg_cluster(B, p.V, p.L, static_cast<int>(sizeof(T)));
  int chunk = ((p.V + 2 * (N - 1)) / N + C - 1) / C * N;  // a row's longest slice
  auto distinct = [&](int tokens) { return static_cast<size_t>(p.L < tokens ? p.L : tokens); };
  auto bytes = [&](int tokens) {
    return LgRing<T, kBias>::kBytes +
           sizeof(uint32_t) * (3 * ((static_cast<size_t>(tokens) + 31) / 32) + 2 + 2 * distinct(tokens));
  };
  while (bytes(chunk) > kLgSmem) chunk = (chunk / 2 + N - 1) / N * N;
  p.chunk = chunk;
  p.words = (chunk + 31) / 32;
  p.distinct = static_cast<int>(distinct(chunk));
  const size_t smem = bytes(chunk);
  auto kernel = logits_kernel<T, kBias>;
  if (ensure_smem_attr(reinterpret_cast<const void*>(kernel), static_cast<int>(smem)) != cudaSuccess)
    return DCR_ERR_CUDA;
  return launch_dependent(kernel, dim3(static_cast<unsigned>(B) * C), dim3(kLgThreads), smem, s, C, p) ==
                 cudaSuccess
             ? DCR_OK
             : DCR_ERR_CUDA;
}

template <typename T>
static int lg_launch_t(const LogitsParams& p, int B, cudaStream_t s) {
  return p.bias != nullptr ? lg_launch<T, true>(p, B, s) : lg_launch<T, false>(p, B, s);
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
  if (B <= 0 || B > (1 << 27) || V <= 0 || V > (1 << 30) || L < 0) return DCR_ERR_SHAPE;
  if (L > 0 && tokens == nullptr) return DCR_ERR_NULL;
  if (l_stride_b < 0 || t_stride_b < 0 || bias_stride_b < 0 || a_stride_b < 0) return DCR_ERR_SHAPE;
  if (B > 1 && o_stride_b < V) return DCR_ERR_SHAPE;
  if (logits_meet(logits, l_stride_b, out, o_stride_b, B, V, dtype == DCR_DTYPE_F32 ? 4 : 2))
    return DCR_ERR_SHAPE;
  if (misaligned(dtype == DCR_DTYPE_F32 ? 4 : 2, logits, out) || misaligned(8, next_token) ||
      misaligned(tokens_are_int64 ? 8 : 4, tokens) ||
      misaligned(4, token_lengths, prompt_lengths, repetition, presence, frequency, bias, allowed))
    return DCR_ERR_ALIGN;
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
    case DCR_DTYPE_BF16: return lg_launch_t<__nv_bfloat16>(p, B, s);
    case DCR_DTYPE_F16: return lg_launch_t<__half>(p, B, s);
    default: return lg_launch_t<float>(p, B, s);
  }
}

}  // extern "C"
