// dcr_rotary.cu — position rotation of query and key heads from frequencies, in place or into other
// rows, or with the append of keys and values into a paged cache (sm_100a).
//
// For token t at position x_t and frequency i < r / 2 (r rotated elements a row, the first ones):
//   a = x_t * inv_freq[i],  c = factor * cos a,  s = factor * sin a
//   (u, w) -> (u c - w s, w c + u s)   for the elements (i, i + r/2), or (2i, 2i + 1) interleaved
// and elements r.. stay as they are. Scaling for long contexts is in the frequencies and the
// factor. With norm weights (the paged form) every row is first x * rsqrt(mean(x^2) + eps) * weight.
// All in fp32 from the stored inputs, rounded once. The angle is taken in turns in 64 bits, x_t *
// (inv_freq / 2 pi) less its nearest integer, so a position of 2^31 loses 2^-22 of a turn at most and
// one of a million 2^-33; an fp32 product would be off by a hundredth of a turn there. The
// reference's step is HF apply_rotary_pos_emb from tables (dcr_attention/models/llama/attention.py:395);
// layouts, parts of a head, pages and norms have no counterpart there.
//
// Bound: the rows, read and written once. A CTA takes a few tokens: their angles, once for all heads,
// go to shared memory while the first rows are on their way. A lane takes two 16-byte chunks that
// hold whole pairs: chunks r/2 elements apart, or neighbours. Where r is not a multiple of two chunks
// a warp takes a row element by element (106 us for 8191 tokens of 40 heads of 80, 20 elements of each
// turned, a sixth of the memory's rate).
// Measured (in a CUDA graph): 16381 tokens of 32 + 8 heads of 128, f16 (336 MB): 54.3 us, 6.2 TB/s; the
// same with the values of 8 more heads into pages, norms, and 96 elements of each head turned in
// neighbouring pairs, bf16 (403 MB): 97 us, 4.2 TB/s (whole heads in halves: 91), bound by instructions: the
// place, angle, weight and pair of each row part are worked out by itself. The append by tables, whose warps hold
// angle and weight as two factors for all rows of a token, takes 68 us for whole heads in halves. 48 tokens: 2.2
// and 4.3 us. With items found by divisions and
// arithmetic that is not packed these took 75 and 121 us; loading each item's successor as soon as it
// was used (95 registers) 59 and 106; six items in flight 62 and 127.
#include <type_traits>

#include "dcr_internal.h"
#include "dcr_paged.cuh"

namespace dcr {

struct RotaryParams {
  const void* q;
  const void* k;
  const void* v;             // paged
  int64_t qst, qsh, kst, ksh, vst, vsh;
  void* q_out;
  void* k_out;               // not paged
  int64_t qost, qosh, kost, kosh;
  const float* inv_freq;     // [rot / 2]
  const void* positions;     // [T] int32 or int64
  int wide;                  // positions are int64
  int interleaved;
  int T, H, H_kv, D, rot;
  int parts;                 // items (two chunks) of a row: all of it, or its rotated part in place
  int per_cta;               // tokens a CTA
  float factor;
  // paged
  PagePool c;
  void* k_pages;
  void* v_pages;
  const int32_t* seq;
  const int32_t* slots;
  int n_seq;
  const void* qw;
  const void* kw;
  float eps;
  float* weights;
  int64_t wsb, wsh;
  int32_t* pos;
  int64_t psb, psh;
};

constexpr int kRoThreads = 128;
constexpr int kRoSteps = 3;        // items a thread has in flight
constexpr int kRoMaxTokens = 16;   // tokens a CTA at most
constexpr int kRoMaxDim = 512;

// Where a token's key and value go.
struct RotaryPlace {
  int64_t k, v;   // element offsets of head 0's row
  int b, slot;    // slot < 0: nowhere
  int64_t position;
};

template <bool Paged>
__device__ __forceinline__ RotaryPlace ro_place(const RotaryParams& p, int t) {
  RotaryPlace r;
  r.position = p.wide ? static_cast<const int64_t*>(p.positions)[t]
                      : static_cast<const int32_t*>(p.positions)[t];
  r.k = r.v = 0;
  r.b = 0;
  r.slot = -1;
  if constexpr (Paged) {
    const int slot = p.slots[t];
    if (slot < 0) return r;
    const int b = p.seq != nullptr ? p.seq[t] : t;
    int pg = -1;
    uint32_t pi = 0;
    if (b >= 0 && b < p.n_seq && slot < p.c.max_pages * static_cast<int>(p.c.page.d)) {
      pi = p.c.page.div(slot);
      pg = page_of(p.c, b, pi);
    }
    if (pg < 0) {  // no such place, or not mapped: the row would be lost
      raise_status(DCR_ERR_DEVICE_INDEX);
      return r;
    }
    const int64_t in = slot - static_cast<int>(pi * p.c.page.d);
    r.k = pg * p.c.ksp + in * p.c.ksr;
    r.v = pg * p.c.vsp + in * p.c.vsr;
    r.b = b;
    r.slot = slot;
  }
  return r;
}

// cos and sin of every token of the CTA, times the factor: cosines [tokens][rot / 2], then sines.
__device__ __forceinline__ void ro_angles(const RotaryParams& p, const RotaryPlace* place, int tokens,
                                          float* turn) {
  const int half = p.rot / 2, n = tokens * half;
  for (int i = threadIdx.x; i < n; i += kRoThreads) {
    const int t = i / half, f = i - t * half;
    const double turns = static_cast<double>(place[t].position) *
                         (static_cast<double>(p.inv_freq[f]) * 0.15915494309189533577);
    float s, c;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
    turn[i] = c * p.factor;
    turn[n + i] = s * p.factor;
  }
}

// A row's source and destination.
template <typename T, bool Paged>
__device__ __forceinline__ const T* ro_source(const RotaryParams& p, int t, int row) {
  if (row < p.H) return static_cast<const T*>(p.q) + t * p.qst + row * p.qsh;
  if (!Paged || row < p.H + p.H_kv) return static_cast<const T*>(p.k) + t * p.kst + (row - p.H) * p.ksh;
  return static_cast<const T*>(p.v) + t * p.vst + (row - p.H - p.H_kv) * p.vsh;
}

template <typename T, bool Paged>
__device__ __forceinline__ T* ro_target(const RotaryParams& p, const RotaryPlace& at, int t, int row) {
  if (row < p.H) return static_cast<T*>(p.q_out) + t * p.qost + row * p.qosh;
  if constexpr (Paged) {
    if (at.slot < 0) return nullptr;
    return row < p.H + p.H_kv ? static_cast<T*>(p.k_pages) + at.k + (row - p.H) * p.c.ksh
                              : static_cast<T*>(p.v_pages) + at.v + (row - p.H - p.H_kv) * p.c.vsh;
  } else {
    return static_cast<T*>(p.k_out) + t * p.kost + (row - p.H) * p.kosh;
  }
}

// The two chunks of item i of a row, the first `turned` items of which are rotated.
__device__ __forceinline__ int2 ro_chunks(int i, int turned, int interleaved) {
  if (i < turned && !interleaved) return make_int2(i, i + turned);
  return make_int2(2 * i, 2 * i + 1);
}

// An item of the CTA: part of a row of a token. Items are kRoThreads apart.
struct RotaryItem {
  int part, row, t;
  __device__ __forceinline__ void next(int parts, int rows) {
    part += kRoThreads % parts;
    row += kRoThreads / parts;
    if (part >= parts) {
      part -= parts;
      ++row;
    }
    while (row >= rows) {
      row -= rows;
      ++t;
    }
  }
};

template <typename T, bool Paged, bool Interleaved, bool Norms>
__global__ void __launch_bounds__(kRoThreads) rotary_kernel(const RotaryParams p) {
  constexpr int N = ElemTraits<T>::kPerChunk;
  extern __shared__ __align__(16) float ro_turn[];
  __shared__ RotaryPlace place[kRoMaxTokens];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const int t0 = blockIdx.x * p.per_cta;
  const int tokens = min(p.per_cta, p.T - t0);
  const int rows = p.H + (Paged ? 2 : 1) * p.H_kv;
  const int parts = p.parts, turned = p.rot / (2 * N);
  uint4 x[kRoSteps][2];
  RotaryItem at[kRoSteps];
  RotaryItem last;  // the item after those loaded
  last.part = static_cast<int>(threadIdx.x) % parts;
  last.row = static_cast<int>(threadIdx.x) / parts;
  last.t = last.row / rows;
  last.row -= last.t * rows;
  auto load = [&]() {
#pragma unroll
    for (int i = 0; i < kRoSteps; ++i) {
      at[i] = last;
      if (last.t < tokens) {
        const uint4* src = reinterpret_cast<const uint4*>(ro_source<T, Paged>(p, t0 + last.t, last.row));
        const int2 ch = ro_chunks(last.part, turned, Interleaved);
        x[i][0] = __ldcs(src + ch.x);
        x[i][1] = __ldcs(src + ch.y);
        last.next(parts, rows);
      } else {
        x[i][0] = x[i][1] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  };
  load();
  __shared__ __align__(16) float weight[Norms ? 2 : 1][Norms ? 128 : 4];
  if (Norms && threadIdx.x < p.D / N * 2) {
    const int k = threadIdx.x >= p.D / N, ch = threadIdx.x - k * (p.D / N);
    const void* w = k ? p.kw : p.qw;
    float g[N];
    if (w != nullptr) {
      ap_load<T, N>(w, ch * N, g);
#pragma unroll
      for (int e = 0; e < N; ++e) weight[k][ch * N + e] = g[e];
    }
  }
  if (threadIdx.x < tokens) place[threadIdx.x] = ro_place<Paged>(p, t0 + threadIdx.x);
  __syncthreads();
  ro_angles(p, place, tokens, ro_turn);
  __syncthreads();
  const int rounds = (tokens * rows * parts + kRoSteps * kRoThreads - 1) / (kRoSteps * kRoThreads);
#pragma unroll 1
  for (int round = 0; round < rounds; ++round) {
    if (round > 0) load();
#pragma unroll
    for (int i = 0; i < kRoSteps; ++i) {
      const int part = at[i].part, t = at[i].t, row = at[i].row;
      const bool in = t < tokens;
      const int2 ch = ro_chunks(part, turned, Interleaved);
      const bool value = Paged && row >= p.H + p.H_kv;
      float2 f[2][N / 2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float y[N];
        ElemTraits<T>::widen(x[i][h], y);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) f[h][e] = make_float2(y[2 * e], y[2 * e + 1]);
      }
      const float2 zero = make_float2(0.0f, 0.0f);
      const bool normed = Norms && !value && (row < p.H ? p.qw : p.kw) != nullptr;
      if constexpr (Norms) {  // all lanes of a row take part
        float2 s2 = zero;
#pragma unroll
        for (int e = 0; e < N / 2; ++e) s2 = ffma2(f[0][e], f[0][e], ffma2(f[1][e], f[1][e], s2));
        float ss = s2.x + s2.y;
        for (int o = parts / 2; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (normed) {
          const float rs = rsqrtf(ss / p.D + p.eps);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4* g = reinterpret_cast<const float4*>(weight[row >= p.H] + (h ? ch.y : ch.x) * N);
#pragma unroll
            for (int e = 0; e < N / 4; ++e) {
              const float4 w = g[e];
              f[h][2 * e] = ffma2(f[h][2 * e], ffma2(make_float2(w.x, w.y), make_float2(rs, rs), zero), zero);
              f[h][2 * e + 1] = ffma2(f[h][2 * e + 1], ffma2(make_float2(w.z, w.w), make_float2(rs, rs), zero), zero);
            }
          }
        }
      }
      if (!in) continue;
      if (!value && part < turned) {
        const float* cs = ro_turn + t * (p.rot / 2) + part * N;
        const float* sn = cs + tokens * (p.rot / 2);
#pragma unroll
        for (int e = 0; e < N / 4; ++e) {
          const float4 c = reinterpret_cast<const float4*>(cs)[e], s = reinterpret_cast<const float4*>(sn)[e];
          if constexpr (Interleaved) {  // the pairs 4 e .. 4 e + 3 of the two chunks
            const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float2& y = f[(4 * e + k) / (N / 2)][(4 * e + k) % (N / 2)];
              y = ffma2(y, make_float2(cc[k], cc[k]), ffma2(make_float2(-y.y, y.x), make_float2(ss[k], ss[k]), zero));
            }
          } else {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float2 ck = k ? make_float2(c.z, c.w) : make_float2(c.x, c.y);
              const float2 sk = k ? make_float2(s.z, s.w) : make_float2(s.x, s.y);
              const float2 a = f[0][2 * e + k], b = f[1][2 * e + k];
              f[0][2 * e + k] = ffma2(a, ck, ffma2(make_float2(-b.x, -b.y), sk, zero));
              f[1][2 * e + k] = ffma2(b, ck, ffma2(a, sk, zero));
            }
          }
        }
      }
      T* dst = ro_target<T, Paged>(p, place[t], t0 + t, row);
      if (dst == nullptr) continue;
      // what no arithmetic touched is stored as it was read
      const bool same = value || (!normed && part >= turned);
      __stcs(reinterpret_cast<uint4*>(dst) + ch.x, same ? x[i][0] : ap_round<T>(f[0]));
      __stcs(reinterpret_cast<uint4*>(dst) + ch.y, same ? x[i][1] : ap_round<T>(f[1]));
      if (Paged && part == 0 && row >= p.H && !value) {
        const int h = row - p.H;
        if (p.weights != nullptr) p.weights[place[t].b * p.wsb + h * p.wsh + place[t].slot] = 0.0f;
        if (p.pos != nullptr)
          p.pos[place[t].b * p.psb + h * p.psh + place[t].slot] = static_cast<int32_t>(place[t].position);
      }
    }
  }
}

// Element by element, a warp a row: any even number of rotated elements.
template <typename T, bool Paged>
__global__ void __launch_bounds__(kRoThreads) rotary_any_kernel(const RotaryParams p) {
  extern __shared__ __align__(16) float ro_turn[];
  __shared__ RotaryPlace place[kRoMaxTokens];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const int t0 = blockIdx.x * p.per_cta;
  const int tokens = min(p.per_cta, p.T - t0);
  const int rows = p.H + (Paged ? 2 : 1) * p.H_kv;
  const int lane = threadIdx.x & 31, half = p.rot / 2;
  if (threadIdx.x < tokens) place[threadIdx.x] = ro_place<Paged>(p, t0 + threadIdx.x);
  __syncthreads();
  ro_angles(p, place, tokens, ro_turn);
  __syncthreads();
  auto value_of = [](const T* row, int i) {
    if constexpr (sizeof(T) == 4) return row[i];
    else return ElemTraits<T>::widen1(reinterpret_cast<const uint16_t*>(row)[i]);
  };
#pragma unroll 1
  for (int item = threadIdx.x >> 5; item < tokens * rows; item += kRoThreads / 32) {
    const int t = item / rows, row = item - t * rows;
    const T* src = ro_source<T, Paged>(p, t0 + t, row);
    T* dst = ro_target<T, Paged>(p, place[t], t0 + t, row);
    const bool value = Paged && row >= p.H + p.H_kv;
    const T* w = Paged && !value ? static_cast<const T*>(row < p.H ? p.qw : p.kw) : nullptr;
    float rs = 1.0f;
    if (w != nullptr) {
      float ss = 0.0f;
      for (int e = lane; e < p.D; e += 32) ss = fmaf(value_of(src, e), value_of(src, e), ss);
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      rs = rsqrtf(ss / p.D + p.eps);
    }
    if (dst == nullptr) continue;
    auto normed = [&](int e) {
      return w != nullptr ? value_of(src, e) * (rs * value_of(w, e)) : value_of(src, e);
    };
    if (!value)
      for (int f = lane; f < half; f += 32) {
        const int i = p.interleaved ? 2 * f : f, j = p.interleaved ? 2 * f + 1 : f + half;
        const float c = ro_turn[t * half + f], s = ro_turn[(tokens + t) * half + f];
        const float a = normed(i), b = normed(j);
        ElemTraits<T>::store(dst, i, a * c - b * s);
        ElemTraits<T>::store(dst, j, b * c + a * s);
      }
    if (dst != src || w != nullptr)
      for (int e = (value ? 0 : p.rot) + lane; e < p.D; e += 32) {
        if (w == nullptr) dst[e] = src[e];
        else ElemTraits<T>::store(dst, e, normed(e));
      }
    if (Paged && lane == 0 && row >= p.H && !value) {
      const int h = row - p.H;
      if (p.weights != nullptr) p.weights[place[t].b * p.wsb + h * p.wsh + place[t].slot] = 0.0f;
      if (p.pos != nullptr)
        p.pos[place[t].b * p.psb + h * p.psh + place[t].slot] = static_cast<int32_t>(place[t].position);
    }
  }
}

template <typename T, bool Paged>
static int ro_launch(RotaryParams p, bool in_place, cudaStream_t s) {
  constexpr int N = ElemTraits<T>::kPerChunk;
  const bool whole = p.D % (2 * N) == 0 && p.rot % (2 * N) == 0;
  p.parts = (in_place ? p.rot : p.D) / (2 * N);
  const int rows = p.H + (Paged ? 2 : 1) * p.H_kv;
  // Tokens a CTA: for a few rounds of kRoSteps items a thread, since a CTA's beginning (places, angles) costs
  // as much as a round (1, 2 and 4 rounds: 58.3, 54.3 and 54.8 us for the first case above, 108.5, 100.6
  // and 96.8 for the second), few enough to fill the SMs.
  constexpr int kRounds = Paged ? 4 : 2;
  int per = whole ? kRounds * kRoSteps * kRoThreads / (rows * p.parts) : 4;
  const int spread = p.T / (4 * device_sm_count());
  if (per > spread) per = spread;
  if (per > kRoMaxTokens) per = kRoMaxTokens;
  if (per < 1) per = 1;
  p.per_cta = per;
  const size_t smem = static_cast<size_t>(per) * p.rot * sizeof(float);
  const dim3 grid((p.T + per - 1) / per);
  const bool norms = Paged && (p.qw != nullptr || p.kw != nullptr);
  auto kernel = rotary_any_kernel<T, Paged>;
  if (whole && norms)
    kernel = p.interleaved ? rotary_kernel<T, Paged, true, Paged> : rotary_kernel<T, Paged, false, Paged>;
  else if (whole)
    kernel = p.interleaved ? rotary_kernel<T, Paged, true, false> : rotary_kernel<T, Paged, false, false>;
  const cudaError_t e = launch_dependent(kernel, grid, dim3(kRoThreads), smem, s, 1, p);
  return e == cudaSuccess ? DCR_OK : DCR_ERR_CUDA;
}

template <bool Paged>
static int ro_launch_t(const RotaryParams& p, int dtype, bool in_place, cudaStream_t s) {
  switch (dtype) {
    case DCR_DTYPE_BF16: return ro_launch<__nv_bfloat16, Paged>(p, in_place, s);
    case DCR_DTYPE_F16: return ro_launch<__half, Paged>(p, in_place, s);
    default: return ro_launch<float, Paged>(p, in_place, s);
  }
}

// Shapes that both forms share.
static int ro_check(int T, int H, int H_kv, int D, int rot) {
  if (T <= 0 || H <= 0 || H_kv <= 0 || rot <= 0 || rot % 2 != 0 || rot > D) return DCR_ERR_SHAPE;
  if (static_cast<int64_t>(T) * (H + 2 * static_cast<int64_t>(H_kv)) > 0x7fffff00ll) return DCR_ERR_SHAPE;
  if (static_cast<int64_t>(H) + 2 * static_cast<int64_t>(H_kv) > 0x10000) return DCR_ERR_SHAPE;
  return DCR_OK;
}

// Whether rows [T, heads, D] of one tensor share bytes with those of another. Slices of one packed
// row per token, the usual case, are told apart by their places in the row.
static bool ro_meet(const void* a, int64_t ast, int64_t ash, int64_t a_heads, const void* b, int64_t bst,
                    int64_t bsh, int64_t b_heads, int64_t T, int64_t D, int64_t element) {
  if (T > 1 && ast == bst && ast > 0) {
    const int64_t period = ast * element, ea = ((a_heads - 1) * (a_heads > 1 ? ash : 0) + D) * element;
    const int64_t eb = ((b_heads - 1) * (b_heads > 1 ? bsh : 0) + D) * element;
    int64_t d = static_cast<int64_t>(reinterpret_cast<uintptr_t>(a) - reinterpret_cast<uintptr_t>(b)) % period;
    if (d < 0) d += period;
    if (d >= eb && d + ea <= period) return false;
  }
  return tables_meet(TableSpan(a, T, a_heads, D, ast, ash, element),
                     TableSpan(b, T, b_heads, D, bst, bsh, element));
}

}  // namespace dcr

using namespace dcr;

extern "C" {

int dcr_rotary(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k,
               int64_t k_stride_t, int64_t k_stride_h, const float* inv_freq, int rotated,
               const void* positions, int positions_are_int64, int interleaved, float factor,
               int dtype, int T, int H, int H_kv, int D, void* q_out, int64_t qo_stride_t,
               int64_t qo_stride_h, void* k_out, int64_t ko_stride_t, int64_t ko_stride_h,
               void* stream) {
  if (q == nullptr || k == nullptr || inv_freq == nullptr || positions == nullptr || q_out == nullptr ||
      k_out == nullptr)
    return DCR_ERR_NULL;
  if (dtype != DCR_DTYPE_BF16 && dtype != DCR_DTYPE_F16 && dtype != DCR_DTYPE_F32) return DCR_ERR_DTYPE;
  const int64_t per16 = dtype == DCR_DTYPE_F32 ? 4 : 8, element = 16 / per16;
  if (D <= 0 || D > kRoMaxDim || D % per16 != 0) return DCR_ERR_SHAPE;
  const int st = ro_check(T, H, H_kv, D, rotated);
  if (st != DCR_OK) return st;
  const int64_t strides[8] = {q_stride_t, q_stride_h, k_stride_t, k_stride_h,
                              qo_stride_t, qo_stride_h, ko_stride_t, ko_stride_h};
  for (int64_t x : strides) {
    if (x < 0) return DCR_ERR_SHAPE;
    if (x % per16 != 0) return DCR_ERR_ALIGN;
  }
  if (misaligned(16, q, k, q_out, k_out) || misaligned(4, inv_freq, positions) ||
      (positions_are_int64 && misaligned(8, positions)))
    return DCR_ERR_ALIGN;
  if (!rows_apart(T, H, D, qo_stride_t, qo_stride_h) || !rows_apart(T, H_kv, D, ko_stride_t, ko_stride_h))
    return DCR_ERR_SHAPE;
  auto same = [](const void* a, int64_t at, int64_t ah, const void* b, int64_t bt, int64_t bh, int T_, int h) {
    return a == b && (T_ <= 1 || at == bt) && (h <= 1 || ah == bh);
  };
  const bool q_in = same(q, q_stride_t, q_stride_h, q_out, qo_stride_t, qo_stride_h, T, H);
  const bool k_in = same(k, k_stride_t, k_stride_h, k_out, ko_stride_t, ko_stride_h, T, H_kv);
  // no output reaches into an input that is not itself, nor into the other output
  if ((!q_in && ro_meet(q, q_stride_t, q_stride_h, H, q_out, qo_stride_t, qo_stride_h, H, T, D, element)) ||
      (!k_in && ro_meet(k, k_stride_t, k_stride_h, H_kv, k_out, ko_stride_t, ko_stride_h, H_kv, T, D, element)) ||
      ro_meet(k, k_stride_t, k_stride_h, H_kv, q_out, qo_stride_t, qo_stride_h, H, T, D, element) ||
      ro_meet(q, q_stride_t, q_stride_h, H, k_out, ko_stride_t, ko_stride_h, H_kv, T, D, element) ||
      ro_meet(q_out, qo_stride_t, qo_stride_h, H, k_out, ko_stride_t, ko_stride_h, H_kv, T, D, element))
    return DCR_ERR_SHAPE;
  RotaryParams p = {};
  p.q = q;
  p.k = k;
  p.qst = q_stride_t;
  p.qsh = q_stride_h;
  p.kst = k_stride_t;
  p.ksh = k_stride_h;
  p.q_out = q_out;
  p.k_out = k_out;
  p.qost = qo_stride_t;
  p.qosh = qo_stride_h;
  p.kost = ko_stride_t;
  p.kosh = ko_stride_h;
  p.inv_freq = inv_freq;
  p.positions = positions;
  p.wide = positions_are_int64 != 0;
  p.interleaved = interleaved != 0;
  p.T = T;
  p.H = H;
  p.H_kv = H_kv;
  p.D = D;
  p.rot = rotated;
  p.factor = factor;
  return ro_launch_t<false>(p, dtype, q_in && k_in, static_cast<cudaStream_t>(stream));
}

int dcr_paged_rotary_append(
    const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k, int64_t k_stride_t,
    int64_t k_stride_h, const void* v, int64_t v_stride_t, int64_t v_stride_h,
    const void* q_weight, const void* k_weight, float eps, const float* inv_freq, int rotated,
    int interleaved, float factor, const int32_t* positions, const int32_t* seq,
    const int32_t* slots, int dtype, int T, int H, int H_kv, int D, void* q_out, void* k_pages,
    void* v_pages, int64_t kp_stride_p, int64_t kp_stride_h, int64_t kp_stride_s,
    int64_t vp_stride_p, int64_t vp_stride_h, int64_t vp_stride_s, int num_pages, int page_size,
    const int32_t* page_table, int64_t table_stride, int n_seq, int max_pages, float* weights,
    int64_t w_stride_b, int64_t w_stride_h, int32_t* pos, int64_t p_stride_b, int64_t p_stride_h,
    void* stream) {
  if (q == nullptr || k == nullptr || v == nullptr || inv_freq == nullptr || positions == nullptr ||
      slots == nullptr || q_out == nullptr)
    return DCR_ERR_NULL;
  int st = ro_check(T, H, H_kv, D, rotated);
  if (st != DCR_OK) return st;
  if (n_seq <= 0 || (seq == nullptr && T > n_seq)) return DCR_ERR_SHAPE;
  st = check_pool(k_pages, v_pages, dtype, kp_stride_p, kp_stride_h, kp_stride_s, vp_stride_p,
                  vp_stride_h, vp_stride_s, num_pages, page_size, page_table, table_stride,
                  max_pages, H_kv, D);
  if (st != DCR_OK) return st;
  if (H % H_kv != 0) return DCR_ERR_SHAPE;
  const int64_t per16 = dtype == DCR_DTYPE_F32 ? 4 : 8;
  const int64_t strides[6] = {q_stride_t, q_stride_h, k_stride_t, k_stride_h, v_stride_t, v_stride_h};
  for (int64_t x : strides) {
    if (x < 0) return DCR_ERR_SHAPE;
    if (x % per16 != 0) return DCR_ERR_ALIGN;
  }
  if (misaligned(16, q, k, v, q_out, q_weight, k_weight) ||
      misaligned(4, inv_freq, positions, seq, slots, weights, pos))
    return DCR_ERR_ALIGN;
  const int64_t max_slots = static_cast<int64_t>(max_pages) * page_size;
  if ((weights != nullptr && (w_stride_b < 0 || w_stride_h < 0 ||
                              !rows_apart(n_seq, H_kv, max_slots, w_stride_b, w_stride_h))) ||
      (pos != nullptr && (p_stride_b < 0 || p_stride_h < 0 ||
                          !rows_apart(n_seq, H_kv, max_slots, p_stride_b, p_stride_h))))
    return DCR_ERR_SHAPE;
  if (rows_meet(q, q_stride_t, q_stride_h, q_out, T, H, D, 16 / per16)) return DCR_ERR_SHAPE;
  // queries written over keys or values that another warp has yet to read would end in the cache
  if (rows_reach(k, k_stride_t, k_stride_h, H_kv, q_out, T, H, D, 16 / per16) ||
      rows_reach(v, v_stride_t, v_stride_h, H_kv, q_out, T, H, D, 16 / per16))
    return DCR_ERR_OVERLAP;
  RotaryParams p = {};
  p.q = q;
  p.k = k;
  p.v = v;
  p.qst = q_stride_t;
  p.qsh = q_stride_h;
  p.kst = k_stride_t;
  p.ksh = k_stride_h;
  p.vst = v_stride_t;
  p.vsh = v_stride_h;
  p.q_out = q_out;
  p.qost = static_cast<int64_t>(H) * D;
  p.qosh = D;
  p.inv_freq = inv_freq;
  p.positions = positions;
  p.interleaved = interleaved != 0;
  p.T = T;
  p.H = H;
  p.H_kv = H_kv;
  p.D = D;
  p.rot = rotated;
  p.factor = factor;
  p.c = make_pool(k_pages, v_pages, kp_stride_p, kp_stride_h, kp_stride_s, vp_stride_p,
                  vp_stride_h, vp_stride_s, num_pages, page_size, page_table, table_stride,
                  max_pages);
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  p.seq = seq;
  p.slots = slots;
  p.n_seq = n_seq;
  p.qw = q_weight;
  p.kw = k_weight;
  p.eps = eps;
  p.weights = weights;
  p.wsb = w_stride_b;
  p.wsh = w_stride_h;
  p.pos = pos;
  p.psb = p_stride_b;
  p.psh = p_stride_h;
  return ro_launch_t<true>(p, dtype, false, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
