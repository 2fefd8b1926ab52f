// dcr_paged_append.cu — query and key norms with the position rotation, and the append of the
// new keys and values into a paged cache, in one launch (sm_100a).
//
// For token t with position pos_t and the tables' rows c = cos[pos_t], s = sin[pos_t], every
// query and key head row x of D elements becomes
//   y = x * rsqrt(mean(x^2) + eps) * w        (skipped without a weight)
//   x' = y * c + rot(y) * s,  rot(y) = [-y[D/2:], y[:D/2]]
// in fp32 from the stored inputs, rounded once. The rotated queries go to q_out; the rotated
// keys and the values go to slot slots[t] of sequence seq[t]'s pages (slots[t] < 0: nowhere),
// where weights[seq][h_kv][slot] = 0 and pos[seq][h_kv][slot] = pos_t are set on request (a
// cache under eviction). The reference's step is HF apply_rotary_pos_emb and a torch.cat
// (dcr_attention/models/llama/attention.py:395-421); the norms have no counterpart there.
//
// Bound: the rows, read and written once; and the issue slots, since a 16-bit element costs a
// conversion, a square, two products and a rounding. A lane holds a 16-byte chunk of a row and the
// chunk half a row further, which the rotation pairs with it, so no element is exchanged or
// converted twice (by shuffles between the lanes of the two halves the prompts below took 78.7
// us). A row takes 4 to 16 lanes, a warp kApSteps times 8 to 2 rows of one token and kind (query,
// key, value): the token's table rows times the norm weights are folded into two factors once,
// x' = rs * (x * (w c) + x_far * (w_far s)), and all its rows are in flight before the first is
// used. Rows are read and written once, as streaming accesses (77.3 us without the hint on both
// sides, 70.0 with it). Measured: 16381 tokens of 32 + 2 x 8 heads of 128 in f16, 404 MB, in 69 to 73
// us by run, 5.5 to 5.9 TB/s, 84 to 90% of the measured copy bandwidth; a warp that took a whole token, the next rows
// on their way meanwhile, needed 126 registers and 83 us.
#include <type_traits>

#include "dcr_internal.h"
#include "dcr_paged.cuh"

namespace dcr {

struct PagedAppendParams {
  PagePool c;
  void* k_pages;
  void* v_pages;
  const void* q;
  const void* k;
  const void* v;
  int64_t qst, qsh, kst, ksh, vst, vsh;
  const void* qw;
  const void* kw;
  const void* cos;
  const void* sin;
  int n_pos;
  const int32_t* positions;
  const int32_t* seq;    // or null: token t belongs to sequence t
  const int32_t* slots;
  int T, H, H_kv, n_seq;
  float eps;
  void* q_out;           // [T][H][D]
  float* weights;
  int64_t wsb, wsh;
  int32_t* pos;
  int64_t psb, psh;
};

constexpr int kApWarps = 4;
constexpr int kApSteps = 2;

// N consecutive elements from a 16-byte (or wider) aligned address, widened.
template <typename T, int N>
__device__ __forceinline__ void ap_load(const void* base, int64_t i, float (&f)[N]) {
  constexpr int kPer = ElemTraits<T>::kPerChunk;
  static_assert(N % kPer == 0, "whole chunks");
  const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(base) + i);
#pragma unroll
  for (int c = 0; c < N / kPer; ++c) {
    float x[kPer];
    ElemTraits<T>::widen(src[c], x);
#pragma unroll
    for (int e = 0; e < kPer; ++e) f[c * kPer + e] = x[e];
  }
}

template <typename T>
__device__ __forceinline__ uint32_t ap_pack(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <typename T>
__device__ __forceinline__ uint4 ap_round(const float2 (&f)[ElemTraits<T>::kPerChunk / 2]) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x),
                      __float_as_uint(f[1].y));
  else
    return make_uint4(ap_pack<T>(f[0].x, f[0].y), ap_pack<T>(f[1].x, f[1].y),
                      ap_pack<T>(f[2].x, f[2].y), ap_pack<T>(f[3].x, f[3].y));
}

template <typename T, typename TC, int D>
__global__ void __launch_bounds__(kApWarps * 32) paged_append_kernel(const PagedAppendParams p) {
  constexpr int N = ElemTraits<T>::kPerChunk;  // elements of a chunk
  constexpr int L = D / (2 * N);               // lanes per row: chunks ch and ch + L
  constexpr int RW = 32 / L;                   // rows per step
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const int lane = threadIdx.x & 31;
  const int ch = lane % L, sub = lane / L;
  const int nq = (p.H + RW * kApSteps - 1) / (RW * kApSteps);
  const int nk = (p.H_kv + RW * kApSteps - 1) / (RW * kApSteps);
  const int blocks = nq + 2 * nk;
  const int item = blockIdx.x * kApWarps + (threadIdx.x >> 5);
  if (item >= p.T * blocks) return;
  const int t = item / blocks;
  int blk = item - t * blocks;
  const int kind = blk < nq ? 0 : blk < nq + nk ? 1 : 2;  // query, key, value
  blk -= kind == 0 ? 0 : kind == 1 ? nq : nq + nk;
  const int heads = kind == 0 ? p.H : p.H_kv;
  const int h0 = blk * RW * kApSteps + sub;  // this lane's heads: h0, h0 + RW, ...
  const char* src = static_cast<const char*>(kind == 0 ? p.q : kind == 1 ? p.k : p.v) + ch * 16;
  const int64_t st = kind == 0 ? p.qst : kind == 1 ? p.kst : p.vst;
  const int64_t sh = (kind == 0 ? p.qsh : kind == 1 ? p.ksh : p.vsh) * static_cast<int64_t>(sizeof(T));
  src += t * st * static_cast<int64_t>(sizeof(T));
  uint4 x[kApSteps][2];
#pragma unroll
  for (int i = 0; i < kApSteps; ++i) {
    const int h = h0 + i * RW;
    const uint4* row = reinterpret_cast<const uint4*>(src + h * sh);
    x[i][0] = h < heads ? __ldcs(row) : make_uint4(0u, 0u, 0u, 0u);
    x[i][1] = h < heads ? __ldcs(row + L) : make_uint4(0u, 0u, 0u, 0u);
  }
  const int position = p.positions[t];
  const bool fine = position >= 0 && position < p.n_pos;
  if (!fine) raise_status(DCR_ERR_DEVICE_INDEX);

  char* dst;
  int64_t dh;  // bytes between heads
  if (kind == 0) {
    dst = static_cast<char*>(p.q_out) + static_cast<int64_t>(t) * p.H * (D * static_cast<int>(sizeof(T)));
    dh = D * static_cast<int>(sizeof(T));
  } else {
    const int slot = p.slots[t];
    if (slot < 0 || !fine) return;
    const int b = p.seq != nullptr ? p.seq[t] : t;
    int pg = -1;
    uint32_t pi = 0;
    if (b >= 0 && b < p.n_seq && slot < p.c.max_pages * static_cast<int>(p.c.page.d)) {
      pi = p.c.page.div(slot);
      pg = page_of(p.c, b, pi);
    }
    if (pg < 0) {  // no such place, or not mapped: the row would be lost
      raise_status(DCR_ERR_DEVICE_INDEX);
      return;
    }
    const int64_t in = slot - static_cast<int>(pi * p.c.page.d);
    const int64_t off = kind == 1 ? pg * p.c.ksp + in * p.c.ksr : pg * p.c.vsp + in * p.c.vsr;
    dst = static_cast<char*>(kind == 1 ? p.k_pages : p.v_pages) + off * static_cast<int64_t>(sizeof(T));
    dh = (kind == 1 ? p.c.ksh : p.c.vsh) * static_cast<int64_t>(sizeof(T));
    if (kind == 1 && ch == 0) {
#pragma unroll
      for (int i = 0; i < kApSteps; ++i) {
        const int h = h0 + i * RW;
        if (h >= heads) break;
        if (p.weights != nullptr) p.weights[b * p.wsb + h * p.wsh + slot] = 0.0f;
        if (p.pos != nullptr) p.pos[b * p.psb + h * p.psh + slot] = position;
      }
    }
  }
  dst += ch * 16;
  if (kind == 2) {
#pragma unroll
    for (int i = 0; i < kApSteps; ++i) {
      if (h0 + i * RW >= heads) break;
      uint4* row = reinterpret_cast<uint4*>(dst + (h0 + i * RW) * dh);
      __stcs(row, x[i][0]);
      __stcs(row + L, x[i][1]);
    }
    return;
  }

  // [half]: x'[half] = rs * (x[half] * near[half] + x[other half] * far[half]), where the first
  // half's far factor has a minus
  float2 near[2][N / 2], far[2][N / 2];
  const void* w = kind == 0 ? p.qw : p.kw;
  {
    const int64_t row = static_cast<int64_t>(fine ? position : 0) * D + ch * N;
    float wt[2][N];
    if (w != nullptr) {
      ap_load<T, N>(w, ch * N, wt[0]);
      ap_load<T, N>(w, ch * N + D / 2, wt[1]);
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float c[N], s[N];
      ap_load<TC, N>(p.cos, row + half * (D / 2), c);
      ap_load<TC, N>(p.sin, row + half * (D / 2), s);
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        near[half][e / 2] = w != nullptr ? make_float2(c[e] * wt[half][e], c[e + 1] * wt[half][e + 1])
                                         : make_float2(c[e], c[e + 1]);
        const float2 f = w != nullptr ? make_float2(s[e] * wt[1 - half][e], s[e + 1] * wt[1 - half][e + 1])
                                      : make_float2(s[e], s[e + 1]);
        far[half][e / 2] = half == 0 ? make_float2(-f.x, -f.y) : f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kApSteps; ++i) {
    float2 a[2][N / 2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float f[N];
      ElemTraits<T>::widen(x[i][half], f);
#pragma unroll
      for (int e = 0; e < N; e += 2) a[half][e / 2] = make_float2(f[e], f[e + 1]);
    }
    const float2 zero = make_float2(0.0f, 0.0f);
    float2 rs = make_float2(1.0f, 1.0f);
    if (w != nullptr) {
      float2 s2 = zero;
#pragma unroll
      for (int e = 0; e < N / 2; ++e) s2 = ffma2(a[1][e], a[1][e], ffma2(a[0][e], a[0][e], s2));
      float ss = s2.x + s2.y;
#pragma unroll
      for (int o = L / 2; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      rs.x = rs.y = rsqrtf(ss * (1.0f / D) + p.eps);
    }
    uint4 r[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float2 out[N / 2];
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        out[e] = ffma2(a[half][e], near[half][e], ffma2(a[1 - half][e], far[half][e], zero));
        if (w != nullptr) out[e] = ffma2(out[e], rs, zero);
      }
      r[half] = ap_round<T>(out);
    }
    if (h0 + i * RW >= heads) continue;
    uint4* row = reinterpret_cast<uint4*>(dst + (h0 + i * RW) * dh);
    __stcs(row, fine ? r[0] : make_uint4(0u, 0u, 0u, 0u));
    __stcs(row + L, fine ? r[1] : make_uint4(0u, 0u, 0u, 0u));
  }
}

template <typename T, typename TC>
static cudaError_t launch_paged_append(const PagedAppendParams& p, int D, cudaStream_t s) {
  const int per = kApSteps * 64 * ElemTraits<T>::kPerChunk / D;  // heads per warp
  const int64_t warps = static_cast<int64_t>(p.T) * ((p.H + per - 1) / per + 2 * ((p.H_kv + per - 1) / per));
  const unsigned grid = static_cast<unsigned>((warps + kApWarps - 1) / kApWarps);
  return launch_dependent(D == 64 ? paged_append_kernel<T, TC, 64> : paged_append_kernel<T, TC, 128>,
                          dim3(grid), dim3(kApWarps * 32), 0, s, 1, p);
}

}  // namespace dcr

using namespace dcr;

extern "C" int dcr_paged_append(
    const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k, int64_t k_stride_t,
    int64_t k_stride_h, const void* v, int64_t v_stride_t, int64_t v_stride_h,
    const void* q_weight, const void* k_weight, float eps, const void* cos, const void* sin,
    int table_dtype, int n_pos, const int32_t* positions, const int32_t* seq,
    const int32_t* slots, int dtype, int T, int H, int H_kv, int D, void* q_out, void* k_pages,
    void* v_pages, int64_t kp_stride_p, int64_t kp_stride_h, int64_t kp_stride_s,
    int64_t vp_stride_p, int64_t vp_stride_h, int64_t vp_stride_s, int num_pages, int page_size,
    const int32_t* page_table, int64_t table_stride, int n_seq, int max_pages, float* weights,
    int64_t w_stride_b, int64_t w_stride_h, int32_t* pos, int64_t p_stride_b,
    int64_t p_stride_h, void* stream) {
  if (q == nullptr || k == nullptr || v == nullptr || cos == nullptr || sin == nullptr ||
      positions == nullptr || slots == nullptr || q_out == nullptr)
    return DCR_ERR_NULL;
  if (T <= 0 || H <= 0 || n_pos <= 0 || n_seq <= 0) return DCR_ERR_SHAPE;
  if (seq == nullptr && T > n_seq) return DCR_ERR_SHAPE;
  const int st = check_pool(k_pages, v_pages, dtype, kp_stride_p, kp_stride_h, kp_stride_s,
                            vp_stride_p, vp_stride_h, vp_stride_s, num_pages, page_size,
                            page_table, table_stride, max_pages, H_kv, D);
  if (st != DCR_OK) return st;
  if (H % H_kv != 0) return DCR_ERR_SHAPE;
  if (static_cast<int64_t>(T) * (H + 2 * static_cast<int64_t>(H_kv)) > 0x7fffff00ll)
    return DCR_ERR_SHAPE;
  if (table_dtype != dtype && table_dtype != DCR_DTYPE_F32) return DCR_ERR_DTYPE;
  const int64_t per16 = dtype == DCR_DTYPE_F32 ? 4 : 8;
  const int64_t strides[6] = {q_stride_t, q_stride_h, k_stride_t, k_stride_h, v_stride_t, v_stride_h};
  for (int i = 0; i < 6; ++i) {
    if (strides[i] < 0) return DCR_ERR_SHAPE;
    if (strides[i] % per16 != 0) return DCR_ERR_ALIGN;
  }
  if (misaligned(16, q, k, v, q_out, cos, sin, q_weight, k_weight) ||
      misaligned(4, positions, seq, slots, weights, pos))
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
  PagedAppendParams p;
  p.c = make_pool(k_pages, v_pages, kp_stride_p, kp_stride_h, kp_stride_s, vp_stride_p,
                  vp_stride_h, vp_stride_s, num_pages, page_size, page_table, table_stride,
                  max_pages);
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  p.q = q;
  p.k = k;
  p.v = v;
  p.qst = q_stride_t;
  p.qsh = q_stride_h;
  p.kst = k_stride_t;
  p.ksh = k_stride_h;
  p.vst = v_stride_t;
  p.vsh = v_stride_h;
  p.qw = q_weight;
  p.kw = k_weight;
  p.cos = cos;
  p.sin = sin;
  p.n_pos = n_pos;
  p.positions = positions;
  p.seq = seq;
  p.slots = slots;
  p.T = T;
  p.H = H;
  p.H_kv = H_kv;
  p.n_seq = n_seq;
  p.eps = eps;
  p.q_out = q_out;
  p.weights = weights;
  p.wsb = w_stride_b;
  p.wsh = w_stride_h;
  p.pos = pos;
  p.psb = p_stride_b;
  p.psh = p_stride_h;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f32_tables = table_dtype == DCR_DTYPE_F32;
  cudaError_t e;
  if (dtype == DCR_DTYPE_BF16)
    e = f32_tables ? launch_paged_append<__nv_bfloat16, float>(p, D, s)
                   : launch_paged_append<__nv_bfloat16, __nv_bfloat16>(p, D, s);
  else if (dtype == DCR_DTYPE_F16)
    e = f32_tables ? launch_paged_append<__half, float>(p, D, s)
                   : launch_paged_append<__half, __half>(p, D, s);
  else
    e = launch_paged_append<float, float>(p, D, s);
  return e == cudaSuccess ? DCR_OK : DCR_ERR_CUDA;
}
