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
// Bound: the rows, read and written once. A row is spread over its 16-byte chunks' lanes (8, 16
// or 32), so a warp takes 4, 2 or 1 rows at a time and every access is 16 bytes a lane; the
// element D/2 away sits in the lane half a row away and comes by shuffle. A warp takes up to
// kApSteps such steps of one token and kind (query, key, value): the token's table rows times
// the norm weight are folded into two factors once, x' = rs * (x * (w c) + x_far * (w_far s)),
// and all its rows are in flight before the first is used.
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
constexpr int kApSteps = 4;

// N consecutive elements from a 16-byte (or wider) aligned address, widened.
template <typename T, int N>
__device__ __forceinline__ void ap_load(const void* base, int64_t i, float (&f)[N]) {
  constexpr int kPer = ElemTraits<T>::kPerChunk;
  static_assert(N % kPer == 0, "whole chunks");
  const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(base) + i);
#pragma unroll
  for (int c = 0; c < N / kPer; ++c) {
    float x[kPer];
    ElemTraits<T>::widen(__ldg(src + c), x);
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

template <typename T, typename TC, int D>
__global__ void __launch_bounds__(kApWarps * 32) paged_append_kernel(const PagedAppendParams p) {
  constexpr int N = ElemTraits<T>::kPerChunk;  // elements per lane
  constexpr int L = D / N;                     // lanes per row
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
  const int64_t sh = kind == 0 ? p.qsh : kind == 1 ? p.ksh : p.vsh;
  uint4 x[kApSteps];
#pragma unroll
  for (int i = 0; i < kApSteps; ++i) {
    const int h = h0 + i * RW;
    x[i] = h < heads ? __ldg(reinterpret_cast<const uint4*>(src + (t * st + h * sh) * static_cast<int64_t>(sizeof(T))))
                     : make_uint4(0u, 0u, 0u, 0u);
  }
  const int position = __ldg(p.positions + t);
  const bool fine = position >= 0 && position < p.n_pos;
  if (!fine) raise_status(DCR_ERR_DEVICE_INDEX);

  char* dst;
  int64_t dh;  // bytes between heads
  if (kind == 0) {
    dst = static_cast<char*>(p.q_out) + static_cast<int64_t>(t) * p.H * (D * static_cast<int>(sizeof(T)));
    dh = D * static_cast<int>(sizeof(T));
  } else {
    const int slot = __ldg(p.slots + t);
    if (slot < 0 || !fine) return;
    const int b = p.seq != nullptr ? __ldg(p.seq + t) : t;
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
    for (int i = 0; i < kApSteps; ++i)
      if (h0 + i * RW < heads) *reinterpret_cast<uint4*>(dst + (h0 + i * RW) * dh) = x[i];
    return;
  }

  // x' = rs * (x * near + x_far * far); the far half of a row enters the near one with a minus
  float near[N], far[N];
  {
    const int64_t row = static_cast<int64_t>(fine ? position : 0) * D + ch * N;
    ap_load<TC, N>(p.cos, row, near);
    ap_load<TC, N>(p.sin, row, far);
    const float sign = ch < L / 2 ? -1.0f : 1.0f;
    const void* w = kind == 0 ? p.qw : p.kw;
    float wn[N], wf[N];
    if (w != nullptr) {
      ap_load<T, N>(w, ch * N, wn);
      ap_load<T, N>(w, (ch ^ (L / 2)) * N, wf);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      near[e] *= w != nullptr ? wn[e] : 1.0f;
      far[e] *= sign * (w != nullptr ? wf[e] : 1.0f);
    }
  }
  const bool norm = (kind == 0 ? p.qw : p.kw) != nullptr;
#pragma unroll
  for (int i = 0; i < kApSteps; ++i) {
    float a[N], b[N];
    ElemTraits<T>::widen(x[i], a);
    uint4 y;
    y.x = __shfl_xor_sync(0xffffffffu, x[i].x, L / 2);
    y.y = __shfl_xor_sync(0xffffffffu, x[i].y, L / 2);
    y.z = __shfl_xor_sync(0xffffffffu, x[i].z, L / 2);
    y.w = __shfl_xor_sync(0xffffffffu, x[i].w, L / 2);
    ElemTraits<T>::widen(y, b);
    float rs = 1.0f;
    if (norm) {
      float2 s2 = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        const float2 v = make_float2(a[e], a[e + 1]);
        s2 = ffma2(v, v, s2);
      }
      float ss = s2.x + s2.y;
#pragma unroll
      for (int o = L / 2; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      rs = rsqrtf(ss * (1.0f / D) + p.eps);
    }
    const float2 rs2 = make_float2(rs, rs), zero = make_float2(0.0f, 0.0f);
    float2 out[N / 2];
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 f = ffma2(make_float2(b[e], b[e + 1]), make_float2(far[e], far[e + 1]), zero);
      const float2 s = ffma2(make_float2(a[e], a[e + 1]), make_float2(near[e], near[e + 1]), f);
      out[e / 2] = norm ? ffma2(s, rs2, zero) : s;
    }
    if (h0 + i * RW >= heads) continue;
    uint4 r;
    if constexpr (N == 8) {
      r = make_uint4(ap_pack<T>(out[0].x, out[0].y), ap_pack<T>(out[1].x, out[1].y),
                     ap_pack<T>(out[2].x, out[2].y), ap_pack<T>(out[3].x, out[3].y));
    } else {
      r = make_uint4(__float_as_uint(out[0].x), __float_as_uint(out[0].y),
                     __float_as_uint(out[1].x), __float_as_uint(out[1].y));
    }
    *reinterpret_cast<uint4*>(dst + (h0 + i * RW) * dh) = fine ? r : make_uint4(0u, 0u, 0u, 0u);
  }
}

template <typename T, typename TC>
static cudaError_t launch_paged_append(const PagedAppendParams& p, int D, cudaStream_t s) {
  const int per = kApSteps * 32 * ElemTraits<T>::kPerChunk / D;  // heads per warp
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
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                         reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(q_out) |
                         reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin) |
                         reinterpret_cast<uintptr_t>(q_weight) | reinterpret_cast<uintptr_t>(k_weight);
  if (ptrs & 15u) return DCR_ERR_ALIGN;
  if ((weights != nullptr && (w_stride_b < 0 || w_stride_h < 0)) ||
      (pos != nullptr && (p_stride_b < 0 || p_stride_h < 0)))
    return DCR_ERR_SHAPE;
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
