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
// One warp per (token, head row); a lane holds the rotation's pairs (i, i + D/2).
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

template <typename T>
__device__ __forceinline__ float ap_elem(const void* p, int64_t i) {
  if constexpr (sizeof(T) == 4)
    return static_cast<const float*>(p)[i];
  else
    return ElemTraits<T>::widen1(static_cast<const uint16_t*>(p)[i]);
}

template <typename T, typename TC, int D>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedAppendParams p) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int heads = p.H + 2 * p.H_kv;
  if (item >= static_cast<int64_t>(p.T) * heads) return;
  const int t = static_cast<int>(item / heads);
  const int r = static_cast<int>(item - static_cast<int64_t>(t) * heads);
  const bool is_q = r < p.H, is_v = r >= p.H + p.H_kv;
  const int h = is_q ? r : is_v ? r - p.H - p.H_kv : r - p.H;
  const void* src = is_q ? p.q : is_v ? p.v : p.k;
  const int64_t at = is_q ? t * p.qst + h * p.qsh : is_v ? t * p.vst + h * p.vsh : t * p.kst + h * p.ksh;
  float x[2][E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    x[0][e] = ap_elem<T>(src, at + lane + 32 * e);
    x[1][e] = ap_elem<T>(src, at + lane + 32 * e + D / 2);
  }
  const int position = p.positions[t];
  const bool fine = position >= 0 && position < p.n_pos;
  if (!fine) raise_status(DCR_ERR_DEVICE_INDEX);
  if (!is_v) {
    const void* w = is_q ? p.qw : p.kw;
    if (w != nullptr) {
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) ss = fmaf(x[0][e], x[0][e], fmaf(x[1][e], x[1][e], ss));
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float rs = rsqrtf(ss / D + p.eps);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x[0][e] *= rs * ap_elem<T>(w, lane + 32 * e);
        x[1][e] *= rs * ap_elem<T>(w, lane + 32 * e + D / 2);
      }
    }
    const int64_t row = static_cast<int64_t>(fine ? position : 0) * D;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int64_t i = row + lane + 32 * e;
      const float a = x[0][e], b = x[1][e];
      x[0][e] = fine ? a * ap_elem<TC>(p.cos, i) - b * ap_elem<TC>(p.sin, i) : 0.0f;
      x[1][e] = fine ? b * ap_elem<TC>(p.cos, i + D / 2) + a * ap_elem<TC>(p.sin, i + D / 2) : 0.0f;
    }
  }
  T* dst;
  if (is_q) {
    dst = static_cast<T*>(p.q_out) + (static_cast<int64_t>(t) * p.H + h) * D;
  } else {
    const int slot = p.slots[t];
    if (slot < 0 || !fine) return;
    const int b = p.seq != nullptr ? p.seq[t] : t;
    if (b < 0 || b >= p.n_seq || slot >= p.c.max_pages * static_cast<int>(p.c.page.d)) {
      raise_status(DCR_ERR_DEVICE_INDEX);
      return;
    }
    const uint32_t pi = p.c.page.div(slot);
    const int pg = page_of(p.c, b, pi);
    if (pg < 0) {  // a key without a mapped page would be lost
      raise_status(DCR_ERR_DEVICE_INDEX);
      return;
    }
    const int in = slot - pi * p.c.page.d;
    dst = is_v ? static_cast<T*>(p.v_pages) + pg * p.c.vsp + h * p.c.vsh + in * p.c.vsr
               : static_cast<T*>(p.k_pages) + pg * p.c.ksp + h * p.c.ksh + in * p.c.ksr;
    if (!is_v && lane == 0) {
      if (p.weights != nullptr) p.weights[b * p.wsb + h * p.wsh + slot] = 0.0f;
      if (p.pos != nullptr) p.pos[b * p.psb + h * p.psh + slot] = position;
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    ElemTraits<T>::store(dst, lane + 32 * e, x[0][e]);
    ElemTraits<T>::store(dst, lane + 32 * e + D / 2, x[1][e]);
  }
}

template <typename T, typename TC>
static void launch_paged_append(const PagedAppendParams& p, int D, cudaStream_t s) {
  const int64_t items = static_cast<int64_t>(p.T) * (p.H + 2 * p.H_kv);
  const unsigned grid = static_cast<unsigned>((items + 7) / 8);
  if (D == 64)
    paged_append_kernel<T, TC, 64><<<grid, 256, 0, s>>>(p);
  else
    paged_append_kernel<T, TC, 128><<<grid, 256, 0, s>>>(p);
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
  if (static_cast<int64_t>(T) * (H + 2 * static_cast<int64_t>(H_kv)) > 0x7fffffffll)
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
  if (dtype == DCR_DTYPE_BF16) {
    if (f32_tables) launch_paged_append<__nv_bfloat16, float>(p, D, s);
    else launch_paged_append<__nv_bfloat16, __nv_bfloat16>(p, D, s);
  } else if (dtype == DCR_DTYPE_F16) {
    if (f32_tables) launch_paged_append<__half, float>(p, D, s);
    else launch_paged_append<__half, __half>(p, D, s);
  } else {
    launch_paged_append<float, float>(p, D, s);
  }
  return cudaGetLastError() == cudaSuccess ? DCR_OK : DCR_ERR_CUDA;
}
