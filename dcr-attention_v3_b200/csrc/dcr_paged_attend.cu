// dcr_paged_attend.cu — attention of one new token per sequence over a paged cache (sm_100a).
//
// For sequence b, query head h and its KV head h / G, over the valid slots i (below the
// sequence's length, among its last `window` slots when window > 0, in a mapped page):
//   z_i = scale * q . k_i,  lse = log sum_i exp(z_i),  O = sum_i exp(z_i - lse) v_i
// and, on request, weights[b][h_kv][i] += sum over the KV head's G query heads of
// exp(z_i - lse). A row without valid slots gets O = 0 and lse = -inf and adds no weight; a
// score of -inf counts as a masked slot. The reference attends to one contiguous cache
// (dcr_attention/models/llama/attention.py:436); pages, windows and weights have no
// counterpart there.
//
// One CTA per (sequence, KV head), a warp per slot: online softmax in base 2, sums in fp32,
// the warps' states merged in shared memory, one rounding to the output type.
#include <math.h>

#include "dcr_internal.h"
#include "dcr_paged.cuh"

namespace dcr {

constexpr int kPaThreads = 256;
constexpr int kPaWarps = kPaThreads / 32;

struct PagedAttendParams {
  PagePool c;
  const void* q;
  int64_t qsb, qsh;
  const int32_t* lengths;
  int B, H, H_kv, G;
  float scale2;  // scale * log2(e)
  int window;
  void* o;        // [B][H][D]
  float* lse;     // [B][H] or null
  float* weights; // [B][H_kv][...] or null
  int64_t wsb, wsh;
};

template <typename T>
__device__ __forceinline__ float pa_elem(const void* p, int64_t i) {
  if constexpr (sizeof(T) == 4)
    return static_cast<const float*>(p)[i];
  else
    return ElemTraits<T>::widen1(static_cast<const uint16_t*>(p)[i]);
}

template <typename T, int D>
__global__ void __launch_bounds__(kPaThreads) paged_attend_kernel(const PagedAttendParams p) {
  constexpr int E = D / 32;
  __shared__ float m_s[kPaWarps], l_s[kPaWarps], o_s[kPaWarps][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.y, hk = blockIdx.x;
  const int n = checked_length(p.c, p.lengths[b]);
  const int lo = p.window > 0 && n > p.window ? n - p.window : 0;
  // z (base 2) of one slot for the query held in q; false if the slot's page is not mapped
  auto score = [&](const float (&q)[E], int i, int& pg, int& in) {
    const uint32_t pi = p.c.page.div(i);
    pg = page_of(p.c, b, pi);
    in = i - pi * p.c.page.d;
    if (pg < 0) return -INFINITY;
    const int64_t at = pg * p.c.ksp + hk * p.c.ksh + in * p.c.ksr;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], pa_elem<T>(p.c.k, at + lane + 32 * e), s);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s * p.scale2;
  };
  for (int pass = 0; pass < (p.weights != nullptr ? 2 : 1); ++pass) {
    for (int g = 0; g < p.G; ++g) {
      const int h = hk * p.G + g;
      float q[E], o[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        q[e] = pa_elem<T>(p.q, b * p.qsb + h * p.qsh + lane + 32 * e);
        o[e] = 0.0f;
      }
      float m = -INFINITY, l = 0.0f;
      const float lse2 = pass == 1 ? p.lse[static_cast<int64_t>(b) * p.H + h] : 0.0f;
      for (int i = lo + warp; i < n; i += kPaWarps) {
        int pg, in;
        const float z = score(q, i, pg, in);
        if (z == -INFINITY) continue;
        if (pass == 1) {  // the same warp adds every head's share of its slots, in head order
          if (lane == 0)
            p.weights[b * p.wsb + hk * p.wsh + i] += exp2f(z - lse2 * 1.4426950408889634f);
          continue;
        }
        const float mn = fmaxf(m, z);
        const float a = m == -INFINITY ? 0.0f : exp2f(m - mn);
        const float w = exp2f(z - mn);
        m = mn;
        l = fmaf(l, a, w);
        const int64_t at = pg * p.c.vsp + hk * p.c.vsh + in * p.c.vsr;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], a, w * pa_elem<T>(p.c.v, at + lane + 32 * e));
      }
      if (pass == 1) continue;
      if (lane == 0) {
        m_s[warp] = m;
        l_s[warp] = l;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) o_s[warp][lane + 32 * e] = o[e];
      __syncthreads();
      if (warp == 0) {
        float M = -INFINITY, L = 0.0f, acc[E] = {};
        for (int w = 0; w < kPaWarps; ++w) M = fmaxf(M, m_s[w]);
        for (int w = 0; w < kPaWarps; ++w) {
          const float a = m_s[w] == -INFINITY ? 0.0f : exp2f(m_s[w] - M);
          L = fmaf(a, l_s[w], L);
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] = fmaf(a, o_s[w][lane + 32 * e], acc[e]);
        }
        const int64_t row = static_cast<int64_t>(b) * p.H + h;
#pragma unroll
        for (int e = 0; e < E; ++e)
          ElemTraits<T>::store(static_cast<T*>(p.o) + row * D, lane + 32 * e,
                               L > 0.0f || L != L ? acc[e] / L : 0.0f);
        if (lane == 0 && p.lse != nullptr)
          p.lse[row] = M == -INFINITY ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
      }
      __syncthreads();
    }
  }
}

}  // namespace dcr

using namespace dcr;

extern "C" {

size_t dcr_paged_workspace_bytes(int B, int H, int H_kv, int D, int max_slots, int with_weights) {
  if (B <= 0 || H_kv <= 0 || H <= 0 || H % H_kv != 0 || (D != 64 && D != 128) || max_slots <= 0)
    return 0;
  return with_weights ? sizeof(float) * static_cast<size_t>(B) * H : 16;
}

int dcr_paged_attend(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* k_pages,
                     const void* v_pages, int dtype, int64_t k_stride_p, int64_t k_stride_h,
                     int64_t k_stride_s, int64_t v_stride_p, int64_t v_stride_h,
                     int64_t v_stride_s, int num_pages, int page_size, const int32_t* page_table,
                     int64_t table_stride, int max_pages, const int32_t* lengths, int B, int H,
                     int H_kv, int D, float scale, int window, void* o, float* lse,
                     float* weights, int64_t w_stride_b, int64_t w_stride_h, void* workspace,
                     size_t workspace_bytes, void* stream) {
  if (q == nullptr || lengths == nullptr || o == nullptr) return DCR_ERR_NULL;
  if (B <= 0 || B > 65535 || H <= 0 || H_kv <= 0 || H % H_kv != 0 || window < 0) return DCR_ERR_SHAPE;
  const int st = check_pool(k_pages, v_pages, dtype, k_stride_p, k_stride_h, k_stride_s,
                            v_stride_p, v_stride_h, v_stride_s, num_pages, page_size, page_table,
                            table_stride, max_pages, H_kv, D);
  if (st != DCR_OK) return st;
  const int64_t per16 = dtype == DCR_DTYPE_F32 ? 4 : 8;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o)) & 15u) ||
      q_stride_b % per16 || q_stride_h % per16)
    return DCR_ERR_ALIGN;
  if (q_stride_b < 0 || q_stride_h < 0) return DCR_ERR_SHAPE;
  const int max_slots = max_pages * page_size;
  if (weights != nullptr && (w_stride_h < 0 || w_stride_b < 0)) return DCR_ERR_SHAPE;
  if (workspace == nullptr ||
      workspace_bytes < dcr_paged_workspace_bytes(B, H, H_kv, D, max_slots, weights != nullptr))
    return DCR_ERR_WORKSPACE;
  PagedAttendParams p;
  p.c = make_pool(k_pages, v_pages, k_stride_p, k_stride_h, k_stride_s, v_stride_p, v_stride_h,
                  v_stride_s, num_pages, page_size, page_table, table_stride, max_pages);
  p.q = q;
  p.qsb = q_stride_b;
  p.qsh = q_stride_h;
  p.lengths = lengths;
  p.B = B;
  p.H = H;
  p.H_kv = H_kv;
  p.G = H / H_kv;
  p.scale2 = scale * 1.4426950408889634f;
  p.window = window;
  p.o = o;
  p.lse = lse != nullptr ? lse : weights != nullptr ? static_cast<float*>(workspace) : nullptr;
  p.weights = weights;
  p.wsb = w_stride_b;
  p.wsh = w_stride_h;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid(H_kv, B);
  switch (dtype * 2 + (D == 128)) {
    case 0: paged_attend_kernel<__nv_bfloat16, 64><<<grid, kPaThreads, 0, s>>>(p); break;
    case 1: paged_attend_kernel<__nv_bfloat16, 128><<<grid, kPaThreads, 0, s>>>(p); break;
    case 2: paged_attend_kernel<__half, 64><<<grid, kPaThreads, 0, s>>>(p); break;
    case 3: paged_attend_kernel<__half, 128><<<grid, kPaThreads, 0, s>>>(p); break;
    case 4: paged_attend_kernel<float, 64><<<grid, kPaThreads, 0, s>>>(p); break;
    default: paged_attend_kernel<float, 128><<<grid, kPaThreads, 0, s>>>(p); break;
  }
  return cudaGetLastError() == cudaSuccess ? DCR_OK : DCR_ERR_CUDA;
}

}  // extern "C"
