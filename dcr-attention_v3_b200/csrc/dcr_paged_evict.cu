// dcr_paged_evict.cu — eviction from a paged cache by accumulated attention weight (sm_100a).
//
// For every (sequence b, KV head) whose n = lengths[b] slots exceed `budget`, keep `budget` of
// them: first the protected ones (position below `sinks`, or among the `recent` last of the
// seen[b] positions so far), then those of the largest weight; equal ones by the lower slot.
// -0 equals +0 and a NaN weight ranks above every number (the library's order of scores). The
// kept slots at or past the budget move, in slot order, into the evicted slots before it, so
// that the first `budget` slots hold what is kept and only rows that have to move are read:
// sources and destinations never overlap. src_out tells, for every slot below min(n, budget),
// the slot its row came from; weights and positions are gathered to new tables. The reference
// has no counterpart (its cache only grows).
//
// Kernel 1, one CTA a row: the budget-th largest 32-bit order key by four 8-bit histogram
// levels in shared memory, then one pass in slot order that matches holes and movers.
// Kernel 2: gathers the tables and moves the K and V rows.
#include "dcr_internal.h"
#include "dcr_paged.cuh"

namespace dcr {

constexpr int kEvThreads = 1024;

struct PagedEvictParams {
  PagePool c;
  void* k_pages;
  void* v_pages;
  const int32_t* lengths;
  const float* weights;
  int64_t wsb, wsh;
  const int32_t* pos;
  int64_t psb, psh;
  const int32_t* seen;
  int H_kv, budget, sinks, recent;
  int32_t* src;         // [B][H_kv][budget]
  float* w_out;
  int64_t wosb, wosh;
  int32_t* pos_out;
  int64_t posb, posh;
  int32_t* len_out;     // [B]
  int32_t* holes;       // [B * H_kv][budget]
};

// Order of a slot's claim to stay, as an unsigned key: larger stays first.
__device__ __forceinline__ uint32_t ev_key(float w, int pos, int sinks, int from) {
  if (pos < sinks || pos >= from) return 0xffffffffu;
  uint32_t u = __float_as_uint(w);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xfffffffeu;
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive sum of a flag over the CTA's threads in order, and the total.
__device__ __forceinline__ int ev_block_rank(bool f, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned b = __ballot_sync(0xffffffffu, f);
  if (lane == 0) warp_sums[warp] = __popc(b);
  __syncthreads();
  const int mine = warp_sums[lane];  // kEvThreads / 32 = 32 warps
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  total = __shfl_sync(0xffffffffu, incl, 31);
  const int before = __shfl_sync(0xffffffffu, incl - mine, warp);
  __syncthreads();
  return before + __popc(b & ((1u << lane) - 1u));
}

__global__ void __launch_bounds__(kEvThreads) paged_evict_select_kernel(const PagedEvictParams p) {
  __shared__ uint32_t hist[256];
  __shared__ int sums[32];
  __shared__ uint32_t found_s[2];
  const int tid = threadIdx.x;
  const int h = blockIdx.x, b = blockIdx.y;
  const int64_t row = static_cast<int64_t>(b) * p.H_kv + h;
  const int n = checked_length(p.c, p.lengths[b]);
  const int from = p.seen[b] - p.recent;
  const float* w = p.weights + b * p.wsb + h * p.wsh;
  const int32_t* ps = p.pos + b * p.psb + h * p.psh;
  int32_t* src = p.src + row * p.budget;
  if (h == 0 && tid == 0) p.len_out[b] = n < p.budget ? n : p.budget;
  if (n <= p.budget) {
    for (int i = tid; i < p.budget; i += kEvThreads) src[i] = i < n ? i : -1;
    return;
  }
  uint32_t prefix = 0, mask = 0, left = p.budget;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kEvThreads) {
      const uint32_t key = ev_key(w[i], ps[i], p.sinks, from);
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid < 32) {
      int bin;
      uint32_t above;
      warp_find_bin(hist, left, bin, above);
      if (tid == 0) {
        found_s[0] = static_cast<uint32_t>(bin);
        found_s[1] = above;
      }
    }
    __syncthreads();
    prefix |= found_s[0] << shift;
    mask |= 255u << shift;
    left -= found_s[1];
    __syncthreads();
  }
  // keys above `prefix` stay, and the first `left` that equal it
  int32_t* holes = p.holes + row * p.budget;
  int ties = 0, n_holes = 0, n_moves = 0;
  for (int base = 0; base < n; base += kEvThreads) {
    const int i = base + tid;
    const bool in = i < n;
    const uint32_t key = in ? ev_key(w[i], ps[i], p.sinks, from) : 0u;
    int total;
    const int tie = ties + ev_block_rank(in && key == prefix, sums, total);
    ties += total;
    const bool keep = in && (key > prefix || (key == prefix && tie < static_cast<int>(left)));
    const bool hole = in && !keep && i < p.budget;
    const int rank_h = n_holes + ev_block_rank(hole, sums, total);
    n_holes += total;
    if (hole) holes[rank_h] = i;
    if (keep && i < p.budget) src[i] = i;
    __syncthreads();  // the holes of this chunk and before are visible to its movers
    const bool move = keep && i >= p.budget;
    const int rank_m = n_moves + ev_block_rank(move, sums, total);
    n_moves += total;
    if (move) src[holes[rank_m]] = i;
  }
}

// One warp per destination slot.
template <int RowBytes>
__global__ void __launch_bounds__(256) paged_evict_move_kernel(const PagedEvictParams p) {
  const int lane = threadIdx.x & 31;
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int h = blockIdx.y, b = blockIdx.z;
  if (i >= p.budget) return;
  const int64_t row = static_cast<int64_t>(b) * p.H_kv + h;
  const int s = p.src[row * p.budget + i];
  if (lane == 0) {
    p.w_out[b * p.wosb + h * p.wosh + i] = s < 0 ? 0.0f : p.weights[b * p.wsb + h * p.wsh + s];
    p.pos_out[b * p.posb + h * p.posh + i] = s < 0 ? -1 : p.pos[b * p.psb + h * p.psh + s];
  }
  if (s < 0 || s == i) return;
  const uint32_t fi = p.c.page.div(s), ti = p.c.page.div(i);
  const int fp = page_of(p.c, b, fi), tp = page_of(p.c, b, ti);
  if (fp < 0 || tp < 0) {
    raise_status(DCR_ERR_DEVICE_INDEX);
    return;
  }
  const int64_t fs = s - static_cast<int64_t>(fi) * p.c.page.d, ts = i - static_cast<int64_t>(ti) * p.c.page.d;
  constexpr int kC = RowBytes / 16;  // strides below are in 16-byte chunks
  uint4* k = static_cast<uint4*>(p.k_pages);
  uint4* v = static_cast<uint4*>(p.v_pages);
  if (lane < kC) {
    k[tp * p.c.ksp + h * p.c.ksh + ts * p.c.ksr + lane] =
        k[fp * p.c.ksp + h * p.c.ksh + fs * p.c.ksr + lane];
    v[tp * p.c.vsp + h * p.c.vsh + ts * p.c.vsr + lane] =
        v[fp * p.c.vsp + h * p.c.vsh + fs * p.c.vsr + lane];
  }
}

}  // namespace dcr

using namespace dcr;

extern "C" {

size_t dcr_paged_evict_workspace_bytes(int B, int H_kv, int budget) {
  if (B <= 0 || H_kv <= 0 || budget <= 0) return 0;
  return sizeof(int32_t) * static_cast<size_t>(B) * H_kv * budget;
}

int dcr_paged_evict(void* k_pages, void* v_pages, int dtype, int64_t k_stride_p,
                    int64_t k_stride_h, int64_t k_stride_s, int64_t v_stride_p,
                    int64_t v_stride_h, int64_t v_stride_s, int num_pages, int page_size,
                    const int32_t* page_table, int64_t table_stride, int max_pages,
                    const int32_t* lengths, const float* weights, int64_t w_stride_b,
                    int64_t w_stride_h, const int32_t* pos, int64_t p_stride_b,
                    int64_t p_stride_h, const int32_t* seen, int B, int H_kv, int D, int budget,
                    int sinks, int recent, int32_t* src_out, float* weights_out,
                    int64_t wo_stride_b, int64_t wo_stride_h, int32_t* pos_out,
                    int64_t po_stride_b, int64_t po_stride_h, int32_t* lengths_out,
                    void* workspace, size_t workspace_bytes, void* stream) {
  if (lengths == nullptr || weights == nullptr || pos == nullptr || seen == nullptr ||
      src_out == nullptr || weights_out == nullptr || pos_out == nullptr || lengths_out == nullptr)
    return DCR_ERR_NULL;
  if (B <= 0 || B > 65535 || H_kv > 65535 || budget <= 0 || sinks < 0 || recent < 0)
    return DCR_ERR_SHAPE;
  const int st = check_pool(k_pages, v_pages, dtype, k_stride_p, k_stride_h, k_stride_s,
                            v_stride_p, v_stride_h, v_stride_s, num_pages, page_size, page_table,
                            table_stride, max_pages, H_kv, D);
  if (st != DCR_OK) return st;
  if (budget > max_pages * page_size) return DCR_ERR_SHAPE;
  // the tables are gathered, not updated in place
  if (weights_out == weights || pos_out == pos || lengths_out == lengths) return DCR_ERR_SHAPE;
  const int64_t strides[8] = {w_stride_b,  w_stride_h,  p_stride_b,  p_stride_h,
                              wo_stride_b, wo_stride_h, po_stride_b, po_stride_h};
  for (int i = 0; i < 8; ++i)
    if (strides[i] < 0) return DCR_ERR_SHAPE;
  if (workspace == nullptr || workspace_bytes < dcr_paged_evict_workspace_bytes(B, H_kv, budget))
    return DCR_ERR_WORKSPACE;
  const int64_t per16 = dtype == DCR_DTYPE_F32 ? 4 : 8;
  PagedEvictParams p;
  p.c = make_pool(k_pages, v_pages, k_stride_p / per16, k_stride_h / per16, k_stride_s / per16,
                  v_stride_p / per16, v_stride_h / per16, v_stride_s / per16, num_pages,
                  page_size, page_table, table_stride, max_pages);
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  p.lengths = lengths;
  p.weights = weights;
  p.wsb = w_stride_b;
  p.wsh = w_stride_h;
  p.pos = pos;
  p.psb = p_stride_b;
  p.psh = p_stride_h;
  p.seen = seen;
  p.H_kv = H_kv;
  p.budget = budget;
  p.sinks = sinks;
  p.recent = recent;
  p.src = src_out;
  p.w_out = weights_out;
  p.wosb = wo_stride_b;
  p.wosh = wo_stride_h;
  p.pos_out = pos_out;
  p.posb = po_stride_b;
  p.posh = po_stride_h;
  p.len_out = lengths_out;
  p.holes = static_cast<int32_t*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  paged_evict_select_kernel<<<dim3(H_kv, B), kEvThreads, 0, s>>>(p);
  if (cudaGetLastError() != cudaSuccess) return DCR_ERR_CUDA;
  const dim3 grid((budget + 7) / 8, H_kv, B);
  const int bytes = D * (dtype == DCR_DTYPE_F32 ? 4 : 2);
  if (bytes == 128) paged_evict_move_kernel<128><<<grid, 256, 0, s>>>(p);
  else if (bytes == 256) paged_evict_move_kernel<256><<<grid, 256, 0, s>>>(p);
  else paged_evict_move_kernel<512><<<grid, 256, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? DCR_OK : DCR_ERR_CUDA;
}

}  // extern "C"
