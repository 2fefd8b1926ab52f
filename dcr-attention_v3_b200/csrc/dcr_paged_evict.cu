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
// Bound: 8 bytes a slot for the selection and the moved rows' 2 * 2 * D * element bytes; with
// few slots, latency.
//
// Kernel 1, a cluster of C CTAs a row: every thread keeps its slots' 32-bit order keys in
// registers (a warp's slots are consecutive, 32 at a time); the budget-th largest key by three
// histogram levels (12, 10 and 10 bits) in shared memory, whose bins every CTA adds to the sums
// of all CTAs of its cluster (only bins that hold anything travel; reading all bins of all CTAs
// instead was 1.3 to 10 times slower); then one exchange of per-warp counts gives every warp the
// ranks of its holes and movers, which ballots spread over its slots in slot order. A table of a
// size that registers cannot hold is read again at every level. Kernel 2 (a programmatic
// dependent) pairs the i-th hole with the i-th mover and copies the rows, 16 bytes a lane. Up to
// kEvFew evictions a row, a decode step's steady state, are found one by one as the smallest claim
// left and moved by the first kernel itself. Measured: 32 rows of 32768 slots to 4916, 134,000 rows
// of 128 bytes moved in K and in V: 30.0 us a call, 2.6 TB/s of the 79 MB it cannot do without; 64 rows
// of 4917 slots, one to go: 7.7 us.
#include <cooperative_groups.h>

#include "dcr_internal.h"
#include "dcr_paged.cuh"

namespace dcr {

namespace cg = cooperative_groups;

constexpr int kEvThreads = 1024;
constexpr int kEvWarps = kEvThreads / 32;
constexpr int kEvBins = 4096;
// Evictions that are taken one by one. One by one / by the histograms, for 1, 2, 3 and 4 of them: 64
// rows of 4917 slots 7.4 / 10.8, 9.2 / 10.8, 11.2 / 11.0, 12.8 / 11.2 us; 256 rows of 1025 8.2 / 11.4,
// 10.2 / 11.5, 12.5 / 11.5, 14.3 / 11.5; 32 rows of 20001 8.8 / 13.3, 11.7 / 13.8, 14.2 / 13.8, 16.3 / 13.8.
constexpr int kEvFew = 2;
constexpr int kEvAllBins = kEvBins + 2048;  // of the three levels

struct PagedEvictParams {
  PagePool c;           // strides in 16-byte chunks
  void* k_pages;
  void* v_pages;
  const int32_t* lengths;
  const float* weights;
  int64_t wsb, wsh;
  const int32_t* pos;
  int64_t psb, psh;
  const int32_t* seen;
  int H_kv, budget, sinks, recent;
  int chunks;           // 16-byte chunks of a row
  int32_t* src;         // [B][H_kv][budget]
  float* w_out;
  int64_t wosb, wosh;
  int32_t* pos_out;
  int64_t posb, posh;
  int32_t* len_out;     // [B]
  int32_t* holes;       // [B * H_kv][budget]
  int32_t* movers;      // [B * H_kv][budget]
  int32_t* n_moves;     // [B * H_kv]
};

// Order of a slot's claim to stay, as an unsigned key (never 0): larger stays first.
__device__ __forceinline__ uint32_t ev_key(float w, int pos, int sinks, int from) {
  if (pos < sinks || pos >= from) return 0xffffffffu;
  uint32_t u = __float_as_uint(w);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xfffffffeu;
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// The whole CTA finds, from the top, the bin in which the k-th largest key of a histogram of
// 1024 * Q bins lies: res = (bin, number of keys above it).
template <int Q>
__device__ __forceinline__ void ev_find(const uint32_t* hist, uint32_t k, uint32_t* sums,
                                        uint32_t* res) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t c[Q], s = 0;
#pragma unroll
  for (int i = 0; i < Q; ++i) {  // descending bins
    c[i] = hist[(kEvThreads - tid) * Q - 1 - i];
    s += c[i];
  }
  const uint32_t incl = warp_incl_scan(s);
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  uint32_t before = lane < warp ? sums[lane] : 0u;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  uint32_t above = before + incl - s;
  if (above < k && k <= above + s) {
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      if (above < k && k <= above + c[i]) {
        res[0] = static_cast<uint32_t>(kEvThreads * Q - 1 - (tid * Q + i));
        res[1] = above;
      }
      above += c[i];
    }
  }
}

template <int VPT>
__global__ void __launch_bounds__(kEvThreads) paged_evict_select_kernel(const PagedEvictParams p) {
  extern __shared__ uint32_t hist[];         // the three levels' bins; clusters: and their sums
  __shared__ uint32_t sums[kEvWarps];
  __shared__ uint32_t res[2];
  __shared__ int4 counts[kEvWarps];          // per warp, then the sums before it
  __shared__ int4 totals[8];                 // per CTA of the cluster
  __shared__ uint64_t least_s[2][kEvWarps], least_c[2][8];
  __shared__ int gone_s[kEvFew];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // not before the wait: the second kernel reads the page table ahead of its own
  asm volatile("griddepcontrol.launch_dependents;");
  const int64_t row = blockIdx.x / C;
  const int b = static_cast<int>(row / p.H_kv), h = static_cast<int>(row - static_cast<int64_t>(b) * p.H_kv);
  const int n = checked_length(p.c, p.lengths[b]);
  const int from = p.seen[b] - p.recent;
  const float* w = p.weights + b * p.wsb + h * p.wsh;
  const int32_t* ps = p.pos + b * p.psb + h * p.psh;
  int32_t* src = p.src + row * p.budget;
  float* wo = p.w_out + b * p.wosb + h * p.wosh;
  int32_t* po = p.pos_out + b * p.posb + h * p.posh;
  if (h == 0 && rank == 0 && tid == 0) p.len_out[b] = n < p.budget ? n : p.budget;
  if (n <= p.budget) {  // nothing to evict: all CTAs of the cluster return
    for (int i = rank * kEvThreads + tid; i < p.budget; i += C * kEvThreads) {
      src[i] = i < n ? i : -1;
      wo[i] = i < n ? w[i] : 0.0f;
      po[i] = i < n ? ps[i] : -1;
    }
    if (rank == 0 && tid == 0) p.n_moves[row] = 0;
    return;
  }

  const int used = (n + C * kEvThreads - 1) / (C * kEvThreads);  // slots per thread
  const int base = (rank * kEvWarps + warp) * 32 * used + lane;  // slot j of this lane: + 32 j
  auto load = [&](int j) {
    const int i = base + 32 * j;
    return i < n ? ev_key(w[i], ps[i], p.sinks, from) : 0u;
  };
  // Every slot below the budget keeps its place at first; the second kernel fills the holes.
  // Batches of loads, so that no load waits for a store.
  constexpr int kBatch = VPT == 0 ? 8 : VPT < 8 ? VPT : 8;
  uint32_t keys[VPT > 0 ? VPT : 1];
#pragma unroll
  for (int j0 = 0; j0 < (VPT > 0 ? VPT : used); j0 += kBatch) {
    if (j0 >= used) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (VPT > 0) keys[VPT > 0 ? j0 + j : 0] = 0u;
      continue;
    }
    float wj[kBatch];
    int pj[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = base + 32 * (j0 + j);
      const bool in = j0 + j < used && i < n;
      wj[j] = in ? w[i] : 0.0f;
      pj[j] = in ? ps[i] : 0;
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = base + 32 * (j0 + j);
      const bool in = j0 + j < used && i < n;
      if (VPT > 0) keys[VPT > 0 ? j0 + j : 0] = in ? ev_key(wj[j], pj[j], p.sinks, from) : 0u;
      if (in && i < p.budget) {
        src[i] = i;
        wo[i] = wj[j];
        po[i] = pj[j];
      }
    }
  }
  auto each = [&](auto&& f) {
    if constexpr (VPT > 0) {
#pragma unroll
      for (int j = 0; j < VPT; ++j)
        if (j < used) f(j, keys[j]);
    } else {
      for (int j = 0; j < used; ++j) f(j, load(j));
    }
  };
  if (n - p.budget <= kEvFew) {
    // Few to evict: one after another the smallest claim, of equal ones the highest slot (the
    // order key above the slot's complement, so that the smallest pair goes).
    const int few = n - p.budget;
    uint64_t last = 0;
    for (int r = 0; r < few; ++r) {
      uint64_t m = ~0ull;
      each([&](int j, uint32_t key) {
        const uint64_t c = (static_cast<uint64_t>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(base + 32 * j));
        if (key != 0u && c > last && c < m) m = c;
      });
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        const uint64_t y = __shfl_xor_sync(0xffffffffu, m, o);
        m = y < m ? y : m;
      }
      if (lane == 0) least_s[r & 1][warp] = m;
      __syncthreads();  // the other half of least_s may still be read
      m = least_s[r & 1][lane];
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        const uint64_t y = __shfl_xor_sync(0xffffffffu, m, o);
        m = y < m ? y : m;
      }
      if (C > 1) {
        if (r == 0) cluster.sync();  // every CTA has begun
        if (tid < C) *cluster.map_shared_rank(&least_c[r & 1][rank], tid) = m;
        cluster.sync();
        for (int x = 0; x < C; ++x) m = least_c[r & 1][x] < m ? least_c[r & 1][x] : m;
      }
      last = m;
      if (tid == 0) gone_s[r] = static_cast<int>(0xffffffffu - static_cast<uint32_t>(m));
    }
    // all places below the budget are written (the barriers above), so the holes can be filled
    __syncthreads();
    if (rank != 0) return;
    if (tid == 0) p.n_moves[row] = 0;  // the second kernel has nothing to do
    if (warp >= few) return;
    // the warp-th hole and mover in slot order: holes are evicted slots below the budget, movers
    // the slots past it that stay
    int hole = -1, mover = -1, holes = 0, movers = 0;
    for (int r = 0; r < few; ++r) {
      const int slot = gone_s[r];
      int before = 0;
      for (int x = 0; x < few; ++x) before += gone_s[x] < slot;
      if (slot < p.budget) {
        if (before == warp) hole = slot;
        ++holes;
      }
    }
    for (int x = 0; x < few; ++x) {
      const int slot = p.budget + x;
      bool stays = true;
      for (int r = 0; r < few; ++r) stays = stays && gone_s[r] != slot;
      if (stays && movers++ == warp) mover = slot;
    }
    if (hole < 0 || mover < 0) return;  // holes and movers are as many
    const uint32_t fi = p.c.page.div(mover), ti = p.c.page.div(hole);
    const int fp = page_of(p.c, b, fi), tp = page_of(p.c, b, ti);
    const bool moves = fp >= 0 && tp >= 0;
    if (lane == 0) {
      src[hole] = moves ? mover : -1;
      wo[hole] = moves ? w[mover] : 0.0f;
      po[hole] = moves ? ps[mover] : -1;
    }
    if (!moves) {  // a row without a mapped page on either side
      raise_status(DCR_ERR_DEVICE_INDEX);
      return;
    }
    const int64_t fs = mover - static_cast<int>(fi * p.c.page.d), ts = hole - static_cast<int>(ti * p.c.page.d);
    uint4* k = static_cast<uint4*>(p.k_pages) + h * p.c.ksh + lane;
    uint4* v = static_cast<uint4*>(p.v_pages) + h * p.c.vsh + lane;
    if (lane < p.chunks) {
      k[tp * p.c.ksp + ts * p.c.ksr] = k[fp * p.c.ksp + fs * p.c.ksr];
      v[tp * p.c.vsp + ts * p.c.vsr] = v[fp * p.c.vsp + fs * p.c.vsr];
    }
    return;
  }

  for (int i = tid; i < (C > 1 ? 2 : 1) * kEvAllBins; i += kEvThreads) hist[i] = 0;
  if (C > 1)
    cluster.sync();
  else
    __syncthreads();

  // the threshold T = prefix, level by level: `left` counts from the top within the prefix
  uint32_t prefix = 0, left = p.budget;
  auto level = [&](int shift, int bits, uint32_t* bins, auto q) {
    constexpr int Q = decltype(q)::value;
    const uint32_t above_mask = bits + shift == 32 ? 0u : 0xffffffffu << (bits + shift);
    each([&](int, uint32_t key) {
      if (key != 0u && ((key ^ prefix) & above_mask) == 0u)
        atomicAdd(bins + ((key >> shift) & ((1u << bits) - 1u)), 1u);
    });
    __syncthreads();
    if (C > 1) {
      for (int i = tid; i < (1 << bits); i += kEvThreads) {
        const uint32_t c = bins[i];
        if (c == 0u) continue;
        for (int r = 0; r < C; ++r) atomicAdd(cluster.map_shared_rank(bins + kEvAllBins + i, r), c);
      }
      cluster.sync();
    }
    ev_find<Q>(C > 1 ? bins + kEvAllBins : bins, left, sums, res);
    __syncthreads();
    prefix |= res[0] << shift;
    left -= res[1];
  };
  level(20, 12, hist, std::integral_constant<int, 4>());
  level(10, 10, hist + kEvBins, std::integral_constant<int, 1>());
  level(0, 10, hist + kEvBins + 1024, std::integral_constant<int, 1>());

  // Keys above T stay, and the first `left` that equal it. Per warp: evicted slots below the
  // budget and kept ones past it, ties aside (x, y), and ties below and past the budget (z, w).
  int4 mine = make_int4(0, 0, 0, 0);
  each([&](int j, uint32_t key) {
    const bool lo = base + 32 * j < p.budget, tie = key == prefix;
    mine.x += __popc(__ballot_sync(0xffffffffu, key != 0u && lo && key < prefix));
    mine.y += __popc(__ballot_sync(0xffffffffu, !lo && key > prefix));
    mine.z += __popc(__ballot_sync(0xffffffffu, lo && tie));
    mine.w += __popc(__ballot_sync(0xffffffffu, !lo && tie));
  });
  if (lane == 0) counts[warp] = mine;
  __syncthreads();
  if (warp == 0) {
    const int4 c = counts[lane];
    int4 s;
    s.x = static_cast<int>(warp_incl_scan(c.x));
    s.y = static_cast<int>(warp_incl_scan(c.y));
    s.z = static_cast<int>(warp_incl_scan(c.z));
    s.w = static_cast<int>(warp_incl_scan(c.w));
    counts[lane] = make_int4(s.x - c.x, s.y - c.y, s.z - c.z, s.w - c.w);
    int4 t;
    t.x = __shfl_sync(0xffffffffu, s.x, 31);
    t.y = __shfl_sync(0xffffffffu, s.y, 31);
    t.z = __shfl_sync(0xffffffffu, s.z, 31);
    t.w = __shfl_sync(0xffffffffu, s.w, 31);
    if (lane < C) *cluster.map_shared_rank(&totals[rank], lane) = t;
  }
  if (C > 1)
    cluster.sync();
  else
    __syncthreads();
  int4 at = counts[warp];
  int past_total = 0, ties_below = 0;
  for (int r = 0; r < C; ++r) {
    const int4 t = totals[r];
    past_total += t.y;
    ties_below += t.z;
    if (r < rank) {
      at.x += t.x;
      at.y += t.y;
      at.z += t.z;
      at.w += t.w;
    }
  }
  const int quota = static_cast<int>(left);
  if (rank == 0 && tid == 0) p.n_moves[row] = past_total + quota - min(quota, ties_below);
  int tie0 = at.z + at.w;                                       // ties before this warp
  int hole0 = at.x + at.z - min(at.z, quota);                   // evicted slots below the budget
  int move0 = at.y + min(quota, tie0) - min(quota, at.z);       // kept slots past it
  int32_t* holes = p.holes + row * p.budget;
  int32_t* movers = p.movers + row * p.budget;
  const unsigned below = (1u << lane) - 1u;
  each([&](int j, uint32_t key) {
    const int i = base + 32 * j;
    const bool lo = i < p.budget, tie = key == prefix;
    const unsigned bt = __ballot_sync(0xffffffffu, tie);
    const bool keep = key > prefix || (tie && tie0 + __popc(bt & below) < quota);
    const bool hole = key != 0u && lo && !keep, move = keep && !lo;
    const unsigned bh = __ballot_sync(0xffffffffu, hole), bm = __ballot_sync(0xffffffffu, move);
    if (hole) holes[hole0 + __popc(bh & below)] = i;
    if (move) movers[move0 + __popc(bm & below)] = i;
    tie0 += __popc(bt);
    hole0 += __popc(bh);
    move0 += __popc(bm);
  });
}

// The i-th mover of a row goes to its i-th hole, kUnroll pairs per lane group at a time. The
// sequence's page table is read into shared memory before the first kernel is done (where it
// fits; an entry is checked where a move uses it, the others may hold anything), and a round's
// pairs while the round before is on its way, so that a round waits for one read of the rows (with
// three dependent reads a round and three waves of CTAs, the call for 134,000 pairs of 128-byte
// rows took 34.0 us instead of 31.9).
constexpr int kEvPages = 4096;

template <int RowBytes>
__global__ void __launch_bounds__(256) paged_evict_move_kernel(const PagedEvictParams p) {
  constexpr int L = RowBytes / 16, RW = 32 / L, kUnroll = 2;
  __shared__ int32_t pages[kEvPages];
  const int lane = threadIdx.x & 31;
  const int ch = lane % L;
  const int64_t row = blockIdx.y;
  const int b = static_cast<int>(row / p.H_kv), h = static_cast<int>(row - static_cast<int64_t>(b) * p.H_kv);
  const bool local = p.c.max_pages <= kEvPages;
  if (local)
    for (int i = threadIdx.x; i < p.c.max_pages; i += 256) pages[i] = p.c.table[b * p.c.tstride + i];
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n = p.n_moves[row];
  const int32_t* holes = p.holes + row * p.budget;
  const int32_t* movers = p.movers + row * p.budget;
  uint4* k = static_cast<uint4*>(p.k_pages) + h * p.c.ksh + ch;
  uint4* v = static_cast<uint4*>(p.v_pages) + h * p.c.vsh + ch;
  const float* w = p.weights + b * p.wsb + h * p.wsh;
  const int32_t* ps = p.pos + b * p.psb + h * p.psh;
  const int step = gridDim.x * 8 * RW * kUnroll;
  int r0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * RW * kUnroll + lane / L;
  int d[kUnroll], f[kUnroll];
  auto pairs = [&](int r) {  // asked for before n is known; what lies past n is not used
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int at = r + i * RW;
      d[i] = at < p.budget ? holes[at] : 0;
      f[i] = at < p.budget ? movers[at] : 0;
    }
  };
  pairs(r0);
  while (r0 < n) {
    uint4 kx[kUnroll], vx[kUnroll];
    int64_t tk[kUnroll], tv[kUnroll];
    int to[kUnroll], from[kUnroll];
    bool moves[kUnroll];
    float wx[kUnroll];
    int px[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      to[i] = r0 + i * RW < n ? d[i] : -1;
      from[i] = f[i];
      moves[i] = false;
      if (to[i] < 0) continue;
      const uint32_t fi = p.c.page.div(from[i]), ti = p.c.page.div(to[i]);
      const int fp = local ? checked_page(p.c, pages[fi]) : page_of(p.c, b, fi);
      const int tp = local ? checked_page(p.c, pages[ti]) : page_of(p.c, b, ti);
      if (ch == 0) {
        wx[i] = w[from[i]];
        px[i] = ps[from[i]];
      }
      if (fp < 0 || tp < 0) {  // a row without a mapped page on either side
        raise_status(DCR_ERR_DEVICE_INDEX);
        from[i] = px[i] = -1;
        wx[i] = 0.0f;
        continue;
      }
      moves[i] = true;
      const int64_t fs = from[i] - static_cast<int>(fi * p.c.page.d), ts = to[i] - static_cast<int>(ti * p.c.page.d);
      kx[i] = k[fp * p.c.ksp + fs * p.c.ksr];
      vx[i] = v[fp * p.c.vsp + fs * p.c.vsr];
      tk[i] = tp * p.c.ksp + ts * p.c.ksr;
      tv[i] = tp * p.c.vsp + ts * p.c.vsr;
    }
    r0 += step;
    pairs(r0);
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      if (to[i] < 0) continue;
      if (ch == 0) {
        p.src[row * p.budget + to[i]] = from[i];
        p.w_out[b * p.wosb + h * p.wosh + to[i]] = wx[i];
        p.pos_out[b * p.posb + h * p.posh + to[i]] = px[i];
      }
      if (!moves[i]) continue;
      k[tk[i]] = kx[i];
      v[tv[i]] = vx[i];
    }
  }
}

// Cluster size and register keys per thread: one CTA takes 8192 slots, since the levels'
// cluster barriers cost more than longer loops up to there (whole calls for rows x slots, C = 1 /
// 2 / 4 / 8: 32 x 8192 14.5 / 14.7 / 13.9 / 19.0 us, 128 x 8192 39.7 / 43.2 / 54.8 / 80.4, 32 x 32768
// 39.5 / 33.8 / 25.3 / 30.8, 8 x 32769 89.4 / 26.3 / 23.6 / 18.0); clusters grow past it
// while all rows' CTAs still fit the GPU at once, or as far as registers need it.
static int ev_launch_select(const PagedEvictParams& p, int rows, int slots, cudaStream_t s) {
  const int sms = device_sm_count();
  int C = 1;
  while (C < 8 && ((rows * 2 * C <= sms && slots > 8192 * C) || slots > 32 * kEvThreads * C)) C *= 2;
  const int need = (slots + C * kEvThreads - 1) / (C * kEvThreads);
  const dim3 grid(static_cast<unsigned>(rows) * C), block(kEvThreads);
  auto kernel = need <= 4    ? paged_evict_select_kernel<4>
                : need <= 8  ? paged_evict_select_kernel<8>
                : need <= 32 ? paged_evict_select_kernel<32>
                             : paged_evict_select_kernel<0>;
  const size_t smem = sizeof(uint32_t) * kEvAllBins * (C > 1 ? 2 : 1);
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), 2 * 4 * kEvAllBins);
  if (e == cudaSuccess) e = launch_dependent(kernel, grid, block, smem, s, C, p);
  return e == cudaSuccess ? DCR_OK : DCR_ERR_CUDA;
}

template <int RowBytes>
static int ev_launch_move(const PagedEvictParams& p, int rows, int most, cudaStream_t s) {
  constexpr int kPer = 8 * (32 * 16 / RowBytes) * 2;  // pairs a CTA takes at once
  int x = (most + kPer - 1) / kPer;
  const int cap = (device_sm_count() * 3 + rows - 1) / rows;  // the GPU full once
  if (x > cap) x = cap;
  return launch_dependent(paged_evict_move_kernel<RowBytes>, dim3(x, rows), dim3(256), 0, s, 1, p) ==
                 cudaSuccess
             ? DCR_OK
             : DCR_ERR_CUDA;
}

}  // namespace dcr

using namespace dcr;

extern "C" {

size_t dcr_paged_evict_workspace_bytes(int B, int H_kv, int budget) {
  if (B <= 0 || H_kv <= 0 || budget <= 0) return 0;
  return sizeof(int32_t) * static_cast<size_t>(B) * H_kv * (2 * static_cast<size_t>(budget) + 1);
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
  if (B <= 0 || static_cast<int64_t>(B) * H_kv > 65535 || budget <= 0 || sinks < 0 || recent < 0)
    return DCR_ERR_SHAPE;
  const int st = check_pool(k_pages, v_pages, dtype, k_stride_p, k_stride_h, k_stride_s,
                            v_stride_p, v_stride_h, v_stride_s, num_pages, page_size, page_table,
                            table_stride, max_pages, H_kv, D);
  if (st != DCR_OK) return st;
  if (budget > max_pages * page_size) return DCR_ERR_SHAPE;
  if (misaligned(4, lengths, weights, pos, seen, src_out, weights_out, pos_out, lengths_out))
    return DCR_ERR_ALIGN;
  // the tables are gathered, not updated in place
  if (weights_out == weights || pos_out == pos || lengths_out == lengths) return DCR_ERR_SHAPE;
  const int64_t strides[8] = {w_stride_b,  w_stride_h,  p_stride_b,  p_stride_h,
                              wo_stride_b, wo_stride_h, po_stride_b, po_stride_h};
  for (int i = 0; i < 8; ++i)
    if (strides[i] < 0) return DCR_ERR_SHAPE;
  if (!rows_apart(B, H_kv, budget, wo_stride_b, wo_stride_h) ||
      !rows_apart(B, H_kv, budget, po_stride_b, po_stride_h))
    return DCR_ERR_SHAPE;
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15u) ||
      workspace_bytes < dcr_paged_evict_workspace_bytes(B, H_kv, budget))
    return DCR_ERR_WORKSPACE;
  const int64_t cap = static_cast<int64_t>(max_pages) * page_size;
  const TableSpan w_in(weights, B, H_kv, cap, w_stride_b, w_stride_h);
  const TableSpan p_in(pos, B, H_kv, cap, p_stride_b, p_stride_h);
  const TableSpan w_to(weights_out, B, H_kv, budget, wo_stride_b, wo_stride_h);
  const TableSpan p_to(pos_out, B, H_kv, budget, po_stride_b, po_stride_h);
  if (tables_meet(w_in, w_to) || tables_meet(p_in, w_to) || tables_meet(w_in, p_to) ||
      tables_meet(p_in, p_to) || tables_meet(w_to, p_to) ||
      tables_meet(TableSpan(lengths, 1, 1, B, 0, 0), TableSpan(lengths_out, 1, 1, B, 0, 0)))
    return DCR_ERR_SHAPE;
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
  p.chunks = static_cast<int>(D / per16);
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
  const int rows = B * H_kv, slots = max_pages * page_size;
  p.holes = static_cast<int32_t*>(workspace);
  p.movers = p.holes + static_cast<int64_t>(rows) * budget;
  p.n_moves = p.movers + static_cast<int64_t>(rows) * budget;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = ev_launch_select(p, rows, slots, s);
  if (rc != DCR_OK || slots == budget) return rc;  // no row holds more than the budget
  const int most = budget < slots - budget ? budget : slots - budget;
  const int bytes = D * (dtype == DCR_DTYPE_F32 ? 4 : 2);
  if (bytes == 128) return ev_launch_move<128>(p, rows, most, s);
  if (bytes == 256) return ev_launch_move<256>(p, rows, most, s);
  return ev_launch_move<512>(p, rows, most, s);
}

}  // extern "C"
