// dcr_paged_rows.cu — attention of many query rows against the same run of pages (sm_100a): a
// prompt's tokens over their sequence's cache, and a batch of single tokens over the prefix they
// share.
//
// A segment is a run of tokens that look into one sequence's page table: the new tokens of one
// sequence (prefill), or one token each of a group of sequences whose first slots are the same
// pages (shared). Its query rows of a KV head are (token, query head of the KV head), G per token;
// row r sees the slots [lo_r, hi_r) in mapped pages:
//   prefill   token i of n, at position x = length - n + i: hi = x + 1 (causal) or length,
//             lo = max(0, x + 1 - window) with a window
//   shared    hi = min(length, prefix), lo = max(0, length - window) with a window
//   z_j = scale * q . k_j,  lse = log sum_j exp(z_j),  O = sum_j exp(z_j - lse) v_j
// A row that sees nothing gets O = 0 and lse = -inf; a score of -inf counts as a masked slot. A
// slot that some row of a tile does not see must not reach it through 0 * inf or 0 * NaN, so where a
// tile is not seen whole, V's elements that are not finite are taken as 0 and the rows that do see
// such a slot become NaN. The reference attends to one contiguous cache and computes prompts densely
// (dcr_attention/models/llama/attention.py:436); pages, windows and shared prefixes have no
// counterpart there.
//
// Shared: the prefix is read once for a group instead of once for each of its sequences. Each
// sequence's own slots go through dcr_paged_attend.cu's kernels into fp32 rows; the parts' (m, l, o)
// are joined by rows_join_kernel, as are those of a run that is split over several CTAs.
//
// Bound: with many rows the exponentials, 16 a cycle and SM, which take 1024 cycles for 128 x 128 scores,
// as long as both products at D = 128 and twice as long at D = 64; with few rows K and V, read once.
// Measured (calls one after another in a CUDA graph; a tile of 256 rows and 128 slots takes 3100 to 3250
// cycles, of which 2080 are what its exponentials need, the rest waits for scores and their loads, and
// a CTA's beginning and end 14000): 2048 tokens on 32768 slots, 32 heads of 128 on 8, f16 (1.13 TFLOP):
// 1.03 to 1.16 ms by the card's power, 0.98 to 1.1 PFLOP/s; six prompts of 740 to 8192 tokens, heads of
// 64, bf16 (0.66 TFLOP): 1.10 ms, 600 TFLOP/s; 48 sequences of 2 to 5 drafted tokens, window 8191, f16
// (556 MB): 136 us, 4.1 TB/s; sequences of 5 tokens on 16000 slots, heads of 128, 8 of them 95 us, 9 (72
// CTAs) 135, 18 (a full wave, 1.2 GB) 178, 19 309; 45 samples of three documents of 7700 to 32768 slots, 64
// heads of 128 on 8, f16 (398 MB): 108 us; three prompts of 236 to 1499 slots in fp32: 237 us, 25 TFLOP/s.
// Tried and not kept: a whole tile's scores at once (1264 us for the six prompts, each step waits for
// its scores then; in halves 1256, before K and V came by the tensor map); the next half's scores loaded
// before this one's exponentials (1427 instead of 1221); an eighth, a quarter or a third of the
// exponentials as polynomials on the FMA pipe (1203, 1235 and more instead of 1221, and 1076, 1162
// instead of 1041 for the heads of 128); turns between the two blocks for the exponentials (1368
// instead of 1220); few rows four times over for shorter steps (no gain: loads set their pace).
#include <cuda.h>
#include <math.h>

#include <type_traits>

#include "dcr_internal.h"
#include "dcr_paged.cuh"
#include "dcr_tc.cuh"

namespace dcr {

struct RowsParams {
  PagePool c;
  const void* q;
  int64_t qst, qsh;
  const int32_t* lengths;  // of the sequences (prefill: segments; shared: tokens)
  const int32_t* starts;   // [nseg + 1] tokens of each segment
  const int32_t* prefix;   // shared: [T]; prefill: null
  int T, nseg, H, H_kv, G;
  FastDiv of_G;            // rows to tokens
  int pieces;              // CTAs that units are cut up for (0: a unit is one CTA's)
  int window, causal;
  float scale2;            // scale * log2(e)
  void* o;                 // [T][H][D]
  float* lse;              // [T][H] natural log, or null
  float* part_o;           // [places][D], or null: o and lse are written at once
  float2* part_ml;         // [places] base of the exponents and sum
  int64_t places;
  int2* part_of;           // [T][H] a row's first place (the next ones are a CTA's rows on) and their number
  int box;                 // neighbouring slots that a tensor-map copy brings in (0: no such copies)
};

// Tensor maps of the pool, for tiles that are whole: boxes of `box` slots of one page.
struct RowsMaps {
  CUtensorMap k, v;
};

// A CTA's rows: BM of a segment's, for one KV head.
struct RowsUnit {
  int seg, tok0, ntok, len;  // the segment, its tokens; prefill: its sequence's length
  int hk, split, parts;      // this CTA's part of the slots
  int row0, rows;            // first row in the segment and their number (0: nothing to do)
  int lo_min, lo_max, hi_min, hi_max;  // over the rows that see a slot
};

// The tokens of segment s; an inverted or outlying pair of starts raises the status.
__device__ __forceinline__ void rows_segment(const RowsParams& p, int s, int& tok0, int& ntok) {
  const int a = p.starts[s], b = p.starts[s + 1];
  if (a < 0 || b < a || b > p.T) {
    raise_status(DCR_ERR_DEVICE_INDEX);
    tok0 = ntok = 0;
    return;
  }
  tok0 = a;
  ntok = b - a;
}

// Row r's slots [x, y).
__device__ __forceinline__ int2 rows_limits(const RowsParams& p, const RowsUnit& u, int r) {
  const int i = static_cast<int>(p.of_G.div(u.row0 + r));
  if (p.prefix != nullptr) {
    const int len = checked_length(p.c, p.lengths[u.tok0 + i]);
    return make_int2(p.window > 0 ? max(0, len - p.window) : 0, min(len, p.prefix[u.tok0 + i]));
  }
  const int x = u.len - u.ntok + i;
  return make_int2(p.window > 0 ? max(0, x + 1 - p.window) : 0, p.causal ? x + 1 : u.len);
}

// Tiles of 128 slots that a segment's rows may see: how units are cut up goes by them, not what they
// see. A shared segment's are found by the whole CTA beforehand, those from the first slot that any of its
// tokens sees to the last, since its first token may wait (a length of 0) or share less than the others.
constexpr int kRowsWeights = 640;  // shared segments; those past them (no call with so many is cut up) count 1

__device__ __forceinline__ int rows_weight(const RowsParams& p, const int* found, int s, int tok0, int ntok) {
  if (ntok == 0) return 0;
  if (p.prefix != nullptr) return s < kRowsWeights ? found[s] : 1;
  const int hi = checked_length(p.c, p.lengths[s]);
  const int lo = p.window > 0 ? hi - ntok + 1 - p.window : 0;
  return max(1, (hi - max(lo, 0) + 127) / 128);
}

// The weights of shared segments, a warp a segment.
__device__ __forceinline__ void rows_find_weights(const RowsParams& p, int* found) {
  const int lane = threadIdx.x & 31, cap = p.c.max_pages * static_cast<int>(p.c.page.d);
#pragma unroll 1
  for (int s = threadIdx.x >> 5; s < min(p.nseg, kRowsWeights); s += blockDim.x >> 5) {
    int tok0, ntok, lo = INT32_MAX, hi = 0;
    rows_segment(p, s, tok0, ntok);
#pragma unroll 4
    for (int t = tok0 + lane; t < tok0 + ntok; t += 32) {
      const int len = min(p.lengths[t], cap), b = min(len, p.prefix[t]);
      const int a = p.window > 0 ? max(0, len - p.window) : 0;
      lo = min(lo, a < b ? a : INT32_MAX);
      hi = max(hi, a < b ? b : 0);
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) found[s] = lo < hi ? (hi - lo + 127) / 128 : 1;
  }
}

constexpr int kRowsMaxParts = 64;
constexpr int kRowsMinPart = 4;  // tiles of 128 slots: smaller parts gain nothing, larger ones idle SMs

// Finds this CTA's rows and their limits. A unit is a KV head's tile of BM rows of a segment. Where
// units are many (pieces = 0) blockIdx.x is one: heads of a tile side by side, a segment's tiles from the
// last to the first, since a causal segment's last rows see most, and segments from the one that sees
// most on, so that the grid ends on short units (up to 64 segments, two a lane; the units of more are so many
// that the grid's end is a small part of it). Else units are cut into parts of at most
// a number of slots, the least for which all parts are no more than the grid. False: nothing to do.
template <int BM>
__device__ __forceinline__ bool rows_begin(const RowsParams& p, RowsUnit& u, int2* limits) {
  __shared__ int found[kRowsWeights];
  const int lane = threadIdx.x & 31;
  if (p.prefix != nullptr) {
    rows_find_weights(p, found);
    __syncthreads();
  }
  if (threadIdx.x < 32) {
    const int per = (p.nseg + 31) >> 5;
    auto tiles_of = [&](int ntok) { return (ntok * p.G + BM - 1) / BM * p.H_kv; };  // units of a segment
    int chunk = 0;
    if (p.pieces > 0) {
      int most = 0;
      for (int j = 0; j < per; ++j) {
        const int s = lane * per + j;
        int tok0, ntok;
        if (s >= p.nseg) break;
        rows_segment(p, s, tok0, ntok);
        most = max(most, rows_weight(p, found, s, tok0, ntok));
      }
      most = __reduce_max_sync(0xffffffffu, most);
      int least = min(most, max(kRowsMinPart, (most + kRowsMaxParts - 1) / kRowsMaxParts));
      while (least < most) {  // parts are no more for a larger chunk
        const int mid = (least + most) >> 1;
        int n = 0;
        for (int j = 0; j < per; ++j) {
          const int s = lane * per + j;
          int tok0, ntok;
          if (s >= p.nseg) break;
          rows_segment(p, s, tok0, ntok);
          n += tiles_of(ntok) * ((rows_weight(p, found, s, tok0, ntok) + mid - 1) / mid);
        }
        n = __reduce_add_sync(0xffffffffu, n);
        if (n > p.pieces) least = mid + 1;
        else most = mid;
      }
      chunk = max(1, most);
    }
    if (lane == 0) u.rows = 0;
    __syncwarp();
    auto take = [&](int s, int tok0, int ntok, int parts, int unit, int split) {
      const int tile = unit / p.H_kv;
      u.seg = s;
      u.tok0 = tok0;
      u.ntok = ntok;
      u.len = p.prefix == nullptr ? checked_length(p.c, p.lengths[s]) : 0;
      u.hk = unit - tile * p.H_kv;
      u.split = split;
      u.parts = parts;
      u.row0 = tile * BM;
      u.rows = min(BM, ntok * p.G - u.row0);
      u.lo_min = u.hi_min = INT32_MAX;
      u.lo_max = u.hi_max = 0;
    };
    const int want = blockIdx.x;
    // with K segments a lane: this lane's, if it has the unit
    auto sorted = [&](auto k) {
      constexpr int K = decltype(k)::value;
      int tok0[K], ntok[K], weight[K], n[K], before[K] = {};
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int s = lane * K + j;
        tok0[j] = ntok[j] = weight[j] = 0;
        if (s < p.nseg) {
          rows_segment(p, s, tok0[j], ntok[j]);
          weight[j] = rows_weight(p, found, s, tok0[j], ntok[j]);
        }
        n[j] = tiles_of(ntok[j]);
      }
      const int lanes = (p.nseg + K - 1) / K;
#pragma unroll 4
      for (int o = 0; o < lanes; ++o)
#pragma unroll
        for (int i = 0; i < K; ++i) {
          const int w = __shfl_sync(0xffffffffu, weight[i], o), m = __shfl_sync(0xffffffffu, n[i], o);
#pragma unroll
          for (int j = 0; j < K; ++j)
            if (w > weight[j] || (w == weight[j] && o * K + i < lane * K + j)) before[j] += m;
        }
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int at = want - before[j];
        if (at >= 0 && at < n[j]) {
          const int tile = at / p.H_kv;  // from the last
          take(lane * K + j, tok0[j], ntok[j], 1, n[j] - (tile + 1) * p.H_kv + (at - tile * p.H_kv), 0);
        }
      }
    };
    if (p.pieces == 0 && p.nseg <= 32) {
      sorted(std::integral_constant<int, 1>());
    } else if (p.pieces == 0 && p.nseg <= 64) {
      sorted(std::integral_constant<int, 2>());
    } else {
      auto parts_of = [&](int s, int tok0, int ntok) {
        return p.pieces > 0 ? (rows_weight(p, found, s, tok0, ntok) + chunk - 1) / chunk : 1;
      };
      int mine = 0;
      for (int j = 0; j < per; ++j) {
        const int s = lane * per + j;
        int tok0, ntok;
        if (s >= p.nseg) break;
        rows_segment(p, s, tok0, ntok);
        mine += tiles_of(ntok) * parts_of(s, tok0, ntok);
      }
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      int before = upto - mine;
      for (int s = lane * per; want >= before && want < upto && s < p.nseg; ++s) {
        int tok0, ntok;
        rows_segment(p, s, tok0, ntok);
        const int parts = parts_of(s, tok0, ntok), n = tiles_of(ntok) * parts;
        if (want < before + n) {
          const int unit = (want - before) / parts;
          take(s, tok0, ntok, parts, unit, want - before - unit * parts);
          break;
        }
        before += n;
      }
    }
  }
  __syncthreads();
  if (u.rows == 0) return false;
  if (threadIdx.x < BM) {
    const int r = threadIdx.x;
    const bool in = r < u.rows;
    const int2 x = in ? rows_limits(p, u, r) : make_int2(0, 0);
    limits[r] = x;
    // A row that sees nothing (a sequence that waits) does not count: a tile that all others see is whole
    // for them. What is computed in its place is dropped in the end.
    const bool sees = in && x.x < x.y;
    const int a = __reduce_min_sync(0xffffffffu, sees ? x.x : INT32_MAX);
    const int b = __reduce_max_sync(0xffffffffu, sees ? x.x : 0);
    const int c = __reduce_min_sync(0xffffffffu, sees ? x.y : INT32_MAX);
    const int d = __reduce_max_sync(0xffffffffu, sees ? x.y : 0);
    if (lane == 0) {
      atomicMin(&u.lo_min, a);
      atomicMax(&u.lo_max, b);
      atomicMin(&u.hi_min, c);
      atomicMax(&u.hi_max, d);
    }
  }
  __syncthreads();
  return true;
}

// The tiles [x, y) of BN slots that are this CTA's.
template <int BN>
__device__ __forceinline__ int2 rows_tiles(const RowsParams& p, const RowsUnit& u) {
  if (u.lo_min >= u.hi_max) return make_int2(0, 0);
  const int a = u.lo_min / BN, n = (u.hi_max + BN - 1) / BN - a;
  return make_int2(a + static_cast<int>(static_cast<int64_t>(n) * u.split / u.parts),
                   a + static_cast<int>(static_cast<int64_t>(n) * (u.split + 1) / u.parts));
}

// Whether the CTA's rows are joined with others' before they are rounded; a whole unit of a prefill is
// written at once, and noted as no parts.
__device__ __forceinline__ bool rows_in_parts(const RowsParams& p, const RowsUnit& u) {
  return p.part_o != nullptr && (p.prefix != nullptr || u.parts > 1);
}

// Where row r of the CTA (output row `row`) leaves its part; the unit's first CTA notes where they are.
template <int BM>
__device__ __forceinline__ int64_t rows_place(const RowsParams& p, const RowsUnit& u, int r, int64_t row) {
  const int64_t at = p.pieces > 0 ? static_cast<int64_t>(blockIdx.x) * BM + r : row;
  if (u.split == 0) p.part_of[row] = make_int2(static_cast<int>(at), u.parts);
  return at;
}

// The page table's row of a segment: its sequence, or its first token's.
__device__ __forceinline__ int rows_table(const RowsParams& p, const RowsUnit& u) {
  return p.prefix != nullptr ? u.tok0 : u.seg;
}

__device__ __forceinline__ float rows_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Element offsets of slot j's K and V rows of the segment's head; false: not mapped, or past the
// last slot that any row sees.
__device__ __forceinline__ bool rows_slot(const RowsParams& p, const RowsUnit& u, int j, int64_t& k,
                                          int64_t& v) {
  k = v = 0;
  if (j < u.lo_min || j >= u.hi_max) return false;
  const uint32_t pi = p.c.page.div(j);
  const int pg = page_of(p.c, rows_table(p, u), pi);
  if (pg < 0) return false;
  const int64_t in = j - static_cast<int>(pi * p.c.page.d);
  k = pg * p.c.ksp + u.hk * p.c.ksh + in * p.c.ksr;
  v = pg * p.c.vsp + u.hk * p.c.vsh + in * p.c.vsr;
  return true;
}

__device__ __forceinline__ bool rows_finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// ---------------------------------------------------------------------------------------
// fp32 rows: 128 query rows against tiles of 64 slots with fp32 FMAs, 128 threads of 8 x 8 scores and 8 x
// D / 8 output elements each. Q and K lie transposed in shared memory, so a step of the inner loop
// reads eight neighbouring rows and eight slots in four 16-byte reads for 64 FMAs; V comes by cp.async while the scores are
// computed. Measured: three prompts of 236 to 1499 slots, 16 heads of 64: 237 us, 344 without cutting
// long units up; 64 rows and 4 x 4 scores a thread, four reads for 32 FMAs, took 314.
// ---------------------------------------------------------------------------------------
constexpr int kRfRows = 128, kRfSlots = 64, kRfThreads = 128;

template <int D>
struct RowsFma {
  static constexpr int WQ = kRfRows + 4, WK = kRfSlots + 4;  // words of a transposed row
  static constexpr int kSmem = 4 * (D * WQ + D * WK + kRfSlots * D + kRfSlots * WQ);
};

template <int D>
__global__ void __launch_bounds__(kRfThreads) rows_fma_kernel(const RowsParams p) {
  using S = RowsFma<D>;
  constexpr int WQ = S::WQ, WK = S::WK, C = D / 4, E = D / 32;  // chunks of a row; groups of 4 output dims
  extern __shared__ __align__(16) float rf_smem[];
  __shared__ RowsUnit u;
  __shared__ int2 limits[kRfRows];
  __shared__ int64_t koff[kRfSlots], voff[kRfSlots];
  __shared__ int flag[kRfSlots];  // 1: mapped; 2: V not finite
  float* qt = rf_smem;
  float* kt = qt + D * WQ;
  float* vs = kt + D * WK;
  float* pt = vs + kRfSlots * D;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  if (!rows_begin<kRfRows>(p, u, limits)) return;
  const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
  // Q and K by neighbouring rows: their elements go to neighbouring words of the transposed tile then
  for (int i = threadIdx.x; i < kRfRows * C; i += kRfThreads) {
    const int r = i % kRfRows, ch = i / kRfRows;
    float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (r < u.rows) {
      const int t = static_cast<int>(p.of_G.div(u.row0 + r)), g = u.row0 + r - t * p.G;
      f = reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + (u.tok0 + t) * p.qst +
                                          (u.hk * p.G + g) * p.qsh)[ch];
    }
    float* at = qt + 4 * ch * WQ + r;
    at[0] = f.x, at[WQ] = f.y, at[2 * WQ] = f.z, at[3 * WQ] = f.w;
  }
  float2 o[8][2 * E] = {};
  float m[8], l[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.0f;
  }
  unsigned poison = 0;  // a bit a row
  const int2 tiles = rows_tiles<kRfSlots>(p, u);
#pragma unroll 1
  for (int t = tiles.x; t < tiles.y; ++t) {
    const int j0 = t * kRfSlots;
    const bool seen = j0 >= u.lo_max && j0 + kRfSlots <= u.hi_min;  // whole, by every row that sees any
    __syncthreads();
    if (threadIdx.x < kRfSlots)
      flag[threadIdx.x] = rows_slot(p, u, j0 + threadIdx.x, koff[threadIdx.x], voff[threadIdx.x]);
    __syncthreads();
#pragma unroll 4
    for (int i = threadIdx.x; i < kRfSlots * C; i += kRfThreads) {
      const int j = i / C, ch = i - j * C;
      cp_async_16(vs + j * D + ch * 4, static_cast<const float*>(p.c.v) + voff[j] + ch * 4, flag[j] ? 16u : 0u);
    }
    cp_async_commit();
#pragma unroll 4
    for (int i = threadIdx.x; i < kRfSlots * C; i += kRfThreads) {
      const int j = i % kRfSlots, ch = i / kRfSlots;
      float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (flag[j]) f = reinterpret_cast<const float4*>(static_cast<const float*>(p.c.k) + koff[j])[ch];
      float* at = kt + 4 * ch * WK + j;
      at[0] = f.x, at[WK] = f.y, at[2 * WK] = f.z, at[3 * WK] = f.w;
    }
    __syncthreads();
    float2 s[8][4] = {};  // [row][slots 4 tx, 4 tx + 2, 32 + 4 tx, 34 + 4 tx and the next one]
#pragma unroll 4
    for (int d = 0; d < D; ++d) {
      const float4 a0 = *reinterpret_cast<const float4*>(qt + d * WQ + 8 * ty);
      const float4 a1 = *reinterpret_cast<const float4*>(qt + d * WQ + 8 * ty + 4);
      const float4 b0 = *reinterpret_cast<const float4*>(kt + d * WK + 4 * tx);
      const float4 b1 = *reinterpret_cast<const float4*>(kt + d * WK + 32 + 4 * tx);
      const float q[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
      const float2 k[4] = {make_float2(b0.x, b0.y), make_float2(b0.z, b0.w), make_float2(b1.x, b1.y),
                           make_float2(b1.z, b1.w)};
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = ffma2(make_float2(q[i], q[i]), k[e], s[i][e]);
    }
    cp_async_wait<0>();
    if (!seen) {  // a thread's own copies
      for (int i = threadIdx.x; i < kRfSlots * C; i += kRfThreads) {
        float* x = vs + i / C * D + i % C * 4;
        bool fine = true;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!rows_finite(x[e])) {
            fine = false;
            x[e] = 0.0f;
          }
        if (!fine) atomicOr(&flag[i / C], 2);
      }
      __syncthreads();
    }
    auto slot = [&](int e) { return e < 4 ? 4 * tx + e : 28 + 4 * tx + e; };
    unsigned held = 0, spoilt = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      held |= static_cast<unsigned>(flag[slot(e)] & 1) << e;
      spoilt |= static_cast<unsigned>(flag[slot(e)] >> 1) << e;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      unsigned in = held;
      if (!seen) {
        const int2 lim = limits[8 * ty + i];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (j0 + slot(e) < lim.x || j0 + slot(e) >= lim.y) in &= ~(1u << e);
        if ((in & spoilt) != 0) poison |= 1u << i;
      }
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][e].x = (in >> (2 * e)) & 1u ? s[i][e].x * p.scale2 : -INFINITY;
        s[i][e].y = (in >> (2 * e + 1)) & 1u ? s[i][e].y * p.scale2 : -INFINITY;
        top = fmaxf(top, fmaxf(s[i][e].x, s[i][e].y));
      }
#pragma unroll
      for (int x = 4; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float mn = fmaxf(m[i], top);
      if (mn > m[i]) {
        const float a = m[i] == -INFINITY ? 0.0f : rows_exp2(m[i] - mn);
        m[i] = mn;
        l[i] *= a;
#pragma unroll
        for (int e = 0; e < 2 * E; ++e) o[i][e] = make_float2(o[i][e].x * a, o[i][e].y * a);
      }
      const float base = mn == -INFINITY ? 0.0f : mn;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][e] = make_float2(rows_exp2(s[i][e].x - base), rows_exp2(s[i][e].y - base));
        l[i] += s[i][e].x + s[i][e].y;
      }
    }
    // the weights of slot(e) in row 8 e + tx, so that the lanes' words lie in different banks
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        auto w = [&](int r) { return e % 2 ? s[r][e / 2].y : s[r][e / 2].x; };
        *reinterpret_cast<float4*>(pt + (8 * e + tx) * WQ + 8 * ty + i) = make_float4(w(i), w(i + 1), w(i + 2), w(i + 3));
      }
    __syncthreads();
#pragma unroll 2
    for (int k = 0; k < kRfSlots; ++k) {
      const int j = k < 32 ? k % 8 * 4 + k / 8 : 28 + k % 8 * 4 + k / 8;
      const float4 a0 = *reinterpret_cast<const float4*>(pt + k * WQ + 8 * ty);
      const float4 a1 = *reinterpret_cast<const float4*>(pt + k * WQ + 8 * ty + 4);
      const float w[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
#pragma unroll
      for (int x = 0; x < E; ++x) {
        const float4 b = *reinterpret_cast<const float4*>(vs + j * D + 32 * x + 4 * tx);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          o[i][2 * x] = ffma2(make_float2(w[i], w[i]), make_float2(b.x, b.y), o[i][2 * x]);
          o[i][2 * x + 1] = ffma2(make_float2(w[i], w[i]), make_float2(b.z, b.w), o[i][2 * x + 1]);
        }
      }
    }
  }
#pragma unroll
  for (int x = 4; x >= 1; x >>= 1) poison |= __shfl_xor_sync(0xffffffffu, poison, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int x = 4; x >= 1; x >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
    const int r = 8 * ty + i;
    if (r >= u.rows) continue;
    if (limits[r].x >= limits[r].y) {  // it sees nothing
      m[i] = -INFINITY;
      l[i] = 0.0f;
    }
    const int t = static_cast<int>(p.of_G.div(u.row0 + r)), g = u.row0 + r - t * p.G;
    const int64_t row = static_cast<int64_t>(u.tok0 + t) * p.H + u.hk * p.G + g;
    const bool parts = rows_in_parts(p, u);
    const int64_t at = parts ? rows_place<kRfRows>(p, u, r, row) : row;
    if (!parts && p.part_of != nullptr) p.part_of[row] = make_int2(0, 0);
    const float spoil = (poison >> i) & 1u ? __int_as_float(0x7fffffff) : 1.0f;
    const bool none = l[i] == 0.0f;  // what is in its o may be anything
    const float by = none ? 0.0f : parts ? spoil : spoil / l[i];
    float* dst = (parts ? p.part_o : static_cast<float*>(p.o)) + at * D + 4 * tx;
#pragma unroll
    for (int x = 0; x < E; ++x) {
      const float2 c = none ? make_float2(0.0f, 0.0f) : o[i][2 * x], d = none ? c : o[i][2 * x + 1];
      *reinterpret_cast<float4*>(dst + 32 * x) = make_float4(c.x * by, c.y * by, d.x * by, d.y * by);
    }
    if (tx != 0) continue;
    if (parts) p.part_ml[at] = make_float2(m[i], l[i]);
    else if (p.lse != nullptr) p.lse[row] = l[i] == 0.0f ? -INFINITY : (m[i] + log2f(l[i])) * kLn2;
  }
}

// ---------------------------------------------------------------------------------------
// 16-bit rows: two blocks of 128 query rows against tiles of 128 slots on the tensor cores.
//
// Warps: two groups of four for the softmax, a row a thread; two groups of two that bring in K and V; two
// that issue the products, one for each softmax group. S = Q K^T of 64 slots goes to one of a group's
// two buffers in tensor memory; the softmax warps read their rows, keep the running base and sum (m, l)
// and write the weights P back over S; O += P V accumulates in tensor memory with P as its A operand.
// While a group computes on one buffer, S of the next 64 slots is made in the other. K and V tiles take
// turns in a ring. Where segments have more than 128 rows on average a CTA takes 256, a block for each
// group; else (Twin) 128, whose tiles the groups halve between them, and join what they hold at the
// end: one group alone would wait on its own chain of steps, at 13 bytes of K and V a cycle and SM.
//
// The base is raised only when a row's score is 8 above the largest it was set by, so O is rescaled
// for few steps, and then when the product of the step before is done. In f16 the base stays 7 below the
// maximum, so that small weights keep their bits (2^-24 of 2^7). A weight enters the second product
// rounded to 16 bits, off by half a step at most, as the output's own rounding. Errors against 64 bits are
// 1.02 to 1.06 times those of fp32 weights for the prompts above, and the square root of 2 times where a row's
// weights are alike and its values have no mean, so that both errors are as large (1200 tokens on 2048 to
// 32768 slots: f16 0.00029 instead of 0.00021, bf16 0.00235 instead of 0.00166). With Parts = 2 a weight's
// remainder goes in as well, in a second product: for shared prefixes, which are bound by their loads. Prompts
// would take 4 to 25% longer (the six 1278 us, the chunk 1246, the drafted tokens 146) for the errors of fp32
// weights, but for the chunk, whose error is that of its sums. Those are of 32 bits and lose a little with each
// product of 16 slots, as if truncated: a row's output is 3.5e-5 of itself too small behind 32768 slots, and
// 1.3e-4 behind 131072.
// ---------------------------------------------------------------------------------------
constexpr int kTcSlots = 128;

template <int D, bool Twin>
struct RowsTc {
  static constexpr int kRows = Twin ? 128 : 256;     // query rows a CTA
  static constexpr int kPanel = 128 * 128;           // bytes of 128 rows of 64 elements
  static constexpr int kTile = D / 64 * kPanel;
  static constexpr int kQ = kRows / 128 * kTile;
  // Places of K and V in turn: an even number, so that each of the two loader groups has its own. (A
  // thread that used another's could find the phase before the last one's parity, and take a place
  // that is still in use for released.)
  static constexpr int kStages = Twin ? (D == 64 ? 12 : 4) : (D == 64 ? 8 : 4);
  static_assert(kStages % 2 == 0, "places of K and V in turn");
  static constexpr int kSmem = 1024 + kQ + kStages * kTile;
  static constexpr int kColumns = 512;
  static constexpr int kLoad0 = 256;                 // first loader thread
  static constexpr int kMma = kLoad0 + 128;          // the issuing warps' first thread
  static constexpr int kThreads = kMma + 128;
  // Registers a thread: at launch, of the softmax warps and of the others.
  static constexpr int kAtLaunch = 128, kOthers = 56, kSoftmax = 200;
  static_assert(kLoad0 * kSoftmax + 256 * kOthers <= kThreads * kAtLaunch, "shares of the launch's registers");
};

struct RowsTcShared {
  RowsUnit u;
  uint64_t q_full, s_full[2][2], p_full[2][2], o_done[2][2], drained[2];  // [block][half]
  uint64_t full[12], empty[12];
  uint32_t tmem;
  uint32_t mask[16][4];         // mapped slots of the tiles in flight
  int64_t off[2][kTcSlots];     // element offsets of a loader group's slots
  int2 limits[256];
  float2 part[128];             // Twin: the second block's bases and sums
  uint8_t spoilt[256];          // rows that see a value that is not finite, in a tile not seen whole
};

template <typename T>
__device__ __forceinline__ uint32_t rows_pack(float a, float b, float& ra, float& rb) {
  uint32_t hi;
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    ra = a - f.x;
    rb = b - f.y;
    hi = *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    ra = a - __uint_as_float(hi << 16);
    rb = b - __uint_as_float(hi & 0xffff0000u);
  }
  return hi;
}

__device__ __forceinline__ float2 fadd2(float2 a, float2 b) { return ffma2(a, make_float2(1.0f, 1.0f), b); }

// Bits [from, to) of a word that begins at 0.
__device__ __forceinline__ uint32_t rows_bits(int from, int to) {
  from = max(0, min(32, from));
  to = max(0, min(32, to));
  const uint32_t below = to == 32 ? 0xffffffffu : (1u << to) - 1u;
  return from == 32 ? 0u : below & (0xffffffffu << from);
}

// Chunk ch of slot row r of a V tile at slot j0: elements that are not finite become 0, and rows that
// see the slot are noted.
template <typename T>
__device__ __forceinline__ void rows_tc_clean(RowsTcShared& sh, uint8_t* column, int j0, int r, int ch) {
  uint16_t* at = reinterpret_cast<uint16_t*>(column + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
  const uint4 w = *reinterpret_cast<const uint4*>(at);
  float f[8];
  ElemTraits<T>::widen(w, f);
  bool finite = true;
#pragma unroll
  for (int x = 0; x < 8; ++x) finite = finite && rows_finite(f[x]);
  if (finite) return;
  for (int x = 0; x < 8; ++x)
    if (!rows_finite(ElemTraits<T>::widen1(at[x]))) at[x] = 0;
  for (int x = 0; x < sh.u.rows; ++x)
    if (j0 + r >= sh.limits[x].x && j0 + r < sh.limits[x].y) sh.spoilt[x] = 1;
}

template <int N>
__device__ __forceinline__ void rows_hide(uint32_t (&s)[N], const uint32_t* words) {
#pragma unroll
  for (int c = 0; c < N; ++c)
    if (!((words[c / 32] >> (c % 32)) & 1u)) s[c] = 0xff800000u;  // -inf
}

// A group of two loader warps: the K or the V tiles of [tiles.x, tiles.y), into every other place of the
// ring. A thread looks up two slots, for the next tile ahead of this one's wait. A tile whose slots are
// all there comes by tensor-map copies of up to a page each, which announce themselves; the others (the
// ends, pages that are not mapped, pages of no multiple of 8 slots) by 16-byte cp.async, zeros for what
// is not there. (One group of four warps for K and V took 1800 cycles a tile of 16-slot pages.)
template <typename T, int D, bool Twin>
__device__ __forceinline__ void rows_tc_load(const RowsParams& p, const RowsMaps& maps, RowsTcShared& sh,
                                             uint8_t* ring, int2 tiles) {
  using S = RowsTc<D, Twin>;
  constexpr int C = D / 8, RP = 64 / C;  // chunks of a row, rows a step
  const RowsUnit& u = sh.u;
  const int kind = (threadIdx.x - S::kLoad0) / 64, gt = threadIdx.x % 64, lane = threadIdx.x & 31;  // 0: K, 1: V
  const int32_t* table = p.c.table + rows_table(p, u) * p.c.tstride;
  const void* map = kind ? &maps.v : &maps.k;
  const int64_t sp = kind ? p.c.vsp : p.c.ksp, sr = kind ? p.c.vsr : p.c.ksr;
  const T* base = static_cast<const T*>(kind ? p.c.v : p.c.k) + u.hk * (kind ? p.c.vsh : p.c.ksh) + gt % C * 8;
  const uint32_t column = (gt % C >> 3) * S::kPanel;
  int64_t* off = sh.off[kind];
  const int n = tiles.y - tiles.x;
  int pg[2];
  // the table's entries for the thread's slots of tile t (below 0: none that any row sees)
  auto look_up = [&](int t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = (tiles.x + t) * kTcSlots + gt + 64 * i;
      pg[i] = t < n && j >= u.lo_min && j < u.hi_max ? table[p.c.page.div(j)] : -1;
    }
  };
  look_up(0);
  int st = kind;
  uint32_t phase = 1;  // of the release before this use of a place: the first use waits for none
  int issued = 0;
  bool fine = true;    // after a wait that ran out a thread only keeps the others company at the barrier
#pragma unroll 1
  for (int t = 0; t < n; ++t) {
    const int j0 = (tiles.x + t) * kTcSlots;
    const bool seen = j0 >= u.lo_max && j0 + kTcSlots <= u.hi_min;  // whole, by every row that sees any
    int page[2], in[2];
    unsigned held[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      page[i] = checked_page(p.c, pg[i]);
      held[i] = __ballot_sync(0xffffffffu, page[i] >= 0);
      in[i] = j0 + gt + 64 * i - static_cast<int>(p.c.page.div(j0 + gt + 64 * i) * p.c.page.d);
    }
    look_up(t + 1);
    uint32_t whole;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
        "bar.red.and.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(whole)
        : "r"(static_cast<uint32_t>(seen && p.box > 0 && (held[0] & held[1]) == 0xffffffffu)), "r"(2 + kind)
        : "memory");
    if (fine && 2 * t >= S::kStages) fine = __all_sync(0xffffffffu, mbar_wait_short(&sh.empty[st], phase));
    // A tile's mask is read by steps that lag its S by two at most, and S of the tile kStages / 2 before
    // this one is done: 16 places are enough.
    if (kind == 0 && lane < 2) sh.mask[t & 15][gt / 32 + 2 * lane] = held[lane];
    __syncwarp();
    uint8_t* tile = ring + st * S::kTile;
    if (whole != 0) {
      if (fine) {
        // a warp announces half the bytes, whoever copies them
        if (lane == 0) mbar_arrive_expect_tx(&sh.full[st], S::kTile / 2);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = gt + 64 * i;
          if ((r & (p.box - 1)) != 0) continue;
#pragma unroll
          for (int x = 0; x < D / 64; ++x)
            tma_load_4d_tile(tile + x * S::kPanel + r * 128, map, &sh.full[st], 64 * x, in[i], u.hk, page[i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) off[gt + 64 * i] = page[i] < 0 ? -1 : page[i] * sp + in[i] * sr;
      asm volatile("bar.sync %0, 64;" ::"r"(2 + kind) : "memory");
      if (fine) {
#pragma unroll 8
        for (int i = 0; i < kTcSlots / RP; ++i) {
          const int r = gt / C + i * RP;
          const int64_t o = off[r];
          cp_async_16(tile + column + r * 128 + (((gt % C & 7) ^ (r & 7)) << 4), base + (o < 0 ? 0 : o),
                      o < 0 ? 0u : 16u);
        }
        cp_async_commit();
        cp_async_wait<0>();
        if (kind == 1 && !seen) {
#pragma unroll 1
          for (int i = 0; i < kTcSlots / RP; ++i)
            rows_tc_clean<T>(sh, tile + column, j0, gt / C + i * RP, gt % C);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.full[st]);
      }
    }
    issued += fine;
    st += 2;
    if (st >= S::kStages) {
      st -= S::kStages;
      phase ^= 1;
    }
  }
  // after a wait that ran out: what was issued before it must not be left on its way into shared memory
  for (int t = max(0, issued - S::kStages / 2); !fine && t < issued; ++t)
    mbar_wait_bounded(&sh.full[kind + 2 * (t % (S::kStages / 2))], (t / (S::kStages / 2)) & 1);
}

// The issuing warp of block x: one of its lanes issues.
template <typename T, int D, bool Twin, int Parts>
__device__ __forceinline__ void rows_tc_issue(RowsTcShared& sh, uint32_t q, uint32_t ring, int n, int x) {
  using S = RowsTc<D, Twin>;
  constexpr uint32_t kS = tc_instruction<T>(kTcSlots / 2, false), kO = tc_instruction<T>(D, true);
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
  const uint64_t q_desc = tc_descriptor(q + (Twin ? 0 : x * S::kTile), 16), k_desc = tc_descriptor(ring, 16),
                 v_desc = tc_descriptor(ring, S::kPanel);
  int k_stage = 0, v_stage = 1;                 // places of the K and V in use
  uint32_t k_phase = 0, v_phase = 0;
  auto next = [](int& stage, uint32_t& phase) {
    stage += 2;
    if (stage >= S::kStages) {
      stage -= S::kStages;
      phase ^= 1;
    }
  };
  auto wait = [](uint64_t* bar, uint32_t phase) {
    return __all_sync(0xffffffffu, mbar_wait_short(bar, phase));
  };
  bool fine = wait(&sh.q_full, 0);
  tc_fence_after();
  // S of a step, buffer b: with Twin this block's half of the next K tile, else half b of it
  auto scores = [&](int b) {
    const int h = Twin ? x : b;
    if (Twin || b == 0) fine = fine && wait(&sh.full[k_stage], k_phase);
    if (!fine) return;
    const uint64_t k0 = k_desc + k_stage * (S::kTile / 16) + h * 512;
    if (tc_elected()) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        constexpr int kStep = S::kPanel / 16;
        tc_mma(tmem + x * 128 + b * 64, q_desc + (k / 4) * kStep + (k % 4) * 2, k0 + (k / 4) * kStep + (k % 4) * 2,
               kS, k > 0);
      }
      tc_commit(&sh.s_full[x][b]);
      if (Twin || b == 1) tc_commit(&sh.empty[k_stage]);
    }
    if (Twin || b == 1) next(k_stage, k_phase);
  };
  const int steps = Twin ? n : 2 * n;
  scores(0);
  if (steps > 1) scores(1);
#pragma unroll 1
  for (int i = 0; fine && i < steps; i += 2) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (i + b >= steps) break;
      const int h = Twin ? x : b;
      if (Twin || b == 0) fine = wait(&sh.full[v_stage], v_phase);
      fine = fine && wait(&sh.p_full[x][b], (i >> 1) & 1);
      if (!fine) break;
      tc_fence_after();
      const uint64_t v = v_desc + v_stage * (S::kTile / 16) + h * 512;
      if (tc_elected()) {
#pragma unroll
        for (int part = 0; part < Parts; ++part)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tc_mma_ts(tmem + 256 + x * D, tmem + x * 128 + b * 64 + part * 32 + k * 8, v + k * 128, kO,
                      i > 0 || b > 0 || part > 0 || k > 0);
        tc_commit(&sh.o_done[x][b]);
        if (Twin || b == 1) tc_commit(&sh.empty[v_stage]);
      }
      if (Twin || b == 1) next(v_stage, v_phase);
      if (i + b + 2 < steps) scores(b);
    }
  }
  // nothing is left in flight when the tensor memory is freed
  if (tc_elected()) tc_commit(&sh.drained[x]);
  wait(&sh.drained[x], 0);
}

// The largest of 64 scores, by chains that do not wait for one another.
__device__ __forceinline__ float rows_max(const uint32_t (&s)[64]) {
  float m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = __uint_as_float(s[i]);
#pragma unroll
  for (int c = 4; c < 64; c += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m[i] = fmaxf(fmaxf(m[i], __uint_as_float(s[c + i])), c + 4 + i < 64 ? __uint_as_float(s[c + 4 + i]) : -INFINITY);
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// A softmax thread: row `r` of the CTA, of which it leaves base and sum in `state`. False: a wait ran
// out.
template <typename T, int D, bool Twin, int Parts>
__device__ __forceinline__ bool rows_tc_softmax(const RowsParams& p, RowsTcShared& sh, int2 tiles, float scale2,
                                                float2& state) {
  constexpr float kBelow = std::is_same<T, __half>::value ? 7.0f : 0.0f;
  const RowsUnit& u = sh.u;
  const int x = threadIdx.x / 128, r = threadIdx.x % 128 + (Twin ? 0 : x * 128);
  const uint32_t lane0 = static_cast<uint32_t>((threadIdx.x % 128) / 32 * 32) << 16;
  const uint32_t s_at = sh.tmem + lane0 + x * 128, o_at = sh.tmem + lane0 + 256 + x * D;
  const int2 lim = sh.limits[r];
  const bool idle = (r & ~31) >= u.rows;  // no row of this warp is one
  float& m = state.x;
  float& l = state.y;
  bool fine = true;
  const int steps = (Twin ? 1 : 2) * (tiles.y - tiles.x);
  auto wait_scores = [&](int i) {
    fine = __all_sync(0xffffffffu, mbar_wait_short(&sh.s_full[x][i & 1], (i >> 1) & 1));
    tc_fence_after();
  };
  // The product of half i is done. Its barrier is at that phase or the one before: the half after the
  // next one has not begun.
  auto wait_output = [&](int i) {
    fine = __all_sync(0xffffffffu, mbar_wait_short(&sh.o_done[x][i & 1], (i >> 1) & 1));
    tc_fence_after();
  };
#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    const int b = i & 1, tile = Twin ? i : i >> 1, h = Twin ? x : b;  // buffer; half of the tile
    const int j0 = (tiles.x + tile) * kTcSlots + h * 64;
    wait_scores(i);
    if (!fine) break;
    if (!idle) {
      uint32_t s[64], words[2];
      tc_load_start(s_at + b * 64, s);
      bool whole = j0 >= u.lo_max && j0 + 64 <= u.hi_min;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        words[w] = *reinterpret_cast<volatile uint32_t*>(&sh.mask[tile & 15][2 * h + w]);
        whole = whole && words[w] == 0xffffffffu;
      }
      tc_load_wait(s);
      if (!whole) {
#pragma unroll
        for (int w = 0; w < 2; ++w) words[w] &= rows_bits(lim.x - j0 - 32 * w, lim.y - j0 - 32 * w);
        rows_hide(s, words);
      }
      const float top = rows_max(s) * scale2;
      if (__any_sync(0xffffffffu, top > m + (8.0f + kBelow))) {
        const float mn = fmaxf(m, top - kBelow);
        const float f = m == -INFINITY ? 0.0f : rows_exp2(m - mn);
        m = mn;
        l *= f;
        if (i > 0) {
          wait_output(i - 1);
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += 32) {
            uint32_t o[32];
            tc_load(o_at + c0, o);
#pragma unroll
            for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
            tc_store(o_at + c0, o);
          }
        }
      }
      const float base = m == -INFINITY ? 0.0f : -m;
      // 64 weights in 16 bits, 2 a word; with Parts = 2 the remainders too
      float2 sum = make_float2(0.0f, 0.0f);
      uint32_t hi[32], lo[32];
#pragma unroll
      for (int c = 0; c < 64; c += 2) {
        const float2 z = ffma2(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])),
                               make_float2(scale2, scale2), make_float2(base, base));
        const float2 w = make_float2(rows_exp2(z.x), rows_exp2(z.y));
        sum = fadd2(sum, w);
        float ra, rb;
        hi[c / 2] = rows_pack<T>(w.x, w.y, ra, rb);
        if constexpr (Parts == 2) {
          float na, nb;
          lo[c / 2] = rows_pack<T>(ra, rb, na, nb);
        }
      }
      tc_store(s_at + b * 64, hi);
      if constexpr (Parts == 2) tc_store(s_at + b * 64 + 32, lo);
      l += sum.x + sum.y;
      tc_wait_stores();
      tc_fence_before();
    }
    mbar_arrive(&sh.p_full[x][b]);
  }
  if (fine) wait_output(steps - 1);
  return fine;
}

// Writes the rows. With Twin the blocks hold two parts of the same rows: the second lays its part out in
// shared memory, element by element of all rows, and the first joins them.
template <typename T, int D, bool Twin>
__device__ __forceinline__ void rows_tc_write(const RowsParams& p, RowsTcShared& sh, float* other, float2 state,
                                              bool fine) {
  const RowsUnit& u = sh.u;
  const int x = threadIdx.x / 128, lr = threadIdx.x % 128, r = lr + (Twin ? 0 : x * 128);
  const uint32_t o_at = sh.tmem + (static_cast<uint32_t>(lr / 32 * 32) << 16) + 256 + x * D;
  const bool works = fine && (r & ~31) < u.rows;  // alike for a warp
  float m = state.x, l = state.y, own = 1.0f, theirs = 0.0f;
  if constexpr (Twin) {
    asm volatile("bar.sync 1, 256;" ::: "memory");  // both blocks' products are done: the ring is free
    if (works && x == 1) {
      sh.part[lr] = state;
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t o[32];
        tc_load(o_at + c0, o);
#pragma unroll
        for (int c = 0; c < 32; ++c) other[(c0 + c) * 128 + lr] = __uint_as_float(o[c]);
      }
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (!works || x == 1) return;
    const float2 b = sh.part[lr];
    const float M = fmaxf(m, b.x);
    own = m == -INFINITY ? 0.0f : rows_exp2(m - M);
    theirs = b.x == -INFINITY ? 0.0f : rows_exp2(b.x - M);
    // a part without a slot (sum 0) counts for nothing; what else is there is finite, or NaN by right
    l = (l == 0.0f ? 0.0f : own * l) + (b.y == 0.0f ? 0.0f : theirs * b.y);
    m = M;
  } else if (!works) {
    return;
  }
  const bool in = r < u.rows;
  const int rr = in ? u.row0 + r : 0;
  const int t = static_cast<int>(p.of_G.div(rr)), g = rr - t * p.G;
  const int64_t row = static_cast<int64_t>(u.tok0 + t) * p.H + u.hk * p.G + g;
  const float nan = __int_as_float(0x7fffffff);
  const float spoil = in && sh.spoilt[r] ? nan : 1.0f;
  const bool parts = rows_in_parts(p, u);
  const int64_t part = in && parts ? rows_place<RowsTc<D, Twin>::kRows>(p, u, r, row) : 0;
  if (in && !parts && p.part_of != nullptr) p.part_of[row] = make_int2(0, 0);
  const float inv = parts ? spoil : l == 0.0f ? 0.0f : spoil / l;
#pragma unroll 1
  for (int c0 = 0; c0 < D; c0 += 32) {
    uint32_t o[32];
    __syncwarp();
    tc_load(o_at + c0, o);
    float f[32];
#pragma unroll
    for (int c = 0; c < 32; ++c) {
      f[c] = __uint_as_float(o[c]);
      if constexpr (Twin) f[c] = fmaf(theirs, other[(c0 + c) * 128 + lr], own * f[c]);
      f[c] = l == 0.0f ? 0.0f : f[c] * inv;
    }
    if (in && parts) {
      float4* dst = reinterpret_cast<float4*>(p.part_o + part * D + c0);
#pragma unroll
      for (int c = 0; c < 32; c += 4) dst[c / 4] = make_float4(f[c], f[c + 1], f[c + 2], f[c + 3]);
    } else if (in) {
      uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.o) + row * D + c0);
#pragma unroll
      for (int c = 0; c < 32; c += 8) {
        float ra, rb;
        uint32_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = rows_pack<T>(f[c + 2 * e], f[c + 2 * e + 1], ra, rb);
        dst[c / 8] = make_uint4(h[0], h[1], h[2], h[3]);
      }
    }
  }
  if (!in) return;
  if (parts) p.part_ml[part] = make_float2(m, l);
  else if (p.lse != nullptr) p.lse[row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <typename T, int D, bool Twin, int Parts>
__global__ void __launch_bounds__(RowsTc<D, Twin>::kThreads, 1) rows_tc_kernel(const RowsParams p, const __grid_constant__ RowsMaps maps) {
  using S = RowsTc<D, Twin>;
  extern __shared__ uint8_t rt_raw[];
  __shared__ RowsTcShared sh;
  uint8_t* q = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(rt_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = q + S::kQ;
  // A shared prefix's kernel is the third of its call and reads nothing that the first two write, so it
  // waits for them last of all (in every CTA: it must not end before them).
  const bool early = p.prefix != nullptr;
  if (!early) asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  auto wait_late = [&]() {
    if (early) asm volatile("griddepcontrol.wait;" ::: "memory");
  };
  if (!rows_begin<S::kRows>(p, sh.u, sh.limits)) {
    wait_late();
    return;
  }
  const RowsUnit& u = sh.u;
  const int2 tiles = rows_tiles<kTcSlots>(p, u);
  const int tid = threadIdx.x, n = tiles.y - tiles.x;
  if (n <= 0) {  // no row of this part sees a slot
    for (int r = tid; r < u.rows; r += S::kThreads) {
      const int t = static_cast<int>(p.of_G.div(u.row0 + r)), g = u.row0 + r - t * p.G;
      const int64_t row = static_cast<int64_t>(u.tok0 + t) * p.H + u.hk * p.G + g;
      if (rows_in_parts(p, u)) {
        p.part_ml[rows_place<S::kRows>(p, u, r, row)] = make_float2(-INFINITY, 0.0f);
        continue;
      }
      if (p.part_of != nullptr) p.part_of[row] = make_int2(0, 0);
      uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.o) + row * D);
      for (int c = 0; c < D / 8; ++c) dst[c] = make_uint4(0u, 0u, 0u, 0u);
      if (p.lse != nullptr) p.lse[row] = -INFINITY;
    }
    wait_late();
    return;
  }
  const int blocks = Twin || u.rows > 128 ? 2 : 1;
  // q on its way: a block's rows are brought in by its threads, with Twin half of them by each block's
  constexpr int C = D / 8, kQRows = Twin ? 64 : 128, kQSteps = kQRows * C / 128;
  auto q_row = [&](int i) { return (tid % 128 + i * 128) / C + tid / 128 * kQRows; };
  auto q_place = [&](int i) {
    const int r = q_row(i), ch = tid % C;
    return reinterpret_cast<uint4*>(q + r / 128 * S::kTile + (ch >> 3) * S::kPanel + r % 128 * 128 +
                                    (((ch & 7) ^ (r & 7)) << 4));
  };
  if (tid / 128 < blocks && tid < S::kLoad0) {
#pragma unroll
    for (int i = 0; i < kQSteps; ++i) {
      const bool in = q_row(i) < u.rows;
      const int rr = in ? u.row0 + q_row(i) : 0;
      const int t = static_cast<int>(p.of_G.div(rr)), g = rr - t * p.G;
      cp_async_16(q_place(i), static_cast<const T*>(p.q) + (u.tok0 + t) * p.qst + (u.hk * p.G + g) * p.qsh + tid % C * 8,
                  in ? 16u : 0u);
    }
    cp_async_commit();
  }
  if (tid == S::kMma) {
    mbar_init(&sh.q_full, blocks * 128);
    for (int x = 0; x < 2; ++x) {
      for (int h = 0; h < 2; ++h) {
        mbar_init(&sh.s_full[x][h], 1);
        mbar_init(&sh.p_full[x][h], 128);
        mbar_init(&sh.o_done[x][h], 1);
      }
      mbar_init(&sh.drained[x], 1);
    }
    for (int e = 0; e < S::kStages; ++e) {
      mbar_init(&sh.full[e], 2);
      mbar_init(&sh.empty[e], blocks);
    }
    fence_mbar_init();
  }
  if (tid < 256) sh.spoilt[tid] = 0;
  __syncwarp();
  if (tid / 32 == S::kMma / 32) tc_alloc(&sh.tmem, S::kColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // scores are scaled by |scale|: its sign goes into q, and for a scale of 0 q is 0
  const float scale2 = p.scale2 == 0.0f ? 1.0f : fabsf(p.scale2);
  if (tid < S::kLoad0) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kSoftmax));
    if (tid / 128 < blocks) {
      cp_async_wait<0>();
      if (p.scale2 <= 0.0f)
        for (int i = 0; i < kQSteps; ++i) {
          uint4* at = q_place(i);
          const uint32_t keep = p.scale2 < 0.0f ? 0xffffffffu : 0u, flip = keep & 0x80008000u;
          *at = make_uint4((at->x & keep) ^ flip, (at->y & keep) ^ flip, (at->z & keep) ^ flip, (at->w & keep) ^ flip);
        }
      fence_proxy_async_smem();
      mbar_arrive(&sh.q_full);
      // a row that sees nothing begins at a base that no score is above, so that it raises none of its warp's
      const int r = tid % 128 + (Twin ? 0 : tid / 128 * 128);
      const bool blind = r < u.rows && sh.limits[r].x >= sh.limits[r].y;
      float2 state = make_float2(blind ? INFINITY : -INFINITY, 0.0f);
      const bool fine = rows_tc_softmax<T, D, Twin, Parts>(p, sh, tiles, scale2, state);
      if (blind) state = make_float2(-INFINITY, 0.0f);
      rows_tc_write<T, D, Twin>(p, sh, reinterpret_cast<float*>(ring), state, fine);
    }
  } else if (tid < S::kMma) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kOthers));
    rows_tc_load<T, D, Twin>(p, maps, sh, ring, tiles);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kOthers));
    const int x = __shfl_sync(0xffffffffu, (tid - S::kMma) / 32, 0);
    if (x < blocks) rows_tc_issue<T, D, Twin, Parts>(sh, smem_u32(q), smem_u32(ring), n, x);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (tid / 32 == S::kMma / 32) tc_free(sh.tmem, S::kColumns);
  wait_late();
}

// Joins a row's parts: those of its CTAs, and with `own` (fp32 rows and (m, 1 / l)) that of its own slots.
// A warp takes a row; parts without a slot (l = 0) have no o.
constexpr int kRjWarps = 4;

template <typename T, int D>
__global__ void __launch_bounds__(kRjWarps * 32) rows_join_kernel(const RowsParams p, int stride,
                                                                  const float* own_o, const float2* own_ml) {
  constexpr int E = D / 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRjWarps + (threadIdx.x >> 5);
  const int64_t rows = static_cast<int64_t>(p.T) * p.H;
  if (row >= rows) return;
  const int t = static_cast<int>(row / p.H);
  const bool held = t >= p.starts[0] && t < p.starts[p.nseg];  // in some segment
  if (!held) {
    if (p.prefix == nullptr) return;  // nobody's token: left as it is
    if (lane == 0) raise_status(DCR_ERR_DEVICE_INDEX);
  }
  // lane x holds parts x and x + 32, then the own part's
  int2 of = held ? p.part_of[row] : make_int2(0, 0);
  if (of.x < 0 || of.y < 0 || of.y > kRowsMaxParts || of.x + (of.y - 1) * static_cast<int64_t>(stride) >= p.places)
    of.y = 0;  // starts out of order: a row that no CTA took
  if (of.y == 0 && p.prefix == nullptr) return;  // written already
  float2 ml[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int s = lane + 32 * i;
    ml[i] = s < of.y ? p.part_ml[of.x + static_cast<int64_t>(s) * stride] : make_float2(-INFINITY, 0.0f);
  }
  float2 own = make_float2(-INFINITY, 0.0f);
  if (own_ml != nullptr) {
    const float2 x = own_ml[row];
    if (x.y != 0.0f) own = make_float2(x.x, 1.0f / x.y);
  }
  float M = fmaxf(fmaxf(ml[0].x, ml[1].x), own.x);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  float w[2], L = 0.0f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    w[i] = ml[i].x == -INFINITY ? 0.0f : rows_exp2(ml[i].x - M);
    L += ml[i].y == 0.0f ? 0.0f : w[i] * ml[i].y;
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  float acc[E] = {};
  if (own.y != 0.0f) {
    const float a = rows_exp2(own.x - M) * own.y;
    L += a;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = a * own_o[row * D + lane + 32 * e];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    unsigned left = __ballot_sync(0xffffffffu, ml[i].y != 0.0f);
    while (left != 0) {
      const int s = __ffs(left) - 1;
      left &= left - 1;
      const float a = __shfl_sync(0xffffffffu, w[i], s);
      const float* src = p.part_o + (of.x + static_cast<int64_t>(s + 32 * i) * stride) * D;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(a, src[lane + 32 * e], acc[e]);
    }
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
  for (int e = 0; e < E; ++e) ElemTraits<T>::store(static_cast<T*>(p.o) + row * D, lane + 32 * e, acc[e] * inv);
  if (lane == 0 && p.lse != nullptr) p.lse[row] = L == 0.0f ? -INFINITY : (M + log2f(L)) * kLn2;
}

// How a call is cut: query rows a CTA, CTAs that units are cut up for (0: a CTA a unit), CTAs.
struct RowsPlan {
  int bm, pieces;
  int64_t units, ctas;
};

static RowsPlan rows_plan(int dtype, int T, int nseg, int H_kv, int G, bool shared) {
  RowsPlan r;
  const int64_t rows = static_cast<int64_t>(T) * G;
  const bool tc = dtype != DCR_DTYPE_F32;
  // two blocks of rows where segments have more than one on average
  r.bm = !tc ? kRfRows : rows > 128ll * nseg ? 256 : 128;
  // every segment adds one tile of rows at most that is not full
  const int64_t units = (rows / r.bm + (nseg < rows ? nseg : rows)) * H_kv;
  // Units are cut up where the grid has more than one CTA for each; fp32 ones, whose longest would set the
  // pace (a tile takes 4 us), up to 4 CTAs an SM. A 16-bit prompt's where it has two: with fewer most units
  // stay whole, and the call pays for parts and join (10 to 16 sequences on 16000 slots, 8 KV heads of 64: 124 us
  // whole, 129 cut; on 2000 slots 23 and 27; 9 sequences, whose units are counted as 80 and are 72, would
  // gain: 125 whole, 75 cut).
  const int64_t slots = static_cast<int64_t>(tc ? 1 : 4) * device_sm_count();
  r.pieces = units <= slots && (shared || !tc || 2 * units <= slots) ? static_cast<int>(slots) : 0;
  r.units = units;
  r.ctas = r.pieces > 0 ? r.pieces : units;
  return r;
}

// Workspace sections.
struct RowsLayout {
  size_t o, ml, of, own_o, own_ml, attend, total;
  int64_t places;
};

static RowsLayout rows_layout(const RowsPlan& r, int T, int H, int D, size_t attend, bool shared) {
  RowsLayout w;
  size_t off = 0;
  auto take = [&](size_t n) {
    const size_t at = off;
    off = (off + n + 255) / 256 * 256;
    return at;
  };
  const size_t rows = static_cast<size_t>(T) * H;
  w.places = r.pieces > 0 ? static_cast<int64_t>(r.pieces) * r.bm : shared ? static_cast<int64_t>(rows) : 0;
  w.o = take(w.places * D * sizeof(float));
  w.ml = take(w.places * sizeof(float2));
  w.of = take(w.places > 0 ? rows * sizeof(int2) : 0);
  w.own_o = take(shared ? rows * D * sizeof(float) : 0);
  w.own_ml = take(shared ? rows * sizeof(float2) : 0);
  w.attend = take(attend);
  w.total = off > 256 ? off : 256;
  return w;
}

// The parts' fields of the parameters.
static void rows_set_parts(RowsParams& p, const RowsPlan& plan, const RowsLayout& w, uint8_t* ws) {
  const bool parts = w.places > 0;
  p.pieces = plan.pieces;
  p.places = w.places;
  p.part_o = parts ? reinterpret_cast<float*>(ws + w.o) : nullptr;
  p.part_ml = parts ? reinterpret_cast<float2*>(ws + w.ml) : nullptr;
  p.part_of = parts ? reinterpret_cast<int2*>(ws + w.of) : nullptr;
  p.box = 0;
}

template <typename Kernel, typename... Args>
static int rows_launch_as(Kernel kernel, int threads, int smem, const RowsPlan& plan, cudaStream_t s,
                          const Args&... args) {
  if (ensure_smem_attr(reinterpret_cast<const void*>(kernel), smem) != cudaSuccess) return DCR_ERR_CUDA;
  return launch_dependent(kernel, dim3(static_cast<unsigned>(plan.ctas)), dim3(threads), smem, s, 1, args...) ==
                 cudaSuccess
             ? DCR_OK
             : DCR_ERR_CUDA;
}

// The pool as tensor maps of boxes of `box` slots; false where its strides are none that a map takes.
template <typename T>
static bool rows_map(CUtensorMap* map, const PagePool& c, const void* base, int64_t sp, int64_t sh,
                     int64_t sr, int H_kv, int D, int box) {
  EncodeTiledFn encode = get_encode_fn();
  if (!encode) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), c.page.d, static_cast<cuuint64_t>(H_kv),
                              static_cast<cuuint64_t>(c.num_pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(sr) * 2, static_cast<cuuint64_t>(sh) * 2,
                                 static_cast<cuuint64_t>(sp) * 2};
  const cuuint32_t size[4] = {64u, static_cast<cuuint32_t>(box), 1u, 1u}, step[4] = {1u, 1u, 1u, 1u};
  return encode(map, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                4, const_cast<void*>(base), dims, strides, size, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, int Parts>
static int rows_launch(const RowsParams& params, const RowsPlan& plan, cudaStream_t s) {
  if constexpr (sizeof(T) == 4) {
    return rows_launch_as(rows_fma_kernel<D>, kRfThreads, RowsFma<D>::kSmem, plan, s, params);
  } else {
    RowsParams p = params;
    RowsMaps maps = {};
    // the largest power of two that divides a page, at most a tile; 8 slots are a swizzle's period
    int box = static_cast<int>(p.c.page.d & (~p.c.page.d + 1));
    if (box > kTcSlots) box = kTcSlots;
    p.box = box >= 8 && rows_map<T>(&maps.k, p.c, p.c.k, p.c.ksp, p.c.ksh, p.c.ksr, p.H_kv, D, box) &&
                    rows_map<T>(&maps.v, p.c, p.c.v, p.c.vsp, p.c.vsh, p.c.vsr, p.H_kv, D, box)
                ? box
                : 0;
    if (plan.bm == 256)
      return rows_launch_as(rows_tc_kernel<T, D, false, Parts>, RowsTc<D, false>::kThreads,
                            RowsTc<D, false>::kSmem, plan, s, p, maps);
    return rows_launch_as(rows_tc_kernel<T, D, true, Parts>, RowsTc<D, true>::kThreads, RowsTc<D, true>::kSmem,
                          plan, s, p, maps);
  }
}

template <typename T, int D>
static int rows_join(const RowsParams& p, const RowsPlan& plan, const float* own_o, const float2* own_ml, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(p.T) * p.H;
  return launch_dependent(rows_join_kernel<T, D>, dim3(static_cast<unsigned>((rows + kRjWarps - 1) / kRjWarps)),
                          dim3(kRjWarps * 32), 0, s, 1, p, plan.bm, own_o, own_ml) == cudaSuccess
             ? DCR_OK
             : DCR_ERR_CUDA;
}

// f(T of the dtype, D as a constant)
template <typename F>
static int rows_dispatch(int dtype, int D, F&& f) {
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  switch (dtype) {
    case DCR_DTYPE_BF16: return D == 64 ? f(__nv_bfloat16(), D64()) : f(__nv_bfloat16(), D128());
    case DCR_DTYPE_F16: return D == 64 ? f(__half(), D64()) : f(__half(), D128());
    default: return D == 64 ? f(0.0f, D64()) : f(0.0f, D128());
  }
}

// What both entry points check of their shapes.
static int rows_check(int T, int H, int H_kv, int window) {
  if (T <= 0 || H <= 0 || H_kv <= 0 || H % H_kv != 0 || window < 0) return DCR_ERR_SHAPE;
  if (static_cast<int64_t>(T) * H > 0x40000000ll) return DCR_ERR_SHAPE;
  return DCR_OK;
}

static int rows_check_rows(const void* q, int64_t qst, int64_t qsh, const void* o, const void* lse,
                           const void* a, const void* b, const void* c, int dtype, int T, int H, int D) {
  const int64_t per16 = dtype == DCR_DTYPE_F32 ? 4 : 8;
  if (misaligned(16, q, o) || misaligned(4, lse, a, b, c) || qst % per16 || qsh % per16)
    return DCR_ERR_ALIGN;
  if (qst < 0 || qsh < 0) return DCR_ERR_SHAPE;
  return rows_meet(q, qst, qsh, o, T, H, D, 16 / per16) ? DCR_ERR_SHAPE : DCR_OK;
}

}  // namespace dcr

using namespace dcr;

extern "C" {

size_t dcr_paged_prefill_workspace_bytes(int dtype, int T, int B, int H, int H_kv, int D) {
  if (B <= 0 || (D != 64 && D != 128) || rows_check(T, H, H_kv, 0) != DCR_OK)
    return 0;
  return rows_layout(rows_plan(dtype, T, B, H_kv, H / H_kv, false), T, H, D, 0, false).total;
}

int dcr_paged_prefill(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_pages,
                      const void* v_pages, int dtype, int64_t k_stride_p, int64_t k_stride_h,
                      int64_t k_stride_s, int64_t v_stride_p, int64_t v_stride_h,
                      int64_t v_stride_s, int num_pages, int page_size, const int32_t* page_table,
                      int64_t table_stride, int max_pages, const int32_t* lengths,
                      const int32_t* starts, int T, int B, int H, int H_kv, int D, float scale,
                      int window, int causal, void* o, float* lse, void* workspace,
                      size_t workspace_bytes, void* stream) {
  if (q == nullptr || lengths == nullptr || starts == nullptr || o == nullptr) return DCR_ERR_NULL;
  if (B <= 0 || (window > 0 && !causal)) return DCR_ERR_SHAPE;
  int st = rows_check(T, H, H_kv, window);
  if (st != DCR_OK) return st;
  st = check_pool(k_pages, v_pages, dtype, k_stride_p, k_stride_h, k_stride_s, v_stride_p,
                  v_stride_h, v_stride_s, num_pages, page_size, page_table, table_stride, max_pages,
                  H_kv, D);
  if (st != DCR_OK) return st;
  st = rows_check_rows(q, q_stride_t, q_stride_h, o, lse, lengths, starts, nullptr, dtype, T, H, D);
  if (st != DCR_OK) return st;
  RowsPlan plan = rows_plan(dtype, T, B, H_kv, H / H_kv, false);
  if (max_pages * page_size <= 128 * kRowsMinPart) {  // nothing to cut up
    plan.pieces = 0;
    plan.ctas = plan.units;
  }
  if (plan.ctas > INT32_MAX) return DCR_ERR_SHAPE;
  const RowsLayout w = rows_layout(plan, T, H, D, 0, false);
  if (workspace == nullptr || misaligned(16, workspace) || workspace_bytes < w.total)
    return DCR_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  RowsParams p;
  p.c = make_pool(k_pages, v_pages, k_stride_p, k_stride_h, k_stride_s, v_stride_p, v_stride_h,
                  v_stride_s, num_pages, page_size, page_table, table_stride, max_pages);
  p.q = q;
  p.qst = q_stride_t;
  p.qsh = q_stride_h;
  p.lengths = lengths;
  p.starts = starts;
  p.prefix = nullptr;
  p.T = T;
  p.nseg = B;
  p.H = H;
  p.H_kv = H_kv;
  p.G = H / H_kv;
  p.of_G = FastDiv::make(static_cast<uint32_t>(p.G));
  p.window = window;
  p.causal = causal != 0;
  p.scale2 = scale * kLog2e;
  p.o = o;
  p.lse = lse;
  rows_set_parts(p, plan, w, ws);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return rows_dispatch(dtype, D, [&](auto type, auto dims) {
    using Ty = decltype(type);
    constexpr int kDim = decltype(dims)::value;
    const int rc = rows_launch<Ty, kDim, 1>(p, plan, s);
    return rc != DCR_OK || plan.pieces == 0 ? rc : rows_join<Ty, kDim>(p, plan, nullptr, nullptr, s);
  });
}

size_t dcr_paged_shared_workspace_bytes(int dtype, int B, int groups, int H, int H_kv, int D) {
  if (groups <= 0 || (D != 64 && D != 128) || rows_check(B, H, H_kv, 0) != DCR_OK)
    return 0;
  return rows_layout(rows_plan(dtype, B, groups, H_kv, H / H_kv, true), B, H, D,
                     pa_layout(B, H, H / H_kv, D, 1, false).total, true).total;
}

int dcr_paged_shared_attend(const void* q, int64_t q_stride_b, int64_t q_stride_h,
                            const void* k_pages, const void* v_pages, int dtype, int64_t k_stride_p,
                            int64_t k_stride_h, int64_t k_stride_s, int64_t v_stride_p,
                            int64_t v_stride_h, int64_t v_stride_s, int num_pages, int page_size,
                            const int32_t* page_table, int64_t table_stride, int max_pages,
                            const int32_t* lengths, const int32_t* groups, int n_groups,
                            const int32_t* prefix, int B, int H, int H_kv, int D, float scale,
                            int window, void* o, float* lse, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (q == nullptr || lengths == nullptr || groups == nullptr || prefix == nullptr || o == nullptr)
    return DCR_ERR_NULL;
  if (n_groups <= 0) return DCR_ERR_SHAPE;
  int st = rows_check(B, H, H_kv, window);
  if (st != DCR_OK) return st;
  st = check_pool(k_pages, v_pages, dtype, k_stride_p, k_stride_h, k_stride_s, v_stride_p,
                  v_stride_h, v_stride_s, num_pages, page_size, page_table, table_stride, max_pages,
                  H_kv, D);
  if (st != DCR_OK) return st;
  st = rows_check_rows(q, q_stride_b, q_stride_h, o, lse, lengths, groups, prefix, dtype, B, H, D);
  if (st != DCR_OK) return st;
  const int G = H / H_kv;
  const RowsPlan plan = rows_plan(dtype, B, n_groups, H_kv, G, true);
  if (plan.ctas > INT32_MAX) return DCR_ERR_SHAPE;
  const PagedAttendLayout a = pa_layout(B, H, G, D, 1, false);
  const RowsLayout w = rows_layout(plan, B, H, D, a.total, true);
  if (workspace == nullptr || misaligned(16, workspace) || workspace_bytes < w.total)
    return DCR_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int HB = pa_head_block(G, D, dtype);
  PagedAttendParams own;
  own.c = make_pool(k_pages, v_pages, k_stride_p, k_stride_h, k_stride_s, v_stride_p, v_stride_h,
                    v_stride_s, num_pages, page_size, page_table, table_stride, max_pages);
  own.q = q;
  own.qsb = q_stride_b;
  own.qsh = q_stride_h;
  own.lengths = lengths;
  own.prefix = prefix;
  own.B = B;
  own.H = H;
  own.H_kv = H_kv;
  own.G = G;
  own.hblocks = (G + HB - 1) / HB;
  own.units = H_kv * own.hblocks;
  own.scale2 = scale * kLog2e;
  own.window = window;
  own.page16 = 0;
  own.o = ws + w.own_o;
  own.lse = nullptr;
  own.stats = reinterpret_cast<float2*>(ws + w.own_ml);
  own.part = reinterpret_cast<float*>(ws + w.attend + a.part);
  own.scores = nullptr;
  own.s_stride = 0;
  RowsParams p;
  p.c = own.c;
  p.q = q;
  p.qst = q_stride_b;
  p.qsh = q_stride_h;
  p.lengths = lengths;
  p.starts = groups;
  p.prefix = prefix;
  p.T = B;
  p.nseg = n_groups;
  p.H = H;
  p.H_kv = H_kv;
  p.G = G;
  p.of_G = FastDiv::make(static_cast<uint32_t>(G));
  p.window = window;
  p.causal = 0;
  p.scale2 = own.scale2;
  p.o = o;
  p.lse = lse;
  rows_set_parts(p, plan, w, ws);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = pa_launch_any<true>(own, dtype, D, HB, a.ctas, s);
  if (rc != DCR_OK) return rc;
  return rows_dispatch(dtype, D, [&](auto type, auto dims) {
    using Ty = decltype(type);
    constexpr int kDim = decltype(dims)::value;
    const int r = rows_launch<Ty, kDim, 2>(p, plan, s);
    return r != DCR_OK ? r
                       : rows_join<Ty, kDim>(p, plan, reinterpret_cast<const float*>(ws + w.own_o),
                                             reinterpret_cast<const float2*>(ws + w.own_ml), s);
  });
}

}  // extern "C"
