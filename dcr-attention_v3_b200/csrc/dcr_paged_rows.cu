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
#include <math.h>

#include <type_traits>

#include "dcr_internal.h"
#include "dcr_paged.cuh"

namespace dcr {

struct RowsParams {
  PagePool c;
  const void* q;
  int64_t qst, qsh;
  const int32_t* lengths;  // of the sequences (prefill: segments; shared: tokens)
  const int32_t* starts;   // [nseg + 1] tokens of each segment
  const int32_t* prefix;   // shared: [T]; prefill: null
  int T, nseg, H, H_kv, G;
  int splits;              // parts that a segment's slots are cut into
  int window, causal;
  float scale2;            // scale * log2(e)
  void* o;                 // [T][H][D]
  float* lse;              // [T][H] natural log, or null
  float* part_o;           // [splits][T][H][D], or null: o and lse are written at once
  float2* part_ml;         // [splits][T][H] base of the exponents and sum
};

// A CTA's rows: BM of a segment's, for one KV head.
struct RowsUnit {
  int seg, tok0, ntok, len;  // the segment, its tokens; prefill: its sequence's length
  int hk, split;
  int row0, rows;            // first row in the segment and their number (0: nothing to do)
  int lo_min, lo_max, hi_min, hi_max;  // over the rows
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
  const int i = (u.row0 + r) / p.G;
  if (p.prefix != nullptr) {
    const int len = checked_length(p.c, p.lengths[u.tok0 + i]);
    return make_int2(p.window > 0 ? max(0, len - p.window) : 0, min(len, p.prefix[u.tok0 + i]));
  }
  const int x = u.len - u.ntok + i;
  return make_int2(p.window > 0 ? max(0, x + 1 - p.window) : 0, p.causal ? x + 1 : u.len);
}

// Finds this CTA's rows (blockIdx.x = (tile * H_kv + head) * splits + split, tiles from the last to
// the first, since a causal segment's last rows see most) and their limits. False: none.
template <int BM>
__device__ __forceinline__ bool rows_begin(const RowsParams& p, RowsUnit& u, int2* limits) {
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    const int rest = blockIdx.x / p.splits;
    const int tile = rest / p.H_kv;
    const int per = (p.nseg + 31) >> 5;
    int mine = 0;
    for (int j = 0; j < per; ++j) {
      const int s = lane * per + j;
      int tok0, ntok;
      if (s < p.nseg) {
        rows_segment(p, s, tok0, ntok);
        mine += (ntok * p.G + BM - 1) / BM;
      }
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    const int want = __shfl_sync(0xffffffffu, upto, 31) - 1 - tile;
    if (lane == 0) u.rows = 0;
    __syncwarp();
    int before = upto - mine;
    if (want >= before && want < upto) {
      for (int s = lane * per;; ++s) {
        int tok0, ntok;
        rows_segment(p, s, tok0, ntok);
        const int n = (ntok * p.G + BM - 1) / BM;
        if (want >= before + n) {
          before += n;
          continue;
        }
        u.seg = s;
        u.tok0 = tok0;
        u.ntok = ntok;
        u.len = p.prefix == nullptr ? checked_length(p.c, p.lengths[s]) : 0;
        u.hk = rest - tile * p.H_kv;
        u.split = blockIdx.x - rest * p.splits;
        u.row0 = (want - before) * BM;
        u.rows = min(BM, ntok * p.G - u.row0);
        u.lo_min = u.hi_min = INT32_MAX;
        u.lo_max = u.hi_max = 0;
        break;
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
    const bool sees = in && x.x < x.y;  // else it widens nothing, but no tile is seen whole
    const int a = __reduce_min_sync(0xffffffffu, sees ? x.x : INT32_MAX);
    const int b = __reduce_max_sync(0xffffffffu, in ? x.x : 0);
    const int c = __reduce_min_sync(0xffffffffu, in ? x.y : INT32_MAX);
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
  return make_int2(a + static_cast<int>(static_cast<int64_t>(n) * u.split / p.splits),
                   a + static_cast<int>(static_cast<int64_t>(n) * (u.split + 1) / p.splits));
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
// fp32 rows: 64 query rows against tiles of 64 slots with fp32 FMAs, 256 threads of 4 x 4 scores
// and 4 x D / 16 output elements each. Q and K lie transposed in shared memory, so a step of the
// inner loop reads four neighbouring rows and four neighbouring slots in two 16-byte reads for
// 8 packed FMAs.
// ---------------------------------------------------------------------------------------
constexpr int kRfRows = 64, kRfSlots = 64, kRfThreads = 256;

template <int D>
struct RowsFma {
  static constexpr int kPad = 4;
  static constexpr int W = kRfRows + kPad;
  static constexpr int kQ = D * W * 4, kK = D * W * 4, kV = kRfSlots * D * 4, kP = kRfSlots * W * 4;
  static constexpr int kSmem = kQ + kK + kV + kP;
};

template <typename T, int D>
__global__ void __launch_bounds__(kRfThreads) rows_fma_kernel(const RowsParams p) {
  using S = RowsFma<D>;
  constexpr int W = S::W, N = ElemTraits<T>::kPerChunk, C = D / N;
  constexpr int E = D / 64;  // groups of 4 output dims a thread
  extern __shared__ __align__(16) float rf_smem[];
  __shared__ RowsUnit u;
  __shared__ int2 limits[kRfRows];
  __shared__ int64_t koff[kRfSlots], voff[kRfSlots];
  __shared__ int flag[kRfSlots];  // 1: mapped; 2: V not finite
  __shared__ int bad;
  float* qt = rf_smem;
  float* kt = qt + D * W;
  float* vs = kt + D * W;
  float* pt = vs + kRfSlots * D;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  if (!rows_begin<kRfRows>(p, u, limits)) return;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int i = threadIdx.x; i < kRfRows * C; i += kRfThreads) {
    const int r = i / C, ch = i - r * C;
    float f[N] = {};
    if (r < u.rows) {
      const int t = (u.row0 + r) / p.G, g = u.row0 + r - t * p.G;
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) +
                                                        (u.tok0 + t) * p.qst + (u.hk * p.G + g) * p.qsh);
      ElemTraits<T>::widen(src[ch], f);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) qt[(ch * N + e) * W + r] = f[e];
  }
  float2 o[4][2 * E] = {};
  float m[4], l[4];
  bool poison[4] = {};
  int2 lim[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.0f;
    lim[i] = limits[4 * ty + i];
  }
  const int2 tiles = rows_tiles<kRfSlots>(p, u);
#pragma unroll 1
  for (int t = tiles.x; t < tiles.y; ++t) {
    const int j0 = t * kRfSlots;
    const bool whole = j0 >= u.lo_max && j0 + kRfSlots <= u.hi_min;
    __syncthreads();
    if (threadIdx.x < kRfSlots)
      flag[threadIdx.x] = rows_slot(p, u, j0 + threadIdx.x, koff[threadIdx.x], voff[threadIdx.x]);
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < kRfSlots * C; i += kRfThreads) {
      const int j = i / C, ch = i - j * C;
      float f[N] = {}, x[N] = {};
      if (flag[j] & 1) {
        ElemTraits<T>::widen(reinterpret_cast<const uint4*>(static_cast<const T*>(p.c.k) + koff[j])[ch], f);
        ElemTraits<T>::widen(reinterpret_cast<const uint4*>(static_cast<const T*>(p.c.v) + voff[j])[ch], x);
        if (!whole) {
          bool fine = true;
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (!rows_finite(x[e])) {
              fine = false;
              x[e] = 0.0f;
            }
          if (!fine) {
            atomicOr(&flag[j], 2);
            bad = 1;
          }
        }
      }
#pragma unroll
      for (int e = 0; e < N; ++e) kt[(ch * N + e) * W + j] = f[e];
#pragma unroll
      for (int e = 0; e < N; e += 4)
        *reinterpret_cast<float4*>(vs + j * D + ch * N + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
    }
    __syncthreads();
    float2 s[4][2] = {};  // [row][slot pair]
#pragma unroll 8
    for (int d = 0; d < D; ++d) {
      const float4 a = *reinterpret_cast<const float4*>(qt + d * W + 4 * ty);
      const float4 b = *reinterpret_cast<const float4*>(kt + d * W + 4 * tx);
      const float q[4] = {a.x, a.y, a.z, a.w};
      const float2 k[2] = {make_float2(b.x, b.y), make_float2(b.z, b.w)};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) s[i][e] = ffma2(make_float2(q[i], q[i]), k[e], s[i][e]);
    }
    int seen = 0, spoilt = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      seen |= (flag[4 * tx + e] & 1) << e;
      spoilt |= (flag[4 * tx + e] >> 1) << e;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float z[4] = {s[i][0].x, s[i][0].y, s[i][1].x, s[i][1].y};
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = j0 + 4 * tx + e;
        const bool in = ((seen >> e) & 1) && j >= lim[i].x && j < lim[i].y;
        z[e] = in ? z[e] * p.scale2 : -INFINITY;
        if (in && ((spoilt >> e) & 1)) poison[i] = true;
        top = fmaxf(top, z[e]);
      }
#pragma unroll
      for (int x = 8; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float mn = fmaxf(m[i], top);
      const float a = m[i] == -INFINITY ? 0.0f : rows_exp2(m[i] - mn);
      const float base = mn == -INFINITY ? 0.0f : mn;
      m[i] = mn;
      l[i] *= a;
#pragma unroll
      for (int e = 0; e < 2 * E; ++e) o[i][e] = make_float2(o[i][e].x * a, o[i][e].y * a);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float w = rows_exp2(z[e] - base);
        l[i] += w;
        pt[(4 * tx + e) * W + 4 * ty + i] = w;
      }
    }
    __syncthreads();
#pragma unroll 4
    for (int j = 0; j < kRfSlots; ++j) {
      const float4 a = *reinterpret_cast<const float4*>(pt + j * W + 4 * ty);
      const float w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int x = 0; x < E; ++x) {
        const float4 b = *reinterpret_cast<const float4*>(vs + j * D + 64 * x + 4 * tx);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[i][2 * x] = ffma2(make_float2(w[i], w[i]), make_float2(b.x, b.y), o[i][2 * x]);
          o[i][2 * x + 1] = ffma2(make_float2(w[i], w[i]), make_float2(b.z, b.w), o[i][2 * x + 1]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int spoilt = poison[i];
#pragma unroll
    for (int x = 8; x >= 1; x >>= 1) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
      spoilt |= __shfl_xor_sync(0xffffffffu, spoilt, x);
    }
    const int r = 4 * ty + i;
    if (r >= u.rows) continue;
    const int t = (u.row0 + r) / p.G, g = u.row0 + r - t * p.G;
    const int64_t row = static_cast<int64_t>(u.tok0 + t) * p.H + u.hk * p.G + g;
    const float nan = __int_as_float(0x7fffffff);
    if (p.part_o != nullptr) {
      const int64_t at = u.split * (static_cast<int64_t>(p.T) * p.H) + row;
      if (tx == 0) p.part_ml[at] = make_float2(m[i], l[i]);
      if (l[i] == 0.0f) continue;  // not read
#pragma unroll
      for (int x = 0; x < E; ++x)
        *reinterpret_cast<float4*>(p.part_o + at * D + 64 * x + 4 * tx) =
            spoilt ? make_float4(nan, nan, nan, nan)
                   : make_float4(o[i][2 * x].x, o[i][2 * x].y, o[i][2 * x + 1].x, o[i][2 * x + 1].y);
      continue;
    }
    const float inv = l[i] == 0.0f ? 0.0f : spoilt ? nan : 1.0f / l[i];
    T* dst = static_cast<T*>(p.o) + row * D;
#pragma unroll
    for (int x = 0; x < E; ++x) {
      const int d = 64 * x + 4 * tx;
      ElemTraits<T>::store(dst, d, o[i][2 * x].x * inv);
      ElemTraits<T>::store(dst, d + 1, o[i][2 * x].y * inv);
      ElemTraits<T>::store(dst, d + 2, o[i][2 * x + 1].x * inv);
      ElemTraits<T>::store(dst, d + 3, o[i][2 * x + 1].y * inv);
    }
    if (tx == 0 && p.lse != nullptr)
      p.lse[row] = l[i] == 0.0f ? -INFINITY : (m[i] + log2f(l[i])) * kLn2;
  }
}

// Joins a row's parts: those of its splits, and with `own` (fp32 rows and (m, 1 / l)) that of its own
// slots. A warp takes a row; parts without a slot (l = 0) have no o.
constexpr int kRowsMaxSplits = 64;
constexpr int kRjWarps = 4;

template <typename T, int D>
__global__ void __launch_bounds__(kRjWarps * 32) rows_join_kernel(const RowsParams p, const float* own_o,
                                                                  const float2* own_ml) {
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
  float2 ml[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int s = lane + 32 * i;
    ml[i] = held && s < p.splits ? p.part_ml[s * rows + row] : make_float2(-INFINITY, 0.0f);
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
      const float* src = p.part_o + ((s + 32 * i) * rows + row) * D;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(a, src[lane + 32 * e], acc[e]);
    }
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
  for (int e = 0; e < E; ++e) ElemTraits<T>::store(static_cast<T*>(p.o) + row * D, lane + 32 * e, acc[e] * inv);
  if (lane == 0 && p.lse != nullptr) p.lse[row] = L == 0.0f ? -INFINITY : (M + log2f(L)) * kLn2;
}

// How a call is cut: rows a CTA, parts a segment's slots are cut into, CTAs.
struct RowsPlan {
  int bm, splits;
  int64_t ctas;
};

static RowsPlan rows_plan(int T, int nseg, int H_kv, int G, int max_slots, int window) {
  RowsPlan r;
  r.bm = kRfRows;
  const int64_t rows = static_cast<int64_t>(T) * G;
  // every segment adds one tile at most that is not full
  const int64_t tiles = rows / r.bm + (nseg < rows ? nseg : rows);
  int64_t slots = max_slots;
  if (window > 0 && static_cast<int64_t>(window) + T < slots) slots = static_cast<int64_t>(window) + T;
  const int64_t most = slots / (4 * kRfSlots) > 1 ? slots / (4 * kRfSlots) : 1;
  int64_t want = (4ll * device_sm_count() + tiles * H_kv - 1) / (tiles * H_kv);
  if (want > most) want = most;
  if (want > kRowsMaxSplits) want = kRowsMaxSplits;
  r.splits = static_cast<int>(want);
  r.ctas = tiles * H_kv * r.splits;
  return r;
}

// Workspace sections.
struct RowsLayout {
  size_t o, ml, own_o, own_ml, attend, total;
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
  const size_t parts = shared || r.splits > 1 ? r.splits : 0;
  w.o = take(parts * rows * D * sizeof(float));
  w.ml = take(parts * rows * sizeof(float2));
  w.own_o = take(shared ? rows * D * sizeof(float) : 0);
  w.own_ml = take(shared ? rows * sizeof(float2) : 0);
  w.attend = take(attend);
  w.total = off > 256 ? off : 256;
  return w;
}

template <typename T, int D>
static int rows_launch(const RowsParams& p, const RowsPlan& plan, cudaStream_t s) {
  auto kernel = rows_fma_kernel<T, D>;
  if (ensure_smem_attr(reinterpret_cast<const void*>(kernel), RowsFma<D>::kSmem) != cudaSuccess)
    return DCR_ERR_CUDA;
  return launch_dependent(kernel, dim3(static_cast<unsigned>(plan.ctas)), dim3(kRfThreads),
                          RowsFma<D>::kSmem, s, 1, p) == cudaSuccess
             ? DCR_OK
             : DCR_ERR_CUDA;
}

template <typename T, int D>
static int rows_join(const RowsParams& p, const float* own_o, const float2* own_ml, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(p.T) * p.H;
  return launch_dependent(rows_join_kernel<T, D>, dim3(static_cast<unsigned>((rows + kRjWarps - 1) / kRjWarps)),
                          dim3(kRjWarps * 32), 0, s, 1, p, own_o, own_ml) == cudaSuccess
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

size_t dcr_paged_prefill_workspace_bytes(int T, int B, int H, int H_kv, int D, int max_slots, int window) {
  if (B <= 0 || max_slots <= 0 || (D != 64 && D != 128) || rows_check(T, H, H_kv, window) != DCR_OK)
    return 0;
  return rows_layout(rows_plan(T, B, H_kv, H / H_kv, max_slots, window), T, H, D, 0, false).total;
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
  const RowsPlan plan = rows_plan(T, B, H_kv, H / H_kv, max_pages * page_size, window);
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
  p.splits = plan.splits;
  p.window = window;
  p.causal = causal != 0;
  p.scale2 = scale * kLog2e;
  p.o = o;
  p.lse = lse;
  p.part_o = plan.splits > 1 ? reinterpret_cast<float*>(ws + w.o) : nullptr;
  p.part_ml = plan.splits > 1 ? reinterpret_cast<float2*>(ws + w.ml) : nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return rows_dispatch(dtype, D, [&](auto type, auto dims) {
    using Ty = decltype(type);
    constexpr int kDim = decltype(dims)::value;
    const int rc = rows_launch<Ty, kDim>(p, plan, s);
    return rc != DCR_OK || plan.splits == 1 ? rc : rows_join<Ty, kDim>(p, nullptr, nullptr, s);
  });
}

size_t dcr_paged_shared_workspace_bytes(int B, int groups, int H, int H_kv, int D, int max_slots) {
  if (groups <= 0 || max_slots <= 0 || (D != 64 && D != 128) || rows_check(B, H, H_kv, 0) != DCR_OK)
    return 0;
  return rows_layout(rows_plan(B, groups, H_kv, H / H_kv, max_slots, 0), B, H, D,
                     pa_layout(B, H, H / H_kv, D, max_slots, false).total, true).total;
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
  const int G = H / H_kv, max_slots = max_pages * page_size;
  const RowsPlan plan = rows_plan(B, n_groups, H_kv, G, max_slots, 0);
  if (plan.ctas > INT32_MAX) return DCR_ERR_SHAPE;
  const PagedAttendLayout a = pa_layout(B, H, G, D, max_slots, false);
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
  p.splits = plan.splits;
  p.window = window;
  p.causal = 0;
  p.scale2 = own.scale2;
  p.o = o;
  p.lse = lse;
  p.part_o = reinterpret_cast<float*>(ws + w.o);
  p.part_ml = reinterpret_cast<float2*>(ws + w.ml);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = pa_launch_any<true>(own, dtype, D, HB, a.ctas, s);
  if (rc != DCR_OK) return rc;
  return rows_dispatch(dtype, D, [&](auto type, auto dims) {
    using Ty = decltype(type);
    constexpr int kDim = decltype(dims)::value;
    const int r = rows_launch<Ty, kDim>(p, plan, s);
    return r != DCR_OK ? r
                       : rows_join<Ty, kDim>(p, reinterpret_cast<const float*>(ws + w.own_o),
                                             reinterpret_cast<const float2*>(ws + w.own_ml), s);
  });
}

}  // extern "C"
