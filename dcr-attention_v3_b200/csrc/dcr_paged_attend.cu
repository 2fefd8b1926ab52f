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
// Bound: the K and V rows, read once (2 * D * element bytes per slot and KV head). The
// arithmetic is 4 * G * D per row, a few per cent of the matrix units, so what matters is how
// many bytes are in flight and that no SM runs dry.
//
// Split. A unit is (sequence, KV head, block of HB = 8 or 16 of its query heads); its slots
// are cut into tiles of R slots on multiples of R. All tiles of all units, in order, are one
// line that the CTAs share out evenly, and each CTA's share its warps: lengths on the device
// may be as unequal as they like. A warp walks its share alone, without barriers: it loads
// rows with 16-byte cp.async into a ring of its own (NH half tiles, K and V in turn; slots
// that are not valid are zero-filled, never read), and keeps the running base, sum and
// output (m, l, o) of the unit it is in. Where a unit lies wholly inside a warp's share the
// warp writes O itself. Otherwise it leaves a piece (m, l, o); the CTA folds its pieces, and
// units that span CTAs are folded from the CTAs' partials in the workspace by a second kernel
// (launched as a programmatic dependent), in a fixed order. Weights take a third kernel: the
// first leaves the scores in the workspace, which costs 8 * G bytes a slot instead of reading
// K again (2 * D bytes).
//
// 16-bit rows go through the tensor cores (mma.sync m16n8k16, A = the query heads as rows): one
// token has at most 16 rows a KV head, so the tile of a tcgen05.mma (64 or 128 rows) would be
// mostly padding and its round trip through TMEM longer than the work. P enters the second
// product as two 16-bit parts (hi = rn(p), lo = rn(p - hi)); with HB = 8 the parts are the two
// row halves of one MMA. In bf16 the parts keep 16 bits of every weight. In f16 they keep 21,
// but end at 2^-24, so f16 weights are taken 2^7 larger (against a base 7 below the maximum):
// they stay below 2^15, and what is lost of a weight is 2^-32 of the row's largest at most. fp32
// rows use fp32 FMAs.
//
// Measured (whole calls back to back in a CUDA graph; the measured copy bandwidth is 6.54 TB/s):
// 4 x 8 KV heads of 64 over 32769 slots, bf16 (268 MB): 47.5 us, 5.65 TB/s, of which some 38 us are
// the stream at 7 TB/s, 4 us its beginning (lengths, page table, first rows) and 5 us the folds; 48
// sequences of 0 to 16000 slots, f16 (747 MB): 120 us, 6.2 TB/s; 16 x 8 heads of 128 in a window of
// 8191, bf16 (537 MB): 92 us, 5.8 TB/s; 3 x 16 heads over 8195 slots in fp32 (201 MB): 38 us, 5.3
// TB/s; 8 x 8 heads over 16385 slots with weights (277 MB): 58.7 us; one sequence of 1000: 7.6 us.
// Tiles of 2 KB instead of 4 needed 453 instead of 261 instructions per 16 slots (66.8 instead of
// 51.7 us for the first case at that step).
#include <math.h>

#include <type_traits>

#include "dcr_internal.h"
#include "dcr_paged.cuh"

namespace dcr {

constexpr int kPaWarps = 8;
constexpr int kPaThreads = kPaWarps * 32;
// Fewest tiles a CTA takes: below it, spreading further costs more in folding than it gains. With
// 4 / 8 / 16 of them, 8 KV heads of 64 over 100 slots take 5.5 / 6.2 / 8.2 us, over 1000 7.1 / 7.6 /
// 8.6, over 4000 9.8 / 8.2 / 9.5, and one KV head of 128 over 8000 14.1 / 10.8 / 10.3.
constexpr int kPaMinTiles = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct PagedAttendParams {
  PagePool c;
  const void* q;
  int64_t qsb, qsh;
  const int32_t* lengths;
  const int32_t* prefix;  // Own: sequence b's first prefix[b] slots are attended elsewhere
  int B, H, H_kv, G;
  int units;      // per sequence: H_kv * blocks of query heads
  int hblocks;    // blocks of query heads per KV head
  float scale2;   // scale * log2(e)
  int window;
  int page16;     // page_size is a multiple of a group: a group lies in one page
  void* o;        // [B][H][D] (Own: fp32)
  float* lse;     // [B][H] natural log, or null
  float2* stats;  // [B][H] (base of the exponents, 1 / sum), with scores and with Own
  float* part;    // [CTAs][2][HB][D + 2]: o, m, l of the open units
  float* scores;  // [B][H][s_stride] base-2 scores, or null
  int64_t s_stride;
};

// Geometry of a variant: T's element bytes, D and the rows of a head block.
template <typename T, int D, int HB>
struct PaShape {
  static constexpr bool k16 = sizeof(T) == 2;
  static constexpr int kRow = D * static_cast<int>(sizeof(T));
  static constexpr int R = 4096 / kRow;                   // slots per tile: 32, 16 or 8
  static constexpr int kChunks = kRow / 16;               // 16-byte chunks per row: 8, 16 or 32
  static constexpr int kHalf = R * kRow;                  // bytes of a K or V half tile
  static constexpr int kRowsPer = 32 / kChunks;           // rows a warp copies per instruction
  static constexpr int kCopies = R / kRowsPer;
  static constexpr int kGroup = R < 16 ? R : 16;          // slots per page lookup
  static constexpr int kGroups = R / kGroup;
  static constexpr int kPiece = HB * (D + 2) * 4;         // a piece (o, m, l)
  static constexpr int kQ = k16 ? 0 : HB * D * 4;         // fp32: the queries, read as broadcasts
  static constexpr int kP = k16 ? 0 : HB * R * 4;         // fp32: the tile's weights
  // ring: an odd number of half tiles (the last half prefetched is of the kind just consumed)
  static constexpr int kFree = (227 * 1024 - 1024) / kPaWarps - kPiece - kQ - kP - 64;
  static constexpr int NHraw = kFree / kHalf;
  static constexpr int NHodd = (NHraw % 2) ? NHraw : NHraw - 1;
  static constexpr int NH = NHodd > 13 ? 13 : NHodd;
  static constexpr int kWarpBytes = NH * kHalf + kPiece + kQ + kP + 64;
  static constexpr int kSmem = kWarpBytes * kPaWarps;
  static_assert(NH >= 3, "the ring holds at least K, V and K");
  static_assert(NH * kHalf >= kPiece, "the ring is reused for the last piece");
};

__device__ __forceinline__ float pa_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row's statistics, with l the sum of exp2(z - m): lse = (m + log2 l) ln 2, and what the
// weights need. Weights are exp2(z - m) / l: a difference of near scores, where lse would be
// rounded once.
__device__ __forceinline__ void pa_store_stats(const PagedAttendParams& p, int64_t row, float m,
                                               float l) {
  if (p.lse != nullptr) p.lse[row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
  if (p.stats != nullptr) p.stats[row] = l == 0.0f ? make_float2(0.0f, 0.0f) : make_float2(m, 1.0f / l);
}

// 8-byte asynchronous global->shared copy.
__device__ __forceinline__ void cp_async_8(void* smem_dst, const void* gsrc) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(smem_dst)), "l"(gsrc) : "memory");
}

// What a state with base m counts for in one with base M >= m; a state without any valid
// slot (m = -inf, sums of 0) counts for nothing.
__device__ __forceinline__ float pa_share(float M, float m) {
  return m == -INFINITY ? 0.0f : pa_exp2(m - M);
}

template <typename T>
__device__ __forceinline__ void pa_store2(T* dst, float a, float b) {
  if constexpr (std::is_same<T, __half>::value)
    *reinterpret_cast<__half2*>(dst) = __floats2half2_rn(a, b);
  else
    *reinterpret_cast<__nv_bfloat162*>(dst) = __floats2bfloat162_rn(a, b);
}

// fp32 output pairs, for the part that is joined with others before it is rounded.
__device__ __forceinline__ void pa_store2(float* dst, float a, float b) {
  *reinterpret_cast<float2*>(dst) = make_float2(a, b);
}

// Tiles of sequence b: its length, first valid slot and tile range. Own: without the prefix.
template <int R, bool Own>
__device__ __forceinline__ void pa_sequence(const PagedAttendParams& p, int b, int& len, int& lo,
                                            int& t_lo, int& t_hi) {
  len = checked_length(p.c, p.lengths[b]);
  lo = p.window > 0 && len > p.window ? len - p.window : 0;
  if constexpr (Own) lo = max(lo, min(p.prefix[b], len));
  t_lo = lo / R;
  t_hi = (len + R - 1) / R;
}

// A place on the line of tiles.
struct PaCursor {
  int b, u, t, t_lo, t_hi, len, lo;
};

template <int R, bool Own>
__device__ __forceinline__ void pa_next(const PagedAttendParams& p, PaCursor& c) {
  if (++c.t < c.t_hi) return;
  if (++c.u == p.units) {
    c.u = 0;
    do {
      if (++c.b >= p.B) return;  // past the end: the caller's count stops here
      pa_sequence<R, Own>(p, c.b, c.len, c.lo, c.t_lo, c.t_hi);
    } while (c.t_lo >= c.t_hi);
  }
  c.t = c.t_lo;
}

__device__ __forceinline__ uint64_t pa_div(uint64_t a, uint32_t b) {
  return (a >> 32) == 0 ? static_cast<uint32_t>(a) / b : a / b;
}

// How the line is shared out: every CTA gets `each` tiles, the first `more` one more. Lane l of
// a warp sums up `per` neighbouring sequences for the search that follows.
struct PaLine {
  int64_t total, each;
  int ctas, more;
  int per;
  int64_t upto;  // tiles per unit of this lane's sequences and all before

  __device__ __forceinline__ int64_t begin(int c) const { return c * each + (c < more ? c : more); }
  __device__ __forceinline__ int cta_of(int64_t place) const {
    const int64_t big = more * (each + 1);
    return place < big ? static_cast<int>(place / (each + 1))
                       : more + static_cast<int>((place - big) / each);
  }
};

template <int R, bool Own>
__device__ __forceinline__ PaLine pa_line(const PagedAttendParams& p, int ctas) {
  const int lane = threadIdx.x & 31;
  PaLine a;
  a.per = (p.B + 31) >> 5;
  a.upto = 0;
#pragma unroll 4
  for (int j = 0; j < a.per; ++j) {
    const int b = lane * a.per + j;
    if (b < p.B) {
      int len, lo, t_lo, t_hi;
      pa_sequence<R, Own>(p, b, len, lo, t_lo, t_hi);
      a.upto += t_hi - t_lo;
    }
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, a.upto, o);
    if (lane >= o) a.upto += y;
  }
  a.total = __shfl_sync(0xffffffffu, a.upto, 31) * p.units;
  const int64_t want = (a.total + kPaMinTiles - 1) / kPaMinTiles;
  a.ctas = want < ctas ? static_cast<int>(want) : ctas;
  a.each = a.ctas > 0 ? pa_div(a.total, a.ctas) : 0;
  a.more = static_cast<int>(a.total - a.each * a.ctas);
  return a;
}

// The cursor at place s (< total) of the line.
template <int R, bool Own>
__device__ __forceinline__ PaCursor pa_seek(const PagedAttendParams& p, const PaLine& line,
                                            int64_t s) {
  const unsigned hit = __ballot_sync(0xffffffffu, s < line.upto * p.units);
  const int l = hit != 0 ? __ffs(hit) - 1 : 31;
  int64_t before = __shfl_sync(0xffffffffu, line.upto, l > 0 ? l - 1 : 0);
  before = l > 0 ? before * p.units : 0;
  PaCursor c;
  c.b = l * line.per;
  pa_sequence<R, Own>(p, c.b, c.len, c.lo, c.t_lo, c.t_hi);
#pragma unroll 1
  while (c.b + 1 < p.B) {
    const int64_t tiles = static_cast<int64_t>(c.t_hi - c.t_lo) * p.units;
    if (s < before + tiles) break;
    before += tiles;
    ++c.b;
    pa_sequence<R, Own>(p, c.b, c.len, c.lo, c.t_lo, c.t_hi);
  }
  const int nt = c.t_hi - c.t_lo;
  const int64_t off = s - before;
  c.u = nt > 0 ? static_cast<int>(pa_div(off, nt)) : 0;
  c.t = c.t_lo + static_cast<int>(off - static_cast<int64_t>(c.u) * nt);
  return c;
}

// The copies of one tile: K's rows, then V's. Where pages hold whole groups of 16 slots (or R,
// if that is less) a page is looked up per group and its rows are a fixed stride apart;
// otherwise every row is looked up by itself, one after the other, which makes the first case
// above 128 us with pages of 8 and 125 with pages of 24 (47 with 16 or 64), the fp32 case 90 with
// pages of 4, 8 or 12 (38). Slots that are not valid are filled with zeros: a copy of no bytes
// reads nothing, whatever its address.
template <typename T, int D, int HB>
struct PaLoader {
  using S = PaShape<T, D, HB>;
  static constexpr uint32_t kAll = 0xffffffffu >> (32 - S::R);
  const char* next_v[S::kGroups];  // this lane's first V row of each group of the tile under way
  int b, hk, slot0;
  uint32_t mask;

  // Issues the tile's K half into `dst` and returns its mask of valid slots.
  __device__ __forceinline__ uint32_t keys(const PagedAttendParams& p, const PaCursor& c,
                                           uint8_t* dst) {
    const int lane = threadIdx.x & 31;
    const int ch = lane % S::kChunks, r0 = lane / S::kChunks;
    b = c.b;
    hk = c.u / p.hblocks;
    slot0 = c.t * S::R;
    const int from = c.lo > slot0 ? c.lo - slot0 : 0;
    const int to = c.len - slot0 < S::R ? c.len - slot0 : S::R;
    mask = (0xffffffffu >> (32 - to)) & (0xffffffffu << from);
    if (!p.page16) {
      mask = copy_each(p, p.c.k, p.c.ksp, p.c.ksh, p.c.ksr, dst);
      return mask;
    }
    const char* src[S::kGroups];
#pragma unroll
    for (int g = 0; g < S::kGroups; ++g) {
      const uint32_t of_group = (0xffffffffu >> (32 - S::kGroup)) << (g * S::kGroup);
      const int s0 = slot0 + g * S::kGroup;
      const uint32_t pi = p.c.page.div(s0);
      const int in = s0 - static_cast<int>(pi * p.c.page.d) + r0;
      int pg = mask & of_group ? page_of(p.c, b, pi) : -1;
      if (pg < 0) {
        mask &= ~of_group;
        pg = 0;
      }
      src[g] = static_cast<const char*>(p.c.k) + ch * 16 +
               (pg * p.c.ksp + hk * p.c.ksh + in * p.c.ksr) * static_cast<int64_t>(sizeof(T));
      next_v[g] = static_cast<const char*>(p.c.v) + ch * 16 +
                  (pg * p.c.vsp + hk * p.c.vsh + in * p.c.vsr) * static_cast<int64_t>(sizeof(T));
    }
    copy_groups(dst, src, p.c.ksr * static_cast<int64_t>(S::kRowsPer * sizeof(T)));
    return mask;
  }

  __device__ __forceinline__ void values(const PagedAttendParams& p, uint8_t* dst) const {
    if (p.page16)
      copy_groups(dst, next_v, p.c.vsr * static_cast<int64_t>(S::kRowsPer * sizeof(T)));
    else
      copy_each(p, p.c.v, p.c.vsp, p.c.vsh, p.c.vsr, dst);
  }

  __device__ __forceinline__ void copy_groups(uint8_t* dst, const char* const (&src)[S::kGroups],
                                              int64_t step) const {
    const int lane = threadIdx.x & 31;
    const uint32_t bits = mask >> (lane / S::kChunks);
    constexpr int kPer = S::kCopies / S::kGroups;
#pragma unroll
    for (int g = 0; g < S::kGroups; ++g) {
      const char* from = src[g];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int r = (g * kPer + i) * S::kRowsPer;
        cp_async_16(dst + at(lane / S::kChunks + r, lane % S::kChunks), from, ((bits >> r) & 1u) * 16u);
        from += step;
      }
    }
  }

  __device__ __forceinline__ uint32_t copy_each(const PagedAttendParams& p, const void* base,
                                                int64_t sp, int64_t sh, int64_t sr,
                                                uint8_t* dst) const {
    const int lane = threadIdx.x & 31;
    const int ch = lane % S::kChunks;
    uint32_t held = 0;
#pragma unroll 1
    for (int i = 0; i < S::kCopies; ++i) {
      const int r = lane / S::kChunks + i * S::kRowsPer;
      bool v = (mask >> r) & 1u;
      int64_t off = 0;
      if (v) {
        const uint32_t pi = p.c.page.div(slot0 + r);
        const int pg = page_of(p.c, b, pi);
        v = pg >= 0;
        if (v) off = pg * sp + hk * sh + (slot0 + r - static_cast<int>(pi * p.c.page.d)) * sr + ch * (16 / static_cast<int>(sizeof(T)));
      }
      cp_async_16(dst + at(r, ch), static_cast<const T*>(base) + off, v ? 16u : 0u);
      const unsigned bal = __ballot_sync(0xffffffffu, v);
#pragma unroll
      for (int j = 0; j < S::kRowsPer; ++j)
        held |= ((bal >> (j * S::kChunks)) & 1u) << (i * S::kRowsPer + j);
    }
    return held;
  }

  // Chunk ch of row r: 16-bit rows by ldmatrix (8 rows of one chunk column at once), fp32 rows
  // by 16-byte reads of two rows' quarters; the swizzles keep both free of bank conflicts.
  __device__ __forceinline__ static uint32_t at(int r, int ch) {
    const int sw = S::k16 ? (ch ^ (r & 7)) : (ch ^ ((r & 1) << 2));
    return static_cast<uint32_t>(r * S::kRow + sw * 16);
  }
};

// The running state of the unit a warp is in. 16-bit: row g of the head block is the MMA row
// lane / 4 (and lane / 4 + 8 when HB = 16), and o holds its dims 8 j + 2 (lane % 4) + {0, 1}.
template <typename T, int D, int HB>
struct PaState16 {
  using S = PaShape<T, D, HB>;
  static constexpr int M = HB / 8;  // row halves in use
  uint32_t qf[D / 16][2 * M];
  float o[D / 8][4];
  float m[M], l[M];
  static constexpr int NT = S::R / 8;
  // m is a base: this much below the largest score so far when it was set
  static constexpr float kBelow = std::is_same<T, __half>::value ? 7.0f : 0.0f;
  uint32_t ph[NT][M], pl[NT][M];  // the tile's weights, hi and lo parts, per 8 slots

  __device__ __forceinline__ void begin(const PagedAttendParams& p, const PaCursor& c, uint8_t*) {
    const int lane = threadIdx.x & 31;
    const int hk = c.u / p.hblocks, h0 = (c.u - hk * p.hblocks) * HB;
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + c.b * p.qsb;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const int g = h0 + lane / 4 + 8 * i;
      const bool in = g < p.G;
      const uint16_t* row = q + (hk * p.G + (in ? g : 0)) * p.qsh + 2 * (lane % 4);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qf[ks][i] = in ? *reinterpret_cast<const uint32_t*>(row + ks * 16) : 0u;
        qf[ks][M + i] = in ? *reinterpret_cast<const uint32_t*>(row + ks * 16 + 8) : 0u;
      }
      m[i] = -INFINITY;
      l[i] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
  }

  __device__ __forceinline__ void scores(const PagedAttendParams& p, const PaCursor& c,
                                         const uint8_t* tile, uint32_t mask, uint8_t*) {
    const int lane = threadIdx.x & 31;
    float z[NT][4] = {};
    const int mat = lane >> 3, r8 = lane & 7;
    const int row = (mat >> 1) * 8 + r8;
    const uint32_t base = smem_u32(tile);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const uint32_t a[4] = {qf[ks][0], M == 2 ? qf[ks][M - 1] : 0u, qf[ks][M],
                             M == 2 ? qf[ks][2 * M - 1] : 0u};
#pragma unroll
      for (int j = 0; j < NT / 2; ++j) {
        uint32_t k0, k1, k2, k3;
        ldsm_x4(base + PaLoader<T, D, HB>::at(row, 2 * ks + (mat & 1)) + j * 16 * S::kRow, k0, k1, k2, k3);
        UnionMma<T>::mma(z[2 * j], a, k0, k1);
        UnionMma<T>::mma(z[2 * j + 1], a, k2, k3);
      }
    }
    const int pos = 2 * (lane & 3);
#pragma unroll
    for (int i = 0; i < M; ++i) {
      float s[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) s[j][e] = z[j][2 * i + e] * p.scale2;
      if (mask != PaLoader<T, D, HB>::kAll) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!((mask >> (8 * j + pos + e)) & 1u)) s[j][e] = -INFINITY;
      }
      if (p.scores != nullptr) {
        const int hk = c.u / p.hblocks;
        const int g = (c.u - hk * p.hblocks) * HB + (lane >> 2) + 8 * i;
        if (g < p.G) {
          float* dst = p.scores + (static_cast<int64_t>(c.b) * p.H + hk * p.G + g) * p.s_stride +
                       c.t * S::R + pos;
#pragma unroll
          for (int j = 0; j < NT; ++j)
            *reinterpret_cast<float2*>(dst + 8 * j) = make_float2(s[j][0], s[j][1]);
        }
      }
      // The base is raised only when some score is 8 above the largest it was set by: weights
      // stay below 2^(8 + kBelow), and most tiles need no rescaling. A NaN score raises nothing
      // and spreads by itself.
      float top = fmaxf(s[0][0], s[0][1]);
#pragma unroll
      for (int j = 1; j < NT; ++j) top = fmaxf(top, fmaxf(s[j][0], s[j][1]));
      if (__any_sync(0xffffffffu, top > m[i] + (8.0f + kBelow))) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float mn = fmaxf(m[i], top - kBelow);
        const float a = m[i] == -INFINITY ? 0.0f : pa_exp2(m[i] - mn);
        m[i] = mn;
        l[i] *= a;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          o[j][2 * i] *= a;
          o[j][2 * i + 1] *= a;
          if (M == 1) {
            o[j][2] *= a;
            o[j][3] *= a;
          }
        }
      }
      const float ms = m[i] == -INFINITY ? 0.0f : m[i];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const float w0 = pa_exp2(s[j][0] - ms), w1 = pa_exp2(s[j][1] - ms);
        l[i] += w0 + w1;
        UnionMma<T>::split(w0, w1, ph[j][i], pl[j][i]);
      }
    }
  }

  __device__ __forceinline__ void values(const uint8_t* tile, uint32_t, uint8_t*) {
    const int lane = threadIdx.x & 31;
    const int mat = lane >> 3, r8 = lane & 7;
    const int row = (mat & 1) * 8 + r8;
    const uint32_t base = smem_u32(tile);
#pragma unroll
    for (int t = 0; t < NT; t += 2) {
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t v0, v1, v2, v3;
        ldsm_x4_t(base + PaLoader<T, D, HB>::at(row, 2 * j + (mat >> 1)) + t * 8 * S::kRow, v0, v1, v2, v3);
        if constexpr (M == 1) {
          const uint32_t a[4] = {ph[t][0], pl[t][0], ph[t + 1][0], pl[t + 1][0]};
          UnionMma<T>::mma(o[2 * j], a, v0, v1);
          UnionMma<T>::mma(o[2 * j + 1], a, v2, v3);
        } else {
          const uint32_t ah[4] = {ph[t][0], ph[t][M - 1], ph[t + 1][0], ph[t + 1][M - 1]};
          const uint32_t al[4] = {pl[t][0], pl[t][M - 1], pl[t + 1][0], pl[t + 1][M - 1]};
          UnionMma<T>::mma(o[2 * j], ah, v0, v1);
          UnionMma<T>::mma(o[2 * j + 1], ah, v2, v3);
          UnionMma<T>::mma(o[2 * j], al, v0, v1);
          UnionMma<T>::mma(o[2 * j + 1], al, v2, v3);
        }
      }
    }
  }

  // The unit's (or share's) end: sums over the lanes of a row.
  __device__ __forceinline__ void close() {
#pragma unroll
    for (int i = 0; i < M; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    if (M == 1) {
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        o[j][0] += o[j][2];
        o[j][1] += o[j][3];
      }
    }
  }

  template <typename TO>
  __device__ __forceinline__ void write(const PagedAttendParams& p, const PaCursor& c) const {
    const int lane = threadIdx.x & 31;
    const int hk = c.u / p.hblocks;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const int g = (c.u - hk * p.hblocks) * HB + (lane >> 2) + 8 * i;
      if (g >= p.G) continue;
      const int64_t row = static_cast<int64_t>(c.b) * p.H + hk * p.G + g;
      const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
      TO* out = static_cast<TO*>(p.o) + row * D + 2 * (lane & 3);
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
        pa_store2(out + 8 * j, o[j][2 * i] * inv, o[j][2 * i + 1] * inv);
      if ((lane & 3) == 0) pa_store_stats(p, row, m[i], l[i]);
    }
  }

  __device__ __forceinline__ void piece(float* dst) const {  // [HB][D + 2]
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      float* r = dst + ((lane >> 2) + 8 * i) * (D + 2);
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
        *reinterpret_cast<float2*>(r + 8 * j + 2 * (lane & 3)) =
            make_float2(o[j][2 * i], o[j][2 * i + 1]);
      if ((lane & 3) == 0) {
        r[D] = m[i];
        r[D + 1] = l[i];
      }
    }
  }
};

// fp32 rows. Scores: lane = (slot lane / 4, quarter lane % 4), which takes every fourth chunk
// of the row; the four partial sums meet by shuffles. Values: a lane holds D / 32 dims of all
// HB rows. m and l are kept by every lane (all lanes agree).
template <typename T, int D, int HB>
struct PaState32 {
  using S = PaShape<T, D, HB>;
  static constexpr int E = D / 32;
  float o[HB][E];
  float m[HB], l[HB];
  int rows;

  __device__ __forceinline__ static float* q_of(uint8_t* own) { return reinterpret_cast<float*>(own); }
  __device__ __forceinline__ static float* p_of(uint8_t* own) {
    return reinterpret_cast<float*>(own + S::kQ);
  }

  __device__ __forceinline__ void begin(const PagedAttendParams& p, const PaCursor& c, uint8_t* own) {
    const int lane = threadIdx.x & 31;
    const int hk = c.u / p.hblocks, h0 = (c.u - hk * p.hblocks) * HB;
    rows = p.G - h0 < HB ? p.G - h0 : HB;
    const float* q = static_cast<const float*>(p.q) + c.b * p.qsb + (hk * p.G + h0) * p.qsh;
    __syncwarp();
    for (int g = 0; g < rows; ++g)
#pragma unroll
      for (int e = 0; e < E; ++e) q_of(own)[g * D + lane + 32 * e] = q[g * p.qsh + lane + 32 * e];
    __syncwarp();
#pragma unroll
    for (int g = 0; g < HB; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) o[g][e] = 0.0f;
    }
  }

  __device__ __forceinline__ void scores(const PagedAttendParams& p, const PaCursor& c,
                                         const uint8_t* tile, uint32_t mask, uint8_t* own) {
    const int lane = threadIdx.x & 31;
    const int r = lane >> 2, qd = lane & 3;
    const int hk = c.u / p.hblocks;
    const int64_t row0 = static_cast<int64_t>(c.b) * p.H + hk * p.G + (c.u - hk * p.hblocks) * HB;
    float4 k[S::R / 8][S::kChunks / 4];
#pragma unroll
    for (int t = 0; t < S::R / 8; ++t)
#pragma unroll
      for (int i = 0; i < S::kChunks / 4; ++i)
        k[t][i] = *reinterpret_cast<const float4*>(tile + PaLoader<T, D, HB>::at(r + 8 * t, 4 * i + qd));
#pragma unroll
    for (int g = 0; g < HB; ++g) {
      if (g >= rows) break;
      const float4* q = reinterpret_cast<const float4*>(q_of(own) + g * D);
      float s[S::R / 8];
      float top = -INFINITY;
#pragma unroll
      for (int t = 0; t < S::R / 8; ++t) {
        float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int i = 0; i < S::kChunks / 4; ++i) {
          const float4 x = q[4 * i + qd];
          s0 = fmaf(k[t][i].x, x.x, s0);
          s1 = fmaf(k[t][i].y, x.y, s1);
          s0 = fmaf(k[t][i].z, x.z, s0);
          s1 = fmaf(k[t][i].w, x.w, s1);
        }
        s[t] = s0 + s1;
        s[t] += __shfl_xor_sync(0xffffffffu, s[t], 1);
        s[t] += __shfl_xor_sync(0xffffffffu, s[t], 2);
        s[t] = (mask >> (r + 8 * t)) & 1u ? s[t] * p.scale2 : -INFINITY;
        if (p.scores != nullptr && qd == 0)
          p.scores[(row0 + g) * p.s_stride + c.t * S::R + r + 8 * t] = s[t];
        top = fmaxf(top, s[t]);
      }
      if (__any_sync(0xffffffffu, top > m[g] + 8.0f)) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float mn = fmaxf(m[g], top);
        const float a = m[g] == -INFINITY ? 0.0f : pa_exp2(m[g] - mn);
        m[g] = mn;
        l[g] *= a;
#pragma unroll
        for (int e = 0; e < E; ++e) o[g][e] *= a;
      }
#pragma unroll
      for (int t = 0; t < S::R / 8; ++t) {
        const float w = pa_exp2(s[t] - (m[g] == -INFINITY ? 0.0f : m[g]));
        l[g] += qd == 0 ? w : 0.0f;
        if (qd == 0) p_of(own)[g * S::R + r + 8 * t] = w;
      }
    }
    __syncwarp();
  }

  __device__ __forceinline__ void values(const uint8_t* tile, uint32_t, uint8_t* own) {
    const int lane = threadIdx.x & 31;
    float v[S::R][E];
#pragma unroll
    for (int r = 0; r < S::R; ++r) {
      const uint8_t* at = tile + PaLoader<T, D, HB>::at(r, lane * E / 4) + (lane * E % 4) * 4;
      if constexpr (E == 2) {
        const float2 x = *reinterpret_cast<const float2*>(at);
        v[r][0] = x.x;
        v[r][1] = x.y;
      } else {
        const float4 x = *reinterpret_cast<const float4*>(at);
        v[r][0] = x.x;
        v[r][1] = x.y;
        v[r][2] = x.z;
        v[r][3] = x.w;
      }
    }
#pragma unroll
    for (int g = 0; g < HB; ++g) {
      if (g >= rows) break;
      const float4* w = reinterpret_cast<const float4*>(p_of(own) + g * S::R);
#pragma unroll
      for (int i = 0; i < S::R / 4; ++i) {
        const float4 x = w[i];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          o[g][e] = fmaf(x.x, v[4 * i][e], o[g][e]);
          o[g][e] = fmaf(x.y, v[4 * i + 1][e], o[g][e]);
          o[g][e] = fmaf(x.z, v[4 * i + 2][e], o[g][e]);
          o[g][e] = fmaf(x.w, v[4 * i + 3][e], o[g][e]);
        }
      }
    }
    __syncwarp();
  }

  __device__ __forceinline__ void close() {
#pragma unroll
    for (int g = 0; g < HB; ++g)
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) l[g] += __shfl_xor_sync(0xffffffffu, l[g], off);
  }

  template <typename TO>
  __device__ __forceinline__ void write(const PagedAttendParams& p, const PaCursor& c) const {
    const int lane = threadIdx.x & 31;
    const int hk = c.u / p.hblocks;
    const int64_t row0 = static_cast<int64_t>(c.b) * p.H + hk * p.G + (c.u - hk * p.hblocks) * HB;
#pragma unroll
    for (int g = 0; g < HB; ++g) {
      if (g >= rows) break;
      float* out = static_cast<float*>(p.o) + (row0 + g) * D + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) out[e] = l[g] == 0.0f ? 0.0f : o[g][e] / l[g];
      if (lane == 0) pa_store_stats(p, row0 + g, m[g], l[g]);
    }
  }

  __device__ __forceinline__ void piece(float* dst) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int g = 0; g < HB; ++g) {
      float* r = dst + g * (D + 2);
#pragma unroll
      for (int e = 0; e < E; ++e) r[lane * E + e] = o[g][e];
      if (lane == 0) {
        r[D] = m[g];
        r[D + 1] = l[g];
      }
    }
  }
};

// A warp's piece: which unit, and whether the unit's tiles go on before or after it.
struct PaPiece {
  int b, u;          // u < 0: none
  int before, after;
};

// Own: only the slots past each sequence's prefix, into fp32 rows and their statistics, which
// are joined with the prefix's afterwards.
template <typename T, int D, int HB, bool Own>
__global__ void __launch_bounds__(kPaThreads, 1) paged_attend_kernel(const PagedAttendParams p) {
  using S = PaShape<T, D, HB>;
  using TO = typename std::conditional<Own, float, T>::type;
  using State = typename std::conditional<S::k16, PaState16<T, D, HB>, PaState32<T, D, HB>>::type;
  extern __shared__ __align__(128) uint8_t pa_smem[];
  __shared__ PaPiece pieces[2 * kPaWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // not before the wait: the call's other kernels read lengths and weights ahead of their own
  asm volatile("griddepcontrol.launch_dependents;");
  uint8_t* ring = pa_smem + warp * (S::NH * S::kHalf);
  uint8_t* own = pa_smem + kPaWarps * (S::NH * S::kHalf) + warp * (S::kPiece + S::kQ + S::kP + 64);
  float* kept = reinterpret_cast<float*>(own);            // the piece that came first
  uint8_t* extra = own + S::kPiece;                       // fp32: queries and weights
  uint32_t* masks = reinterpret_cast<uint32_t*>(own + S::kPiece + S::kQ + S::kP);  // [16]

  const PaLine line = pa_line<S::R, Own>(p, gridDim.x);
  const bool works = static_cast<int>(blockIdx.x) < line.ctas;
  const int64_t c0 = line.begin(blockIdx.x);
  const int n_cta = works ? static_cast<int>(line.each) + (static_cast<int>(blockIdx.x) < line.more) : 0;
  const int rest = n_cta % kPaWarps;
  const int n = n_cta / kPaWarps + (warp < rest);
  const int64_t s0 = c0 + warp * (n_cta / kPaWarps) + (warp < rest ? warp : rest);
  if (lane == 0) pieces[2 * warp].u = pieces[2 * warp + 1].u = -1;

  if (n > 0) {
    PaCursor in = pa_seek<S::R, Own>(p, line, s0);  // where loads are
    PaCursor at = in;                          // where the arithmetic is
    PaLoader<T, D, HB> load;
    State st;
    constexpr int kAhead = (S::NH - 1) / 2;  // tiles in flight
    int hs_in = 0;                           // ring places of the loads and of the arithmetic
    int hs = 0;
    int first = at.t;                        // its first tile in this share
    st.begin(p, at, extra);
    // the first kAhead turns only load; every turn's loads are kAhead tiles ahead
#pragma unroll 1
    for (int i = -kAhead; i < n; ++i) {
      const int j = i + kAhead;
      cp_async_wait<2 * kAhead - 1>();
      __syncwarp();
      if (j < n) {
        const uint32_t m = load.keys(p, in, ring + hs_in * S::kHalf);
        if (lane == 0) masks[j & 15] = m;
      }
      cp_async_commit();
      hs_in = hs_in + 1 == S::NH ? 0 : hs_in + 1;
      const uint32_t mask = masks[i & 15];
      if (i >= 0) {
        st.scores(p, at, ring + hs * S::kHalf, mask, extra);
        hs = hs + 1 == S::NH ? 0 : hs + 1;
        cp_async_wait<2 * kAhead - 1>();
        __syncwarp();
      }
      if (j < n) {
        load.values(p, ring + hs_in * S::kHalf);
        if (j + 1 < n) pa_next<S::R, Own>(p, in);
      }
      cp_async_commit();
      hs_in = hs_in + 1 == S::NH ? 0 : hs_in + 1;
      if (i < 0) continue;
      st.values(ring + hs * S::kHalf, mask, extra);
      hs = hs + 1 == S::NH ? 0 : hs + 1;
      const bool ends = at.t + 1 == at.t_hi;
      if (ends || i + 1 == n) {
        st.close();
        const bool before = first > at.t_lo;
        if (!before && ends) {
          st.template write<TO>(p, at);
        } else {
          // before: the only piece that can be followed by others, so it has its own place;
          // a piece that goes on after the share is the last, and the ring is free then
          float* dst = kept;
          if (!before) {
            cp_async_wait<0>();
            __syncwarp();
            dst = reinterpret_cast<float*>(ring);
          }
          st.piece(dst);
          if (lane == 0) {
            PaPiece& pc = pieces[2 * warp + (before ? 0 : 1)];
            pc.b = at.b;
            pc.u = at.u;
            pc.before = before;
            pc.after = !ends;
          }
        }
        if (i + 1 < n) {
          pa_next<S::R, Own>(p, at);
          first = at.t;
          st.begin(p, at, extra);
        }
      } else {
        ++at.t;
      }
    }
    cp_async_wait<0>();
  }
  __syncthreads();

  // Fold the CTA's pieces: the rows of all its units are dealt out to the warps. Lane x holds
  // piece x; the pieces of a unit are neighbours. Odd pieces are in the rings, even ones in the
  // warps' own places.
  const PaPiece mine = pieces[lane % (2 * kPaWarps)];
  const bool have = lane < 2 * kPaWarps && mine.u >= 0;
  auto piece_at = [&](int x) {
    return reinterpret_cast<const float*>(
        (x & 1) ? pa_smem + (x >> 1) * (S::NH * S::kHalf)
                : pa_smem + kPaWarps * (S::NH * S::kHalf) + (x >> 1) * (S::kPiece + S::kQ + S::kP + 64));
  };
  const float* own_piece = piece_at(lane % (2 * kPaWarps));
  unsigned todo = __ballot_sync(0xffffffffu, have);
  int dealt = warp;  // rows until this warp's next one
  while (todo != 0) {
    const int lead = __ffs(todo) - 1;
    const int b = __shfl_sync(0xffffffffu, mine.b, lead), u = __shfl_sync(0xffffffffu, mine.u, lead);
    const unsigned run = __ballot_sync(0xffffffffu, have && mine.b == b && mine.u == u);
    todo &= ~run;
    const bool before = __shfl_sync(0xffffffffu, mine.before, lead);
    const bool after = __shfl_sync(0xffffffffu, mine.after, 31 - __clz(run));
    const int hk = u / p.hblocks, h0 = (u - hk * p.hblocks) * HB;
    const int rows = p.G - h0 < HB ? p.G - h0 : HB;
    for (; dealt < rows; dealt += kPaWarps) {
      const int g = dealt;
      const bool in = (run >> lane) & 1u;
      const float m = in ? own_piece[g * (D + 2) + D] : -INFINITY;
      float M = m;
#pragma unroll
      for (int o = kPaWarps; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
      M = __shfl_sync(0xffffffffu, M, lead);  // pieces are in the first 2 * kPaWarps lanes
      const float a = pa_share(M, m);
      float L = in ? a * own_piece[g * (D + 2) + D + 1] : 0.0f;
#pragma unroll
      for (int o = kPaWarps; o >= 1; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
      L = __shfl_sync(0xffffffffu, L, lead);
      float acc[D / 32] = {};
#pragma unroll 1
      for (unsigned left = run; left != 0; left &= left - 1) {
        const int x = __ffs(left) - 1;
        const float ax = __shfl_sync(0xffffffffu, a, x);
        const float* src = piece_at(x) + g * (D + 2);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) acc[e] = fmaf(ax, src[lane + 32 * e], acc[e]);
      }
      if (!before && !after) {
        const int64_t row = static_cast<int64_t>(b) * p.H + hk * p.G + h0 + g;
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
        for (int e = 0; e < D / 32; ++e)
          ElemTraits<TO>::store(static_cast<TO*>(p.o) + row * D, lane + 32 * e, acc[e] * inv);
        if (lane == 0) pa_store_stats(p, row, M, L);
      } else {
        float* dst = p.part + ((2 * static_cast<int64_t>(blockIdx.x) + (before ? 0 : 1)) * HB + g) * (D + 2);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) dst[lane + 32 * e] = acc[e];
        if (lane == 0) {
          dst[D] = M;
          dst[D + 1] = L;
        }
      }
    }
    dealt -= rows;
  }

  // rows of empty sequences
#pragma unroll 1
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    int len, lo, t_lo, t_hi;
    pa_sequence<S::R, Own>(p, b, len, lo, t_lo, t_hi);
    if (t_lo < t_hi) continue;
    const int64_t row0 = static_cast<int64_t>(b) * p.H;
    for (int i = threadIdx.x; i < p.H * D; i += kPaThreads)
      ElemTraits<TO>::store(static_cast<TO*>(p.o) + row0 * D, i, 0.0f);
    for (int i = threadIdx.x; i < p.H; i += kPaThreads) pa_store_stats(p, row0 + i, 0.0f, 0.0f);
  }
}

// Folds the partials of the unit that begins in CTA blockIdx.x of the first kernel and ends in
// a later one; blockIdx.y is the row of the head block. What there is to fold follows from the
// lengths, so it is known before the first kernel is done; then up to kFoldParts partials are
// copied to shared memory at once and folded from there. The code is kept small and rolled up:
// it runs once, from a cold instruction cache. (CTAs with nothing to fold leave at once, all but
// the first: the kernel must not end before the one it waits for.)
constexpr int kFoldThreads = 128, kFoldParts = 32;

template <typename T, int D, int HB, bool Own>
__global__ void __launch_bounds__(kFoldThreads) paged_fold_kernel(const PagedAttendParams p) {
  using S = PaShape<T, D, HB>;
  using TO = typename std::conditional<Own, float, T>::type;
  constexpr int W = D + 2;              // o, m, l
  __shared__ __align__(8) float part[kFoldParts * W];
  asm volatile("griddepcontrol.launch_dependents;");
  const PaLine line = pa_line<S::R, Own>(p, gridDim.x);
  const int c0 = blockIdx.x;
  const int64_t end_cta = line.begin(c0 + 1);
  bool open = c0 + 1 < line.ctas;
  PaCursor c;
  int last = 0, hk = 0, h = 0;
  if (open) {
    c = pa_seek<S::R, Own>(p, line, end_cta - 1);
    const int64_t begin = end_cta - 1 - (c.t - c.t_lo), end = begin + (c.t_hi - c.t_lo);
    hk = c.u / p.hblocks;
    h = (c.u - hk * p.hblocks) * HB + blockIdx.y;
    open = begin >= line.begin(c0) && end > end_cta && h < p.G;
    if (open) last = line.cta_of(end - 1);
  }
  if (!open && blockIdx.x + blockIdx.y > 0) return;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!open) return;
  const int d = threadIdx.x;
  float M = -INFINITY, L = 0.0f, acc = 0.0f;
#pragma unroll 1
  for (int c1 = c0; c1 <= last; c1 += kFoldParts) {
    const int count = min(kFoldParts, last + 1 - c1);
    if (c1 > c0) __syncthreads();
#pragma unroll 1
    for (int i = threadIdx.x; i < count * (W / 2); i += kFoldThreads) {
      const int x = i / (W / 2), e = i - x * (W / 2);
      const float* src = p.part + ((2 * static_cast<int64_t>(c1 + x) + (c1 + x == c0 ? 1 : 0)) * HB + blockIdx.y) * W;
      cp_async_8(part + x * W + 2 * e, src + 2 * e);
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    // lane x holds partial x's statistics, in every warp
    const int lane = threadIdx.x & 31;
    const float m = lane < count ? part[lane * W + D] : -INFINITY;
    float top = fmaxf(M, m);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float old = pa_share(top, M);
    L *= old;
    acc *= old;
    M = top;
    const float a = pa_share(M, m);
    float l = lane < count ? a * part[lane * W + D + 1] : 0.0f;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    L += l;
#pragma unroll 8
    for (int x = 0; x < count; ++x)
      acc = fmaf(__shfl_sync(0xffffffffu, a, x), part[x * W + (d < D ? d : 0)], acc);
  }
  if (d >= D) return;
  const int64_t row = static_cast<int64_t>(c.b) * p.H + hk * p.G + h;
  ElemTraits<TO>::store(static_cast<TO*>(p.o) + row * D, d, L == 0.0f ? 0.0f : acc / L);
  if (d == 0) pa_store_stats(p, row, M, L);
}

// weights[b][h_kv][i] += sum over the G heads of exp2(score - m) / l, in head order. A thread
// takes kWeightSlots neighbouring slots; the old weights, which no kernel before this one of the
// call touches, are loaded while those still run.
constexpr int kWeightThreads = 256, kWeightSlots = 4;

__global__ void __launch_bounds__(kWeightThreads) paged_weights_kernel(const PagedAttendParams p,
                                                                       float* weights, int64_t wsb,
                                                                       int64_t wsh) {
  const int hk = blockIdx.y;
  const int i0 = (blockIdx.x * kWeightThreads + threadIdx.x) * kWeightSlots;
  bool waited = false;
  for (int b = blockIdx.z; b < p.B; b += gridDim.z) {
    const int n = checked_length(p.c, p.lengths[b]);
    const int lo = p.window > 0 && n > p.window ? n - p.window : 0;
    float* dst = weights + b * wsb + hk * wsh + i0;
    float w[kWeightSlots], add[kWeightSlots] = {};
#pragma unroll
    for (int e = 0; e < kWeightSlots; ++e) w[e] = i0 + e >= lo && i0 + e < n ? dst[e] : 0.0f;
    if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
    waited = true;
    if (i0 >= n || i0 + kWeightSlots <= lo) continue;
    const int64_t row0 = static_cast<int64_t>(b) * p.H + hk * p.G;
    const float* src = p.scores + row0 * p.s_stride + i0;
#pragma unroll 4
    for (int g = 0; g < p.G; ++g) {
      const float2 ml = p.stats[row0 + g];
      const float4 s4 = *reinterpret_cast<const float4*>(src + g * p.s_stride);
      const float s[kWeightSlots] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
      for (int e = 0; e < kWeightSlots; ++e)
        add[e] += s[e] == -INFINITY ? 0.0f : pa_exp2(s[e] - ml.x) * ml.y;
    }
#pragma unroll
    for (int e = 0; e < kWeightSlots; ++e)
      if (i0 + e >= lo && i0 + e < n) dst[e] = w[e] + add[e];
  }
}

// Workspace sections.
struct PagedAttendLayout {
  size_t part, stats, scores, total;
  int64_t s_stride;
  int ctas;
};

// Query heads per block: all of a KV head's up to 16, so that its rows are read once. Single
// precision with D = 128 keeps to 8: the queries and pieces of 16 would leave no ring.
static int pa_head_block(int G, int D, int dtype) {
  return G <= 8 || (D == 128 && dtype == DCR_DTYPE_F32) ? 8 : 16;
}

static PagedAttendLayout pa_layout(int B, int H, int G, int D, int max_slots, bool weights) {
  PagedAttendLayout w;
  w.ctas = device_sm_count();
  size_t off = 0;
  auto take = [&](size_t n) {
    const size_t at = off;
    off = (off + n + 255) / 256 * 256;
    return at;
  };
  w.part = take(sizeof(float) * 2 * w.ctas * (G <= 8 ? 8 : 16) * (D + 2));
  w.stats = weights ? take(sizeof(float2) * static_cast<size_t>(B) * H) : 0;
  w.s_stride = (static_cast<int64_t>(max_slots) + 31) / 32 * 32;  // whole tiles are stored
  w.scores = weights ? take(sizeof(float) * static_cast<size_t>(B) * H * w.s_stride) : 0;
  w.total = off;
  return w;
}

template <typename T, int D, int HB, bool Own>
static int pa_launch(const PagedAttendParams& p, int ctas, cudaStream_t s) {
  using S = PaShape<T, D, HB>;
  auto kernel = paged_attend_kernel<T, D, HB, Own>;
  if (ensure_smem_attr(reinterpret_cast<const void*>(kernel), S::kSmem) != cudaSuccess)
    return DCR_ERR_CUDA;
  PagedAttendParams q = p;
  q.page16 = p.c.page.d % S::kGroup == 0;
  const int rows = p.G < HB ? p.G : HB;
  if (launch_dependent(kernel, dim3(ctas), dim3(kPaThreads), S::kSmem, s, 1, q) != cudaSuccess ||
      launch_dependent(paged_fold_kernel<T, D, HB, Own>, dim3(ctas, rows), dim3(kFoldThreads), 0, s, 1, q) != cudaSuccess)
    return DCR_ERR_CUDA;
  return DCR_OK;
}

template <typename T, bool Own>
static int pa_launch_t(const PagedAttendParams& p, int D, int HB, int ctas, cudaStream_t s) {
  if (D == 64) return HB == 8 ? pa_launch<T, 64, 8, Own>(p, ctas, s) : pa_launch<T, 64, 16, Own>(p, ctas, s);
  if constexpr (sizeof(T) == 2) {
    if (HB == 16) return pa_launch<T, 128, 16, Own>(p, ctas, s);
  }
  return pa_launch<T, 128, 8, Own>(p, ctas, s);
}

template <bool Own>
static int pa_launch_any(const PagedAttendParams& p, int dtype, int D, int HB, int ctas, cudaStream_t s) {
  switch (dtype) {
    case DCR_DTYPE_BF16: return pa_launch_t<__nv_bfloat16, Own>(p, D, HB, ctas, s);
    case DCR_DTYPE_F16: return pa_launch_t<__half, Own>(p, D, HB, ctas, s);
    default: return pa_launch_t<float, Own>(p, D, HB, ctas, s);
  }
}

}  // namespace dcr

using namespace dcr;

extern "C" {

size_t dcr_paged_workspace_bytes(int B, int H, int H_kv, int D, int max_slots, int with_weights) {
  if (B <= 0 || H_kv <= 0 || H <= 0 || H % H_kv != 0 || (D != 64 && D != 128) || max_slots <= 0)
    return 0;
  return pa_layout(B, H, H / H_kv, D, max_slots, with_weights != 0).total;
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
  if (B <= 0 || H <= 0 || H_kv <= 0 || H_kv > 65535 || H % H_kv != 0 || window < 0)
    return DCR_ERR_SHAPE;
  const int st = check_pool(k_pages, v_pages, dtype, k_stride_p, k_stride_h, k_stride_s,
                            v_stride_p, v_stride_h, v_stride_s, num_pages, page_size, page_table,
                            table_stride, max_pages, H_kv, D);
  if (st != DCR_OK) return st;
  const int64_t per16 = dtype == DCR_DTYPE_F32 ? 4 : 8;
  if (misaligned(16, q, o) || misaligned(4, lengths, lse, weights) || q_stride_b % per16 ||
      q_stride_h % per16)
    return DCR_ERR_ALIGN;
  if (q_stride_b < 0 || q_stride_h < 0) return DCR_ERR_SHAPE;
  const int max_slots = max_pages * page_size;
  if (weights != nullptr && (w_stride_h < 0 || w_stride_b < 0 ||
                             !rows_apart(B, H_kv, max_slots, w_stride_b, w_stride_h)))
    return DCR_ERR_SHAPE;
  const int G = H / H_kv;
  const PagedAttendLayout w = pa_layout(B, H, G, D, max_slots, weights != nullptr);
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15u) ||
      workspace_bytes < w.total)
    return DCR_ERR_WORKSPACE;
  if (rows_meet(q, q_stride_b, q_stride_h, o, B, H, D, 16 / per16)) return DCR_ERR_SHAPE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int HB = pa_head_block(G, D, dtype);
  PagedAttendParams p;
  p.c = make_pool(k_pages, v_pages, k_stride_p, k_stride_h, k_stride_s, v_stride_p, v_stride_h,
                  v_stride_s, num_pages, page_size, page_table, table_stride, max_pages);
  p.q = q;
  p.qsb = q_stride_b;
  p.qsh = q_stride_h;
  p.lengths = lengths;
  p.prefix = nullptr;
  p.B = B;
  p.H = H;
  p.H_kv = H_kv;
  p.G = G;
  p.hblocks = (G + HB - 1) / HB;
  p.units = H_kv * p.hblocks;
  p.scale2 = scale * kLog2e;
  p.window = window;
  p.page16 = 0;
  p.o = o;
  p.lse = lse;
  p.stats = weights != nullptr ? reinterpret_cast<float2*>(ws + w.stats) : nullptr;
  p.part = reinterpret_cast<float*>(ws + w.part);
  p.scores = weights != nullptr ? reinterpret_cast<float*>(ws + w.scores) : nullptr;
  p.s_stride = w.s_stride;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = pa_launch_any<false>(p, dtype, D, HB, w.ctas, s);
  if (rc != DCR_OK || weights == nullptr) return rc;
  const int chunk = kWeightThreads * kWeightSlots;
  const dim3 grid((max_slots + chunk - 1) / chunk, H_kv, B < 65535 ? B : 65535);
  return launch_dependent(paged_weights_kernel, grid, dim3(kWeightThreads), 0, s, 1, p, weights,
                          w_stride_b, w_stride_h) == cudaSuccess
             ? DCR_OK
             : DCR_ERR_CUDA;
}

}  // extern "C"
