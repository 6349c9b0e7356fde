// Attention over a paged cache in 4 bits (mx_kv4.hip), for single tokens, drafts and prompts.
//
// S = c q K^T over the tokens that a row sees, with the running maximum m and sum l of a softmax; O = P V / (l + sink).
//
// A wave holds 32 query rows (a row: one head of one token; the heads of a key head and the tokens of a sequence share
// their keys) and takes 32 cached tokens a step, transposed: S^T = K Q^T has a query row in every lane, so that the
// softmax's maximum, sum and scaling need no exchange but one between the wave's halves, and its registers are the right
// operand of O^T = V^T P^T as they are.
//   S^T: V_MFMA_SCALE_F32_32X32X64_F8F6F4 on the codes and scales as they lie in the cache, with the query as two E4M3
//        terms: a BF16 value has 8 significant bits, the first term takes 4 of them and the second, 2^-4 of its scale, the
//        rest, so the products are those of the BF16 query (to 2^-20 of a block's largest). At the rate of E4M3, two terms
//        cost what one BF16 product does, and the keys need no conversion.
//   O^T: V_MFMA_F32_32X32X16_BF16. A scale belongs to a token and 32 columns, but this product runs over the tokens, so
//        the values become BF16 (exactly: two significant bits and a power of two) by V_CVT_SCALEF32_PK_BF16_FP4, in the
//        row order in which they lie, and go through LDS, whose transposing reads give each lane its column's tokens.
//
// Work is divided evenly over the device: a unit is the row tile of one sequence and key head, an iteration one step of all
// the workgroup's token groups, and workgroup g takes the iterations [g per, (g + 1) per) of all units in a row. Units that
// a workgroup has alone go straight to out; the others' parts go to the workspace and join_kernel adds them up.
#include <algorithm>
#include <type_traits>

#include "mx_kv4.h"

namespace {

using namespace mxh;
using namespace mxk;

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef mxd::v8i v8i;

constexpr int kCus = 256, kXcds = 8;
constexpr int kInlineTiles = 1024;   // sequences, and row tiles of all of them, that every workgroup counts for itself
constexpr float kLowest = -3e38f;    // the maximum of a row that has seen nothing yet
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Byte offsets of the workspace.
struct Space {
  int64_t units, stats, rows, base, prefix, total;
};

struct AttendArgs {
  mx_kv4 cache;
  mx_kv4_query q;
  int group;           // query heads of a key head
  int page_shift;
  int tiles;           // row tiles of all sequences, at most
  float c;             // scale log2(e)
  uint8_t* space;
  Space at;
};

// A workgroup's last unit, where the next workgroups go on with it: who adds it up, and over how many workgroups.
struct Shared {
  int32_t b, h, tile, parts, slot;
};

struct Sequence {
  int first, n;        // query rows in tokens
  int held;            // cached tokens
  int64_t end;         // the length, which may be more than the table holds
};

__device__ __forceinline__ Sequence sequence(const AttendArgs& a, int b) {
  Sequence s;
  if (a.q.q_first) {
    s.first = min(max(a.q.q_first[b], 0), a.q.tokens);
    s.n = min(max(a.q.q_first[b + 1], s.first), a.q.tokens) - s.first;
  } else {
    s.n = a.q.tokens / a.q.batch, s.first = b * s.n;
  }
  const int length = a.q.lengths[b];
  s.end = length;
  s.held = (int)min<int64_t>(max(length, 0), (int64_t)a.q.columns << a.page_shift);
  return s;
}

// The tokens that query token i of the sequence sees.
__device__ __forceinline__ void seen(const AttendArgs& a, const Sequence& s, int i, int& lo, int& hi) {
  const int64_t end = s.end - s.n + i + 1;
  hi = (int)min<int64_t>(max<int64_t>(end, 0), s.held);
  lo = a.q.window ? (int)min<int64_t>(max<int64_t>(end - a.q.window, 0), hi) : 0;
}

// Tokens [lo, hi) that some row of row tile `tile` sees (lo at a whole step), and its iterations of `step` tokens: one at
// least, which writes the rows that see nothing.
__device__ __forceinline__ int tile_iterations(const AttendArgs& a, const Sequence& s, int tile, int rows, int step, int& lo, int& hi) {
  const int64_t row0 = (int64_t)tile * rows, all = (int64_t)s.n * a.group;
  int l1, h0;
  seen(a, s, (int)(row0 / a.group), lo, h0);
  seen(a, s, (int)((min<int64_t>(row0 + rows, all) - 1) / a.group), l1, hi);
  lo &= ~31;
  return max(1, (hi - lo + step - 1) / step);
}

// The plan: base[b] = row tiles of the sequences before b, prefix[i] = iterations (of one key head) of the row tiles before
// i. Made by a workgroup of N threads in its LDS, or by plan_kernel in the workspace.
struct Plan {
  int32_t* base;
  int64_t* prefix;
};

template <int N>
__device__ __forceinline__ int64_t scan(int64_t v, int64_t* sums, int64_t& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t s = v;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int64_t o = __shfl_up(s, m, 64);
    s += lane >= m ? o : 0;
  }
  __syncthreads();
  if (lane == 63) sums[wave] = s;
  __syncthreads();
  int64_t before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < N / 64; ++w) {
    before += w < wave ? sums[w] : 0;
    all += sums[w];
  }
  return before + s - v;
}

__device__ __forceinline__ int find(const int32_t* base, int n, int i) {   // the last b with base[b] <= i
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (base[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

template <int N>
__device__ __forceinline__ void make_plan(const AttendArgs& a, Plan p, int64_t* sums, int rows, int step) {
  int64_t tiles = 0, all;
  for (int b0 = 0; b0 < a.q.batch; b0 += N) {
    const int b = b0 + threadIdx.x;
    int64_t n = 0;
    if (b < a.q.batch) n = ((int64_t)sequence(a, b).n * a.group + rows - 1) / rows;
    const int64_t before = scan<N>(n, sums, all);
    // (no more than there is room for: a q_first that does not ascend could name more rows than there are)
    if (b < a.q.batch) p.base[b] = (int)min<int64_t>(tiles + before, a.tiles);
    tiles += all;
  }
  tiles = min<int64_t>(tiles, a.tiles);
  if (threadIdx.x == 0) p.base[a.q.batch] = (int)tiles;
  __syncthreads();
  int64_t sum = 0;
  for (int i0 = 0; i0 < tiles; i0 += N) {
    const int i = i0 + threadIdx.x;
    int64_t n = 0;
    if (i < tiles) {
      const int b = find(p.base, a.q.batch, i);
      int lo, hi;
      n = tile_iterations(a, sequence(a, b), i - p.base[b], rows, step, lo, hi);
    }
    const int64_t before = scan<N>(n, sums, all);
    if (i < tiles) p.prefix[i] = sum + before;
    sum += all;
  }
  if (threadIdx.x == 0) p.prefix[tiles] = sum;
  __syncthreads();
}

__global__ __launch_bounds__(1024) void plan_kernel(AttendArgs a, int rows, int step) {
  __shared__ int64_t sums[16];
  make_plan<1024>(a, {(int32_t*)(a.space + a.at.base), (int64_t*)(a.space + a.at.prefix)}, sums, rows, step);
}

// Two E4M3 terms of 16 query values (BF16 pairs w) under the scale 2^(exponent - 127), which takes them into [-256, 256]:
// the nearest code, and of what is left the nearest code under 2^-4 of the scale.
__device__ __forceinline__ void split16(const uint32_t (&w)[8], uint32_t exponent, uint32_t* high, uint32_t* low) {
  typedef short v2s __attribute__((ext_vector_type(2)));
  typedef __bf16 v2b __attribute__((ext_vector_type(2)));
  const float scale = mx::u2f(exponent << 23), fine = mx::u2f((exponent - 4u) << 23);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v2s h = {0, 0}, l = {0, 0};
    h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h, __builtin_bit_cast(v2b, w[2 * j]), scale, false);
    h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h, __builtin_bit_cast(v2b, w[2 * j + 1]), scale, true);
    high[j] = __builtin_bit_cast(uint32_t, h);
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(high[j], scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(high[j], scale, true);
    l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, mx::u2f(w[2 * j] << 16) - a[0], mx::u2f(w[2 * j] & 0xFFFF0000u) - a[1], fine, false);
    l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, mx::u2f(w[2 * j + 1] << 16) - b[0], mx::u2f(w[2 * j + 1] & 0xFFFF0000u) - b[1], fine, true);
    low[j] = __builtin_bit_cast(uint32_t, l);
  }
}

// The scale exponent of a block of 32 query values whose magnitudes' largest (as BF16 bits) is top: [128, 256) 2^e. 255
// (NaN) where a value is not finite; blocks below 2^-107 lose their last bits.
__device__ __forceinline__ uint32_t query_exponent(uint32_t top) {
  return top >= 0x7F80u ? 255u : max(top >> 7, 20u) - 7u;
}
__device__ __forceinline__ uint32_t pair_max(uint32_t a, uint32_t b) {   // of two 16-bit numbers each
  typedef unsigned short v2u __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(v2u, a), __builtin_bit_cast(v2u, b)));
}

// Into the accumulation registers: where a wave has all 512 registers of a lane, the queries, which only products read,
// stay in the half that other instructions cannot use.
__device__ __forceinline__ void keep(v8i& v) { asm volatile("" : "+a"(v)); }

template <int kA, int kB>
__device__ __forceinline__ v16f scores(uint4 k, const v8i& q, v16f c, uint32_t ks, uint32_t qs) {
  const v8i av = {(int)k.x, (int)k.y, (int)k.z, (int)k.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, q, c, 4, 0, kA, (int)ks, kB, (int)qs);
}

// Whether one of the used bytes of w is 0xFF.
__device__ __forceinline__ uint32_t marks(uint32_t w) {
  const uint32_t x = ~w;
  return (x - 0x01010101u) & ~x & 0x80808080u;
}

__device__ __forceinline__ float other_half_max(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
  return fmaxf(__int_as_float(p[0]), __int_as_float(p[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
  return __int_as_float(p[0]) + __int_as_float(p[1]);
}

// Waves that a SIMD holds (so workgroups a CU), by what their registers allow.
__host__ __device__ constexpr int waves(int value_width) { return value_width <= 64 ? 3 : value_width <= 128 ? 2 : 1; }

// WK, WV: widths of a key and of a value; kApart: values have codes of their own; RG: the workgroup's row groups of 32. A
// step is 4 / RG tiles of 32 tokens, each of which RG waves (one a row group) score and, in parts, convert.
//
// kSplit (latents): 32 rows of 512 columns and their queries would be 390 registers of a lane's 512 before anything else,
// so a wave multiplies all of the step's tiles by WV RG / 4 columns of the values, and the waves of a row group exchange
// their probabilities through LDS. Otherwise a wave keeps to its tile, and the waves' sums are added at the end.
template <int WK, int WV, bool kApart, int RG>
struct Attend {
  static constexpr bool kSplit = WV >= 512;
  static constexpr int TG = 4 / RG, kRows = 32 * RG, kStep = 32 * TG;
  static constexpr int KS = WK / 64, VS = WV / 64, DB = WV / 32 / (kSplit ? TG : 1);
  static constexpr int KW = scale_pitch(WK) / 4, VW = scale_pitch(WV) / 4;
  static constexpr int VO = (VS + RG - 1) / RG;            // 64-column pieces of the values that a wave converts
  static constexpr int kTile = 64 * WV;                    // bytes of 32 tokens' values in BF16
  // of the values, where others read what a wave has written: two, so that one barrier a step is enough, if they fit
  static constexpr int kBuffers = (RG > 1 || kSplit) && 2 * TG * kTile <= 131072 ? 2 : 1;
  static constexpr int kExchange = kSplit ? 2 * 4 * 64 * 32 : 16;   // probabilities
  static constexpr int CB = WV < 64 ? WV : 64;             // columns that go out at a time
  static constexpr int kOut = 32 * (CB + 4) * 4;           // bytes of a wave's
  static constexpr int kLds = TG * kBuffers * kTile > 4 * kOut ? TG * kBuffers * kTile : 4 * kOut;
  static constexpr int kWaves = waves(WV), kGroups = kCus * kWaves;
};

// Where a row of a unit goes (in values; -1: nowhere), and its factor.
struct Place {
  int64_t at;
  float by;
};

struct RowOut {
  float inv, lse;
};
__device__ __forceinline__ RowOut row_out(const AttendArgs& a, int head, float m, float l) {
  const float sink = a.q.sinks && l != 0.f ? __builtin_amdgcn_exp2f(fmaf(a.q.sinks[head], kLog2e, -m)) : 0.f;
  return {l == 0.f ? 0.f : 1.f / (l + sink), l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2};
}

__device__ __forceinline__ float power(float from, float to) {   // 2^(from - to), 1 where they are equal (infinities too)
  return from == to ? 1.f : __builtin_amdgcn_exp2f(from - to);
}

template <int WK, int WV, bool kApart, int RG>
__global__ __launch_bounds__(256, (Attend<WK, WV, kApart, RG>::kWaves)) void attend_kernel(AttendArgs a, int inline_plan) {
  using A = Attend<WK, WV, kApart, RG>;
  constexpr bool kSplit = A::kSplit;
  constexpr int TG = A::TG, KS = A::KS, VS = A::VS, DB = A::DB, KW = A::KW, VW = A::VW, VO = A::VO, CB = A::CB;
  __shared__ __attribute__((aligned(16))) uint8_t lds[A::kLds];
  __shared__ __attribute__((aligned(16))) uint8_t exchange[A::kExchange];
  __shared__ float tops[2][4][32];
  __shared__ float stats[4][32][2];
  __shared__ Place places[A::kRows];
  __shared__ int64_t plan_prefix[kInlineTiles + 1];
  __shared__ int32_t plan_base[kInlineTiles + 1];
  __shared__ int64_t sums[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rg = wave % RG, tg = wave / RG;
  const int col = lane & 31, half = lane >> 5;   // the lane's query row of the products; as a loader, its token

  Plan plan{(int32_t*)(a.space + a.at.base), (int64_t*)(a.space + a.at.prefix)};
  if (inline_plan) {
    plan = {plan_base, plan_prefix};
    make_plan<256>(a, plan, sums, A::kRows, A::kStep);
  }
  const int64_t all = plan.prefix[plan.base[a.q.batch]] * a.cache.heads;
  constexpr int groups = A::kGroups;
  const int64_t per = max<int64_t>((all + groups - 1) / groups, 1);
  // workgroups go round the XCDs: neighbours in the work, which share keys, to one L2
  const int g = (int)(blockIdx.x % kXcds) * (groups / kXcds) + (int)blockIdx.x / kXcds;
  int64_t x = min(g * per, all);
  const int64_t end = min(x + per, all);
  Shared* shared = (Shared*)(a.space + a.at.units) + g;
  if (tid == 0 && x >= end) shared->parts = 0;

  // LDS places: a loader's 16-byte pieces of its token, and a reader's 8 bytes; pieces of neighbouring tokens lie apart
  const int spread = 2 * (col & 3) + ((col >> 2) & 1);
  uint32_t put[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) put[i] = col * (2 * WV) + ((4 * half + i) ^ spread) * 16;
  const int rt = (lane & 15) >> 2, rc = lane & 3, rs = 2 * rt + half;
  const uint32_t get0 = (4 * half + rt) * (2 * WV) + ((2 * ((lane >> 4) & 1) + rc / 2) ^ rs) * 16 + (rc & 1) * 8;
  const uint32_t get1 = get0 ^ 64;

  while (x < end) {
    // -- the unit of iteration x --
    int b;
    {
      int lo = 0, hi = a.q.batch;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (plan.prefix[plan.base[mid]] * a.cache.heads <= x) lo = mid; else hi = mid;
      }
      b = lo;
    }
    const int t0 = plan.base[b], t1 = plan.base[b + 1];
    const int64_t p0 = plan.prefix[t0], span = plan.prefix[t1] - p0;
    const int64_t in = x - p0 * a.cache.heads;
    const int h = (in | span) >> 32 ? (int)(in / span) : (int)((uint32_t)in / (uint32_t)span);
    const int64_t rest = in - h * span;
    int tile;
    {
      int lo = t0, hi = t1;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (plan.prefix[mid] - p0 <= rest) lo = mid; else hi = mid;
      }
      tile = lo - t0;
    }
    const int64_t unit0 = x - (rest - (plan.prefix[t0 + tile] - p0)), unit1 = unit0 + plan.prefix[t0 + tile + 1] - plan.prefix[t0 + tile];
    const Sequence s = sequence(a, b);
    int lo, hi;
    tile_iterations(a, s, tile, A::kRows, A::kStep, lo, hi);
    const int it0 = (int)(x - unit0), it1 = (int)(min(unit1, end) - unit0);

    // -- the wave's query rows --
    const int rows = s.n * a.group;   // at most 2^30
    const int row0 = tile * A::kRows + rg * 32, row = min(row0 + col, rows - 1);
    const int i = row / a.group;
    int row_lo, row_hi;
    seen(a, s, i, row_lo, row_hi);
    // tokens [all_lo, all_hi) are seen by all of the wave's rows
    int all_lo, all_hi, unused;
    seen(a, s, min(row0, rows - 1) / a.group, unused, all_hi);
    seen(a, s, min(row0 + 31, rows - 1) / a.group, all_lo, unused);

    float m = kLowest, l = 0.f;   // the maximum is a whole number: every rescaling is exact
    v16f o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) {
#pragma unroll
      for (int n = 0; n < 16; ++n) o[d][n] = 0.f;
    }

    // -- loads: the lane's token of a step, its page a step ahead --
    const int32_t* table = a.q.table + (int64_t)b * a.q.columns;
    auto token_of = [&](int it) { return lo + (it * TG + tg) * 32 + col; };
    auto page_of = [&](int it) {
      const int t = token_of(it);
      return it < it1 && t < hi ? table[t >> a.page_shift] : -1;
    };
    uint4 kreg[KS], vreg[VO];
    uint32_t kscale[KW], vscale[VW];
    bool valid = false;
    auto load = [&](int it, int page) {
      valid = page >= 0 && page < a.cache.pages;
      const int64_t at = ((int64_t)(valid ? page : 0) * a.cache.heads + h << a.page_shift) + (token_of(it) & ((1 << a.page_shift) - 1));
      const uint8_t* p = a.cache.k_codes + at * (WK / 2) + 16 * half;
#pragma unroll
      for (int k = 0; k < KS; ++k) kreg[k] = mxd::ldg128(p + 32 * k);
#pragma unroll
      for (int w = 0; w < KW; ++w) kscale[w] = mxd::ldg32(a.cache.k_scales + at * scale_pitch(WK) + 4 * w);
      if constexpr (kApart) {
#pragma unroll
        for (int w = 0; w < VW; ++w) vscale[w] = mxd::ldg32(a.cache.v_scales + at * scale_pitch(WV) + 4 * w);
        const uint8_t* pv = a.cache.v_codes + at * (WV / 2) + 16 * half;
#pragma unroll
        for (int k = 0; k < VO; ++k)
          if (k * RG + rg < VS) vreg[k] = mxd::ldg128(pv + 32 * (k * RG + rg));
      }
    };
    load(it0, page_of(it0));
    int page_next = page_of(it0 + 1);

    v8i qh[KS], ql[KS];
    uint32_t qs[(KS + 1) / 2] = {};
    {
      // 64 values of a step, 2 x 16 a lane; the waves of a row group take turns and exchange what they made
      const uint16_t* q = a.q.q + (s.first + i) * a.q.q_stride + (int64_t)(h * a.group + row % a.group) * WK;
      uint4* made = (uint4*)lds + rg * (KS * 256) + lane;
      uint32_t* made_scales = (uint32_t*)(lds + RG * KS * 4096) + rg * (KS * 64) + lane;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        if (TG > 1 && k % TG != tg) continue;
        uint32_t w[2][8], top[2], high[8], low[8];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint4 v = mxd::ldg128((const uint8_t*)(q + 64 * k + 32 * e + 16 * half + 8 * j));
            w[e][4 * j] = v.x, w[e][4 * j + 1] = v.y, w[e][4 * j + 2] = v.z, w[e][4 * j + 3] = v.w;
          }
          top[e] = w[e][0] & 0x7FFF7FFFu;
#pragma unroll
          for (int j = 1; j < 8; ++j) top[e] = pair_max(top[e], w[e][j] & 0x7FFF7FFFu);
          top[e] = max(top[e] & 0xFFFFu, top[e] >> 16);
          top[e] = max(top[e], (uint32_t)__shfl_xor((int)top[e], 32, 64));
        }
        const uint32_t e0 = query_exponent(top[0]), e1 = query_exponent(top[1]), own = half ? e1 : e0;
        split16(w[0], min(e0, 247u), high, low);
        split16(w[1], min(e1, 247u), high + 4, low + 4);
        const uint32_t scales = own | (own == 255u ? 255u : own - 4u) << 8;
        if constexpr (TG > 1) {
          made[k * 256] = make_uint4(high[0], high[1], high[2], high[3]), made[k * 256 + 64] = make_uint4(high[4], high[5], high[6], high[7]);
          made[k * 256 + 128] = make_uint4(low[0], low[1], low[2], low[3]), made[k * 256 + 192] = make_uint4(low[4], low[5], low[6], low[7]);
          made_scales[k * 64] = scales;
        } else {
#pragma unroll
          for (int n = 0; n < 8; ++n) qh[k][n] = (int)high[n], ql[k][n] = (int)low[n];
          qs[k / 2] |= scales << (16 * (k & 1));
        }
      }
      if constexpr (TG > 1) {
        mxd::lds_barrier();
#pragma unroll
        for (int k = 0; k < KS; ++k) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint4 u = made[k * 256 + 64 * j], v = made[k * 256 + 128 + 64 * j];
            qh[k][4 * j] = (int)u.x, qh[k][4 * j + 1] = (int)u.y, qh[k][4 * j + 2] = (int)u.z, qh[k][4 * j + 3] = (int)u.w;
            ql[k][4 * j] = (int)v.x, ql[k][4 * j + 1] = (int)v.y, ql[k][4 * j + 2] = (int)v.z, ql[k][4 * j + 3] = (int)v.w;
          }
          qs[k / 2] |= made_scales[k * 64] << (16 * (k & 1));
        }
        mxd::lds_barrier();   // before the values come where they were
      }
      if constexpr (A::kWaves == 1) {
#pragma unroll
        for (int k = 0; k < KS; ++k) keep(qh[k]), keep(ql[k]);
      }
    }


    for (int it = it0; it < it1; ++it) {
      // -- scores --
      uint32_t bad = 0;
#pragma unroll
      for (int w = 0; w < (kApart ? VW : KW); ++w) {
        const uint32_t word = kApart ? vscale[w] : kscale[w];
        constexpr int used = (kApart ? WV : WK) / 32;
        bad |= marks(4 * w + 4 <= used ? word : word & ((1u << 8 * (used & 3)) - 1u));
      }
      const bool hide = bad || !valid;   // its values count as zero; who sees a NaN token sees it in the score
      uint32_t ks[KW];
#pragma unroll
      for (int w = 0; w < KW; ++w) ks[w] = kApart && bad ? ~0u : kscale[w] >> (8 * half);
      v16f sc;
#pragma unroll
      for (int n = 0; n < 16; ++n) sc[n] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        if (k & 1) {
          sc = scores<2, 2>(kreg[k], qh[k], sc, ks[k / 2], qs[k / 2]);
          sc = scores<2, 3>(kreg[k], ql[k], sc, ks[k / 2], qs[k / 2]);
        } else {
          sc = scores<0, 0>(kreg[k], qh[k], sc, ks[k / 2], qs[k / 2]);
          sc = scores<0, 1>(kreg[k], ql[k], sc, ks[k / 2], qs[k / 2]);
        }
      }
      // -- values to BF16 --
      const int turn = A::kBuffers > 1 ? it & 1 : 0;
      uint8_t* buffer = lds + turn * (TG * A::kTile);
#pragma unroll
      for (int k = 0; k < VO; ++k) {
        const int piece = k * RG + rg;   // columns [64 piece, + 64), the lane's half of them
        if (VO * RG > VS && piece >= VS) break;
        uint4 w;
        uint32_t word;
        if constexpr (kApart) {
          w = vreg[k];
          word = VW == 1 ? vscale[0] : vscale[piece / 2];
        } else {
          w = kreg[k * RG], word = kscale[k * RG / 2];
#pragma unroll
          for (int r = 1; r < RG; ++r)
            if (rg == r) w = kreg[k * RG + r], word = kscale[(k * RG + r) / 2];
        }
        const uint32_t e = word >> (8 * half + 16 * (piece & 1)) & 255u;
        const float scale = mx::u2f((hide ? 127u : e) << 23);
        const uint32_t u[4] = {hide ? 0u : w.x, hide ? 0u : w.y, hide ? 0u : w.z, hide ? 0u : w.w};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          uint4 v;
          v.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u[n], scale, 0));
          v.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u[n], scale, 1));
          v.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u[n], scale, 2));
          v.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u[n], scale, 3));
          *(uint4*)(buffer + tg * A::kTile + put[n] + 128 * piece) = v;
        }
      }
      const uint32_t shown = (uint32_t)__ballot(valid);
      const int first = lo + (it * TG + tg) * 32;
      load(it + 1, page_next);
      page_next = page_of(it + 2);
      // -- softmax --
      if (shown != ~0u || first < all_lo || first + 32 > all_hi) {
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          const int t = 8 * (n / 4) + 4 * half + (n & 3);
          if (!(shown >> t & 1) || first + t < row_lo || first + t >= row_hi) sc[n] = -INFINITY;
        }
      }
      float top = fmaxf(sc[0], sc[1]);
#pragma unroll
      for (int n = 2; n < 16; ++n) top = fmaxf(top, sc[n]);
      top = other_half_max(top) * a.c;
      // the maximum stays until it is 2^8 too low: probabilities up to 2^8 lose nothing
      float own = top > m + 8.f ? ceilf(top) : m;
      auto rescale = [&](float next) {
        const float by = power(m, next);
        m = next, l *= by;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
#pragma unroll
          for (int n = 0; n < 16; ++n) o[d][n] *= by;
        }
      };
      if constexpr (!kSplit)
        if (__any(own != m)) rescale(own);
      uint32_t p[8];
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const float p0_ = __builtin_amdgcn_exp2f(fmaf(sc[2 * n], a.c, -own)), p1_ = __builtin_amdgcn_exp2f(fmaf(sc[2 * n + 1], a.c, -own));
        sum += p0_ + p1_;
        p[n] = mxd::bf16_pair(p0_, p1_);
      }
      if constexpr (kSplit) {
        uint4* to = (uint4*)(exchange + ((it & 1) * 4 + wave) * 2048) + lane;
        to[0] = make_uint4(p[0], p[1], p[2], p[3]), to[64] = make_uint4(p[4], p[5], p[6], p[7]);
        if (half == 0) tops[it & 1][wave][col] = own;
      } else {
        l += sum;
      }
      if (RG > 1 || kSplit) mxd::lds_barrier();
      if constexpr (kSplit) {
        float next = own;
#pragma unroll
        for (int t = 1; t < TG; ++t) next = fmaxf(next, tops[it & 1][(tg + t) % TG * RG + rg][col]);
        if (__any(next != m)) rescale(next);
        l += sum * power(own, next);
      }
      // -- O^T += V^T P^T --
#pragma unroll
      for (int t = 0; t < (kSplit ? TG : 1); ++t) {
        if constexpr (kSplit) {
          const uint4* from = (const uint4*)(exchange + ((it & 1) * 4 + t * RG + rg) * 2048) + lane;
          const uint4 p0_ = from[0], p1_ = from[64];
          p[0] = p0_.x, p[1] = p0_.y, p[2] = p0_.z, p[3] = p0_.w, p[4] = p1_.x, p[5] = p1_.y, p[6] = p1_.z, p[7] = p1_.w;
          const float theirs = tops[it & 1][t * RG + rg][col];
          if (__any(theirs != m)) {   // whole powers of two: exact
            const float by = power(theirs, m);
#pragma unroll
            for (int n = 0; n < 8; ++n) p[n] = mxd::bf16_pair(mx::u2f(p[n] << 16) * by, mx::u2f(p[n] & 0xFFFF0000u) * by);
          }
        }
        const uint8_t* from = buffer + (kSplit ? t : tg) * A::kTile + (kSplit ? tg * (DB * 64) : 0);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const v8b pv = __builtin_bit_cast(v8b, make_uint4(p[4 * k], p[4 * k + 1], p[4 * k + 2], p[4 * k + 3]));
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            const uint8_t* at = from + (d & 1 ? get1 : get0) + 128 * (d / 2) + 16 * k * (2 * WV);
            typedef __attribute__((address_space(3))) v4s lds_v4s;
            v4s w[2];
            w[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at);
            w[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 8 * (2 * WV)));
            const v8b vv = __builtin_bit_cast(v8b, w);
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vv, pv, o[d], 0, 0, 0);
          }
        }
      }
      if (kSplit && A::kBuffers == 1) mxd::lds_barrier();
    }

    // -- the token groups' sums together, and out --
    l = halves_sum(l);
    if (half == 0) stats[wave][col][0] = m, stats[wave][col][1] = l;
    __syncthreads();   // and everybody has read its values
    const bool alone = x == unit0 && unit1 <= end;
    const int64_t slot = 2 * g + (g * per < unit0 ? 1 : 0);
    float most = kLowest, all_l = 0.f;
#pragma unroll
    for (int t = 0; t < TG; ++t) most = fmaxf(most, stats[t * RG + rg][col][0]);
#pragma unroll
    for (int t = 0; t < TG; ++t) all_l += stats[t * RG + rg][col][1] * power(stats[t * RG + rg][col][0], most);
    if (tg == 0 && half == 0) {
      const int r = rg * 32 + col;
      Place to{-1, 1.f};
      if (row0 + col < rows) {
        if (alone) {
          const int head = h * a.group + row % a.group;
          const int64_t token = s.first + i;
          const RowOut f = row_out(a, head, most, all_l);
          to = {token * a.q.out_stride + (int64_t)head * WV, f.inv};
          if (a.q.lse) a.q.lse[token * a.q.heads + head] = f.lse;
        } else {
          to.at = (slot * A::kRows + r) * WV;
          ((float2*)(a.space + a.at.stats))[slot * A::kRows + r] = make_float2(most, all_l);
        }
      }
      places[r] = to;
    }
    __syncthreads();
    float* part = (float*)(a.space + a.at.rows);
    auto put_out = [&](int r, int c, float4 v) {   // four columns of a row
      const Place to = places[r];
      if (to.at < 0) return;
      if (alone) {
        uint2 w;
        w.x = mxd::bf16_pair(v.x * to.by, v.y * to.by), w.y = mxd::bf16_pair(v.z * to.by, v.w * to.by);
        *(uint2*)(a.q.out + to.at + c) = w;
      } else {
        *(float4*)(part + to.at + c) = v;
      }
    };
    float* own_out = (float*)(lds + wave * A::kOut);
    const float by = power(m, most);
#pragma unroll
    for (int d0 = 0; d0 < DB; d0 += CB / 32) {
#pragma unroll
      for (int d = 0; d < CB / 32; ++d)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const v16f& v = o[d0 + d];
          *(float4*)(own_out + col * (CB + 4) + 32 * d + 8 * n + 4 * half) =
              make_float4(v[4 * n] * by, v[4 * n + 1] * by, v[4 * n + 2] * by, v[4 * n + 3] * by);
        }
      constexpr int L = CB / 4;   // lanes a row
      if constexpr (kSplit || TG == 1) {
        const int c = lane % L * 4;
#pragma unroll 4
        for (int r = lane / L; r < 32; r += 64 / L)
          put_out(rg * 32 + r, (kSplit ? tg * DB * 32 : 0) + d0 * 32 + c, *(const float4*)(own_out + r * (CB + 4) + c));
      } else {
        __syncthreads();
#pragma unroll 1
        for (int e = tid; e < A::kRows * L; e += 256) {
          const int r = e / L, c = e % L * 4;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int t = 0; t < TG; ++t) {
            const float4 w = *(const float4*)((const float*)(lds + (t * RG + r / 32) * A::kOut) + r % 32 * (CB + 4) + c);
            v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
          }
          put_out(r, d0 * 32 + c, v);
        }
        __syncthreads();
      }
    }
    __syncthreads();
    if (tid == 0 && unit1 >= end) {   // the workgroup's last: it joins the unit if it began it and does not end it
      Shared v{b, h, tile, 0};
      if (!alone && x == unit0) v.parts = (int)((unit1 - 1) / per - g + 1);
      v.slot = (int)(slot & 1);
      *shared = v;
    }
    x = min(unit1, end);
  }
}

// A unit that several workgroups had, four columns a thread: blockIdx.x the workgroup that began it.
template <int WV>
__global__ __launch_bounds__(256) void join_kernel(AttendArgs a, int tile_rows) {
  const Shared s = ((const Shared*)(a.space + a.at.units))[blockIdx.x];
  if (s.parts < 2) return;
  const int e = blockIdx.y * 256 + threadIdx.x, r = e / (WV / 4), c = e % (WV / 4) * 4;
  const Sequence q = sequence(a, s.b);
  const int row = s.tile * tile_rows + r;
  if (row >= q.n * a.group) return;
  const float2* stats = (const float2*)(a.space + a.at.stats);
  const float* parts = (const float*)(a.space + a.at.rows);
  // the others' first pieces of work
  auto slot = [&](int i) { return (int64_t)2 * (blockIdx.x + i) + (i ? 0 : s.slot); };
  float most = kLowest;
#pragma unroll 8
  for (int i = 0; i < s.parts; ++i) most = fmaxf(most, stats[slot(i) * tile_rows + r].x);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 8
  for (int i = 0; i < s.parts; ++i) {
    const float2 st = stats[slot(i) * tile_rows + r];
    const float4 p = *(const float4*)(parts + (slot(i) * tile_rows + r) * WV + c);
    const float by = power(st.x, most);
    sum += st.y * by;
    v.x += p.x * by, v.y += p.y * by, v.z += p.z * by, v.w += p.w * by;
  }
  const int head = s.h * a.group + row % a.group;
  const int64_t token = q.first + row / a.group;
  const RowOut f = row_out(a, head, most, sum);
  uint2 w;
  w.x = mxd::bf16_pair(v.x * f.inv, v.y * f.inv), w.y = mxd::bf16_pair(v.z * f.inv, v.w * f.inv);
  *(uint2*)(a.q.out + token * a.q.out_stride + (int64_t)head * WV + c) = w;
  if (a.q.lse && c == 0) a.q.lse[token * a.q.heads + head] = f.lse;
}

int check_attend(const char* who, const mx_kv4* c, int32_t heads, int32_t tokens, int32_t batch) {
  if (int s = check_cache(who, c)) return s;
  MX_REQUIRE(heads >= 1 && heads <= (1 << 16) && heads % c->heads == 0, "%s: %d query heads for %d key heads", who, heads, c->heads);
  MX_REQUIRE(tokens >= 0 && tokens <= kMaxTokens, "%s: token count %d outside [0, %d]", who, tokens, kMaxTokens);
  MX_REQUIRE(batch >= 0 && batch <= kMaxBatch, "%s: %d sequences outside [0, %d]", who, batch, kMaxBatch);
  MX_REQUIRE((int64_t)tokens * heads <= (1ll << 30), "%s: more than 2^30 query rows in all", who);
  return MX_OK;
}

// fn(WK, WV, apart) of a checked cache.
template <typename F>
auto by_widths(const mx_kv4* c, F fn) {
  using std::integral_constant;
  if (c->width == 512) return fn(integral_constant<int, 512>(), integral_constant<int, 512>(), std::false_type());
  if (c->width == 576) return fn(integral_constant<int, 576>(), integral_constant<int, 512>(), std::false_type());
  if (c->width == 64) return fn(integral_constant<int, 64>(), integral_constant<int, 64>(), std::true_type());
  if (c->width == 128) return fn(integral_constant<int, 128>(), integral_constant<int, 128>(), std::true_type());
  return fn(integral_constant<int, 256>(), integral_constant<int, 256>(), std::true_type());
}

int workgroups(int value_width) { return kCus * waves(value_width); }

// Row tiles of all sequences at most: each sequence's last one may be partly full.
int64_t most_tiles(int64_t rows, int batch, int tile_rows) { return rows / tile_rows + batch; }

Space space_of(const mx_kv4* c, int group, int tokens, int batch, int tile_rows) {
  const int64_t n = workgroups(c->value_width), tiles = most_tiles((int64_t)tokens * group, batch, tile_rows);
  auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  Space s;
  s.units = 0;
  s.stats = up(n * (int64_t)sizeof(Shared));
  s.rows = s.stats + up(2 * n * tile_rows * 8);
  s.base = s.rows + 2 * n * tile_rows * c->value_width * 4;
  s.prefix = s.base + up((batch + 1) * 4ll);
  s.total = s.prefix + up((tiles + 1) * 8);
  return s;
}

}  // namespace

using mxi::as_stream;
using mxi::use;

extern "C" {

uint64_t mx_kv4_workspace_bytes(mx_ctx* ctx, const mx_kv4* cache, int32_t heads, int32_t tokens, int32_t batch) {
  if (check_attend("mx_kv4_workspace_bytes", cache, heads, tokens, batch)) return 0;
  const int group = heads / cache->heads;
  int64_t most = 0;
  for (int rg = 1; rg <= 4; rg *= 2) most = std::max(most, space_of(cache, group, tokens, batch, 32 * rg).total);
  return (uint64_t)most;
}

int mx_kv4_attend(mx_ctx* ctx, const mx_kv4* cache, const mx_kv4_query* query, void* workspace, uint64_t workspace_bytes,
                  void* stream) {
  const char* who = "mx_kv4_attend";
  MX_REQUIRE(query, "%s: null query", who);
  const mx_kv4_query& q = *query;
  if (int s = check_attend(who, cache, q.heads, q.tokens, q.batch)) return s;
  MX_REQUIRE(q.columns >= 1 && (int64_t)q.columns * cache->page <= (1ll << 30), "%s: %d columns of pages of %d tokens", who, q.columns,
             cache->page);
  MX_REQUIRE(q.q_first || (q.batch ? q.tokens % q.batch == 0 : q.tokens == 0), "%s: %d rows do not divide among %d sequences", who,
             q.tokens, q.batch);
  MX_REQUIRE(q.window >= 0, "%s: window %d", who, q.window);
  MX_REQUIRE(q.scale > 0.f && q.scale <= 3.4e38f, "%s: scale must be finite and positive", who);
  MX_REQUIRE(q.q_stride >= (int64_t)q.heads * cache->width && q.q_stride % 8 == 0 && q.q_stride < (1ll << 40) &&
                 q.out_stride >= (int64_t)q.heads * cache->value_width && q.out_stride % 8 == 0 && q.out_stride < (1ll << 40),
             "%s: token strides must be multiples of 8 that hold the heads", who);
  if (q.tokens && q.batch) {
    MX_REQUIRE(q.q && q.out && q.table && q.lengths, "%s: null pointer", who);
    MX_REQUIRE(aligned(q.q, 16) && aligned(q.out, 16) && aligned(q.q_first, 4) && aligned(q.table, 4) && aligned(q.lengths, 4) &&
                   aligned(q.sinks, 4) && aligned(q.lse, 4),
               "%s: q and out must be 16-byte aligned, the others to their elements", who);
  }
  const uint64_t need = mx_kv4_workspace_bytes(ctx, cache, q.heads, q.tokens, q.batch);
  MX_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= need, "%s: %llu bytes of workspace, 16-byte aligned, needed", who,
             (unsigned long long)need);
  if (int s = use(ctx)) return s;
  if (!q.tokens || !q.batch) return MX_OK;
  AttendArgs a{};
  a.cache = *cache, a.q = q, a.group = q.heads / cache->heads, a.c = q.scale * kLog2e, a.space = (uint8_t*)workspace;
  while (1 << a.page_shift < cache->page) ++a.page_shift;
  // as many row groups as an average sequence's rows fill
  const int64_t rows = ((int64_t)q.tokens + q.batch - 1) / q.batch * a.group;
  const int rg = rows <= 32 ? 1 : rows <= 64 || !cache->v_codes ? 2 : 4, tile_rows = 32 * rg, step = 128 / rg;
  a.at = space_of(cache, a.group, q.tokens, q.batch, tile_rows);
  const int64_t tiles = most_tiles((int64_t)q.tokens * a.group, q.batch, tile_rows);
  a.tiles = (int)tiles;
  const bool inline_plan = tiles <= kInlineTiles;   // at least as many as sequences
  hipStream_t st = as_stream(stream);
  if (!inline_plan) {
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(1024), 0, st, a, tile_rows, step);
    MX_LAUNCH_CHECK("plan_kernel");
  }
  return by_widths(cache, [&](auto wk, auto wv, auto apart) {
    constexpr int WK = decltype(wk)::value, WV = decltype(wv)::value;
    constexpr bool kApart = decltype(apart)::value;
    const int n = workgroups(WV);
    const dim3 grid(n), threads(256);
    if (rg == 1) hipLaunchKernelGGL((attend_kernel<WK, WV, kApart, 1>), grid, threads, 0, st, a, (int)inline_plan);
    else if (rg == 2) hipLaunchKernelGGL((attend_kernel<WK, WV, kApart, 2>), grid, threads, 0, st, a, (int)inline_plan);
    if constexpr (kApart)
      if (rg == 4) hipLaunchKernelGGL((attend_kernel<WK, WV, kApart, 4>), grid, threads, 0, st, a, (int)inline_plan);
    MX_LAUNCH_CHECK("attend_kernel");
    hipLaunchKernelGGL(join_kernel<WV>, dim3(n, tile_rows * WV / 1024), threads, 0, st, a, tile_rows);
    MX_LAUNCH_CHECK("join_kernel");
    return MX_OK;
  });
}

}  // extern "C"
