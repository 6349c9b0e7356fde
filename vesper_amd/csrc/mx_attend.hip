// Attention over a paged cache in 4 bits (mx_kv4.hip), for single tokens, drafts and prompts.
//
// S = c q K^T over the tokens that a row sees, with the running maximum m and sum l of a softmax; O = P V / (l + sink).
//
// Rows are the heads of a key head and the tokens of a sequence, which share their keys: a row is one head of one token.
// Products are transposed: S^T = K Q^T has a query row in every lane, so that the softmax's maximum, sum and scaling need
// little exchange (between a wave's halves where the values are apart), and its registers are the right operand of
// O^T = V^T P^T as they are.
//   S^T: V_MFMA_SCALE_F32_32X32X64_F8F6F4 on the codes and scales as they lie in the cache, with the query as two E4M3
//        terms: a BF16 value has 8 significant bits, the first term takes 4 of them and the second, 2^-4 of its scale, the
//        rest, so the products are those of the BF16 query (to 2^-21 of a block's largest). At the rate of E4M3, two terms
//        cost what one BF16 product does, and the keys need no conversion. The instruction cuts each of eight neighbouring
//        products towards zero at 2^-13 of the largest power of two that two factors of one make, and adds those up exactly
//        (measured, bit for bit; a code of 0.5 counts as 1 there, a product of zero not at all; between eights it keeps 24
//        bits). So seven products lose up to 2^-12 of the largest each, in both terms 7 (1 + 2 2^-4) 2^-12 < 2^-9 of the
//        eights' largest products: no more than rounding the query's value to BF16 may have changed that product by. On normal
//        values logits are off by some 2^-19 of the sum of their products' magnitudes; with one channel of the query 100 times
//        its neighbours by 0.002 at most and 2e-4 on average (2-norm) where they are about 3 and the rounding of the query is
//        0.004, with it 1000 times by 0.05 and 0.004 of 22 (rounding 0.025).
//   O^T: V_MFMA_F32_32X32X16_BF16. A scale belongs to a token and 32 columns, but this product runs over the tokens, so
//        the values become BF16 (exactly: two significant bits and a power of two) by V_CVT_SCALEF32_PK_BF16_FP4, in the
//        row order in which they lie, and go through LDS, whose transposing reads give each lane its column's tokens.
//
// Work is divided evenly over the device. A unit is the row tile of one sequence and key head; it costs its iterations (a step
// of all the workgroup's token groups each) and kBegin more for its queries and its way out. Workgroup g takes the costs
// [g per, (g + 1) per) of all units in a row, or, where units are short, those whose costs begin there. Units that a workgroup
// has alone go straight to out; the others' parts go to the workspace and a second kernel adds them up.
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
constexpr int kInlineTiles = 1024;   // row tiles of all sequences that every workgroup counts for itself
// Where the plan is made: in the workspace by a launch of its own, in every workgroup's LDS, or, up to 64 tiles, in the
// registers of every wave.
constexpr int kInSpace = 0, kInLds = 1, kByWave = 2;
// What a unit's beginning and end cost, in iterations. With 3, 4, 5 and 6: the 48 sequences below 60.5, 59.8, 60.6 and 60.9 us,
// drafts over 576-wide latents 78.6, 78.4, 80.4 and 79.7, single tokens of grouped queries 74.8, 73.6, 73.0 and 73.2.
constexpr int kBegin = 4;
constexpr float kLowest = -3e38f;    // the maximum of a row that has seen nothing yet
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Byte offsets of the workspace.
struct Space {
  int64_t units, stats, rows, base, prefix, total;
};

// n / d for n below 2^31: with m = floor(2^(31 + s) / d) + 1, s = ceil(log2 d), n m exceeds n 2^(31 + s) / d by less than
// 2^(31 + s) / d.
struct Divide {
  uint32_t m, d;
  int shift;
  Divide() = default;
  explicit Divide(int by) : d(by) {
    int s = 0;
    while ((1ll << s) < by) ++s;
    shift = 31 + s, m = (uint32_t)((1ull << shift) / by + 1);
  }
  __device__ __forceinline__ int of(int n) const { return (int)((uint64_t)(uint32_t)n * m >> shift); }
  __device__ __forceinline__ int rest(int n) const { return n - of(n) * (int)d; }
};

struct AttendArgs {
  mx_kv4 cache;
  mx_kv4_query q;
  int group;           // query heads of a key head
  Divide by_group;
  int rows_each, tiles_each;   // query tokens and row tiles of a sequence, where all have as many
  Divide by_tiles;             // by the latter
  int page_shift;
  int tiles;           // row tiles of all sequences, at most
  bool whole;          // units stay whole: with the workgroup in whose costs they begin
  float c;             // scale log2(e)
  uint8_t* space;
  Space at;
};

// A workgroup's last unit, where the next workgroups go on with it: who adds it up, and over how many workgroups.
struct Shared {
  int32_t b, h, tile, parts, slot;
};

// (the library's minimum and maximum of 64-bit integers go through doubles)
__device__ __forceinline__ int64_t lesser(int64_t a, int64_t b) { return a < b ? a : b; }
__device__ __forceinline__ int64_t larger(int64_t a, int64_t b) { return a > b ? a : b; }

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
    s.n = a.rows_each, s.first = b * s.n;
  }
  const int length = a.q.lengths[b];
  s.end = length;
  s.held = (int)lesser(max(length, 0), (int64_t)a.q.columns << a.page_shift);
  return s;
}

// The tokens that query token i of the sequence sees.
__device__ __forceinline__ void seen(const AttendArgs& a, const Sequence& s, int i, int& lo, int& hi) {
  const int64_t end = s.end - s.n + i + 1;
  hi = (int)lesser(larger(end, 0), s.held);
  lo = a.q.window ? (int)lesser(larger(end - a.q.window, 0), hi) : 0;
}

// Tokens [lo, hi) that some row of row tile `tile` sees (lo at a whole step), and its iterations of `step` tokens: one at
// least, which writes the rows that see nothing.
__device__ __forceinline__ int tile_iterations(const AttendArgs& a, const Sequence& s, int tile, int rows, int step, int& lo, int& hi) {
  const int row0 = tile * rows, all = s.n * a.group;   // at most 2^30
  int l1, h0;
  seen(a, s, a.by_group.of(row0), lo, h0);
  seen(a, s, a.by_group.of(min(row0 + rows, all) - 1), l1, hi);
  lo &= ~31;
  return max(1, (hi - lo + step - 1) / step);
}

// The plan: base[b] = row tiles of the sequences before b (where they differ), prefix[i] = costs (of one key head) of the
// row tiles before i. Made by a workgroup of N threads in its LDS, or by plan_kernel in the workspace.
struct Plan {
  int32_t* base;
  int64_t* prefix;
};

// Sum of s over the wave's lanes up to this one.
__device__ __forceinline__ uint32_t wave_scan(uint32_t s) {
  s += __builtin_amdgcn_update_dpp(0, s, 0x111, 0xF, 0xF, false);   // within 16 lanes, from 1, 2, 4 and 8 before
  s += __builtin_amdgcn_update_dpp(0, s, 0x112, 0xF, 0xF, false);
  s += __builtin_amdgcn_update_dpp(0, s, 0x114, 0xF, 0xF, false);
  s += __builtin_amdgcn_update_dpp(0, s, 0x118, 0xF, 0xF, false);
  s += __builtin_amdgcn_update_dpp(0, s, 0x142, 0xA, 0xF, false);   // rows 1 and 3 from the last lane before them
  s += __builtin_amdgcn_update_dpp(0, s, 0x143, 0xC, 0xF, false);   // rows 2 and 3 from lane 31
  return s;
}
// Sum of v over the threads before this one, and over all N; v below 2^26.
template <int N>
__device__ __forceinline__ int64_t scan(uint32_t v, uint32_t* sums, int64_t& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t s = wave_scan(v);
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

// The last i in [0, n) for which at_most(i), which 0 is and none after one that is not: by a thread, and by a wave, which
// looks at 64 at a time.
template <typename T>
__device__ __forceinline__ int find(int n, T at_most) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (at_most(mid)) lo = mid; else hi = mid;
  }
  return lo;
}
template <typename T>
__device__ __forceinline__ int find_by_wave(int n, T at_most) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, i = lo + (int)(threadIdx.x & 63) * step;
    lo += (__popcll(__ballot(i < hi && at_most(min(i, n - 1)))) - 1) * step;
    hi = min(lo + step, hi);
  }
  return lo;
}

template <int N>
__device__ __forceinline__ void make_plan(const AttendArgs& a, Plan p, uint32_t* sums, int rows, int step) {
  int64_t tiles = (int64_t)a.q.batch * a.tiles_each, all;
  const bool each = !a.q.q_first;
  if (!each) {
    for (int b0 = 0; b0 < a.q.batch; b0 += N) {
      const int b = b0 + threadIdx.x;
      uint32_t n = 0;
      if (b < a.q.batch) n = (uint32_t)(((int64_t)sequence(a, b).n * a.group + rows - 1) / rows);
      const int64_t before = scan<N>(n, sums, all);
      // (no more than there is room for: a q_first that does not ascend could name more rows than there are)
      if (b < a.q.batch) p.base[b] = (int)lesser(tiles + before, a.tiles);
      tiles += all;
    }
    tiles = lesser(tiles, a.tiles);
    if (threadIdx.x == 0) p.base[a.q.batch] = (int)tiles;
    __syncthreads();
  }
  int64_t sum = 0;
  for (int i0 = 0; i0 < tiles; i0 += N) {
    const int i = i0 + threadIdx.x;
    uint32_t n = 0;
    if (i < tiles) {
      const int b = each ? a.by_tiles.of(i) : find(a.q.batch, [&](int k) { return p.base[k] <= i; });
      int lo, hi;
      n = kBegin + tile_iterations(a, sequence(a, b), each ? a.by_tiles.rest(i) : i - p.base[b], rows, step, lo, hi);
    }
    const int64_t before = scan<N>(n, sums, all);
    if (i < tiles) p.prefix[i] = sum + before;
    sum += all;
  }
  if (threadIdx.x == 0) p.prefix[tiles] = sum;
  __syncthreads();
}

__global__ __launch_bounds__(1024) void plan_kernel(AttendArgs a, int rows, int step) {
  __shared__ uint32_t sums[16];
  make_plan<1024>(a, {(int32_t*)(a.space + a.at.base), (int64_t*)(a.space + a.at.prefix)}, sums, rows, step);
}

// What every lane holds, in scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}
__device__ __forceinline__ Sequence uniform(Sequence s) {
  s.first = uniform(s.first), s.n = uniform(s.n), s.held = uniform(s.held), s.end = uniform(s.end);
  return s;
}

// A workgroup's way through the units, in the order key head, sequence, row tile.
struct Units {
  int64_t x, end;           // the costs that are the workgroup's, from x on
  int b, h, tile, tiles;    // the unit, and row tiles of its sequence
  Sequence s;
  int lo, hi;               // the tokens that its rows see
  int64_t unit0;            // its costs begin here
  int n, it0, it1;          // its iterations, and the workgroup's of them
  bool first;               // nothing came before it in this workgroup
};

__device__ __forceinline__ void share(const AttendArgs& a, Units& u) {
  if (a.whole) {
    u.it0 = u.unit0 < u.x ? u.n : 0, u.it1 = u.n;
  } else {
    u.it0 = (int)larger(u.x - u.unit0 - kBegin, 0), u.it1 = (int)lesser(u.end - u.unit0 - kBegin, u.n);
  }
}
__device__ __forceinline__ void enter(const AttendArgs& a, Units& u, int rows, int step) {
  u.n = uniform(tile_iterations(a, u.s, u.tile, rows, step, u.lo, u.hi));
  u.lo = uniform(u.lo), u.hi = uniform(u.hi);
  share(a, u);
}

__device__ __forceinline__ int tiles_of(const AttendArgs& a, const Sequence& s, int rows) {
  return (int)(((int64_t)s.n * a.group + rows - 1) / rows);
}

__device__ __forceinline__ void next_unit(const AttendArgs& a, Units& u, int rows, int step) {
  u.first &= u.it1 <= u.it0;
  u.x = u.unit0 = u.unit0 + kBegin + u.n;
  if (u.x >= u.end) return;
  if (++u.tile == u.tiles) {
    u.tile = 0;
    do {   // (there is another, since costs are left, unless somebody changes the sequences meanwhile)
      if (++u.b == a.q.batch) {
        u.b = 0;
        if (++u.h == a.cache.heads) {
          u.x = u.end;
          return;
        }
      }
      u.s = uniform(sequence(a, u.b));
      u.tiles = tiles_of(a, u.s, rows);
    } while (u.tiles == 0);
  }
  enter(a, u, rows, step);
}

// in / span, which is below 2^16: the quotient in FP32 is within 1 of it.
__device__ __forceinline__ int few(int64_t in, int64_t span) {
  int q = (int)((float)in / (float)span);
  q -= q * span > in;
  q += (q + 1) * span <= in;
  return q;
}

// Workgroup g's share of the units: where it begins. By each thread of N its share of an LDS plan (found: two words), else
// by each wave. Whether there is anything.
template <int N>
__device__ __forceinline__ bool first_unit(const AttendArgs& a, const Plan& p, bool in_lds, int g, int64_t& per, int groups, int32_t* found,
                                           Units& u, int rows, int step) {
  const bool each = !a.q.q_first;
  const int tiles = each ? a.q.batch * a.tiles_each : uniform(p.base[a.q.batch]);
  const int64_t total = uniform(p.prefix[tiles]), all = total * a.cache.heads;
  per = larger((all + groups - 1) / groups, 1);
  u.x = lesser(g * per, all), u.end = lesser(u.x + per, all), u.first = true;
  if (u.x >= u.end) return false;
  u.h = a.cache.heads > 1 ? uniform(few(u.x, total)) : 0;
  const int64_t before = u.h * total, rest = u.x - before;
  int t;
  if (in_lds) {
    for (int i = threadIdx.x; i < tiles; i += N)
      if (p.prefix[i] <= rest && rest < p.prefix[i + 1]) found[0] = i;
    __syncthreads();
    t = uniform(found[0]);
    if (!each) {
      for (int b = threadIdx.x; b < a.q.batch; b += N)
        if (p.base[b] <= t && t < p.base[b + 1]) found[1] = b;
      __syncthreads();
    }
    u.b = each ? a.by_tiles.of(t) : uniform(found[1]);
  } else {
    t = uniform(find_by_wave(tiles, [&](int i) { return p.prefix[i] <= rest; }));
    u.b = each ? a.by_tiles.of(t) : uniform(find_by_wave(a.q.batch, [&](int b) { return p.base[b] <= t; }));
  }
  u.s = uniform(sequence(a, u.b));
  u.tiles = tiles_of(a, u.s, rows);
  u.tile = t - (each ? u.b * a.tiles_each : uniform(p.base[u.b]));
  if (u.tile >= u.tiles) return false;   // (somebody has changed the sequences meanwhile: it may have no row left to read)
  u.unit0 = before + uniform(p.prefix[t]);
  enter(a, u, rows, step);
  return true;
}

// The same for at most 64 row tiles, one a lane, by every wave for itself: without LDS and barriers, which saves 0.8 to 0.9 us
// of a call (16 x 1000 tokens of 8 key heads 17.9 to 17.0, one session of latents over 4099 19.5 to 18.7).
__device__ __forceinline__ bool first_of_few(const AttendArgs& a, int g, int64_t& per, int groups, Units& u, int rows, int step) {
  const int lane = threadIdx.x & 63;
  int b, tile, tiles;
  if (!a.q.q_first) {
    tiles = a.q.batch * a.tiles_each;
    b = a.by_tiles.of(min(lane, tiles - 1)), tile = a.by_tiles.rest(lane);
  } else {
    const uint32_t own = lane < a.q.batch ? tiles_of(a, sequence(a, lane), rows) : 0, upto = wave_scan(own);
    tiles = (int)min((uint32_t)__builtin_amdgcn_readlane(upto, 63), (uint32_t)a.tiles);
    b = 0;   // the last sequence that begins at or before the lane's tile
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) {
      const int begin = __shfl((int)(upto - own), min(b + s, 63), 64);
      b += b + s < a.q.batch && begin <= lane ? s : 0;
    }
    tile = lane - __shfl((int)(upto - own), b, 64);
  }
  if (tiles == 0) return false;
  Sequence s{};
  int lo = 0, hi = 0;
  uint32_t n = 0;
  if (lane < tiles) {
    s = sequence(a, b);
    n = kBegin + tile_iterations(a, s, tile, rows, step, lo, hi);
  }
  const uint32_t upto = wave_scan(n);
  const int64_t total = (uint32_t)__builtin_amdgcn_readlane(upto, 63), all = total * a.cache.heads;
  per = larger((all + groups - 1) / groups, 1);
  u.x = lesser(g * per, all), u.end = lesser(u.x + per, all), u.first = true;
  if (u.x >= u.end) return false;
  u.h = a.cache.heads > 1 ? uniform(few(u.x, total)) : 0;
  const int64_t before = u.h * total, rest = u.x - before;
  const int at = __builtin_ctzll(__ballot(upto > rest));
  auto of = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
  u.b = of(b), u.tile = of(tile), u.n = of((int)n) - kBegin, u.lo = of(lo), u.hi = of(hi);
  u.s.first = of(s.first), u.s.n = of(s.n), u.s.held = of(s.held);
  u.s.end = (int64_t)((uint64_t)(uint32_t)of((int)(s.end >> 32)) << 32 | (uint32_t)of((int)s.end));
  u.tiles = tiles_of(a, u.s, rows);
  if (u.tile >= u.tiles) return false;   // (as above)
  u.unit0 = before + (uint32_t)of((int)upto) - (u.n + kBegin);
  share(a, u);
  return true;
}

// The unit's end in this workgroup: `alone` it has all of it. The workgroup's last unit, if it began it and does not end it,
// is joined from there on.
__device__ __forceinline__ bool is_alone(const Units& u) { return u.it0 == 0 && u.it1 == u.n; }
__device__ __forceinline__ void note(const Units& u, int64_t per, int g, int groups, Shared* shared) {
  Shared v{u.b, u.h, u.tile, 0, u.first ? 0 : 1};
  const int64_t end = u.unit0 + kBegin + u.n;
  if (u.it0 == 0 && u.it1 > 0 && u.it1 < u.n) v.parts = min(few(end - 1, per), groups - 1) - g + 1;
  *shared = v;
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

// Query values of a step as the right operand of the scores' products: a lane's 2 x 16 in two terms, and their scale bytes.
// 32x32x64: the lane's row is lane % 32, the 16s from 16 half and 32 + 16 half on; 16x16x128: lane % 16, from 16 quad and
// 64 + 16 quad on. A lane gives the scales of block half (quad) of 32, not those of the values it holds.
struct QueryStep {
  uint32_t high[8], low[8], scales;
};
struct QueryWords {
  uint32_t w[2][8];
};

template <int kApart = 64>
__device__ __forceinline__ QueryWords query_words(const uint16_t* q, bool first_only = false) {
  QueryWords r;
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (e == 0 || !first_only) v = mxd::ldg128((const uint8_t*)(q + kApart * e + 8 * j));
      r.w[e][4 * j] = v.x, r.w[e][4 * j + 1] = v.y, r.w[e][4 * j + 2] = v.z, r.w[e][4 * j + 3] = v.w;
    }
  return r;
}

__device__ __forceinline__ uint32_t largest(const uint32_t (&w)[8]) {
  uint32_t top = w[0] & 0x7FFF7FFFu;
#pragma unroll
  for (int j = 1; j < 8; ++j) top = pair_max(top, w[j] & 0x7FFF7FFFu);
  return max(top & 0xFFFFu, top >> 16);
}
__device__ __forceinline__ uint32_t scale_bytes(uint32_t e) { return e | (e == 255u ? 255u : e - 4u) << 8; }

__device__ __forceinline__ QueryStep query_step(const QueryWords& q, int half) {
  QueryStep r;
  uint32_t e[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t top = largest(q.w[i]);
    const auto both = __builtin_amdgcn_permlane32_swap(top, top, false, false);
    e[i] = query_exponent(max((uint32_t)both[0], (uint32_t)both[1]));
    split16(q.w[i], min(e[i], 247u), r.high + 4 * i, r.low + 4 * i);
  }
  r.scales = scale_bytes(half ? e[1] : e[0]);
  return r;
}

__device__ __forceinline__ QueryStep query_step16(const QueryWords& q, int l16, int quad) {
  QueryStep r;
  uint32_t e[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {   // blocks quad / 2 and 2 + quad / 2, halved between quads
    const uint32_t top = largest(q.w[i]);
    const auto both = __builtin_amdgcn_permlane16_swap(top, top, false, false);
    e[i] = query_exponent(max((uint32_t)both[0], (uint32_t)both[1]));
    split16(q.w[i], min(e[i], 247u), r.high + 4 * i, r.low + 4 * i);
  }
  const int from = (quad & 1) * 32 + l16;   // a lane of block `quad`
  const uint32_t e0 = (uint32_t)__shfl((int)e[0], from, 64), e1 = (uint32_t)__shfl((int)e[1], from, 64);
  r.scales = scale_bytes(quad < 2 ? e0 : e1);
  return r;
}

// 16 bytes at any multiple of 4.
__device__ __forceinline__ uint4 words4(const uint8_t* p) {
  typedef mxd::u32x4_t words __attribute__((aligned(4)));
  const words v = *(const __attribute__((address_space(1))) words*)p;
  return make_uint4(v.x, v.y, v.z, v.w);
}

// Where a row of a unit goes (in values; -1: nowhere), and its factor.
struct Place {
  int64_t at;
  float by;
};

// The maximum m with a step's largest logit: the logit itself at first, so that one token alone has probability 1. After that
// it stays until it is 2^8 too low (probabilities up to 2^8 lose nothing) and is raised by whole numbers, which scale
// what is in BF16 exactly.
__device__ __forceinline__ float raised(float m, float top) {
  return top > m + 8.f ? (m == kLowest ? top : m + ceilf(top - m)) : m;
}

// A maximum so far from zero that FP32 holds it to whole numbers only: c s - m, rounded once, would not be about zero where s
// is the largest logit (its power overflows from 2^31 on). There c s is rounded by itself, as m is.
__device__ __forceinline__ bool far_off(float m) { return fabsf(m) >= 0x1p24f && m != kLowest; }
// What a step's largest logit has to pass for the maximum to be looked at: anything, where it is far off.
__device__ __forceinline__ float bar_of(float m) { return far_off(m) ? -INFINITY : m + 8.f; }

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

// Latents. A step is 64 tokens, for 64 (RG = 2) or 32 rows, of eight waves, two a SIMD:
//   four score waves: 16 rows and 64 (32) tokens each, by V_MFMA_SCALE_F32_16X16X128_F8F6F4 with the rows' queries in 64
//     registers; and the softmax of these, 16 tokens' beside the next ones' scores, under the maximum so far (drafts over
//     576-wide latents 78.6 us, with all scores first 82.9), and the probabilities to LDS;
//   four value waves: 128 columns and all rows each. Each converts its columns of the step's tokens into an LDS tile of its
//     own, between the products of the last step's values with the last step's probabilities.
// So the matrix units have a score wave's and a value wave's products to choose from, and each wave's other instructions go
// on under the other's products; one barrier a step. Codes and scales come to LDS by copies that nobody waits for, kStages -
// 1 steps ahead, once for all waves.
//
// A workgroup's first queries are converted by all eight waves, later units' by the score waves while the value waves finish
// the unit before; its first copies are asked for before its last products.
//
// Measured at 64 heads of 512 over 48 sequences of 200 to 30,000 tokens (86 MB, 39 GFLOP): 57 us and 10 us for the joining,
// 680 TFLOP/s in the first. A step takes about 3,500 clocks, its products 2,048 of a SIMD's and its LDS traffic about 1,950; a
// workgroup has its first queries after about 17,000 (5,500 for the division, the rest the queries, from the caches beside
// the first copies), and its way out takes 5,000. Before the roles were parted, with eight waves that all scored and
// multiplied, both took 120 us. Not faster: priorities for either role (61 to 63 us for both kernels in place of 61), all of a
// unit's first copies before the rows of the one before go out (windows of 128 over prompts 124 us in place of 122).
constexpr int kLatentStep = 64;
template <int WK, int RG>
struct Latent {
  static constexpr int WV = 512, RQ = 2 * RG, TT = 4 / RQ, T2 = 4 / TT, kRows = 32 * RG, kStep = kLatentStep;
  static constexpr bool kPart = WK % 128 != 0;             // a last step of 64 columns of the keys
  static constexpr int KS = (WK + 127) / 128;
  static constexpr int kStages = kPart ? 3 : 4;
  // LDS: the values' tiles [4 waves][64 tokens][128 columns], the step's probabilities by 16 tokens, twice, and the stages:
  // codes [64][256 B], scales [64][16 B], and of a last step codes [64][32 B] and scales [64][4 B]
  static constexpr int kTile = 64 * 256, kValues = 4 * kTile;
  static constexpr int kWeights = 4 * kRows * 32;
  static constexpr int kScales = 64 * 256, kTail = kScales + 64 * 16, kTailScales = kTail + 64 * 32;
  static constexpr int kStage = kPart ? kTailScales + 64 * 4 : kTail;
  static constexpr int kRing = kValues + 2 * kWeights, kLds = kRing + kStages * kStage;
  static constexpr int kCopies = kPart ? 7 : 5;            // of a value wave and step
  // the first queries' exchange, over the tiles and probabilities
  static constexpr int kMade = 4 * 256 + (kPart ? 128 : 0);
  static_assert(RQ * (kMade * 16 + KS * 256) <= kRing, "the queries lie before the stages");
  static_assert(8 * (kInlineTiles + 1) + 4 * (kInlineTiles + 2) <= kRing, "and so does the plan");
};

template <int kA, int kB>
__device__ __forceinline__ mxd::v4f scores16(uint4 k, const v8i& q, mxd::v4f c, uint32_t ks, uint32_t qs) {
  const v8i av = {(int)k.x, (int)k.y, (int)k.z, (int)k.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, q, c, 4, 0, kA, (int)ks, kB, (int)qs);
}
// Step K of the scores, both terms.
template <int K>
__device__ __forceinline__ mxd::v4f score_step(uint4 k, const v8i& high, const v8i& low, mxd::v4f c, uint32_t ks, uint32_t qs) {
  c = scores16<K & 3, 2 * (K & 1)>(k, high, c, ks, qs);
  return scores16<K & 3, 2 * (K & 1) + 1>(k, low, c, ks, qs);
}

// Over the four lanes of a row (lane % 16).
__device__ __forceinline__ float row_max4(float v) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
  return other_half_max(fmaxf(__int_as_float(p[0]), __int_as_float(p[1])));
}
__device__ __forceinline__ float row_sum4(float v) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
  return halves_sum(__int_as_float(p[0]) + __int_as_float(p[1]));
}

template <int WK, int RG>
__global__ __launch_bounds__(512, 2) void latent_kernel(AttendArgs a, int by) {
  using A = Latent<WK, RG>;
  constexpr int WV = A::WV, RQ = A::RQ, TT = A::TT, T2 = A::T2, KS = A::KS;
  constexpr bool kPart = A::kPart;
  __shared__ __attribute__((aligned(16))) uint8_t lds[A::kLds];
  __shared__ float tops[2][A::kRows][TT];
  __shared__ float stats[A::kRows][TT][2];
  __shared__ Place places[A::kRows];
  __shared__ uint32_t sums[8];
  __shared__ int32_t found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, quad = lane >> 4, col = lane & 31, half = lane >> 5;
  const int rq = wave % RQ, tt = wave % 4 / RQ;   // a score wave's 16 rows and tokens
  const int cg = wave - 4;                        // a value wave's columns
  uint8_t* weights = lds + A::kValues;

  Plan plan{(int32_t*)(a.space + a.at.base), (int64_t*)(a.space + a.at.prefix)};
  if (by == kInLds) {
    plan = {(int32_t*)(lds + 8 * (kInlineTiles + 1)), (int64_t*)lds};
    make_plan<512>(a, plan, sums, A::kRows, A::kStep);
  }
  // workgroups go round the XCDs: neighbours in the work, which share keys, to one L2
  const int g = (int)(blockIdx.x % kXcds) * (kCus / kXcds) + (int)blockIdx.x / kXcds;
  Shared* shared = (Shared*)(a.space + a.at.units) + g;
  if (tid == 0) shared->parts = 0;
  int64_t per;
  Units u;
  if (!(by == kByWave ? first_of_few(a, g, per, kCus, u, A::kRows, A::kStep)
                      : first_unit<512>(a, plan, by == kInLds, g, per, kCus, found, u, A::kRows, A::kStep)))
    return;

  const int spread = 2 * (l16 & 3) + ((l16 >> 2) & 1);   // pieces of 16 bytes of neighbouring tokens' values lie apart
  // To the next unit of which iterations are this workgroup's, from `ahead` units on: whether there is one. Every wave goes
  // its own way through the same units.
  auto go_on = [&](int ahead) {
    for (;; ahead = 1) {
      if (ahead) {
        if (u.end <= u.unit0 + kBegin + u.n && tid == 0) note(u, per, g, kCus, shared);
        next_unit(a, u, A::kRows, A::kStep);
        if (u.x >= u.end) return false;
      }
      if (u.it1 > u.it0) return true;
    }
  };
  if (!go_on(0)) return;
  // -- pages: 16 tokens have one --
  typedef const __attribute__((address_space(4))) int32_t Entry;
  auto table_of = [&] { return (Entry*)(a.q.table + (int64_t)u.b * a.q.columns); };
  auto entry_of = [&](Entry* table, int hi, int t) { return table[min(t, max(hi - 1, 0)) >> a.page_shift]; };
  auto is_there = [&](int hi, int t, int entry) { return t < hi && (uint32_t)entry < (uint32_t)a.cache.pages; };
  // a step's four entries are asked for a step before they are looked at, so that nobody waits for them; bit t: 16 tokens
  int entries[4];
  auto ask = [&](Entry* table, int lo, int hi, int it) {
#pragma unroll
    for (int t = 0; t < 4; ++t) entries[t] = entry_of(table, hi, lo + it * A::kStep + 16 * t);
  };
  auto shown_of = [&](int lo, int hi, int it) {
    uint32_t shown = 0;
#pragma unroll
    for (int t = 0; t < 4; ++t) shown |= is_there(hi, lo + it * A::kStep + 16 * t, entries[t]) ? 1u << t : 0u;
    return shown;
  };
  // -- a value wave's copies of step `it`: its 16 tokens, on page `entry` --
  auto copy = [&](int h, int lo, int hi, int it, int entry) {
    const int t = lo + it * A::kStep + 16 * cg, page = is_there(hi, t, entry) ? entry : 0;
    const int64_t at = (((int64_t)page * a.cache.heads + h) << a.page_shift) + (t & ((1 << a.page_shift) - 1));
    const uint8_t* codes = a.cache.k_codes + at * (WK / 2);
    const uint8_t* scales = a.cache.k_scales + at * scale_pitch(WK);
    auto stage = [&](int at) { return (uint32_t)uniform((int)(mxd::lds_addr(lds) + A::kRing + (it % A::kStages) * A::kStage) + at); };
#pragma unroll
    for (int j = 0; j < 4; ++j) {   // four tokens, their pieces changed about by the token
      const uint32_t token = 4 * j + quad, piece = l16 ^ (token & 7);
      mxd::global_to_lds16(codes + (token * (WK / 2) + piece * 16), stage((16 * cg + 4 * j) * 256));
    }
    if (lane < 16) mxd::global_to_lds16(scales + lane * scale_pitch(WK), stage(A::kScales + 256 * cg));
    if constexpr (kPart) {
      if (lane < 32) mxd::global_to_lds16(codes + ((lane >> 1) * (WK / 2) + 256 + (lane & 1) * 16), stage(A::kTail + 512 * cg));
      if (lane < 16) mxd::global_to_lds4(scales + lane * scale_pitch(WK) + 16, stage(A::kTailScales + 64 * cg));
    }
  };
  auto begin = [&] {   // a unit's first step, asked for while the unit before ends
    copy(u.h, u.lo, u.hi, u.it0, entry_of(table_of(), u.hi, u.lo + u.it0 * A::kStep + 16 * cg));
  };
  auto query_row = [&] {   // a lane's, of the 16 of row quarter rq
    const int row = min(u.tile * A::kRows + rq * 16 + l16, u.s.n * a.group - 1);
    return a.q.q + (u.s.first + a.by_group.of(row)) * a.q.q_stride + (int64_t)(u.h * a.group + a.by_group.rest(row)) * WK + 16 * quad;
  };
  // -- the first unit's queries, KS steps of 128 values, converted by the rows' 8 / RQ waves together and exchanged --
  uint4* const made = (uint4*)lds + rq * A::kMade + lane;
  uint32_t* const made_scales = (uint32_t*)(lds + RQ * A::kMade * 16) + rq * (KS * 64) + lane;
  {
    constexpr int kSharers = 8 / RQ, kEach = (KS + kSharers - 1) / kSharers;
    const int sharer = wave / RQ;
    const uint16_t* q = query_row();
    QueryWords words[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int k = e * kSharers + sharer;
      if (KS % kSharers == 0 || k < KS) words[e] = query_words(q + 128 * k, kPart && k == KS - 1);
    }
    if (wave >= 4) begin();
    if (by == kInLds) __syncthreads();   // the plan has been read
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int k = e * kSharers + sharer;
      if (KS % kSharers && k >= KS) break;
      const QueryStep s = query_step16(words[e], l16, quad);
      made[k * 256] = make_uint4(s.high[0], s.high[1], s.high[2], s.high[3]);
      const int low = kPart && k == 4 ? 64 : 128;   // a last step has nothing in its second halves
      made[k * 256 + low] = make_uint4(s.low[0], s.low[1], s.low[2], s.low[3]);
      if (!kPart || k < 4) {
        made[k * 256 + 64] = make_uint4(s.high[4], s.high[5], s.high[6], s.high[7]);
        made[k * 256 + 192] = make_uint4(s.low[4], s.low[5], s.low[6], s.low[7]);
      }
      made_scales[k * 64] = s.scales;
    }
  }
  if (wave < 4) {
    // -- further units': by the score waves, asked for while the unit before ends, where the registers hold them --
    constexpr bool kAhead = !kPart;
    QueryWords words[KS];
    auto load = [&] {
      const uint16_t* q = query_row();
#pragma unroll
      for (int k = 0; k < KS; ++k) words[k] = query_words(q + 128 * k, kPart && k == KS - 1);
    };
    bool exchanged = true;
    mxd::lds_barrier();
    for (;;) {
      const int it0 = u.it0, it1 = u.it1, lo = u.lo, hi = u.hi;
      Entry* const table = table_of();
      const bool alone = is_alone(u);
      const int64_t slot = 2 * g + (u.first ? 0 : 1);
      ask(table, lo, hi, it0);
      uint32_t shown = shown_of(lo, hi, it0);
      const int h = u.h, first_token = u.s.first, rows = u.s.n * a.group, row0 = u.tile * A::kRows;   // rows at most 2^30
      v8i qh[KS], ql[KS];
      uint32_t qs[(KS + 1) / 2] = {};
      if (exchanged) {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const bool last = kPart && k == 4;
          const uint4 h0 = made[k * 256], l0 = made[k * 256 + (last ? 64 : 128)];
          const uint4 h1 = last ? make_uint4(0u, 0u, 0u, 0u) : made[k * 256 + 64], l1 = last ? make_uint4(0u, 0u, 0u, 0u) : made[k * 256 + 192];
          qh[k] = {(int)h0.x, (int)h0.y, (int)h0.z, (int)h0.w, (int)h1.x, (int)h1.y, (int)h1.z, (int)h1.w};
          ql[k] = {(int)l0.x, (int)l0.y, (int)l0.z, (int)l0.w, (int)l1.x, (int)l1.y, (int)l1.z, (int)l1.w};
          qs[k / 2] |= made_scales[k * 64] << (16 * (k & 1));
        }
      } else {
        if (!kAhead) load();
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const QueryStep s = query_step16(words[k], l16, quad);
#pragma unroll
          for (int n = 0; n < 8; ++n) qh[k][n] = (int)s.high[n], ql[k][n] = (int)s.low[n];
          qs[k / 2] |= s.scales << (16 * (k & 1));
        }
      }
      exchanged = false;
      int row_lo, row_hi;
      seen(a, u.s, a.by_group.of(min(row0 + rq * 16 + l16, rows - 1)), row_lo, row_hi);
      // tokens [all_lo, all_hi) are seen by all of the wave's rows
      int all_lo, all_hi, unused;
      seen(a, u.s, a.by_group.of(min(row0 + rq * 16, rows - 1)), unused, all_hi);
      seen(a, u.s, a.by_group.of(min(row0 + rq * 16 + 15, rows - 1)), all_lo, unused);
      all_lo = uniform(all_lo), all_hi = uniform(all_hi);
      const uint32_t get_k = tt * T2 * 4096 + l16 * 256 + ((quad ^ (l16 & 7)) * 16);
      // probabilities: [16 tokens][row][half][8 tokens of it], as the products take them
      uint8_t* const put_w = weights + (tt * T2 * A::kRows + rq * 16 + l16) * 32 + (quad & 1) * 16 + (quad >> 1) * 8;
      float m = kLowest, l = 0.f;
      float own = kLowest, sum = 0.f;
      bool far = false;   // one of the wave's maxima is far off
      mxd::copy_barrier();   // the first step is there, and exchanged queries have been read
      for (int it = it0; it < it1; ++it) {
        const uint8_t* stage = lds + A::kRing + (it % A::kStages) * A::kStage;
        const int first = lo + it * A::kStep + tt * T2 * 16;
        ask(table, lo, hi, it + 1);
        mxd::v4f sc[T2];
        uint32_t ks[T2], klast[T2];
#pragma unroll
        for (int t = 0; t < T2; ++t) {
          const uint4 w = *(const uint4*)(stage + A::kScales + (tt * T2 + t) * 256 + l16 * 16);
          const uint32_t pick = 0x0C0C0400u + 0x0101u * quad;   // byte `quad` of the four words
          ks[t] = __builtin_amdgcn_perm(w.y, w.x, pick) | __builtin_amdgcn_perm(w.w, w.z, pick) << 16;
          sc[t] = {0.f, 0.f, 0.f, 0.f};
          if constexpr (kPart) {
            const uint32_t v = *(const uint32_t*)(stage + A::kTailScales + ((tt * T2 + t) * 16 + l16) * 4);
            klast[t] = quad > 1 ? 127u : v >> (8 * quad);
          }
        }
        auto codes = [&](int k, int t) { return *(const uint4*)(stage + (get_k ^ (k & 1 ? 64 : 0)) + 128 * (k >> 1) + 4096 * t); };
        auto score = [&](int t) {
          sc[t] = score_step<0>(codes(0, t), qh[0], ql[0], sc[t], ks[t], qs[0]);
          sc[t] = score_step<1>(codes(1, t), qh[1], ql[1], sc[t], ks[t], qs[0]);
          sc[t] = score_step<2>(codes(2, t), qh[2], ql[2], sc[t], ks[t], qs[1]);
          sc[t] = score_step<3>(codes(3, t), qh[3], ql[3], sc[t], ks[t], qs[1]);
          if constexpr (kPart) {
            uint4 w = *(const uint4*)(stage + A::kTail + ((tt * T2 + t) * 16 + l16) * 32 + (quad & 1) * 16);
            w = quad > 1 ? make_uint4(0u, 0u, 0u, 0u) : w;
            sc[t] = score_step<4>(w, qh[KS - 1], ql[KS - 1], sc[t], klast[t], qs[2]);
          }
        };
        if constexpr (TT > 1) {
          if (it > it0) {   // the maximum with the last step's of the row's other waves
            float next = kLowest;
#pragma unroll
            for (int t = 0; t < TT; ++t) next = fmaxf(next, tops[(it - 1) & 1][rq * 16 + l16][t]);
            l = l * power(m, next) + sum * power(own, next);
            m = next, far = __any(far_off(m));
          }
        }
        own = m, sum = 0.f;
        float top = -INFINITY, c = a.c;
        auto weigh = [&](int t) {   // the probabilities of 16 tokens
          float p[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) p[n] = __builtin_amdgcn_exp2f(fmaf(sc[t][n], c, -own));
          sum += (p[0] + p[1]) + (p[2] + p[3]);
          *(uint2*)(put_w + (it & 1) * A::kWeights + t * (A::kRows * 32)) = make_uint2(mxd::bf16_pair(p[0], p[1]), mxd::bf16_pair(p[2], p[3]));
        };
        auto look = [&](int t) { top = fmaxf(top, fmaxf(fmaxf(sc[t][0], sc[t][1]), fmaxf(sc[t][2], sc[t][3]))); };
        const bool plain = shown == 15u && first >= all_lo && first + 16 * T2 <= all_hi && !far;
        if (plain) {   // under the maximum so far, which seldom rises: 16 tokens' probabilities beside the next ones' scores
          score(0);
#pragma unroll
          for (int t = 0; t < T2; ++t) {
            if (t + 1 < T2) score(t + 1);
            look(t), weigh(t);
          }
        } else {
#pragma unroll
          for (int t = 0; t < T2; ++t) score(t);
#pragma unroll
          for (int t = 0; t < T2; ++t) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const int at = first + 16 * t + 4 * quad + n;
              sc[t][n] = (shown >> (tt * T2 + t) & 1) && at >= row_lo && at < row_hi ? sc[t][n] : -INFINITY;
            }
            look(t);
          }
        }
        top = row_max4(top) * a.c;
        const bool rises = __any(top > m + 8.f);
        if (rises) own = raised(m, top);
        if (!plain || rises) {
          far = __any(far_off(own));
          if (far) {
#pragma unroll
            for (int t = 0; t < T2; ++t)
#pragma unroll
              for (int n = 0; n < 4; ++n) sc[t][n] *= a.c;
            c = 1.f;
          }
          sum = 0.f;
#pragma unroll
          for (int t = 0; t < T2; ++t) weigh(t);
        }
        if (quad == 0) tops[it & 1][rq * 16 + l16][tt] = own;
        if constexpr (TT == 1) {
          l = l * power(m, own) + sum;
          m = own;
        }
        shown = shown_of(lo, hi, it + 1);
        mxd::copy_barrier();
      }
      const bool more = go_on(1);
      if (kAhead && more) load();
      if constexpr (TT > 1) {
        float next = kLowest;
#pragma unroll
        for (int t = 0; t < TT; ++t) next = fmaxf(next, tops[(it1 - 1) & 1][rq * 16 + l16][t]);
        l = l * power(m, next) + sum * power(own, next);
        m = next;
      }
      l = row_sum4(l);
      if (quad == 0) stats[rq * 16 + l16][tt][0] = m, stats[rq * 16 + l16][tt][1] = l;
      __syncthreads();
      // where the rows go
      if (tid < A::kRows) {
        const int r = tid;
        float all_l = 0.f;
#pragma unroll
        for (int t = 0; t < TT; ++t) all_l += stats[r][t][1];
        Place to{-1, 1.f};
        if (row0 + r < rows) {
          if (alone) {
            const int head = h * a.group + a.by_group.rest(row0 + r);
            const int64_t token = first_token + a.by_group.of(row0 + r);
            const RowOut f = row_out(a, head, stats[r][0][0], all_l);
            to = {token * a.q.out_stride + (int64_t)head * WV, f.inv};
            if (a.q.lse) a.q.lse[token * a.q.heads + head] = f.lse;
          } else {
            ((float2*)(a.space + a.at.stats))[slot * A::kRows + r] = make_float2(stats[r][0][0], all_l);
          }
        }
        places[r] = to;
      }
      __syncthreads();
      if (!more) return;
    }
  } else {
    // LDS places of the wave's values: a converter's 16-byte pieces of its token, and a reader's 8 bytes
    uint8_t* tile = lds + cg * A::kTile;
    uint32_t put[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) put[n] = l16 * 256 + 128 * (quad >> 1) + ((4 * (quad & 1) + n) ^ spread) * 16;
    const int rt = l16 >> 2, rc = lane & 3, rs = 2 * rt + half;
    const uint32_t get0 = (4 * half + rt) * 256 + ((2 * (quad & 1) + rc / 2) ^ rs) * 16 + (rc & 1) * 8, get1 = get0 ^ 64;
    const uint32_t get_c = l16 * 256 + (((4 * (cg & 1) + quad) ^ (l16 & 7)) * 16) + 128 * (cg >> 1);   // the columns' codes
    const uint32_t get_s = A::kScales + l16 * 16 + 4 * cg;
    bool exchanged = true;
    for (;;) {
      const int it0 = u.it0, it1 = u.it1, lo = u.lo, hi = u.hi;
      Entry* const table = table_of();
      const bool alone = is_alone(u);
      const int64_t slot = 2 * g + (u.first ? 0 : 1);
      ask(table, lo, hi, it0);
      uint32_t shown = shown_of(lo, hi, it0);
      const int h = u.h;
#pragma unroll
      for (int k = 1; k < A::kStages - 1; ++k)
        if (it0 + k < it1) copy(h, lo, hi, it0 + k, entry_of(table, hi, lo + (it0 + k) * A::kStep + 16 * cg));
      if (exchanged) mxd::lds_barrier();   // (the queries)
      exchanged = false;
      float m[RG];
      v16f o[RG][4];
#pragma unroll
      for (int r = 0; r < RG; ++r) {
        m[r] = kLowest;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int n = 0; n < 16; ++n) o[r][d][n] = 0.f;
      }
      // 16 tokens' columns of a step: their codes, and to BF16
      struct Codes {
        uint4 w;
        uint32_t scales;
        bool valid;
      };
      auto codes_of = [&](int it, int t) {
        const uint8_t* stage = lds + A::kRing + (it % A::kStages) * A::kStage;
        return Codes{*(const uint4*)(stage + get_c + 4096 * t), *(const uint32_t*)(stage + get_s + 256 * t),
                     l16 < (shown >> t & 1 ? hi - (lo + it * A::kStep + 16 * t) : 0)};
      };
      auto convert = [&](const Codes& v, int t) {
        // NaN blocks count as tiny here, as what no token of the sequence has left: who sees a NaN token has NaN from its
        // score, and for the others 0 times this is 0
        const uint32_t e = v.scales >> (8 * quad) & 255u;
        const float scale = mx::u2f((e != 255u && v.valid ? e : 0u) << 23);
        const uint32_t c[4] = {v.w.x, v.w.y, v.w.z, v.w.w};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          uint4 w;
          w.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[n], scale, 0));
          w.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[n], scale, 1));
          w.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[n], scale, 2));
          w.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[n], scale, 3));
          *(uint4*)(tile + put[n] + 4096 * t) = w;
        }
      };
      bool moved = false;
      float theirs[RG][TT];
      auto settle = [&](int it) {   // the maxima with step `it`'s
        bool any = false;
        float next[RG];
#pragma unroll
        for (int r = 0; r < RG; ++r) {
          next[r] = kLowest;
#pragma unroll
          for (int t = 0; t < TT; ++t) {
            theirs[r][t] = tops[it & 1][r * 32 + col][t];
            next[r] = fmaxf(next[r], theirs[r][t]);
          }
          any |= next[r] != m[r];
        }
        moved = __any(any);
        if (moved) {
#pragma unroll
          for (int r = 0; r < RG; ++r) {
            const float by = power(m[r], next[r]);
            m[r] = next[r];
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
              for (int n = 0; n < 16; ++n) o[r][d][n] *= by;
          }
        }
      };
      // 16 tokens' values and probabilities of step `it`, and O^T += V^T P^T of them
      struct Operands {
        v8b v[4], p[RG];
      };
      auto operands = [&](int it, int t) {
        Operands r;
#pragma unroll
        for (int i = 0; i < RG; ++i)
          r.p[i] = __builtin_bit_cast(v8b, *(const uint4*)(weights + (it & 1) * A::kWeights + (t * A::kRows + i * 32 + col) * 32 + half * 16));
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const uint8_t* at = tile + (d & 1 ? get1 : get0) + 128 * (d / 2) + 4096 * t;
          typedef __attribute__((address_space(3))) v4s lds_v4s;
          v4s w[2];
          w[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at);
          w[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 2048));
          r.v[d] = __builtin_bit_cast(v8b, w);
        }
        return r;
      };
      auto multiply = [&](Operands& r, int t) {
        if (TT > 1 && moved) {   // by powers of two, but for a unit's first step
#pragma unroll
          for (int i = 0; i < RG; ++i) {
            const float f = power(theirs[i][t / T2], m[i]);
            auto scaled = [&](uint32_t v) { return mxd::bf16_pair(mx::u2f(v << 16) * f, mx::u2f(v & 0xFFFF0000u) * f); };
            const uint4 w = __builtin_bit_cast(uint4, r.p[i]);
            r.p[i] = __builtin_bit_cast(v8b, make_uint4(scaled(w.x), scaled(w.y), scaled(w.z), scaled(w.w)));
          }
        }
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int i = 0; i < RG; ++i) o[i][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(r.v[d], r.p[i], o[i][d], 0, 0, 0);
      };
      int entry = entry_of(table, hi, lo + (it0 + A::kStages - 1) * A::kStep + 16 * cg);   // of the next copies
      auto next_entry = [&](int it) { return entry_of(table, hi, lo + (it + A::kStages) * A::kStep + 16 * cg); };
      // this wave's copies of the step after `it` have landed; those of later steps may be on their way
      auto landed = [&](int it) {
        if (it + A::kStages - 1 < it1) {
          copy(h, lo, hi, it + A::kStages - 1, entry);
          __builtin_amdgcn_s_waitcnt(mxd::vm_wait_imm(A::kCopies * (A::kStages - 2)));
        } else {
          __builtin_amdgcn_s_waitcnt(mxd::vm_wait_imm(0));
        }
        asm volatile("" ::: "memory");
      };
      if (it0 + A::kStages - 1 <= it1) {   // the first step's copies have landed
        __builtin_amdgcn_s_waitcnt(mxd::vm_wait_imm(A::kCopies * (A::kStages - 2)));
      } else {
        __builtin_amdgcn_s_waitcnt(mxd::vm_wait_imm(0));
      }
      asm volatile("" ::: "memory");
      mxd::copy_barrier();
#pragma unroll
      for (int t = 0; t < 4; ++t) convert(codes_of(it0, t), t);
      ask(table, lo, hi, it0 + 1);
      int asked = next_entry(it0);
      landed(it0);
      entry = asked;
      shown = shown_of(lo, hi, it0 + 1);
      mxd::copy_barrier();
      for (int it = it0 + 1; it < it1; ++it) {
        // everything is read from LDS a turn before it is used: 16 tokens' products, under which the next ones' operands come
        // and this step's take the place of those just read
        asked = next_entry(it);
        Codes next[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) next[t] = codes_of(it, t);
        ask(table, lo, hi, it + 1);
        Operands now = operands(it - 1, 0);
        settle(it - 1);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          Operands after;
          if (t < 3) after = operands(it - 1, t + 1);
          multiply(now, t);
          convert(next[t], t);
          if (t < 3) now = after;
        }
        landed(it);
        entry = asked;
        shown = shown_of(lo, hi, it + 1);
        mxd::copy_barrier();
      }
      const bool more = go_on(1);   // (the stages are free, and the values are read last)
      if (more) begin();
      settle(it1 - 1);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        Operands now = operands(it1 - 1, t);
        multiply(now, t);
      }
      __syncthreads();
      __syncthreads();
      if (alone) {
        // a lane has 4 of every 8 columns of its row: the halves exchange fours, and each stores 8 in a row
#pragma unroll
        for (int r = 0; r < RG; ++r) {
          const Place to = places[r * 32 + col];
          if (to.at < 0) continue;
          uint16_t* out = a.q.out + to.at + cg * 128 + 8 * half;
#pragma unroll
          for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int n = 0; n < 16; n += 8) {
              const v16f& v = o[r][d];
              const auto x = __builtin_amdgcn_permlane32_swap(mxd::bf16_pair(v[n] * to.by, v[n + 1] * to.by),
                                                              mxd::bf16_pair(v[n + 4] * to.by, v[n + 5] * to.by), false, false);
              const auto y = __builtin_amdgcn_permlane32_swap(mxd::bf16_pair(v[n + 2] * to.by, v[n + 3] * to.by),
                                                              mxd::bf16_pair(v[n + 6] * to.by, v[n + 7] * to.by), false, false);
              *(uint4*)(out + 32 * d + 2 * n) = make_uint4(x[0], y[0], x[1], y[1]);
            }
        }
      } else {   // parts as the registers have them: [wave][row group][block][4 registers][lane]
        float4* part = (float4*)(a.space + a.at.rows) + (slot * 4 + cg) * (RG * 4 * 4 * 64) + lane;
#pragma unroll
        for (int r = 0; r < RG; ++r)
#pragma unroll
          for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int n = 0; n < 4; ++n)
              part[((r * 4 + d) * 4 + n) * 64] = make_float4(o[r][d][4 * n], o[r][d][4 * n + 1], o[r][d][4 * n + 2], o[r][d][4 * n + 3]);
      }
      if (!more) return;
    }
  }
}

// Waves of the grouped kernel that a SIMD holds (so workgroups a CU), by what their registers allow.
__host__ __device__ constexpr int waves(int width) { return width <= 64 ? 3 : width <= 128 ? 2 : 1; }

// Values apart from their keys. A wave holds 32 rows and takes 32 tokens a step. A step is TG = 4 / RG tiles of 32 tokens, a
// tile the work of RG waves, one a row group, which share its values; a wave keeps to its tile, and the token groups' sums are
// added at the end.
//
// Measured: one token of 32 heads of 128 over 8 key heads and 64 sequences of 500 to 16,000 tokens, 317 MB: 65 us, 4.9 TB/s
// (a large copy's reads and writes 5.1). Two prompts' 2048 tokens over 4500 and 8192, 322 GFLOP: 357 us, the matrix units busy
// in 39 % of the cycles: a step's products take 512 clocks of a SIMD and its other instructions (converting, softmax) about
// as many again from each of two waves.
template <int W, int RG>
struct Grouped {
  static constexpr int TG = 4 / RG, kRows = 32 * RG, kStep = 32 * TG;
  static constexpr int KS = W / 64, DB = W / 32, KW = scale_pitch(W) / 4;
  static constexpr int VO = (KS + RG - 1) / RG;            // 64-column pieces of the values that a wave converts
  static constexpr int kTile = 64 * W;                     // bytes of 32 tokens' values in BF16
  static constexpr int kBuffers = RG > 1 ? 2 : 1;          // others read what a wave has written: with two, one barrier a step
  static constexpr int CB = 64, kOut = 32 * (CB + 4) * 4;  // columns that go out at a time, and a wave's bytes of them
  static constexpr int kValues = TG * kBuffers * kTile, kLds = kValues > 4 * kOut ? kValues : 4 * kOut;
  static constexpr int kWaves = waves(W), kGroups = kCus * kWaves;
};

template <int W, int RG>
__global__ __launch_bounds__(256, (Grouped<W, RG>::kWaves)) void grouped_kernel(AttendArgs a, int by) {
  using A = Grouped<W, RG>;
  constexpr int TG = A::TG, KS = A::KS, DB = A::DB, KW = A::KW, VO = A::VO, CB = A::CB;
  __shared__ __attribute__((aligned(16))) uint8_t lds[A::kLds];
  __shared__ float stats[4][32][2];
  __shared__ Place places[A::kRows];
  __shared__ uint32_t sums[4];
  __shared__ int32_t found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rg = wave % RG, tg = wave / RG;
  const int col = lane & 31, half = lane >> 5;   // the lane's query row of the products; as a loader, its token

  Plan plan{(int32_t*)(a.space + a.at.base), (int64_t*)(a.space + a.at.prefix)};
  if (by == kInLds) {
    plan = {(int32_t*)(lds + 8 * (kInlineTiles + 1)), (int64_t*)lds};
    make_plan<256>(a, plan, sums, A::kRows, A::kStep);
  }
  constexpr int groups = A::kGroups;
  // workgroups go round the XCDs: neighbours in the work, which share keys, to one L2
  const int g = (int)(blockIdx.x % kXcds) * (groups / kXcds) + (int)blockIdx.x / kXcds;
  Shared* shared = (Shared*)(a.space + a.at.units) + g;
  if (tid == 0) shared->parts = 0;
  int64_t per;
  Units u;
  if (!(by == kByWave ? first_of_few(a, g, per, groups, u, A::kRows, A::kStep)
                      : first_unit<256>(a, plan, by == kInLds, g, per, groups, found, u, A::kRows, A::kStep)))
    return;

  // LDS places: a loader's 16-byte pieces of its token, and a reader's 8 bytes; pieces of neighbouring tokens lie apart
  const int spread = 2 * (col & 3) + ((col >> 2) & 1);
  uint32_t put[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) put[i] = tg * A::kTile + col * (2 * W) + ((4 * half + i) ^ spread) * 16;
  const int rt = (lane & 15) >> 2, rc = lane & 3, rs = 2 * rt + half;
  const uint32_t get0 = tg * A::kTile + (4 * half + rt) * (2 * W) + ((2 * ((lane >> 4) & 1) + rc / 2) ^ rs) * 16 + (rc & 1) * 8;
  const uint32_t get1 = get0 ^ 64;

  auto go_on = [&] {   // to the next unit, if there is one
    if (u.end <= u.unit0 + kBegin + u.n && tid == 0) note(u, per, g, groups, shared);
    next_unit(a, u, A::kRows, A::kStep);
    return u.x < u.end;
  };
  for (;;) {
    if (u.it1 <= u.it0) {   // only what the unit's beginning costs is this workgroup's
      if (!go_on()) return;
      continue;
    }
    const int it0 = u.it0, it1 = u.it1;
    // -- the wave's query rows --
    const int rows = u.s.n * a.group;   // at most 2^30
    const int row0 = u.tile * A::kRows + rg * 32, row = min(row0 + col, rows - 1);
    const int i = a.by_group.of(row);
    int row_lo, row_hi;
    seen(a, u.s, i, row_lo, row_hi);
    // tokens [all_lo, all_hi) are seen by all of the wave's rows
    int all_lo, all_hi, unused;
    seen(a, u.s, a.by_group.of(min(row0, rows - 1)), unused, all_hi);
    seen(a, u.s, a.by_group.of(min(row0 + 31, rows - 1)), all_lo, unused);
    all_lo = uniform(all_lo), all_hi = uniform(all_hi);

    // -- loads: the lane's token of a step, its page a step ahead --
    const int32_t* table = a.q.table + (int64_t)u.b * a.q.columns;
    const int lo = u.lo, hi = u.hi, h = u.h;
    auto token_of = [&](int it) { return lo + (it * TG + tg) * 32 + col; };
    auto page_of = [&](int it) {
      const int t = token_of(it);
      return it < it1 && t < hi ? table[t >> a.page_shift] : -1;
    };
    uint4 kreg[KS], vreg[VO];
    uint32_t kscale[KW], vscale[KW];
    bool valid = false;
    auto load = [&](int it, int page) {
      valid = page >= 0 && page < a.cache.pages;
      const int64_t at = (((int64_t)(valid ? page : 0) * a.cache.heads + h) << a.page_shift) + (token_of(it) & ((1 << a.page_shift) - 1));
      const uint8_t* p = a.cache.k_codes + at * (W / 2) + 16 * half;
      const uint8_t* pv = a.cache.v_codes + at * (W / 2) + 16 * half;
#pragma unroll
      for (int k = 0; k < KS; ++k) kreg[k] = mxd::ldg128(p + 32 * k);
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        kscale[w] = mxd::ldg32(a.cache.k_scales + at * scale_pitch(W) + 4 * w);
        vscale[w] = mxd::ldg32(a.cache.v_scales + at * scale_pitch(W) + 4 * w);
      }
#pragma unroll
      for (int k = 0; k < VO; ++k)
        if (k * RG + rg < KS) vreg[k] = mxd::ldg128(pv + 32 * (k * RG + rg));
    };
    load(it0, page_of(it0));
    int page_next = page_of(it0 + 1);

    // -- the queries: a row group's waves convert KS / TG steps of 64 values each and exchange them --
    v8i qh[KS], ql[KS];
    uint32_t qs[(KS + 1) / 2] = {};
    {
      const uint16_t* q = a.q.q + (u.s.first + i) * a.q.q_stride + (int64_t)(h * a.group + a.by_group.rest(row)) * W;
      constexpr int kEach = (KS + TG - 1) / TG;
      QueryWords words[kEach];
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (e * TG + tg < KS) words[e] = query_words<32>(q + 64 * (e * TG + tg) + 16 * half);
      uint4* made = (uint4*)lds + rg * (KS * 256) + lane;
      uint32_t* made_scales = (uint32_t*)(lds + RG * KS * 4096) + rg * (KS * 64) + lane;
      __syncthreads();   // the plan, or the last unit's rows, have been read
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int k = e * TG + tg;
        if (k >= KS) break;
        const QueryStep s = query_step(words[e], half);
        if constexpr (TG > 1) {
          made[k * 256] = make_uint4(s.high[0], s.high[1], s.high[2], s.high[3]), made[k * 256 + 64] = make_uint4(s.high[4], s.high[5], s.high[6], s.high[7]);
          made[k * 256 + 128] = make_uint4(s.low[0], s.low[1], s.low[2], s.low[3]), made[k * 256 + 192] = make_uint4(s.low[4], s.low[5], s.low[6], s.low[7]);
          made_scales[k * 64] = s.scales;
        } else {
#pragma unroll
          for (int n = 0; n < 8; ++n) qh[e][n] = (int)s.high[n], ql[e][n] = (int)s.low[n];
          qs[e / 2] |= s.scales << (16 * (e & 1));
        }
      }
      if constexpr (TG > 1) {
        mxd::lds_barrier();
#pragma unroll
        for (int k = 0; k < KS; ++k) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint4 w = made[k * 256 + 64 * j], v = made[k * 256 + 128 + 64 * j];
            qh[k][4 * j] = (int)w.x, qh[k][4 * j + 1] = (int)w.y, qh[k][4 * j + 2] = (int)w.z, qh[k][4 * j + 3] = (int)w.w;
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

    float m = kLowest, bar = kLowest, l = 0.f;
    v16f o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int n = 0; n < 16; ++n) o[d][n] = 0.f;

    for (int it = it0; it < it1; ++it) {
      // -- scores --
      uint32_t bad = 0;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        constexpr int used = W / 32;
        bad |= marks(4 * w + 4 <= used ? vscale[w] : vscale[w] & ((1u << 8 * (used & 3)) - 1u));
      }
      const bool hide = bad || !valid;   // its values count as zero; who sees a NaN token sees it in the score
      uint32_t ks[KW];
#pragma unroll
      for (int w = 0; w < KW; ++w) ks[w] = bad ? ~0u : kscale[w] >> (8 * half);
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
      __builtin_amdgcn_sched_barrier(0);   // what follows runs beside the products
      // -- values to BF16 --
      uint8_t* buffer = lds + (A::kBuffers > 1 ? (it & 1) * (TG * A::kTile) : 0);
#pragma unroll
      for (int k = 0; k < VO; ++k) {
        const int piece = k * RG + rg;   // columns [64 piece, + 64), the lane's half of them
        if (VO * RG > KS && piece >= KS) break;
        const uint32_t word = KW == 1 || piece < 2 ? vscale[0] : vscale[KW - 1];
        const uint32_t e = word >> (8 * half + 16 * (piece & 1)) & 255u;
        const float scale = mx::u2f((hide ? 127u : e) << 23);
        const uint32_t c[4] = {hide ? 0u : vreg[k].x, hide ? 0u : vreg[k].y, hide ? 0u : vreg[k].z, hide ? 0u : vreg[k].w};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          uint4 v;
          v.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[n], scale, 0));
          v.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[n], scale, 1));
          v.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[n], scale, 2));
          v.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[n], scale, 3));
          *(uint4*)(buffer + put[n] + 128 * piece) = v;
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
          sc[n] = (shown >> t & 1) && first + t >= row_lo && first + t < row_hi ? sc[n] : -INFINITY;
        }
      }
      float top = fmaxf(sc[0], sc[1]);
#pragma unroll
      for (int n = 2; n < 16; ++n) top = fmaxf(top, sc[n]);
      top = other_half_max(top) * a.c;
      float c = a.c;   // far off: 1, and c s in the scores' place (prompts of 128 wide 379 us with this, 374 without)
      if (__any(top > bar)) {
        const float own = raised(m, top), by = power(m, own);
        m = own, bar = bar_of(m), l *= by;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int n = 0; n < 16; ++n) o[d][n] *= by;
        if (__any(far_off(m))) {
#pragma unroll
          for (int n = 0; n < 16; ++n) sc[n] *= a.c;
          c = 1.f;
        }
      }
      uint32_t p[8];
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[2 * n], c, -m)), p1 = __builtin_amdgcn_exp2f(fmaf(sc[2 * n + 1], c, -m));
        l += p0 + p1;
        p[n] = mxd::bf16_pair(p0, p1);
      }
      if (RG > 1) mxd::lds_barrier();
      // -- O^T += V^T P^T, the values read two products ahead --
      v8b vv[3];
      auto read = [&](int n) {
        const int k = n / DB, d = n % DB;
        const uint8_t* at = buffer + (d & 1 ? get1 : get0) + 128 * (d / 2) + 16 * k * (2 * W);
        typedef __attribute__((address_space(3))) v4s lds_v4s;
        v4s w[2];
        w[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at);
        w[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 8 * (2 * W)));
        vv[n % 3] = __builtin_bit_cast(v8b, w);
      };
      read(0), read(1);
#pragma unroll
      for (int n = 0; n < 2 * DB; ++n) {
        const int k = n / DB, d = n % DB;
        if (n + 2 < 2 * DB) read(n + 2);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vv[n % 3], __builtin_bit_cast(v8b, make_uint4(p[4 * k], p[4 * k + 1], p[4 * k + 2], p[4 * k + 3])),
                                                       o[d], 0, 0, 0);
      }
    }

    // -- the token groups' sums together, and out --
    l = halves_sum(l);
    if (half == 0) stats[wave][col][0] = m, stats[wave][col][1] = l;
    __syncthreads();   // and everybody has read its values
    const bool alone = is_alone(u);
    const int64_t slot = 2 * g + (u.first ? 0 : 1);
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
          const int head = h * a.group + a.by_group.rest(row);
          const int64_t token = u.s.first + i;
          const RowOut f = row_out(a, head, most, all_l);
          to = {token * a.q.out_stride + (int64_t)head * W, f.inv};
          if (a.q.lse) a.q.lse[token * a.q.heads + head] = f.lse;
        } else {
          to.at = (slot * A::kRows + r) * W;
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
      if constexpr (TG == 1) {
        const int c = lane % L * 4;
#pragma unroll 4
        for (int r = lane / L; r < 32; r += 64 / L) put_out(rg * 32 + r, d0 * 32 + c, *(const float4*)(own_out + r * (CB + 4) + c));
      } else {
        __syncthreads();
#pragma unroll 2
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
    if (!go_on()) return;
  }
}

// The units that several workgroups had, in pieces of 64 times four values. Where there are more waves than pieces a
// workgroup's waves share a piece's parts; else each takes a piece. Every wave finds the units for itself, in the
// workgroups' last ones, all of them at once. Bound by memory: 39 MB of parts (the 48 sequences above) in 10 us, 4.6 MB (one
// sequence) in 5; a list of the units made in LDS by each workgroup before it began took 22.
//
// piece(e, r, c): the row and first column of the e-th four values of a unit, as its parts have them.
template <int kGroups, int kRows, int WV, typename Piece>
__device__ __forceinline__ void join(const AttendArgs& a, Piece piece) {
  __shared__ float4 sums[4][64];
  __shared__ float2 tops[4][64];
  constexpr int kLook = kGroups / 64, kPieces = kRows * WV / 256;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Shared* units = (const Shared*)(a.space + a.at.units);
  uint64_t masks[kLook];
  int n = 0;
#pragma unroll
  for (int j = 0; j < kLook; ++j) masks[j] = __ballot(units[64 * j + lane].parts > 1);
#pragma unroll
  for (int j = 0; j < kLook; ++j) n += __popcll(masks[j]);
  const bool together = n * kPieces < (int)gridDim.x * 2;
  const int stride = together ? (int)gridDim.x : 4 * (int)gridDim.x;
  const float4* parts = (const float4*)(a.space + a.at.rows);
  for (int k = together ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave; k < n * kPieces; k += stride) {
    int nth = k / kPieces, g = 0;   // the nth set bit
#pragma unroll
    for (int j = 0; j < kLook; ++j) {
      const int here = __popcll(masks[j]);
      if (nth >= 0 && nth < here) {
        uint64_t m = masks[j];
        for (; nth > 0; --nth) m &= m - 1;
        g = 64 * j + __builtin_ctzll(m);
        nth = -1;
      }
      nth -= nth >= 0 ? here : 0;
    }
    const Shared s = units[g];
    const int e = k % kPieces * 64 + lane;
    int r, c;
    piece(e, r, c);
    const float2* stats = (const float2*)(a.space + a.at.stats) + r;
    // the first workgroup's part lies in its slot s.slot, the others' in their first
    auto slot = [&](int i) { return (int64_t)2 * (g + i) + (i ? 0 : s.slot); };
    float most = kLowest, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](auto count, int i0, int step) {   // so many parts at a time
      constexpr int N = decltype(count)::value;
      float2 st[N];
      float4 p[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int64_t at = slot(min(i0 + step * j, s.parts - 1));
        st[j] = stats[at * kRows];
        p[j] = parts[at * (kRows * WV / 4) + e];
      }
      float next = most;
#pragma unroll
      for (int j = 0; j < N; ++j) next = fmaxf(next, st[j].x);
      const float by = power(most, next);
      most = next, sum *= by;
      v.x *= by, v.y *= by, v.z *= by, v.w *= by;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const bool use = i0 + step * j < s.parts;   // (not by a factor of zero: a part may hold NaN)
        const float f = power(st[j].x, most);
        sum += use ? st[j].y * f : 0.f;
        v.x += use ? p[j].x * f : 0.f, v.y += use ? p[j].y * f : 0.f, v.z += use ? p[j].z * f : 0.f, v.w += use ? p[j].w * f : 0.f;
      }
    };
    constexpr std::integral_constant<int, 2> two{};
    constexpr std::integral_constant<int, 8> eight{};
    if (together) {
      if (s.parts <= 8) {
        if (wave < s.parts) add(two, wave, 4);
      } else {
        for (int i0 = wave; i0 < s.parts; i0 += 32) add(eight, i0, 4);
      }
      __syncthreads();
      sums[wave][lane] = v, tops[wave][lane] = make_float2(most, sum);
      __syncthreads();
      if (wave) continue;
#pragma unroll
      for (int w = 1; w < 4; ++w) most = fmaxf(most, tops[w][lane].x);
      sum = 0.f, v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = power(tops[w][lane].x, most);
        const float4 p = sums[w][lane];
        sum += tops[w][lane].y * f;
        v.x += p.x * f, v.y += p.y * f, v.z += p.z * f, v.w += p.w * f;
      }
    } else {
      if (s.parts <= 4) {
        for (int i0 = 0; i0 < s.parts; i0 += 2) add(two, i0, 1);
      } else {
        for (int i0 = 0; i0 < s.parts; i0 += 8) add(eight, i0, 1);
      }
    }
    const Sequence q = sequence(a, s.b);
    const int row = s.tile * kRows + r;
    if (row >= q.n * a.group) continue;
    const int head = s.h * a.group + a.by_group.rest(row);
    const int64_t token = q.first + a.by_group.of(row);
    const RowOut f = row_out(a, head, most, sum);
    uint2 w;
    w.x = mxd::bf16_pair(v.x * f.inv, v.y * f.inv), w.y = mxd::bf16_pair(v.z * f.inv, v.w * f.inv);
    *(uint2*)(a.q.out + token * a.q.out_stride + (int64_t)head * WV + c) = w;
    if (a.q.lse && c == 0) a.q.lse[token * a.q.heads + head] = f.lse;
  }
}

template <int RG>
__global__ __launch_bounds__(256) void join_latent_kernel(AttendArgs a) {
  using A = Latent<512, RG>;
  join<kCus, A::kRows, A::WV>(a, [](int e, int& r, int& c) {
    const int lane = e & 63, n = e >> 6 & 3, d = e >> 8 & 3, rg = e >> 10 & (RG - 1), wave = e / (1024 * RG);
    r = rg * 32 + (lane & 31), c = wave * 128 + 32 * d + 8 * n + 4 * (lane >> 5);
  });
}

template <int W, int RG>
__global__ __launch_bounds__(256) void join_grouped_kernel(AttendArgs a) {
  using A = Grouped<W, RG>;
  join<A::kGroups, A::kRows, W>(a, [](int e, int& r, int& c) { r = e / (W / 4), c = e % (W / 4) * 4; });
}

int check_attend(const char* who, const mx_kv4* c, int32_t heads, int32_t tokens, int32_t batch) {
  if (int s = check_cache(who, c)) return s;
  MX_REQUIRE(heads >= 1 && heads <= (1 << 16) && heads % c->heads == 0, "%s: %d query heads for %d key heads", who, heads, c->heads);
  MX_REQUIRE(tokens >= 0 && tokens <= kMaxTokens, "%s: token count %d outside [0, %d]", who, tokens, kMaxTokens);
  MX_REQUIRE(batch >= 0 && batch <= kMaxBatch, "%s: %d sequences outside [0, %d]", who, batch, kMaxBatch);
  MX_REQUIRE((int64_t)tokens * heads <= (1ll << 30), "%s: more than 2^30 query rows in all", who);
  return MX_OK;
}

// The most row groups of 32 that a workgroup takes.
int most_groups(const mx_kv4* c) { return c->v_codes ? 4 : 2; }

int workgroups(const mx_kv4* c) { return kCus * (c->v_codes ? waves(c->width) : 1); }

// Row tiles of all sequences at most: each sequence's last one may be partly full.
int64_t most_tiles(int64_t rows, int batch, int tile_rows) { return rows / tile_rows + batch; }

Space space_of(const mx_kv4* c, int group, int tokens, int batch, int tile_rows) {
  const int64_t n = workgroups(c), tiles = most_tiles((int64_t)tokens * group, batch, tile_rows);
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
  for (int rg = 1; rg <= most_groups(cache); rg *= 2) most = std::max(most, space_of(cache, group, tokens, batch, 32 * rg).total);
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
  MX_REQUIRE(q.scale > 0.f && q.scale <= 2.3e38f, "%s: scale must be positive and at most 2.3e38", who);   // (times log2(e))
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
  // As many row groups as an average sequence's rows fill, and fewer where little is to do: each lengthens every workgroup's
  // beginning and end, and saves the others' reading and converting. By the steps of 32 rows and 32 tokens that a wave has
  // when the tables are full. Latents of 64 heads: 128 x 300 tokens (5 steps) 20.9 us with one and 33.2 with two, 1 x 4099
  // (2) 19.5 and 22.1, 16 x 4000 (4) 32.0 and 33.1, 16 x 16000 (16) 69.6 and 55.9. Values apart, 32 heads of 128 over 8 key
  // heads: 64 rows of 600 tokens (1 step) 17.3, 20.5 and 21.3 us with one, two and four, 256 of 2000 (8) 28.7, 29.3 and
  // 33.4, 4 x 64 of 4000 (16) 43.1, 38.9 and 42.9, 2048 of 2048 (64) 72.1, 65.1 and 80.0, 2048 of 8192 (256) 292, 275 and 270.
  const int n = workgroups(cache);
  const int64_t tokens_each = ((int64_t)q.tokens + q.batch - 1) / q.batch, rows = tokens_each * a.group;
  const int64_t held = std::min<int64_t>((int64_t)q.columns * cache->page, q.window ? q.window + tokens_each : INT64_MAX);
  const double steps = (double)q.batch * cache->heads * ((rows + 31) / 32) * ((held + 31) / 32) / (4. * n);
  int rg = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  rg = std::min({rg, most_groups(cache), steps <= (cache->v_codes ? 8 : 5) ? 1 : steps <= 128 ? 2 : 4});
  const int tile_rows = 32 * rg, step = cache->v_codes ? 128 / rg : kLatentStep;
  a.by_group = Divide(a.group);
  if (!q.q_first) a.rows_each = q.tokens / q.batch, a.tiles_each = (int)(((int64_t)a.rows_each * a.group + tile_rows - 1) / tile_rows);
  a.by_tiles = Divide(std::max(a.tiles_each, 1));
  a.at = space_of(cache, a.group, q.tokens, q.batch, tile_rows);
  const int64_t tiles = most_tiles((int64_t)q.tokens * a.group, q.batch, tile_rows);
  a.tiles = (int)tiles;
  const int by = tiles <= 64 ? kByWave : tiles <= kInlineTiles ? kInLds : kInSpace;   // (at least as many as sequences)
  hipStream_t st = as_stream(stream);
  // Units of few iterations stay whole, by what the tables can hold: parts cost another beginning, their way out and the
  // second launch, some 9 us. One token each, split and whole: latents of 64 heads 128 x 500 tokens (8 iterations) 26.1 and
  // 23.9 us, 400 x 500 64.2 and 52.9, of one row group 64 x 700 (11) 33.9 and 27.6, 64 x 1000 (16) 36.1 and 34.8, 256 x 1000 of
  // 16 heads 41.3 and 39.1, but 1 x 320 (5) 12.2 and 14.7 and 1 x 500 12.7 and 19.3; 32 heads over 8 key heads 64 x 1000 (8)
  // 22.7 and 19.5, 1 x 800 (7) 13.4 and 13.1, 1 x 1000 13.1 and 13.9; prompts of 1000 with a window of 128 (2) 36.5 and 27.4.
  const int64_t span = std::min<int64_t>(held, q.window ? (int64_t)q.window + 31 + (tile_rows + a.group - 1) / a.group : INT64_MAX);
  const bool few_units = (int64_t)q.batch * cache->heads * ((rows + tile_rows - 1) / tile_rows) < 16;
  a.whole = span <= (int64_t)step * (few_units ? cache->v_codes ? 7 : 4 : cache->v_codes || rg > 1 ? 8 : 16);
  if (by == kInSpace) {
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(1024), 0, st, a, tile_rows, step);
    MX_LAUNCH_CHECK("plan_kernel");
  }
  const int joiners = 8 * kCus;
  auto latent = [&](auto wk, auto groups) {
    constexpr int WK = decltype(wk)::value, RG = decltype(groups)::value;
    static_assert(Latent<WK, RG>::kRows == 32 * RG && Latent<WK, RG>::kStep == kLatentStep, "the plan is of these tiles and steps");
    hipLaunchKernelGGL((latent_kernel<WK, RG>), dim3(n), dim3(512), 0, st, a, by);
    MX_LAUNCH_CHECK("latent_kernel");
    if (a.whole) return MX_OK;
    hipLaunchKernelGGL(join_latent_kernel<RG>, dim3(joiners), dim3(256), 0, st, a);
    MX_LAUNCH_CHECK("join_latent_kernel");
    return MX_OK;
  };
  auto grouped = [&](auto w, auto groups) {
    constexpr int W = decltype(w)::value, RG = decltype(groups)::value;
    static_assert(Grouped<W, RG>::kRows == 32 * RG && Grouped<W, RG>::kStep == 128 / RG, "the plan is of these tiles and steps");
    hipLaunchKernelGGL((grouped_kernel<W, RG>), dim3(n), dim3(256), 0, st, a, by);
    MX_LAUNCH_CHECK("grouped_kernel");
    if (a.whole) return MX_OK;
    hipLaunchKernelGGL((join_grouped_kernel<W, RG>), dim3(joiners), dim3(256), 0, st, a);
    MX_LAUNCH_CHECK("join_grouped_kernel");
    return MX_OK;
  };
  using std::integral_constant;
  auto by_rows = [&](auto launch, auto w) {
    if (rg == 1) return launch(w, integral_constant<int, 1>());
    if (rg == 2) return launch(w, integral_constant<int, 2>());
    return launch(w, integral_constant<int, 4>());
  };
  auto two = [&](auto w) { return rg == 1 ? latent(w, integral_constant<int, 1>()) : latent(w, integral_constant<int, 2>()); };
  switch (cache->width) {
    case 64: return by_rows(grouped, integral_constant<int, 64>());
    case 128: return by_rows(grouped, integral_constant<int, 128>());
    case 256: return by_rows(grouped, integral_constant<int, 256>());
    case 512: return two(integral_constant<int, 512>());
    default: return two(integral_constant<int, 576>());
  }
}

}  // extern "C"
