// Tokens sorted by expert and back: the plan, the rows in expert order, the weighted sum per token, and the gradients
// of both, for experts of any format (the fused MXFP4 layer, mx_moe_prefill, keeps a plan and rows of its own).
//
// P = T k pairs p = t k + j; key(p) = ids[p] where that is in [0, G), else G. The plan is the stable order by key:
//   row(p) = #{q: key(q) < key(p)} + #{q < p: key(q) = key(p)},   first[g] = #{q: key(q) < g}
// so a group's rows are in ascending token order, as the reference's participation orders them
// (src/vesper/moe.py:18-30), and pairs without a group come last. A pair's place comes from counts and ballots over the
// ids (the only atomics add up counts), so the plan is the same on every run.
//
// combine adds a token's rows in ascending row (so ascending expert) order in FP32 from zero, the shared row last, and
// rounds once: without weights the sums of MoEAccumulator (src/vesper/moe.py:42-148), bit for bit.
//
// All of it is memory traffic: each row is read once and written once, and the calls reach 5.4 to 5.9 TB/s of a plain
// copy's 5.0 and a read's 6.9 on 4096 tokens of 8 rows of 7168 BF16 values. Small calls are one launch, 4 to 5 us from
// the host.
#include <algorithm>

#include "mx_device.h"
#include "mx_internal.h"
#include "mx_numerics.h"

namespace {

constexpr int kMaxTokens = 1 << 18;   // keeps every grid below 2^32 threads
constexpr int kMaxTopK = 32, kMaxGroups = 1024;
constexpr int64_t kMaxWidth = 1 << 24;
// Calls that move more than this go past the caches with what they touch once. The sum of a token counts only with all
// its pairs here: an expert-parallel rank moves a fraction of what the host can tell. Through the caches and past them,
// rows of 7168 BF16 values, 8 a token, three sets of buffers in turn: combine of 600 tokens 19.4 and 21.3 us, of 800
// 26.2 and 25.2, of 4096 118 and 107; its gradient 400: 20.3 and 20.3, 600: 32.9 and 29.2; dispatch 600: 16.8 and 17.8,
// 800: 25.0 and 22.5. 600 tokens are 77 MB (the gradient 146), 800 are 103. Dispatch, which writes each row once, goes by
// all the pairs that the host knows of: on a rank that holds a part of them it may write past the caches what would fit.
constexpr int64_t kStreamBytes = 96 << 20;

// ---- plan ----

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

struct PlanArgs {
  const int32_t* ids;
  int32_t pairs, groups;
  int32_t* first;
  int32_t* pair_row;
  int32_t* row_pair;
};

// Workgroup g places the pairs of key g (kAbsent: g = G, the pairs without a group). Each wave takes a contiguous
// section of the pairs, 64 at a time: every lane counts the smaller keys and its own key among its pairs (as unsigned
// numbers, ids below zero are no smaller key; pairs past the section count as ids past the last), and the second walk
// places the key's pairs in order. kBatch loads are in flight together, and a section of one batch stays in registers
// for the second walk: 8, 16 or 32 by the pairs (16384 pairs of 256 groups: 5.8 us with 16, 9.8 with 32). Every
// workgroup reads all the ids, from the L2s: what counts is the instructions per 64 of them and the loads' latency
// (32768 pairs: 8.9 us; with the ids counted by scalar code from ballots 17, with fewer loads in flight 21).
template <bool kAbsent, int kBatch>
__device__ __forceinline__ void place_key(const PlanArgs& a, int g, int (*sums)[2]) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int section = (a.pairs + kPlanThreads - 1) / kPlanThreads * 64;
  const int p0 = min(wave * section, a.pairs), p1 = min(p0 + section, a.pairs);
  uint32_t id[kBatch];
  auto load = [&](int at) {
    if (at + 64 * kBatch <= p1) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) id[i] = (uint32_t)a.ids[at + 64 * i + lane];
    } else {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) id[i] = (uint32_t)a.ids[min(at + 64 * i + lane, a.pairs - 1)];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) id[i] = at + 64 * i + lane < p1 ? id[i] : ~0u;
    }
  };
  auto own = [&](int at, int i) {
    if constexpr (kAbsent) return id[i] >= (uint32_t)g && at + 64 * i + lane < p1;
    return id[i] == (uint32_t)g;
  };
  int less = 0, same = 0;
  for (int at = p0; at < p1; at += 64 * kBatch) {
    load(at);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      less += id[i] < (uint32_t)g;
      same += own(at, i);
    }
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    less += __shfl_xor(less, m, 64);
    same += __shfl_xor(same, m, 64);
  }
  if (lane == 0) {
    sums[wave][0] = less;
    sums[wave][1] = same;
  }
  __syncthreads();
  int base = 0, row = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    base += sums[w][0];
    row += w < wave ? sums[w][1] : 0;
  }
  if (tid == 0) a.first[g] = base;
  if (__builtin_amdgcn_readfirstlane(same) == 0) return;
  row += base;
  const bool reload = section > 64 * kBatch;
  for (int at = p0; at < p1; at += 64 * kBatch) {
    if (reload) load(at);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const bool mine = own(at, i);
      const uint64_t mask = __ballot(mine);
      if (mask == 0) continue;
      if (mine) {
        const int r = row + __popcll(mask & ((1ull << lane) - 1)), p = at + 64 * i + lane;
        a.row_pair[r] = p;
        a.pair_row[p] = kAbsent ? -1 : r;
      }
      row += __popcll(mask);
    }
  }
}

template <int kBatch>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a) {
  __shared__ int sums[kPlanWaves][2];
  const int g = blockIdx.x;
  if (g == a.groups) place_key<true, kBatch>(a, g, sums);
  else place_key<false, kBatch>(a, g, sums);
}

// Many pairs: the pairs in up to kMaxChunks contiguous chunks and three launches, work in proportion to the pairs and
// to chunks x groups: count each chunk's keys; each chunk's first row of each group; place each chunk's pairs. There is
// no workspace: a chunk's counts lie in its own part of row_pair and its first rows in its own part of pair_row, which
// its workgroup has read before anyone writes there, so a chunk has at least G + 1 pairs.
//
// One launch against three, random ids, 8 a token: of 256 groups 32768 pairs 8.9 and 13.7 us, 131072 28 and 14, 2^21
// 383 and 31; of 1024 groups, whose workgroups are not all resident at once, 16384 pairs 12.7 and 17.7, 32768 20.7 and
// 18.1, 2^23 3961 and 128.
constexpr int kMaxChunks = 256, kChunkPairs = 2048;   // at least
constexpr int kChunkedPairs = 3 << 14;                // above this over the walk's rounds (512 workgroups each)
static_assert(kChunkPairs > kMaxGroups, "a chunk's part holds a number for every key");

struct ChunkArgs {
  PlanArgs plan;
  int32_t chunks;
  __device__ __forceinline__ int begin(int c) const { return (int)((int64_t)plan.pairs * c / chunks); }
};

__global__ __launch_bounds__(kPlanThreads) void plan_count_kernel(ChunkArgs a) {
  __shared__ int count[kMaxGroups + 1];
  const int tid = threadIdx.x, groups = a.plan.groups, p0 = a.begin(blockIdx.x), p1 = a.begin(blockIdx.x + 1);
  for (int g = tid; g <= groups; g += kPlanThreads) count[g] = 0;
  __syncthreads();
  constexpr int kBatch = 8;
  for (int at = p0 + tid; at < p1; at += kBatch * kPlanThreads) {
    uint32_t id[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) id[i] = (uint32_t)a.plan.ids[min(at + i * kPlanThreads, p1 - 1)];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (at + i * kPlanThreads < p1) atomicAdd(&count[min(id[i], (uint32_t)groups)], 1);
  }
  __syncthreads();
  for (int g = tid; g <= groups; g += kPlanThreads) a.plan.row_pair[p0 + g] = count[g];
}

// A workgroup 16 keys: thread (key, share of four chunks). What comes before its keys it counts for itself.
constexpr int kBaseKeys = 16, kShares = kPlanThreads / kBaseKeys, kPerShare = kMaxChunks / kShares;

__global__ __launch_bounds__(kPlanThreads) void plan_base_kernel(ChunkArgs a) {
  __shared__ int before[kPlanWaves], waves[kPlanWaves][kBaseKeys];
  const int tid = threadIdx.x, lane = tid & 63, groups = a.plan.groups, g0 = kBaseKeys * blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int key = g0 + tid % kBaseKeys, c0 = tid / kBaseKeys * kPerShare;
  int count[kPerShare], sum = 0;
#pragma unroll
  for (int i = 0; i < kPerShare; ++i) {
    const int v = a.plan.row_pair[a.begin(min(c0 + i, a.chunks - 1)) + min(key, groups)];
    count[i] = c0 + i < a.chunks && key <= groups ? v : 0;
    sum += count[i];
  }
  int below = 0;   // the smaller keys of chunks wave, wave + 16, ...
  for (int c = wave; c < a.chunks; c += 4 * kPlanWaves)
    for (int g = lane; g < g0; g += 64) {
      int v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = a.plan.row_pair[a.begin(min(c + i * kPlanWaves, a.chunks - 1)) + g];
#pragma unroll
      for (int i = 0; i < 4; ++i) below += c + i * kPlanWaves < a.chunks ? v[i] : 0;
    }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) below += __shfl_xor(below, m, 64);
  int upto = sum;   // of the wave's shares of this key up to this one
#pragma unroll
  for (int d = kBaseKeys; d < 64; d <<= 1) {
    const int o = __shfl_up(upto, d, 64);
    if (lane >= d) upto += o;
  }
  if (lane == 0) before[wave] = below;
  if (lane >= 64 - kBaseKeys) waves[wave][lane % kBaseKeys] = upto;
  __syncthreads();
  int row = upto - sum, total = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    row += before[w] + (w < wave ? waves[w][tid % kBaseKeys] : 0);
    total += waves[w][tid % kBaseKeys];
  }
  int smaller = total;
#pragma unroll
  for (int d = 1; d < kBaseKeys; d <<= 1) {
    const int o = __shfl_up(smaller, d, kBaseKeys);
    if (tid % kBaseKeys >= d) smaller += o;
  }
  row += smaller - total;
  if (key > groups) return;
  if (tid < kBaseKeys) a.plan.first[key] = row;
#pragma unroll
  for (int i = 0; i < kPerShare; ++i)
    if (c0 + i < a.chunks) {
      a.plan.pair_row[a.begin(c0 + i) + key] = row;
      row += count[i];
    }
}

// A chunk's waves take a contiguous section each and count its keys; the next row of each key and wave then stands in
// LDS, and 64 pairs at a time find their place among those of their key by a ballot for each bit of the key.
__global__ __launch_bounds__(kPlanThreads) void plan_place_kernel(ChunkArgs a, int bits) {
  extern __shared__ int next[];   // [kPlanWaves][groups + 1]
  const int tid = threadIdx.x, lane = tid & 63, groups = a.plan.groups;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int begin = a.begin(blockIdx.x), end = a.begin(blockIdx.x + 1);
  const int section = (end - begin + kPlanThreads - 1) / kPlanThreads * 64;
  const int p0 = min(begin + wave * section, end), p1 = min(p0 + section, end);
  int* own = next + wave * (groups + 1);
  for (int g = lane; g <= groups; g += 64) own[g] = 0;
  __syncthreads();
  constexpr int kBatch = 8;
  uint32_t key[kBatch];
  auto load = [&](int at) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) key[i] = min((uint32_t)a.plan.ids[min(at + 64 * i + lane, p1 - 1)], (uint32_t)groups);
  };
  for (int at = p0; at < p1; at += 64 * kBatch) {
    load(at);
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (at + 64 * i + lane < p1) atomicAdd(&own[key[i]], 1);
  }
  __syncthreads();
  for (int g = tid; g <= groups; g += kPlanThreads) {
    int row = a.plan.pair_row[begin + g];
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
      const int count = next[w * (groups + 1) + g];
      next[w * (groups + 1) + g] = row;
      row += count;
    }
  }
  __syncthreads();   // the chunk's part of pair_row has been read
  for (int at = p0; at < p1; at += 64 * kBatch) {
    if (section > 64 * kBatch) load(at);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int p = at + 64 * i + lane;
      if (at + 64 * i >= p1) break;
      uint64_t mask = __ballot(p < p1);   // the lanes with this lane's key
      for (int b = 0; b < bits; ++b) {
        const bool set = key[i] >> b & 1;
        const uint64_t with = __ballot(set);
        mask &= set ? with : ~with;
      }
      if (p < p1) {
        const int place = __popcll(mask & ((1ull << lane) - 1)), r = own[key[i]] + place;
        a.plan.row_pair[r] = p;
        a.plan.pair_row[p] = key[i] == (uint32_t)groups ? -1 : r;
        __builtin_amdgcn_wave_barrier();   // every lane has read its key's row before the first of the key moves it on
        if (place == 0) own[key[i]] = r + __popcll(mask);
      }
    }
  }
}

// Access to rows that the call touches once: past the caches where the call moves more than they hold (kStream).
template <bool kStream, typename R>
__device__ __forceinline__ R load_once(const R* p) {
  if constexpr (!kStream) {
    return *p;
  } else if constexpr (sizeof(R) == 16) {
    return __builtin_bit_cast(R, __builtin_nontemporal_load((const mxd::u32x4_t*)p));
  } else {
    return __builtin_nontemporal_load(p);
  }
}
template <bool kStream, typename R>
__device__ __forceinline__ void store_once(R* p, const R& v) {
  if constexpr (!kStream) {
    *p = v;
  } else if constexpr (sizeof(R) == 16) {
    __builtin_nontemporal_store(__builtin_bit_cast(mxd::u32x4_t, v), (mxd::u32x4_t*)p);
  } else {
    __builtin_nontemporal_store(v, p);
  }
}

struct DispatchArgs {
  PlanArgs plan;
  int32_t tokens, k;
  const uint8_t* x;
  uint8_t* rows;
  int64_t units;          // units of the copy per row
  const float* weights;
  float* row_weights;
};

// With the plan made in the same launch every workgroup counts for itself: a pair's key and index as one number, key <<
// 11 | p, orders the pairs, so row(p) is the count of smaller numbers and first[g] that of numbers below g << 11. One
// launch against the plan and the rows by it, 8 a token: 64 tokens 6.5 and 8.4 us, 128 8.1 and 9.1, 256 10.7 and 10.7,
// 512 16.0 and 14.9; one token 5.3.
constexpr int kIndexBits = 11, kFusedPairs = 1 << kIndexBits, kTargets = 8;

// count[n] = how many pairs come before target[n], for up to kTargets targets at once (the others' are not used): a
// thread holds P / 256 pairs, two counts share a register, and the waves' sums meet in LDS. `order` is this thread's
// pairs.
__device__ __forceinline__ void count_before(const uint32_t* order, int pairs, const uint32_t* target, int (*part)[kTargets],
                                             int* count) {
  const int tid = threadIdx.x;
  int low[kTargets / 2], high[kTargets / 2];
#pragma unroll
  for (int n = 0; n < kTargets / 2; ++n) low[n] = high[n] = 0;
#pragma unroll
  for (int i = 0; i < kFusedPairs / 256; ++i)
    if (256 * i < pairs) {
#pragma unroll
      for (int n = 0; n < kTargets / 2; ++n) {
        low[n] += order[i] < target[2 * n];
        high[n] += order[i] < target[2 * n + 1];
      }
    }
#pragma unroll
  for (int n = 0; n < kTargets / 2; ++n) {
    int both = low[n] | high[n] << 16;   // at most 512 a wave
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) both += __shfl_xor(both, m, 64);
    if ((tid & 63) == 0) {
      part[tid >> 6][2 * n] = both & 0xFFFF;
      part[tid >> 6][2 * n + 1] = both >> 16;
    }
  }
  __syncthreads();
  if (tid < kTargets) count[tid] = part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid];
  __syncthreads();
}

// The token's row is read once and written to each of its rows. U is the widest unit that the row's bytes and the
// pointers allow.
//
// By a plan: one wave per token and piece of 64 units (chunks pieces a row; more units, more rounds). 4096 tokens to 8
// rows of 7168 BF16 values each: 90 us, 5.9 TB/s, against 72 for a fill of the same rows; with plain stores 104, with
// loads past the caches too 108, a row's workgroup fetching its token 128, workgroups of 448 threads 93.
template <typename U, bool kStream>
__global__ __launch_bounds__(64) void move_rows_kernel(DispatchArgs a, int chunks) {
  const int t = blockIdx.x / chunks, chunk = blockIdx.x % chunks, lane = threadIdx.x, k = a.k, pairs = a.tokens * k;
  if (a.row_weights && chunk == 0 && lane < k) {
    const int r = a.plan.pair_row[t * k + lane];
    if (r >= 0 && r < pairs) a.row_weights[r] = a.weights[t * k + lane];
  }
  const U* x = (const U*)a.x + (int64_t)t * a.units;
  for (int64_t c = 64 * chunk + lane; c < a.units; c += 64 * chunks) {
    const U v = x[c];
    for (int j = 0; j < k; ++j) {
      const int r = a.plan.pair_row[t * k + j];
      if (r >= 0 && r < pairs) store_once<kStream>((U*)a.rows + (int64_t)r * a.units + c, v);
    }
  }
}

// With the plan, in one launch for few pairs: grid (T + workgroups of kTargets groups, chunks); every workgroup finds
// its own token's rows, the first chunk's writes them, and the workgroups past the tokens the groups' first rows.
template <typename U, bool kStream>
__global__ __launch_bounds__(256) void dispatch_kernel(DispatchArgs a) {
  __shared__ int dst[kMaxTopK];
  __shared__ int part[4][kTargets];
  __shared__ int count[kTargets];
  const int t = blockIdx.x, tid = threadIdx.x, k = a.k, pairs = a.plan.pairs;
  if (t >= a.tokens && blockIdx.y > 0) return;
  uint32_t order[kFusedPairs / 256];
#pragma unroll
  for (int i = 0; i < kFusedPairs / 256; ++i)
    if (256 * i < pairs) order[i] = (uint32_t)a.plan.ids[min(256 * i + tid, pairs - 1)];
#pragma unroll
  for (int i = 0; i < kFusedPairs / 256; ++i)
    if (256 * i < pairs) {
      const int p = 256 * i + tid;
      const uint32_t key = min(order[i], (uint32_t)a.plan.groups);   // ids below zero are large as unsigned numbers
      order[i] = p < pairs ? key << kIndexBits | p : ~0u;
    }
  uint32_t target[kTargets];
  if (t >= a.tokens) {
    const int g0 = (t - a.tokens) * kTargets;
#pragma unroll
    for (int n = 0; n < kTargets; ++n) target[n] = (uint32_t)(g0 + n) << kIndexBits;
    count_before(order, pairs, target, part, count);
    if (tid < kTargets && g0 + tid <= a.plan.groups) a.plan.first[g0 + tid] = count[tid];
    return;
  }
  for (int j0 = 0; j0 < k; j0 += kTargets) {
#pragma unroll
    for (int n = 0; n < kTargets; ++n) {
      const int p = t * k + min(j0 + n, k - 1);
      target[n] = min((uint32_t)a.plan.ids[p], (uint32_t)a.plan.groups) << kIndexBits | p;
    }
    count_before(order, pairs, target, part, count);
    const int j = j0 + tid;
    if (tid < kTargets && j < k) {
      const int p = t * k + j, r = count[tid];
      const bool absent = (uint32_t)a.plan.ids[p] >= (uint32_t)a.plan.groups;
      if (blockIdx.y == 0) {
        a.plan.row_pair[r] = p;
        a.plan.pair_row[p] = absent ? -1 : r;
        if (!absent && a.row_weights) a.row_weights[r] = a.weights[p];
      }
      dst[j] = absent ? -1 : r;
    }
  }
  __syncthreads();
  const U* x = (const U*)a.x + (int64_t)t * a.units;
  for (int64_t c = (int64_t)blockIdx.y * 256 + tid; c < a.units; c += (int64_t)gridDim.y * 256) {
    const U v = x[c];
    for (int j = 0; j < k; ++j) {
      const int r = __builtin_amdgcn_readfirstlane(dst[j]);
      if (r >= 0) store_once<kStream>((U*)a.rows + (int64_t)r * a.units + c, v);
    }
  }
}

// ---- units of a row as FP32 values ----

template <int kType, int V>
struct Unit;

template <>
struct Unit<MX_ROWS_BF16, 8> {
  typedef uint4 Raw;
  static __device__ __forceinline__ void values(const Raw& r, float* v) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = mx::u2f(w[i] << 16);
      v[2 * i + 1] = mx::u2f(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ Raw round(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = mxd::bf16_pair(v[2 * i], v[2 * i + 1]);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

template <>
struct Unit<MX_ROWS_BF16, 1> {
  typedef uint16_t Raw;
  static __device__ __forceinline__ void values(const Raw& r, float* v) { v[0] = mx::bf16_value(r); }
  static __device__ __forceinline__ Raw round(const float* v) { return (uint16_t)mx::bf16_bits(v[0]); }
};

template <>
struct Unit<MX_ROWS_F32, 4> {
  typedef uint4 Raw;
  static __device__ __forceinline__ void values(const Raw& r, float* v) {
    v[0] = mx::u2f(r.x), v[1] = mx::u2f(r.y), v[2] = mx::u2f(r.z), v[3] = mx::u2f(r.w);
  }
  static __device__ __forceinline__ Raw round(const float* v) {
    return make_uint4(mx::f2u(v[0]), mx::f2u(v[1]), mx::f2u(v[2]), mx::f2u(v[3]));
  }
};

template <>
struct Unit<MX_ROWS_F32, 1> {
  typedef float Raw;
  static __device__ __forceinline__ void values(const Raw& r, float* v) { v[0] = r; }
  static __device__ __forceinline__ Raw round(const float* v) { return v[0]; }
};

// ---- combine, and the backward pass of dispatch ----

struct CombineArgs {
  const void* rows;
  const int32_t* pair_row;
  const float* weights;        // [T][k] or null
  const void* shared;          // [T][width] or null
  void* y;
  int32_t tokens, k;
  int64_t units;               // units per row
  const float* row_weights;    // dispatch_backward: the gradient of each row's weight, and
  float* dweights;             // where it goes
  bool stream;
};

// acc += (w *) rows, N of them in flight together; row and weight j are those of lane j0 + j.
template <int N, bool kStream, typename X, int V>
__device__ __forceinline__ void add_rows(const typename X::Raw* rows, int64_t units, int64_t c, int row, float weight,
                                         int j0, bool weighted, float* acc) {
  typename X::Raw raw[N];
#pragma unroll
  for (int j = 0; j < N; ++j)
    raw[j] = load_once<kStream>(rows + (int64_t)__builtin_amdgcn_readlane(row, j0 + j) * units + c);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float v[V];
    X::values(raw[j], v);
    const float w = mx::u2f(__builtin_amdgcn_readlane(mx::f2u(weight), j0 + j));
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = acc[i] + (weighted ? w * v[i] : v[i]);
  }
}

template <int kType, int V, bool kStream>
__device__ __forceinline__ void combine_units(const CombineArgs& a, int t, int64_t c0, int64_t step, int row,
                                              float weight, int n) {
  using X = Unit<kType, V>;
  using Raw = typename X::Raw;
  const Raw* rows = (const Raw*)a.rows;
  const bool weighted = a.weights != nullptr;
  for (int64_t c = c0; c < a.units; c += step) {
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    Raw shared{};
    if (a.shared) shared = load_once<kStream>((const Raw*)a.shared + (int64_t)t * a.units + c);
    int j = 0;
    for (; j + 8 <= n; j += 8) add_rows<8, kStream, X, V>(rows, a.units, c, row, weight, j, weighted, acc);
    if (n & 4) add_rows<4, kStream, X, V>(rows, a.units, c, row, weight, j, weighted, acc), j += 4;
    if (n & 2) add_rows<2, kStream, X, V>(rows, a.units, c, row, weight, j, weighted, acc), j += 2;
    if (n & 1) add_rows<1, kStream, X, V>(rows, a.units, c, row, weight, j, weighted, acc);
    if (a.shared) {
      float v[V];
      X::values(shared, v);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = acc[i] + v[i];
    }
    ((Raw*)a.y)[(int64_t)t * a.units + c] = X::round(acc);
  }
}

// One wave per token and piece of 64 units (chunks pieces a row; more units, more rounds), a unit of 16 bytes (or one
// value) a lane, up to eight rows in flight. Lane j holds the token's pair j; each counts the rows before its own and
// sends it to the lane of that number.
//
// Bound by HBM reads: 4096 x 8 rows of 7168 (529 MB read, 59 written) take 99 us, 5.9 TB/s. At most five waves a SIMD,
// so that the rows in flight fit what the memory takes in order: six or eight 107, four 101, three 104; the unweighted
// sum 98 / 91 / 95 / 99. Calls of rows from the caches neither gain nor lose by it: 16 tokens 5.1 us, 333 of 6 FP32 rows
// of 5120 unweighted 9.7 (9.8 without).
template <int kType, int V>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(1, 5))) void combine_kernel(CombineArgs a, int chunks) {
  const int t = blockIdx.x / chunks, chunk = blockIdx.x % chunks, lane = threadIdx.x, k = a.k, pairs = a.tokens * k;
  int r = -1;
  float w = 1.f;
  if (lane < k) {
    r = a.pair_row[t * k + lane];
    r = r >= 0 && r < pairs ? r : -1;
    if (a.weights) w = a.weights[t * k + lane];
  }
  if (a.dweights && chunk == 0 && lane < k) a.dweights[t * k + lane] = r >= 0 ? a.row_weights[r] : 0.f;
  int before = 0;
  for (int j = 0; j < k; ++j) {
    const int o = __builtin_amdgcn_readlane(r, j);
    before += o >= 0 && (o < r || (o == r && j < lane));
  }
  const int n = __popcll(__ballot(r >= 0));
  const int to = 4 * (r >= 0 ? before : 63);   // lane 63 is no one's: k <= 32
  const int row = __builtin_amdgcn_ds_permute(to, r);
  const float weight = mx::u2f(__builtin_amdgcn_ds_permute(to, (int)mx::f2u(w)));
  const int64_t c0 = 64 * (int64_t)chunk + lane, step = 64 * (int64_t)chunks;
  if (a.stream && n == k) combine_units<kType, V, true>(a, t, c0, step, row, weight, n);
  else combine_units<kType, V, false>(a, t, c0, step, row, weight, n);
}

// ---- the backward pass of combine ----

constexpr int kInFlight = 4;   // units of a row, and of dy, that a thread has in flight

struct CombineBwdArgs {
  const void* dy;
  const void* rows;            // null: no gradient of the weights
  const int32_t* pair_row;
  const float* weights;
  void* drows;                 // null: no gradient of the rows
  float* dweights;
  int32_t tokens, k;
  int64_t units;
  bool stream;
};

template <int kType, int V, bool kStream>
__device__ __forceinline__ float backward_units(const CombineBwdArgs& a, int t, int r, float w) {
  using X = Unit<kType, V>;
  using Raw = typename X::Raw;
  const Raw* dy = (const Raw*)a.dy + (int64_t)t * a.units;
  const Raw* row = (const Raw*)a.rows + (int64_t)r * a.units;
  Raw* out = (Raw*)a.drows + (int64_t)r * a.units;
  const int threads = blockDim.x;
  float dot = 0.f;
  for (int64_t c0 = threadIdx.x; c0 < a.units; c0 += kInFlight * threads) {
    Raw dy_raw[kInFlight], row_raw[kInFlight];
#pragma unroll
    for (int s = 0; s < kInFlight; ++s) {
      const int64_t c = c0 + s * threads;
      if (c < a.units) {
        if (a.dweights) row_raw[s] = load_once<kStream>(row + c);
        dy_raw[s] = dy[c];
      }
    }
#pragma unroll
    for (int s = 0; s < kInFlight; ++s) {
      const int64_t c = c0 + s * threads;
      if (c >= a.units) continue;
      float g[V], v[V];
      X::values(dy_raw[s], g);
      if (a.dweights) {
        X::values(row_raw[s], v);
#pragma unroll
        for (int e = 0; e < V; ++e) dot = dot + g[e] * v[e];
      }
      if (a.drows) {
#pragma unroll
        for (int e = 0; e < V; ++e) g[e] = a.weights ? w * g[e] : g[e];
        store_once<kStream>(out + c, X::round(g));
      }
    }
  }
  return dot;
}

// One workgroup a pair: drows[row] = w dy[t] and dw = <rows[row], dy[t]>, both from one read of dy and of the row. Each
// thread adds its products in order, the lanes are added as a tree and the waves in order. A token's pairs run on one
// XCD (workgroups go round the eight of them), so its dy comes from HBM once and from that L2 after. 4096 x 8 rows of
// 7168 BF16 values (998 MB): 178 us, 5.6 TB/s; pairs in plain order 195, rows read through the caches 189, gradients
// written through them 195; two units a thread of 512 instead of four of 256: 181. At most five waves a SIMD: 179 without
// that, and 1500 tokens of FP32 rows of 5120, an eighth of their six held, 12.8 in place of 13.2, which it costs.
template <int kType, int V>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 5))) void combine_backward_kernel(CombineBwdArgs a) {
  __shared__ float part[4];
  const int tid = threadIdx.x, lane = tid & 63, k = a.k, pairs = a.tokens * k;
  const int i = blockIdx.x >> 3;
  const int t = i / k * 8 + (blockIdx.x & 7), j = i % k;
  if (t >= a.tokens) return;
  int own = -1;
  if (lane < k) own = a.pair_row[t * k + lane];
  const int n = __popcll(__ballot(own >= 0));
  const int r = __builtin_amdgcn_readlane(own, j);
  if (r < 0 || r >= pairs) {
    if (a.dweights && tid == 0) a.dweights[t * k + j] = 0.f;
    return;
  }
  const float w = a.weights ? a.weights[t * k + j] : 1.f;
  float dot = a.stream && n == k ? backward_units<kType, V, true>(a, t, r, w) : backward_units<kType, V, false>(a, t, r, w);
  if (!a.dweights) return;
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) dot = dot + __shfl_xor(dot, m, 64);
  if (lane == 0) part[tid >> 6] = dot;
  __syncthreads();
  if (tid == 0) {
    float sum = part[0];
    for (int v = 1; v < (int)blockDim.x / 64; ++v) sum = sum + part[v];
    a.dweights[t * k + j] = sum;
  }
}

bool is_aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

int check_routing(const char* who, int32_t tokens, int32_t top_k) {
  MX_REQUIRE(tokens >= 0 && tokens <= kMaxTokens, "%s: token count %d outside [0, %d]", who, tokens, kMaxTokens);
  MX_REQUIRE(top_k >= 1 && top_k <= kMaxTopK, "%s: %d groups per token outside [1, %d]", who, top_k, kMaxTopK);
  return MX_OK;
}

int check_plan(const char* who, const mx_row_plan* plan) {
  MX_REQUIRE(plan && plan->first && plan->pair_row && plan->row_pair, "%s: plan pointer is null", who);
  MX_REQUIRE(is_aligned(plan->first, 4) && is_aligned(plan->pair_row, 4) && is_aligned(plan->row_pair, 4),
             "%s: plan arrays must be 4-byte aligned", who);
  return MX_OK;
}

int check_rows(const char* who, int32_t dtype, int64_t width, bool bytes_too) {
  MX_REQUIRE(dtype == MX_ROWS_BF16 || dtype == MX_ROWS_F32 || (bytes_too && dtype == MX_ROWS_U8), "%s: row type %d",
             who, dtype);
  MX_REQUIRE(width >= 1 && width <= kMaxWidth, "%s: row width %lld outside [1, %lld]", who, (long long)width,
             (long long)kMaxWidth);
  return MX_OK;
}

int64_t element_bytes(int32_t dtype) { return dtype == MX_ROWS_F32 ? 4 : dtype == MX_ROWS_BF16 ? 2 : 1; }

// Pieces of 64 units of a row, as many as keep the grid below 2^25 waves.
int chunks_of(int tokens, int64_t units) { return (int)std::min<int64_t>((units + 63) / 64, (1 << 25) / tokens); }

// Whether a call of `row_bytes` rows, `moves` of them a pair and one a token, goes past the caches.
bool streams(int tokens, int k, int64_t row_bytes, int moves) {
  return (int64_t)tokens * (moves * k + 1) * row_bytes > kStreamBytes;
}

template <typename U>
int launch_dispatch(DispatchArgs a, int64_t row_bytes, bool fused, hipStream_t st) {
  a.units = row_bytes / (int64_t)sizeof(U);
  const bool stream = streams(a.tokens, a.k, row_bytes, 1);
  if (fused) {
    // a row in pieces only where the tokens leave room: each piece's workgroup counts anew
    const unsigned chunks = (unsigned)std::min<int64_t>((a.units + 255) / 256, std::max(1, 1024 / std::max(a.tokens, 1)));
    const dim3 grid(a.tokens + (a.plan.groups + kTargets) / kTargets, chunks);
    hipLaunchKernelGGL((stream ? dispatch_kernel<U, true> : dispatch_kernel<U, false>), grid, dim3(256), 0, st, a);
  } else {
    const int chunks = chunks_of(a.tokens, a.units);
    hipLaunchKernelGGL((stream ? move_rows_kernel<U, true> : move_rows_kernel<U, false>), dim3(a.tokens * chunks),
                       dim3(64), 0, st, a, chunks);
  }
  MX_LAUNCH_CHECK("dispatch_kernel");
  return MX_OK;
}

template <int kType, int V>
int launch_combine(CombineArgs a, int64_t width, hipStream_t st) {
  a.units = width / V;
  const int chunks = chunks_of(a.tokens, a.units);
  a.stream = streams(a.tokens, a.k, a.units * (int64_t)sizeof(typename Unit<kType, V>::Raw), 1);
  hipLaunchKernelGGL((combine_kernel<kType, V>), dim3(a.tokens * chunks), dim3(64), 0, st, a, chunks);
  MX_LAUNCH_CHECK("combine_kernel");
  return MX_OK;
}

int combine_any(const CombineArgs& a, int32_t dtype, int64_t width, hipStream_t st) {
  const bool wide = (width * element_bytes(dtype)) % 16 == 0 && is_aligned(a.rows, 16) && is_aligned(a.y, 16) &&
                    (!a.shared || is_aligned(a.shared, 16));
  if (dtype == MX_ROWS_BF16)
    return wide ? launch_combine<MX_ROWS_BF16, 8>(a, width, st) : launch_combine<MX_ROWS_BF16, 1>(a, width, st);
  return wide ? launch_combine<MX_ROWS_F32, 4>(a, width, st) : launch_combine<MX_ROWS_F32, 1>(a, width, st);
}

template <int kType, int V>
int launch_combine_backward(CombineBwdArgs a, int64_t width, hipStream_t st) {
  a.units = width / V;
  const unsigned grid = (unsigned)((a.tokens + 7) / 8 * 8 * a.k);
  // as few equal rounds as kInFlight units a thread of 256 allow
  const int64_t rounds = (a.units + 256 * kInFlight - 1) / (256 * kInFlight), per = rounds * kInFlight;
  const unsigned threads = (unsigned)(((a.units + per - 1) / per + 63) / 64 * 64);
  a.stream = streams(a.tokens, a.k, a.units * (int64_t)sizeof(typename Unit<kType, V>::Raw), 2);
  hipLaunchKernelGGL((combine_backward_kernel<kType, V>), dim3(grid), dim3(threads), 0, st, a);
  MX_LAUNCH_CHECK("combine_backward_kernel");
  return MX_OK;
}

}  // namespace

using mxi::as_stream;
using mxi::use;

int mxi::row_plan(const int32_t* ids, int32_t pairs, int32_t groups, const mx_row_plan& plan, hipStream_t st) {
  const PlanArgs a{ids, pairs, groups, plan.first, plan.pair_row, plan.row_pair};
  if (pairs > kChunkedPairs / (groups / 512 + 1)) {
    const ChunkArgs c{a, std::min(kMaxChunks, pairs / kChunkPairs)};
    hipLaunchKernelGGL(plan_count_kernel, dim3(c.chunks), dim3(kPlanThreads), 0, st, c);
    MX_LAUNCH_CHECK("plan_count_kernel");
    hipLaunchKernelGGL(plan_base_kernel, dim3(groups / kBaseKeys + 1), dim3(kPlanThreads), 0, st, c);
    MX_LAUNCH_CHECK("plan_base_kernel");
    int bits = 1;
    while (groups >> bits) ++bits;
    hipLaunchKernelGGL(plan_place_kernel, dim3(c.chunks), dim3(kPlanThreads), kPlanWaves * (groups + 1) * sizeof(int), st, c,
                       bits);
    MX_LAUNCH_CHECK("plan_place_kernel");
    return MX_OK;
  }
  if (pairs <= 8 * kPlanThreads) hipLaunchKernelGGL(plan_kernel<8>, dim3(groups + 1), dim3(kPlanThreads), 0, st, a);
  else if (pairs <= 16 * kPlanThreads) hipLaunchKernelGGL(plan_kernel<16>, dim3(groups + 1), dim3(kPlanThreads), 0, st, a);
  else hipLaunchKernelGGL(plan_kernel<32>, dim3(groups + 1), dim3(kPlanThreads), 0, st, a);
  MX_LAUNCH_CHECK("plan_kernel");
  return MX_OK;
}

extern "C" {

int mx_dispatch(mx_ctx* ctx, const int32_t* ids, int32_t tokens, int32_t top_k, int32_t groups, const mx_row_plan* plan,
                const void* x, int32_t dtype, int64_t width, const float* weights, void* rows, float* row_weights,
                void* stream) {
  const char* who = "mx_dispatch";
  if (int s = check_routing(who, tokens, top_k)) return s;
  MX_REQUIRE(groups >= 1 && groups <= kMaxGroups, "%s: %d groups outside [1, %d]", who, groups, kMaxGroups);
  if (int s = check_plan(who, plan)) return s;
  MX_REQUIRE((x == nullptr) == (rows == nullptr), "%s: x and rows are given together or not at all", who);
  MX_REQUIRE((weights == nullptr) == (row_weights == nullptr), "%s: weights and row_weights are given together", who);
  MX_REQUIRE(ids || x, "%s: neither ids for a plan nor rows to move", who);
  MX_REQUIRE(x || !weights, "%s: weights move with rows", who);
  MX_REQUIRE(is_aligned(ids, 4) && is_aligned(weights, 4) && is_aligned(row_weights, 4),
             "%s: ids and weights must be 4-byte aligned", who);
  if (x) {
    if (int s = check_rows(who, dtype, width, true)) return s;
    MX_REQUIRE(is_aligned(x, element_bytes(dtype)) && is_aligned(rows, element_bytes(dtype)),
               "%s: x and rows must be aligned to their elements", who);
    MX_REQUIRE(rows != x, "%s: rows may not be x", who);
  }
  if (int s = use(ctx)) return s;
  hipStream_t st = as_stream(stream);
  const int32_t pairs = tokens * top_k;
  const bool fused = ids && x && pairs <= kFusedPairs;
  if (ids && !fused)
    if (int s = mxi::row_plan(ids, pairs, groups, *plan, st)) return s;
  if (!x || (!tokens && !fused)) return MX_OK;
  DispatchArgs a{{ids, pairs, groups, plan->first, plan->pair_row, plan->row_pair}, tokens, top_k, (const uint8_t*)x,
                 (uint8_t*)rows, 0, weights, row_weights};
  const int64_t bytes = width * element_bytes(dtype);
  const uint64_t low = (uint64_t)(uintptr_t)x | (uint64_t)(uintptr_t)rows | (uint64_t)bytes;
  if (low % 16 == 0) return launch_dispatch<uint4>(a, bytes, fused, st);
  if (low % 4 == 0) return launch_dispatch<uint32_t>(a, bytes, fused, st);
  if (low % 2 == 0) return launch_dispatch<uint16_t>(a, bytes, fused, st);
  return launch_dispatch<uint8_t>(a, bytes, fused, st);
}

int mx_combine(mx_ctx* ctx, const void* rows, int32_t dtype, const int32_t* pair_row, const float* weights,
               const void* shared, int32_t tokens, int32_t top_k, int64_t width, void* y, void* stream) {
  const char* who = "mx_combine";
  if (int s = check_routing(who, tokens, top_k)) return s;
  if (int s = check_rows(who, dtype, width, false)) return s;
  MX_REQUIRE(rows && pair_row && y, "%s: null pointer", who);
  const int64_t size = element_bytes(dtype);
  MX_REQUIRE(is_aligned(rows, size) && is_aligned(y, size) && is_aligned(shared, size) && is_aligned(pair_row, 4) &&
                 is_aligned(weights, 4),
             "%s: pointers must be aligned to their elements", who);
  MX_REQUIRE(y != rows, "%s: y may not be rows", who);
  if (int s = use(ctx)) return s;
  if (!tokens) return MX_OK;
  const CombineArgs a{rows, pair_row, weights, shared, y, tokens, top_k, 0, nullptr, nullptr, false};
  return combine_any(a, dtype, width, as_stream(stream));
}

int mx_combine_backward(mx_ctx* ctx, const void* dy, const void* rows, int32_t dtype, const int32_t* pair_row,
                        const float* weights, int32_t tokens, int32_t top_k, int64_t width, void* drows,
                        float* dweights, void* stream) {
  const char* who = "mx_combine_backward";
  if (int s = check_routing(who, tokens, top_k)) return s;
  if (int s = check_rows(who, dtype, width, false)) return s;
  MX_REQUIRE(dy && pair_row, "%s: null pointer", who);
  MX_REQUIRE(drows || dweights, "%s: no gradient asked for", who);
  MX_REQUIRE(!dweights || rows, "%s: the gradient of the weights needs the rows", who);
  const int64_t size = element_bytes(dtype);
  MX_REQUIRE(is_aligned(dy, size) && is_aligned(rows, size) && is_aligned(drows, size) && is_aligned(pair_row, 4) &&
                 is_aligned(weights, 4) && is_aligned(dweights, 4),
             "%s: pointers must be aligned to their elements", who);
  MX_REQUIRE(drows != dy, "%s: drows may not be dy", who);
  if (int s = use(ctx)) return s;
  if (!tokens) return MX_OK;
  const CombineBwdArgs a{dy, rows, pair_row, weights, drows, dweights, tokens, top_k, 0, false};
  const bool wide = (width * size) % 16 == 0 && is_aligned(dy, 16) && (!dweights || is_aligned(rows, 16)) &&
                    is_aligned(drows, 16);
  hipStream_t st = as_stream(stream);
  if (dtype == MX_ROWS_BF16)
    return wide ? launch_combine_backward<MX_ROWS_BF16, 8>(a, width, st)
                : launch_combine_backward<MX_ROWS_BF16, 1>(a, width, st);
  return wide ? launch_combine_backward<MX_ROWS_F32, 4>(a, width, st)
              : launch_combine_backward<MX_ROWS_F32, 1>(a, width, st);
}

int mx_dispatch_backward(mx_ctx* ctx, const void* drows, int32_t dtype, const int32_t* pair_row,
                         const float* drow_weights, int32_t tokens, int32_t top_k, int64_t width, void* dx,
                         float* dweights, void* stream) {
  const char* who = "mx_dispatch_backward";
  if (int s = check_routing(who, tokens, top_k)) return s;
  if (int s = check_rows(who, dtype, width, false)) return s;
  MX_REQUIRE(drows && pair_row && dx, "%s: null pointer", who);
  MX_REQUIRE((drow_weights == nullptr) == (dweights == nullptr), "%s: drow_weights and dweights are given together",
             who);
  const int64_t size = element_bytes(dtype);
  MX_REQUIRE(is_aligned(drows, size) && is_aligned(dx, size) && is_aligned(pair_row, 4) &&
                 is_aligned(drow_weights, 4) && is_aligned(dweights, 4),
             "%s: pointers must be aligned to their elements", who);
  MX_REQUIRE(dx != drows, "%s: dx may not be drows", who);
  if (int s = use(ctx)) return s;
  if (!tokens) return MX_OK;
  const CombineArgs a{drows, pair_row, nullptr, nullptr, dx, tokens, top_k, 0, drow_weights, dweights, false};
  return combine_any(a, dtype, width, as_stream(stream));
}

}  // extern "C"
