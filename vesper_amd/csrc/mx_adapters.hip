// Low-rank adapters of many requests beside a projection: y[t] = base[t] + scale_a up_a (down_a x[t]), a = ids[t].
//
// The quantized base weights cannot take an adapter in, so each token's pair of thin matrices runs beside them: down
// [rank][K] then up [N][rank], both BF16, with the projection's output (BF16, or its FP32 sums) as base and one
// rounding. Both products run on V_MFMA_F32_16X16X32_BF16 with the weights as operand A and tokens as operand B's
// columns:
//   A lane l = row l % 16, K 8 (l / 16) + 0..7; B lane l = column l % 16, same K; D lane l register i = row 4 (l / 16)
//   + i, column l % 16.
// So down's D gives lane (token, q) the ranks 4q..4q+3 of a 16-rank tile, which is what up's operand B wants of that
// lane. h = scale * (down x) is FP32 up to there and loses nothing: its 24 bits are three BF16 terms of 8 (the top half
// of its bits, the top half of what that leaves, and the rest, as far as BF16's smallest numbers reach). A tile's 16
// ranks take one MFMA, K slots 0..3 of a lane holding its ranks' first terms and 4..7 their second against up's values
// given twice, and a second one, or half of one that two tiles share, for the third. No load of up is repeated.
//
// The bank stores each slot in operand order, padded with zeros to whole tiles:
//   down: [rank tile][K chunk of 32][lane] 16 bytes: rank 16 rt + l % 16, K 32 c + 8 (l / 16) + 0..7
//   up: [block of 64 outputs][rank tile][half][lane] 16 bytes: two tiles j = 0, 1 of four ranks each; row m of tile j of
//   a half is output 64 b + 32 half + 8 (m / 4) + 4 j + m % 4, so a lane's D registers of a half's two tiles are 8
//   consecutive outputs of its token and the four lanes of a token 32 (64 bytes of y).
//
// Three forms. Calls of few tokens are bound by the weights of the adapters they name and by their launches, so each
// token's workgroups find the tokens that share its adapter by a ballot, one launch or two. Larger calls sort the
// tokens by adapter into tiles of 64 and read each weight once a tile; x, base and y, once each, then bound them.
#include <algorithm>
#include <cmath>
#include <new>

#include "mx_device.h"
#include "mx_internal.h"
#include "mx_numerics.h"

namespace {

using mxd::ldg128;
using mxd::v4f;

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

constexpr int kMaxTokens = 1 << 18, kMaxSlots = 1024, kMaxRank = 256;
constexpr int kMaxWidth = 1 << 20;
constexpr int kFewTokens = 128;    // a wave holds the ids of this many tokens, in two registers
constexpr int kTileTokens = 64;    // tokens of a workgroup in the grouped form
constexpr int kColumns = kTileTokens / 16;
constexpr int kMostTiles = 8;      // rank tiles that up's waves hold at once; of more, kTurnTiles in turn
constexpr int kTurnTiles = 4;
constexpr int kMaxParts = 32;      // parts of K
// A call of few tokens is one launch if down and the x of its tokens (of 64 at most, since the tokens of a workgroup
// are 16 of one adapter) are no more than this: each of its workgroups reads all of down. One launch and two, rank 12
// (one rank tile), BF16 base, tokens of adapters: 1536 columns and 24576 rows, 1 of 1 4.5 and 7.1 us, 16 of 16 7.2 and
// 9.8, 120 of 2 13.0 and 14.9; 5120 and 1280, 1 of 1 5.7 and 8.4, 16 of 4 6.9 and 8.6, 40 of 9 7.2 and 8.8, 64 of 3 10.3
// and 9.0; 7168 and 1536, 4 of 4 6.8 and 8.4, 16 of 1 9.8 and 8.5, of 16 7.4 and 8.5, 64 of 3 12.4 and 9.1; 16384 and
// 7168, 1 of 1 10.9 and 8.6. Rank 32: 1536 and 24576, 120 of 2 15.9 and 16.6; 7168 and 1536, 1 of 1 8.6 and 8.4. Four
// rank tiles take too many registers: 10.2 and 7.1.
constexpr int kFusedBytes = 320 << 10;
// Calls whose x, base and y exceed this read x past the caches, which leaves them to the weights, base and y. Past them
// and through, three sets in turn, BF16 base, 8 adapters: of rank 64, 1000 tokens of 16384 to 7168 (62 MB) 30.9 and 31.0
// us, 1500 (92 MB) 34.8 and 38.5, 2000 (123 MB) 41.7 and 46.9, 4096 (252 MB) 74.0 and 73.9; of rank 32, 2500 of 7168 to
// 1536 (51 MB) 24.2 and 22.7, 4000 (82 MB) 29.8 and 28.8. (For y it makes no difference.)
constexpr int64_t kStreamBytes = 80 << 20;
constexpr int kWantGroups = 512;   // workgroups that the split of K aims at

struct AdapterSlot {
  int32_t rank;   // 0: empty
  float scale;
};

struct Bank {
  const uint8_t* down;
  const uint8_t* up;
  const AdapterSlot* table;
  int32_t n, k, slots;
  int32_t rank_tiles, chunks, blocks;   // of the largest rank; K chunks of 32 (an even count); blocks of 64 outputs
  __host__ __device__ int64_t down_bytes() const { return (int64_t)rank_tiles * chunks * 1024; }
  __host__ __device__ int64_t up_bytes() const { return (int64_t)blocks * rank_tiles * 2048; }
  // a block of a slot; what is past the bank repeats its last block, and no slot is the first
  __device__ __forceinline__ const uint8_t* up_at(int slot, int block) const {
    return up + max(slot, 0) * up_bytes() + (int64_t)min(block, blocks - 1) * rank_tiles * 2048;
  }
};

__device__ __forceinline__ v8bf as_bf(uint4 v) { return __builtin_bit_cast(v8bf, v); }

// ---- loading a slot ----

__global__ __launch_bounds__(64) void adapter_store_down_kernel(Bank b, uint8_t* bank, int slot, const uint16_t* src,
                                                                int rank) {
  const int lane = threadIdx.x, c = blockIdx.x, rt = blockIdx.y;
  const int r = 16 * rt + (lane & 15), k0 = 32 * c + 8 * (lane >> 4);
  uint32_t w[4] = {0, 0, 0, 0};
  for (int i = 0; i < 8; ++i) {
    const uint32_t v = r < rank && k0 + i < b.k ? src[(int64_t)r * b.k + k0 + i] : 0;
    w[i >> 1] |= v << (16 * (i & 1));
  }
  uint8_t* dst = bank + slot * b.down_bytes() + ((int64_t)rt * b.chunks + c) * 1024 + 16 * lane;
  *(uint4*)dst = make_uint4(w[0], w[1], w[2], w[3]);
}

__global__ __launch_bounds__(128) void adapter_store_up_kernel(Bank b, uint8_t* bank, AdapterSlot* table, int slot,
                                                         const uint16_t* src, int rank, float scale) {
  const int lane = threadIdx.x & 63, half = threadIdx.x >> 6, block = blockIdx.x, rt = blockIdx.y;
  if (block == 0 && rt == 0 && threadIdx.x == 0) table[slot] = AdapterSlot{rank, scale};
  if (rank == 0) return;
  const int m = lane & 15, r0 = 16 * rt + 4 * (lane >> 4);
  uint32_t w[4] = {0, 0, 0, 0};
  for (int i = 0; i < 8; ++i) {
    const int n = 64 * block + 32 * half + 8 * (m >> 2) + 4 * (i >> 2) + (m & 3), r = r0 + (i & 3);
    const uint32_t v = n < b.n && r < rank ? src[(int64_t)n * rank + r] : 0;
    w[i >> 1] |= v << (16 * (i & 1));
  }
  uint8_t* dst = bank + slot * b.up_bytes() + ((int64_t)block * b.rank_tiles + rt) * 2048 + 1024 * half + 16 * lane;
  *(uint4*)dst = make_uint4(w[0], w[1], w[2], w[3]);
}

// threadIdx.x, of which the compiler keeps nothing from one turn of a workgroup's loop to the next: the addresses of a
// second turn, which few calls have, would take 30 registers of the first.
__device__ __forceinline__ int thread_here() {
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  return tid;
}

// ---- the tokens of a workgroup ----

struct Tile {
  int slot, rows;   // slot -1: tokens without an adapter; rows 0: no tile of this number
};

struct Call {
  Bank bank;
  const uint16_t* x;
  int64_t x_stride;
  const int32_t* ids;
  const int32_t* first;      // grouped form: the plan of ids (slots groups), or null: every workgroup counts for itself
  const int32_t* row_pair;
  Tile* tile;                // grouped form: what down found, for up: the tiles, then {parts, tiles},
  int32_t* tile_token;       // and the tokens of their 64 columns
  int32_t tokens, parts;
  float* low;                // [parts][T][16 rank_tiles]: partial sums of down x
  const void* base;
  int64_t base_stride;
  uint16_t* y;
  int64_t y_stride;
  int32_t tiles;             // grouped form: the most tiles that there can be; parts: the most parts
};

// Workgroups go round the eight XCDs; this numbers them so that each XCD takes a contiguous range of `count`.
__device__ __forceinline__ int on_xcd(int id, int count) { return (id & 7) * ((count + 7) >> 3) + (id >> 3); }

// What a workgroup of down does: a part of K and a group of rank tiles for a tile. The split of K follows the tiles
// that there are, which only the device knows: the slots that no token names make none (600 tokens of 8 adapters of
// rank 64 by 16384 in a bank of 1024 slots 27 us, split by the tiles that there could be 78), and a slot of fewer ranks
// than the bank's largest has fewer pieces (4096 tokens of rank 16 by 16384 in a bank of 256 ranks 73 us, with idle
// workgroups for the other ranks some 50 more; in a bank of 16 ranks 60).
struct Work {
  Tile tile;
  int index, part, rank_group;   // index -1: nothing
  int tiles, pieces, parts;      // in all; pieces: groups of rank tiles that the tiles have together
};

// Piece `id` of down's work: the groups' tiles, kTileTokens tokens of a group each (a group's last one short), the
// tokens without an adapter last as group `slots`, each for every RT rank tiles that its slot has, then the next part
// of K; each XCD has a contiguous range of it. count(g) gives the tokens of a group, -1 if the plan is none: then there
// is nothing to do. Thread i of the workgroup has the groups from i `per` on. place: the tile's group and the place in
// it of its first token.
constexpr int kThreadGroups = kMaxSlots / 256 + 1;
constexpr int kPieceShift = 13;   // tiles and pieces are counted in one number: up to 5120 and 20480
static_assert(kMaxTokens / kTileTokens + kMaxSlots + 1 < 1 << kPieceShift, "a count of tiles has 13 bits");

template <int RT, typename Count>
__device__ __forceinline__ Work locate(const Call& c, int id, Count count, int (&found)[8], int2& place) {
  const int tid = threadIdx.x, lane = tid & 63, slots = c.bank.slots, per = (slots + 256) / 256, first = tid * per;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int n[kThreadGroups], each[kThreadGroups], mine = 0;   // each: pieces of a tile
#pragma unroll
  for (int i = 0; i < kThreadGroups; ++i)
    if (i < per) {
      n[i] = first + i <= slots ? count(first + i) : 0;
      each[i] = c.bank.rank_tiles > RT && first + i < slots ? max((c.bank.table[first + i].rank + 16 * RT - 1) / (16 * RT), 1) : 1;
      mine += (n[i] + kTileTokens - 1) / kTileTokens * (1 + (each[i] << kPieceShift));
    }
  int upto = mine;   // of the wave's threads up to this one
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(upto, d, 64);
    if (lane >= d) upto += o;
  }
  bool none = false;
#pragma unroll
  for (int i = 0; i < kThreadGroups; ++i) none |= i < per && n[i] < 0;
  none = __any(none);
  if (lane == 63) found[4 + wave] = none ? -1 : upto;
  __syncthreads();
  int total = 0, before = upto - mine;
  none = false;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    none |= found[4 + w] < 0;
    before += w < wave ? found[4 + w] : 0;
    total += found[4 + w];
  }
  total = __builtin_amdgcn_readfirstlane(none ? 0 : total);
  Work w;
  w.tile = Tile{-1, 0};
  w.tiles = total & ((1 << kPieceShift) - 1);
  w.pieces = total >> kPieceShift;
  w.parts = min(c.parts, max(kWantGroups / max(w.pieces, 1), 1));
  w.index = -1;
  w.part = w.rank_group = 0;
  const int all = w.parts * w.pieces, piece = on_xcd(id, all);
  if (id >= (all + 7) / 8 * 8 || piece >= all) return w;
  w.part = piece / w.pieces;
  int skip = piece - w.part * w.pieces - (before >> kPieceShift);   // pieces from this thread's first on
  if (skip >= 0 && skip < mine >> kPieceShift) {
    int index = before & ((1 << kPieceShift) - 1);
#pragma unroll
    for (int i = 0; i < kThreadGroups; ++i)
      if (i < per) {
        const int tiles = (n[i] + kTileTokens - 1) / kTileTokens, tile = each[i] == 1 ? skip : skip / each[i];
        if (skip >= 0 && tile < tiles) {
          found[0] = first + i;
          found[1] = tile * kTileTokens;
          found[2] = min(kTileTokens, n[i] - tile * kTileTokens);
          found[3] = (index + tile) << 4 | (skip - tile * each[i]);
        }
        skip -= tiles * each[i];
        index += tiles;
      }
  }
  __syncthreads();
  place.x = __builtin_amdgcn_readfirstlane(found[0]);
  place.y = __builtin_amdgcn_readfirstlane(found[1]);
  const int at = __builtin_amdgcn_readfirstlane(found[3]);
  w.index = at >> 4;
  w.rank_group = at & 15;
  w.tile = Tile{place.x < slots ? place.x : -1, __builtin_amdgcn_readfirstlane(found[2])};
  return w;
}

// Piece `id` by the plan of ids; `token` is that of this lane's column (those past the last repeat it).
template <int RT>
__device__ __forceinline__ Work plan_work(const Call& c, int id, int (&found)[8], int& token) {
  const int slots = c.bank.slots;
  int2 place;
  const Work work = locate<RT>(c, id, [&](int g) {
    const int lo = c.first[g], hi = g < slots ? c.first[g + 1] : c.tokens;
    return lo >= 0 && (g || !lo) && lo <= hi && hi <= c.tokens ? hi - lo : -1;
  }, found, place);
  if (work.index >= 0) {
    token = c.row_pair[c.first[place.x] + place.y + min((int)(threadIdx.x & 63), work.tile.rows - 1)];
    token = token >= 0 && token < c.tokens ? token : 0;
  }
  return work;
}

// The same from the ids themselves, by a workgroup of four waves for itself: it counts the groups in `lds`, finds its
// tile and picks out the tile's tokens in ascending order. The waves hold the ids, a contiguous section each. About 2
// us in each round of workgroups, where the plan is a launch of 5 and 1 more to read it: 1000 tokens of 8 adapters of
// rank 32, 7168 columns and 1536 rows, 17.9 us, by a plan made for the call 20.4; 16384 columns and 7168 rows, 4096 of
// rank 64 74.1 and 74.4, 4000 of 4 of rank 256, in four rank groups, 151 and 152.
constexpr int kOwnIds = 16, kOwnTokens = 4 * 64 * kOwnIds;
constexpr int kCopies = 8;   // of each count, by lane: neighbours of one group take few turns at one of them
constexpr int kOwnLds = (kMaxSlots + 1) * kCopies + 4 + kTileTokens;   // numbers

template <int RT>
__device__ __forceinline__ Work own_work(const Call& c, int id, int (&found)[8], int* lds, int& token) {
  const int tid = threadIdx.x, lane = tid & 63, slots = c.bank.slots;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int* count = lds;
  int* part = lds + (kMaxSlots + 1) * kCopies;
  int* list = part + 4;
  const int section = (c.tokens + 255) / 256 * 64, p0 = wave * section + lane;
  int key[kOwnIds];   // -1: past the last token; tokens without an adapter are group `slots`
#pragma unroll
  for (int i = 0; i < kOwnIds; ++i)
    if (64 * i < section) key[i] = c.ids[min(p0 + 64 * i, c.tokens - 1)];
  for (int n = tid; n < (slots + 1) * (kCopies / 4); n += 256) ((uint4*)count)[n] = make_uint4(0, 0, 0, 0);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kOwnIds; ++i)
    if (64 * i < section) {
      key[i] = p0 + 64 * i >= c.tokens ? -1 : key[i] >= 0 && key[i] < slots ? key[i] : slots;
      if (key[i] >= 0) atomicAdd(&count[key[i] * kCopies + lane % kCopies], 1);
    }
  __syncthreads();
  int2 place;
  const Work work = locate<RT>(c, id, [&](int g) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) n += count[g * kCopies + i];
    return n;
  }, found, place);
  if (work.index < 0) return work;
  int own = 0;
#pragma unroll
  for (int i = 0; i < kOwnIds; ++i)
    if (64 * i < section) own += __popcll(__ballot(key[i] == place.x));
  if (lane == 0) part[wave] = own;
  __syncthreads();
  int at = -place.y;
  for (int w = 0; w < wave; ++w) at += part[w];
#pragma unroll
  for (int i = 0; i < kOwnIds; ++i)
    if (64 * i < section) {
      const uint64_t mask = __ballot(key[i] == place.x);
      const int column = at + __popcll(mask & ((1ull << lane) - 1));
      if (key[i] == place.x && column >= 0 && column < kTileTokens) list[column] = p0 + 64 * i;
      at += __popcll(mask);
    }
  __syncthreads();
  token = list[min(lane, work.tile.rows - 1)];
  __syncthreads();   // before the stages
  return work;
}

// Few tokens: the workgroups of token t take the tokens of t's adapter, up to 16 a workgroup. The first of each 16 does
// it; rows = 0 for the others. (Tokens are the grid's slow dimension: as its fast one, a count of them that eight
// divides puts all the workgroups of a token on one XCD, and 64 tokens of 16 adapters take 27 us where 65 take 17.)
struct Few {
  int slot, rows;
  int token;   // of this lane's column, lane % 16; columns past the last repeat it
};

__device__ __forceinline__ Few few_tokens(const Call& c, int t) {
  const int lane = threadIdx.x & 63;
  int id[2], place[2];
  uint64_t mask[2];   // the tokens of t's adapter, 64 tokens each
#pragma unroll
  for (int i = 0; i < 2; ++i) id[i] = c.ids[min(64 * i + lane, c.tokens - 1)];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    id[i] = 64 * i + lane >= c.tokens ? -2 : id[i] >= 0 && id[i] < c.bank.slots ? id[i] : -1;
  const int slot = __builtin_amdgcn_readlane(t < 64 ? id[0] : id[1], t & 63);
#pragma unroll
  for (int i = 0; i < 2; ++i) mask[i] = __ballot(id[i] == slot);
  const int first = __popcll(mask[0]), total = first + __popcll(mask[1]);
  const uint64_t below = (1ull << (t & 63)) - 1, under = (1ull << lane) - 1;
  const int before = t < 64 ? __popcll(mask[0] & below) : first + __popcll(mask[1] & below);
  const int rows = before & 15 ? 0 : min(16, total - before);
  place[0] = __popcll(mask[0] & under) - before;
  place[1] = first + __popcll(mask[1] & under) - before;
#pragma unroll
  for (int i = 0; i < 2; ++i) {   // column n's token goes to lane n; lane 63 is no column's
    const bool mine = id[i] == slot && place[i] >= 0 && place[i] < 16;
    id[i] = __builtin_amdgcn_ds_permute(4 * (mine ? place[i] : 63), 64 * i + lane);
  }
  const int column = min(lane & 15, max(rows, 1) - 1);
  const int low = __shfl(id[0], column, 64), high = __shfl(id[1], column, 64);
  return Few{slot, rows, before + column < first ? low : high};
}

// Four ranks of h, from r0 on; past the slot's rank zero.
__device__ __forceinline__ v4f h_of(const AdapterSlot& slot, int r0, v4f s) {
  v4f h;
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = r0 + i < slot.rank ? slot.scale * s[i] : 0.f;
  return h;
}

// Four ranks of h as up's operand B: the first two terms of each, and the third.
struct Terms {
  uint4 two;
  uint2 third;
};

__device__ __forceinline__ Terms split(v4f h) {
  uint32_t t[3][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t[0][i] = mx::f2u(h[i]);
    const bool finite = (t[0][i] & 0x7F800000u) != 0x7F800000u;   // infinities and NaN are their first term
    const float rest = finite ? h[i] - mx::u2f(t[0][i] & 0xFFFF0000u) : 0.f;
    t[1][i] = mx::f2u(rest);
    t[2][i] = mx::f2u(rest - mx::u2f(t[1][i] & 0xFFFF0000u));
  }
  uint32_t w[3][2];   // the upper halves of two
#pragma unroll
  for (int n = 0; n < 3; ++n)
#pragma unroll
    for (int k = 0; k < 2; ++k) w[n][k] = __builtin_amdgcn_perm(t[n][2 * k + 1], t[n][2 * k], 0x07060302u);
  return Terms{make_uint4(w[0][0], w[0][1], w[1][0], w[1][1]), make_uint2(w[2][0], w[2][1])};
}

__device__ __forceinline__ v4f load_h(const float* p) { return __builtin_bit_cast(v4f, ldg128((const uint8_t*)p)); }

// The parts first, first + step, ... of four ranks added in that order, eight of them in flight.
__device__ __forceinline__ v4f sum_parts(const float* p, int64_t stride, int first, int step, int parts) {
  v4f sum = v4f{0.f, 0.f, 0.f, 0.f};
  for (int n = first; n < parts; n += 8 * step) {
    uint4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = ldg128((const uint8_t*)(p + min(n + i * step, parts - 1) * stride));
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i * step < parts) sum = sum + __builtin_bit_cast(v4f, v[i]);
  }
  return sum;
}

// ---- down: partial sums of h ----

// Few tokens, grid (parts, T), 4 waves: a part of K for up to 16 tokens of an adapter, RT rank tiles at a time (those
// past the last repeat it). Bound by down's bytes: 24 tokens of 16 adapters of rank 64 by 16384 (33 MB) 8.0 us. The
// waves take the K units (of 64: two chunks) in turn, the next one's loads in flight while one is multiplied, and their
// sums are added in wave order.
template <int RT>
__device__ __forceinline__ void few_down(const Call& c, const Few& f, int r0, int tiles, int first_tiles,
                                         v4f (*red)[RT][64]) {
  const Bank& b = c.bank;
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int units = b.chunks / 2, whole = b.k / 64;
  const int u1 = (int)((int64_t)units * (blockIdx.x + 1) / c.parts);
  int u = (int)((int64_t)units * blockIdx.x / c.parts) + wave;
  const uint8_t* x = (const uint8_t*)(c.x + f.token * c.x_stride) + 16 * q;
  const int64_t tile_bytes = (int64_t)b.chunks * 1024;
  const uint8_t* w = b.down + f.slot * b.down_bytes() + r0 * tile_bytes + 16 * lane;
  struct Unit {
    uint4 x[2], w[2][RT];
  } unit[2];
  v4f acc[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) acc[r] = v4f{0.f, 0.f, 0.f, 0.f};
  auto load_w = [&](Unit& n, int at, int last) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int r = 0; r < RT; ++r) n.w[s][r] = ldg128(w + min(r, last) * tile_bytes + 2048 * (int64_t)at + 1024 * s);
  };
  auto load = [&](Unit& n, int at, int last) {
    load_w(n, at, last);
#pragma unroll
    for (int s = 0; s < 2; ++s) n.x[s] = ldg128(x + 128 * at + 64 * s);
  };
  auto multiply = [&](const Unit& n) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int r = 0; r < RT; ++r)
        acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(n.w[s][r]), as_bf(n.x[s]), acc[r], 0, 0, 0);
  };
  const int end = min(u1, whole);
  if (u < end) {
    load(unit[0], u, first_tiles - 1);
    const int last = max(tiles - r0 - 1, 0);
    while (true) {
      load(unit[1], min(u + 4, end - 1), last);
      multiply(unit[0]);
      u += 4;
      if (u >= end) break;
      load(unit[0], min(u + 4, end - 1), last);
      multiply(unit[1]);
      u += 4;
      if (u >= end) break;
    }
  }
  if (tiles <= r0) return;
  if (u < u1) {   // the last unit of a K that is no multiple of 64: zeros past the end of x
    load_w(unit[0], u, tiles - r0 - 1);
#pragma unroll
    for (int s = 0; s < 2; ++s)
      unit[0].x[s] = 64 * u + 32 * s + 8 * q < b.k ? ldg128(x + 128 * u + 64 * s) : make_uint4(0, 0, 0, 0);
    multiply(unit[0]);
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) red[wave][r][lane] = acc[r];
  __syncthreads();
  for (int r = wave; r < RT; r += 4)
    if (r0 + r < tiles && (lane & 15) < f.rows) {
      const v4f s = ((red[0][r][lane] + red[1][r][lane]) + red[2][r][lane]) + red[3][r][lane];
      *(v4f*)(c.low + ((int64_t)blockIdx.x * c.tokens + f.token) * (16 * b.rank_tiles) + 16 * (r0 + r) + 4 * q) = s;
    }
  __syncthreads();
}

// The first unit's weights are asked for by the bank's largest rank, before the slot's own has arrived.
template <int RT>
__global__ __launch_bounds__(256) void adapter_few_down_kernel(Call c) {
  __shared__ v4f red[4][RT][64];
  const Few f = few_tokens(c, blockIdx.y);
  if (f.rows == 0 || f.slot < 0) return;
  const int tiles = (c.bank.table[f.slot].rank + 15) >> 4;
  few_down<RT>(c, f, 0, tiles, min(RT, c.bank.rank_tiles), red);
  for (int r0 = RT; r0 < tiles; r0 += RT) few_down<RT>(c, f, r0, tiles, min(RT, tiles - r0), red);
}

// Grouped form: a part of K for a tile of 64 tokens and RT rank tiles, 4 waves. x comes through LDS in stages of 256 K,
// so that rows are read 512 bytes at a time (in operand order a load takes 64 bytes of each of 16 rows: with rows a
// power of two apart those meet in the same memory channels); each wave multiplies its K unit of 64 of every stage, its
// weights straight from the L2 of its XCD, which holds one part's. Two stages: one in flight while one is multiplied.
// 4096 tokens of 8 adapters of rank 64 by 16384: 36 to 39 us, by a plan 35, of which x (134 MB) alone, read so, takes 25;
// without LDS 46; tiles of 128 tokens 34, but 62 against 55 with two rank groups. The rows of a pair lie 512 bytes
// apart and the pairs 1040, and a second row's 16-byte pieces are swapped in halves of 128 bytes, so that the 16 rows
// of an operand read lie in different banks.
constexpr int kStageK = 256, kPairBytes = 1040, kStageBytes = kTileTokens / 2 * kPairBytes;
static_assert(4 * kOwnLds <= 2 * kStageBytes, "the counts lie where the stages come after them");

template <int RT, bool kStream>
__device__ __forceinline__ void down_piece(const Call& c, const Work& work, int tokens, uint4* stage_lds) {
  const Bank& b = c.bank;
  const Tile t = work.tile;
  const int part = work.part, r0 = RT * work.rank_group;
  const AdapterSlot slot = b.table[t.slot];
  const int tiles = (slot.rank + 15) >> 4;
  if (r0 >= tiles) return;
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int stages = (b.k + kStageK - 1) / kStageK, units = b.chunks / 2;
  const int s0 = (int)((int64_t)stages * part / work.parts), s1 = (int)((int64_t)stages * (part + 1) / work.parts);
  const uint32_t lds = mxd::lds_addr(stage_lds);
  const int piece = (lane & 31) ^ (lane >> 5 << 3);   // of its row that this lane copies
  const uint8_t* src[kColumns * 2];
#pragma unroll
  for (int j = 0; j < kColumns * 2; ++j)
    src[j] = (const uint8_t*)(c.x + __shfl(tokens, 2 * (wave + 4 * j) + (lane >> 5), 64) * c.x_stride);
  auto copy = [&](int stage, int buffer) {
    const bool in = kStageK * stage + 8 * piece < b.k;
    const int64_t at = in ? (int64_t)(2 * kStageK) * stage + 16 * piece : 0;
#pragma unroll
    for (int j = 0; j < kColumns * 2; ++j)
      if (2 * (wave + 4 * j) < t.rows) {
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds + buffer * kStageBytes + (wave + 4 * j) * kPairBytes);
        if constexpr (kStream) mxd::global_to_lds16_nt(src[j] + at, to);
        else mxd::global_to_lds16(src[j] + at, to);
      }
  };
  const int64_t tile_bytes = (int64_t)b.chunks * 1024;
  const uint8_t* w = b.down + t.slot * b.down_bytes() + r0 * tile_bytes + 16 * lane;
  const int last = tiles - r0 - 1;
  auto load_w = [&](uint4 (*n)[RT], int stage) {
    const int u = min(4 * stage + wave, units - 1);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int r = 0; r < RT; ++r) n[s][r] = ldg128(w + min(r, last) * tile_bytes + 2048 * (int64_t)u + 1024 * s);
  };
  v4f acc[kColumns][RT];
#pragma unroll
  for (int i = 0; i < kColumns; ++i)
#pragma unroll
    for (int r = 0; r < RT; ++r) acc[i][r] = v4f{0.f, 0.f, 0.f, 0.f};
  // this lane's row of column tile 0: pair (l % 16) / 2, half l % 2
  const uint8_t* rows = (const uint8_t*)stage_lds + ((lane & 15) >> 1) * kPairBytes + (lane & 1) * 512;
  auto multiply = [&](const uint4 (*n)[RT], int stage, int buffer) {
    const int u = 4 * stage + wave;
    if (64 * u >= b.k) return;
    const bool ragged = 64 * u + 64 > b.k;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int at = 16 * ((8 * wave + 4 * s + q) ^ ((lane & 1) << 3));
      uint4 x[kColumns];
#pragma unroll
      for (int i = 0; i < kColumns; ++i) x[i] = *(const uint4*)(rows + buffer * kStageBytes + i * 8 * kPairBytes + at);
      if (ragged && 64 * u + 32 * s + 8 * q >= b.k) {
#pragma unroll
        for (int i = 0; i < kColumns; ++i) x[i] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < kColumns; ++i)
          acc[i][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(n[s][r]), as_bf(x[i]), acc[i][r], 0, 0, 0);
    }
  };
  uint4 wv[2][2][RT];
  // the weights before the copies: the wait for the weights then leaves the copies behind them in flight
  load_w(wv[0], s0);
  copy(s0, 0);
  for (int stage = s0; stage < s1; stage += 2) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if (stage + n >= s1) break;
      __builtin_amdgcn_s_waitcnt(mxd::vm_wait_imm(0));
      mxd::copy_barrier();
      if (stage + n + 1 < s1) {
        load_w(wv[n ^ 1], stage + n + 1);
        copy(stage + n + 1, n ^ 1);
      }
      multiply(wv[n], stage + n, n);
    }
  }
  mxd::copy_barrier();
  v4f* red = (v4f*)stage_lds;
#pragma unroll
  for (int i = 0; i < kColumns; ++i)
#pragma unroll
    for (int r = 0; r < RT; ++r) red[((wave * kColumns + i) * RT + r) * 64 + lane] = acc[i][r];
  __syncthreads();
  const int col = 16 * wave + (lane & 15), token = __shfl(tokens, col, 64);   // wave i finishes column tile i
  if (col >= t.rows) return;
  float* low = c.low + ((int64_t)part * c.tokens + token) * (16 * b.rank_tiles) + 16 * r0 + 4 * q;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    if (r0 + r >= tiles) break;
    v4f s = red[(wave * RT + r) * 64 + lane];
#pragma unroll
    for (int v = 1; v < 4; ++v) s = s + red[((v * kColumns + wave) * RT + r) * 64 + lane];
    *(v4f*)(low + 16 * r) = c.parts == 1 ? h_of(slot, 16 * (r0 + r) + 4 * q, s) : s;
  }
}

template <int RT, bool kStream>
__global__ __launch_bounds__(256, 2) void adapter_down_kernel(Call c) {
  extern __shared__ uint4 stage_lds[];   // two stages; then the waves' sums [4][kColumns][RT][64]
  __shared__ int found[8];   // of the tile: group, first token's place in it, tokens, number and rank group; then sums
  int tokens = 0;
  const Work work = c.first ? plan_work<RT>(c, blockIdx.x, found, tokens)
                            : own_work<RT>(c, blockIdx.x, found, (int*)stage_lds, tokens);
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) c.tile[c.tiles] = Tile{work.parts, work.tiles};
    for (int i = work.tiles + threadIdx.x; i < c.tiles; i += 256) c.tile[i] = Tile{-1, 0};
  }
  if (work.index < 0) return;
  if (work.part == 0 && work.rank_group == 0) {
    if (threadIdx.x < 64) c.tile_token[work.index * kTileTokens + threadIdx.x] = tokens;
    if (threadIdx.x == 0) c.tile[work.index] = work.tile;
  }
  if (work.tile.rows > 0 && work.tile.slot >= 0) down_piece<RT, kStream>(c, work, tokens, stage_lds);
}

// Grouped form of more than 16 ranks: the parts of four ranks of a token added, as h in the first part's place;
// more than eight of them, which a thread has in flight at once, by four lanes whose sums are added as a tree. A launch
// of its own, 3 to 5 us: in up every workgroup of a tile would add them anew, which 4096 tokens of rank 64 pay with 18
// us and 3056 beside 24576 rows with 41, and even rank 32 with 1. Of up to 16 ranks up does it: 1010 tokens of rank 8,
// 7168 columns and 576 rows, 12.4 us in all, with this launch 1.9 more.
template <int kShares>
__global__ __launch_bounds__(256) void adapter_sum_kernel(Call c) {
  const Bank& b = c.bank;
  const int per = 4 * b.rank_tiles, share = (threadIdx.x & 63) / (64 / kShares);   // entries of a token
  const int e = (blockIdx.x * 256 + (threadIdx.x & ~63)) / kShares + threadIdx.x % (64 / kShares);
  if (e >= c.tokens * per) return;
  const int id = c.ids[e / per], r0 = 4 * (e % per);
  if (id < 0 || id >= b.slots) return;
  const AdapterSlot slot = b.table[id];
  if (r0 >= slot.rank) return;   // what lies past a slot's rank no one has written, and up takes as zero
  float* p = c.low + 4 * (int64_t)e;
  v4f s = sum_parts(p, (int64_t)c.tokens * 4 * per, share, kShares, min(c.tile[c.tiles].slot, c.parts));
#pragma unroll
  for (int d = 64 / kShares; d < 64; d <<= 1)   // the lanes of an entry are here or gone together
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = s[i] + __shfl_xor(s[i], d, 64);
  if (share == 0) *(v4f*)p = h_of(slot, r0, s);
}

// ---- up: y = base + up h ----

template <bool kF32>
struct Eight;   // 8 consecutive values of base

template <>
struct Eight<true> {
  float4 v[2];
  __device__ __forceinline__ void load(const Call& c, int64_t at) {
    const float4* s = (const float4*)((const float*)c.base + at);
    v[0] = s[0], v[1] = s[1];
  }
  __device__ __forceinline__ v4f four(int j) const { return v4f{v[j].x, v[j].y, v[j].z, v[j].w}; }
};

// Four of the eight BF16 values, the second four with `second`.
__device__ __forceinline__ v4f four_of(uint4 v, int second) {
  const uint32_t a = second ? v.z : v.x, b = second ? v.w : v.y;
  return v4f{mx::u2f(a << 16), mx::u2f(a & 0xFFFF0000u), mx::u2f(b << 16), mx::u2f(b & 0xFFFF0000u)};
}

template <>
struct Eight<false> {
  uint4 v;
  __device__ __forceinline__ void load(const Call& c, int64_t at) { v = *(const uint4*)((const uint16_t*)c.base + at); }
  __device__ __forceinline__ v4f four(int j) const { return four_of(v, j); }
};

__device__ __forceinline__ uint4 eight_bf16(v4f a, v4f b) {
  return make_uint4(mxd::bf16_pair(a[0], a[1]), mxd::bf16_pair(a[2], a[3]), mxd::bf16_pair(b[0], b[1]),
                    mxd::bf16_pair(b[2], b[3]));
}

// Two 16-byte pieces a lane between operand order and memory order. In operand order lane (column, q) holds pieces q of
// the first and of the second 64 bytes of its column's token, so an access takes 64 bytes of 16 rows; in memory order
// the lanes of columns 0-7 hold first pieces and those of 8-15 second ones, of column % 8 and then of 8 + column % 8:
// 128 bytes, a whole line, of 8 rows. The lanes eight apart swap one piece; the same swap leads back.
// (A plain copy of 4096 rows of 7168 in these orders: 26 and 18 us.)
__device__ __forceinline__ void swap8(uint4& first, uint4& second, bool low) {
  const uint32_t a[4] = {first.x, first.y, first.z, first.w}, b[4] = {second.x, second.y, second.z, second.w};
  uint32_t u[4], v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {   // in numbers: a choice between structures would go through memory
    const uint32_t give = low ? b[i] : a[i];
    const uint32_t got = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)give, 0x128, 0xF, 0xF, false);   // row_ror:8
    u[i] = low ? a[i] : got;
    v[i] = low ? got : b[i];
  }
  first = make_uint4(u[0], u[1], u[2], u[3]);
  second = make_uint4(v[0], v[1], v[2], v[3]);
}

// 16 rows (of two tiles of a half each) against operand B `h`: K slots 0..3 are the ranks of up's tile a, 4..7 those of b
// (their two halves). acc[0..3] are the tiles of the block.
__device__ __forceinline__ void up_mfma(uint4 a0, uint4 a1, uint4 b0, uint4 b1, uint4 h, v4f (&acc)[4]) {
  const v8bf v = as_bf(h);
  acc[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(make_uint4(a0.x, a0.y, b0.x, b0.y)), v, acc[0], 0, 0, 0);
  acc[1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(make_uint4(a0.z, a0.w, b0.z, b0.w)), v, acc[1], 0, 0, 0);
  acc[2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(make_uint4(a1.x, a1.y, b1.x, b1.y)), v, acc[2], 0, 0, 0);
  acc[3] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(make_uint4(a1.z, a1.w, b1.z, b1.w)), v, acc[3], 0, 0, 0);
}

// Up of RT rank tiles at most, `count` of them the slot's (up's others may hold anything). This lane's terms of tile r of
// a column tile lie at two[64 r] and, the third ones of two tiles together, at third[64 (r / 2)]. 4096 tokens of 8 adapters
// of rank 128 and 256 (BF16 base), 1536 columns and 24576 rows: 136 and 210 us, with an MFMA for the third terms of each
// tile 147 and 220; of rank 64 no different.
template <int RT>
__device__ __forceinline__ void up_tiles(const uint4 (&w)[RT][2], const uint4* two, const uint4* third, int count,
                                         v4f (&acc)[4]) {
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    if (r >= count) continue;
    up_mfma(w[r][0], w[r][1], w[r][0], w[r][1], two[64 * r], acc);
    const uint4 rest = third[64 * (r / 2)];
    if (r % 2) up_mfma(w[r - 1][0], w[r - 1][1], w[r][0], w[r][1], rest, acc);
    else if (r + 1 >= count) up_mfma(w[r][0], w[r][1], w[r][0], w[r][1], make_uint4(rest.x, rest.y, 0, 0), acc);
  }
}

// Few tokens, grid (output blocks / 4, T), 4 waves, a block of 64 outputs each for up to 16 tokens of an adapter (24
// tokens of 16 adapters of rank 64, 7168 outputs, 15 MB of up: 5.8 to 7.1 us). What does not depend on h is asked for before h
// is put together: thread (entry e, share s) adds the parts s, s + shares, ... of four ranks of a token, and the shares
// are added in order. (Two waves a SIMD at least, as adapter_up_kernel and for the same reason.)
template <bool kF32>
__global__ __launch_bounds__(256, 2) void adapter_few_up_kernel(Call c) {
  constexpr int RT = 4;   // rank tiles in registers at once
  __shared__ v4f sums[256];
  __shared__ uint4 h_lds[kMaxRank / 16 * 64];
  __shared__ uint4 third_lds[kMaxRank / 32 * 64];
  const Few f = few_tokens(c, blockIdx.y);
  if (f.rows == 0) return;
  const Bank& b = c.bank;
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int block = 4 * blockIdx.x + wave, n = 64 * block + 8 * q;   // past the last block: no output is a lane's
  const uint8_t* up = b.up_at(f.slot, block) + 16 * lane;
  uint4 w[RT][2];
  auto load_up = [&](int r0, int count) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int at = r0 + min(r, count - 1);
      w[r][0] = ldg128(up + 2048 * at), w[r][1] = ldg128(up + 2048 * at + 1024);
    }
  };
  Eight<kF32> base[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) base[k].load(c, f.token * c.base_stride + (n + 32 * k < b.n ? n + 32 * k : 0));
  load_up(0, min(RT, b.rank_tiles));   // of the largest rank: the slot's own is still on its way
  const AdapterSlot slot = f.slot >= 0 ? b.table[f.slot] : AdapterSlot{0, 0.f};
  const int tiles = (slot.rank + 15) >> 4;
  // entry e: ranks 4 (e / rows) .. of column e % rows
  const int entries = 4 * tiles * f.rows, shares = entries ? max(256 / entries, 1) : 0;
  const int64_t part_stride = (int64_t)c.tokens * 16 * b.rank_tiles;
  for (int e0 = 0; e0 < entries; e0 += 256) {
    const int e = e0 + (shares > 1 ? tid % entries : tid), share = shares > 1 ? tid / entries : 0;
    const int column = e % f.rows, token = __shfl(f.token, column, 64);
    const bool in = e < entries && share < shares;
    v4f sum = v4f{0.f, 0.f, 0.f, 0.f};
    if (in)
      sum = sum_parts(c.low + (int64_t)token * 16 * b.rank_tiles + 4 * (e / f.rows), part_stride, share, shares, c.parts);
    if (shares > 1) {
      sums[tid] = sum;
      __syncthreads();
      if (tid < entries)
        for (int m = 1; m < min(shares, c.parts); ++m) sum = sum + sums[m * entries + tid];
    }
    if (in && share == 0) {
      const Terms h = split(h_of(slot, 4 * (e / f.rows), sum));
      const int four = e / f.rows, at = four % 4 * 16 + column;
      h_lds[four / 4 * 64 + at] = h.two;
      ((uint2*)third_lds)[2 * (four / 8 * 64 + at) + four / 4 % 2] = h.third;
    }
  }
  __syncthreads();
  v4f acc[4] = {base[0].four(0), base[0].four(1), base[1].four(0), base[1].four(1)};
  for (int r0 = 0; r0 < tiles; r0 += RT) {
    if (r0) load_up(r0, min(RT, tiles - r0));
    up_tiles<RT>(w, h_lds + 64 * r0 + lane, third_lds + 32 * r0 + lane, tiles - r0, acc);
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if ((lane & 15) < f.rows && n + 32 * k < b.n)
      *(uint4*)(c.y + f.token * c.y_stride + n + 32 * k) = eight_bf16(acc[2 * k], acc[2 * k + 1]);
}

// Few tokens in one launch, for a down that every workgroup can read for itself: grid (output blocks / 16, T), 16
// waves. A chain of two loads' latencies and a launch: one token of 24576 outputs 4.5 to 5.5 us. The waves take the K units of 64 in turn, two
// of them in flight, h is put together through LDS, and each wave finishes a block of 64 outputs whose up and base were
// asked for at the start.
template <int RT, bool kF32>
__global__ __launch_bounds__(1024) void adapter_few_kernel(Call c) {
  __shared__ v4f sums[16][RT][64];
  __shared__ uint4 h_lds[RT][64];
  __shared__ uint4 third_lds[64];
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Bank& b = c.bank;
  const Few f = few_tokens(c, blockIdx.y);
  if (f.rows == 0) return;
  const int block = 16 * blockIdx.x + wave, n = 64 * block + 8 * q;
  const int units = b.chunks / 2, last = b.rank_tiles - 1;
  const int64_t tile_bytes = (int64_t)b.chunks * 1024;
  const uint8_t* x = (const uint8_t*)(c.x + f.token * c.x_stride) + 16 * q;
  const uint8_t* down = b.down + max(f.slot, 0) * b.down_bytes() + 16 * lane;
  const uint8_t* up = b.up_at(f.slot, block) + 16 * lane;
  struct Unit {
    uint4 x[2], w[2][RT];
  } unit[2];
  auto load = [&](Unit& m, int at) {   // a unit past the last repeats it; what lies past the end of x is zero
    at = min(at, units - 1);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const bool in = 64 * at + 32 * s + 8 * q < b.k;
      const uint4 v = ldg128(in ? x + 128 * at + 64 * s : x - 16 * q);
      m.x[s] = in ? v : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < RT; ++r) m.w[s][r] = ldg128(down + min(r, last) * tile_bytes + 2048 * (int64_t)at + 1024 * s);
    }
  };
  Eight<kF32> base[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) base[k].load(c, f.token * c.base_stride + (n + 32 * k < b.n ? n + 32 * k : 0));
  uint4 w[RT][2];
  v4f acc[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) acc[r] = v4f{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const Unit& m) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int r = 0; r < RT; ++r)
        acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(m.w[s][r]), as_bf(m.x[s]), acc[r], 0, 0, 0);
  };
  if (f.slot >= 0) {
    load(unit[0], wave);
    load(unit[1], wave + 16);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      w[r][0] = ldg128(up + 2048 * min(r, last));
      w[r][1] = ldg128(up + 2048 * min(r, last) + 1024);
    }
    for (int u = wave; u < units; u += 32) {
      multiply(unit[0]);
      if (u + 32 < units) load(unit[0], u + 32);
      if (u + 16 < units) {
        multiply(unit[1]);
        if (u + 48 < units) load(unit[1], u + 48);
      }
    }
  }
  const AdapterSlot slot = f.slot >= 0 ? b.table[f.slot] : AdapterSlot{0, 0.f};
  const int tiles = (slot.rank + 15) >> 4;
#pragma unroll
  for (int r = 0; r < RT; ++r) sums[wave][r][lane] = acc[r];
  __syncthreads();
  if (wave < RT) {   // wave r puts rank tile r together
    v4f sum = sums[0][wave][lane];
#pragma unroll
    for (int v = 1; v < 16; ++v) sum = sum + sums[v][wave][lane];
    const Terms h = split(h_of(slot, 16 * wave + 4 * q, sum));
    h_lds[wave][lane] = h.two;
    ((uint2*)third_lds)[2 * lane + wave] = h.third;
  }
  __syncthreads();
  v4f out[4] = {base[0].four(0), base[0].four(1), base[1].four(0), base[1].four(1)};
  up_tiles<RT>(w, h_lds[0] + lane, third_lds + lane, tiles, out);
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if ((lane & 15) < f.rows && n + 32 * k < b.n)
      *(uint4*)(c.y + f.token * c.y_stride + n + 32 * k) = eight_bf16(out[2 * k], out[2 * k + 1]);
}

// Base of the tile's tokens at a block, in memory order (see swap8): this lane's pieces are of two tokens of each
// column tile, eight columns apart. Lanes without an output repeat another's address.
template <bool kF32>
__device__ __forceinline__ void load_base(const Call& c, int tokens, int n, int lane, uint4 (&base)[kColumns][kF32 ? 4 : 2],
                                          int64_t (&token)[kColumns][2]) {
  const bool low = (lane & 15) < 8;
#pragma unroll
  for (int i = 0; i < kColumns; ++i)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      token[i][k] = __shfl(tokens, 16 * i + 8 * k + (lane & 7), 64);
      if constexpr (kF32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = n + 32 * h < c.bank.n ? n + 32 * h + (low ? 0 : 4) : 0;
          base[i][2 * h + k] = ldg128((const uint8_t*)((const float*)c.base + token[i][k] * c.base_stride + at));
        }
      } else {
        const int at = n + (low ? 0 : 32) < c.bank.n ? n + (low ? 0 : 32) : 0;
        base[i][k] = ldg128((const uint8_t*)((const uint16_t*)c.base + token[i][k] * c.base_stride + at));
      }
    }
}

// A column tile's base as what its sums start from.
template <bool kF32>
__device__ __forceinline__ void from_base(uint4 (&base)[kF32 ? 4 : 2], bool low, v4f (&acc)[4]) {
  if constexpr (kF32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      swap8(base[2 * h], base[2 * h + 1], low);
      acc[2 * h] = __builtin_bit_cast(v4f, base[2 * h]);
      acc[2 * h + 1] = __builtin_bit_cast(v4f, base[2 * h + 1]);
    }
  } else {
    swap8(base[0], base[1], low);
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = four_of(base[k >> 1], k & 1);
  }
}

// Column tile i of y, of `rows` tokens in all; `at` is this lane's output in memory order.
__device__ __forceinline__ void store_y(const Call& c, int rows, int i, int at, int lane, bool low,
                                        const int64_t (&token)[2], const v4f (&acc)[4]) {
  uint4 out[2] = {eight_bf16(acc[0], acc[1]), eight_bf16(acc[2], acc[3])};
  swap8(out[0], out[1], low);
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (16 * i + 8 * k + (lane & 7) < rows && at < c.bank.n) *(uint4*)(c.y + token[k] * c.y_stride + at) = out[k];
}

// A column tile's terms into LDS for up_tiles; `ranks` is how many ranks the slot has from this lane's first on: the sums
// past them are not its own.
template <int RT>
__device__ __forceinline__ void put_h(const v4f (&h)[RT], int ranks, uint4* two, uint4* third) {
  Terms t[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    t[r] = split(ranks > 16 * r ? h[r] : v4f{0.f, 0.f, 0.f, 0.f});
    two[64 * r] = t[r].two;
    if (r % 2) third[64 * (r / 2)] = make_uint4(t[r - 1].third.x, t[r - 1].third.y, t[r].third.x, t[r].third.y);
    else if (r + 1 == RT) third[64 * (r / 2)] = make_uint4(t[r].third.x, t[r].third.y, 0, 0);
  }
}

// Grouped form: a tile of 64 tokens and four blocks of 64 outputs, one a wave, its weights of all ranks in registers
// for the tile's columns, 16 tokens at a time. What does not depend on h is asked for before h goes to LDS. Bound by
// base and y: 4096 tokens of 7168 outputs (117 MB) 30 to 32 us; with accesses of 64 bytes 7 more.
template <int RT, bool kF32>
__device__ __forceinline__ void up_blocks(const Call& c, int index, const Tile& t, int group, int parts, int tid, uint4* h_lds,
                                          uint4* third_lds) {
  constexpr int kPairs = (RT + 1) / 2;
  const Bank& b = c.bank;
  const int tokens = c.tile_token[index * kTileTokens + (tid & 63)];
  const AdapterSlot slot = t.slot >= 0 ? b.table[t.slot] : AdapterSlot{0, 0.f};
  const int tiles = (slot.rank + 15) >> 4;
  const int lane = tid & 63, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int block = 4 * group + wave, n = 64 * block + 8 * q;   // past the last block: no output is a lane's
  // every load below goes out before the first of them is waited for; lanes without an output repeat another's address
  const int64_t rank_stride = 16 * b.rank_tiles;
  const float* low_h = c.low + __shfl(tokens, 16 * wave + (lane & 15), 64) * rank_stride + 4 * q;
  v4f h[RT];   // of the wave's column tile
  if (RT > 1 || c.parts == 1) {
#pragma unroll
    for (int r = 0; r < RT; ++r) h[r] = load_h(low_h + 16 * max(min(r, tiles - 1), 0));
  }
  uint4 w[RT][2];
  {
    const uint8_t* p = b.up_at(t.slot, block) + 16 * lane;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int at = max(min(r, tiles - 1), 0);
      w[r][0] = ldg128(p + 2048 * at), w[r][1] = ldg128(p + 2048 * at + 1024);
    }
  }
  const bool low = (lane & 15) < 8;
  uint4 base[kColumns][kF32 ? 4 : 2];
  int64_t token[kColumns][2];
  load_base<kF32>(c, tokens, n, lane, base, token);
  if constexpr (RT == 1)
    if (c.parts > 1 && tiles) h[0] = h_of(slot, 4 * q, sum_parts(low_h, c.tokens * rank_stride, 0, 1, parts));
  put_h(h, slot.rank - 4 * q, h_lds + wave * RT * 64 + lane, third_lds + wave * kPairs * 64 + lane);
  mxd::lds_barrier();
  const int at_y = n + (low ? 0 : 32);
#pragma unroll
  for (int i = 0; i < kColumns; ++i) {
    if (16 * i >= t.rows) break;
    v4f acc[4];
    from_base<kF32>(base[i], low, acc);
    const uint4 *two = h_lds + i * RT * 64 + lane, *third = third_lds + i * kPairs * 64 + lane;
    if (tiles == RT) up_tiles<RT>(w, two, third, RT, acc);
    else up_tiles<RT>(w, two, third, tiles, acc);
    store_y(c, t.rows, i, at_y, lane, low, token[i], acc);
  }
}

// The same in a bank of more than 128 ranks: the blocks' sums of all 64 tokens stay in registers, and the ranks go
// through 64 at a time, only the slot's own. 4096 tokens of 8 adapters of rank 256, 64 and 16 in a bank of 256, 1536
// columns and 24576 outputs, BF16 base: 202, 114 and 105 us in all; all 16 rank tiles at once 340, 248 and 211. (In a bank
// of 128 ranks eight at once and four in turn: rank 128 127 and 144 us, rank 64 115 and 113.)
template <bool kF32>
__device__ __forceinline__ void up_blocks_many(const Call& c, int index, const Tile& t, int group, int tid, uint4* h_lds,
                                               uint4* third_lds) {
  constexpr int RT = kTurnTiles, kPairs = RT / 2;
  const Bank& b = c.bank;
  const int tokens = c.tile_token[index * kTileTokens + (tid & 63)];
  const AdapterSlot slot = t.slot >= 0 ? b.table[t.slot] : AdapterSlot{0, 0.f};
  const int tiles = (slot.rank + 15) >> 4;
  const int lane = tid & 63, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int block = 4 * group + wave, n = 64 * block + 8 * q;   // past the last block: no output is a lane's
  const float* low_h = c.low + __shfl(tokens, 16 * wave + (lane & 15), 64) * (int64_t)(16 * b.rank_tiles) + 4 * q;
  const uint8_t* up = b.up_at(t.slot, block) + 16 * lane;
  const bool low = (lane & 15) < 8;
  uint4 base[kColumns][kF32 ? 4 : 2];
  int64_t token[kColumns][2];
  load_base<kF32>(c, tokens, n, lane, base, token);
  v4f acc[kColumns][4];
#pragma unroll
  for (int i = 0; i < kColumns; ++i) from_base<kF32>(base[i], low, acc[i]);
  for (int r0 = 0; r0 < tiles; r0 += RT) {
    v4f h[RT];
    uint4 w[RT][2];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int at = min(r0 + r, tiles - 1);
      h[r] = load_h(low_h + 16 * at);
      w[r][0] = ldg128(up + 2048 * at), w[r][1] = ldg128(up + 2048 * at + 1024);
    }
    if (r0) __syncthreads();   // the h before this has been read
    put_h(h, slot.rank - 16 * r0 - 4 * q, h_lds + wave * RT * 64 + lane, third_lds + wave * kPairs * 64 + lane);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kColumns; ++i)
      if (16 * i < t.rows)
        up_tiles<RT>(w, h_lds + i * RT * 64 + lane, third_lds + i * kPairs * 64 + lane, tiles - r0, acc[i]);
  }
#pragma unroll
  for (int i = 0; i < kColumns; ++i)
    if (16 * i < t.rows) store_y(c, t.rows, i, n + (low ? 0 : 32), lane, low, token[i], acc[i]);
}

// RT rank tiles, or in turns if there are more. kTurns: for fewer workgroups than there can be tiles. With room for two
// waves a SIMD or more the compiler keeps the sums in VGPRs. It must: where it had them in AGPRs, its copy of a base that
// no rank tile adds to (a tile without an adapter) held the first of four values four times. At most three waves: rank 64,
// 8 adapters, 4096 tokens, 1536 columns and 24576 rows take 106 us (FP32 base 131), with no such limit 112 (137).
template <int RT, bool kF32, bool kTurns>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 3))) void adapter_up_kernel(Call c) {
  constexpr int kHeld = RT > kMostTiles ? kTurnTiles : RT;
  __shared__ uint4 h_lds[kColumns * kHeld * 64];
  __shared__ uint4 third_lds[kColumns * ((kHeld + 1) / 2) * 64];
  const int groups = (c.bank.blocks + 3) / 4, group = blockIdx.x % groups;
  int index = blockIdx.x / groups;
  Tile t = c.tile[index];
  const Tile all = c.tile[c.tiles];
  if (t.rows == 0) return;
  auto blocks = [&](const Tile& tile, int tid) {
    if constexpr (RT <= kMostTiles) up_blocks<RT, kF32>(c, index, tile, group, all.slot, tid, h_lds, third_lds);
    else up_blocks_many<kF32>(c, index, tile, group, tid, h_lds, third_lds);
  };
  blocks(t, threadIdx.x);
  if constexpr (kTurns)
    for (index += gridDim.x / groups; index < all.rows; index += gridDim.x / groups) {
      __syncthreads();   // before the next tile's h
      blocks(c.tile[index], thread_here());
    }
}

bool is_aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
uint64_t round256(uint64_t n) { return (n + 255) & ~(uint64_t)255; }

// Tiles that T tokens in `slots` groups and the one without can make at most.
int tiles_of(const Bank& b, int tokens) {
  const int groups = std::min(b.slots + 1, tokens);
  return (int)(((int64_t)tokens + (int64_t)groups * (kTileTokens - 1)) / kTileTokens);
}

// Which calls are of few tokens: up to 64, and with at most 64 ranks to the 128 that a wave can hold. Few and grouped,
// BF16 base, 16384 columns and 7168 rows: 16 adapters of rank 64, 64 tokens 17.2 and 20.4 us, 128 22.6 and 20.5; 2 of rank
// 16, 128 tokens 10.8 and 13.3; 16 of rank 128, 32 tokens 25.4 and 27.5, 64 31.8 and 29.1, 128 41.3 and 28.6. 16 of rank
// 128, 64 tokens, 1536 columns and 24576 rows 32.0 and 33.3, 7168 and 1536 16.6 and 19.3. 1536 and 24576, 16 of rank 32:
// 64 tokens 14.3 and 18.0, 128 19.9 and 18.0; 7168 and 576, 4 of rank 64: 120 tokens 14.0 and 16.8.
bool is_few(const Bank& b, int tokens) { return tokens <= (b.rank_tiles <= 4 ? kFewTokens : kFewTokens / 2); }

// Parts of K. Few tokens: as many as give each wave a unit of 64, since how many adapters the tokens share is not known
// here. Grouped form: the most that down may take (locate): as many as are resident together (two a CU) and no more,
// since a few beyond would run alone after the rest, if every tile is full; at least two stages each. In both, parts T is
// at most kWantGroups kTileTokens + T.
int parts_of(const Bank& b, int tokens) {
  if (is_few(b, tokens)) return std::max(1, std::min(kMaxParts, b.chunks / 8));
  return std::max(1, std::min({kMaxParts, b.k / (2 * kStageK), kWantGroups * kTileTokens / tokens}));
}

}  // namespace

struct mx_adapters {
  mx_ctx* ctx;
  Bank bank;
  uint8_t* down;
  uint8_t* up;
  AdapterSlot* table;
  int32_t max_rank;
};

using mxi::as_stream;
using mxi::use;

namespace {

struct Workspace {
  uint64_t pair_row, row_pair, tile, tile_token, low, bytes;   // offsets; the plan's first at 0
};

Workspace workspace_of(const Bank& b, int32_t tokens) {
  const uint64_t rows = std::min((uint64_t)tokens * kMaxParts, (uint64_t)kWantGroups * kTileTokens + tokens);
  Workspace w;
  w.pair_row = round256(4 * ((uint64_t)b.slots + 1));
  w.row_pair = w.pair_row + round256(4 * (uint64_t)tokens);
  w.tile = w.row_pair + round256(4 * (uint64_t)tokens);
  w.tile_token = w.tile + round256(sizeof(Tile) * ((uint64_t)tiles_of(b, tokens) + 1));
  w.low = w.tile_token + round256(4 * kTileTokens * (uint64_t)tiles_of(b, tokens));
  w.bytes = w.low + round256(rows * 64 * b.rank_tiles);
  return w;
}

template <int RT>
int launch_fused(const Call& c, bool f32, hipStream_t st) {
  const dim3 grid((c.bank.blocks + 15) / 16, c.tokens);
  hipLaunchKernelGGL((f32 ? adapter_few_kernel<RT, true> : adapter_few_kernel<RT, false>), grid, dim3(1024), 0, st, c);
  MX_LAUNCH_CHECK("adapter_few_kernel");
  return MX_OK;
}

int launch_few(const Call& c, bool f32, hipStream_t st) {
  const int rt = c.bank.rank_tiles;
  if (rt <= 2 && (16 * rt + std::min(c.tokens, 64)) * c.bank.chunks <= kFusedBytes / 64)
    return rt == 1 ? launch_fused<1>(c, f32, st) : launch_fused<2>(c, f32, st);
  hipLaunchKernelGGL((rt == 1   ? adapter_few_down_kernel<1>
                      : rt == 2 ? adapter_few_down_kernel<2>
                                : adapter_few_down_kernel<4>),
                     dim3(c.parts, c.tokens), dim3(256), 0, st, c);
  MX_LAUNCH_CHECK("adapter_few_down_kernel");
  const dim3 grid((c.bank.blocks + 3) / 4, c.tokens);
  hipLaunchKernelGGL((f32 ? adapter_few_up_kernel<true> : adapter_few_up_kernel<false>), grid, dim3(256), 0, st, c);
  MX_LAUNCH_CHECK("adapter_few_up_kernel");
  return MX_OK;
}

unsigned round8(int64_t n) { return (unsigned)((n + 7) / 8 * 8); }

template <int RT, bool kStream>
int launch_down(const Call& c, hipStream_t st) {
  const int most = c.tiles * ((c.bank.rank_tiles + RT - 1) / RT);
  constexpr size_t lds = std::max(2 * kStageBytes, 4 * kColumns * RT * 1024);
  hipLaunchKernelGGL((adapter_down_kernel<RT, kStream>), dim3(round8(std::max(std::min(c.parts * most, kWantGroups), most))),
                     dim3(256), lds, st, c);
  MX_LAUNCH_CHECK("adapter_down_kernel");
  return MX_OK;
}

template <int RT, bool kTurns>
int launch_up(const Call& c, int tiles, bool f32, hipStream_t st) {
  const int groups = (c.bank.blocks + 3) / 4;
  hipLaunchKernelGGL((f32 ? adapter_up_kernel<RT, true, kTurns> : adapter_up_kernel<RT, false, kTurns>),
                     dim3((unsigned)(groups * tiles)), dim3(256), 0, st, c);
  MX_LAUNCH_CHECK("adapter_up_kernel");
  return MX_OK;
}

// How many tiles the tokens make only the device knows; a bank of many slots could make far more than they do. Up has
// workgroups for the full ones and 32 more, or as many as are resident together, and takes the rest in turns: 1536
// columns, 24576 rows, rank 16, 200 tokens of 8 of 64 slots in any order 15.4 us, with 64 more 16.7; 7168 columns, 1536
// rows (of which 170 tiles are resident), 600 tokens of 64 of 1024 slots 16.7, with 32 and 16 more some 2 and 4 above.
template <int RT>
int launch_up(const Call& c, bool f32, hipStream_t st) {
  const int tiles = c.tokens / kTileTokens + std::max(32, 1024 / ((c.bank.blocks + 3) / 4));
  return tiles < c.tiles ? launch_up<RT, true>(c, tiles, f32, st) : launch_up<RT, false>(c, c.tiles, f32, st);
}

int launch_groups(const Call& c, bool f32, hipStream_t st) {
  const int rt = c.bank.rank_tiles;
  const bool stream = rt <= 4 &&   // with more rank tiles x is read again
                      (int64_t)c.tokens * (2 * (int64_t)c.bank.k + (f32 ? 6 : 4) * (int64_t)c.bank.n) > kStreamBytes;
  if (int s = rt == 1   ? (stream ? launch_down<1, true>(c, st) : launch_down<1, false>(c, st))
              : rt == 2 ? (stream ? launch_down<2, true>(c, st) : launch_down<2, false>(c, st))
                        : (stream ? launch_down<4, true>(c, st) : launch_down<4, false>(c, st)))
    return s;
  if (c.parts > 1 && rt > 1) {
    const int entries = c.tokens * 4 * rt;
    if (c.parts > 8) hipLaunchKernelGGL(adapter_sum_kernel<4>, dim3((entries + 63) / 64), dim3(256), 0, st, c);
    else hipLaunchKernelGGL(adapter_sum_kernel<1>, dim3((entries + 255) / 256), dim3(256), 0, st, c);
    MX_LAUNCH_CHECK("adapter_sum_kernel");
  }
  if (rt == 1) return launch_up<1>(c, f32, st);
  if (rt == 2) return launch_up<2>(c, f32, st);
  if (rt <= 4) return launch_up<4>(c, f32, st);
  return rt <= kMostTiles ? launch_up<kMostTiles>(c, f32, st) : launch_up<kMaxRank / 16>(c, f32, st);
}

}  // namespace

extern "C" {

int mx_adapters_create(mx_ctx* ctx, int32_t n, int32_t k, int32_t slots, int32_t max_rank, mx_adapters** out) {
  const char* who = "mx_adapters_create";
  MX_REQUIRE(out != nullptr, "%s: null output", who);
  MX_REQUIRE(n >= 8 && n % 8 == 0 && n <= kMaxWidth && k >= 8 && k % 8 == 0 && k <= kMaxWidth,
             "%s: rows %d and width %d must be multiples of 8 in [8, %d]", who, n, k, kMaxWidth);
  MX_REQUIRE(slots >= 1 && slots <= kMaxSlots, "%s: %d slots outside [1, %d]", who, slots, kMaxSlots);
  MX_REQUIRE(max_rank >= 1 && max_rank <= kMaxRank, "%s: rank %d outside [1, %d]", who, max_rank, kMaxRank);
  if (int s = use(ctx)) return s;
  Bank b{};
  b.n = n, b.k = k, b.slots = slots;
  b.rank_tiles = (max_rank + 15) / 16, b.chunks = (k + 63) / 64 * 2, b.blocks = (n + 63) / 64;
  const uint64_t down = (uint64_t)slots * b.down_bytes(), up = (uint64_t)slots * b.up_bytes();
  void* base = nullptr;
  if (int s = mx_malloc(ctx, down + up + round256(slots * sizeof(AdapterSlot)), &base)) return s;
  uint8_t* p = (uint8_t*)base;
  mx_adapters* a = new (std::nothrow) mx_adapters{ctx, b, p, p + down, (AdapterSlot*)(p + down + up), max_rank};
  if (!a || hipMemset(a->table, 0, slots * sizeof(AdapterSlot)) != hipSuccess ||
      hipStreamSynchronize(nullptr) != hipSuccess) {
    (void)hipGetLastError();
    delete a;
    (void)mx_free(ctx, base);
    return mxi::fail(MX_ERR_MEMORY, "%s: no memory for the bank", who);
  }
  a->bank.down = a->down, a->bank.up = a->up, a->bank.table = a->table;
  *out = a;
  return MX_OK;
}

int mx_adapters_destroy(mx_adapters* a) {
  if (!a) return MX_OK;
  const int status = mx_free(a->ctx, a->down);
  delete a;
  return status;
}

int mx_adapters_load(mx_adapters* a, int32_t slot, const uint16_t* down, const uint16_t* up, int32_t rank, float scale,
                     void* stream) {
  const char* who = "mx_adapters_load";
  if (!a) return mxi::fail(MX_ERR_STATE, "%s: bank is closed", who);
  MX_REQUIRE(slot >= 0 && slot < a->bank.slots, "%s: slot %d outside [0, %d)", who, slot, a->bank.slots);
  MX_REQUIRE(rank >= 0 && rank <= a->max_rank, "%s: rank %d outside [0, %d]", who, rank, a->max_rank);
  MX_REQUIRE(rank == 0 || (down && up), "%s: null pointer", who);
  MX_REQUIRE(is_aligned(down, 2) && is_aligned(up, 2), "%s: weights must be 2-byte aligned", who);
  MX_REQUIRE(std::isfinite(scale), "%s: the scale must be finite", who);
  if (int s = use(a->ctx)) return s;
  const Bank& b = a->bank;
  hipStream_t st = as_stream(stream);
  const int tiles = (rank + 15) / 16;
  if (rank) {
    hipLaunchKernelGGL(adapter_store_down_kernel, dim3(b.chunks, tiles), dim3(64), 0, st, b, a->down, slot, down, rank);
    MX_LAUNCH_CHECK("adapter_store_down_kernel");
  }
  hipLaunchKernelGGL(adapter_store_up_kernel, dim3(rank ? b.blocks : 1, rank ? tiles : 1), dim3(128), 0, st, b, a->up,
                     a->table, slot, up, rank, scale);
  MX_LAUNCH_CHECK("adapter_store_up_kernel");
  return MX_OK;
}

uint64_t mx_adapters_workspace_bytes(const mx_adapters* a, int32_t tokens) {
  return a && tokens >= 1 && tokens <= kMaxTokens ? workspace_of(a->bank, tokens).bytes : 0;
}

int mx_adapters_apply(mx_adapters* a, const uint16_t* x, int64_t x_stride, const int32_t* ids, const mx_row_plan* plan,
                      int32_t tokens, const void* base, int32_t base_type, int64_t base_stride, uint16_t* y,
                      int64_t y_stride, void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* who = "mx_adapters_apply";
  if (!a) return mxi::fail(MX_ERR_STATE, "%s: bank is closed", who);
  const Bank& b = a->bank;
  MX_REQUIRE(tokens >= 0 && tokens <= kMaxTokens, "%s: token count %d outside [0, %d]", who, tokens, kMaxTokens);
  MX_REQUIRE(base_type == MX_ROWS_BF16 || base_type == MX_ROWS_F32, "%s: base type %d", who, base_type);
  if (!tokens) return use(a->ctx);
  MX_REQUIRE(x && ids && base && y && workspace, "%s: null pointer", who);
  const bool f32 = base_type == MX_ROWS_F32;
  MX_REQUIRE(x_stride >= b.k && base_stride >= b.n && y_stride >= b.n && x_stride % 8 == 0 && y_stride % 8 == 0 &&
                 base_stride % (f32 ? 4 : 8) == 0 && x_stride <= INT32_MAX && y_stride <= INT32_MAX &&
                 base_stride <= INT32_MAX,
             "%s: row strides must hold a row and keep rows 16-byte aligned", who);
  MX_REQUIRE(is_aligned(x, 16) && is_aligned(base, 16) && is_aligned(y, 16) && is_aligned(ids, 4),
             "%s: x, base and y must be 16-byte and ids 4-byte aligned", who);
  MX_REQUIRE((const void*)y != base || (!f32 && y_stride == base_stride),
             "%s: y may be base only with the same type and stride", who);
  MX_REQUIRE(y != x, "%s: y may not be x", who);
  const Workspace w = workspace_of(b, tokens);
  MX_REQUIRE(is_aligned(workspace, 256) && workspace_bytes >= w.bytes,
             "%s: workspace must be 256-byte aligned and hold %llu bytes", who, (unsigned long long)w.bytes);
  if (plan) {
    MX_REQUIRE(plan->first && plan->pair_row && plan->row_pair, "%s: plan pointer is null", who);
    MX_REQUIRE(is_aligned(plan->first, 4) && is_aligned(plan->row_pair, 4), "%s: plan arrays must be 4-byte aligned",
               who);
  }
  if (int s = use(a->ctx)) return s;
  hipStream_t st = as_stream(stream);
  uint8_t* ws = (uint8_t*)workspace;
  Call c{b, x, x_stride, ids, nullptr, nullptr, (Tile*)(ws + w.tile), (int32_t*)(ws + w.tile_token), tokens,
         parts_of(b, tokens), (float*)(ws + w.low), base, base_stride, y, y_stride, 0};
  if (w.low + (uint64_t)c.parts * tokens * 64 * b.rank_tiles > w.bytes)   // parts_of and workspace_of belong together
    return mxi::fail(MX_ERR_STATE, "%s: %d parts of %d tokens exceed the workspace", who, c.parts, tokens);
  if (is_few(b, tokens)) return launch_few(c, f32, st);
  mx_row_plan own{(int32_t*)ws, (int32_t*)(ws + w.pair_row), (int32_t*)(ws + w.row_pair)};
  if (!plan && tokens > kOwnTokens) {
    if (int s = mxi::row_plan(ids, tokens, b.slots, own, st)) return s;
    plan = &own;
  }
  if (plan) c.first = plan->first, c.row_pair = plan->row_pair;
  c.tiles = tiles_of(b, tokens);
  return launch_groups(c, f32, st);
}

}  // extern "C"
