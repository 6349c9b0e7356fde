// Low-rank adapters of many requests beside a projection: y[t] = base[t] + scale_a up_a (down_a x[t]), a = ids[t].
//
// The quantized base weights cannot take an adapter in, so each token's pair of thin matrices runs beside them: down
// [rank][K] then up [N][rank], both BF16, with the projection's output (BF16, or its FP32 sums) as base and one rounding.
// Both products run on V_MFMA_F32_16X16X32_BF16 with the weights as operand A and tokens as operand B's columns:
//   A lane l = row l % 16, K 8 (l / 16) + 0..7; B lane l = column l % 16, same K; D lane l register i = row 4 (l / 16)
//   + i, column l % 16.
// So down's D gives lane (token, q) the ranks 4q..4q+3 of a 16-rank tile, which is what up's operand B wants of that
// lane: up takes the 16 ranks of a tile in one MFMA of 32, K slots 0..3 of a lane holding its ranks of bf16(h) and 4..7
// those of bf16(h - bf16(h)) against up's values given twice. h = scale * (down x) keeps about 16 significant bits that
// way, for no further load of up.
//
// The bank stores each slot in operand order, padded with zeros to whole tiles:
//   down: [rank tile][K chunk of 32][lane] 16 bytes: rank 16 rt + l % 16, K 32 c + 8 (l / 16) + 0..7
//   up: [block of 64 outputs][rank tile][half][lane] 16 bytes: two tiles j = 2 half, 2 half + 1 of four ranks each;
//   row m of tile j is output 64 b + 16 (m / 4) + 4 j + m % 4, so a lane's D registers of the four tiles are 16
//   consecutive outputs of its token.
#include <algorithm>
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
constexpr int kTokenForm = 32;     // calls of up to this many tokens run a token at a time
constexpr int kColumns = 2;        // 16-token column tiles of a workgroup in the grouped form
constexpr int kTileTokens = 16 * kColumns;
constexpr int kMaxParts = 32;      // parts of K
constexpr int kWantGroups = 512;   // workgroups that the split of K aims at
constexpr int kRankGroup = 4;      // rank tiles in registers at once

struct AdapterSlot {
  int32_t rank;   // 0: empty
  float scale;
};

struct Bank {
  const uint8_t* down;
  const uint8_t* up;
  const AdapterSlot* table;
  int32_t n, k, slots;
  int32_t rank_tiles, chunks, blocks;   // of the largest rank; K chunks of 32; blocks of 64 outputs
  __host__ __device__ int64_t down_bytes() const { return (int64_t)rank_tiles * chunks * 1024; }
  __host__ __device__ int64_t up_bytes() const { return (int64_t)blocks * rank_tiles * 2048; }
};

__device__ __forceinline__ v8bf as_bf(uint4 v) { return __builtin_bit_cast(v8bf, v); }

// ---- loading a slot ----

__global__ __launch_bounds__(64) void adapter_down_kernel(Bank b, uint8_t* bank, int slot, const uint16_t* src, int rank) {
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

__global__ __launch_bounds__(128) void adapter_up_kernel(Bank b, uint8_t* bank, AdapterSlot* table, int slot,
                                                         const uint16_t* src, int rank, float scale) {
  const int lane = threadIdx.x & 63, half = threadIdx.x >> 6, block = blockIdx.x, rt = blockIdx.y;
  if (block == 0 && rt == 0 && threadIdx.x == 0) table[slot] = AdapterSlot{rank, scale};
  if (rank == 0) return;
  const int m = lane & 15, r0 = 16 * rt + 4 * (lane >> 4);
  uint32_t w[4] = {0, 0, 0, 0};
  for (int i = 0; i < 8; ++i) {
    const int n = 64 * block + 16 * (m >> 2) + 4 * (2 * half + (i >> 2)) + (m & 3), r = r0 + (i & 3);
    const uint32_t v = n < b.n && r < rank ? src[(int64_t)n * rank + r] : 0;
    w[i >> 1] |= v << (16 * (i & 1));
  }
  uint8_t* dst = bank + slot * b.up_bytes() + ((int64_t)block * b.rank_tiles + rt) * 2048 + 1024 * half + 16 * lane;
  *(uint4*)dst = make_uint4(w[0], w[1], w[2], w[3]);
}

// ---- the tokens of a workgroup ----

struct Call {
  Bank bank;
  const uint16_t* x;
  int64_t x_stride;
  const int32_t* ids;
  const int32_t* first;      // grouped form: the plan of ids (slots groups)
  const int32_t* row_pair;
  int32_t tokens, parts;
  float* low;                // [parts][T][16 rank_tiles]: partial sums of down x
  const void* base;
  int64_t base_stride;
  uint16_t* y;
  int64_t y_stride;
  int32_t blocks_per_group;  // output blocks of a workgroup
};

struct Tile {
  int slot;        // -1: tokens without an adapter
  int row, rows;   // grouped: sorted rows; token form: the token, 1
};

// Tile `index` of the plan's groups, kTileTokens sorted rows each (a group's last one short), the tokens without an
// adapter last; rows = 0 past the end. Every wave searches for itself, 64 groups at a time.
__device__ __forceinline__ Tile find_tile(const Call& c, int index) {
  const int lane = threadIdx.x & 63, slots = c.bank.slots;
  int before = 0;
  for (int g0 = 0; g0 <= slots; g0 += 64) {
    const int g = g0 + lane;
    int lo = g <= slots ? c.first[g] : c.tokens, hi = g < slots ? c.first[g + 1] : c.tokens;
    lo = min(max(lo, 0), c.tokens);
    hi = min(max(hi, lo), c.tokens);
    const int count = (hi - lo + kTileTokens - 1) / kTileTokens;
    int upto = count;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(upto, d, 64);
      if (lane >= d) upto += o;
    }
    const int total = __shfl(upto, 63, 64);
    if (index < before + total) {
      const int at = __ffsll((unsigned long long)__ballot(upto > index - before)) - 1;
      const int skip = index - before - (__shfl(upto, at, 64) - __shfl(count, at, 64));
      const int l = __shfl(lo, at, 64) + skip * kTileTokens, h = __shfl(hi, at, 64);
      return Tile{g0 + at < slots ? g0 + at : -1, l, min(kTileTokens, h - l)};
    }
    before += total;
  }
  return Tile{-1, 0, 0};
}

template <bool kGrouped>
__device__ __forceinline__ Tile tile_of(const Call& c) {
  Tile t;
  if constexpr (kGrouped) {
    t = find_tile(c, blockIdx.x);
  } else {
    const int id = c.ids[blockIdx.x];
    t = Tile{id >= 0 && id < c.bank.slots ? id : -1, (int)blockIdx.x, 1};
  }
  return Tile{__builtin_amdgcn_readfirstlane(t.slot), __builtin_amdgcn_readfirstlane(t.row),
              __builtin_amdgcn_readfirstlane(t.rows)};
}

// The token of column `col` of the tile; columns past the last repeat it.
template <bool kGrouped>
__device__ __forceinline__ int token_of(const Call& c, const Tile& t, int col) {
  if constexpr (!kGrouped) return t.row;
  const int p = c.row_pair[t.row + min(col, t.rows - 1)];
  return p >= 0 && p < c.tokens ? p : 0;
}

// ---- down: partial sums of h ----

// grid (tiles, parts), 4 waves: a part of the K chunks for the tile's tokens and all ranks, the waves taking the chunks
// in turn and added in wave order.
template <bool kGrouped>
__global__ __launch_bounds__(256) void adapter_down_gemm_kernel(Call c) {
  constexpr int CT = kGrouped ? kColumns : 1;
  __shared__ v4f red[4][CT][kRankGroup][64];
  const Tile t = tile_of<kGrouped>(c);
  if (t.rows == 0 || t.slot < 0) return;
  const Bank& b = c.bank;
  const int rank = b.table[t.slot].rank, tiles = (rank + 15) >> 4;
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c0 = (int)((int64_t)b.chunks * blockIdx.y / c.parts), c1 = (int)((int64_t)b.chunks * (blockIdx.y + 1) / c.parts);
  int token[CT];
  const uint8_t* x[CT];
#pragma unroll
  for (int i = 0; i < CT; ++i) {
    token[i] = token_of<kGrouped>(c, t, 16 * i + (lane & 15));
    x[i] = (const uint8_t*)(c.x + token[i] * c.x_stride) + 16 * q;
  }
  const uint8_t* w = b.down + t.slot * b.down_bytes() + 16 * lane;
  for (int r0 = 0; r0 < tiles; r0 += kRankGroup) {
    v4f acc[CT][kRankGroup];
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
      for (int r = 0; r < kRankGroup; ++r) acc[i][r] = v4f{0.f, 0.f, 0.f, 0.f};
    for (int ch = c0 + wave; ch < c1; ch += 4) {
      uint4 xv[CT], wv[kRankGroup];
#pragma unroll
      for (int i = 0; i < CT; ++i)
        xv[i] = 32 * ch + 8 * q < b.k ? ldg128(x[i] + 64 * ch) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < kRankGroup; ++r)
        if (r0 + r < tiles) wv[r] = ldg128(w + ((int64_t)(r0 + r) * b.chunks + ch) * 1024);
#pragma unroll
      for (int r = 0; r < kRankGroup; ++r)
        if (r0 + r < tiles)
#pragma unroll
          for (int i = 0; i < CT; ++i)
            acc[i][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(wv[r]), as_bf(xv[i]), acc[i][r], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
      for (int r = 0; r < kRankGroup; ++r) red[wave][i][r][lane] = acc[i][r];
    __syncthreads();
    for (int e = wave; e < CT * kRankGroup; e += 4) {
      const int i = e / kRankGroup, r = e % kRankGroup, col = 16 * i + (lane & 15);
      if (r0 + r < tiles && col < t.rows) {
        const v4f s = ((red[0][i][r][lane] + red[1][i][r][lane]) + red[2][i][r][lane]) + red[3][i][r][lane];
        const int tok = token_of<kGrouped>(c, t, col);
        *(v4f*)(c.low + ((int64_t)blockIdx.y * c.tokens + tok) * (16 * b.rank_tiles) + 16 * (r0 + r) + 4 * q) = s;
      }
    }
    __syncthreads();
  }
}

// ---- up: y = base + up h ----

template <bool kF32>
struct BaseValues;   // 16 consecutive values of base, the second eight where they exist

template <>
struct BaseValues<true> {
  float4 v[4];
  __device__ __forceinline__ void load(const void* p, bool second) {
    const float4* s = (const float4*)p;
    v[0] = s[0], v[1] = s[1];
    if (second) v[2] = s[2], v[3] = s[3];
  }
  __device__ __forceinline__ v4f four(int j) const { return v4f{v[j].x, v[j].y, v[j].z, v[j].w}; }
};

template <>
struct BaseValues<false> {
  uint4 v[2];
  __device__ __forceinline__ void load(const void* p, bool second) {
    const uint4* s = (const uint4*)p;
    v[0] = s[0];
    if (second) v[1] = s[1];
  }
  __device__ __forceinline__ v4f four(int j) const {
    const uint4 u = v[j >> 1];
    const uint32_t a = j & 1 ? u.z : u.x, b = j & 1 ? u.w : u.y;
    return v4f{mx::u2f(a << 16), mx::u2f(a & 0xFFFF0000u), mx::u2f(b << 16), mx::u2f(b & 0xFFFF0000u)};
  }
};

// grid (tiles, groups of output blocks), 4 waves. The tile's h (the parts' sums, in order, times the slot's scale) goes
// to LDS as operand B; then each wave takes output blocks of 64 in turn.
template <bool kGrouped, bool kF32>
__global__ __launch_bounds__(256) void adapter_up_gemm_kernel(Call c) {
  constexpr int CT = kGrouped ? kColumns : 1;
  extern __shared__ uint4 h_lds[];   // [CT][rank tiles][64]
  const Tile t = tile_of<kGrouped>(c);
  if (t.rows == 0) return;
  const Bank& b = c.bank;
  const AdapterSlot slot = t.slot >= 0 ? b.table[t.slot] : AdapterSlot{0, 0.f};
  const int tiles = (slot.rank + 15) >> 4;
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t rank_stride = 16 * b.rank_tiles;
  for (int e = tid; e < CT * tiles * 64; e += 256) {
    const int l = e & 63, r = (e >> 6) % tiles, i = (e >> 6) / tiles;
    const int tok = token_of<kGrouped>(c, t, 16 * i + (l & 15)), r0 = 16 * r + 4 * (l >> 4);
    const float* p = c.low + tok * rank_stride + r0;
    v4f s = *(const v4f*)p;
    for (int n = 1; n < c.parts; ++n) s = s + *(const v4f*)(p + n * c.tokens * rank_stride);
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float h = r0 + k < slot.rank ? slot.scale * s[k] : 0.f;
      hi[k] = mx::bf16_bits(h);
      const bool finite = (hi[k] & 0x7F80u) != 0x7F80u;   // an infinite h has no second term
      lo[k] = finite ? mx::bf16_bits(h - mx::bf16_value(hi[k])) : 0u;
    }
    h_lds[e] = make_uint4(hi[0] | hi[1] << 16, hi[2] | hi[3] << 16, lo[0] | lo[1] << 16, lo[2] | lo[3] << 16);
  }
  __syncthreads();
  int64_t at_base[CT], at_y[CT];
  bool live[CT];
#pragma unroll
  for (int i = 0; i < CT; ++i) {
    const int col = 16 * i + (lane & 15);
    const int64_t tok = token_of<kGrouped>(c, t, col);
    live[i] = col < t.rows;
    at_base[i] = tok * c.base_stride;
    at_y[i] = tok * c.y_stride;
  }
  const uint8_t* up = b.up + (t.slot >= 0 ? t.slot : 0) * b.up_bytes() + 16 * lane;
  const int b0 = blockIdx.y * c.blocks_per_group, b1 = min(b0 + c.blocks_per_group, b.blocks);
  for (int block = b0 + wave; block < b1; block += 4) {
    const int n = 64 * block + 16 * q;
    const bool any = n < b.n, second = n + 8 < b.n;
    BaseValues<kF32> base[CT];
#pragma unroll
    for (int i = 0; i < CT; ++i)
      if (live[i] && any)
        base[i].load(kF32 ? (const void*)((const float*)c.base + at_base[i] + n)
                          : (const void*)((const uint16_t*)c.base + at_base[i] + n), second);
    v4f acc[CT][4];
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    const uint8_t* w = up + (int64_t)block * b.rank_tiles * 2048;
    for (int r = 0; r < tiles; ++r) {
      const uint4 w01 = ldg128(w + 2048 * r), w23 = ldg128(w + 2048 * r + 1024);
      const uint4 a[4] = {make_uint4(w01.x, w01.y, w01.x, w01.y), make_uint4(w01.z, w01.w, w01.z, w01.w),
                          make_uint4(w23.x, w23.y, w23.x, w23.y), make_uint4(w23.z, w23.w, w23.z, w23.w)};
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        const v8bf h = as_bf(h_lds[(i * tiles + r) * 64 + lane]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(a[j]), h, acc[i][j], 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < CT; ++i) {
      if (!live[i] || !any || (!kGrouped && (lane & 15))) continue;
      uint32_t out[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v4f v = base[i].four(j);
        if (tiles) v = v + acc[i][j];
        out[2 * j] = mx::bf16_bits(v[0]) | mx::bf16_bits(v[1]) << 16;
        out[2 * j + 1] = mx::bf16_bits(v[2]) | mx::bf16_bits(v[3]) << 16;
      }
      uint4* y = (uint4*)(c.y + at_y[i] + n);
      y[0] = make_uint4(out[0], out[1], out[2], out[3]);
      if (second) y[1] = make_uint4(out[4], out[5], out[6], out[7]);
    }
  }
}

bool is_aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
uint64_t round256(uint64_t n) { return (n + 255) & ~(uint64_t)255; }

// Parts of K for T tokens: enough workgroups for the chip, at least 8 chunks a part. parts T <= 16 kWantGroups kColumns + T.
int parts_of(int chunks, int tokens) {
  const int tiles = tokens <= kTokenForm ? tokens : (tokens + kTileTokens - 1) / kTileTokens;
  const int most = std::min(kMaxParts, std::max(1, chunks / 8));
  return std::max(1, std::min(most, (kWantGroups + tiles - 1) / tiles));
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
  uint64_t pair_row, row_pair, low, bytes;   // offsets; the plan's first at 0
};

Workspace workspace_of(const Bank& b, int32_t tokens) {
  const uint64_t rows = std::min((uint64_t)tokens * kMaxParts, (uint64_t)kWantGroups * kTileTokens + tokens);
  Workspace w;
  w.pair_row = round256(4 * ((uint64_t)b.slots + 1));
  w.row_pair = w.pair_row + round256(4 * (uint64_t)tokens);
  w.low = w.row_pair + round256(4 * (uint64_t)tokens);
  w.bytes = w.low + round256(rows * 64 * b.rank_tiles);
  return w;
}

template <bool kGrouped>
int launch(const Call& c, int tiles, bool f32, hipStream_t st) {
  const Bank& b = c.bank;
  hipLaunchKernelGGL((adapter_down_gemm_kernel<kGrouped>), dim3(tiles, c.parts), dim3(256), 0, st, c);
  MX_LAUNCH_CHECK("adapter_down_gemm_kernel");
  const size_t lds = (size_t)(kGrouped ? kColumns : 1) * b.rank_tiles * 1024;
  const dim3 grid(tiles, (b.blocks + c.blocks_per_group - 1) / c.blocks_per_group);
  if (f32) hipLaunchKernelGGL((adapter_up_gemm_kernel<kGrouped, true>), grid, dim3(256), lds, st, c);
  else hipLaunchKernelGGL((adapter_up_gemm_kernel<kGrouped, false>), grid, dim3(256), lds, st, c);
  MX_LAUNCH_CHECK("adapter_up_gemm_kernel");
  return MX_OK;
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
  b.rank_tiles = (max_rank + 15) / 16, b.chunks = (k + 31) / 32, b.blocks = (n + 63) / 64;
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
  if (int s = use(a->ctx)) return s;
  const Bank& b = a->bank;
  hipStream_t st = as_stream(stream);
  const int tiles = (rank + 15) / 16;
  if (rank) {
    hipLaunchKernelGGL(adapter_down_kernel, dim3(b.chunks, tiles), dim3(64), 0, st, b, a->down, slot, down, rank);
    MX_LAUNCH_CHECK("adapter_down_kernel");
  }
  hipLaunchKernelGGL(adapter_up_kernel, dim3(rank ? b.blocks : 1, rank ? tiles : 1), dim3(128), 0, st, b, a->up,
                     a->table, slot, up, rank, scale);
  MX_LAUNCH_CHECK("adapter_up_kernel");
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
  Call c{b, x, x_stride, ids, nullptr, nullptr, tokens, parts_of(b.chunks, tokens), (float*)(ws + w.low),
         base, base_stride, y, y_stride, 4};
  if (tokens <= kTokenForm) return launch<false>(c, tokens, f32, st);
  mx_row_plan own{(int32_t*)ws, (int32_t*)(ws + w.pair_row), (int32_t*)(ws + w.row_pair)};
  if (!plan) {
    if (int s = mxi::row_plan(ids, tokens, b.slots, own, st)) return s;
    plan = &own;
  }
  c.first = plan->first;
  c.row_pair = plan->row_pair;
  c.blocks_per_group = 16;
  const int groups = std::min(b.slots + 1, tokens);
  const int tiles = (int)(((int64_t)tokens + (int64_t)groups * (kTileTokens - 1)) / kTileTokens);
  return launch<true>(c, tiles, f32, st);
}

}  // extern "C"
