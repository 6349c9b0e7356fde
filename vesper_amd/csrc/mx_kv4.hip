// Appending to a paged key/value cache in 4 bits.
#include <algorithm>
#include <type_traits>

#include "mx_kv4.h"

namespace {

using namespace mxh;
using namespace mxk;

// ---- append ----

struct AppendArgs {
  mx_kv4 cache;
  mx_kv4_rows rows;
  mx_rotation rot;
  int64_t total;   // key rows, then value rows
  bool wide;
};

// Latency: a row's chain of loads, sums and one store. 4096 latents of 576 in 7.0 us (11.8 MB), 16 in 3.4, an empty launch
// about 2.
//
// A row on L lanes: normalized, rotated and rounded to BF16; then each quad of lanes holds a block of 32 values, whose
// largest magnitude (as integers, so that an infinity or NaN is the largest) gives the scale.
template <int L, int NI, bool F32>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  const int g = threadIdx.x % L;
  const int64_t mine = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L, r = mine < a.total ? mine : a.total - 1;
  const int heads = a.cache.heads;
  const int64_t key_rows = (int64_t)a.rows.tokens * heads;
  const bool value = r >= key_rows;
  const uint32_t row = (uint32_t)(value ? r - key_rows : r), t = row / (uint32_t)heads, h = row - t * (uint32_t)heads;
  const int64_t slot = a.rows.slots[t];
  const int width = value ? a.cache.value_width : a.cache.width;
  const int64_t size = F32 ? 4 : 2;
  const void* x = value ? (const uint8_t*)a.rows.v + (t * a.rows.v_stride + (int64_t)h * width) * size
                        : (const uint8_t*)a.rows.k + (t * a.rows.k_stride + (int64_t)h * width) * size;
  Raw8<F32> raw[NI];
  load_row<L, NI>(x, a.wide, 0, width, g, raw);
  mx_rotation rot = a.rot;
  const float* angles = nullptr;
  const bool placed = place_of(rot, t, angles);
  if (value) rot.norm = 0, angles = nullptr;
  Columns<NI> cols;
  weights_of<L>(rot, a.rows.weight, 0, g, cols);
  angles_of<L>(rot, angles, 0, width, g, cols);
  float v[NI][8];
  finish_row<L, NI>(x, a.wide, rot, cols, 0, g, raw, v);
  const int64_t page = slot / a.cache.page;
  if (mine >= a.total || slot < 0 || page >= a.cache.pages || !placed) return;
  const int64_t at = (page * heads + h) * a.cache.page + slot % a.cache.page;
  uint8_t* codes = (value ? a.cache.v_codes : a.cache.k_codes) + at * (width / 2);
  uint8_t* scales = (value ? a.cache.v_scales : a.cache.k_scales) + at * scale_pitch(width);
  uint16_t* rounded = value ? a.rows.v_rounded : a.rows.k_rounded;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = 8 * (i * L + g);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[i][j] = mxd::bf16_round_sel(v[i][j]);
      top = max(top, mx::f2u(v[i][j]) & 0x7FFFFFFFu);
    }
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, false));
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, false));
    if (c >= width) continue;
    // amax = m 2^k: 6 2^e >= amax from e = k - 2 on where m <= 1.5, else from k - 1
    const bool finite = top < 0x7F800000u;
    const uint32_t amax = max(top, mx::kAmaxFloorBits);
    uint32_t e8 = (amax >> 23) - ((amax & 0x7FFFFFu) <= 0x400000u ? 2 : 1);
    e8 = finite ? min(e8, 252u) : 255u;
    const float scale = mx::u2f(e8 << 23);
    uint32_t w = 0;
    if (finite) {
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[i][0], v[i][1], scale, 0);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[i][2], v[i][3], scale, 1);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[i][4], v[i][5], scale, 2);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[i][6], v[i][7], scale, 3);
    }
    *(uint32_t*)(codes + c / 2) = w;
    if ((g & 3) == 0) scales[c / 32] = (uint8_t)e8;
    if (rounded) {
      uint4 o;
      o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
      o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
      o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
      o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
      *(uint4*)(rounded + ((int64_t)t * heads + h) * width + c) = o;
    }
  }
}

}  // namespace

int mxk::check_cache(const char* who, const mx_kv4* c) {
  MX_REQUIRE(c, "%s: null cache", who);
  MX_REQUIRE(c->page >= 16 && c->page <= 1024 && (c->page & (c->page - 1)) == 0, "%s: page of %d tokens not a power of two in [16, 1024]",
             who, c->page);
  MX_REQUIRE(c->heads >= 1 && c->heads <= 1024, "%s: %d key heads outside [1, 1024]", who, c->heads);
  MX_REQUIRE(c->pages >= 1 && (int64_t)c->pages * c->heads * c->page <= (1ll << 40), "%s: %d pages", who, c->pages);
  const bool apart = c->v_codes || c->v_scales;
  if (apart)
    MX_REQUIRE((c->width == 64 || c->width == 128 || c->width == 256) && c->value_width == c->width,
               "%s: keys of %d and values of %d; 64, 128 or 256 of both are supported", who, c->width, c->value_width);
  else
    MX_REQUIRE((c->width == 512 || c->width == 576) && c->value_width == 512,
               "%s: latents of %d with values of %d; 512 or 576 with 512 are supported", who, c->width, c->value_width);
  MX_REQUIRE(c->k_codes && c->k_scales && (!apart || (c->v_codes && c->v_scales)), "%s: null cache array", who);
  MX_REQUIRE(aligned(c->k_codes, 16) && aligned(c->k_scales, 16) && aligned(c->v_codes, 16) && aligned(c->v_scales, 16),
             "%s: cache arrays must be 16-byte aligned", who);
  return MX_OK;
}

using mxi::as_stream;
using mxi::use;

extern "C" {

int mx_kv4_append(mx_ctx* ctx, const mx_kv4* cache, const mx_kv4_rows* rows, const mx_rotation* rotation, void* stream) {
  const char* who = "mx_kv4_append";
  if (int s = check_cache(who, cache)) return s;
  MX_REQUIRE(rows, "%s: null rows", who);
  MX_REQUIRE(rows->tokens >= 0 && rows->tokens <= kMaxTokens, "%s: token count %d outside [0, %d]", who, rows->tokens, kMaxTokens);
  MX_REQUIRE((int64_t)rows->tokens * cache->heads < (1ll << 30), "%s: 2^30 rows or more in all", who);
  MX_REQUIRE(rows->type == MX_ROWS_BF16 || rows->type == MX_ROWS_F32, "%s: row type %d", who, rows->type);
  const bool apart = cache->v_codes != nullptr;
  MX_REQUIRE(rows->k && rows->slots && (rows->v != nullptr) == apart, "%s: keys, slots and, where the cache holds them, values", who);
  MX_REQUIRE(apart || !rows->v_rounded, "%s: latents have no values of their own", who);
  const int64_t size = rows->type == MX_ROWS_F32 ? 4 : 2;
  MX_REQUIRE(rows->k_stride >= (int64_t)cache->heads * cache->width && rows->k_stride < (1ll << 40) &&
                 (!apart || (rows->v_stride >= (int64_t)cache->heads * cache->value_width && rows->v_stride < (1ll << 40))),
             "%s: token strides below the tokens' values", who);
  MX_REQUIRE(aligned(rows->k, size) && aligned(rows->v, size) && aligned(rows->weight, 4) && aligned(rows->slots, 8),
             "%s: pointers must be aligned to their elements", who);
  MX_REQUIRE(aligned(rows->k_rounded, 16) && aligned(rows->v_rounded, 16), "%s: rounded rows must be 16-byte aligned", who);
  AppendArgs a{};
  a.cache = *cache, a.rows = *rows;
  if (rotation) {
    if (int s = check_rotation(who, rotation)) return s;
    MX_REQUIRE(rotation->width == cache->width, "%s: a rotation of %d values for keys of %d", who, rotation->width, cache->width);
    a.rot = *rotation;
  }
  a.wide = aligned(rows->k, 16) && aligned(rows->v, 16) && rows->k_stride * size % 16 == 0 && rows->v_stride * size % 16 == 0;
  if (int s = use(ctx)) return s;
  if (!rows->tokens) return MX_OK;
  return by_lanes(cache->width, [&](auto l, auto n) {
    constexpr int L = decltype(l)::value, NI = decltype(n)::value;
    const auto kernel = rows->type == MX_ROWS_F32 ? append_kernel<L, NI, true> : append_kernel<L, NI, false>;
    // As many tokens a launch as leave it below 2^32 threads, nearly always all. (With the rows in turns of its workgroups 4096
    // latents took 8.4 us in place of 6.6.)
    const int64_t token_rows = (int64_t)cache->heads * (apart ? 2 : 1), most = (1ll << 31) / (L * token_rows);
    for (int64_t t = 0; t < rows->tokens; t += most) {
      mx_kv4_rows& r = a.rows;
      r.tokens = (int32_t)std::min<int64_t>(rows->tokens - t, most), a.total = r.tokens * token_rows;
      r.k = (const uint8_t*)rows->k + t * rows->k_stride * size, r.slots = rows->slots + t;
      if (r.v) r.v = (const uint8_t*)rows->v + t * rows->v_stride * size;
      if (r.k_rounded) r.k_rounded = rows->k_rounded + t * cache->heads * cache->width;
      if (r.v_rounded) r.v_rounded = rows->v_rounded + t * cache->heads * cache->value_width;
      if (a.rot.positions) a.rot.positions = rotation->positions + t;
      hipLaunchKernelGGL(kernel, dim3((unsigned)((a.total + 256 / L - 1) / (256 / L))), dim3(256), 0, as_stream(stream), a);
      MX_LAUNCH_CHECK("append_kernel");
    }
    return MX_OK;
  });
}

}  // extern "C"
