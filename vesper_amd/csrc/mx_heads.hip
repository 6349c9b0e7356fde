// Heads normalized and rotated in one pass, and the gradients of that.
//
// y = R(p) n,  n = w x r on the first `norm` values,  r = 1 / sqrt(mean(x^2) + eps).  With g = R(p)^T dy and u = x r:
//   dx = r (w g - u mean(w g u)) on those values and g on the others,   dw = sum over tokens and heads of g u.
//
// Memory traffic alone: a row is read once into registers, eight values a lane, by as many lanes as it has eights.
// Measured for 4096 tokens of 32 + 8 heads of 128 in BF16, all of each turned: forward 20.2 us for 86 MB (4.3 TB/s; 27.3 with
// a row at a time, whose loads waited for the token's position), backward 29.2 us for 128 MB (4.4 TB/s) and 4.5 for the
// workgroups' parts of dweight (46 and 9.4 with 512 workgroups for either set).
#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "mx_heads.h"

namespace {

using namespace mxh;

constexpr int kMaxTokens = 1 << 20, kMaxWidth = 4096;
constexpr int kGradBlocks = 1280;   // workgroups that add up dweight, of both sets together (and one more of each)

// A piece is K heads of one token and set on a group of L lanes: its rows are asked for at once, its angles and weights once.
struct Pieces {
  int of[2];   // of a token, by set
  __host__ __device__ int per_token() const { return of[0] + of[1]; }
};

struct HeadsArgs {
  mx_heads set[2];
  Pieces n;
  int tokens;
  mx_rotation rot;
  int y_type;
  bool wide;
  int from, to;   // the columns that the call touches
};

template <int L, int NI, int K, bool F32>
__global__ __launch_bounds__(256) void rotate_kernel(HeadsArgs a) {
  const int g = threadIdx.x % L;
  const uint32_t each = a.n.per_token(), pieces = (uint32_t)a.tokens * each;
  for (uint32_t first = blockIdx.x * (256 / L); first < pieces; first += gridDim.x * (256 / L)) {
    const uint32_t mine = first + threadIdx.x / L, p = min(mine, pieces - 1), t = p / each;
    const int j = p - t * each;
    const bool second = j >= a.n.of[0];
    const mx_heads& s = a.set[second];
    const int h = (second ? j - a.n.of[0] : j) * K;
    const int64_t xe = F32 ? 4 : 2, ye = a.y_type == MX_ROWS_F32 ? 4 : 2;
    const uint8_t* x = (const uint8_t*)s.x + (t * s.x_stride + (int64_t)h * a.rot.width) * xe;
    uint8_t* y = (uint8_t*)s.y + (t * s.y_stride + (int64_t)h * a.rot.width) * ye;
    const int heads = s.heads - h;   // of the piece, if below K
    Raw8<F32> raw[K][NI];
#pragma unroll
    for (int k = 0; k < K; ++k) load_row<L, NI>(x + (int64_t)min(k, heads - 1) * a.rot.width * xe, a.wide, a.from, a.to, g, raw[k]);
    Columns<NI> cols;
    const float* angles = nullptr;
    const bool live = place_of(a.rot, t, angles) && mine < pieces;
    weights_of<L>(a.rot, s.weight, a.from, g, cols);
    angles_of<L>(a.rot, angles, a.from, a.to, g, cols);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float v[NI][8];
      finish_row<L, NI>(x + (int64_t)min(k, heads - 1) * a.rot.width * xe, a.wide, a.rot, cols, a.from, g, raw[k], v);
      if (!live || k >= heads) continue;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int c = a.from + 8 * (i * L + g);
        if (c < a.to) store8(y + (int64_t)k * a.rot.width * ye, a.y_type, a.wide, c, v[i]);
      }
    }
  }
}

struct GradArgs {
  mx_heads_grad set[2];
  int tokens;
  mx_rotation rot;
  bool wide;
  int blocks[2];   // workgroups of each set
  float* parts;    // [blocks[0] + blocks[1]][norm]
};

// A row at a time here: two or four a lane (37 and 38 us for both kernels in place of 36) or one asked for ahead (41 to 52)
// take registers that more waves use better. The first blocks[0] workgroups have the first set. A lane keeps its columns' sums for dweight over its rows; the
// workgroup's go to parts.
template <int L, int NI, bool F32>
__global__ __launch_bounds__(256) void rotate_backward_kernel(GradArgs a) {
  extern __shared__ float sums[];   // [256 / L][8 L NI] where dweight is asked for
  const bool second = (int)blockIdx.x >= a.blocks[0];
  const mx_heads_grad& s = a.set[second];
  const int g = threadIdx.x % L, norm = a.rot.norm, width = a.rot.width;
  constexpr int64_t size = F32 ? 4 : 2;
  constexpr int type = F32 ? MX_ROWS_F32 : MX_ROWS_BF16;
  const float sign = a.rot.inverse ? 1.f : -1.f;   // R^T turns back
  Columns<NI> cols;
  weights_of<L>(a.rot, s.weight, 0, g, cols);
  float dw[NI][8] = {};
  const uint32_t each = s.heads, rows = (uint32_t)a.tokens * each, step = a.blocks[second] * (256 / L);
  const uint32_t begin = (blockIdx.x - (second ? a.blocks[0] : 0)) * (256 / L);
  for (uint32_t first = begin; first < rows; first += step) {
    const uint32_t mine = first + threadIdx.x / L, p = min(mine, rows - 1), t = p / each;
    const int64_t head = (int64_t)(p - t * each) * width;
    const uint8_t* dy = (const uint8_t*)s.dy + (t * s.dy_stride + head) * size;
    uint8_t* dx = (uint8_t*)s.dx + (t * s.dx_stride + head) * size;
    Raw8<F32> raw_d[NI], raw_x[NI];
    load_row<L, NI>(dy, a.wide, 0, width, g, raw_d);
    load_row<L, NI>((const uint8_t*)s.x + (t * s.x_stride + head) * size, a.wide, 0, norm, g, raw_x);
    const float* angles = nullptr;
    const bool there = mine < rows, counts = place_of(a.rot, t, angles) && there;
    angles_of<L>(a.rot, angles, 0, width, g, cols);
    float d[NI][8], u[NI][8];
    double sum = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      values(raw_d[i], d[i]), values(raw_x[i], u[i]);
      if (__all(counts)) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) d[i][j] = counts ? d[i][j] : 0.f, u[i][j] = counts ? u[i][j] : 0.f;   // (they may hold NaN)
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      turn8(a.rot, cols.a[i], sign, d[i], [&](float (&q)[8]) {
        if constexpr (NI == 1) {
          partner_lane<L>(a.rot, cols.a[0], g, d[0], q);
        } else if (cols.a[i].on) {   // (from memory once more)
          values(load_raw<F32>(dy, a.wide, 8 * (i * L + g) + (cols.a[i].low ? a.rot.dims / 2 : -(a.rot.dims / 2))), q);
#pragma unroll
          for (int j = 0; j < 8; ++j) q[j] = counts ? q[j] : 0.f;
        }
      });
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fma((double)u[i][j], (double)u[i][j], sum);
    }
    if (norm) {
      const float whole = root(group_sum<L>(sum), norm, a.rot.eps), r = counts ? whole : 0.f;   // (infinite where eps is zero)
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        if (!cols.normed[i]) continue;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          u[i][j] *= r;
          dw[i][j] += d[i][j] * u[i][j];
          d[i][j] *= cols.w[i][j];
          dot += d[i][j] * u[i][j];
        }
      }
      const float mean = group_sum<L>(dot) / norm;
#pragma unroll
      for (int i = 0; i < NI; ++i)
        if (cols.normed[i])
#pragma unroll
          for (int j = 0; j < 8; ++j) d[i][j] = r * (d[i][j] - u[i][j] * mean);
    }
    if (!__all(counts)) {   // zero whatever the weights are
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) d[i][j] = counts ? d[i][j] : 0.f;
    }
    if (!there) continue;
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (8 * (i * L + g) < width) store8(dx, type, a.wide, 8 * (i * L + g), d[i]);
  }
  if (!s.dweight) return;
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[threadIdx.x / L * (8 * L * NI) + 8 * (i * L + g) + j] = dw[i][j];
  __syncthreads();
  float* part = a.parts + (int64_t)blockIdx.x * norm;
  for (int c = threadIdx.x; c < norm; c += 256) {
    float v = 0.f;
#pragma unroll 4
    for (int k = 0; k < 256 / L; ++k) v += sums[k * (8 * L * NI) + c];
    part[c] = v;
  }
}

// dweight from the workgroups' parts, 32 columns a workgroup: 128 rows of eight lanes, eight parts in flight each.
__global__ __launch_bounds__(1024) void dweight_kernel(GradArgs a) {
  __shared__ float4 sums[16][8];
  const int set = blockIdx.y, norm = a.rot.norm;
  float* out = a.set[set].dweight;
  if (!out) return;
  const int lane = threadIdx.x & 7, c = blockIdx.x * 32 + 4 * lane, blocks = a.blocks[set];
  const float* part = a.parts + (int64_t)(set ? a.blocks[0] : 0) * norm + min(c, norm - 4);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int b0 = threadIdx.x / 8; b0 < blocks; b0 += 1024) {
    float4 p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = *(const float4*)(part + (int64_t)min(b0 + 128 * i, blocks - 1) * norm);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (b0 + 128 * i < blocks) v.x += p[i].x, v.y += p[i].y, v.z += p[i].z, v.w += p[i].w;
  }
#pragma unroll
  for (int m = 8; m < 64; m <<= 1)
    v.x += __shfl_xor(v.x, m, 64), v.y += __shfl_xor(v.y, m, 64), v.z += __shfl_xor(v.z, m, 64), v.w += __shfl_xor(v.w, m, 64);
  if ((threadIdx.x & 63) < 8) sums[threadIdx.x / 64][lane] = v;
  __syncthreads();
  if (threadIdx.x >= 8 || c >= norm) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) v.x += sums[i][lane].x, v.y += sums[i][lane].y, v.z += sums[i][lane].z, v.w += sums[i][lane].w;
  out[c] = v.x, out[c + 1] = v.y, out[c + 2] = v.z, out[c + 3] = v.w;
}

// fn(K, F32) for a call's rows: four heads a piece where that still leaves every SIMD four waves.
template <int L, int NI, typename F>
int by_piece(int64_t rows, bool f32, F fn) {
  using std::integral_constant;
  using std::bool_constant;
  if constexpr (NI == 1) {
    if (rows * L / 64 >= 4 * 16 * 256) return f32 ? fn(integral_constant<int, 4>(), bool_constant<true>()) : fn(integral_constant<int, 4>(), bool_constant<false>());
  }
  return f32 ? fn(integral_constant<int, 1>(), bool_constant<true>()) : fn(integral_constant<int, 1>(), bool_constant<false>());
}

int check_type(const char* who, int32_t type) {
  MX_REQUIRE(type == MX_ROWS_BF16 || type == MX_ROWS_F32, "%s: row type %d", who, type);
  return MX_OK;
}

int check_sets(const char* who, int32_t n_sets, int32_t tokens, const mx_rotation* rot, int64_t heads) {
  MX_REQUIRE(tokens >= 0 && tokens <= kMaxTokens, "%s: token count %d outside [0, %d]", who, tokens, kMaxTokens);
  MX_REQUIRE((int64_t)tokens * heads < (1ll << 31), "%s: 2^31 heads or more in all", who);
  return mxh::check_rotation(who, rot);
}

int check_set(const char* who, int32_t heads, int64_t stride, int width) {
  MX_REQUIRE(heads >= 1 && heads <= (1 << 16), "%s: %d heads outside [1, 65536]", who, heads);
  MX_REQUIRE(stride >= (int64_t)heads * width && stride < (1ll << 40), "%s: token stride %lld below %lld values", who, (long long)stride,
             (long long)heads * width);
  return MX_OK;
}

}  // namespace

int mxh::check_rotation(const char* who, const mx_rotation* r) {
  MX_REQUIRE(r, "%s: null rotation", who);
  MX_REQUIRE(r->width >= 8 && r->width % 8 == 0 && r->width <= kMaxWidth, "%s: head width %d not a multiple of 8 in [8, %d]", who,
             r->width, kMaxWidth);
  MX_REQUIRE(r->norm >= 0 && r->norm % 8 == 0 && r->norm <= r->width, "%s: norm of %d values of %d", who, r->norm, r->width);
  MX_REQUIRE(r->style == MX_ROTATE_PAIRS || r->style == MX_ROTATE_HALVES, "%s: rotation style %d", who, r->style);
  const int unit = r->style == MX_ROTATE_HALVES ? 16 : 8;
  MX_REQUIRE(r->dims >= 0 && r->dims % unit == 0 && r->first >= 0 && r->first % 8 == 0 && r->dims <= r->width - r->first,
             "%s: rotated values [%d, +%d) of %d", who, r->first, r->dims, r->width);
  MX_REQUIRE(!r->norm || (r->eps >= 0.f && r->eps <= 3.4e38f), "%s: eps must be finite and not negative", who);
  MX_REQUIRE(r->inverse == 0 || r->inverse == 1, "%s: inverse is 0 or 1", who);
  if (r->dims) {
    MX_REQUIRE(r->table && r->positions && r->table_positions >= 1, "%s: a rotation needs its table and positions", who);
    MX_REQUIRE(aligned(r->table, 16) && aligned(r->positions, 4), "%s: table must be 16-byte, positions 4-byte aligned", who);
  }
  return MX_OK;
}

using mxi::as_stream;
using mxi::use;

extern "C" {

int mx_rotate_heads(mx_ctx* ctx, const mx_heads* sets, int32_t n_sets, int32_t tokens, const mx_rotation* rotation,
                    int32_t x_type, int32_t y_type, void* stream) {
  const char* who = "mx_rotate_heads";
  MX_REQUIRE(sets && (n_sets == 1 || n_sets == 2), "%s: one or two sets of heads", who);
  int64_t heads = 0;
  for (int i = 0; i < n_sets; ++i) heads += std::max(sets[i].heads, 0);
  if (int s = check_sets(who, n_sets, tokens, rotation, heads)) return s;
  if (int s = check_type(who, x_type)) return s;
  if (int s = check_type(who, y_type)) return s;
  HeadsArgs a{};
  a.tokens = tokens, a.rot = *rotation, a.y_type = y_type;
  a.to = rotation->width;
  const int64_t xe = x_type == MX_ROWS_F32 ? 4 : 2, ye = y_type == MX_ROWS_F32 ? 4 : 2;
  bool wide = true, in_place = true;
  for (int i = 0; i < n_sets; ++i) {
    const mx_heads& s = sets[i];
    if (int e = check_set(who, s.heads, s.x_stride, rotation->width)) return e;
    if (int e = check_set(who, s.heads, s.y_stride, rotation->width)) return e;
    MX_REQUIRE(s.x && s.y, "%s: null pointer", who);
    MX_REQUIRE(aligned(s.x, xe) && aligned(s.y, ye) && aligned(s.weight, 4), "%s: pointers must be aligned to their elements", who);
    MX_REQUIRE(s.x != s.y || (x_type == y_type && s.x_stride == s.y_stride), "%s: y may be x only with its type and stride", who);
    wide &= aligned(s.x, 16) && aligned(s.y, 16) && s.x_stride * xe % 16 == 0 && s.y_stride * ye % 16 == 0;
    in_place &= s.x == s.y;
    a.set[i] = s;
  }
  if (n_sets == 1) a.set[1] = a.set[0];
  a.wide = wide;
  if (in_place && !rotation->norm) a.from = rotation->first, a.to = rotation->first + rotation->dims;   // nothing else changes
  if (int s = use(ctx)) return s;
  if (!tokens || a.to == a.from) return MX_OK;
  return mxh::by_lanes(a.to - a.from, [&](auto l, auto n) {
    constexpr int L = decltype(l)::value, NI = decltype(n)::value;
    return by_piece<L, NI>(tokens * heads, x_type == MX_ROWS_F32, [&](auto k, auto f32) {
      constexpr int K = decltype(k)::value;
      for (int i = 0; i < n_sets; ++i) a.n.of[i] = (sets[i].heads + K - 1) / K;
      const int64_t pieces = (int64_t)tokens * a.n.per_token();
      const unsigned grid = (unsigned)std::min<int64_t>((pieces + 256 / L - 1) / (256 / L), 1 << 16);
      hipLaunchKernelGGL((rotate_kernel<L, NI, K, decltype(f32)::value>), dim3(grid), dim3(256), 0, as_stream(stream), a);
      MX_LAUNCH_CHECK("rotate_kernel");
      return MX_OK;
    });
  });
}

uint64_t mx_rotate_heads_workspace_bytes(int32_t norm) {
  if (norm < 0 || norm > kMaxWidth) return 0;
  return (uint64_t)(kGradBlocks + 2) * norm * sizeof(float);
}

int mx_rotate_heads_backward(mx_ctx* ctx, const mx_heads_grad* sets, int32_t n_sets, int32_t tokens, const mx_rotation* rotation,
                             int32_t type, void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* who = "mx_rotate_heads_backward";
  MX_REQUIRE(sets && (n_sets == 1 || n_sets == 2), "%s: one or two sets of heads", who);
  int64_t heads = 0;
  for (int i = 0; i < n_sets; ++i) heads += std::max(sets[i].heads, 0);
  if (int s = check_sets(who, n_sets, tokens, rotation, heads)) return s;
  if (int s = check_type(who, type)) return s;
  const int64_t size = type == MX_ROWS_F32 ? 4 : 2;
  GradArgs a{};
  a.tokens = tokens, a.rot = *rotation, a.parts = (float*)workspace;
  bool wide = true, weights = false;
  for (int i = 0; i < n_sets; ++i) {
    const mx_heads_grad& s = sets[i];
    if (int e = check_set(who, s.heads, s.dy_stride, rotation->width)) return e;
    if (int e = check_set(who, s.heads, s.dx_stride, rotation->width)) return e;
    if (rotation->norm)
      if (int e = check_set(who, s.heads, s.x_stride, rotation->width)) return e;
    MX_REQUIRE(s.dy && s.dx && (s.x || !rotation->norm), "%s: null pointer", who);
    MX_REQUIRE(aligned(s.x, size) && aligned(s.dy, size) && aligned(s.dx, size) && aligned(s.weight, 4) && aligned(s.dweight, 4),
               "%s: pointers must be aligned to their elements", who);
    MX_REQUIRE(s.dx != s.dy || s.dx_stride == s.dy_stride, "%s: dx may be dy only with its stride", who);
    MX_REQUIRE(s.dx != s.x || s.dx_stride == s.x_stride, "%s: dx may be x only with its stride", who);
    MX_REQUIRE(!s.dweight || rotation->norm, "%s: no norm has no weights", who);
    wide &= aligned(s.dy, 16) && aligned(s.dx, 16) && s.dy_stride * size % 16 == 0 && s.dx_stride * size % 16 == 0;
    if (rotation->norm) wide &= aligned(s.x, 16) && s.x_stride * size % 16 == 0;
    weights |= s.dweight != nullptr;
    a.set[i] = s;
  }
  a.wide = wide;
  if (n_sets == 2 && sets[0].dweight && sets[1].dweight) {
    const intptr_t apart = (const uint8_t*)sets[1].dweight - (const uint8_t*)sets[0].dweight;
    MX_REQUIRE(std::abs(apart) >= rotation->norm * (intptr_t)sizeof(float), "%s: the sets' dweight share memory", who);
  }
  if (weights)
    MX_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= mx_rotate_heads_workspace_bytes(rotation->norm),
               "%s: the gradient of weights needs %llu bytes of workspace, 16-byte aligned", who,
               (unsigned long long)mx_rotate_heads_workspace_bytes(rotation->norm));
  if (int s = use(ctx)) return s;
  if (!tokens && !weights) return MX_OK;
  return mxh::by_lanes(rotation->width, [&](auto l, auto n) {
    constexpr int L = decltype(l)::value, NI = decltype(n)::value;
    int64_t steps[2] = {0, 0};
    for (int i = 0; i < n_sets; ++i) steps[i] = ((int64_t)tokens * sets[i].heads + 256 / L - 1) / (256 / L);
    // as many turns for every workgroup, whichever its set
    const int64_t most = weights ? kGradBlocks : 1 << 16, turns = std::max<int64_t>((steps[0] + steps[1] + most - 1) / most, 1);
    for (int i = 0; i < n_sets; ++i) a.blocks[i] = (int)std::max<int64_t>((steps[i] + turns - 1) / turns, 1);
    const auto kernel = type == MX_ROWS_F32 ? rotate_backward_kernel<L, NI, true> : rotate_backward_kernel<L, NI, false>;
    hipLaunchKernelGGL(kernel, dim3(a.blocks[0] + a.blocks[1]), dim3(256), weights ? 256 * NI * 8 * sizeof(float) : 0, as_stream(stream), a);
    MX_LAUNCH_CHECK("rotate_backward_kernel");
    if (weights) {
      hipLaunchKernelGGL(dweight_kernel, dim3((rotation->norm + 31) / 32, n_sets), dim3(1024), 0, as_stream(stream), a);
      MX_LAUNCH_CHECK("dweight_kernel");
    }
    return MX_OK;
  });
}

}  // extern "C"
