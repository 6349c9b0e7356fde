// Heads normalized and rotated in one pass, and the gradients of that.
//
// y = R(p) n,  n = w x r on the first `norm` values,  r = 1 / sqrt(mean(x^2) + eps).  With g = R(p)^T dy and u = x r:
//   dx = r (w g - u mean(w g u)) on those values and g on the others,   dw = sum over tokens and heads of g u.
//
// Memory traffic alone: a row is read once into registers, eight values a lane, by as many lanes as it has eights.
#include <algorithm>
#include <type_traits>

#include "mx_heads.h"

namespace {

using namespace mxh;

constexpr int kMaxTokens = 1 << 20, kMaxWidth = 4096;
constexpr int kGradBlocks = 512;   // workgroups of one set of heads that add up dweight

struct HeadsArgs {
  mx_heads set[2];
  int heads;           // of both sets
  int64_t rows;        // tokens * heads
  mx_rotation rot;
  int x_type, y_type;
  bool wide;
  int from, to;        // the columns that the call touches
};

template <int L, int NI>
__global__ __launch_bounds__(256) void rotate_kernel(HeadsArgs a) {
  const int g = threadIdx.x % L;
  const int64_t step = (int64_t)gridDim.x * (256 / L);
  for (int64_t r = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L; r < a.rows; r += step) {
    const uint32_t t = (uint32_t)r / (uint32_t)a.heads;
    int h = (uint32_t)r - t * (uint32_t)a.heads;
    const float* angles = nullptr;
    if (!place_of(a.rot, t, angles)) continue;
    const int second = h >= a.set[0].heads;
    const mx_heads& s = a.set[second];
    h -= second ? a.set[0].heads : 0;
    const int64_t xe = a.x_type == MX_ROWS_F32 ? 4 : 2, ye = a.y_type == MX_ROWS_F32 ? 4 : 2;
    const void* x = (const uint8_t*)s.x + (t * s.x_stride + (int64_t)h * a.rot.width) * xe;
    void* y = (uint8_t*)s.y + (t * s.y_stride + (int64_t)h * a.rot.width) * ye;
    float v[NI][8];
    normalized_row<L, NI>(x, a.x_type, a.wide, a.rot, angles, s.weight, a.from, a.to, g, v);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = a.from + 8 * (i * L + g);
      if (c < a.to) store8(y, a.y_type, a.wide, c, v[i]);
    }
  }
}

struct GradArgs {
  mx_heads_grad set[2];
  int tokens;
  mx_rotation rot;
  int type;
  bool wide;
  float* parts;   // [2][kGradBlocks][norm]
};

// blockIdx.y: the set. A lane keeps its columns' sums for dweight over its rows; the workgroup's go to parts.
template <int L, int NI>
__global__ __launch_bounds__(256) void rotate_backward_kernel(GradArgs a) {
  extern __shared__ float sums[];   // [256 / L][8 L NI] where dweight is asked for
  const mx_heads_grad& s = a.set[blockIdx.y];
  const int g = threadIdx.x % L, norm = a.rot.norm, width = a.rot.width;
  const int64_t size = a.type == MX_ROWS_F32 ? 4 : 2;
  const float sign = a.rot.inverse ? 1.f : -1.f;   // R^T turns back
  float dw[NI][8] = {};
  const int64_t rows = (int64_t)a.tokens * s.heads, step = (int64_t)gridDim.x * (256 / L);
  for (int64_t r = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L; r < rows; r += step) {
    const uint32_t t = (uint32_t)r / (uint32_t)s.heads;
    const int64_t head = (int64_t)((uint32_t)r - t * (uint32_t)s.heads) * width;
    const uint8_t* dy = (const uint8_t*)s.dy + (t * s.dy_stride + head) * size;
    const uint8_t* x = (const uint8_t*)s.x + (t * s.x_stride + head) * size;
    uint8_t* dx = (uint8_t*)s.dx + (t * s.dx_stride + head) * size;
    const float* angles = nullptr;
    const bool live = place_of(a.rot, t, angles);
    float d[NI][8], u[NI][8];
    double sum = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = 8 * (i * L + g);
#pragma unroll
      for (int j = 0; j < 8; ++j) d[i][j] = u[i][j] = 0.f;
      if (c >= width || !live) continue;
      load8(dy, a.type, a.wide, c, d[i]);
      if (c < norm) load8(x, a.type, a.wide, c, u[i]);
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = 8 * (i * L + g);
      if (c < width && live) turn8(a.rot, angles, sign, c, d[i], [&](int at, float (&p)[8]) { load8(dy, a.type, a.wide, at, p); });
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fma((double)u[i][j], (double)u[i][j], sum);
    }
    if (norm) {
      const float r = root(group_sum<L>(sum), norm, a.rot.eps);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int c = 8 * (i * L + g);
        if (c >= norm) continue;
        float w[8];
        weights8(s.weight, c, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          u[i][j] *= r;
          dw[i][j] += d[i][j] * u[i][j];
          d[i][j] *= w[j];
          dot += d[i][j] * u[i][j];
        }
      }
      const float mean = group_sum<L>(dot) / norm;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        if (8 * (i * L + g) >= norm) continue;
#pragma unroll
        for (int j = 0; j < 8; ++j) d[i][j] = r * (d[i][j] - u[i][j] * mean);
      }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (8 * (i * L + g) < width) store8(dx, a.type, a.wide, 8 * (i * L + g), d[i]);
  }
  if (!s.dweight) return;
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[threadIdx.x / L * (8 * L * NI) + 8 * (i * L + g) + j] = dw[i][j];
  __syncthreads();
  float* part = a.parts + ((int64_t)blockIdx.y * kGradBlocks + blockIdx.x) * norm;
  for (int c = threadIdx.x; c < norm; c += 256) {
    float v = 0.f;
#pragma unroll 4
    for (int k = 0; k < 256 / L; ++k) v += sums[k * (8 * L * NI) + c];
    part[c] = v;
  }
}

// dweight from the workgroups' parts: 16 rows of 64 columns add up every 16th part.
__global__ __launch_bounds__(1024) void dweight_kernel(GradArgs a, int blocks) {
  __shared__ float sums[16][64];
  float* out = a.set[blockIdx.y].dweight;
  if (!out) return;
  const int c = blockIdx.x * 64 + threadIdx.x % 64, k = threadIdx.x / 64;
  const float* part = a.parts + (int64_t)blockIdx.y * kGradBlocks * a.rot.norm;
  float v = 0.f;
  if (c < a.rot.norm)
    for (int b = k; b < blocks; b += 16) v += part[(int64_t)b * a.rot.norm + c];
  sums[k][threadIdx.x % 64] = v;
  __syncthreads();
  if (k == 0 && c < a.rot.norm) {
#pragma unroll
    for (int i = 1; i < 16; ++i) v += sums[i][threadIdx.x];
    out[c] = v;
  }
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
  a.heads = (int)heads, a.rows = tokens * heads, a.rot = *rotation, a.x_type = x_type, a.y_type = y_type;
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
    const unsigned grid = (unsigned)std::min<int64_t>((a.rows + 256 / L - 1) / (256 / L), 1 << 14);
    hipLaunchKernelGGL((rotate_kernel<L, NI>), dim3(grid), dim3(256), 0, as_stream(stream), a);
    MX_LAUNCH_CHECK("rotate_kernel");
    return MX_OK;
  });
}

uint64_t mx_rotate_heads_workspace_bytes(int32_t norm) {
  if (norm < 0 || norm > kMaxWidth) return 0;
  return 2ull * kGradBlocks * norm * sizeof(float);
}

int mx_rotate_heads_backward(mx_ctx* ctx, const mx_heads_grad* sets, int32_t n_sets, int32_t tokens, const mx_rotation* rotation,
                             int32_t type, void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* who = "mx_rotate_heads_backward";
  MX_REQUIRE(sets && (n_sets == 1 || n_sets == 2), "%s: one or two sets of heads", who);
  int64_t heads = 0, most = 1;
  for (int i = 0; i < n_sets; ++i) heads += std::max(sets[i].heads, 0), most = std::max<int64_t>(most, sets[i].heads);
  if (int s = check_sets(who, n_sets, tokens, rotation, heads)) return s;
  if (int s = check_type(who, type)) return s;
  const int64_t size = type == MX_ROWS_F32 ? 4 : 2;
  GradArgs a{};
  a.tokens = tokens, a.rot = *rotation, a.type = type, a.parts = (float*)workspace;
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
  if (weights)
    MX_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= mx_rotate_heads_workspace_bytes(rotation->norm),
               "%s: the gradient of weights needs %llu bytes of workspace, 16-byte aligned", who,
               (unsigned long long)mx_rotate_heads_workspace_bytes(rotation->norm));
  if (int s = use(ctx)) return s;
  if (!tokens && !weights) return MX_OK;
  return mxh::by_lanes(rotation->width, [&](auto l, auto n) {
    constexpr int L = decltype(l)::value, NI = decltype(n)::value;
    const int64_t steps = std::max<int64_t>((tokens * most + 256 / L - 1) / (256 / L), 1);
    const unsigned grid = (unsigned)(weights ? std::min<int64_t>((steps + 3) / 4, kGradBlocks) : std::min<int64_t>(steps, 1 << 14));
    hipLaunchKernelGGL((rotate_backward_kernel<L, NI>), dim3(grid, n_sets), dim3(256), weights ? 256 * NI * 8 * sizeof(float) : 0,
                       as_stream(stream), a);
    MX_LAUNCH_CHECK("rotate_backward_kernel");
    if (weights) {
      hipLaunchKernelGGL(dweight_kernel, dim3((rotation->norm + 63) / 64, n_sets), dim3(1024), 0, as_stream(stream), a, (int)grid);
      MX_LAUNCH_CHECK("dweight_kernel");
    }
    return MX_OK;
  });
}

}  // extern "C"
