// A head's row on a group of L lanes: eight values a lane and step, loaded, normalized and rotated (mx_heads.hip; on the
// way into the cache, mx_kv4.hip).
#pragma once
#include "mx_device.h"
#include "mx_internal.h"

namespace mxh {

// The eight values of a row from column c on. wide: 16-byte loads.
__device__ __forceinline__ void load8(const void* row, int type, bool wide, int c, float (&v)[8]) {
  if (type == MX_ROWS_BF16) {
    const uint16_t* p = (const uint16_t*)row + c;
    uint32_t w[4];
    if (wide) {
      const uint4 q = mxd::ldg128((const uint8_t*)p);
      w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = p[2 * j] | (uint32_t)p[2 * j + 1] << 16;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = mx::u2f(w[j] << 16);
      v[2 * j + 1] = mx::u2f(w[j] & 0xFFFF0000u);
    }
  } else {
    const float* p = (const float*)row + c;
    if (wide) {
      const uint4 a = mxd::ldg128((const uint8_t*)p), b = mxd::ldg128((const uint8_t*)(p + 4));
      v[0] = mx::u2f(a.x), v[1] = mx::u2f(a.y), v[2] = mx::u2f(a.z), v[3] = mx::u2f(a.w);
      v[4] = mx::u2f(b.x), v[5] = mx::u2f(b.y), v[6] = mx::u2f(b.z), v[7] = mx::u2f(b.w);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = p[j];
    }
  }
}

__device__ __forceinline__ void store8(void* row, int type, bool wide, int c, const float (&v)[8]) {
  if (type == MX_ROWS_BF16) {
    uint16_t* p = (uint16_t*)row + c;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = mxd::bf16_pair(v[2 * j], v[2 * j + 1]);
    if (wide) {
      *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) p[2 * j] = (uint16_t)w[j], p[2 * j + 1] = (uint16_t)(w[j] >> 16);
    }
  } else {
    float* p = (float*)row + c;
    if (wide) {
      *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
      *(float4*)(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = v[j];
    }
  }
}

__device__ __forceinline__ void weights8(const float* weight, int c, float (&w)[8]) {
  if (weight) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = mxd::ldgf(weight + c + j);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = 1.f;
  }
}

// Sum over the L lanes of a group, in every lane of it.
template <int L, typename T>
__device__ __forceinline__ T group_sum(T v) {
#pragma unroll
  for (int m = L / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// 1 / sqrt(sum / n + eps) rounded to FP32: the FP32 reciprocal root, within 2^-22 of it, and one Newton step in 64 bits,
// which squares its error. A sum whose FP32 value leaves the normal range goes through the 64-bit root.
__device__ __forceinline__ float root(double sum, int n, float eps) {
  const double m = sum / n + (double)eps;
  if (m > 1e-37 && m < 1e37) {
    const double r = (double)__builtin_amdgcn_rsqf((float)m);
    return (float)(r * (1.5 - 0.5 * m * r * r));
  }
  return (float)(1.0 / sqrt(m));
}

// Whether token t takes part: its position is in the table (or nothing is rotated).
__device__ __forceinline__ bool place_of(const mx_rotation& rot, int64_t t, const float*& angles) {
  if (!rot.dims) return true;
  const int p = rot.positions[t];
  if (p < 0 || p >= rot.table_positions) return false;
  angles = rot.table + (int64_t)p * rot.dims;
  return true;
}

// Columns [8 c, 8 c + 8) of a row turned by the token's angles (sign 1, or -1 for the inverse), where they lie in the
// rotated range. partner(c, p) gives the eight values dims / 2 away (halves).
template <typename Partner>
__device__ __forceinline__ void turn8(const mx_rotation& rot, const float* angles, float sign, int c, float (&v)[8], Partner partner) {
  const int j = c - rot.first;
  if (j < 0 || j >= rot.dims) return;
  const int half = rot.dims / 2;
  if (rot.style == MX_ROTATE_PAIRS) {
    const float4 co = *(const float4*)(angles + j / 2), si = *(const float4*)(angles + half + j / 2);
    const float cs[4] = {co.x, co.y, co.z, co.w}, sn[4] = {si.x, si.y, si.z, si.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = v[2 * i], b = v[2 * i + 1], s = sign * sn[i];
      v[2 * i] = a * cs[i] - b * s;
      v[2 * i + 1] = b * cs[i] + a * s;
    }
  } else {
    const bool low = j < half;
    const int k = low ? j : j - half;
    float p[8];
    partner(low ? c + half : c - half, p);
    const float4 c0 = *(const float4*)(angles + k), c1 = *(const float4*)(angles + k + 4);
    const float4 s0 = *(const float4*)(angles + half + k), s1 = *(const float4*)(angles + half + k + 4);
    const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    const float sn[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
    const float turn = low ? -sign : sign;   // a c - b s, b c + a s
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * cs[i] + p[i] * (turn * sn[i]);
  }
}

// A row of `width` values from column `from` on, normalized and rotated into v.
template <int L, int NI>
__device__ __forceinline__ void normalized_row(const void* row, int type, bool wide, const mx_rotation& rot, const float* angles,
                                               const float* weight, int from, int to, int g, float (&v)[NI][8]) {
  double sum = 0;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = from + 8 * (i * L + g);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    if (c < to) load8(row, type, wide, c, v[i]);
    if (c < rot.norm) {
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fma((double)v[i][j], (double)v[i][j], sum);
    }
  }
  float r = 1.f;
  if (rot.norm) {
    r = root(group_sum<L>(sum), rot.norm, rot.eps);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = from + 8 * (i * L + g);
      if (c >= rot.norm) continue;
      float w[8];
      weights8(weight, c, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * r * w[j];
    }
  }
  if (!rot.dims) return;
  const float sign = rot.inverse ? -1.f : 1.f;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = from + 8 * (i * L + g);
    if (c >= to) continue;
    turn8(rot, angles, sign, c, v[i], [&](int at, float (&p)[8]) {
      load8(row, type, wide, at, p);
      if (at < rot.norm) {
        float w[8];
        weights8(weight, at, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = p[j] * r * w[j];
      }
    });
  }
}

// Host: the checks of a rotation that both files make. x_needed: whether positions must be given.
int check_rotation(const char* who, const mx_rotation* rot);

inline bool aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// fn(std::integral_constant L, NI) for rows of n values on as few lanes as hold them.
template <typename F>
int by_lanes(int n, F fn) {
  using std::integral_constant;
  const int chunks = (n + 7) / 8;
  if (chunks <= 8) return fn(integral_constant<int, 8>(), integral_constant<int, 1>());
  if (chunks <= 16) return fn(integral_constant<int, 16>(), integral_constant<int, 1>());
  if (chunks <= 32) return fn(integral_constant<int, 32>(), integral_constant<int, 1>());
  if (chunks <= 64) return fn(integral_constant<int, 64>(), integral_constant<int, 1>());
  if (chunks <= 128) return fn(integral_constant<int, 64>(), integral_constant<int, 2>());
  return fn(integral_constant<int, 64>(), integral_constant<int, 8>());
}

}  // namespace mxh
