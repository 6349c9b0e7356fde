// A head's row on a group of L lanes: eight values a lane and step, loaded, normalized and rotated (mx_heads.hip; on the
// way into the cache, mx_kv4.hip).
#pragma once
#include "mx_device.h"
#include "mx_internal.h"

namespace mxh {

// Eight values of a row as they lie in memory.
template <bool F32>
struct Raw8 {
  uint4 w[F32 ? 2 : 1];
};

// From column c on. wide: 16-byte loads.
template <bool F32>
__device__ __forceinline__ Raw8<F32> load_raw(const void* row, bool wide, int c) {
  Raw8<F32> r;
  const uint8_t* p = (const uint8_t*)row + (int64_t)c * (F32 ? 4 : 2);
#pragma unroll
  for (int i = 0; i < (F32 ? 2 : 1); ++i) {
    if (wide) {
      r.w[i] = mxd::ldg128(p + 16 * i);
    } else if (F32) {
      const uint32_t* q = (const uint32_t*)p + 4 * i;
      r.w[i] = make_uint4(q[0], q[1], q[2], q[3]);
    } else {
      const uint16_t* q = (const uint16_t*)p;
      r.w[i] = make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16, q[6] | (uint32_t)q[7] << 16);
    }
  }
  return r;
}

template <bool F32>
__device__ __forceinline__ void values(const Raw8<F32>& r, float (&v)[8]) {
  if constexpr (F32) {
    v[0] = mx::u2f(r.w[0].x), v[1] = mx::u2f(r.w[0].y), v[2] = mx::u2f(r.w[0].z), v[3] = mx::u2f(r.w[0].w);
    v[4] = mx::u2f(r.w[1].x), v[5] = mx::u2f(r.w[1].y), v[6] = mx::u2f(r.w[1].z), v[7] = mx::u2f(r.w[1].w);
  } else {
    const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[2 * j] = mx::u2f(w[j] << 16), v[2 * j + 1] = mx::u2f(w[j] & 0xFFFF0000u);
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

// Whether column c is normalized, with its weights (ones where there are none).
__device__ __forceinline__ bool weights8(const float* weight, int norm, int c, float (&w)[8]) {
  typedef float __attribute__((ext_vector_type(4), aligned(4))) four;
  const bool on = c < norm;
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = 1.f;
  if (on && weight) {
    const four a = *(const four*)(weight + c), b = *(const four*)(weight + c + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = a[j], w[4 + j] = b[j];
  }
  return on;
}

// What lane i ^ m of each 16 holds, or for m of 4 and 8 a lane of the other half of 8 or 16: the same to a butterfly.
template <int m>
__device__ __forceinline__ int across(int v) {
  constexpr int how = m == 1 ? 0xB1 : m == 2 ? 0x4E : m == 4 ? 0x141 : 0x140;   // quads' lanes, mirrored halves, mirrored rows
  return __builtin_amdgcn_mov_dpp(v, how, 0xF, 0xF, false);
}
template <int m>
__device__ __forceinline__ float across(float v) {
  if constexpr (m > 8) return __shfl_xor(v, m, 64);
  return __int_as_float(across<m>(__float_as_int(v)));
}
template <int m>
__device__ __forceinline__ double across(double v) {
  if constexpr (m > 8) return __shfl_xor(v, m, 64);
  return __hiloint2double(across<m>(__double2hiint(v)), across<m>(__double2loint(v)));
}

// Sum over the L lanes of a group, in every lane of it. Every lane of the wave comes here.
template <int L, int m = 1, typename T>
__device__ __forceinline__ T group_sum(T v) {
  v += across<m>(v);
  if constexpr (2 * m < L) return group_sum<L, 2 * m>(v);
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

// The cosines and sines of columns [c, c + 8) of a row, where they are turned; pairs have four of each.
struct Angles8 {
  float c[8], s[8];
  bool on, low;   // of halves, c is in the first
};
__device__ __forceinline__ Angles8 angles8(const mx_rotation& rot, const float* angles, int c) {
  Angles8 a;
  const int j = c - rot.first, half = rot.dims / 2;
  a.on = angles && j >= 0 && j < rot.dims, a.low = j < half;
#pragma unroll
  for (int i = 0; i < 8; ++i) a.c[i] = 1.f, a.s[i] = 0.f;
  if (!a.on) return a;
  const float* p = angles + (rot.style == MX_ROTATE_PAIRS ? j / 2 : a.low ? j : j - half);
  const float4 c0 = *(const float4*)p, s0 = *(const float4*)(p + half);
  a.c[0] = c0.x, a.c[1] = c0.y, a.c[2] = c0.z, a.c[3] = c0.w, a.s[0] = s0.x, a.s[1] = s0.y, a.s[2] = s0.z, a.s[3] = s0.w;
  if (rot.style == MX_ROTATE_HALVES) {
    const float4 c1 = *(const float4*)(p + 4), s1 = *(const float4*)(p + half + 4);
    a.c[4] = c1.x, a.c[5] = c1.y, a.c[6] = c1.z, a.c[7] = c1.w, a.s[4] = s1.x, a.s[5] = s1.y, a.s[6] = s1.z, a.s[7] = s1.w;
  }
  return a;
}

// Eight values turned by their angles (sign 1, or -1 for the inverse): (a, b) -> (a c - b s, b c + a s). partner(p): the
// eight values half the range away, asked of every lane where halves are turned.
template <typename Partner>
__device__ __forceinline__ void turn8(const mx_rotation& rot, const Angles8& a, float sign, float (&v)[8], Partner partner) {
  if (!rot.dims) return;
  if (rot.style == MX_ROTATE_PAIRS) {
    if (!a.on) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = v[2 * i], y = v[2 * i + 1], s = sign * a.s[i];
      v[2 * i] = x * a.c[i] - y * s;
      v[2 * i + 1] = y * a.c[i] + x * s;
    }
  } else {
    float p[8];
    partner(p);
    if (!a.on) return;
    const float turn = a.low ? -sign : sign;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * a.c[i] + p[i] * (turn * a.s[i]);
  }
}

// The partner of a row that its L lanes hold in one step: from the lane that has it.
template <int L>
__device__ __forceinline__ void partner_lane(const mx_rotation& rot, const Angles8& a, int g, const float (&v)[8], float (&p)[8]) {
  const int from = a.on ? g + (a.low ? rot.dims / 16 : -(rot.dims / 16)) : g;
#pragma unroll
  for (int j = 0; j < 8; ++j) p[j] = __shfl(v[j], from, L);
}

// What the lane's columns of all rows of one token need: weights and angles.
template <int NI>
struct Columns {
  float w[NI][8];
  const float* weight;
  bool normed[NI];
  Angles8 a[NI];
};
template <int L, int NI>
__device__ __forceinline__ void weights_of(const mx_rotation& rot, const float* weight, int from, int g, Columns<NI>& cols) {
  cols.weight = weight;
#pragma unroll
  for (int i = 0; i < NI; ++i) cols.normed[i] = weights8(weight, rot.norm, from + 8 * (i * L + g), cols.w[i]);
}
template <int L, int NI>
__device__ __forceinline__ void angles_of(const mx_rotation& rot, const float* angles, int from, int to, int g, Columns<NI>& cols) {
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = from + 8 * (i * L + g);
    cols.a[i] = angles8(rot, c < to ? angles : nullptr, c);
  }
}

template <int L, int NI, bool F32>
__device__ __forceinline__ void load_row(const void* row, bool wide, int from, int to, int g, Raw8<F32> (&raw)[NI]) {
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = from + 8 * (i * L + g);
    if (c < to) {
      raw[i] = load_raw<F32>(row, wide, c);
    } else {
#pragma unroll
      for (int j = 0; j < (F32 ? 2 : 1); ++j) raw[i].w[j] = make_uint4(0, 0, 0, 0);
    }
  }
}

// A row normalized and rotated into v. Every lane of the wave comes here.
template <int L, int NI, bool F32>
__device__ __forceinline__ void finish_row(const void* row, bool wide, const mx_rotation& rot, const Columns<NI>& cols, int from, int g,
                                           const Raw8<F32> (&raw)[NI], float (&v)[NI][8]) {
  double sum = 0;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    values(raw[i], v[i]);
    if (cols.normed[i])
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fma((double)v[i][j], (double)v[i][j], sum);
  }
  float r = 1.f;
  if (rot.norm) {
    r = root(group_sum<L>(sum), rot.norm, rot.eps);
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (cols.normed[i])
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * r * cols.w[i][j];
  }
  const float sign = rot.inverse ? -1.f : 1.f;
#pragma unroll
  for (int i = 0; i < NI; ++i)
    turn8(rot, cols.a[i], sign, v[i], [&](float (&p)[8]) {
      if constexpr (NI == 1) {
        partner_lane<L>(rot, cols.a[0], g, v[0], p);
      } else if (cols.a[i].on) {   // (from memory once more)
        const int c = from + 8 * (i * L + g) + (cols.a[i].low ? rot.dims / 2 : -(rot.dims / 2));
        values(load_raw<F32>(row, wide, c), p);
        float w[8];
        const float* weight = cols.weight;
        if (weights8(weight, rot.norm, c, w))
#pragma unroll
          for (int j = 0; j < 8; ++j) p[j] = p[j] * r * w[j];
      }
    });
}

// Host: the checks of a rotation that both files make.
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
