// What the files of the 4-bit cache share: appending (mx_kv4.hip) and attention (mx_attend.hip).
#pragma once
#include "mx_heads.h"

namespace mxk {

constexpr int kMaxTokens = 1 << 20, kMaxBatch = 1 << 16;

// Bytes from one token's scales to the next's.
__host__ __device__ constexpr int scale_pitch(int width) { return (width + 127) / 128 * 4; }

int check_cache(const char* who, const mx_kv4* cache);

}  // namespace mxk
