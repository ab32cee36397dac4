// What the kernels and entry points of the paged key-value cache share.
#pragma once

#include "common.hpp"

namespace cv3 {

// A value that the whole wave holds alike, moved to the scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)(uint32_t)uniform((int)v) | (int64_t)uniform((int)(v >> 32)) << 32;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// 2^(x - top), 0 where x is -inf whatever top is
__device__ __forceinline__ float weight_of(float x, float top) { return x == -INFINITY ? 0.f : exp2_fast(x - top); }

// A maximum for keys that are there and score -inf every one, with a sum of 0: their softmax is 0 / 0 = NaN, unless
// another part has a score that is a number, beside which it weighs nothing.  -inf says that no key is there.
constexpr float kNoScore = -3.402823466e38f;

// Workgroups of a launch, which has fewer than 2^32 threads: one less where they have 512.
constexpr int64_t kLaunchBlocks = 1 << 23;

inline int elem_size(int type) { return type == CV3_F32 ? 4 : 2; }

// What every call on a cache checks.
inline int check_cache(int type, const void* k, const void* v, int64_t pages, int64_t page, int kv_heads, int d) {
  CV3_REQUIRE(type == CV3_F32 || type == CV3_F16 || type == CV3_BF16, CV3_EINVAL, "unknown cache type %d", type);
  CV3_REQUIRE(page >= 1 && page <= 65536, CV3_EINVAL, "a page holds 1 to 65536 keys, not %lld", (long long)page);
  CV3_REQUIRE(pages >= 1 && pages <= INT32_MAX, CV3_EINVAL, "a cache has 1 to 2^31 - 1 pages, not %lld",
              (long long)pages);
  CV3_REQUIRE(kv_heads >= 1 && kv_heads <= 1024, CV3_EINVAL, "1 to 1024 kv heads, not %d", kv_heads);
  CV3_REQUIRE(d >= 8 && d <= 256 && d % 8 == 0, CV3_EINVAL, "the head dim must be a multiple of 8, 8 to 256, not %d", d);
  CV3_REQUIRE(k && v, CV3_EINVAL, "null cache");
  CV3_REQUIRE(((uintptr_t)k | (uintptr_t)v) % 16 == 0, CV3_EINVAL, "the caches must be 16-byte aligned");
  return CV3_OK;
}

}  // namespace cv3
