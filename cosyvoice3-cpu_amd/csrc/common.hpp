// Shared helpers for the cv3hip kernels: status codes, thread-local error text,
// the calling thread's stream, and wavefront (64-lane) reductions for gfx950.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <string>

#include "../../include/cv3hip.h"

namespace cv3 {

// Sets the calling thread's error message; returns `code`.
int fail(int code, const char* fmt, ...);
// The stream a call runs on: `s` if non-null, else the calling thread's own
// non-blocking stream (created on first use).
hipStream_t stream_of(cv3_stream_t s);
// True once cv3_shutdown has run: every block is freed and every stream destroyed, so
// no entry point may enqueue work any more.
bool shut_down();

// Memory for the launches that one entry point makes on st, from the caching allocator: ordered behind the block's
// earlier uses on st itself, given back behind st (scratch_free follows the last launch), owned by the graph if st
// is capturing (where the next call on st takes it again).  CV3_ENOMEM if there is none: out of memory, or nothing
// cached and the thread or st is capturing.
int scratch_alloc(void** ptr, size_t bytes, hipStream_t st);
int scratch_free(void* ptr, hipStream_t st);

// Memory that a call reads or writes.  Doubles hold the sizes: those of a mistaken call may pass 2^63 bytes.
struct Run {
  const void* p;
  double bytes;
};
inline bool overlap(const Run& a, const Run& b) {
  const double x = (double)(uintptr_t)a.p, y = (double)(uintptr_t)b.p;
  return a.p && b.p && a.bytes > 0 && b.bytes > 0 && x < y + b.bytes && y < x + a.bytes;
}
// Whether a call's results share nothing with its inputs or each other.
template <int N, int M>
bool apart(const Run (&out)[N], const Run (&in)[M]) {
  for (int i = 0; i < N; ++i) {
    for (int j = 0; j < M; ++j)
      if (overlap(out[i], in[j])) return false;
    for (int j = 0; j < i; ++j)
      if (overlap(out[i], out[j])) return false;
  }
  return true;
}
// n rows of wa floats, la apart, against n of wb, lb apart: whether they are the same rows, or share nothing (rows of
// one pitch may lie between each other).  A row that is rewritten by who reads it may be the same; what lies across
// two rows may be written before it is read.
inline bool rows_alike_or_apart(const float* a, int64_t la, int64_t wa, const float* b, int64_t lb, int64_t wb, int64_t n) {
  const double pa = 4.0 * la, pb = 4.0 * lb, sa = 4.0 * wa, sb = 4.0 * wb;
  if (a == b && (la == lb || n == 1)) return true;
  if (!overlap({a, (n - 1) * pa + sa}, {b, (n - 1) * pb + sb})) return true;
  if (n == 1 || la != lb) return false;
  double at = fmod((double)(uintptr_t)b - (double)(uintptr_t)a, pa);
  if (at < 0) at += pa;
  return at >= sa && at + sb <= pa;
}

constexpr int kWave = 64;

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, kWave));
  return v;
}

// Block-wide sum for blockDim.x a multiple of 64 and <= 1024.  `red` must hold
// blockDim.x/64 floats of shared memory.  Every thread receives the result.
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, nw = blockDim.x >> 6;
  __syncthreads();
  if (lane == 0) red[wid] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < nw; ++i) t += red[i];
  return t;
}

__device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, nw = blockDim.x >> 6;
  __syncthreads();
  if (lane == 0) red[wid] = v;
  __syncthreads();
  float t = red[0];
  for (int i = 1; i < nw; ++i) t = fmaxf(t, red[i]);
  return t;
}

__host__ __device__ inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace cv3

#define CV3_HIP(expr)                                                              \
  do {                                                                             \
    hipError_t e_ = (expr);                                                        \
    if (e_ != hipSuccess)                                                          \
      return cv3::fail(CV3_EHIP, "%s failed: %s", #expr, hipGetErrorString(e_));  \
  } while (0)

#define CV3_LAUNCHED()                                                             \
  do {                                                                             \
    hipError_t e_ = hipGetLastError();                                             \
    if (e_ != hipSuccess)                                                          \
      return cv3::fail(CV3_EHIP, "kernel launch failed: %s", hipGetErrorString(e_)); \
  } while (0)

#define CV3_REQUIRE(cond, code, ...)                                               \
  do {                                                                             \
    if (!(cond)) return cv3::fail((code), __VA_ARGS__);                            \
  } while (0)

// First statement of every entry point that enqueues device work.
#define CV3_ALIVE() CV3_REQUIRE(!cv3::shut_down(), CV3_EINVAL, "the library has been shut down")
