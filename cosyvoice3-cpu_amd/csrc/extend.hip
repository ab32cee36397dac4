// Attention of several new tokens per sequence over the paged cache: prompts in slices, drafted tokens, texts to score.
// Every query sees its sequence's keys up to itself (sdpa with a causal mask, cv3cpu/ops.py:267-300; the reference runs
// one sequence's prompt at a time over a contiguous cache, cv3cpu/models/qwen2.py:139-179).
//
// The queries are a ragged list: rows starts[b] .. starts[b + 1] are sequence b's last tokens, the last of them at
// position lengths[b] - 1.  Page ids, lengths and starts come from device memory and are checked where they are used.
#include "paged_common.hpp"

#include <algorithm>

using namespace cv3;

namespace {

struct __attribute__((packed, aligned(4))) f32x4u {
  float v[4];
};

struct ExtArgs {
  const float* q;
  int64_t ldq;
  const void* k;
  const void* v;
  const int32_t* tables;
  const int32_t* lengths;
  const int32_t* starts;
  float* out;
  int64_t ldo;
  int64_t pages, blocks, n;
  int window;                  // keys that a query sees at most
  int batch, page, heads, kv_heads, group, d;
  float scale;                 // times log2(e)
};

template <typename E>
__device__ __forceinline__ float to_float(E x) { return (float)x; }

// Rows of sequence b in the list, [first, first + count), and the position of the first of them.
struct Seq {
  int first, count, base, len;
};
__device__ __forceinline__ Seq seq_of(const ExtArgs& a, int b) {
  Seq s;
  s.first = (int)min((int64_t)max(a.starts[b], 0), a.n);
  s.count = (int)min((int64_t)max(a.starts[b + 1], s.first), a.n) - s.first;
  s.len = (int)min((int64_t)max(a.lengths[b], 0), a.blocks * a.page);
  s.base = s.len - s.count;
  return s;
}

// One query over keys [lo, hi) by one wave, in float32 throughout: a key a lane for the scores, four channels a lane
// for the sum.  Outputs are summed and then divided.
template <typename E>
struct RowSum {
  float o[4], top, sum;
  bool there;                  // a key, whatever its score

  __device__ __forceinline__ void run(const ExtArgs& a, int b, int kvh, const float* q, int lo, int hi) {
    const int lane = threadIdx.x & 63;
    const int32_t* table = a.tables + (int64_t)b * a.blocks;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = 0.f;
    top = -INFINITY;
    sum = 0.f;
    there = false;
#pragma unroll 1
    for (int k0 = lo; k0 < hi; k0 += 64) {
      const int key = k0 + lane;
      int64_t off = -1;
      if (key < hi) {
        const uint32_t blk = (uint32_t)key / (uint32_t)a.page;
        const int32_t id = table[blk];
        if ((uint32_t)id < (uint64_t)a.pages)
          off = (((int64_t)id * a.kv_heads + kvh) * a.page + (key - (int64_t)blk * a.page)) * a.d;
      }
      float x = -INFINITY;
      if (off >= 0) {
        const E* kr = (const E*)a.k + off;
        float dot = 0.f;
#pragma unroll 2
        for (int c = 0; c < a.d; c += 4) {
          const f32x4u qv = *(const f32x4u*)(q + c);
#pragma unroll
          for (int i = 0; i < 4; ++i) dot = fmaf(qv.v[i], to_float(kr[c + i]), dot);
        }
        x = dot * a.scale;
      }
      uint64_t seen = __ballot(off >= 0);
      if (!seen) continue;
      there = true;
      const float now = fmaxf(top, wave_max(x));
      const float f = weight_of(top, now), ref = now == -INFINITY ? 0.f : now;
      top = now;
      const float p = off >= 0 ? exp2_fast(x - ref) : 0.f;
      sum = sum * f + p;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] *= f;
      while (seen) {
        const int j = uniform(__ffsll((unsigned long long)seen) - 1);
        seen &= seen - 1;
        const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), j));
        const E* vr = (const E*)a.v + uniform(__shfl(off, j, kWave));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (64 * i + lane < a.d) o[i] = fmaf(w, to_float(vr[64 * i + lane]), o[i]);
      }
    }
    sum = wave_sum(sum);
  }
};

// One wave a query.
template <typename E>
__global__ __launch_bounds__(256) void k_extend_rows(ExtArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + uniform((int)threadIdx.x >> 6);
  const int64_t row = item / a.heads;
  const int head = (int)(item % a.heads);
  if (row >= a.n) return;
  int b = -1;
  Seq s{};
  for (int i = 0; i < a.batch; ++i) {
    s = seq_of(a, i);
    if (row >= s.first && row < s.first + s.count) {
      b = i;
      break;
    }
  }
  if (b < 0) return;
  const int hi = max(0, s.base + (int)(row - s.first) + 1), lo = max(0, hi - a.window);
  RowSum<E> r;
  r.run(a, b, head / a.group, a.q + row * a.ldq + (int64_t)head * a.d, lo, hi);
  float* out = a.out + row * a.ldo + (int64_t)head * a.d;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (64 * i + lane < a.d) out[64 * i + lane] = r.there ? r.o[i] / r.sum : 0.f;
}

}  // namespace

extern "C" {

int cv3_paged_extend(const float* q, int64_t ldq, int64_t n, int heads, int kv_heads, int d, int cache_type,
                     const void* k_cache, const void* v_cache, int64_t pages, int64_t page, const int32_t* tables,
                     int64_t blocks, const int32_t* lengths, const int32_t* starts, int64_t batch, int64_t window,
                     float scale, float* out, int64_t ldo, cv3_stream_t s) {
  CV3_ALIVE();
  CV3_REQUIRE(kv_heads >= 1 && heads >= 1 && heads % kv_heads == 0, CV3_EINVAL,
              "%d query heads is not a multiple of %d kv heads", heads, kv_heads);
  if (int rc = check_cache(cache_type, k_cache, v_cache, pages, page, kv_heads, d)) return rc;
  CV3_REQUIRE(heads <= 65536, CV3_EINVAL, "at most 65536 query heads, not %d", heads);
  CV3_REQUIRE(blocks >= 1 && blocks <= (INT32_MAX - 65536) / page, CV3_EINVAL,
              "tables of %lld blocks of %lld keys pass 2^31 keys", (long long)blocks, (long long)page);
  CV3_REQUIRE(n >= 0 && batch >= 0 && n <= kLaunchBlocks / heads && batch <= kLaunchBlocks / heads, CV3_EINVAL,
              "%lld rows of %lld sequences are too many for one call", (long long)n, (long long)batch);
  CV3_REQUIRE(window >= 1, CV3_EINVAL, "a window of %lld keys", (long long)window);
  CV3_REQUIRE(ldq >= (int64_t)heads * d && ldo >= (int64_t)heads * d, CV3_EINVAL, "rows are too short for %d heads of %d",
              heads, d);
  if (n == 0 || batch == 0) return CV3_OK;
  CV3_REQUIRE(q && tables && lengths && starts && out, CV3_EINVAL, "null operand");
  CV3_REQUIRE(rows_alike_or_apart(q, ldq, (int64_t)heads * d, out, ldo, (int64_t)heads * d, n), CV3_EINVAL,
              "out and q overlap: out may be q itself, at its pitch");
  const double cache = (double)pages * page * kv_heads * d * elem_size(cache_type);
  const Run in[] = {{k_cache, cache}, {v_cache, cache}, {tables, 4.0 * batch * blocks}, {lengths, 4.0 * batch},
                    {starts, 4.0 * (batch + 1)}};
  const Run res[] = {{out, 4.0 * ((n - 1) * (double)ldo + (double)heads * d)}};
  CV3_REQUIRE(apart(res, in), CV3_EINVAL, "out overlaps the caches, the tables, the lengths or the starts");
  ExtArgs a{q, ldq, k_cache, v_cache, tables, lengths, starts, out, ldo, pages, blocks, n,
            (int)std::min<int64_t>(window, INT32_MAX), (int)batch, (int)page, heads, kv_heads, heads / kv_heads, d,
            scale * 1.4426950408889634f};
  hipStream_t st = stream_of(s);
  const dim3 grid((unsigned)ceil_div(n * heads, 4));
  if (cache_type == CV3_F32) hipLaunchKernelGGL(k_extend_rows<float>, grid, dim3(256), 0, st, a);
  else if (cache_type == CV3_F16) hipLaunchKernelGGL(k_extend_rows<_Float16>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(k_extend_rows<__bf16>, grid, dim3(256), 0, st, a);
  CV3_LAUNCHED();
  return CV3_OK;
}

}  // extern "C"
