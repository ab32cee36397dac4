// Log probabilities of given tokens, the entropy of their distributions and the best alternatives, from logits: what a
// program reads off when it scores texts or reports a choice (log_softmax, cv3cpu/ops.py:90-93).
#include "common.hpp"
#include "decode_common.hpp"   // DPP lane exchanges
#include "rank.hpp"

#include <algorithm>

using namespace cv3;

namespace {

constexpr int kTop = 32;             // alternatives of a row
constexpr int kVocabMax = 1 << 19;   // at most 64 slices of 8192 logits
constexpr int kThreads = 256;
constexpr int kList = 256;           // logits of a slice that may pass its bar by value alone

struct ScoreArgs {
  const float* logits;
  const int64_t* tokens;
  float* logprobs;
  float* entropy;
  int64_t* ids;
  float* values;
  uint64_t* keys;        // [rows, slices, top]: a slice's best logits, best first
  double* sums;          // [rows, slices, 2]: sums of e = exp(x - the slice's largest), and of e (x - the largest)
  float* tops;           // [rows, slices]
  int64_t vocab;
  int top, slices, slice;
};

struct Dist {            // of a whole row: log of the sum of exponentials, entropy
  double lse, entropy;
};
__device__ __forceinline__ Dist dist_of(double top, double s, double es) {
  if (!(top > -INFINITY)) return Dist{(double)NAN, (double)NAN};       // -inf alone: 0 / 0
  const double l = log(s);
  return Dist{top + l, l - es / s};
}

__device__ __forceinline__ void store_row(const ScoreArgs& a, int64_t row, const Dist& d) {
  const int64_t t = a.tokens[row];
  a.logprobs[row] = t >= 0 && t < a.vocab ? (float)((double)a.logits[row * a.vocab + t] - d.lse) : 0.f;
  a.entropy[row] = (float)d.entropy;
}
__device__ __forceinline__ void store_top(const ScoreArgs& a, int64_t row, int r, uint64_t key, const Dist& d) {
  a.ids[row * a.top + r] = (int64_t)(uint32_t)~(uint32_t)key;
  a.values[row * a.top + r] = (float)((double)rank_value((uint32_t)(key >> 32)) - d.lse);
}

// One slice of one row, E logits a thread, all loads in flight together; a row of one slice is finished here.
//
// The best `top`: of the 64 groups of four threads each has a largest logit, and what is among the slice's best W
// is no less than the W-th of those.  A few more than W logits pass that bar as a rule and are ranked by counting.
// A key is the logit's rank over the complement of its token, so no two are equal and equal logits go by the lower
// token.  Where more pass than the list holds (many equal logits) or the bar is -inf, the bar is set by whole keys:
// what passes it lies in W groups, at most 4 W E keys.  W is the most that `top` may be, 0 where none are asked for.
//
// Bound by HBM where there is much, each logit read once: 500 rows of 128000 45.8 us, 5.6 TB/s; 6 of 6761 6.0 us, the chain
// load, maximum, bar, sums, ranking.
template <int E, int W>
__global__ __launch_bounds__(kThreads) void k_score_slices(ScoreArgs a) {
  constexpr int kMost = W ? std::max(4 * W * E, kList) : 1;
  __shared__ uint64_t s_list[kMost];
  __shared__ uint64_t s_key[W ? 64 : 1];
  __shared__ float s_group[W ? 64 : 1];
  __shared__ float s_max[4];
  __shared__ double s_sum[4], s_prod[4];
  __shared__ int s_count;
  const int64_t row = blockIdx.x / (unsigned)a.slices;
  const int slice = (int)(blockIdx.x % (unsigned)a.slices);
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  struct __attribute__((packed, aligned(4))) Four {
    float v[4];
  };
  const int lo = slice * a.slice, hi = (int)min((int64_t)lo + a.slice, a.vocab);
  const float* x = a.logits + row * a.vocab;
  const int first = lo + tid * 4;      // this thread's tokens: first + 4 * kThreads * i + 0 .. 3
  float v[E], four[E / 4];
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    const int t = first + e * kThreads;
    if (t + 4 <= hi) {
      const Four f = *(const Four*)(x + t);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[e + i] = f.v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[e + i] = t + i < hi ? x[t + i] : -INFINITY;
    }
  }
  float mx = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    four[e / 4] = fmaxf(fmaxf(v[e], v[e + 1]), fmaxf(v[e + 2], v[e + 3]));
    mx = fmaxf(mx, four[e / 4]);
  }
  if constexpr (W > 0) {
    float best = mx;
    best = fmaxf(best, __uint_as_float(dpp32<kDppXor1>(__float_as_uint(best))));
    best = fmaxf(best, __uint_as_float(dpp32<kDppXor2>(__float_as_uint(best))));
    if ((lane & 3) == 0) s_group[tid >> 2] = best;
  }
  mx = wave_max_dpp(mx);
  if (lane == 0) s_max[wv] = mx;
  if (tid == 0) s_count = 0;
  __syncthreads();
  mx = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));

  bool whole_keys = false;
  if constexpr (W > 0) {
    // the W-th largest of the groups, by every wave for itself: the least that fewer than `top` surpass
    const float mine = s_group[lane];
    int above = 0;
#pragma unroll 16
    for (int i = 0; i < 64; ++i)
      above += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), i)) > mine ? 1 : 0;
    const float bar = -wave_max_dpp(above < a.top ? -mine : -INFINITY);
    whole_keys = bar == -INFINITY;
    if (!whole_keys) {
#pragma unroll
      for (int e = 0; e < E; e += 4)
        if (four[e / 4] >= bar) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (v[e + i] >= bar) {
              const int n = atomicAdd(&s_count, 1);      // the order goes: keys are ranked
              const uint32_t t = (uint32_t)(first + e * kThreads + i);
              if (n < kList) s_list[n] = (uint64_t)rank_bits(v[e + i]) << 32 | (uint32_t)~t;
            }
        }
    }
  }
  // Sums of four in float32, then float64.  A NaN, or +inf - +inf, makes both NaN; -inf adds nothing to either: its
  // exponential is 0, and the difference is held at -200, where exponentials have long been 0.
  const float ref = mx == -INFINITY ? 0.f : mx;
  double sum = 0.0, prod = 0.0;
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    float s = 0.f, p = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = v[e + i] - ref, z = __builtin_amdgcn_exp2f(y * kLog2E);
      s += z;
      p = fmaf(z, fmaxf(y, -200.f), p);
    }
    sum += (double)s;
    prod += (double)p;
  }
  sum = wave_sum_dpp(sum);
  prod = wave_sum_dpp(prod);
  if (lane == 0) s_sum[wv] = sum, s_prod[wv] = prod;
  __syncthreads();
  sum = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
  prod = s_prod[0] + s_prod[1] + s_prod[2] + s_prod[3];
  const bool alone = a.slices == 1;
  const Dist d = alone ? dist_of((double)mx, sum, prod) : Dist{};
  const int64_t at = row * a.slices + slice;
  if (tid == 0) {
    if (alone) {
      store_row(a, row, d);
    } else {
      a.sums[2 * at] = sum;
      a.sums[2 * at + 1] = prod;
      a.tops[at] = mx;
    }
  }
  if constexpr (W > 0) {
    int n = s_count;
    if (whole_keys || n > kList) {
      // rolled loops over the logits again, from L2: this is rare, and the code small
      auto key_at = [&](int e) -> uint64_t {
        const int t = first + (e >> 2) * 4 * kThreads + (e & 3);
        return t < hi ? (uint64_t)rank_bits(x[t]) << 32 | (uint32_t)~(uint32_t)t : 0;
      };
      uint64_t k = 0;
#pragma unroll 1
      for (int e = 0; e < E; ++e) k = max(k, key_at(e));
      k = max(k, dpp64<kDppXor1>(k));
      k = max(k, dpp64<kDppXor2>(k));
      if ((lane & 3) == 0) s_key[tid >> 2] = k;
      __syncthreads();                     // every thread has read s_count, and the keys are there
      if (tid == 0) s_count = 0;
      const uint64_t own = s_key[lane];
      int over = 0;
#pragma unroll 1
      for (int i = 0; i < 64; ++i) over += readlane64(own, i) > own ? 1 : 0;
      const uint64_t least = max(wave_max_u64(over >= a.top - 1 ? own : 0), (uint64_t)1);
      __syncthreads();
#pragma unroll 1
      for (int e = 0; e < E; ++e) {
        const uint64_t u = key_at(e);
        if (u >= least) s_list[atomicAdd(&s_count, 1)] = u;
      }
      __syncthreads();
      n = s_count;
    }
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t k = s_list[i];
      int r = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) r += s_list[j] > k ? 1 : 0;
      if (r < a.top) {
        if (alone) store_top(a, row, r, k, d);
        else a.keys[at * a.top + r] = k;
      }
    }
    if (!alone && tid >= n && tid < a.top) a.keys[at * a.top + tid] = 0;     // a last slice with fewer logits
  }
}

// The slices of a row, one workgroup each: sums over the largest of their maxima, and the best of their sorted lists.
// The W-th best of the lists' heads is a bar that at most W lists pass.  500 rows of 16 slices: 4.8 us, a launch and its chain.
__global__ __launch_bounds__(kThreads) void k_score_join(ScoreArgs a) {
  __shared__ uint64_t s_list[kTop * 64];
  __shared__ uint64_t s_pass[kTop * kTop];
  __shared__ Dist s_dist;
  __shared__ int s_count;
  const int64_t row = blockIdx.x, list0 = row * a.slices;
  const int tid = threadIdx.x, lane = tid & 63;
  const int candidates = a.slices * a.top;
  for (int i = tid; i < candidates; i += kThreads) s_list[i] = a.keys[list0 * a.top + i];
  if (tid < 64) {              // at most 64 slices: a lane each
    const float top = lane < a.slices ? a.tops[list0 + lane] : -INFINITY;
    double s = lane < a.slices ? a.sums[2 * (list0 + lane)] : 0.0, p = lane < a.slices ? a.sums[2 * (list0 + lane) + 1] : 0.0;
    const float all = wave_max_dpp(top);
    if (top != all) {
      const double down = (double)top - (double)all, f = exp(down);      // 0 where the slice is -inf
      p = top > -INFINITY ? f * (p + down * s) : f * s;                  // f * s: NaN where the slice's NaN hides in s
      s *= f;
    }
    s = wave_sum_dpp(s);
    p = wave_sum_dpp(p);
    if (lane == 0) {
      s_dist = dist_of((double)all, s, p);
      s_count = 0;
      store_row(a, row, s_dist);
    }
  }
  __syncthreads();
  if (a.top == 0) return;
  const Dist d = s_dist;
  uint64_t bar = 1;
  if (a.slices > a.top) {
    const uint64_t head = lane < a.slices ? s_list[lane * a.top] : 0;
    int above = 0;
    for (int i = 0; i < a.slices; ++i) above += readlane64(head, i) > head ? 1 : 0;
    bar = max(bar, wave_max_u64(above >= a.top - 1 ? head : 0));
  }
  for (int i = tid; i < candidates; i += kThreads)
    if (s_list[i] >= bar) s_pass[atomicAdd(&s_count, 1)] = s_list[i];
  __syncthreads();
  const int n = s_count;
  for (int i = tid; i < n; i += kThreads) {
    const uint64_t k = s_pass[i];
    int r = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) r += s_pass[j] > k ? 1 : 0;
    if (r < a.top) store_top(a, row, r, k, d);
  }
}

// Up to 2048 and 4096 logits a row, slices as long: 2000 rows of 2000 15.6 us with 32 logits a thread, 11.6 with 8; 1000 of
// 4000 10.4 and 8.7 with 16; 3 of 2000 6.7 and 6.9.
template <int E>
void launch_slices(const ScoreArgs& a, int64_t rows, hipStream_t st) {
  const dim3 grid((unsigned)(rows * a.slices)), block(kThreads);
  if (a.top == 0) hipLaunchKernelGGL((k_score_slices<E, 0>), grid, block, 0, st, a);
  else if (a.top <= 8) hipLaunchKernelGGL((k_score_slices<E, 8>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((k_score_slices<E, kTop>), grid, block, 0, st, a);
}

}  // namespace

extern "C" {

int cv3_token_logprobs(const float* logits, int64_t rows, int64_t vocab, const int64_t* tokens, int top,
                       float* logprobs, float* entropy, int64_t* top_ids, float* top_logprobs, cv3_stream_t s) {
  CV3_ALIVE();
  CV3_REQUIRE(vocab >= 1 && vocab <= kVocabMax, CV3_EINVAL, "a vocabulary of 1 to %d tokens, not %lld", kVocabMax,
              (long long)vocab);
  CV3_REQUIRE(top >= 0 && top <= kTop && top <= vocab, CV3_EINVAL, "0 to %d alternatives out of %lld tokens, not %d", kTop,
              (long long)vocab, top);
  // a launch has fewer than 2^32 threads: 256 a slice
  CV3_REQUIRE(rows >= 0 && rows <= ((1 << 24) - 1) / ceil_div(vocab, 32 * kThreads), CV3_EINVAL,
              "%lld rows of %lld logits are too many for one call", (long long)rows, (long long)vocab);
  if (rows == 0) return CV3_OK;
  CV3_REQUIRE(logits && tokens && logprobs && entropy && (top == 0 || (top_ids && top_logprobs)), CV3_EINVAL, "null operand");
  const double n = (double)rows;
  const Run in[] = {{logits, 4 * n * vocab}, {tokens, 8 * n}};
  const Run out[] = {{logprobs, 4 * n}, {entropy, 4 * n}, {top_ids, 8 * n * top}, {top_logprobs, 4 * n * top}};
  CV3_REQUIRE(apart(out, in), CV3_EINVAL, "results that overlap each other, the logits or the tokens");
  ScoreArgs a{logits, tokens, logprobs, entropy, top_ids, top_logprobs, nullptr, nullptr, nullptr, vocab, top, 1, 32 * kThreads};
  a.slices = (int)ceil_div(vocab, a.slice);
  hipStream_t st = stream_of(s);
  if (a.slices == 1) {
    if (vocab <= 8 * kThreads) launch_slices<8>(a, rows, st);
    else if (vocab <= 16 * kThreads) launch_slices<16>(a, rows, st);
    else launch_slices<32>(a, rows, st);
    CV3_LAUNCHED();
    return CV3_OK;
  }
  const int64_t lists = rows * a.slices;
  void* work = nullptr;
  if (int rc = scratch_alloc(&work, (size_t)lists * (top * 8 + 20), st)) return rc;
  a.sums = (double*)work;
  a.keys = (uint64_t*)(a.sums + 2 * lists);
  a.tops = (float*)(a.keys + lists * top);
  launch_slices<32>(a, rows, st);
  hipLaunchKernelGGL(k_score_join, dim3((unsigned)rows), dim3(kThreads), 0, st, a);
  const hipError_t err = hipGetLastError();
  const int rc = scratch_free(work, st);
  CV3_REQUIRE(err == hipSuccess, CV3_EHIP, "kernel launch failed: %s", hipGetErrorString(err));
  return rc;
}

}  // extern "C"
