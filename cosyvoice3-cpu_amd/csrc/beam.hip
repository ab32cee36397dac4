// Beam search over the paged cache: the best continuations over beams and vocabulary, and the
// tables and part-filled pages that follow the chosen beams.  The reference draws one token for one
// sequence (log_softmax, cv3cpu/ops.py:90-93; _sample, cv3cpu/models/llm.py:125-149).
#include "common.hpp"
#include "decode_common.hpp"   // DPP lane exchanges
#include "rank.hpp"

#include <algorithm>

using namespace cv3;

namespace {

constexpr int kBeams = 16;           // beams of a request
constexpr int kVocabMax = 1 << 19;   // at most 64 slices of 8192 logits
constexpr int kSelThreads = 256;

struct SelectArgs {
  const float* logits;
  const float* scores;
  const uint8_t* done;
  uint64_t* keys;        // [rows, slices, beams]: a slice's best logits, best first
  double* sums;          // [rows, slices]: sum of exp(logit - the slice's largest)
  float* tops;           // [rows, slices]
  int64_t* tokens;
  int32_t* parents;
  float* scores_out;
  uint8_t* done_out;
  int64_t vocab, stop_lo, stop_hi, ban_lo, ban_hi, pad;
  int beams, slices, slice;
};

constexpr int kList = 512;     // logits of a slice that may pass its bar by value alone

// Best `beams` logits of one slice of one row, and its part of the softmax's sum; HBM-bound, the
// logits read once, E a thread, all loads in flight together.
//
// Of the 64 groups of four threads each has a largest logit.  What is among the slice's best W is no
// less than the W-th of those: a few more than W logits pass that bar as a rule, and are ranked by
// counting.  A key is the logit's rank over the complement of its token, so no two are equal and
// equal logits go by the lower token.  Where more pass than the list holds (many equal logits), the
// bar is -inf or some of the slice's tokens are banned, the bar is set by whole keys: whatever passes
// it then lies in W groups, at most 4 W E keys.  24 x 8 rows of 128000: 21.6 us, 4.6 TB/s; 4 rows of 6761:
// 4.8 us, the chain of load, two joins of the waves and a ranking.
template <int E>
__global__ __launch_bounds__(kSelThreads, 6) void k_select_slices(SelectArgs a) {
  constexpr int kMost = 4 * kBeams * E;
  __shared__ uint64_t s_list[kMost > kList ? kMost : kList];
  __shared__ uint64_t s_key[64];
  __shared__ float s_group[64];
  __shared__ float s_max[4];
  __shared__ double s_sum[4];
  __shared__ int s_count;
  const int row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  if (a.done[row]) return;             // its one continuation needs no logits
  struct __attribute__((packed, aligned(4))) Four {
    float v[4];
  };
  const int lo = slice * a.slice, hi = (int)min((int64_t)lo + a.slice, a.vocab);
  const float* x = a.logits + (int64_t)row * a.vocab;
  const int first = lo + tid * 4;      // this thread's tokens: first + 4 * kSelThreads * i + 0 .. 3
  float v[E], four[E / 4];
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    const int t = first + e * kSelThreads;
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
  float best = mx;
  best = fmaxf(best, __uint_as_float(dpp32<kDppXor1>(__float_as_uint(best))));
  best = fmaxf(best, __uint_as_float(dpp32<kDppXor2>(__float_as_uint(best))));
  if ((lane & 3) == 0) s_group[tid >> 2] = best;
  mx = wave_max_dpp(mx);
  if (lane == 0) s_max[wv] = mx;
  if (tid == 0) s_count = 0;
  __syncthreads();
  mx = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));

  // the W-th largest of the groups, by every wave for itself: the least that fewer than W surpass
  const float mine = s_group[lane];
  int above = 0;
#pragma unroll 16
  for (int i = 0; i < 64; ++i)
    above += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), i)) > mine ? 1 : 0;
  const float bar = -wave_max_dpp(above < a.beams ? -mine : -INFINITY);
  const bool whole_keys = bar == -INFINITY || (a.ban_lo < hi && a.ban_hi > lo);
  if (!whole_keys) {
#pragma unroll
    for (int e = 0; e < E; e += 4)
      if (four[e / 4] >= bar) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (v[e + i] >= bar) {
            const int n = atomicAdd(&s_count, 1);
            const uint32_t t = (uint32_t)(first + e * kSelThreads + i);
            if (n < kList) s_list[n] = (uint64_t)rank_bits(v[e + i]) << 32 | ~t;
          }
      }
  }
  // Sums of four in float32, then float64: a NaN, or +inf - +inf, makes the row's sum NaN.
  const float ref = mx == -INFINITY ? 0.f : mx;
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) s += __builtin_amdgcn_exp2f((v[e + i] - ref) * kLog2E);
    sum += (double)s;
  }
  sum = wave_sum_dpp(sum);
  if (lane == 0) s_sum[wv] = sum;
  __syncthreads();
  int n = s_count;
  if (whole_keys || n > kList) {
    // rolled loops over the logits again, from L2: this is rare, and the code small
    auto key_at = [&](int e) -> uint64_t {
      const int t = first + (e >> 2) * 4 * kSelThreads + (e & 3);
      return t < hi && !(t >= a.ban_lo && t < a.ban_hi) ? (uint64_t)rank_bits(x[t]) << 32 | ~(uint32_t)t : 0;
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
    const uint64_t least = max(wave_max_u64(over >= a.beams - 1 ? own : 0), (uint64_t)1);
    __syncthreads();
#pragma unroll 1
    for (int e = 0; e < E; ++e) {
      const uint64_t u = key_at(e);
      if (u >= least) s_list[atomicAdd(&s_count, 1)] = u;
    }
    __syncthreads();
    n = s_count;
  }
  const int64_t at = (int64_t)row * a.slices + slice;
  uint64_t* out = a.keys + at * a.beams;
  for (int i = tid; i < n; i += kSelThreads) {
    const uint64_t k = s_list[i];
    int r = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) r += s_list[j] > k ? 1 : 0;
    if (r < a.beams) out[r] = k;
  }
  if (tid >= n && tid < a.beams) out[tid] = 0;
  if (tid == 0) {
    a.sums[at] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
    a.tops[at] = mx;
  }
}

struct Pick {            // larger is better: the value, then the lower beam, the larger logit, the lower token
  uint64_t hi, lo;
  __device__ bool operator>(const Pick& o) const { return hi != o.hi ? hi > o.hi : lo > o.lo; }
};

constexpr int kPickThreads = 512;
constexpr int kLists = kBeams * 64;            // of a request: its beams' slices
constexpr int kListsEach = kLists / kPickThreads;
constexpr int kPicks = kBeams * kListsEach * kBeams;
constexpr int kEarly = 2;                     // candidates of a thread that are loaded with the heads

// One workgroup per request; bound by the chain of its few loads (24 requests of 8 x 16 lists 6.4 us, one of
// 4 x 4 lists 4.7).  The slices' lists are sorted, so
// the best of a thread's lists are their heads.  As above, the W-th largest value of 64 groups of
// threads is a bar that a few more than W pass; where equal values bring more than the list holds, the
// W-th best head of the threads, whole, bounds them by W lists a thread x W threads x W keys.
__global__ __launch_bounds__(kPickThreads) void k_select_beams(SelectArgs a) {
  __shared__ double s_lse[kBeams], s_score[kBeams];
  __shared__ int s_done[kBeams];
  __shared__ double s_sum[kLists];
  __shared__ float s_top[kLists];
  __shared__ Pick s_best[kPickThreads];
  __shared__ Pick s_list[kPicks];
  __shared__ Pick s_out[kBeams];
  __shared__ Pick s_bar;
  __shared__ uint32_t s_high[kPickThreads];
  __shared__ int s_count;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t row0 = (int64_t)blockIdx.x * a.beams;
  const int lists = a.beams * a.slices;
  // An ended beam's lists hold whatever the memory held: they are not looked at.
  const int64_t list0 = row0 * a.slices;
  const uint64_t* keys = a.keys + list0 * a.beams;
  const unsigned beams = (unsigned)a.beams, slices = (unsigned)a.slices, candidates = (unsigned)lists * beams;
  const uint64_t head = tid < lists ? keys[tid * a.beams] : 0;
  uint64_t early[kEarly];                      // this thread's first candidates, loaded with the heads
#pragma unroll
  for (int i = 0; i < kEarly; ++i) early[i] = tid + i * kPickThreads < candidates ? keys[tid + i * kPickThreads] : 0;
#pragma unroll 1
  for (int l = tid; l < lists; l += kPickThreads) {
    s_sum[l] = a.sums[list0 + l];
    s_top[l] = a.tops[list0 + l];
  }
  if (tid < a.beams) {
    s_score[tid] = (double)a.scores[row0 + tid];
    s_done[tid] = a.done[row0 + tid];
  }
  if (tid < kBeams) s_out[tid] = Pick{0, 0};
  if (tid == 0) {
    s_count = 0;
    s_bar = Pick{0, 1};
  }
  __syncthreads();
  for (int b = wv; b < a.beams; b += kPickThreads / 64) {
    // at most 64 slices: a lane each
    const float top = lane < a.slices ? s_top[b * a.slices + lane] : -INFINITY;
    const float all = wave_max_dpp(top);
    double sum = lane < a.slices ? s_sum[b * a.slices + lane] : 0.0;
    if (top != all) sum *= exp((double)top - (double)all);     // 0 or NaN where the slice is -inf
    sum = wave_sum_dpp(sum);
    if (lane == 0) s_lse[b] = all > -INFINITY ? (double)all + log(sum) : (double)NAN;
  }
  __syncthreads();
  // The candidate of beam b that key k, of that rank in one of its lists, stands for.
  auto pick = [&](int b, bool leads, uint64_t k) -> Pick {
    const uint64_t order = (uint64_t)(31 - b) << 59;
    if (s_done[b]) return leads ? Pick{rank_bits(s_score[b]), order} : Pick{0, 0};
    if (!k) return Pick{0, 0};
    const double value = s_score[b] + ((double)rank_value((uint32_t)(k >> 32)) - s_lse[b]);
    return Pick{rank_bits(value), order | (k >> 32) << 27 | (k & 0x7ffffff)};
  };
  Pick best{0, 0};
#pragma unroll 1
  for (int l = tid; l < lists; l += kPickThreads) {
    const unsigned b = (unsigned)l / slices;
    const Pick p = pick(b, l == b * slices, l == tid ? head : keys[l * a.beams]);
    if (p > best) best = p;
  }
  s_best[tid] = best;
  s_high[tid] = (uint32_t)(best.hi >> 32);     // the upper half of a value's rank is enough for the bar
  __syncthreads();
  uint32_t group = 0;                          // of threads 64 apart: one beam's lists are neighbours
#pragma unroll
  for (int i = 0; i < kPickThreads; i += 64) group = max(group, s_high[i + lane]);
  int above = 0;
#pragma unroll
  for (int i = 0; i < 64; ++i) above += (uint32_t)__builtin_amdgcn_readlane((int)group, i) > group ? 1 : 0;
  // the least that fewer than W surpass; 0 (there are fewer heads): everything
  uint32_t least = above < a.beams ? ~group : 0;
  least = max(least, dpp32<kDppXor1>(least));
  least = max(least, dpp32<kDppXor2>(least));
  least = max(least, dpp32<kDppHalfMirror>(least));
  least = max(least, dpp32<kDppMirror>(least));
  least = ~max(max((uint32_t)__builtin_amdgcn_readlane((int)least, 0), (uint32_t)__builtin_amdgcn_readlane((int)least, 16)),
               max((uint32_t)__builtin_amdgcn_readlane((int)least, 32), (uint32_t)__builtin_amdgcn_readlane((int)least, 48)));
  Pick bar{(uint64_t)least << 32, 0};
#pragma unroll 1
  for (bool whole = false;; whole = true) {
    // Every candidate against the bar, a thread each.
#pragma unroll 1
    for (unsigned c = tid, i = 0; c < candidates; c += kPickThreads, ++i) {
      const unsigned list = c / beams, b = list / slices;
      if (s_high[list % kPickThreads] < (uint32_t)(bar.hi >> 32)) continue;      // the list's head does not pass
      uint64_t k = early[0];
      if (i > 0) k = i == 1 ? early[1] : keys[c];
      const Pick p = pick(b, list * beams == c && list == b * slices, k);
      if (p.hi && !(bar > p)) {
        const int at = atomicAdd(&s_count, 1);
        if (at < kPicks) s_list[at] = p;
      }
    }
    __syncthreads();
    if (whole || s_count <= kPicks) break;
    // more equal values than the list holds: a bar of one whole head
    const int heads = min(lists, kPickThreads);
    above = 0;
#pragma unroll 1
    for (int i = 0; i < heads; ++i) above += s_best[i] > best ? 1 : 0;
    if (tid < heads && above == a.beams - 1 && best.hi) s_bar = best;
    __syncthreads();                           // every thread has read s_count
    if (tid == 0) s_count = 0;
    bar = s_bar;
    __syncthreads();
  }
  const int n = s_count;
  for (int i = tid; i < n; i += kPickThreads) {
    const Pick p = s_list[i];
    int r = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) r += s_list[j] > p ? 1 : 0;
    if (r < a.beams) s_out[r] = p;
  }
  __syncthreads();
  if (tid < a.beams) {                         // scores_out and done_out may be scores and done: those are read
    const Pick p = s_out[tid];
    int parent = 31 - (int)(p.lo >> 59);
    if (parent < 0 || parent >= a.beams) parent = 0;
    const bool ended = s_done[parent] != 0;
    const int64_t token = ended ? a.pad : (int64_t)(0x7ffffff - (p.lo & 0x7ffffff));
    a.tokens[row0 + tid] = token;
    a.parents[row0 + tid] = parent;
    a.scores_out[row0 + tid] = (float)rank_value(p.hi);
    a.done_out[row0 + tid] = ended || (token >= a.stop_lo && token < a.stop_hi) ? 1 : 0;
  }
}

template <int E>
void launch_slices(const SelectArgs& a, int64_t rows, hipStream_t st) {
  hipLaunchKernelGGL(k_select_slices<E>, dim3((unsigned)(rows * a.slices)), dim3(kSelThreads), 0, st, a);
}

// ------------------------------------------------------------------------------------------------

struct ReorderArgs {
  const int32_t* parents;
  int32_t* tables;
  const int32_t* own;
  const int32_t* lengths;
  uint4* k;
  uint4* v;
  int64_t pages, blocks, layers;
  int beams, kv_heads, page, row_vecs;   // 16-byte vectors of a key row
  int parts, table_parts;                // workgroups of a run of rows, and of a request's table
};

// Copies move a part-filled page's rows between the beams' own pages, in place and in any order: a
// thread holds the same 16 bytes of every beam's page, reads all it needs and only then writes.
// HBM-bound (16 requests of 8 beams, 24 layers of bfloat16, pages of 64: 19.6 us, 16.7 at best, 4.4 - 5.2 TB/s); a beam
// that stays itself costs nothing.  Of a request's workgroups
// the last table_parts turn its table, column by column, in the same way.
template <int W>
__global__ __launch_bounds__(256) void k_beam_reorder(ReorderArgs a) {
  const int64_t copies = a.layers * a.kv_heads * 2 * a.parts, r = blockIdx.y, in = blockIdx.x;
  const int64_t cap = a.blocks * a.page;
  const int64_t len = min((int64_t)max(a.lengths[r], 0), cap);
  const int64_t full = len / a.page, rest = len - full * a.page;
  const int32_t* parents = a.parents + r * a.beams;
  if (in >= copies) {
    int32_t* table = a.tables + r * a.beams * a.blocks;
    const int32_t* own = a.own + r * a.beams * a.blocks;
    const int64_t c = (in - copies) * 256 + threadIdx.x;
    if (c >= a.blocks) return;
    int32_t id[W];
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (w < a.beams) {
        const int p = parents[w];
        id[w] = (unsigned)p >= (unsigned)a.beams ? table[w * a.blocks + c]
                : c < full                       ? table[p * a.blocks + c]
                                                 : own[w * a.blocks + c];
      }
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (w < a.beams) table[w * a.blocks + c] = id[w];
    return;
  }
  const int vec = (int)(in % a.parts) * 256 + (int)threadIdx.x;
  if (vec >= rest * a.row_vecs) return;
  const int64_t lane_of = in / a.parts;          // [layer][k or v][kv head]
  const int kv = (int)(lane_of % a.kv_heads);
  uint4* cache = (lane_of / a.kv_heads) % 2 ? a.v : a.k;
  const int64_t layer = lane_of / a.kv_heads / 2;
  const int32_t* own = a.own + r * a.beams * a.blocks + full;
  const int64_t run = (int64_t)a.page * a.row_vecs, page_vecs = run * a.kv_heads;
  uint4* base = cache + layer * a.pages * page_vecs + kv * run + vec;
  uint4 x[W];
  int64_t to[W];           // -1: this beam's rows stay
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int p = w < a.beams ? parents[w] : w;
    const bool other = p != w && (unsigned)p < (unsigned)a.beams;
    const int64_t from = other ? own[p * a.blocks] : -1;
    to[w] = other ? own[w * a.blocks] : -1;
    if (from < 0 || from >= a.pages || to[w] >= a.pages) to[w] = -1;
    x[w] = to[w] >= 0 ? base[from * page_vecs] : uint4{};
  }
#pragma unroll
  for (int w = 0; w < W; ++w)
    if (to[w] >= 0) base[to[w] * page_vecs] = x[w];
}

}  // namespace

extern "C" {

int cv3_beam_select(const float* logits, int64_t requests, int beams, int64_t vocab, const float* scores,
                    const uint8_t* done, int64_t stop_lo, int64_t stop_hi, int64_t ban_lo, int64_t ban_hi, int64_t pad,
                    int64_t* tokens, int32_t* parents, float* scores_out, uint8_t* done_out, cv3_stream_t s) {
  CV3_ALIVE();
  CV3_REQUIRE(beams >= 1 && beams <= kBeams, CV3_EINVAL, "1 to %d beams, not %d", kBeams, beams);
  CV3_REQUIRE(vocab >= 1 && vocab <= kVocabMax, CV3_EINVAL, "a vocabulary of 1 to %d tokens, not %lld", kVocabMax,
              (long long)vocab);
  // a launch has fewer than 2^32 threads: 512 a request, 256 a slice
  CV3_REQUIRE(requests >= 0 && requests < (1 << 23) && requests * beams <= (1 << 23) / ceil_div(vocab, 8 * kSelThreads), CV3_EINVAL,
              "%lld requests of %d beams are too many for one call", (long long)requests, beams);
  const int64_t banned = std::max<int64_t>(0, std::min(ban_hi, vocab) - std::max<int64_t>(ban_lo, 0));
  CV3_REQUIRE(vocab - banned >= beams, CV3_EINVAL, "%lld tokens to choose from are fewer than %d beams",
              (long long)(vocab - banned), beams);
  if (requests == 0) return CV3_OK;
  CV3_REQUIRE(logits && scores && done && tokens && parents && scores_out && done_out, CV3_EINVAL, "null operand");
  const int64_t rows = requests * beams;
  const double n = (double)rows;
  const Run in[] = {{logits, 4 * n * vocab}, {scores, scores == scores_out ? 0 : 4 * n}, {done, done == done_out ? 0 : n}};
  const Run out[] = {{tokens, 8 * n}, {parents, 4 * n}, {scores_out, 4 * n}, {done_out, n}};
  CV3_REQUIRE(apart(out, in), CV3_EINVAL, "results that overlap: only scores_out may be scores, and done_out done");
  // 2048 logits a workgroup where 8192 would leave half the CUs idle (16 x 4 rows of 6761: 10.0 us a call
  // against 11.1; 64 x 4: 11.9 against 11.2; 2 x 8 of 128000: 13.8 against 12.3), and a list a lane is enough
  const int e = rows * ceil_div(vocab, 32 * kSelThreads) < 128 && vocab <= 64 * 8 * kSelThreads ? 8 : 32;
  SelectArgs a{logits, scores, done, nullptr, nullptr, nullptr, tokens, parents, scores_out, done_out, vocab, stop_lo,
               stop_hi, ban_lo, ban_hi, pad, beams, 0, e * kSelThreads};
  a.slices = (int)ceil_div(vocab, a.slice);
  hipStream_t st = stream_of(s);
  const int64_t lists = rows * a.slices;
  void* work = nullptr;
  if (int rc = scratch_alloc(&work, (size_t)lists * (beams * 8 + 16), st)) return rc;
  a.keys = (uint64_t*)work;
  a.sums = (double*)(a.keys + lists * beams);
  a.tops = (float*)(a.sums + lists);
  e == 8 ? launch_slices<8>(a, rows, st) : launch_slices<32>(a, rows, st);
  hipLaunchKernelGGL(k_select_beams, dim3((unsigned)requests), dim3(kPickThreads), 0, st, a);
  const hipError_t err = hipGetLastError();
  const int rc = scratch_free(work, st);
  CV3_REQUIRE(err == hipSuccess, CV3_EHIP, "kernel launch failed: %s", hipGetErrorString(err));
  return rc;
}

int cv3_beam_reorder(const int32_t* parents, int64_t requests, int beams, int32_t* tables, const int32_t* own,
                     int64_t blocks, const int32_t* lengths, int cache_type, void* k_cache, void* v_cache,
                     int64_t layers, int64_t pages, int kv_heads, int64_t page, int d, cv3_stream_t s) {
  CV3_ALIVE();
  CV3_REQUIRE(cache_type == CV3_F32 || cache_type == CV3_F16 || cache_type == CV3_BF16, CV3_EINVAL,
              "unknown cache type %d", cache_type);
  CV3_REQUIRE(beams >= 1 && beams <= kBeams, CV3_EINVAL, "1 to %d beams, not %d", kBeams, beams);
  CV3_REQUIRE(page >= 1 && page <= 65536, CV3_EINVAL, "a page holds 1 to 65536 keys, not %lld", (long long)page);
  CV3_REQUIRE(pages >= 1 && pages <= INT32_MAX && layers >= 1 && layers <= 65536 && kv_heads >= 1 && kv_heads <= 1024,
              CV3_EINVAL, "bad cache shape");
  CV3_REQUIRE(d >= 8 && d <= 256 && d % 8 == 0, CV3_EINVAL, "the head dim must be a multiple of 8, 8 to 256, not %d", d);
  CV3_REQUIRE(blocks >= 1 && blocks <= (INT32_MAX - 65536) / page, CV3_EINVAL,
              "tables of %lld blocks of %lld keys pass 2^31 keys", (long long)blocks, (long long)page);
  CV3_REQUIRE(requests >= 0, CV3_EINVAL, "negative number of requests");
  if (requests == 0) return CV3_OK;
  CV3_REQUIRE(parents && tables && own && lengths && k_cache && v_cache, CV3_EINVAL, "null operand");
  CV3_REQUIRE(((uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0, CV3_EINVAL, "the caches must be 16-byte aligned");
  const double n = (double)requests * beams,
               cache = (double)layers * pages * kv_heads * page * d * (cache_type == CV3_F32 ? 4 : 2);
  const Run in[] = {{parents, 4 * n}, {own, 4 * n * blocks}, {lengths, 4.0 * requests}};
  const Run out[] = {{tables, 4 * n * blocks}, {k_cache, cache}, {v_cache, cache}};
  CV3_REQUIRE(apart(out, in), CV3_EINVAL, "tables, caches, parents, lengths and the beams' own pages overlap");
  const int row_vecs = d * (cache_type == CV3_F32 ? 4 : 2) / 16;
  ReorderArgs a{parents, tables, own, lengths, (uint4*)k_cache, (uint4*)v_cache, pages, blocks, layers, beams, kv_heads,
                (int)page, row_vecs, (int)ceil_div(page * row_vecs, 256), (int)ceil_div(blocks, 256)};
  const int64_t per = layers * kv_heads * 2 * a.parts + a.table_parts;
  CV3_REQUIRE(requests <= 65535 && per < (1 << 24), CV3_EINVAL, "%lld requests, or pages of %lld copies, are too many for one call",
              (long long)requests, (long long)per);
  const dim3 grid((unsigned)per, (unsigned)requests), block(256);
  hipStream_t st = stream_of(s);
  if (beams <= 4) hipLaunchKernelGGL(k_beam_reorder<4>, grid, block, 0, st, a);
  else if (beams <= 8) hipLaunchKernelGGL(k_beam_reorder<8>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(k_beam_reorder<16>, grid, block, 0, st, a);
  CV3_LAUNCHED();
  return CV3_OK;
}

}  // extern "C"
