// Pages of the paged key-value cache as sequences come and go: sequences that go on from others, the list of pages
// that nobody holds any more, and the move of what is held into another cache.  The reference has one contiguous cache
// that grows and is dropped whole (KVCache, cv3cpu/models/qwen2.py:74-121).
//
// Who holds a page is told by the tables and lengths alone: sequence b holds the first ceil(lengths[b] / page) entries
// of its table.  No counts are kept beside them that could come apart from them.  Every id and length is checked where
// it is used; ids outside the cache count as absent.
#include "paged_common.hpp"

#include <algorithm>

using namespace cv3;

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));     // 16 bytes

constexpr int kForks = 4096, kForkRows = 65536;   // forks of a call, sequences of its tables
// Workgroups of a call's copies, about, and 16-byte vectors of a thread in flight: what every workgroup does before its
// copies is most of a small call.
constexpr int kForkGroups = 1024, kForkAhead = 6;
constexpr int kThreads = 256;

struct ForkArgs {
  const int32_t* parents;
  const int32_t* children;
  int32_t* tables;
  int32_t* lengths;
  const int32_t* free_pages;
  const int32_t* taken;
  int32_t* taken_out;
  u32x4* k;
  u32x4* v;
  int64_t pages, blocks, free_count, layers;
  int forks, rows, kv_heads, page, row_vecs;
};

// The keys of sequence r, and the blocks that they begin.
__device__ __forceinline__ int held_of(const int32_t* lengths, int64_t r, int64_t blocks, int page) {
  return (int)min((int64_t)max(lengths[r], 0), blocks * page);
}
__device__ __forceinline__ int live_of(const int32_t* lengths, int64_t r, int64_t blocks, int page) {
  return (int)(((uint32_t)held_of(lengths, r, blocks, page) + (uint32_t)page - 1) / (uint32_t)page);
}

// Workgroups (x, i) make fork i: all of them copy its part-filled page, the first writes its table and length.  Every
// one finds by itself which forks of the call are made and so which free page is i's: a bit a sequence says whether it
// is a parent, is named as a child, is named again.  3 forks of a sequence 5.1 us, the chain of loads that ends in a page's
// id; 112 of 16 (24 layers of 2 x 64 bfloat16, pages of 64) 18 us, 2.8 TB/s of the 50 MB that move.  Forks into a parent of the call or into a child that is named
// twice are not made, so what is read here (parents) is nowhere written (children).
__global__ __launch_bounds__(kThreads) void k_fork(ForkArgs a) {
  extern __shared__ uint32_t s_bits[];           // [3][words]
  __shared__ int s_before, s_all;
  const int words = (a.rows + 31) / 32, i = blockIdx.y, tid = threadIdx.x;
  uint32_t *parent = s_bits, *child = s_bits + words, *again = s_bits + 2 * words;
  for (int w = tid; w < 3 * words; w += kThreads) s_bits[w] = 0;
  if (tid == 0) s_before = s_all = 0;
  __syncthreads();
  // this fork's numbers and every fork's, together; the lengths of kForksEach x 256 of them at a time
  constexpr int kForksEach = 4;
  const uint32_t p = a.forks ? (uint32_t)a.parents[i] : ~0u, c = a.forks ? (uint32_t)a.children[i] : ~0u;
  const int len = p < (uint32_t)a.rows ? held_of(a.lengths, p, a.blocks, a.page) : 0, full = len / a.page, rest = len - full * a.page;
  const int32_t* from = a.tables + (int64_t)(p < (uint32_t)a.rows ? p : 0) * a.blocks;
  const int32_t source = rest ? from[full] : -1;
  uint32_t ps[kForksEach], cs[kForksEach];
  int keys[kForksEach];
  bool part[kForksEach];
  // a part-filled last page is copied, and takes a page, if it is there: of an absent one a child has no keys either
  auto last = [&](uint32_t fp, int n) {
    return n % a.page ? (uint32_t)a.tables[(int64_t)fp * a.blocks + n / a.page] : ~0u;
  };
  const bool once = a.forks <= kForksEach * kThreads;
#pragma unroll
  for (int e = 0; e < kForksEach; ++e) {
    const int f = tid + e * kThreads;
    ps[e] = f < a.forks ? (uint32_t)a.parents[f] : ~0u;
    cs[e] = f < a.forks ? (uint32_t)a.children[f] : ~0u;
  }
#pragma unroll
  for (int e = 0; e < kForksEach; ++e) keys[e] = ps[e] < (uint32_t)a.rows ? held_of(a.lengths, ps[e], a.blocks, a.page) : 0;
#pragma unroll
  for (int e = 0; e < kForksEach; ++e) part[e] = last(ps[e], keys[e]) < (uint64_t)a.pages;
  auto enter = [&](uint32_t fp, uint32_t fc) {
    if (fp < (uint32_t)a.rows) atomicOr(&parent[fp >> 5], 1u << (fp & 31));
    if (fc < (uint32_t)a.rows && atomicOr(&child[fc >> 5], 1u << (fc & 31)) >> (fc & 31) & 1)
      atomicOr(&again[fc >> 5], 1u << (fc & 31));
  };
#pragma unroll
  for (int e = 0; e < kForksEach; ++e) enter(ps[e], cs[e]);
  for (int f = tid + kForksEach * kThreads; f < a.forks; f += kThreads) enter((uint32_t)a.parents[f], (uint32_t)a.children[f]);
  __syncthreads();
  auto made = [&](uint32_t fp, uint32_t fc) {
    return fp < (uint32_t)a.rows && fc < (uint32_t)a.rows && !((parent[fc >> 5] | again[fc >> 5]) >> (fc & 31) & 1);
  };
  int before = 0, all = 0;
  auto count = [&](int f, uint32_t fp, uint32_t fc, bool takes) {
    if (takes && made(fp, fc)) {
      ++all;
      if (f < i) ++before;
    }
  };
#pragma unroll
  for (int e = 0; e < kForksEach; ++e) count(tid + e * kThreads, ps[e], cs[e], part[e]);
  if (!once)
    for (int f = tid + kForksEach * kThreads; f < a.forks; f += kThreads) {
      const uint32_t fp = (uint32_t)a.parents[f];
      const int n = fp < (uint32_t)a.rows ? held_of(a.lengths, fp, a.blocks, a.page) : 0;
      count(f, fp, (uint32_t)a.children[f], last(fp, n) < (uint64_t)a.pages);
    }
  if (before) atomicAdd(&s_before, before);
  if (all) atomicAdd(&s_all, all);
  __syncthreads();
  const int64_t taken = a.taken[0];
  if (blockIdx.x == 0 && i == 0 && tid == 0) a.taken_out[0] = (int32_t)min(taken + s_all, (int64_t)INT32_MAX);
  if (!made(p, c)) return;
  const int64_t at = taken + s_before;
  const bool takes = (uint32_t)source < (uint64_t)a.pages;
  const int32_t to = takes && at >= 0 && at < a.free_count ? a.free_pages[at] : -1;
  if (blockIdx.x == 0) {
    for (int64_t b = tid; b < a.blocks; b += kThreads)
      a.tables[(int64_t)c * a.blocks + b] = b < full ? from[b] : b == full ? to : -1;
    if (tid == 0) a.lengths[c] = len;
  }
  if (!takes || (uint32_t)to >= (uint64_t)a.pages || source == to) return;
  // rows [0, rest) of every (layer, kv head, k or v): runs that follow each other, 16 bytes a thread
  const uint32_t run = (uint32_t)rest * a.row_vecs, runs = (uint32_t)(a.layers * 2 * a.kv_heads);
  const int64_t head_vecs = (int64_t)a.page * a.row_vecs, page_vecs = head_vecs * a.kv_heads;
  const int64_t vecs = (int64_t)runs * run, step = (int64_t)gridDim.x * kThreads;
  for (int64_t x0 = (int64_t)blockIdx.x * kThreads + tid; x0 < vecs; x0 += step * kForkAhead) {
    u32x4 got[kForkAhead];
    u32x4* dst[kForkAhead];
#pragma unroll
    for (int u = 0; u < kForkAhead; ++u) {
      const int64_t x = x0 + u * step;
      dst[u] = nullptr;
      got[u] = u32x4{};
      if (x >= vecs) continue;
      const uint32_t which = vecs <= UINT32_MAX ? (uint32_t)x / run : (uint32_t)(x / run), vec = (uint32_t)(x - (int64_t)which * run);
      const uint32_t head = which >> 1, layer = head / (uint32_t)a.kv_heads;
      u32x4* base = (which & 1 ? a.v : a.k) + (int64_t)layer * a.pages * page_vecs +
                    (int64_t)(head - layer * a.kv_heads) * head_vecs + vec;
      got[u] = base[source * page_vecs];
      dst[u] = base + to * page_vecs;
    }
#pragma unroll
    for (int u = 0; u < kForkAhead; ++u)
      if (dst[u]) *dst[u] = got[u];
  }
}

// ------------------------------------------------------------------------------------------------
// which pages are held
// ------------------------------------------------------------------------------------------------

constexpr int64_t kPagesMost = 1 << 24;       // pages of a cache
constexpr int kRange = 8192;                  // pages of a workgroup of the list
constexpr int kRanges = (int)(kPagesMost / kRange);
constexpr int kListThreads = 1024;
// Up to here one launch does it: bits and lengths lie in LDS, and every workgroup goes over all entries.
constexpr int64_t kOnePages = 1 << 17, kOneEntries = 1 << 16;
constexpr int kOneRows = 4096, kOneShare = 4096;        // pages that a workgroup lists

struct HeldArgs {
  const int32_t* tables;
  const int32_t* lengths;
  uint32_t* bits;              // a bit a page: held
  int32_t* counts;             // [ranges]: pages of the range that are listed
  int32_t* list;               // those pages, ascending
  int32_t* rank;               // [pages]: a held page's place among the held; NULL: the free ones are listed, -1 behind
  int32_t* count;              // how many
  int64_t rows, blocks, pages;
  int page;
};

__device__ __forceinline__ void hold(const HeldArgs& a, uint32_t* bits, uint32_t id) {
  if (id < (uint64_t)a.pages) atomicOr(&bits[id >> 5], 1u << (id & 31));
}

// Lists the pages of [p0, p1) that are asked for, from place `at` on; `scan` is LDS, a word a wave.
template <int T>
__device__ __forceinline__ void list_range(const HeldArgs& a, const uint32_t* bits, int64_t p0, int64_t p1, int32_t at,
                                           int32_t* scan) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  constexpr int kWaves = T / 64;
  // every wave takes an equal run of 64-page steps: first how many it has, then their places
  const int64_t steps = ceil_div(p1 - p0, 64), each = ceil_div(steps, kWaves);
  const int64_t s0 = min((int64_t)wv * each, steps), s1 = min(s0 + each, steps);
  auto listed = [&](int64_t p) {
    if (p >= p1) return false;
    const bool held = bits[p >> 5] >> (p & 31) & 1;
    return held == (a.rank != nullptr);
  };
  // the run's words, a lane each: pages past p1 lie in its last word alone
  int mine = 0;
  for (int64_t w = (p0 + s0 * 64) / 32 + lane; w * 32 < min(p0 + s1 * 64, p1); w += 64) {
    const int64_t in = p1 - w * 32;
    mine += __popc((a.rank ? bits[w] : ~bits[w]) & (in >= 32 ? ~0u : (1u << in) - 1));
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mine += __shfl_xor(mine, o, kWave);
  if (lane == 0) scan[wv] = mine;
  __syncthreads();
  int32_t place = at;
  for (int w = 0; w < wv; ++w) place += scan[w];
#pragma unroll 4
  for (int64_t s = s0; s < s1; ++s) {
    const int64_t p = p0 + s * 64 + lane;
    const bool on = listed(p);
    const uint64_t mask = __ballot(on);
    const int32_t to = place + __popcll(mask & (((uint64_t)1 << lane) - 1));
    if (on) {
      a.list[to] = (int32_t)p;
      if (a.rank) a.rank[p] = to;
    }
    place += __popcll(mask);
  }
}

// Small caches, in one launch: every workgroup marks all held pages in its LDS, every entry of the tables a thread's,
// kEntriesAhead of them in flight, and lists a share of the pages.  Bound by its instructions, a dozen an entry: 8 sequences
// 4.5 us, 384 of 119 blocks 12.4 (45.7 thousand entries; 26 with one workgroup).
constexpr int kEntriesAhead = 8;
__global__ __launch_bounds__(kListThreads) void k_held_one(HeldArgs a) {
  extern __shared__ uint32_t s_bits[];
  __shared__ int32_t s_live[kOneRows];
  __shared__ int32_t s_scan[kListThreads / 64], s_before[kListThreads / 64], s_all[kListThreads / 64];
  const int words = (int)ceil_div(a.pages, 32), tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const uint32_t blocks = (uint32_t)a.blocks, entries = (uint32_t)(a.rows * a.blocks);
  for (int r = tid; r < a.rows; r += kListThreads) s_live[r] = live_of(a.lengths, r, a.blocks, a.page);
  for (int w = tid; w < words; w += kListThreads) s_bits[w] = 0;
  __syncthreads();
  const uint32_t rows_on = kListThreads / blocks, on = kListThreads - rows_on * blocks;
  uint32_t row = (uint32_t)tid / blocks, col = (uint32_t)tid - row * blocks;
  for (uint32_t e = tid; e < entries; e += kListThreads * kEntriesAhead) {
    uint32_t id[kEntriesAhead];
#pragma unroll
    for (int i = 0; i < kEntriesAhead; ++i) {
      const uint32_t at = e + i * kListThreads;
      id[i] = 0xffffffffu;
      if (at < entries && (int)col < s_live[row]) id[i] = (uint32_t)a.tables[at];
      row += rows_on, col += on;
      if (col >= blocks) ++row, col -= blocks;
    }
#pragma unroll
    for (int i = 0; i < kEntriesAhead; ++i) hold(a, s_bits, id[i]);
  }
  __syncthreads();
  // this workgroup's share, and what is listed ahead of it
  const int64_t each = ceil_div(ceil_div(a.pages, 64), gridDim.x) * 64, p0 = min((int64_t)blockIdx.x * each, a.pages);
  int before = 0, all = 0;
  for (int w = tid; w < words; w += kListThreads) {
    const int64_t in = a.pages - (int64_t)w * 32;
    const int n = __popc((a.rank ? s_bits[w] : ~s_bits[w]) & (in >= 32 ? ~0u : (1u << in) - 1));
    all += n;
    if ((int64_t)w * 32 < p0) before += n;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    before += __shfl_xor(before, o, kWave);
    all += __shfl_xor(all, o, kWave);
  }
  if (lane == 0) s_before[wv] = before, s_all[wv] = all;
  __syncthreads();
  before = all = 0;
  for (int w = 0; w < kListThreads / 64; ++w) before += s_before[w], all += s_all[w];
  list_range<kListThreads>(a, s_bits, p0, min(p0 + each, a.pages), before, s_scan);
  if (blockIdx.x == 0 && tid == 0) a.count[0] = all;
  if (!a.rank)
    for (int64_t i = max((int64_t)all, p0) + tid; i < min(p0 + each, a.pages); i += kListThreads) a.list[i] = -1;
}

__global__ __launch_bounds__(kThreads) void k_held_clear(HeldArgs a) {
  const int64_t words = ceil_div(a.pages, 32);
  for (int64_t w = (int64_t)blockIdx.x * kThreads + threadIdx.x; w < words; w += (int64_t)gridDim.x * kThreads) a.bits[w] = 0;
}
__global__ __launch_bounds__(kThreads) void k_held_mark(HeldArgs a) {       // a wave a row of the table
  const int lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * (kThreads / 64) + uniform((int)threadIdx.x >> 6); r < a.rows;
       r += (int64_t)gridDim.x * (kThreads / 64)) {
    const int live = live_of(a.lengths, r, a.blocks, a.page);
#pragma unroll 4
    for (int b = lane; b < live; b += 64) hold(a, a.bits, (uint32_t)a.tables[r * a.blocks + b]);
  }
}
__global__ __launch_bounds__(kThreads) void k_held_count(HeldArgs a) {
  __shared__ int32_t s_sum[kThreads / 64];
  const int64_t p0 = (int64_t)blockIdx.x * kRange, words = ceil_div(a.pages, 32), w = p0 / 32 + threadIdx.x;
  static_assert(kRange / 32 == kThreads, "a word a thread");
  int n = 0;
  if (w < words) {
    const int64_t in = min(a.pages - w * 32, (int64_t)32);
    const uint32_t there = in == 32 ? ~0u : (1u << in) - 1;
    n = __popc((a.rank ? a.bits[w] : ~a.bits[w]) & there);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, kWave);
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) a.counts[blockIdx.x] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
}
__global__ __launch_bounds__(kThreads) void k_held_list(HeldArgs a) {
  __shared__ int32_t s_scan[kThreads / 64], s_before[kThreads / 64], s_all[kThreads / 64];
  const int ranges = gridDim.x, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int before = 0, all = 0;
  for (int r = threadIdx.x; r < ranges; r += kThreads) {
    const int n = a.counts[r];
    all += n;
    if (r < (int)blockIdx.x) before += n;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    before += __shfl_xor(before, o, kWave);
    all += __shfl_xor(all, o, kWave);
  }
  if (lane == 0) s_before[wv] = before, s_all[wv] = all;
  __syncthreads();
  before = all = 0;
  for (int w = 0; w < kThreads / 64; ++w) before += s_before[w], all += s_all[w];
  const int64_t p0 = (int64_t)blockIdx.x * kRange, p1 = min(p0 + kRange, a.pages);
  list_range<kThreads>(a, a.bits, p0, p1, before, s_scan);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.count[0] = all;
  if (!a.rank)                                   // -1 behind the last, a share of it each
    for (int64_t i = p0 + threadIdx.x; i < p1; i += kThreads)
      if (i >= all) a.list[i] = -1;
}

// The lists of k_held_one or the four kernels; scratch for bits and counts is the caller's.
int64_t held_scratch(int64_t rows, int64_t blocks, int64_t pages) {
  if (pages <= kOnePages && rows <= kOneRows && rows * blocks <= kOneEntries) return 0;
  return 4 * (ceil_div(pages, 32) + kRanges);
}
void list_held(HeldArgs a, void* work, hipStream_t st) {
  const int64_t words = ceil_div(a.pages, 32);
  if (!work) {
    hipLaunchKernelGGL(k_held_one, dim3((unsigned)ceil_div(a.pages, kOneShare)), dim3(kListThreads), (size_t)words * 4, st, a);
    return;
  }
  a.bits = (uint32_t*)work;
  a.counts = (int32_t*)(a.bits + words);
  hipLaunchKernelGGL(k_held_clear, dim3((unsigned)std::min<int64_t>(ceil_div(words, kThreads), 1024)), dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL(k_held_mark, dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(a.rows, kThreads / 64), 2048))),
                     dim3(kThreads), 0, st, a);
  const dim3 ranges((unsigned)ceil_div(a.pages, kRange));
  hipLaunchKernelGGL(k_held_count, ranges, dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL(k_held_list, ranges, dim3(kThreads), 0, st, a);
}

// ------------------------------------------------------------------------------------------------
// the move
// ------------------------------------------------------------------------------------------------

struct MoveArgs {
  const int32_t* tables;
  const int32_t* lengths;
  int32_t* tables_new;
  const int32_t* list;
  const int32_t* rank;
  const int32_t* used;
  const u32x4* k;
  const u32x4* v;
  u32x4* k_new;
  u32x4* v_new;
  int64_t rows, blocks, pages, pages_new, layers, page_vecs;
  int page, table_groups, most;      // most: pages that may be held
};

// The first table_groups workgroups turn the tables, the others copy: a wave a run of one page in one layer, its K or V.
// Bound by HBM where there is much: 48 sequences, 371 MB of reads and writes, 66.6 us, 5.6 TB/s; 4 of them 7.
constexpr int kMoveAhead = 8;
__global__ __launch_bounds__(kThreads) void k_move_pages(MoveArgs a) {
  const int lane = threadIdx.x & 63, wv = uniform((int)threadIdx.x >> 6);
  constexpr int kWaves = kThreads / 64;
  if ((int)blockIdx.x < a.table_groups) {
    for (int64_t r = (int64_t)blockIdx.x * kWaves + wv; r < a.rows; r += (int64_t)a.table_groups * kWaves) {
      const int live = live_of(a.lengths, r, a.blocks, a.page);
      for (int64_t b = lane; b < a.blocks; b += 64) {
        int32_t id = -1;
        if (b < live) {
          const uint32_t old = (uint32_t)a.tables[r * a.blocks + b];
          if (old < (uint64_t)a.pages) id = a.rank[old];
          if (id >= a.pages_new) id = -1;
        }
        a.tables_new[r * a.blocks + b] = id;
      }
    }
    return;
  }
  // a wave a (plane, page): as many pages as there may be, so that the list is read beside its length
  const uint32_t at = (blockIdx.x - a.table_groups) * kWaves + wv, plane = at / (uint32_t)a.most;
  const int64_t to = at - plane * (uint32_t)a.most, layer = plane >> 1;
  if (layer >= a.layers) return;
  const int64_t n = min((int64_t)a.used[0], a.pages_new), from = a.list[to];
  if (to >= n) return;
  const u32x4* src = (plane & 1 ? a.v : a.k) + (layer * a.pages + from) * a.page_vecs;
  u32x4* dst = (plane & 1 ? a.v_new : a.k_new) + (layer * a.pages_new + to) * a.page_vecs;
  for (int64_t x0 = lane; x0 < a.page_vecs; x0 += 64 * kMoveAhead) {
    u32x4 got[kMoveAhead];
#pragma unroll
    for (int i = 0; i < kMoveAhead; ++i) got[i] = src[min(x0 + 64 * i, a.page_vecs - 1)];
#pragma unroll
    for (int i = 0; i < kMoveAhead; ++i)
      if (x0 + 64 * i < a.page_vecs) dst[x0 + 64 * i] = got[i];
  }
}

// What calls on tables check.
int check_tables(int64_t rows, int64_t blocks, int64_t page) {
  CV3_REQUIRE(page >= 1 && page <= 65536, CV3_EINVAL, "a page holds 1 to 65536 keys, not %lld", (long long)page);
  CV3_REQUIRE(blocks >= 1 && blocks <= (INT32_MAX - 65536) / page, CV3_EINVAL,
              "tables of %lld blocks of %lld keys pass 2^31 keys", (long long)blocks, (long long)page);
  CV3_REQUIRE(rows >= 0 && rows <= INT32_MAX, CV3_EINVAL, "bad number of sequences: %lld", (long long)rows);
  return CV3_OK;
}

}  // namespace

extern "C" {

int cv3_paged_fork(const int32_t* parents, const int32_t* children, int64_t forks, int32_t* tables, int64_t rows,
                   int64_t blocks, int32_t* lengths, const int32_t* free_pages, int64_t free_count,
                   const int32_t* taken, int32_t* taken_out, int cache_type, void* k_cache, void* v_cache,
                   int64_t layers, int64_t pages, int kv_heads, int64_t page, int d, cv3_stream_t s) {
  CV3_ALIVE();
  if (int rc = check_cache(cache_type, k_cache, v_cache, pages, page, kv_heads, d)) return rc;
  if (int rc = check_tables(rows, blocks, page)) return rc;
  CV3_REQUIRE(layers >= 1 && layers <= 65536, CV3_EINVAL, "1 to 65536 layers, not %lld", (long long)layers);
  CV3_REQUIRE(forks >= 0 && forks <= kForks, CV3_EINVAL, "at most %d forks a call, not %lld", kForks, (long long)forks);
  CV3_REQUIRE(rows <= kForkRows, CV3_EINVAL, "at most %d sequences, not %lld", kForkRows, (long long)rows);
  CV3_REQUIRE(free_count >= 0 && free_count <= INT32_MAX, CV3_EINVAL, "bad number of free pages");
  CV3_REQUIRE(taken && taken_out && (free_pages || free_count == 0) &&
                  (forks == 0 || (parents && children && tables && lengths)), CV3_EINVAL, "null operand");
  const double cache = (double)layers * pages * kv_heads * page * d * elem_size(cache_type), n = (double)rows;
  const Run in[] = {{parents, 4.0 * forks}, {children, 4.0 * forks}, {free_pages, 4.0 * free_count}, {taken, 4}};
  const Run out[] = {{tables, 4 * n * blocks}, {lengths, 4 * n}, {taken_out, 4}, {k_cache, cache}, {v_cache, cache}};
  CV3_REQUIRE(apart(out, in), CV3_EINVAL, "tables, lengths, caches and the count of pages overlap each other or the inputs");
  const int row_vecs = d * elem_size(cache_type) / 16;
  ForkArgs a{parents, children, tables, lengths, free_pages, taken, taken_out, (u32x4*)k_cache, (u32x4*)v_cache, pages,
             blocks, free_count, layers, (int)forks, (int)rows, kv_heads, (int)page, row_vecs};
  CV3_REQUIRE((double)layers * 2 * kv_heads < 2147483648.0, CV3_EINVAL, "bad cache shape");
  // at least one workgroup, so that the pages taken are passed on
  const int64_t vecs = layers * 2 * kv_heads * page * row_vecs, count = std::max<int64_t>(forks, 1);
  // where it may be, a multiple of the XCDs: children of one parent then find its rows in their L2 (84 forks of 12 parents,
  // 24 layers of 2 x 80 float32, 23 us with 13 workgroups each, 19 with 16)
  const int64_t share = std::max<int64_t>(1, kForkGroups / count);
  const int64_t each = std::max<int64_t>(1, std::min(ceil_div(vecs, kThreads * kForkAhead), share >= 8 ? (share + 4) / 8 * 8 : share));
  if (forks == 0) a.rows = 0;
  hipLaunchKernelGGL(k_fork, dim3((unsigned)each, (unsigned)count), dim3(kThreads), (size_t)3 * ((a.rows + 31) / 32) * 4,
                     stream_of(s), a);
  CV3_LAUNCHED();
  return CV3_OK;
}

int cv3_paged_free(const int32_t* tables, int64_t rows, int64_t blocks, const int32_t* lengths, int64_t page,
                   int64_t pages, int32_t* free_pages, int32_t* count, cv3_stream_t s) {
  CV3_ALIVE();
  if (int rc = check_tables(rows, blocks, page)) return rc;
  CV3_REQUIRE(pages >= 1 && pages <= kPagesMost, CV3_EINVAL, "1 to %lld pages, not %lld", (long long)kPagesMost,
              (long long)pages);
  CV3_REQUIRE(free_pages && count && (rows == 0 || (tables && lengths)), CV3_EINVAL, "null operand");
  const double n = (double)rows;
  const Run in[] = {{tables, 4 * n * blocks}, {lengths, 4 * n}};
  const Run out[] = {{free_pages, 4.0 * pages}, {count, 4}};
  CV3_REQUIRE(apart(out, in), CV3_EINVAL, "results that overlap each other, the tables or the lengths");
  hipStream_t st = stream_of(s);
  void* work = nullptr;
  if (const int64_t bytes = held_scratch(rows, blocks, pages))
    if (int rc = scratch_alloc(&work, (size_t)bytes, st)) return rc;
  list_held(HeldArgs{tables, lengths, nullptr, nullptr, free_pages, nullptr, count, rows, blocks, pages, (int)page}, work, st);
  const hipError_t err = hipGetLastError();
  const int rc = work ? scratch_free(work, st) : CV3_OK;
  CV3_REQUIRE(err == hipSuccess, CV3_EHIP, "kernel launch failed: %s", hipGetErrorString(err));
  return rc;
}

int cv3_paged_compact(const int32_t* tables, int64_t rows, int64_t blocks, const int32_t* lengths, int cache_type,
                      const void* k_cache, const void* v_cache, int64_t layers, int64_t pages, int kv_heads,
                      int64_t page, int d, void* k_new, void* v_new, int64_t pages_new, int32_t* tables_new,
                      int32_t* used, cv3_stream_t s) {
  CV3_ALIVE();
  if (int rc = check_cache(cache_type, k_cache, v_cache, pages, page, kv_heads, d)) return rc;
  if (int rc = check_cache(cache_type, k_new, v_new, pages_new, page, kv_heads, d)) return rc;
  if (int rc = check_tables(rows, blocks, page)) return rc;
  CV3_REQUIRE(layers >= 1 && layers <= 65536, CV3_EINVAL, "1 to 65536 layers, not %lld", (long long)layers);
  CV3_REQUIRE(pages <= kPagesMost, CV3_EINVAL, "at most %lld pages, not %lld", (long long)kPagesMost, (long long)pages);
  CV3_REQUIRE(used && (rows == 0 || (tables && lengths && tables_new)), CV3_EINVAL, "null operand");
  const int row_vecs = d * elem_size(cache_type) / 16;
  const double n = (double)rows, one = 16.0 * layers * kv_heads * page * row_vecs;
  const Run in[] = {{tables, 4 * n * blocks}, {lengths, 4 * n}, {k_cache, one * pages}, {v_cache, one * pages}};
  const Run out[] = {{tables_new, 4 * n * blocks}, {used, 4}, {k_new, one * pages_new}, {v_new, one * pages_new}};
  CV3_REQUIRE(apart(out, in), CV3_EINVAL, "the new cache, its tables and their count overlap each other or what is read");
  CV3_REQUIRE((double)std::min({(double)pages, (double)pages_new, n * blocks}) * layers * 2 / 4 < kLaunchBlocks, CV3_EINVAL,
              "%lld pages of %lld layers are too many for one call", (long long)pages, (long long)layers);
  hipStream_t st = stream_of(s);
  const int64_t bits = held_scratch(rows, blocks, pages);
  void* work = nullptr;
  if (int rc = scratch_alloc(&work, (size_t)(8 * pages + bits), st)) return rc;
  int32_t *list = (int32_t*)work, *rank = list + pages;
  list_held(HeldArgs{tables, lengths, nullptr, nullptr, list, rank, used, rows, blocks, pages, (int)page},
            bits ? (void*)(rank + pages) : nullptr, st);
  const int64_t most = std::min({pages, pages_new, rows * blocks});       // pages to copy; the list is as long as the cache
  const int64_t copies = ceil_div(most * layers * 2, kThreads / 64), tables_by = std::min<int64_t>(ceil_div(rows, kThreads / 64), 256);
  MoveArgs a{tables, lengths, tables_new, list, rank, used, (const u32x4*)k_cache, (const u32x4*)v_cache, (u32x4*)k_new,
             (u32x4*)v_new, rows, blocks, pages, pages_new, layers, kv_heads * page * row_vecs, (int)page, (int)tables_by, (int)most};
  if (copies + tables_by > 0)
    hipLaunchKernelGGL(k_move_pages, dim3((unsigned)(copies + tables_by)), dim3(kThreads), 0, st, a);
  const hipError_t err = hipGetLastError();
  const int rc = scratch_free(work, st);
  CV3_REQUIRE(err == hipSuccess, CV3_EHIP, "kernel launch failed: %s", hipGetErrorString(err));
  return rc;
}

}  // extern "C"
