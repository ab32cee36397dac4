// The paged key-value cache: block tables and slots from request lengths, rotary with the cache
// write, and the attention of one new token per sequence over the cache.  It is the form for
// several sequences of what the reference holds for one (KVCache, cv3cpu/models/qwen2.py:74-121;
// apply_rope, qwen2.py:64-71; sdpa at one query, cv3cpu/ops.py:267-300).
//
// A cache is [pages, kv_heads, page, d]: the rows of one head in one page are one contiguous run.
// Key j of sequence b lies in page tables[b][j / page], row j % page.  Offsets are 64-bit; page
// ids, lengths and slots come from device memory, so every one is checked against its bounds
// where it is used, and what lies outside counts as absent.
#include "bf16x3.hpp"
#include "paged_common.hpp"

#include <algorithm>

using namespace cv3;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
// 16 bytes at any 4-byte boundary
struct __attribute__((packed, aligned(4))) f32x4u {
  float v[4];
};

__device__ __forceinline__ uint16_t bf16_bits(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }

// ------------------------------------------------------------------------------------------------
// block tables
// ------------------------------------------------------------------------------------------------

constexpr int kTabThreads = 256, kTabEach = 4;   // requests and tokens of a thread at a time
constexpr int kTabRequests = 4096;               // a call's requests: two int32 of LDS each

struct TabArgs {
  const int32_t* lengths;
  const int32_t* fresh;
  const int32_t* free_pages;
  const int32_t* taken;
  int32_t* tables;
  int32_t* total;
  int32_t* taken_out;
  int32_t* starts;
  int64_t* slots;
  int32_t* positions;
  int64_t free_count;
  int requests, page, blocks, tokens;
};

// Sum over the threads before this one, at most 2^32 - 1; *all receives the sum of all of them.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* red, uint32_t* all) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  uint32_t up = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = __shfl_up(up, o, kWave);
    if (lane >= o) up = __builtin_elementwise_add_sat(up, u);
  }
  __syncthreads();
  if (lane == 63) red[wid] = up;
  __syncthreads();
  uint32_t before = __shfl_up(up, 1, kWave), sum = 0;
  if (lane == 0) before = 0;
#pragma unroll
  for (int i = 0; i < kTabThreads / 64; ++i) {
    const uint32_t r = red[i];
    if (i < wid) before = __builtin_elementwise_add_sat(before, r);
    sum = __builtin_elementwise_add_sat(sum, r);
  }
  *all = sum;
  return before;
}

// Every workgroup sums over the requests by itself (a few kilobytes from L2, no wait between
// workgroups), then lists a share of the tokens, four neighbours a thread.  A token finds its request
// among the starts in LDS; the token that opens a page also enters it into the table.  Pages before
// `have` are the request's own already; page have + i is free_pages[first + i].  Bound by the chain of
// its loads: 5.0 us for a decode step of eight requests, 7.9 us for 384 prompts of up to 1200 tokens.
__global__ __launch_bounds__(kTabThreads) void k_block_tables(TabArgs a) {
  __shared__ int32_t s_start[kTabRequests + 1];
  __shared__ int32_t s_first[kTabRequests];   // index of the request's first new page among the free ones
  __shared__ uint32_t s_red[kTabThreads / 64];
  const uint32_t page = (uint32_t)a.page, cap = (uint32_t)a.blocks * page, most = (uint32_t)a.tokens;
  const bool reserved = !a.free_pages;        // the tables hold every page already
  const int64_t taken = reserved ? 0 : a.taken[0];
  uint32_t tok = 0, pages = 0;                // of the requests so far; tok at most `most`
  for (int r0 = 0; r0 < a.requests; r0 += kTabThreads * kTabEach) {
    const int r = r0 + (int)threadIdx.x * kTabEach;
    uint32_t held[kTabEach], want[kTabEach], sum = 0, all;
#pragma unroll
    for (int i = 0; i < kTabEach; ++i) {
      held[i] = r + i < a.requests ? (uint32_t)max(a.lengths[r + i], 0) : 0;
      const uint32_t fresh = r + i < a.requests ? (uint32_t)max(a.fresh[r + i], 0) : 0;
      want[i] = min(fresh, held[i] < cap ? cap - held[i] : 0);
      sum = __builtin_elementwise_add_sat(sum, want[i]);
    }
    // the tokens that a call may list go to the first requests: the running sums, cut at that number
    uint32_t at = __builtin_elementwise_add_sat(tok, block_scan(sum, s_red, &all));
    tok = min(__builtin_elementwise_add_sat(tok, all), most);
    uint32_t start[kTabEach], now[kTabEach], need[kTabEach], more = 0;
#pragma unroll
    for (int i = 0; i < kTabEach; ++i) {
      start[i] = min(at, most);
      at = __builtin_elementwise_add_sat(at, want[i]);
      now[i] = held[i] + (min(at, most) - start[i]);
      need[i] = reserved ? 0 : (now[i] + page - 1) / page - (held[i] + page - 1) / page;
      more += need[i];
    }
    uint32_t upto = pages + block_scan(more, s_red, &all);
    pages += all;
#pragma unroll
    for (int i = 0; i < kTabEach; ++i) {
      if (r + i < a.requests) {
        s_start[r + i] = (int32_t)start[i];
        s_first[r + i] = (int32_t)min(taken + upto, (int64_t)INT32_MAX);
        if (blockIdx.x == 0) {
          a.starts[r + i] = (int32_t)start[i];
          a.total[r + i] = (int32_t)now[i];
        }
      }
      upto += need[i];
    }
  }
  if (threadIdx.x == 0) s_start[a.requests] = (int32_t)tok;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.starts[a.requests] = (int32_t)tok;
    if (!reserved) a.taken_out[0] = (int32_t)min(taken + pages, (int64_t)INT32_MAX);
  }
  __syncthreads();
  for (int64_t t0 = ((int64_t)blockIdx.x * kTabThreads + threadIdx.x) * kTabEach; t0 < a.tokens;
       t0 += (int64_t)gridDim.x * kTabThreads * kTabEach) {
    struct __attribute__((packed, aligned(4))) Out {
      int64_t slot[kTabEach];
    } out;
    struct __attribute__((packed, aligned(4))) Pos {
      int32_t pos[kTabEach];
    } where;
    int r = 0, top = a.requests;       // the last request that starts at or before t0: those without tokens lie before it
    while (t0 < tok && top - r > 1) {
      const int mid = (r + top) >> 1;
      if (s_start[mid] <= t0) r = mid; else top = mid;
    }
#pragma unroll
    for (int i = 0; i < kTabEach; ++i) {
      const int64_t t = t0 + i;
      out.slot[i] = -1;
      where.pos[i] = -1;
      if (t >= tok) continue;
      while (s_start[r + 1] <= t) ++r;         // ends: tok, behind the last request, is past t
      const uint32_t held = (uint32_t)max(a.lengths[r], 0), pos = held + (uint32_t)(t - s_start[r]);
      const uint32_t block = pos / page, row = pos - block * page, have = (held + page - 1) / page;
      int32_t* entry = a.tables + (int64_t)r * a.blocks + block;
      int32_t id;
      if (block < have || reserved) {
        id = *entry;
      } else {
        const int64_t n = (int64_t)s_first[r] + (block - have);
        id = n >= 0 && n < a.free_count ? a.free_pages[n] : -1;
        if (row == 0) *entry = id;
      }
      if (id >= 0) out.slot[i] = (int64_t)id * page + row;
      where.pos[i] = (int32_t)pos;
    }
    if (t0 + kTabEach <= a.tokens) {
      *(Out*)(a.slots + t0) = out;
      *(Pos*)(a.positions + t0) = where;
    } else {
#pragma unroll
      for (int i = 0; i < kTabEach; ++i)
        if (t0 + i < a.tokens) {
          a.slots[t0 + i] = out.slot[i];
          a.positions[t0 + i] = where.pos[i];
        }
    }
  }
}

// ------------------------------------------------------------------------------------------------
// rotary and cache write
// ------------------------------------------------------------------------------------------------

struct AppendArgs {
  const float* rows;
  int64_t n, ld;
  const int32_t* positions;
  const int64_t* slots;
  const float* cos_tab;
  const float* sin_tab;
  int64_t rope_rows;
  void* k;
  void* v;
  int64_t slot_count;
  float* q;
  int64_t ldq;
  int page, heads, kv_heads, d;
};

template <int V, bool PAST>
__device__ __forceinline__ void store_elems(void* base, int type, int64_t at, const float* x) {
  if (type == CV3_F32) {
    float* p = (float*)base + at;
    if constexpr (V == 4) {
      const f32x4 v = {x[0], x[1], x[2], x[3]};
      if constexpr (PAST) __builtin_nontemporal_store(v, (f32x4*)p);
      else *(f32x4*)p = v;
    } else {
      p[0] = x[0];
    }
    return;
  }
  uint16_t b[V];
#pragma unroll
  for (int i = 0; i < V; ++i)
    b[i] = type == CV3_F16 ? __builtin_bit_cast(uint16_t, (_Float16)x[i]) : bf16_bits(x[i]);
  uint16_t* p = (uint16_t*)base + at;
  if constexpr (V == 4)
    *(uint2*)p = make_uint2((uint32_t)b[0] | (uint32_t)b[1] << 16, (uint32_t)b[2] | (uint32_t)b[3] << 16);
  else p[0] = b[0];
}

// One thread per V channels j.. of a head's first half and the V at j + d/2 that rotate with them:
// out[j] = x[j] cos[j] - x[j + d/2] sin[j], out[j + d/2] = x[j + d/2] cos[j + d/2] + x[j] sin[j + d/2].
// HBM-bound: each row is read once, q written in float32, k and v rounded (to nearest even) to the
// cache's type as they are written.  PAST: rows and q go past the caches, for calls that move more
// than the 256 MB of the last one (6001 tokens of 32 + 2 x 8 heads of 128, bfloat16, 272 MB: 46.7 us,
// 5.8 TB/s, against 50.2).
template <int V, bool PAST>
__global__ __launch_bounds__(256) void k_append(AppendArgs a, int type, unsigned per_row, unsigned blocks_per_row) {
  const int64_t n = blockIdx.x / blocks_per_row;
  const unsigned item = (blockIdx.x % blocks_per_row) * blockDim.x + threadIdx.x;
  if (item >= per_row) return;
  const int half = a.d / 2;
  const unsigned per_head = half / V;
  const int head = item / per_head, j = (int)(item % per_head) * V;
  const int64_t pos = a.positions ? a.positions[n] : 0;
  const bool turns = a.cos_tab && head < a.heads + a.kv_heads;
  const bool placed = !a.cos_tab || (pos >= 0 && pos < a.rope_rows);
  const float* src = a.rows + n * a.ld + (int64_t)head * a.d + j;
  float x[V], y[V], u[V], w[V];
  if constexpr (V == 4) {
    f32x4 lo, hi;
    if constexpr (PAST) {
      lo = __builtin_nontemporal_load((const f32x4*)src);
      hi = __builtin_nontemporal_load((const f32x4*)(src + half));
    } else {
      lo = *(const f32x4*)src;
      hi = *(const f32x4*)(src + half);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = lo[i], y[i] = hi[i];
  } else {
    x[0] = src[0];
    y[0] = src[half];
  }
#pragma unroll
  for (int i = 0; i < V; ++i) u[i] = x[i], w[i] = y[i];
  if (turns && placed) {
    const float* c = a.cos_tab + pos * a.d + j;
    const float* s = a.sin_tab + pos * a.d + j;
    struct __attribute__((packed, aligned(4))) Vec {
      float v[V];
    };
    const Vec c0 = *(const Vec*)c, c1 = *(const Vec*)(c + half), s0 = *(const Vec*)s, s1 = *(const Vec*)(s + half);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      u[i] = x[i] * c0.v[i] + (-y[i]) * s0.v[i];
      w[i] = y[i] * c1.v[i] + x[i] * s1.v[i];
    }
  }
  if (head < a.heads) {
    if (!a.q) return;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      u[i] = placed ? u[i] : 0.f;
      w[i] = placed ? w[i] : 0.f;
    }
    float* dst = a.q + n * a.ldq + (int64_t)head * a.d + j;
    store_elems<V, PAST>(dst, CV3_F32, 0, u);
    store_elems<V, PAST>(dst, CV3_F32, half, w);
    return;
  }
  const int64_t slot = a.slots[n];
  if (!placed || slot < 0 || slot >= a.slot_count) return;
  const int64_t id = a.slot_count <= INT32_MAX ? (uint32_t)slot / (uint32_t)a.page : slot / a.page;
  const int h = head - a.heads, kv = h % a.kv_heads;
  void* cache = h < a.kv_heads ? a.k : a.v;
  const int64_t at = ((id * a.kv_heads + kv) * a.page + (slot - id * a.page)) * a.d + j;
  store_elems<V, PAST>(cache, type, at, u);
  store_elems<V, PAST>(cache, type, at + half, w);
}

// ------------------------------------------------------------------------------------------------
// attention of one new token per sequence
// ------------------------------------------------------------------------------------------------

constexpr int kTile = 64;       // keys of a work unit
constexpr int kStrip = 16;      // keys that one wave multiplies at a time
constexpr int kWaves = 4;       // of an attention workgroup
// Workgroups of the split form: two a CU are all resident at once, and fewer parts are left to join than
// with more (3 x 100001 float16 keys: 39 us with 512, 37 with 768, 45 with 1024; 96 ragged
// sequences in bfloat16, 32 on 8 heads of 128: 236 us with 512, 250 with 768, 233 with 1024).
constexpr int kGroups = 512;
constexpr int64_t kWholeBytes = 192 << 10;

struct AttnArgs {
  const float* q;
  int64_t ldq;
  const void* k;
  const void* v;
  const int32_t* tables;
  const int32_t* lengths;
  const int32_t* starts;
  float* out;
  int64_t ldo;
  float* part;                  // [2 groups][heads of a tile][d + 2]: o, m, l
  int2* pairs;                  // [batch][kv heads][head tiles]
  int64_t pages, blocks;
  int batch, page, heads, kv_heads, group, gtiles, htile, d, groups;
  float scale;                  // times log2(e)
};

// What of sequence b is seen: keys [lo, hi), and how many 64-key units hold them.
struct Span {
  int lo, hi, tiles;
};

__device__ __forceinline__ Span span_of(const AttnArgs& a, int b) {
  Span s{0, 0, 0};
  if (b >= a.batch) return s;
  const int64_t cap = a.blocks * a.page;
  s.hi = (int)min((int64_t)max(a.lengths[b], 0), cap);
  s.lo = a.starts ? min(max(a.starts[b], 0), s.hi) : 0;
  s.tiles = s.hi > s.lo ? (s.hi + kTile - 1) / kTile - s.lo / kTile : 0;
  return s;
}

__device__ __forceinline__ Span uniform_span(const AttnArgs& a, int b) {
  const Span s = span_of(a, b);
  return Span{uniform(s.lo), uniform(s.hi), uniform(s.tiles)};
}

// A workgroup's share of the units: [at, end) of them, the first in sequence b, `before` units of
// one head ahead of that sequence.  n workgroups have a share.
struct Share {
  int64_t units, at, end, before;
  int n, b;
};

__device__ __forceinline__ int64_t wave_scan(int64_t v) {      // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t u = __shfl_up(v, o, kWave);
    if (lane >= o) v += u;
  }
  return v;
}

// Every wave finds its workgroup's share by itself: a lane sums a 64th of the sequences, the lane
// that holds the share's first unit is found, then the sequence among that lane's.
__device__ __forceinline__ Share share_of(const AttnArgs& a, int w) {
  const int lane = threadIdx.x & 63, per = a.kv_heads * a.gtiles, each = (a.batch + 63) / 64;
  Share s{};
  int64_t mine = 0;
#pragma unroll 4
  for (int i = 0; i < each; ++i) mine += span_of(a, lane * each + i).tiles;
  int64_t up = wave_scan(mine);
  s.units = uniform(__shfl(up, 63, kWave)) * per;
  s.n = (int)min((int64_t)a.groups, s.units);
  if (w >= s.n) return s;
  s.at = s.units * w / s.n;
  s.end = s.units * (w + 1) / s.n;
  const int64_t want = s.at / per;
  int from = __ffsll((unsigned long long)__ballot(want < up)) - 1;     // the first lane that passes it
  s.before = uniform(__shfl(up - mine, from, kWave));
  s.b = uniform(from) * each;
  for (int i = 0; each > 1 && i < each; i += 64) {
    const int64_t t = i + lane < each ? span_of(a, s.b + i + lane).tiles : 0;
    up = s.before + wave_scan(t);
    const uint64_t hit = __ballot(want < up);
    from = hit ? __ffsll((unsigned long long)hit) - 1 : 63;
    s.before = uniform(__shfl(hit ? up - t : up, from, kWave));
    if (hit) {
      s.b += i + uniform(from);
      break;
    }
  }
  return s;
}

template <typename E>
struct Elem;
template <>
struct Elem<float> {
  typedef uint4 VRaw;
  static __device__ __forceinline__ void wide(const uint4& r, float* f) {
    f[0] = __uint_as_float(r.x), f[1] = __uint_as_float(r.y), f[2] = __uint_as_float(r.z), f[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ void four(const uint4& r, float* f) { wide(r, f); }
};
template <>
struct Elem<_Float16> {
  typedef uint2 VRaw;
  static __device__ __forceinline__ void two(uint32_t r, float* f) {
    f[0] = (float)__builtin_bit_cast(_Float16, (uint16_t)r);
    f[1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(r >> 16));
  }
  static __device__ __forceinline__ void wide(const uint4& r, float* f) {
    two(r.x, f), two(r.y, f + 2), two(r.z, f + 4), two(r.w, f + 6);
  }
  static __device__ __forceinline__ void four(const uint2& r, float* f) { two(r.x, f), two(r.y, f + 2); }
};
template <>
struct Elem<__bf16> {
  typedef uint2 VRaw;
  static __device__ __forceinline__ void two(uint32_t r, float* f) {
    f[0] = __uint_as_float(r << 16);
    f[1] = __uint_as_float(r & 0xffff0000u);
  }
  static __device__ __forceinline__ void wide(const uint4& r, float* f) {
    two(r.x, f), two(r.y, f + 2), two(r.z, f + 4), two(r.w, f + 6);
  }
  static __device__ __forceinline__ void four(const uint2& r, float* f) { two(r.x, f), two(r.y, f + 2); }
};

// What one wave has of up to 16 query heads: lane (g, m) = (lane / 16, lane % 16) holds head m's
// channels d = 64 jj + 16 g + 4 r + c in o[jj][c][r], its running maximum, and its keys' part of the sum.
template <int NJ>
struct Wave {
  f32x4 o[NJ][4];
  float top, sum;

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[j][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    top = -INFINITY;
    sum = 0.f;
  }
};

// The keys that one workgroup looks at for one kv head: strips [.., s1) of 16.
template <typename E, int NJ, bool FULL>
struct Keys {
  typedef typename Elem<E>::VRaw VRaw;
  static constexpr int KC = 16 / sizeof(E);        // channels of a lane's 16 bytes
  static constexpr int NK = 64 * NJ / (4 * KC);    // such loads a key row
  const int32_t* table;
  const E* k;
  const E* v;
  int64_t stride;
  uint32_t pages, page;
  int d, lo, hi, s1, m, g;

  __device__ __forceinline__ Keys(const AttnArgs& a, int b, int kvh, const Span& sp, int end) {
    const int lane = threadIdx.x & 63;
    m = lane & 15, g = lane >> 4;
    d = FULL ? 64 * NJ : a.d;
    table = a.tables + (int64_t)b * a.blocks;
    k = (const E*)a.k + (int64_t)kvh * a.page * d;
    v = (const E*)a.v + (int64_t)kvh * a.page * d;
    stride = (int64_t)a.kv_heads * a.page;
    pages = (uint32_t)a.pages, page = (uint32_t)a.page;
    lo = sp.lo, hi = sp.hi, s1 = end;
  }
  // Offset of key 16 s + m in the cache, -1 where there is none to see.
  __device__ __forceinline__ int64_t locate(int s) const {
    const int key = s * kStrip + m;
    if (s >= s1 || key < lo || key >= hi) return -1;
    const uint32_t blk = (uint32_t)key / page;
    const int32_t id = table[blk];
    if ((uint32_t)id >= pages) return -1;
    return ((int64_t)id * stride + ((uint32_t)key - blk * page)) * d;
  }
  // Key row m, the lane's 16 bytes of each 64 (a key that is not there reads the first page's row).
  __device__ __forceinline__ void load_k(int64_t off, uint4 (&r)[NK]) const {
    const E* p = k + max(off, (int64_t)0) + KC * g;
#pragma unroll
    for (int j = 0; j < NK; ++j) r[j] = FULL || 4 * KC * j + KC * g < d ? *(const uint4*)(p + 4 * KC * j) : uint4{};
  }
  // Rows of keys 4g .. 4g + 3, channels 64 jj + 4 m ..; ov: their offsets.
  __device__ __forceinline__ void load_v(int64_t off, VRaw (&r)[4][NJ], int64_t (&ov)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ov[i] = __shfl(off, 4 * g + i, kWave);
      const E* p = v + max(ov[i], (int64_t)0) + 4 * m;
#pragma unroll
      for (int j = 0; j < NJ; ++j) r[i][j] = FULL || 64 * j + 4 * m < d ? *(const VRaw*)(p + 64 * j) : VRaw{};
    }
  }
};

// The query's channels from c on, times scale * log2(e); zeros past the head's and for heads that are not there.
template <int N, bool FULL>
__device__ __forceinline__ void load_q(const AttnArgs& a, const float* q, bool on, int c, int d, float* f) {
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    f32x4u x{};
    if (on && (FULL || c + e < d)) x = *(const f32x4u*)(q + c + e);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[e + i] = x.v[i] * a.scale;
  }
}

// The running maximum moves only when a score passes it by more than 2^slack: with 8, weights stay below
// 2^8, and float32 sums lose nothing by it but their top eight powers of two.  Returns the factor for
// what has been summed (1: nothing moved).
__device__ __forceinline__ float raise(float mx, float& top, float slack) {
  if (!__any(!(mx <= top + slack) && mx != -INFINITY)) return 1.f;   // NaN scores too: they reach the output
  float t = fmaxf(mx, __shfl_xor(mx, 16, kWave));
  t = fmaxf(fmaxf(t, __shfl_xor(t, 32, kWave)), top);
  const float f = weight_of(top, t);
  top = t;
  return f;
}

// Whether what a wave has summed, for the heads that there are, is finite and small enough for the sums of
// hundreds of waves.
template <int NJ>
__device__ __forceinline__ bool in_bounds(const Wave<NJ>& w, bool on) {
  bool bad = !(w.sum < 0x1p110f);
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) bad = bad || !(fabsf(w.o[j][c][r]) < 0x1p110f);
  return !__any(on && bad);
}

// Strips s, s + NW, .. on the float32 matrix cores, whatever the cache's type: 16x16x4 products take
// 1024 cycles a strip at d = 64, room for 19 TB/s of float32 cache, so HBM bounds it for one query
// head a kv head as for sixteen.  Scores are formed as K . q^T, so that lane (g, m) holds those of keys
// 4g .. 4g + 3 and head m.  That is also where V^T . P^T wants its second operand: step i takes keys
// {i, 4 + i, 8 + i, 12 + i}, lane (g, m) its own p[i].  Nothing goes through LDS or across lanes.  K is
// loaded in the first operand's layout with the sum over channels permuted so that a lane's share
// is 16 contiguous bytes, V with the output channels permuted alike (64 jj + 4 m + c in tile (jj, c)).
template <typename E, int NJ, bool FULL, int NW>
__device__ __forceinline__ void strips_f32(const AttnArgs& a, const Keys<E, NJ, FULL>& keys, const float* q, bool on,
                                           int s, float slack, Wave<NJ>& w) {
  typedef Keys<E, NJ, FULL> K;
  float qf[K::NK * K::KC];
#pragma unroll
  for (int j = 0; j < K::NK; ++j)
    load_q<K::KC, FULL>(a, q, on, 4 * K::KC * j + K::KC * keys.g, keys.d, qf + j * K::KC);
  uint4 kr[K::NK];
  typename K::VRaw vr[4][NJ];
  int64_t ov[4];
  w.clear();
  int64_t off = keys.locate(s), next = keys.locate(s + NW);
  keys.load_k(off, kr);
  keys.load_v(off, vr, ov);
  for (; s < keys.s1; s += NW) {
    // scores of this strip; then its K registers take the next one's rows
    f32x4 sc{0.f, 0.f, 0.f, 0.f}, sc1{0.f, 0.f, 0.f, 0.f};     // two chains: shorter, and the rounding less
#pragma unroll
    for (int j = 0; j < K::NK; ++j) {
      float kf[K::KC];
      Elem<E>::wide(kr[j], kf);
#pragma unroll
      for (int e = 0; e < K::KC; e += 2) {
        sc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], qf[j * K::KC + e], sc, 0, 0, 0);
        sc1 = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e + 1], qf[j * K::KC + e + 1], sc1, 0, 0, 0);
      }
    }
    sc += sc1;
    keys.load_k(next, kr);
    const int64_t after = keys.locate(s + 2 * NW);
    // masked keys: score -inf, and V zeroed (a NaN there would survive a zero weight)
    const bool all = __all(off >= 0);
    if (!all) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[i] = ov[i] >= 0 ? sc[i] : -INFINITY;
    }
    const float f = raise(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), w.top, slack);
    if (__any(f != 1.f)) {
      w.sum *= f;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) w.o[j][c] *= f;
    }
    const float ref = w.top == -INFINITY ? 0.f : w.top;
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = exp2_fast(sc[i] - ref);
      w.sum += p[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        float vf[4];
        Elem<E>::four(vr[i][j], vf);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float x = all || ov[i] >= 0 ? vf[c] : 0.f;
          w.o[j][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, p[i], w.o[j][c], 0, 0, 0);
        }
      }
    keys.load_v(next, vr, ov);
    off = next;
    next = after;
  }
}

// Two-byte keys and values are whole operands of the two-byte matrix products, which run at sixteen
// times the float32 rate; only the queries and the weights, float32, are split into planes.
template <typename E>
struct Planes;
template <>
struct Planes<__bf16> {      // three planes carry all 24 bits
  static constexpr int N = 3;
  static __device__ __forceinline__ void split(const float* x, uint4* p) {
    split_x3(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]), p[0], p[1], p[2]);
  }
  static __device__ __forceinline__ f32x4 mul(const uint4& a, const uint4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  }
};
template <>
struct Planes<_Float16> {    // two planes of 11 bits, the second 2^11 times what the first leaves: within 2^-22
  static constexpr int N = 2;
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ void split(const float* x, uint4* p) {
    h8 a, b;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = (_Float16)x[i];
      b[i] = (_Float16)((x[i] - (float)a[i]) * 2048.f);
    }
    p[0] = __builtin_bit_cast(uint4, a);
    p[1] = __builtin_bit_cast(uint4, b);
  }
  static __device__ __forceinline__ f32x4 mul(const uint4& a, const uint4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  }
};

// The same strips two at a time (s and s + NW) on the two-byte matrix cores.  Scores: 16 keys by 32
// channels by 16 heads a product, K straight from memory.  V^T . P^T sums over both strips' 32 keys in
// one product, keys 4g .. 4g + 3 of each in lane group g: the weights' planes again stay in their
// lanes, and V's four rows a lane are turned into channels by eight byte permutations a 4 x 4 block.
// float16 weights are held 2^7 up and queries scaled to one by their head's largest, so that both
// planes stay in float16's range.  An infinity among what is seen has no planes of its own: the caller
// forms outputs that are not finite again in float32.
template <typename E, int NJ, bool FULL, int NW>
__device__ __forceinline__ void strips_16(const AttnArgs& a, const Keys<E, NJ, FULL>& keys, const float* q, bool on,
                                          int s, Wave<NJ>& w) {
  typedef Keys<E, NJ, FULL> K;
  typedef Planes<E> P;
  constexpr bool kHalf = P::N == 2;
  constexpr float kUp = kHalf ? 7.f : 0.f;
  uint4 qp[P::N][K::NK];
  float unit = 1.f;            // float16: 2^E of this head's largest |q|
  {
    float qf[K::NK][8];
    float big = 0.f;
#pragma unroll
    for (int j = 0; j < K::NK; ++j) {
      load_q<8, FULL>(a, q, on, 32 * j + 8 * keys.g, keys.d, qf[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(qf[j][e]));
    }
    if constexpr (kHalf) {
      big = fmaxf(big, __shfl_xor(big, 16, kWave));
      big = fmaxf(big, __shfl_xor(big, 32, kWave));
      const int e2 = big > 0.f && big < INFINITY ? max(min(__builtin_amdgcn_frexp_expf(big), 126), -126) : 0;
      unit = ldexpf(1.f, e2);
      const float down = ldexpf(1.f, -e2);
#pragma unroll
      for (int j = 0; j < K::NK; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) qf[j][e] *= down;
    }
#pragma unroll
    for (int j = 0; j < K::NK; ++j) {
      uint4 t[P::N];
      P::split(qf[j], t);
#pragma unroll
      for (int n = 0; n < P::N; ++n) qp[n][j] = t[n];
    }
  }
  uint4 kr[2][K::NK];
  typename K::VRaw vr[2][4][NJ];
  int64_t ov[2][4], off[2], next[2], after[2];
  f32x4 low[NJ][4];            // float16: the second plane's sums, 2^11 up
  w.clear();
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) low[j][c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    off[t] = keys.locate(s + t * NW);
    next[t] = keys.locate(s + (2 + t) * NW);
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    keys.load_k(off[t], kr[t]);
    keys.load_v(off[t], vr[t], ov[t]);
  }
  for (; s < keys.s1; s += 2 * NW) {
    f32x4 sc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4 big{0.f, 0.f, 0.f, 0.f}, small{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < K::NK; ++j) {
        big = P::mul(kr[t][j], qp[0][j], big);
        small = P::mul(kr[t][j], qp[1][j], small);
        if constexpr (P::N == 3) small = P::mul(kr[t][j], qp[2][j], small);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sc[t][i] = kHalf ? fmaf(small[i], 0x1p-11f, big[i]) * unit : big[i] + small[i];
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      keys.load_k(next[t], kr[t]);
      after[t] = keys.locate(s + (4 + t) * NW);
    }
    const bool all = __all(off[0] >= 0 && off[1] >= 0);
    if (!all) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool there = ov[t][i] >= 0;
          sc[t][i] = there ? sc[t][i] : -INFINITY;
#pragma unroll
          for (int j = 0; j < NJ; ++j) vr[t][i][j] = there ? vr[t][i][j] : typename K::VRaw{};
        }
    }
    float mx = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3]));
    mx = fmaxf(mx, fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
    const float f = raise(mx, w.top, 8.f);
    if (__any(f != 1.f)) {
      w.sum *= f;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          w.o[j][c] *= f;
          if constexpr (kHalf) low[j][c] *= f;
        }
    }
    const float ref = (w.top == -INFINITY ? 0.f : w.top) - kUp;
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = exp2_fast(sc[i / 4][i % 4] - ref);
      w.sum += p[i];
    }
    uint4 pp[P::N];
    P::split(p, pp);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t x[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[t][i] = c < 2 ? vr[t][i][j].x : vr[t][i][j].y;
        const uint32_t sel = c % 2 ? 0x07060302u : 0x05040100u;
        const uint4 av = {__builtin_amdgcn_perm(x[0][1], x[0][0], sel), __builtin_amdgcn_perm(x[0][3], x[0][2], sel),
                          __builtin_amdgcn_perm(x[1][1], x[1][0], sel), __builtin_amdgcn_perm(x[1][3], x[1][2], sel)};
        w.o[j][c] = P::mul(av, pp[0], w.o[j][c]);
        if constexpr (kHalf) {
          low[j][c] = P::mul(av, pp[1], low[j][c]);
        } else {
          w.o[j][c] = P::mul(av, pp[1], w.o[j][c]);
          w.o[j][c] = P::mul(av, pp[2], w.o[j][c]);
        }
      }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      keys.load_v(next[t], vr[t], ov[t]);
      off[t] = next[t];
      next[t] = after[t];
    }
  }
  if constexpr (kHalf) {
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) w.o[j][c] = (low[j][c] * 0x1p-11f + w.o[j][c]) * 0x1p-7f;
    w.sum *= 0x1p-7f;
  }
}

// Attention of up to 16 query heads that share kv head `kvh` over strips [s0, s1) of sequence b, by
// the NW waves of a workgroup, which are then joined through LDS.
template <typename E, int NJ, bool FULL, int NW>
__device__ __forceinline__ void attend(const AttnArgs& a, int b, int kvh, int gt, const Span& sp, int s0, int s1,
                                       float* s_o, float* s_ml) {
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wv = uniform((int)threadIdx.x >> 6);
  const int d = FULL ? 64 * NJ : a.d;
  const int hg = min(a.htile, a.group - gt * a.htile);   // heads of this tile
  const int head = kvh * a.group + gt * a.htile + m;
  const bool on = m < hg;
  const float* q = a.q + (int64_t)b * a.ldq + (int64_t)(on ? head : 0) * d;
  const Keys<E, NJ, FULL> keys(a, b, kvh, sp, s1);
  Wave<NJ> w;
  // What is not finite, or near the largest float, is formed again in float32 with weights of at most one:
  // the slack alone may have brought it there.
  float slack = 8.f;
  bool fine = false;
  if constexpr (sizeof(E) == 2) {
    strips_16<E, NJ, FULL, NW>(a, keys, q, on, s0 + wv, w);
    fine = in_bounds(w, on);
    slack = 0.f;
  }
#pragma unroll 1
  for (; !fine; slack = 0.f) {
    strips_f32<E, NJ, FULL, NW>(a, keys, q, on, s0 + wv, slack, w);
    fine = slack == 0.f || in_bounds(w, on);
  }
  float sum = w.sum;
  sum += __shfl_xor(sum, 16, kWave);
  sum += __shfl_xor(sum, 32, kWave);
  if (__any(on && w.top == -INFINITY)) {         // rare: no score that is a number.  Is there a key at all?
    bool there = false;
#pragma unroll 1
    for (int s = s0 + wv; s < s1 && !there; s += NW) there = __any(keys.locate(s) >= 0);
    if (there) w.top = fmaxf(w.top, kNoScore);
  }

  // The waves' maxima and sums, then their outputs 64 channels at a time: s_o[wave][head][64 + 4].
  if (g == 0) {
    s_ml[(wv * 16 + m) * 2] = w.top;
    s_ml[(wv * 16 + m) * 2 + 1] = sum;
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    if (on) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float4 x = make_float4(w.o[j][0][r], w.o[j][1][r], w.o[j][2][r], w.o[j][3][r]);
        *(float4*)(s_o + (wv * 16 + m) * 68 + 16 * g + 4 * r) = x;
      }
    }
    __syncthreads();
    for (int h = wv; h < hg; h += NW) {
      float t = -INFINITY;
#pragma unroll
      for (int u = 0; u < NW; ++u) t = fmaxf(t, s_ml[(u * 16 + h) * 2]);
      float l = 0.f, x = 0.f;
#pragma unroll
      for (int u = 0; u < NW; ++u) {
        const float f = weight_of(s_ml[(u * 16 + h) * 2], t);
        l += f * s_ml[(u * 16 + h) * 2 + 1];
        x += f * s_o[(u * 16 + h) * 68 + lane];
      }
      const int c = 64 * j + lane;
      const bool whole = s_ml[NW * 32] != 0.f;    // the pair's every key was here: this is the output
      if (c < d) {
        if (whole) {
          a.out[(int64_t)b * a.ldo + (int64_t)(kvh * a.group + gt * a.htile + h) * d + c] =
              t != -INFINITY ? x / l : 0.f;
        } else {
          float* dst = a.part + ((int64_t)__float_as_int(s_ml[NW * 32 + 1]) * a.htile + h) * (d + 2);
          dst[c] = x;
          if (j == 0 && lane == 0) {
            dst[d] = t;
            dst[d + 1] = l;
          }
        }
      }
    }
    __syncthreads();
  }
}

// Waves a SIMD that the registers are held to: what they need is 16 NJ floats each of output, keys
// and values, and the query (half as much again as planes).
template <typename E, int NJ>
constexpr int waves_per_simd() {
  return NJ == 1 ? (sizeof(E) == 2 ? 3 : 4) : NJ == 2 ? 2 : 1;
}

// One workgroup per (sequence, kv head, tile of query heads): one launch, for caches short enough.
// Eight waves where a key row is short: 6.9 us against 7.6 with four at one sequence of 256 float32 keys
// (14 on 2 heads of 64); at d = 128 they only crowd the CU (256 bfloat16 keys of 128 sequences, 32 on 8
// heads: 37 us against 27).
template <int NJ>
constexpr int kWholeWaves = NJ == 1 ? 8 : 4;

template <typename E, int NJ, bool FULL>
__global__ __launch_bounds__(kWholeWaves<NJ> * 64, (waves_per_simd<E, NJ>())) void k_paged_whole(AttnArgs a) {
  constexpr int NW = kWholeWaves<NJ>;
  __shared__ float s_o[NW * 16 * 68];
  __shared__ float s_ml[NW * 32 + 2];
  const int per = a.kv_heads * a.gtiles, b = blockIdx.x / per, p = blockIdx.x % per;
  const Span sp = uniform_span(a, b);
  if (threadIdx.x == 0) s_ml[NW * 32] = 1.f;
  __syncthreads();
  attend<E, NJ, FULL, NW>(a, b, p / a.gtiles, p % a.gtiles, sp, sp.lo / kStrip, (sp.hi + kStrip - 1) / kStrip, s_o,
                          s_ml);
}

// HBM-bound for large batches: 96 ragged sequences of up to 6000 bfloat16 keys, 32 on 8 heads of 128, 1.2 GB in
// 248 us, 4.7 TB/s (232 at best); 3 x 100001 float16 keys, 14 on 2 heads of 64, 36.3 us, 4.2 TB/s with its start;
// 24 x 1000 and fewer keys by five dependent latencies, 7 - 10 us.
//
// The units of all sequences and heads, in order, shared out evenly over `groups` workgroups by the
// lengths on the device: a ragged batch fills the machine as an even one does, and a captured
// launch serves every length.  A pair (sequence, tile of heads) that one workgroup holds whole is
// written by it; of a pair that crosses workgroups each leaves its maximum, sum and output in `part`
// (slot 2 w, or 2 w + 1 where the pair begins inside w's share), and k_paged_join adds them up.
// The workgroup that begins a pair enters it into `pairs`: its first slot and last workgroup, or -1.
template <typename E, int NJ, bool FULL>
__global__ __launch_bounds__(kWaves * 64, (waves_per_simd<E, NJ>())) void k_paged_split(AttnArgs a) {
  __shared__ float s_o[kWaves * 16 * 68];
  __shared__ float s_ml[kWaves * 32 + 2];
  const int per = a.kv_heads * a.gtiles, w = blockIdx.x;
  const Share sh = share_of(a, w);
  if (w >= sh.n) return;
  int64_t at = sh.at, in = at - sh.before * per;  // the unit, and the unit within the sequence: [pair][tile]
  int b = sh.b;
  Span sp = uniform_span(a, b);
  while (at < sh.end) {
    while (in >= (int64_t)sp.tiles * per) {
      in -= (int64_t)sp.tiles * per;
      if (++b >= a.batch) return;                 // lengths that changed under the call
      sp = uniform_span(a, b);
    }
    const int p = (int)(in / sp.tiles), t = (int)(in - (int64_t)p * sp.tiles);
    const int take = (int)min((int64_t)(sp.tiles - t), sh.end - at), slot = 2 * w + (at == sh.at ? 0 : 1);
    const bool whole = take == sp.tiles;
    if (threadIdx.x == 0) {
      s_ml[kWaves * 32] = whole ? 1.f : 0.f;
      s_ml[kWaves * 32 + 1] = __int_as_float(slot);
      if (t == 0)
        a.pairs[(int64_t)b * per + p] =
            make_int2(whole ? -1 : slot, whole ? 0 : (int)(((at + sp.tiles) * sh.n - 1) / sh.units));
    }
    __syncthreads();
    const int t0 = sp.lo / kTile + t, per_tile = kTile / kStrip;
    attend<E, NJ, FULL, kWaves>(a, b, p / a.gtiles, p % a.gtiles, sp, max(t0 * per_tile, sp.lo / kStrip),
                                min((t0 + take) * per_tile, (sp.hi + kStrip - 1) / kStrip), s_o, s_ml);
    at += take;
    in += take;
  }
}

constexpr int kJoinWaves = 4, kJoinAhead = 8;

// One workgroup per (sequence, query head), 3.4 us for one sequence, 5.4 for 42 heads of 85 parts each, 8 for
// 3.1 thousand heads of one or two: the parts of a pair that crossed workgroups, and zeros
// for a sequence with no key to see.  The waves take the parts in turn, eight at a time so that
// their loads are in flight together, then meet in LDS.
template <int NJ>
__global__ __launch_bounds__(kJoinWaves * 64) void k_paged_join(AttnArgs a) {
  __shared__ float s_o[kJoinWaves * 64 * NJ];
  __shared__ float s_ml[kJoinWaves * 2];
  const int lane = threadIdx.x & 63, wv = uniform((int)threadIdx.x >> 6);
  const int b = blockIdx.x / a.heads, head = blockIdx.x % a.heads, kvh = head / a.group, gh = head % a.group;
  const int h = gh % a.htile;
  const int2 pair = a.pairs[((int64_t)b * a.kv_heads + kvh) * a.gtiles + gh / a.htile];
  float* out = a.out + (int64_t)b * a.ldo + (int64_t)head * a.d;
  if (span_of(a, b).tiles == 0) {
    for (int c = threadIdx.x; c < a.d; c += kJoinWaves * 64) out[c] = 0.f;
    return;
  }
  if (pair.x < 0) return;                       // written by the one workgroup that held it
  const int w0 = min(pair.x >> 1, a.groups - 1), count = min(pair.y, a.groups - 1) - w0 + 1;
  float x[NJ], top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int j = 0; j < NJ; ++j) x[j] = 0.f;
  for (int i = wv; i < count; i += kJoinWaves * kJoinAhead) {
    float y[kJoinAhead][NJ], t[kJoinAhead], l[kJoinAhead];
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) {
      const int n = i + u * kJoinWaves;
      const float* src = a.part + ((int64_t)(n ? 2 * (w0 + min(n, count - 1)) : 2 * w0 + (pair.x & 1)) * a.htile + h) * (a.d + 2);
      t[u] = n < count ? src[a.d] : -INFINITY;
      l[u] = src[a.d + 1];
#pragma unroll
      for (int j = 0; j < NJ; ++j) y[u][j] = 64 * j + lane < a.d ? src[64 * j + lane] : 0.f;
    }
    float now = top;
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) now = fmaxf(now, t[u]);
    const float f = weight_of(top, now);
    sum *= f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) x[j] *= f;
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) {
      if (i + u * kJoinWaves < count) {
        const float g = weight_of(t[u], now);
        sum += g * l[u];
#pragma unroll
        for (int j = 0; j < NJ; ++j) x[j] += g * y[u][j];
      }
    }
    top = now;
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) s_o[(wv * NJ + j) * 64 + lane] = x[j];
  if (lane == 0) {
    s_ml[2 * wv] = top;
    s_ml[2 * wv + 1] = sum;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.d; c += kJoinWaves * 64) {
    float t = -INFINITY, l = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) t = fmaxf(t, s_ml[2 * w]);
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) {
      const float f = weight_of(s_ml[2 * w], t);
      l += f * s_ml[2 * w + 1];
      y += f * s_o[w * NJ * 64 + c];
    }
    out[c] = t != -INFINITY ? y / l : 0.f;
  }
}

template <typename E, int NJ, bool FULL>
void launch_attention(const AttnArgs& a, bool whole, hipStream_t st) {
  if (whole) {
    hipLaunchKernelGGL((k_paged_whole<E, NJ, FULL>), dim3(a.batch * a.kv_heads * a.gtiles), dim3(kWholeWaves<NJ> * 64), 0,
                       st, a);
  } else {
    hipLaunchKernelGGL((k_paged_split<E, NJ, FULL>), dim3(a.groups), dim3(kWaves * 64), 0, st, a);
    hipLaunchKernelGGL(k_paged_join<NJ>, dim3(a.batch * a.heads), dim3(kJoinWaves * 64), 0, st, a);
  }
}

template <typename E>
void attention_for(const AttnArgs& a, bool whole, hipStream_t st) {
  switch ((a.d + 63) / 64) {
    case 1: a.d == 64 ? launch_attention<E, 1, true>(a, whole, st) : launch_attention<E, 1, false>(a, whole, st); break;
    case 2: a.d == 128 ? launch_attention<E, 2, true>(a, whole, st) : launch_attention<E, 2, false>(a, whole, st); break;
    case 3: launch_attention<E, 3, false>(a, whole, st); break;
    default: a.d == 256 ? launch_attention<E, 4, true>(a, whole, st) : launch_attention<E, 4, false>(a, whole, st);
  }
}

}  // namespace

extern "C" {

int cv3_paged_tables(const int32_t* lengths, const int32_t* new_tokens, int64_t requests, int64_t page,
                     const int32_t* free_pages, int64_t free_count, const int32_t* taken, int32_t* tables,
                     int64_t blocks, int64_t tokens, int32_t* total, int32_t* taken_out, int32_t* starts,
                     int64_t* slots, int32_t* positions, cv3_stream_t s) {
  CV3_ALIVE();
  CV3_REQUIRE(requests >= 0 && requests <= kTabRequests, CV3_EINVAL, "at most %d requests a call, not %lld",
              kTabRequests, (long long)requests);
  CV3_REQUIRE(page >= 1 && page <= 65536, CV3_EINVAL, "a page holds 1 to 65536 keys, not %lld", (long long)page);
  CV3_REQUIRE(blocks >= 1 && blocks <= (INT32_MAX - 65536) / page, CV3_EINVAL,
              "tables of %lld blocks of %lld keys pass 2^31 keys", (long long)blocks, (long long)page);
  CV3_REQUIRE(tokens >= 0 && tokens <= INT32_MAX - 65536, CV3_EINVAL, "too many tokens: %lld", (long long)tokens);
  CV3_REQUIRE(free_count >= 0 && free_count <= INT32_MAX, CV3_EINVAL, "bad number of free pages");
  CV3_REQUIRE(starts && (requests == 0 || (lengths && new_tokens && tables && total)) &&
                  (tokens == 0 || (slots && positions)) && (free_pages ? taken && taken_out : free_count == 0),
              CV3_EINVAL, "null operand");
  const double r = (double)requests, t = (double)tokens, one = free_pages ? 4 : 0;
  const Run in[] = {{lengths, 4 * r}, {new_tokens, 4 * r}, {free_pages, 4.0 * free_count}, {taken, one}};
  const Run out[] = {{tables, 4 * r * blocks}, {total, 4 * r}, {taken_out, one}, {starts, 4 * (r + 1)}, {slots, 8 * t},
                     {positions, 4 * t}};
  CV3_REQUIRE(apart(out, in), CV3_EINVAL,
              "results that overlap: every workgroup reads the lengths, the counts and the free pages while others write");
  TabArgs a{lengths, new_tokens, free_pages, taken, tables, total, taken_out, starts, slots, positions,
            free_count, (int)requests, (int)page, (int)blocks, (int)tokens};
  const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(tokens, kTabThreads * kTabEach), 1024));
  hipLaunchKernelGGL(k_block_tables, dim3(grid), dim3(kTabThreads), 0, stream_of(s), a);
  CV3_LAUNCHED();
  return CV3_OK;
}

int cv3_paged_append(const float* rows, int64_t n, int64_t ld, int heads, int kv_heads, int d,
                     const int32_t* positions, const int64_t* slots, const float* cos_tab, const float* sin_tab,
                     int64_t rope_rows, int cache_type, void* k_cache, void* v_cache, int64_t pages, int64_t page,
                     float* q, int64_t ldq, cv3_stream_t s) {
  CV3_ALIVE();
  if (int rc = check_cache(cache_type, k_cache, v_cache, pages, page, kv_heads, d)) return rc;
  CV3_REQUIRE(heads >= 0 && heads <= 65536, CV3_EINVAL, "0 to 65536 query heads, not %d", heads);
  CV3_REQUIRE(n >= 0, CV3_EINVAL, "negative number of rows");
  CV3_REQUIRE(ld >= (int64_t)(heads + 2 * kv_heads) * d, CV3_EINVAL, "rows of %lld floats are too short for %d + 2 x %d heads of %d",
              (long long)ld, heads, kv_heads, d);
  CV3_REQUIRE(!q || ldq >= (int64_t)heads * d, CV3_EINVAL, "q rows of %lld floats are too short", (long long)ldq);
  CV3_REQUIRE(!cos_tab == !sin_tab, CV3_EINVAL, "the rotary needs both tables");
  CV3_REQUIRE(!cos_tab || (positions && rope_rows >= 1), CV3_EINVAL, "the rotary needs positions and table rows");
  if (n == 0) return CV3_OK;
  CV3_REQUIRE(rows && slots, CV3_EINVAL, "null operand");
  const double cache = (double)pages * page * kv_heads * d * elem_size(cache_type);
  CV3_REQUIRE(!overlap({k_cache, cache}, {v_cache, cache}), CV3_EINVAL, "the caches of keys and values overlap");
  CV3_REQUIRE(!q || rows_alike_or_apart(rows, ld, (int64_t)(heads + 2 * kv_heads) * d, q, ldq, (int64_t)heads * d, n),
              CV3_EINVAL, "q and the rows overlap: q may be the rows themselves, at their pitch");
  AppendArgs a{rows, n, ld, positions, slots, cos_tab, sin_tab, rope_rows, k_cache, v_cache, pages * page, q, ldq,
               (int)page, heads, kv_heads, d};
  // four channels a thread where rows start on 16 bytes (the tables are read by single floats)
  const bool wide = (uintptr_t)rows % 16 == 0 && ld % 4 == 0 && (!q || ((uintptr_t)q % 16 == 0 && ldq % 4 == 0));
  const unsigned per_row = (unsigned)(heads + 2 * kv_heads) * (d / 2) / (wide ? 4 : 1);
  const unsigned threads = std::min(256u, (per_row + 63) / 64 * 64), per = (per_row + threads - 1) / threads;
  CV3_REQUIRE(n <= (int64_t)kLaunchBlocks / per, CV3_EINVAL, "too many rows for one call: %lld", (long long)n);
  const int64_t bytes = n * ((2 * heads + 2 * kv_heads) * (int64_t)d * 4 + 2 * kv_heads * (int64_t)d * elem_size(cache_type));
  const auto kernel = !wide ? k_append<1, false> : bytes > (256 << 20) ? k_append<4, true> : k_append<4, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)n * per), dim3(threads), 0, stream_of(s), a, cache_type, per_row, per);
  CV3_LAUNCHED();
  return CV3_OK;
}

int cv3_paged_attention(const float* q, int64_t ldq, int64_t batch, int heads, int kv_heads, int d, int cache_type,
                        const void* k_cache, const void* v_cache, int64_t pages, int64_t page, const int32_t* tables,
                        int64_t blocks, const int32_t* lengths, const int32_t* starts, float scale, float* out,
                        int64_t ldo, cv3_stream_t s) {
  CV3_ALIVE();
  CV3_REQUIRE(kv_heads >= 1 && heads >= 1 && heads % kv_heads == 0, CV3_EINVAL,
              "%d query heads is not a multiple of %d kv heads", heads, kv_heads);
  if (int rc = check_cache(cache_type, k_cache, v_cache, pages, page, kv_heads, d)) return rc;
  CV3_REQUIRE(heads <= 65536, CV3_EINVAL, "at most 65536 query heads, not %d", heads);
  CV3_REQUIRE(blocks >= 1 && blocks <= (INT32_MAX - 65536) / page, CV3_EINVAL,
              "tables of %lld blocks of %lld keys pass 2^31 keys", (long long)blocks, (long long)page);
  CV3_REQUIRE(batch >= 0 && batch <= (kLaunchBlocks - 1) / heads, CV3_EINVAL, "%lld sequences of %d heads are too many for one call",
              (long long)batch, heads);
  CV3_REQUIRE(ldq >= (int64_t)heads * d && ldo >= (int64_t)heads * d, CV3_EINVAL, "rows are too short for %d heads of %d",
              heads, d);
  if (batch == 0) return CV3_OK;
  CV3_REQUIRE(q && tables && lengths && out, CV3_EINVAL, "null operand");
  CV3_REQUIRE(rows_alike_or_apart(q, ldq, (int64_t)heads * d, out, ldo, (int64_t)heads * d, batch), CV3_EINVAL,
              "out and q overlap: out may be q itself, at its pitch");
  const int group = heads / kv_heads, htile = std::min(group, 16), gtiles = (group + htile - 1) / htile;
  AttnArgs a{q, ldq, k_cache, v_cache, tables, lengths, starts, out, ldo, nullptr, nullptr, pages, blocks, (int)batch, (int)page,
             heads, kv_heads, group, gtiles, htile, d, 0, scale * 1.4426950408889634f};
  hipStream_t st = stream_of(s);
  // One workgroup a pair where a full table's keys and values are few: it takes 5.5 us and 1.3 more each
  // 64 KB, the split form 9.7 and hardly more (one sequence, 14 on 2 heads of 64: 256 float32 keys 6.9
  // against 9.6 us, 512 keys 10.7 against 9.6; 512 bfloat16 keys 7.2 against 9.7, 1024 10.6 against 9.7).
  bool whole = blocks * page * 2 * d * elem_size(cache_type) <= kWholeBytes;
  if (!whole) {
    a.groups = kGroups;
    const size_t parts = (size_t)2 * a.groups * htile * (d + 2) * sizeof(float);   // a multiple of 8
    void* work = nullptr;
    const int rc = scratch_alloc(&work, parts + (size_t)batch * kv_heads * gtiles * sizeof(int2), st);
    if (rc == CV3_ENOMEM) whole = true;      // one workgroup a pair needs no memory of its own
    else if (rc) return rc;
    a.part = (float*)work;
    a.pairs = (int2*)((char*)work + parts);
  }
  if (cache_type == CV3_F32) attention_for<float>(a, whole, st);
  else if (cache_type == CV3_F16) attention_for<_Float16>(a, whole, st);
  else attention_for<__bf16>(a, whole, st);
  const hipError_t e = hipGetLastError();
  const int rc = whole ? CV3_OK : scratch_free(a.part, st);
  CV3_REQUIRE(e == hipSuccess, CV3_EHIP, "kernel launch failed: %s", hipGetErrorString(e));
  return rc;
}

}  // extern "C"
