// The paged key-value cache: block tables and slots from request lengths, rotary with the cache
// write, and the attention of one new token per sequence over the cache.  It is the form for
// several sequences of what the reference holds for one (KVCache, cv3cpu/models/qwen2.py:74-121;
// apply_rope, qwen2.py:64-71; sdpa at one query, cv3cpu/ops.py:267-300).
//
// A cache is [pages, kv_heads, page, d]: the rows of one head in one page are one contiguous run.
// Key j of sequence b lies in page tables[b][j / page], row j % page.  Offsets are 64-bit; page
// ids, lengths and slots come from device memory, so every one is checked against its bounds
// where it is used, and what lies outside counts as absent.
#include "common.hpp"

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

constexpr int kTabThreads = 1024;
constexpr int kTabRequests = 4096;   // a call's requests: two int32 of LDS each

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

// Inclusive sum over the workgroup's threads; *all receives the sum of all of them.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* red, int64_t* all) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t u = __shfl_up(v, o, kWave);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 63) red[wid] = v;
  __syncthreads();
  int64_t before = 0, sum = 0;
  for (int i = 0; i < kTabThreads / 64; ++i) {
    const int64_t r = red[i];
    if (i < wid) before += r;
    sum += r;
  }
  *all = sum;
  return v + before;
}

// Every workgroup sums over the requests by itself (a few kilobytes from L2, no wait between
// workgroups), then lists a share of the tokens.  A token finds its request among the starts in
// LDS; the token that opens a page also enters it into the table.  Pages before `have` are the
// request's own already; page have + i is free_pages[first + i].
__global__ __launch_bounds__(kTabThreads) void k_block_tables(TabArgs a) {
  __shared__ int32_t s_start[kTabRequests + 1];
  __shared__ int32_t s_first[kTabRequests];   // index of the request's first new page among the free ones
  __shared__ int64_t s_red[kTabThreads / 64];
  const int64_t cap = (int64_t)a.blocks * a.page;
  const int64_t taken = a.taken[0];
  int64_t tok = 0, pages = 0;
  for (int r0 = 0; r0 < a.requests; r0 += kTabThreads) {
    const int r = r0 + (int)threadIdx.x;
    const bool on = r < a.requests;
    const int64_t held = on ? max(a.lengths[r], 0) : 0;
    const int64_t want = on ? max((int64_t)0, min((int64_t)a.fresh[r], cap - held)) : 0;
    int64_t all;
    // the tokens that a call may list go to the first requests: the running sums, cut at that number
    const int64_t sum = block_scan(want, s_red, &all);
    const int64_t end = min(tok + sum, (int64_t)a.tokens), start = min(tok + sum - want, (int64_t)a.tokens);
    tok = min(tok + all, (int64_t)a.tokens);
    const int64_t now = held + (end - start);
    const int64_t have = (uint32_t)(held + a.page - 1) / (uint32_t)a.page;
    const int64_t need = (int64_t)((uint32_t)(now + a.page - 1) / (uint32_t)a.page) - have;
    const int64_t upto = block_scan(need, s_red, &all);
    if (on) {
      s_start[r] = (int32_t)start;
      s_first[r] = (int32_t)min(taken + pages + upto - need, (int64_t)INT32_MAX);
      if (blockIdx.x == 0) {
        a.starts[r] = (int32_t)start;
        a.total[r] = (int32_t)now;
      }
    }
    pages += all;
  }
  if (threadIdx.x == 0) s_start[a.requests] = (int32_t)tok;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.starts[a.requests] = (int32_t)tok;
    a.taken_out[0] = (int32_t)min(taken + pages, (int64_t)INT32_MAX);
  }
  __syncthreads();
  for (int64_t t = (int64_t)blockIdx.x * kTabThreads + threadIdx.x; t < a.tokens;
       t += (int64_t)gridDim.x * kTabThreads) {
    int64_t slot = -1;
    int32_t pos = -1;
    if (t < tok) {
      int lo = 0, hi = a.requests;   // the last request that starts at or before t: requests without tokens lie before it
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_start[mid] <= t) lo = mid; else hi = mid;
      }
      const int32_t held = max(a.lengths[lo], 0);
      pos = held + (int32_t)(t - s_start[lo]);
      const int block = (uint32_t)pos / (uint32_t)a.page, row = pos - block * a.page;
      const int have = (uint32_t)(held + a.page - 1) / (uint32_t)a.page;
      int32_t* entry = a.tables + (int64_t)lo * a.blocks + block;
      int32_t id;
      if (block < have) {
        id = *entry;
      } else {
        const int64_t i = (int64_t)s_first[lo] + (block - have);
        id = i >= 0 && i < a.free_count ? a.free_pages[i] : -1;
        if (row == 0) *entry = id;
      }
      if (id >= 0) slot = (int64_t)id * a.page + row;
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
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

template <int V>
__device__ __forceinline__ void store_elems(void* base, int type, int64_t at, const float* x) {
  if (type == CV3_F32) {
    float* p = (float*)base + at;
    if constexpr (V == 4) *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
    else p[0] = x[0];
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
// cache's type as they are written.
template <int V>
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
    *(float4*)x = *(const float4*)src;
    *(float4*)y = *(const float4*)(src + half);
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
    store_elems<V>(dst, CV3_F32, 0, u);
    store_elems<V>(dst, CV3_F32, half, w);
    return;
  }
  const int64_t slot = a.slots[n];
  if (!placed || slot < 0 || slot >= a.slot_count) return;
  const int64_t id = a.slot_count <= INT32_MAX ? (uint32_t)slot / (uint32_t)a.page : slot / a.page;
  const int h = head - a.heads, kv = h % a.kv_heads;
  void* cache = h < a.kv_heads ? a.k : a.v;
  const int64_t at = ((id * a.kv_heads + kv) * a.page + (slot - id * a.page)) * a.d + j;
  store_elems<V>(cache, type, at, u);
  store_elems<V>(cache, type, at + half, w);
}

// ------------------------------------------------------------------------------------------------
// attention of one new token per sequence
// ------------------------------------------------------------------------------------------------

constexpr int kTile = 64;       // keys of a work unit
constexpr int kStrip = 16;      // keys that one wave multiplies at a time
constexpr int kSplitWaves = 4, kWholeWaves = 8;

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

// Units of all sequences, and the sequence that unit-of-one-head `at` (in [0, total)) falls in: *b,
// and *before, the units of the sequences ahead of it.  Every wave finds them by itself; a lane
// sums four sequences.  With at < 0: the units ahead of sequence *b.
__device__ __forceinline__ int64_t find_units(const AttnArgs& a, int64_t at, int* b, int64_t* before) {
  const int lane = threadIdx.x & 63;
  int64_t total = 0;
  bool found = false;
  const int want = *b;
  for (int c = 0; c < a.batch; c += 256) {
    int t[4];
    int64_t mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = span_of(a, c + lane * 4 + i).tiles;
      mine += t[i];
    }
    int64_t up = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t u = __shfl_up(up, o, kWave);
      if (lane >= o) up += u;
    }
    int64_t ahead = total + up - mine;
    if (!found) {
      int in = -1;
      int64_t first = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = c + lane * 4 + i;
        const bool here = at >= 0 ? at >= ahead && at < ahead + t[i] : n == want;
        if (here) in = n, first = ahead;
        ahead += t[i];
      }
      const uint64_t hit = __ballot(in >= 0);
      if (hit) {
        const int from = __ffsll((unsigned long long)hit) - 1;
        *b = __builtin_amdgcn_readfirstlane(__shfl(in, from, kWave));
        *before = __shfl(first, from, kWave);
        found = true;
      }
    }
    total += __shfl(up, 63, kWave);
  }
  return total;
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

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// 2^(x - top), 0 where x is -inf whatever top is
__device__ __forceinline__ float weight_of(float x, float top) { return x == -INFINITY ? 0.f : exp2_fast(x - top); }

// Attention of up to 16 query heads that share kv head `kvh` over strips [s0, s1) of sequence b.
//
// Both products run on the float32 matrix cores, whatever the cache's type: 16x16x4 products take
// 1024 cycles a strip of 16 keys at d = 64, room for 19 TB/s of float32 cache, so the kernel is
// bound by HBM for one query head a kv head as for sixteen.  Scores are formed as K . q^T, so that
// lane (g, m) = (lane / 16, lane % 16) holds those of keys 4g .. 4g + 3 and head m.  That is also
// where V^T . P^T wants its second operand: step i takes keys {i, 4 + i, 8 + i, 12 + i}, lane (g, m)
// its own p[i].  Nothing goes through LDS before the waves are joined.  K is loaded in the first
// operand's layout with the sum over channels permuted so that a lane's share is 16 contiguous
// bytes, V with the output channels permuted alike (d = 64 jj + 4 m + c in tile (jj, c)).
//
// The running maximum is kept for a whole wave's strips and moved only when a score passes it by
// more than 2^8: p stays below 2^8 and the sums in float32 lose nothing.
template <typename E, int NJ, bool FULL, int NW>
__device__ void attend(const AttnArgs& a, int b, int kvh, int gt, const Span& sp, int s0, int s1, float* s_o,
                       float* s_ml) {
  constexpr int KC = 16 / sizeof(E);              // channels of a lane's 16 bytes
  constexpr int NK = 64 * NJ / (4 * KC);          // such loads a key row
  typedef typename Elem<E>::VRaw VRaw;
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int d = FULL ? 64 * NJ : a.d;
  const int hg = min(a.htile, a.group - gt * a.htile);   // heads of this tile
  const int head = kvh * a.group + gt * a.htile + m;

  float qf[NK * KC];
#pragma unroll
  for (int j = 0; j < NK; ++j)
#pragma unroll
    for (int e = 0; e < KC; e += 4) {
      const int c = 4 * KC * j + KC * g + e;
      f32x4u x{};
      if (m < hg && (FULL || c < d)) x = *(const f32x4u*)(a.q + (int64_t)b * a.ldq + (int64_t)head * d + c);
#pragma unroll
      for (int i = 0; i < 4; ++i) qf[j * KC + e + i] = x.v[i] * a.scale;
    }

  const int32_t* table = a.tables + (int64_t)b * a.blocks;
  const E* kb = (const E*)a.k + (int64_t)kvh * a.page * d;
  const E* vb = (const E*)a.v + (int64_t)kvh * a.page * d;
  const int64_t stride = (int64_t)a.kv_heads * a.page;

  // Offset of key 16 s + m in the cache, -1 where there is none to see.
  auto locate = [&](int s) -> int64_t {
    const int key = s * kStrip + m;
    if (s >= s1 || key < sp.lo || key >= sp.hi) return -1;
    const int blk = (uint32_t)key / (uint32_t)a.page;
    const int32_t id = table[blk];
    if ((uint32_t)id >= (uint64_t)a.pages) return -1;
    return ((int64_t)id * stride + (key - blk * a.page)) * d;
  };
  uint4 kr[NK];
  VRaw vr[4][NJ];
  auto load_k = [&](int64_t off) {
    const E* p = kb + max(off, (int64_t)0) + KC * g;      // a key that is not there reads the first page's
#pragma unroll
    for (int j = 0; j < NK; ++j)
      kr[j] = FULL || 4 * KC * j + KC * g < d ? *(const uint4*)(p + 4 * KC * j) : uint4{};
  };
  int64_t ov[4];
  auto load_v = [&](int64_t off) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ov[i] = __shfl(off, 4 * g + i, kWave);
      const E* p = vb + max(ov[i], (int64_t)0) + 4 * m;
#pragma unroll
      for (int j = 0; j < NJ; ++j) vr[i][j] = FULL || 64 * j + 4 * m < d ? *(const VRaw*)(p + 64 * j) : VRaw{};
    }
  };

  f32x4 o[NJ][4];
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) o[j][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = 0.f;

  int s = s0 + wv;
  int64_t off = locate(s), next = locate(s + NW);
  load_k(off);
  load_v(off);
  for (; s < s1; s += NW) {
    // scores of this strip; then its K registers take the next one's rows
    f32x4 sc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      float kf[KC];
      Elem<E>::wide(kr[j], kf);
#pragma unroll
      for (int e = 0; e < KC; ++e) sc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], qf[j * KC + e], sc, 0, 0, 0);
    }
    load_k(next);
    const int64_t after = locate(s + 2 * NW);

    // masked keys: score -inf, and V zeroed (a NaN there would survive a zero weight)
    const bool all = __all(off >= 0);
    if (!all) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[i] = ov[i] >= 0 ? sc[i] : -INFINITY;
    }
    const float mx = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
    if (__any(!(mx <= top + 8.f) && mx != -INFINITY)) {     // NaN scores too: they reach the output
      float t = mx;
      t = fmaxf(t, __shfl_xor(t, 16, kWave));
      t = fmaxf(t, __shfl_xor(t, 32, kWave));
      t = fmaxf(t, top);
      const float f = weight_of(top, t);
      sum *= f;
      top = t;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[j][c] *= f;
    }
    const float ref = top == -INFINITY ? 0.f : top;
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = exp2_fast(sc[i] - ref);
      sum += p[i];
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
          o[j][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, p[i], o[j][c], 0, 0, 0);
        }
      }
    load_v(next);
    off = next;
    next = after;
  }
  sum += __shfl_xor(sum, 16, kWave);
  sum += __shfl_xor(sum, 32, kWave);

  // The waves' maxima and sums, then their outputs 64 channels at a time: s_o[wave][head][64 + 4].
  if (g == 0) {
    s_ml[(wv * 16 + m) * 2] = top;
    s_ml[(wv * 16 + m) * 2 + 1] = sum;
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    if (m < hg) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float4 x = make_float4(o[j][0][r], o[j][1][r], o[j][2][r], o[j][3][r]);
        *(float4*)(s_o + (wv * 16 + m) * 68 + 16 * g + 4 * r) = x;
      }
    }
    __syncthreads();
    for (int h = wv; h < hg; h += NW) {
      float t = -INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w) t = fmaxf(t, s_ml[(w * 16 + h) * 2]);
      float l = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = weight_of(s_ml[(w * 16 + h) * 2], t);
        l += f * s_ml[(w * 16 + h) * 2 + 1];
        x += f * s_o[(w * 16 + h) * 68 + lane];
      }
      const int c = 64 * j + lane;
      const bool whole = s_ml[NW * 32] != 0.f;    // the pair's every key was here: this is the output
      if (c < d) {
        if (whole) {
          a.out[(int64_t)b * a.ldo + (int64_t)(kvh * a.group + gt * a.htile + h) * d + c] = l != 0.f ? x / l : 0.f;
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

// One workgroup per (sequence, kv head, tile of query heads): one launch, for caches short enough.
template <typename E, int NJ, bool FULL>
__global__ __launch_bounds__(kWholeWaves * 64) void k_paged_whole(AttnArgs a) {
  __shared__ float s_o[kWholeWaves * 16 * 68];
  __shared__ float s_ml[kWholeWaves * 32 + 2];
  const int per = a.kv_heads * a.gtiles, b = blockIdx.x / per, p = blockIdx.x % per;
  const Span sp = span_of(a, b);
  if (threadIdx.x == 0) s_ml[kWholeWaves * 32] = 1.f;
  __syncthreads();
  attend<E, NJ, FULL, kWholeWaves>(a, b, p / a.gtiles, p % a.gtiles, sp, sp.lo / kStrip,
                                   (sp.hi + kStrip - 1) / kStrip, s_o, s_ml);
}

// The units of all sequences and heads, in order, shared out evenly over `groups` workgroups by the
// lengths on the device: a ragged batch fills the machine as an even one does, and a captured
// launch serves every length.  A pair that one workgroup holds whole is written by it; of a pair
// that crosses workgroups each leaves its maximum, sum and output in `part` (slot 2 w, or 2 w + 1
// where the pair begins inside w's share), and k_paged_join adds them up.
__device__ __forceinline__ int groups_for(const AttnArgs& a, int64_t units) {
  return (int)min((int64_t)a.groups, units);
}

template <typename E, int NJ, bool FULL>
__global__ __launch_bounds__(kSplitWaves * 64) void k_paged_split(AttnArgs a) {
  __shared__ float s_o[kSplitWaves * 16 * 68];
  __shared__ float s_ml[kSplitWaves * 32 + 2];
  const int per = a.kv_heads * a.gtiles;
  // total first, then the sequence of this workgroup's first unit
  int b = 0;
  int64_t before = 0;
  const int64_t units = find_units(a, 0, &b, &before) * per;
  const int n = groups_for(a, units), w = blockIdx.x;
  if (w >= n) return;
  int64_t at = units * w / n;
  const int64_t end = units * (w + 1) / n;
  find_units(a, at / per, &b, &before);
  Span sp = span_of(a, b);
  int64_t in = at - before * per;                 // unit within the sequence: [pair][tile]
  const int64_t first = at;
  while (at < end) {
    while (in >= (int64_t)sp.tiles * per) {
      in -= (int64_t)sp.tiles * per;
      if (++b >= a.batch) return;                 // lengths that changed under the call
      sp = span_of(a, b);
    }
    const int p = (int)(in / sp.tiles), t = (int)(in % sp.tiles);
    const int take = (int)min((int64_t)(sp.tiles - t), end - at);
    if (threadIdx.x == 0) {
      s_ml[kSplitWaves * 32] = take == sp.tiles ? 1.f : 0.f;
      s_ml[kSplitWaves * 32 + 1] = __int_as_float(2 * w + (at == first ? 0 : 1));
    }
    __syncthreads();
    const int t0 = sp.lo / kTile + t, per_tile = kTile / kStrip;
    attend<E, NJ, FULL, kSplitWaves>(a, b, p / a.gtiles, p % a.gtiles, sp, max(t0 * per_tile, sp.lo / kStrip),
                                     min((t0 + take) * per_tile, (sp.hi + kStrip - 1) / kStrip), s_o, s_ml);
    at += take;
    in += take;
  }
}

constexpr int kJoinWaves = 8;

// One workgroup per (sequence, query head): the parts of a pair that crossed workgroups, and zeros
// for a sequence with no key to see.  The waves take the parts in turn, then meet in LDS.
__global__ __launch_bounds__(kJoinWaves * 64) void k_paged_join(AttnArgs a) {
  __shared__ float s_o[kJoinWaves * 256];
  __shared__ float s_ml[kJoinWaves * 2];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int want = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
  const int per = a.kv_heads * a.gtiles, kvh = head / a.group, gh = head % a.group;
  const int p = kvh * a.gtiles + gh / a.htile, h = gh % a.htile;
  int b = want;
  int64_t before = 0;
  const int64_t units = find_units(a, -1, &b, &before) * per;
  const Span sp = span_of(a, b);
  float* out = a.out + (int64_t)b * a.ldo + (int64_t)head * a.d;
  if (sp.tiles == 0) {
    for (int c = threadIdx.x; c < a.d; c += kJoinWaves * 64) out[c] = 0.f;
    return;
  }
  const int n = groups_for(a, units);
  const int64_t t0 = before * per + (int64_t)p * sp.tiles, t1 = t0 + sp.tiles - 1;
  const int w0 = (int)(((t0 + 1) * n - 1) / units), w1 = (int)(((t1 + 1) * n - 1) / units);
  if (w0 == w1) return;                         // written by the one workgroup that held it
  const int first = 2 * w0 + (units * w0 / n == t0 ? 0 : 1);
  float x[4] = {0.f, 0.f, 0.f, 0.f}, top = -INFINITY, sum = 0.f;
  for (int w = w0 + wv; w <= w1; w += kJoinWaves) {
    const float* src = a.part + ((int64_t)(w == w0 ? first : 2 * w) * a.htile + h) * (a.d + 2);
    const float t = fmaxf(top, src[a.d]), f = weight_of(top, t), u = weight_of(src[a.d], t);
    sum = sum * f + u * src[a.d + 1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = 64 * j + lane;
      x[j] = x[j] * f + (c < a.d ? u * src[c] : 0.f);
    }
    top = t;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) s_o[wv * 256 + 64 * j + lane] = x[j];
  if (lane == 0) {
    s_ml[2 * wv] = top;
    s_ml[2 * wv + 1] = sum;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.d; c += kJoinWaves * 64) {
    float t = -INFINITY, l = 0.f, y = 0.f;
    for (int w = 0; w < kJoinWaves; ++w) t = fmaxf(t, s_ml[2 * w]);
    for (int w = 0; w < kJoinWaves; ++w) {
      const float f = weight_of(s_ml[2 * w], t);
      l += f * s_ml[2 * w + 1];
      y += f * s_o[w * 256 + c];
    }
    out[c] = l != 0.f ? y / l : 0.f;
  }
}

template <typename E, int NJ, bool FULL>
void launch_attention(const AttnArgs& a, bool whole, hipStream_t st) {
  if (whole) {
    hipLaunchKernelGGL((k_paged_whole<E, NJ, FULL>), dim3(a.batch * a.kv_heads * a.gtiles), dim3(kWholeWaves * 64), 0,
                       st, a);
  } else {
    hipLaunchKernelGGL((k_paged_split<E, NJ, FULL>), dim3(a.groups), dim3(kSplitWaves * 64), 0, st, a);
    hipLaunchKernelGGL(k_paged_join, dim3(a.batch * a.heads), dim3(kJoinWaves * 64), 0, st, a);
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

int elem_size(int type) { return type == CV3_F32 ? 4 : 2; }

// What every call on a cache checks.
int check_cache(int type, const void* k, const void* v, int64_t pages, int64_t page, int kv_heads, int d) {
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
  CV3_REQUIRE(taken && taken_out && starts && (requests == 0 || (lengths && new_tokens && tables && total)) &&
                  (tokens == 0 || (slots && positions)) && (free_count == 0 || free_pages),
              CV3_EINVAL, "null operand");
  CV3_REQUIRE((requests == 0 || (const void*)total != (const void*)lengths) && taken_out != taken, CV3_EINVAL,
              "total and taken_out are arrays of their own: every workgroup reads lengths and taken");
  TabArgs a{lengths, new_tokens, free_pages, taken, tables, total, taken_out, starts, slots, positions,
            free_count, (int)requests, (int)page, (int)blocks, (int)tokens};
  const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(tokens, kTabThreads), 512));
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
  AppendArgs a{rows, n, ld, positions, slots, cos_tab, sin_tab, rope_rows, k_cache, v_cache, pages * page, q, ldq,
               (int)page, heads, kv_heads, d};
  // four channels a thread where rows start on 16 bytes (the tables are read by single floats)
  const bool wide = (uintptr_t)rows % 16 == 0 && ld % 4 == 0 && (!q || ((uintptr_t)q % 16 == 0 && ldq % 4 == 0));
  const unsigned per_row = (unsigned)(heads + 2 * kv_heads) * (d / 2) / (wide ? 4 : 1);
  const unsigned threads = std::min(256u, (per_row + 63) / 64 * 64), per = (per_row + threads - 1) / threads;
  CV3_REQUIRE(n <= (int64_t)INT32_MAX / per, CV3_EINVAL, "too many rows: %lld", (long long)n);
  if (wide)
    hipLaunchKernelGGL(k_append<4>, dim3((unsigned)n * per), dim3(threads), 0, stream_of(s), a, cache_type, per_row, per);
  else
    hipLaunchKernelGGL(k_append<1>, dim3((unsigned)n * per), dim3(threads), 0, stream_of(s), a, cache_type, per_row, per);
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
  CV3_REQUIRE(batch >= 0 && batch <= INT32_MAX / heads, CV3_EINVAL, "bad batch of %lld", (long long)batch);
  CV3_REQUIRE(ldq >= (int64_t)heads * d && ldo >= (int64_t)heads * d, CV3_EINVAL, "rows are too short for %d heads of %d",
              heads, d);
  if (batch == 0) return CV3_OK;
  CV3_REQUIRE(q && tables && lengths && out, CV3_EINVAL, "null operand");
  const int group = heads / kv_heads, htile = std::min(group, 16), gtiles = (group + htile - 1) / htile;
  AttnArgs a{q, ldq, k_cache, v_cache, tables, lengths, starts, out, ldo, nullptr, pages, blocks, (int)batch, (int)page,
             heads, kv_heads, group, gtiles, htile, d, 0, scale * 1.4426950408889634f};
  hipStream_t st = stream_of(s);
  bool whole = blocks * page <= 1024;
  if (!whole) {
    a.groups = 1024;
    void* part = nullptr;
    const int rc = scratch_alloc(&part, (size_t)2 * a.groups * htile * (d + 2) * sizeof(float), st);
    if (rc == CV3_ENOMEM) whole = true;      // one workgroup a pair needs no memory of its own
    else if (rc) return rc;
    a.part = (float*)part;
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
