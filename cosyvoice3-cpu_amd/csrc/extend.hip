// Attention of several new tokens per sequence over the paged cache: prompts in slices, drafted tokens, texts to score.
// Every query sees its sequence's keys up to itself (sdpa with a causal mask, cv3cpu/ops.py:267-300; the reference runs
// one sequence's prompt at a time over a contiguous cache, cv3cpu/models/qwen2.py:139-179).
//
// The queries are a ragged list: rows starts[b] .. starts[b + 1] are sequence b's last tokens, the last of them at
// position lengths[b] - 1.  Page ids, lengths and starts come from device memory and are checked where they are used.
#include "decode_common.hpp"   // DPP lane exchanges
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
  uint32_t page_inv;           // (2^32 - 1) / page
  int batch, page, heads, kv_heads, group, d, slots;
  float scale;                 // times log2(e)
  float* part;                 // [2 groups][rows of a tile][d + 2]: output, maximum, sum of a part of a row's keys
  int2* pairs;                 // [slots][kv heads]
  int groups, part_rows;
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

// ------------------------------------------------------------------------------------------------
// tiles on the matrix cores
// ------------------------------------------------------------------------------------------------

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kRows = 128;          // (token, head) rows of a workgroup: 32 a wave
constexpr int kThreads = 256;
constexpr int kSplitSlots = 2048;   // tiles of rows whose keys may be shared out
// Weights are held 2^10 up against a reference that a row's largest score has passed by so little that the 32 of a lane
// sum to no more than kMost, which float16 holds; so small planes end 2^-35 below the largest weight or lower.
constexpr float kUp = 10.f, kMost = 60000.f;

// How a cache's numbers become float16 operands.  float32: two planes, x 2^s = hi + lo within 2^-23 of x or 2^-25.
// bfloat16: one plane that holds x 2^s whole, down to 2^-17 of the largest's.  float16: as it is.
template <typename E>
struct Cell;
template <>
struct Cell<float> {
  typedef uint4 Raw;                // four channels
  static constexpr int N = 2;
  static constexpr bool SCALED = true;
  static __device__ __forceinline__ void four(const uint4& r, float* f) {
    f[0] = __uint_as_float(r.x), f[1] = __uint_as_float(r.y), f[2] = __uint_as_float(r.z), f[3] = __uint_as_float(r.w);
  }
};
template <>
struct Cell<__bf16> {
  typedef uint2 Raw;
  static constexpr int N = 1;
  static constexpr bool SCALED = true;
  static __device__ __forceinline__ void four(const uint2& r, float* f) {
    f[0] = __uint_as_float(r.x << 16), f[1] = __uint_as_float(r.x & 0xffff0000u);
    f[2] = __uint_as_float(r.y << 16), f[3] = __uint_as_float(r.y & 0xffff0000u);
  }
};
template <>
struct Cell<_Float16> {
  typedef uint2 Raw;
  static constexpr int N = 1;
  static constexpr bool SCALED = false;
  static __device__ __forceinline__ void four(const uint2&, float*) {}
};

// x up = hi + lo, each rounded to float16 from the exact sum of product and addend (mixed multiply-adds; `zero` and `one`
// are kept from folding, which would bring back a multiplication and two conversions).
struct Exact {
  float zero, one;
  __device__ __forceinline__ Exact() {
    zero = 0.f, one = 1.f;
    asm("" : "+s"(zero), "+s"(one));
  }
  __device__ __forceinline__ _Float16 scaled(float x, float up) const { return (_Float16)fmaf(x, up, zero); }
  static __device__ __forceinline__ _Float16 rest(float x, float up, _Float16 hi) { return (_Float16)fmaf(x, up, -(float)hi); }
};
__device__ __forceinline__ h2 half2_of(float a, float b) { return __builtin_convertvector((f32x2{a, b}), h2); }

// 2^15 over the power of two above x: what brings numbers of at most x below the largest float16.
__device__ __forceinline__ int up_of(float x) {
  return x > 0.f && x < INFINITY ? min(15 - __builtin_amdgcn_frexp_expf(x), 126) : 15;
}

// A tile of rows: rows row0 .. row0 + rows of sequence b's count * group (token, head of the group) rows, for one kv head.
struct Item {
  int b, kvh, first, base, len, row0, rows;
  __device__ __forceinline__ int hi_of(const ExtArgs& a, int r) const {     // keys seen: [lo, hi)
    return max(0, base + (row0 + r) / a.group + 1);
  }
  static __device__ __forceinline__ int lo_of(const ExtArgs& a, int hi) { return max(0, hi - a.window); }
};

// Slots: sequence b's tiles are those from floor(starts[b] group / 128) + b on, so that no two sequences share one.
__device__ __forceinline__ int slot_of(const ExtArgs& a, int first, int b) {
  return (int)((int64_t)first * a.group / kRows) + b;
}
__device__ __forceinline__ bool item_of(const ExtArgs& a, int b, int tile, Item& it) {
  const Seq s = seq_of(a, b);
  it.b = b;
  it.first = uniform(s.first), it.base = uniform(s.base), it.len = uniform(s.len);
  const int64_t left = (int64_t)uniform(s.count) * a.group - (int64_t)tile * kRows;
  if (tile < 0 || left <= 0) return false;
  it.row0 = tile * kRows;
  it.rows = (int)min(left, (int64_t)kRows);
  return true;
}
// Its tiles of KT keys: [t0, t1).
template <int KT>
__device__ __forceinline__ void tiles_of(const ExtArgs& a, const Item& it, int& t0, int& t1) {
  const int hi = it.hi_of(a, it.rows - 1);
  t0 = Item::lo_of(a, it.hi_of(a, 0)) / KT;
  t1 = max(t0, (hi + KT - 1) / KT);
  if (hi == 0) t1 = t0;
}
// The sequence of a slot, by every thread of the workgroup alike: how many begin at or before it.
__device__ __forceinline__ bool find_item(const ExtArgs& a, int slot, Item& it) {
  int before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
    const int b = b0 + (int)threadIdx.x;
    const bool at = b < a.batch && slot_of(a, (int)min((int64_t)max(a.starts[b], 0), a.n), b) <= slot;
    before += __syncthreads_count(at);
  }
  if (before == 0) return false;
  const int b = uniform(before - 1);
  return item_of(a, b, slot - uniform(slot_of(a, (int)min((int64_t)max(a.starts[b], 0), a.n), b)), it);
}

template <typename E, int ND>
struct Shape {
  static constexpr int DP = 32 * ND;                   // channels, padded
  static constexpr int N = Cell<E>::N;
  // Keys of a tile: 64 where the registers hold what a thread fetches of it ahead (8 x 800 queries over 5800 keys, 32 on 8
  // heads of 128: float32 2.98 ms with 64, 2.39 with 32; bfloat16 1.93 and 1.50; float16, not widened, 1.25 and 1.29).
  static constexpr int KT = ND <= 2 || (ND <= 4 && N == 1 && !Cell<E>::SCALED) ? 64 : 32;
  static constexpr int KS = DP + 8;                    // 16 rows, each this much on, lie in distinct banks
  static constexpr int BLOCKS = KT / 4 * (DP / 4), NB = (BLOCKS + kThreads - 1) / kThreads;
  // Where eight keys of a channel lie: step u takes keys 16 u + {0 .. 3, 8 .. 11} and {4 .. 7, 12 .. 15}, run r = 2 u + 0
  // and 1.  Runs are exchanged by channel bits so that 16 channels' reads of a run fall into distinct banks, and likewise
  // the writes of 16 threads, whose channels are 4 apart.
  static __device__ __forceinline__ int v_at(int channel, int run) {
    const int turn = KT == 64 ? (channel >> 1 & 7) ^ (channel >> 4 & 1) : (channel >> 2 & 3) ^ (channel >> 4 & 3);
    return channel * KT + 8 * (run ^ turn);
  }
  struct Mem {
    alignas(16) _Float16 k[N][KT * KS];                // [key][channel]
    alignas(16) _Float16 v[N][DP * KT];                // [channel][key], see v_at
    int64_t off[KT];
    uint64_t mask;
    float mx[kThreads / 64][2];
  };
};

// Rows of one item over key tiles [t0, t1).
//
// S^T = K Q^T on 32 keys x 32 rows x 16 channels: a lane has one row (two lanes share it) and half the keys of each 8,
// which is what O^T = V^T P^T wants as its second operand once V's keys lie in that order, so the weights stay in their
// lanes and the softmax needs one exchange between two lanes a tile.  Everything enters the float16 matrix cores as
// planes: queries and weights as two (float32 in 22 bits), keys and values by their type (Cell); lo x lo is left out
// (2^-24).  That is 3 products a product for float32 caches, 2 for the two-byte ones, where bfloat16 planes would take 6
// and 3.  Keys are scaled by a power of two a tile, values by one that only grows over the tiles.  What that loses, small
// numbers beside large ones, is looked for: a row whose scores could be off (their factor is large), whose outputs are
// below 2^-15 of the largest value, or whose results are not finite is formed again in float32 (RowSum).
template <typename E, int ND, bool FULL>
__device__ __forceinline__ void attend(const ExtArgs& a, const Item& it, int t0, int t1, int whole_t0, int whole_t1,
                                       float* part, typename Shape<E, ND>::Mem& mem) {
  typedef Shape<E, ND> S;
  typedef Cell<E> C;
  typedef typename C::Raw Raw;
  constexpr int KT = S::KT, DP = S::DP, N = S::N, KS = S::KS, NB = S::NB, CG = DP / 4;
  const int tid = threadIdx.x, lane = tid & 63, wv = uniform(tid >> 6), n = lane & 31, g = lane >> 5;
  const int d = FULL ? DP : a.d;
  const int row = wv * 32 + n;
  const bool valid = row < it.rows;
  const int flat = it.row0 + (valid ? row : 0);
  const int tok = it.first + flat / a.group, head = it.kvh * a.group + flat % a.group;
  const int hi = valid ? it.hi_of(a, row) : 0, lo = Item::lo_of(a, hi);
  // of the wave: keys that any of its rows sees [w_lo, w_hi), and that all of them see [s_lo, s_hi)
  const bool active = wv * 32 < it.rows;
  const int w_hi = active ? it.hi_of(a, min(it.rows, wv * 32 + 32) - 1) : 0, s_hi = active ? it.hi_of(a, wv * 32) : 0;
  const int w_lo = Item::lo_of(a, s_hi), s_lo = Item::lo_of(a, w_hi);
  const float* q = a.q + (int64_t)tok * a.ldq + (int64_t)head * d;

  const Exact exact;
  // the row's channels 16 s + 8 g .. + 8, in two planes
  h8 qh[DP / 16], ql[DP / 16];
  float factor;                        // of the row's scores: |scale| log2(e) over its power of two
  {
    float x[DP / 16][8], big = 0.f;
    const float sign = a.scale < 0.f ? -1.f : 1.f;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const int c = 16 * s + 8 * g + e;
        f32x4u y{};
        if (valid && (FULL || c < d)) y = *(const f32x4u*)(q + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[s][e + i] = sign * y.v[i];
          big = fmaxf(big, fabsf(y.v[i]));
        }
      }
    big = fmaxf(big, __shfl_xor(big, 32, kWave));
    const int up = up_of(big);
    factor = ldexpf(fabsf(a.scale), -up);
    const float unit = ldexpf(1.f, up);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        qh[s][e] = exact.scaled(x[s][e], unit);
        ql[s][e] = Exact::rest(x[s][e], unit, qh[s][e]);
      }
  }

  const int32_t* table = a.tables + (int64_t)it.b * a.blocks;
  const E* kc = (const E*)a.k + (int64_t)it.kvh * a.page * d;
  const E* vc = (const E*)a.v + (int64_t)it.kvh * a.page * d;
  // page id and row of this thread's key of tile t; -1: not there
  auto lookup = [&](int t, int32_t& id, uint32_t& in) {
    id = -1;
    in = 0;
    const int key = t * KT + tid;
    if (tid < KT && t < t1 && key < it.len) {
      uint32_t blk = __umulhi((uint32_t)key, a.page_inv);          // the quotient, or one less
      in = (uint32_t)key - blk * (uint32_t)a.page;
      if (in >= (uint32_t)a.page) ++blk, in -= (uint32_t)a.page;
      id = table[blk];
    }
  };
  auto place = [&](int32_t id, uint32_t in) {
    if (tid < 64) {
      const bool there = (uint32_t)id < (uint64_t)a.pages;
      if (tid < KT) mem.off[tid] = there ? ((int64_t)id * a.kv_heads * a.page + in) * d : -1;
      const uint64_t mask = __ballot(there);
      if (tid == 0) mem.mask = mask;
    }
  };
  // this thread's blocks of 4 keys x 4 channels
  Raw kr[NB][4], vr[NB][4];
  constexpr uint64_t kAll = ~(uint64_t)0 >> (64 - KT);
  uint64_t mask = 0;
  auto fetch = [&]() {
    mask = mem.mask;
    mask = (uint64_t)uniform((int64_t)mask);
    const bool all = mask == kAll;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int at = tid + j * kThreads, cg = at % CG, kg = at / CG;
      const bool on = (S::BLOCKS % kThreads == 0 || at < S::BLOCKS) && (FULL || 4 * cg < d);
      int64_t off[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) off[i] = mem.off[(S::BLOCKS % kThreads == 0 ? 4 * kg : 4 * kg % KT) + i];
#pragma unroll
      for (int i = 0; i < 4; ++i) kr[j][i] = vr[j][i] = Raw{};
      if (all) {
        if (on) {
#pragma unroll
          for (int i = 0; i < 4; ++i) kr[j][i] = *(const Raw*)(kc + off[i] + 4 * cg);
#pragma unroll
          for (int i = 0; i < 4; ++i) vr[j][i] = *(const Raw*)(vc + off[i] + 4 * cg);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (on && off[i] >= 0) {
            kr[j][i] = *(const Raw*)(kc + off[i] + 4 * cg);
            vr[j][i] = *(const Raw*)(vc + off[i] + 4 * cg);
          }
      }
    }
  };

  f32x16 o[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
  float top = -INFINITY, sum = 0.f;
  bool there = false, coarse = false;
  float v_big = 0.f;                   // largest |v| so far
  int v_up = 126, o_up = 126;          // powers of two of the values now, and of o

  if (t0 < t1) {
    int32_t id;
    uint32_t in;
    lookup(t0, id, in);
    place(id, in);
    __syncthreads();
    fetch();
    lookup(t0 + 1, id, in);
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      const uint64_t now = mask;
      float kx[NB][4][4], vx[NB][4][4];
      if constexpr (C::SCALED) {
        float km = 0.f, vm = 0.f;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            C::four(kr[j][i], kx[j][i]);
            C::four(vr[j][i], vx[j][i]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              km = fmaxf(km, fabsf(kx[j][i][c]));
              vm = fmaxf(vm, fabsf(vx[j][i][c]));
            }
          }
        km = wave_max_dpp(km);
        vm = wave_max_dpp(vm);
        if (lane == 0) mem.mx[wv][0] = km, mem.mx[wv][1] = vm;
      }
      __syncthreads();                 // the last tile is done with, and the maxima are there
      float down = 1.f;                // of the keys
      if constexpr (C::SCALED) {
        float km = 0.f;
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) {
          km = fmaxf(km, mem.mx[w][0]);
          v_big = fmaxf(v_big, mem.mx[w][1]);
        }
        const int up = uniform(up_of(km));
        down = ldexpf(1.f, -up);
        if (!(km < INFINITY)) coarse = true;
        v_up = uniform(min(v_up, v_big > 0.f ? up_of(v_big) : 126));
        const float ku = ldexpf(1.f, up), vu = ldexpf(1.f, v_up);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          const int at = tid + j * kThreads, cg = at % CG, kg = at / CG;
          if (S::BLOCKS % kThreads != 0 && at >= S::BLOCKS) continue;
          const int run = 2 * (kg >> 2) + (kg & 1), half = 4 * (kg >> 1 & 1);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            h4 h, l;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              h[c] = exact.scaled(kx[j][i][c], ku);
              if constexpr (N == 2) l[c] = Exact::rest(kx[j][i][c], ku, h[c]);
            }
            *(h4*)&mem.k[0][(4 * kg + i) * KS + 4 * cg] = h;
            if constexpr (N == 2) *(h4*)&mem.k[1][(4 * kg + i) * KS + 4 * cg] = l;
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            h4 h, l;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              h[i] = exact.scaled(vx[j][i][c], vu);
              if constexpr (N == 2) l[i] = Exact::rest(vx[j][i][c], vu, h[i]);
            }
            *(h4*)&mem.v[0][S::v_at(4 * cg + c, run) + half] = h;
            if constexpr (N == 2) *(h4*)&mem.v[1][S::v_at(4 * cg + c, run) + half] = l;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          const int at = tid + j * kThreads, cg = at % CG, kg = at / CG;
          if (S::BLOCKS % kThreads != 0 && at >= S::BLOCKS) continue;
          const int run = 2 * (kg >> 2) + (kg & 1), half = 4 * (kg >> 1 & 1);
          uint32_t x[4][2];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint2 kw = __builtin_bit_cast(uint2, kr[j][i]), vw = __builtin_bit_cast(uint2, vr[j][i]);
            *(uint2*)&mem.k[0][(4 * kg + i) * KS + 4 * cg] = kw;
            x[i][0] = vw.x, x[i][1] = vw.y;
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {      // 4 x 4 two-byte values turned by byte permutations
            const uint32_t sel = c % 2 ? 0x07060302u : 0x05040100u;
            *(uint2*)&mem.v[0][S::v_at(4 * cg + c, run) + half] = make_uint2(__builtin_amdgcn_perm(x[1][c / 2], x[0][c / 2], sel),
                                                                     __builtin_amdgcn_perm(x[3][c / 2], x[2][c / 2], sel));
          }
        }
      }
      place(id, in);
      __syncthreads();                 // the tile is there
      if (t + 1 < t1) {
        fetch();
        lookup(t + 2, id, in);
      }
      const int k0 = t * KT;
      if (k0 >= w_hi || k0 + KT <= w_lo) continue;

      f32x16 sc[KT / 32];
#pragma unroll
      for (int u = 0; u < KT / 32; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[u][r] = 0.f;
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        // products of one accumulator are kept apart: one that follows on another of the same waits for it
        h8 kx8[N][KT / 32];
#pragma unroll
        for (int u = 0; u < KT / 32; ++u)
#pragma unroll
          for (int j = 0; j < N; ++j) kx8[j][u] = *(const h8*)&mem.k[j][(32 * u + n) * KS + 16 * s + 8 * g];
#pragma unroll
        for (int u = 0; u < KT / 32; ++u) sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kx8[0][u], qh[s], sc[u], 0, 0, 0);
#pragma unroll
        for (int u = 0; u < KT / 32; ++u) sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kx8[0][u], ql[s], sc[u], 0, 0, 0);
        if constexpr (N == 2) {
#pragma unroll
          for (int u = 0; u < KT / 32; ++u) sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kx8[1][u], qh[s], sc[u], 0, 0, 0);
        }
      }
      // register r of sc[u]: key 32 u + 8 (r / 4) + 4 g + r % 4
      const bool every = now == kAll && k0 + KT <= s_hi && k0 >= s_lo;
      if (every) {
        there = true;
      } else {
        const int b0 = max(lo - k0, 0), b1 = min(hi - k0, KT);
        uint64_t m = b1 > b0 ? now & (~(uint64_t)0 >> (64 - b1)) & (~(uint64_t)0 << b0) : 0;
        there = there || m != 0;
        m >>= 4 * g;
#pragma unroll
        for (int u = 0; u < KT / 32; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const uint32_t bits = (uint32_t)(m >> 32 * u);
            sc[u][r] = bits >> (8 * (r / 4) + r % 4) & 1 ? sc[u][r] : -INFINITY;
          }
      }
      const float c = factor * down;
      // a score's terms are up to 2^30 c, and off by 2^-10 c where the small planes end: 2^-23 with 16 of them
      coarse = coarse || !(c <= (C::SCALED ? 0x1p-17f : 0x1p-8f));
      if (C::SCALED && o_up != v_up) {
        const float f = ldexpf(1.f, v_up - o_up);
        o_up = v_up;
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[i][r] *= f;
      }
      // Half by half, 32 keys: weights against the reference so far, whose sum of positive numbers shows whether one of
      // them is too large for float16.  Only then, and for rows that have met no key before, the largest score is found
      // and the reference moved.  The products of one half run beside the weights of the next.
#pragma unroll
      for (int w = 0; w < KT / 32; ++w) {
        h8 ph[2], pl[2];
        float part_sum;
        auto weigh = [&]() {
          const float ref = (top == -INFINITY ? 0.f : top) - kUp;
          part_sum = 0.f;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float x = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const float p0 = exp2_fast(fmaf(sc[w][8 * u + e], c, -ref)), p1 = exp2_fast(fmaf(sc[w][8 * u + e + 1], c, -ref));
              x += p0 + p1;
              const h2 h = half2_of(p0, p1);
              ph[u][e] = h[0], ph[u][e + 1] = h[1];
              pl[u][e] = Exact::rest(p0, exact.one, h[0]), pl[u][e + 1] = Exact::rest(p1, exact.one, h[1]);
            }
            part_sum += x;
          }
        };
        weigh();
        if (__any(!(part_sum <= kMost) || top == -INFINITY)) {
          float mx = sc[w][0];
#pragma unroll
          for (int r = 1; r < 16; ++r) mx = fmaxf(mx, sc[w][r]);
          const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
          mx = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])) * c;
          const float up = fmaxf(mx, top), f = weight_of(top, up);
          top = up;
          sum *= f;
#pragma unroll
          for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] *= f;
          weigh();
        }
        sum += part_sum;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          // products of one accumulator are kept apart, as above
          h8 vx8[N][ND];
#pragma unroll
          for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) vx8[j][i] = *(const h8*)&mem.v[j][S::v_at(32 * i + n, 4 * w + 2 * u + g)];
#pragma unroll
          for (int i = 0; i < ND; ++i) o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vx8[0][i], ph[u], o[i], 0, 0, 0);
#pragma unroll
          for (int i = 0; i < ND; ++i) o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vx8[0][i], pl[u], o[i], 0, 0, 0);
          if constexpr (N == 2) {
#pragma unroll
            for (int i = 0; i < ND; ++i) o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vx8[1][i], ph[u], o[i], 0, 0, 0);
          }
        }
      }
    }
  }

  // register r of o[i]: channel 32 i + 8 (r / 4) + 4 g + r % 4
  sum += __shfl_xor(sum, 32, kWave);
  const float inv = 1.f / sum;
  float big = 0.f;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      o[i][r] *= inv;
      odd = odd || !(fabsf(o[i][r]) < INFINITY);
      big = fmaxf(big, fabsf(o[i][r]));
    }
  big = fmaxf(big, __shfl_xor(big, 32, kWave));
  odd = odd || coarse || !(sum > 0.f && sum < INFINITY) || (C::SCALED && big < 1.f && v_big > 0.f);
  odd = __shfl_xor((int)odd, 32, kWave) || odd;
  const bool again = valid && there && odd, whole = t0 == whole_t0 && t1 == whole_t1;
  const float unit = C::SCALED ? ldexpf(1.f, -o_up) : 1.f;
  float* dst = whole ? a.out + (int64_t)tok * a.ldo + (int64_t)head * d : part + (int64_t)row * (d + 2);
  if (valid && !again) {
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int c = 32 * i + 8 * (r / 4) + 4 * g;
        f32x4u x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x.v[e] = there ? o[i][r + e] * unit : 0.f;
        if (FULL || c < d) *(f32x4u*)(dst + c) = x;
      }
    if (!whole && g == 0) {
      dst[d] = there ? top : -INFINITY;
      dst[d + 1] = there ? sum : 0.f;
    }
  }
  uint64_t rest = __ballot(again && g == 0);
  while (rest) {
    const int r = uniform(__ffsll((unsigned long long)rest) - 1);
    rest &= rest - 1;
    const int r_tok = uniform(__shfl(tok, r, kWave)), r_head = uniform(__shfl(head, r, kWave));
    const int r_hi = min(uniform(__shfl(hi, r, kWave)), t1 * KT), r_lo = max(uniform(__shfl(lo, r, kWave)), t0 * KT);
    RowSum<E> x;
    x.run(a, it.b, it.kvh, a.q + (int64_t)r_tok * a.ldq + (int64_t)r_head * d, r_lo, r_hi);
    const bool none = x.there && x.top == -INFINITY;       // scores of -inf alone
    float* to = whole ? a.out + (int64_t)r_tok * a.ldo + (int64_t)r_head * d : part + (int64_t)(wv * 32 + r) * (d + 2);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (64 * i + lane < d) to[64 * i + lane] = !x.there || (none && !whole) ? 0.f : x.o[i] / x.sum;
    if (!whole && lane == 0) {
      to[d] = none ? kNoScore : x.top;
      to[d + 1] = x.sum * 0x1p10f;
    }
  }
}

// One workgroup a (tile of rows, kv head).
template <typename E, int ND, bool FULL>
__global__ __launch_bounds__(kThreads, ND <= 4 ? 2 : 1) void k_extend_whole(ExtArgs a) {
  __shared__ typename Shape<E, ND>::Mem mem;
  Item it;
  // the last tiles of a sequence see the most keys: they go first
  if (!find_item(a, a.slots - 1 - (int)(blockIdx.x / (unsigned)a.kv_heads), it)) return;
  it.kvh = (int)(blockIdx.x % (unsigned)a.kv_heads);
  int t0, t1;
  tiles_of<Shape<E, ND>::KT>(a, it, t0, t1);
  attend<E, ND, FULL>(a, it, t0, t1, t0, t1, nullptr, mem);
}

// A workgroup's share of the (slot, kv head, key tile) units, in that order.
struct Plan {
  int64_t before[kSplitSlots + 1];   // key tiles of one kv head in the slots ahead
  int32_t slot[kSplitSlots];         // a sequence's first slot
  int64_t sum[kThreads / 64];
};
// The last i of [0, n) with v[i] <= x; v[0] <= x.
template <typename T>
__device__ __forceinline__ int last_at(const T* v, int n, T x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// The units shared out evenly over `groups` workgroups by what the device holds: a long cache with few rows, a ragged
// batch and a causal triangle all fill the machine, and a captured launch serves every length.  Every workgroup sums
// over the slots by itself.  An item (slot, kv head) that one workgroup holds whole is written by it; of one that
// crosses workgroups each leaves its rows' outputs, maxima and sums in `part` (slot 2 w, or 2 w + 1 where the item
// begins inside w's share), and k_extend_join adds them up.  The workgroup that begins an item enters it into `pairs`:
// its first part and last workgroup, or -1.  Shares that follow each other go to one XCD, whose L2 they share keys in.
template <typename E, int ND, bool FULL>
__global__ __launch_bounds__(kThreads, ND <= 4 ? 2 : 1) void k_extend_split(ExtArgs a) {
  constexpr int KT = Shape<E, ND>::KT;
  __shared__ union {
    typename Shape<E, ND>::Mem mem;
    Plan plan;
  } lds;
  Plan& p = lds.plan;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, slots = a.slots;
  const int w = (int)(blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8);
  for (int b = tid; b < a.batch; b += kThreads)
    p.slot[b] = slot_of(a, (int)min((int64_t)max(a.starts[b], 0), a.n), b);
  __syncthreads();
  constexpr int kEach = kSplitSlots / kThreads;
  const int each = (slots + kThreads - 1) / kThreads;
  int64_t mine[kEach], all = 0;
#pragma unroll 1
  for (int i = 0; i < each; ++i) {
    const int s = tid * each + i;
    int64_t units = 0;
    if (s < slots && p.slot[0] <= s) {
      const int b = last_at(p.slot, a.batch, (int32_t)s);
      const Seq q = seq_of(a, b);
      const int64_t row0 = (int64_t)(s - p.slot[b]) * kRows, rows = min((int64_t)q.count * a.group - row0, (int64_t)kRows);
      if (row0 >= 0 && rows > 0) {
        Item it{b, 0, q.first, q.base, q.len, (int)row0, (int)rows};
        int t0, t1;
        tiles_of<KT>(a, it, t0, t1);
        units = t1 - t0;
      }
    }
    mine[i] = units;
    all += units;
  }
  int64_t up = all;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t u = __shfl_up(up, o, kWave);
    if (lane >= o) up += u;
  }
  if (lane == 63) p.sum[wv] = up;
  __syncthreads();
  int64_t at = up - all, total = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    if (i < wv) at += p.sum[i];
    total += p.sum[i];
  }
#pragma unroll 1
  for (int i = 0; i < each; ++i) {
    const int s = tid * each + i;
    if (s < slots) p.before[s] = at;
    at += mine[i];
  }
  __syncthreads();
  total = uniform(total) * a.kv_heads;
  const int64_t n = min((int64_t)a.groups, total);
  if (w >= n) return;
  const int64_t first = total * w / n, end = total * (w + 1) / n;
  int slot = uniform(last_at(p.before, slots, first / a.kv_heads));
  int64_t in = first - uniform(p.before[slot]) * a.kv_heads;          // the unit within the slot: [kv head][key tile]
  int b = uniform(last_at(p.slot, a.batch, (int32_t)slot));
  __syncthreads();                     // the plan's memory is the tiles' from here on

  at = first;
  while (at < end) {
    Item it{};
    int t0 = 0, t1 = 0;
    const int tile = slot - slot_of(a, uniform((int)min((int64_t)max(a.starts[b], 0), a.n)), b);
    if (item_of(a, b, tile, it)) tiles_of<KT>(a, it, t0, t1);
    const int units = t1 - t0;
    if (in >= (int64_t)units * a.kv_heads) {           // the next slot; of the next sequence, where it begins there
      in -= (int64_t)units * a.kv_heads;
      if (++slot >= slots) return;                     // lengths that changed under the call
      while (b + 1 < a.batch && slot_of(a, uniform((int)min((int64_t)max(a.starts[b + 1], 0), a.n)), b + 1) <= slot) ++b;
      continue;
    }
    it.kvh = (int)(in / units);
    const int t = (int)(in - (int64_t)it.kvh * units), take = (int)min((int64_t)(units - t), end - at);
    const int place = 2 * w + (at == first ? 0 : 1);
    if (tid == 0 && t == 0) {
      const bool whole = take == units;
      a.pairs[(int64_t)slot * a.kv_heads + it.kvh] =
          make_int2(whole ? -1 : place, whole ? 0 : (int)(((at + units) * n - 1) / total));
    }
    attend<E, ND, FULL>(a, it, t0 + t, t0 + t + take, t0, t1, a.part + (int64_t)place * a.part_rows * (a.d + 2), lds.mem);
    __syncthreads();                   // before the next item's first page ids
    at += take;
    in += take;
  }
}

// Rows of items that crossed workgroups, and zeros for those with no key to see: a wave a row at a time, eight rows each.
constexpr int kJoinRows = 32;
__global__ __launch_bounds__(kThreads) void k_extend_join(ExtArgs a) {
  const int lane = threadIdx.x & 63, wv = uniform((int)threadIdx.x >> 6);
  const int slot = (int)(blockIdx.x / (unsigned)a.kv_heads), row0 = blockIdx.y * kJoinRows;
  Item it;
  if (!find_item(a, slot, it) || row0 >= it.rows) return;
  it.kvh = (int)(blockIdx.x % (unsigned)a.kv_heads);
  const bool none = it.hi_of(a, it.rows - 1) == 0;
  const int2 pair = none ? make_int2(0, 0) : a.pairs[blockIdx.x];
  if (pair.x < 0) return;              // written by the one workgroup that held it
  const int w0 = min(pair.x >> 1, a.groups - 1), count = none ? 0 : min(pair.y, a.groups - 1) - w0 + 1;
  for (int r = row0 + wv; r < min(row0 + kJoinRows, it.rows); r += kThreads / 64) {
    const int flat = it.row0 + r, head = it.kvh * a.group + flat % a.group;
    float* out = a.out + (int64_t)(it.first + flat / a.group) * a.ldo + (int64_t)head * a.d;
    float x[4], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = 0.f;
    constexpr int kAhead = 4;
    for (int i = 0; i < count; i += kAhead) {
      float y[kAhead][4], t[kAhead], l[kAhead], now = top;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int m = min(i + u, count - 1);
        const float* src = a.part + ((int64_t)(m ? 2 * (w0 + m) : pair.x) * a.part_rows + r) * (a.d + 2);
        t[u] = i + u < count ? src[a.d] : -INFINITY;
        l[u] = src[a.d + 1];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[u][j] = 64 * j + lane < a.d ? src[64 * j + lane] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) now = fmaxf(now, t[u]);
      const float f = weight_of(top, now);
      sum *= f;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] *= f;
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (t[u] != -INFINITY) {
          const float g = weight_of(t[u], now) * l[u];
          sum += g;
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] += g * y[u][j];
        }
      top = now;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (64 * j + lane < a.d) out[64 * j + lane] = top != -INFINITY ? x[j] / sum : 0.f;
  }
}

constexpr int groups_of(int d) { return d <= 128 ? 512 : 256; }     // workgroups that the registers let run at once

template <typename E, int ND, bool FULL>
void launch_tiles(const ExtArgs& a, hipStream_t st) {
  if (!a.part) {
    hipLaunchKernelGGL((k_extend_whole<E, ND, FULL>), dim3((unsigned)a.slots * a.kv_heads), dim3(kThreads), 0, st, a);
    return;
  }
  hipLaunchKernelGGL((k_extend_split<E, ND, FULL>), dim3(a.groups), dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL(k_extend_join, dim3((unsigned)a.slots * a.kv_heads, (unsigned)ceil_div(a.part_rows, kJoinRows)), dim3(kThreads),
                     0, st, a);
}

template <typename E>
void extend_for(const ExtArgs& a, hipStream_t st) {
  switch ((a.d + 31) / 32) {
    case 1:
    case 2: a.d == 64 ? launch_tiles<E, 2, true>(a, st) : launch_tiles<E, 2, false>(a, st); break;
    case 3: launch_tiles<E, 3, false>(a, st); break;
    case 4: a.d == 128 ? launch_tiles<E, 4, true>(a, st) : launch_tiles<E, 4, false>(a, st); break;
    case 5:
    case 6: launch_tiles<E, 6, false>(a, st); break;
    default: launch_tiles<E, 8, false>(a, st);
  }
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
            (int)std::min<int64_t>(window, INT32_MAX), (uint32_t)(0xffffffffu / (uint32_t)page), (int)batch, (int)page, heads, kv_heads, heads / kv_heads, d,
            (int)(n * (heads / kv_heads) / kRows + batch), scale * 1.4426950408889634f, nullptr, nullptr, 0, 0};
  hipStream_t st = stream_of(s);
  const int64_t cap = blocks * page, items = (int64_t)a.slots * kv_heads;
  const bool whole = a.slots > kSplitSlots || cap <= 256 || items >= 8192;
  if (!whole) {
    a.groups = groups_of(d);
    a.part_rows = (int)std::min<int64_t>(kRows, n * a.group);
    const size_t parts = (size_t)2 * a.groups * a.part_rows * (d + 2) * sizeof(float);      // a multiple of 8
    void* work = nullptr;
    const int rc = scratch_alloc(&work, parts + (size_t)items * sizeof(int2), st);
    if (rc && rc != CV3_ENOMEM) return rc;     // without memory: one workgroup an item
    a.part = (float*)work;
    a.pairs = (int2*)((char*)work + parts);
  }
  if (cache_type == CV3_F32) extend_for<float>(a, st);
  else if (cache_type == CV3_F16) extend_for<_Float16>(a, st);
  else extend_for<__bf16>(a, st);
  const hipError_t err = hipGetLastError();
  const int rc = a.part ? scratch_free(a.part, st) : CV3_OK;
  CV3_REQUIRE(err == hipSuccess, CV3_EHIP, "kernel launch failed: %s", hipGetErrorString(err));
  return rc;
}

}  // extern "C"
