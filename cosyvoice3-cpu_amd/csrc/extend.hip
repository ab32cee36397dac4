// Attention of several new tokens per sequence over the paged cache: prompts in slices, drafted tokens, texts to score.
// Every query sees its sequence's keys up to itself (sdpa with a causal mask, cv3cpu/ops.py:267-300; the reference runs
// one sequence's prompt at a time over a contiguous cache, cv3cpu/models/qwen2.py:139-179).
//
// The queries are a ragged list: rows starts[b] .. starts[b + 1] are sequence b's last tokens, the last of them at
// position lengths[b] - 1.  Page ids, lengths and starts come from device memory and are checked where they are used.
#include "decode_common.hpp"   // DPP lane exchanges
#include "paged_common.hpp"

#include <algorithm>
#include <type_traits>

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
  float* part;                 // [places][rows of a tile][d]: outputs of parts of the rows' keys
  float2* part_ml;             // [places][rows of a tile]: their maxima and sums
  struct Piece* pieces;        // parts of items, a workgroup each
  struct Piece* cuts;          // the first part of every item that has several
  int* counts;                 // of cuts and pieces; whether these are sorted
  int groups, part_rows, pieces_most, places, cuts_most;
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
// for the sum.
template <typename E>
struct RowSum {
  float o[4], top, sum;
  bool there;                  // a key, whatever its score

  // The outputs, divided; sums of values near the largest float, which leave its range, once more with weights 2^-40 down.
  __device__ __forceinline__ void run(const ExtArgs& a, int b, int kvh, const float* q, int lo, int hi) {
    float down = 1.f;
#pragma unroll 1
    for (;; down = 0x1p-40f) {
      sums(a, b, kvh, q, lo, hi, down);
      bool out = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) out = out || !(fabsf(o[i]) < INFINITY);
      if (down != 1.f || !(__any(out) && sum < INFINITY)) break;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] / sum / down;
  }
  __device__ __forceinline__ void sums(const ExtArgs& a, int b, int kvh, const float* q, int lo, int hi, float down) {
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
      // the values of kAhead keys at a time
      constexpr int kAhead = 8;
      auto add = [&](auto many) {
        constexpr int N = decltype(many)::value;
        float w[N], v[N][4];
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int j = uniform(__ffsll((unsigned long long)seen) - 1);
          seen &= seen - 1;
          w[k] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), j)) * down;
          const E* vr = (const E*)a.v + (int64_t)readlane64((uint64_t)off, j);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[k][i] = 64 * i + lane < a.d ? to_float(vr[64 * i + lane]) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = fmaf(w[k], v[k][i], o[i]);
      };
      while (__popcll(seen) >= kAhead) add(std::integral_constant<int, kAhead>());
      while (seen) add(std::integral_constant<int, 1>());
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

constexpr int kWaveRows = 32;       // (token, head) rows of a wave
constexpr int kSplitSlots = 1024;   // tiles of rows whose keys may be shared out
// Tables up to here are not worth a plan: 12 prompts of up to 900 tokens (14 on 2 heads of 64, float32) 49 us without, 62 with,
// float16 37 and 49.  The table's width decides, since the host knows no lengths: the same prompts in wider tables are planned.
constexpr int kWholeKeys = 1024;
// And up to here where items nearly fill the machine and are taken in their order: 8 ragged prompts of up to 2000 tokens (14
// on 2 heads of 64, float32) 114 us planned, 102 whole.  Further up one long sequence among short ones would be the last by
// far (a slice of 500 over 4000 keys among 16 prompts of 500: 100 planned, 160 whole), with fewer items the machine is not
// full (a prompt of 2000: 63 and 80).
constexpr int kOrderKeys = 2048;
// Items from which their order counts, more than one a compute unit: 12 prompts of up to 900 tokens 66 us by slots, 50 with
// the longest first, 16 of 1000 156 and 136; where all are alike (24 x 60 queries over 360 keys) 52 and 53.
constexpr int kOrderItems = 256;
// Rows a sequence, on average, that one wave takes: 4 tokens of 7 heads a kv head over 504 keys 12 us, 16 with four waves.
// For d > 64 one wave fetches too slowly (8 x 9 queries over 709 keys, 4 heads of 128 a kv head, 65 us against 35).
constexpr int kFewRows = 48;

// Weights are held 2^12 up against a reference that a row's largest score has passed by so little that no eight of them sum
// to more than kMost, which float16 holds; so small planes end 2^-37 below the largest weight or lower.
constexpr float kUp = 12.f, kMost = 60000.f;

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

__device__ __forceinline__ h2 half2_of(float a, float b) { return __builtin_convertvector((f32x2{a, b}), h2); }

// Two numbers times `up`, and what float16 leaves of them: two mixed multiply-adds each, into the halves of a register, of
// which the compiler makes three.  h of rest2_of depends on the numbers, so that an instruction lies between an exponential
// and its use there; what the matrix cores read passes settled() first, since the compiler does not see that these are vector
// instructions.
__device__ __forceinline__ h2 scaled2_of(float x0, float x1, float up) {
  h2 h;
  asm("v_fma_mixlo_f16 %0, %1, %2, 0" : "=v"(h) : "v"(x0), "s"(up));
  asm("v_fma_mixhi_f16 %0, %1, %2, 0" : "+v"(h) : "v"(x1), "s"(up));
  return h;
}
__device__ __forceinline__ h2 rest2_of(float x0, float x1, float up, h2 h) {
  h2 l;
  asm("v_fma_mixlo_f16 %0, %1, %2, -%3 op_sel_hi:[0,0,1]" : "=v"(l) : "v"(x0), "s"(up), "v"(h));
  asm("v_fma_mixhi_f16 %0, %1, %2, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(l) : "v"(x1), "s"(up), "v"(h));
  return l;
}
// The largest of x, |a| and |b|, NaN if one is: v_max3 would pass NaNs over, but forget x for a signalling one.  (fmaxf first
// makes quiet what it is given, an instruction a number.)
__device__ __forceinline__ float max_abs(float x, float a, float b) {
  asm("v_maximum3_f32 %0, %0, |%1|, |%2|" : "+v"(x) : "v"(a), "v"(b));
  return x;
}
// 2^e of the whole wave, e from -126 to 127
__device__ __forceinline__ float power_of(int e) { return __int_as_float((127 + e) << 23); }
__device__ __forceinline__ void settled(h8& x) { asm("s_nop 1" : "+v"(x)); }

// 2^15 over the power of two above x: what brings numbers of at most x below the largest float16.
__device__ __forceinline__ int up_of(float x) {
  return x > 0.f && x < INFINITY ? min(15 - __builtin_amdgcn_frexp_expf(x), 126) : 15;
}

// A tile of rows, a workgroup's: rows row0 .. row0 + rows of sequence b's count * group (token, head of the group) rows,
// for one kv head.
struct Item {
  int b, kvh, first, base, len, row0, rows;
  __device__ __forceinline__ int hi_of(const ExtArgs& a, int r) const {     // keys seen: [lo, hi)
    return max(0, base + (row0 + r) / a.group + 1);
  }
  static __device__ __forceinline__ int lo_of(const ExtArgs& a, int hi) { return max(0, hi - a.window); }
};

// Slots: sequence b's tiles of W waves are those from floor(starts[b] group / (32 W)) + b on, so that no two sequences
// share one.
template <int W>
__device__ __forceinline__ int slot_of(const ExtArgs& a, int first, int b) {
  return (int)((int64_t)first * a.group / (kWaveRows * W)) + b;
}
template <int W>
__device__ __forceinline__ int first_slot(const ExtArgs& a, int b) {
  return slot_of<W>(a, (int)min((int64_t)max(a.starts[b], 0), a.n), b);
}
template <int W>
__device__ __forceinline__ bool item_of(const ExtArgs& a, int b, int tile, Item& it) {
  constexpr int kRows = kWaveRows * W;
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
template <int W, int WAVES = W>
__device__ __forceinline__ bool find_item(const ExtArgs& a, int slot, Item& it) {
  int before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64 * WAVES) {
    const int b = b0 + (int)threadIdx.x;
    before += __syncthreads_count(b < a.batch && first_slot<W>(a, b) <= slot);
  }
  if (before == 0) return false;
  const int b = uniform(before - 1);
  return item_of<W>(a, b, slot - uniform(first_slot<W>(a, b)), it);
}

// One value of a wave's 64, by lane exchanges within rows of 16 and four lane reads.
template <typename F>
__device__ __forceinline__ uint32_t wave_fold(uint32_t v, F f) {
  v = f(v, dpp32<kDppXor1>(v));
  v = f(v, dpp32<kDppXor2>(v));
  v = f(v, dpp32<kDppHalfMirror>(v));
  v = f(v, dpp32<kDppMirror>(v));
  return f(f((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16)),
           f((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48)));
}
__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v) {
  return wave_fold(v, [](uint32_t x, uint32_t y) { return x + y; });
}
// Of numbers that are not negative, by their bits; NaN if one is.
__device__ __forceinline__ float wave_most(float v) {
  return __uint_as_float(wave_fold(__float_as_uint(v), [](uint32_t x, uint32_t y) { return max(x, y); }));
}
// Item `at` of up to 64 sequences in the order of their last key's tile, the furthest first: a sequence a lane, the level
// by bisection of how many lie at or above it, by every wave for itself.
template <int KT, int W>
__device__ __forceinline__ bool find_by_keys(const ExtArgs& a, int at, Item& it) {
  constexpr int kRows = kWaveRows * W;
  const int lane = threadIdx.x & 63;
  const Seq s = lane < a.batch ? seq_of(a, lane) : Seq{};
  const int all = (s.count * a.group + kRows - 1) / kRows;
  // how many of the sequence's tiles of rows see a key past L tiles of keys: its last ones
  auto past = [&](int L) {
    const int64_t x = (int64_t)L * KT - s.base;      // tokens before the first that does
    return L < 0 || x <= 0 ? all : x >= s.count ? 0 : all - (int)x * a.group / kRows;
  };
  int lo = -1, hi = (int)((a.blocks * a.page + KT - 1) / KT);
  if ((uint32_t)at >= wave_sum_u32((uint32_t)all)) return false;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (wave_sum_u32((uint32_t)past(mid)) > (uint32_t)at) lo = mid; else hi = mid;
  }
  const int above = past(hi), mine = past(lo) - above;
  int up = mine, before = (int)wave_sum_u32((uint32_t)above);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(up, o, kWave);
    if (lane >= o) up += u;
  }
  before += up - mine;                       // items ahead of this sequence's at the level
  const int b = uniform(__ffsll((unsigned long long)__ballot(at >= before && at < before + mine)) - 1);
  return item_of<W>(a, b, __builtin_amdgcn_readlane(all - above - 1 - (at - before), b), it);
}

// The sum over a query's channels that lie where its small plane ends, up to 2^-18 of its largest, of the largest key of
// [lo, hi) there; by one wave.
template <typename E>
__device__ __forceinline__ float key_ends(const ExtArgs& a, int b, int kvh, const float* q, int lo, int hi) {
  const int lane = threadIdx.x & 63;
  const int32_t* table = a.tables + (int64_t)b * a.blocks;
  float big = 0.f, sum = 0.f;
#pragma unroll 1
  for (int c = lane; c < a.d; c += 64) big = fmaxf(big, fabsf(q[c]));
  const float unit = ldexpf(1.f, up_of(wave_most(big)));
#pragma unroll 1
  for (int c = 0; c < a.d; ++c) {
    const float x = fabsf(__uint_as_float((uint32_t)uniform((int)__float_as_uint(q[c]))) * unit);
    if (x == 0.f || !(x < 0x1p-3f)) continue;
    float most = 0.f;
#pragma unroll 4
    for (int key = lo + lane; key < hi; key += 64) {
      const uint32_t blk = (uint32_t)key / (uint32_t)a.page;
      const int32_t id = table[blk];
      if ((uint32_t)id < (uint64_t)a.pages)
        most = fmaxf(most, fabsf(to_float(((const E*)a.k)[(((int64_t)id * a.kv_heads + kvh) * a.page + (key - (int64_t)blk * a.page)) * a.d + c])));
    }
    sum += wave_most(most);
  }
  return sum;
}

template <typename E, int ND, int W>
struct Shape {
  static constexpr int T = 64 * W;                     // threads
  static constexpr int DP = 32 * ND;                   // channels, padded
  static constexpr int N = Cell<E>::N;
  // Keys of a tile: 64 where the registers hold what a thread fetches of it ahead (8 x 800 queries over 5800 keys, 32 on 8
  // heads of 128: float32 2.98 ms with 64, 2.39 with 32; bfloat16 1.93 and 1.50; float16, not widened, 1.25 and 1.29).
  // One wave alone fetches all of a tile: 32.
  static constexpr int KT = W > 1 && (ND <= 2 || (ND <= 4 && N == 1 && !Cell<E>::SCALED)) ? 64 : 32;
  static constexpr int KS = DP + 8;                    // 16 rows, each this much on, lie in distinct banks
  static constexpr int BLOCKS = KT / 4 * (DP / 4), NB = (BLOCKS + T - 1) / T;
  // Where eight keys of a channel lie: step u takes keys 16 u + {0 .. 3, 8 .. 11} and {4 .. 7, 12 .. 15}, run r = 2 u + 0
  // and 1.  Runs are exchanged by channel bits so that 16 channels' reads of a run fall into distinct banks, and likewise
  // the writes of 16 threads, whose channels are 4 apart.
  static __device__ __forceinline__ int v_at(int channel, int run) {
    const int turn = KT == 64 ? (channel >> 1 & 7) ^ (channel >> 4 & 1) : (channel >> 2 & 3) ^ (channel >> 4 & 3);
    return channel * KT + 8 * (run ^ turn);
  }
  // v_at(32 i + n, run + g) from v_at(n, g), run even
  static __device__ __forceinline__ int v_at(int first, int i, int run) {
    return 32 * i * KT + (first ^ 8 * (KT == 64 ? run : run ^ 2 * (i & 1)));
  }
  struct Mem {
    alignas(16) _Float16 k[N][KT * KS];                // [key][channel]
    alignas(16) _Float16 v[N][DP * KT];                // [channel][key], see v_at
    int64_t off[KT];
    uint64_t mask;
    float mx[W][2];
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
// numbers beside large ones, is looked for: a row whose scores could be off by 2^-20 of the largest (its largest number and
// the keys' are in different channels, and far above what makes its scores), whose outputs are
// below 2^-15 of the largest value or so small that many keys of next to no weight could be missed in them, or whose results
// are not finite is formed again in float32 (RowSum).
//
// Bound by the matrix cores and the vector units, which share a wave's time: of some 3900 cycles a tile of 64 keys (float16,
// d = 64, two workgroups a CU) the products with their operands take about half, exponentials and planes of the weights a
// quarter, addresses and loads 750, barriers 430; float32 widens its tile for another 900.  500 queries over 60501 keys
// (14 on 2 heads, float16) 266 us, 410 TFLOP/s of 4 d flops a score: twice that in products, where a library's large
// product of float16 reaches 1060.  12 slices of up to 800 over 5800 keys (32 on 8 heads of 128, bfloat16) 640 us, 420.
// From 193 channels on, float32 and bfloat16 spill (100 bytes a lane): one prompt of 500 (8 on 2 heads of 256) 96 and 80 us.
template <typename E, int ND, bool FULL, int W>
__device__ __forceinline__ void attend(const ExtArgs& a, const Item& it, int t0, int t1, bool whole, float* part,
                                       float2* part_ml, typename Shape<E, ND, W>::Mem& mem) {
  typedef Shape<E, ND, W> S;
  typedef Cell<E> C;
  typedef typename C::Raw Raw;
  constexpr int KT = S::KT, DP = S::DP, N = S::N, KS = S::KS, NB = S::NB, CG = DP / 4;
  const int tid = threadIdx.x, lane = tid & 63, wv = uniform(tid >> 6), n = lane & 31, g = lane >> 5;
  const int d = FULL ? DP : a.d;
  const int row = wv * kWaveRows + n;
  const bool valid = row < it.rows;
  auto token_of = [&](int r) { return it.first + (it.row0 + r) / a.group; };
  auto head_of = [&](int r) { return it.kvh * a.group + (it.row0 + r) % a.group; };
  // worked out where they are needed, rather than held over the keys
  auto row_now = [&]() {
    int t = tid;
    asm volatile("" : "+v"(t));
    return wv * kWaveRows + (t & 31);
  };
  auto hi_now = [&]() { return valid ? it.hi_of(a, row_now()) : 0; };
  // of the wave: keys that any of its rows sees [w_lo, w_hi), and that all of them see [s_lo, s_hi)
  const bool active = wv * kWaveRows < it.rows;
  const int w_hi = active ? it.hi_of(a, min(it.rows, (wv + 1) * kWaveRows) - 1) : 0;
  const int s_hi = active ? it.hi_of(a, wv * kWaveRows) : 0;
  const int w_lo = Item::lo_of(a, s_hi), s_lo = Item::lo_of(a, w_hi);

  // Weights come up by 2^kUp after the exponential (kHold) where keys and values are widened: in its argument 12 costs 3 bits
  // of the weights near the largest (12 prompts, bfloat16: 2.4e-7 of the results' root mean square against 2.8e-7).  float16
  // caches have it in the argument (kRef): no row of theirs has fewer bits than a row of the one-token form.
  constexpr float kHold = C::SCALED ? 0x1p12f : 1.f, kRef = C::SCALED ? 0.f : kUp;
  // the row's channels 16 s + 8 g .. + 8, in two planes
  h8 qh[DP / 16], ql[DP / 16];
  float factor;                        // of the row's scores: |scale| log2(e) over its power of two
  bool ends = true;                    // the row has numbers of up to 2^-18 of its largest, where its small plane ends
  {
    const float* q = a.q + (int64_t)token_of(valid ? row : 0) * a.ldq + (int64_t)head_of(valid ? row : 0) * d;
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
    if constexpr (!C::SCALED) {          // elsewhere the keys' own size tells that they hardly matter
      uint32_t least = ~0u;
#pragma unroll
      for (int s = 0; s < DP / 16; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) least = min(least, __float_as_uint(fabsf(x[s][e])) - 1);
      least = min(least, (uint32_t)__shfl_xor((int)least, 32, kWave));
      ends = least < __float_as_uint(ldexpf(0x1p-3f, -up)) - 1;
    }
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        qh[s][e] = (_Float16)(x[s][e] * unit);
        ql[s][e] = (_Float16)fmaf(x[s][e], unit, -(float)qh[s][e]);
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
      const int at = tid + j * S::T, cg = at % CG, kg = at / CG;
      const bool on = (S::BLOCKS % S::T == 0 || at < S::BLOCKS) && (FULL || 4 * cg < d);
      int64_t off[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) off[i] = mem.off[(S::BLOCKS % S::T == 0 ? 4 * kg : 4 * kg % KT) + i];
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
  bool there = false, broken = false;
  int up_least = 126;                  // of the keys' powers of two
  int v_first = S::v_at(n, g);
  float v_big = 0.f;                   // largest |v| so far
  float v_sq = 0.f;                    // of float16 values, this thread's sum of squares
  float v_sum = 0.f;                   // of the others, the largest of each tile summed, as o
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
            for (int c = 0; c < 4; c += 2) {
              km = max_abs(km, kx[j][i][c], kx[j][i][c + 1]);
              vm = max_abs(vm, vx[j][i][c], vx[j][i][c + 1]);
            }
          }
        km = wave_most(km);
        vm = wave_most(vm);
        if (lane == 0) mem.mx[wv][0] = km, mem.mx[wv][1] = vm;
      }
      __syncthreads();                 // the last tile is done with, and the maxima are there
      float down = 1.f, v_most = 0.f;  // of the keys; the tile's largest |v|
      int up = 0;
      bool endless = false;            // a key of the tile, or a value that is none
      if constexpr (C::SCALED) {
        uint32_t km_bits = 0, vm_bits = 0;       // as wave_most: a NaN is the largest
#pragma unroll
        for (int w = 0; w < W; ++w) {
          km_bits = max(km_bits, __float_as_uint(mem.mx[w][0]));
          vm_bits = max(vm_bits, __float_as_uint(mem.mx[w][1]));
        }
        const float km = __uint_as_float(km_bits), vm = __uint_as_float(vm_bits);
        v_big = fmaxf(v_big, vm);
        v_most = vm;
        up = uniform(up_of(km));
        down = power_of(-up);
        endless = !(km < INFINITY) || vm != vm;
        v_up = uniform(min(v_up, v_big > 0.f ? up_of(v_big) : 126));
        const float ku = power_of(up), vu = power_of(v_up);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          const int at = tid + j * S::T, cg = at % CG, kg = at / CG;
          if (S::BLOCKS % S::T != 0 && at >= S::BLOCKS) continue;
          const int run = 2 * (kg >> 2) + (kg & 1), half = 4 * (kg >> 1 & 1);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            h4 h, l;
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
              const h2 y = scaled2_of(kx[j][i][c], kx[j][i][c + 1], ku);
              h[c] = y[0], h[c + 1] = y[1];
              if constexpr (N == 2) {
                const h2 z = rest2_of(kx[j][i][c], kx[j][i][c + 1], ku, y);
                l[c] = z[0], l[c + 1] = z[1];
              }
            }
            *(h4*)&mem.k[0][(4 * kg + i) * KS + 4 * cg] = h;
            if constexpr (N == 2) *(h4*)&mem.k[1][(4 * kg + i) * KS + 4 * cg] = l;
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            h4 h, l;
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const h2 y = scaled2_of(vx[j][i][c], vx[j][i + 1][c], vu);
              h[i] = y[0], h[i + 1] = y[1];
              if constexpr (N == 2) {
                const h2 z = rest2_of(vx[j][i][c], vx[j][i + 1][c], vu, y);
                l[i] = z[0], l[i + 1] = z[1];
              }
            }
            *(h4*)&mem.v[0][S::v_at(4 * cg + c, run) + half] = h;
            if constexpr (N == 2) *(h4*)&mem.v[1][S::v_at(4 * cg + c, run) + half] = l;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          const int at = tid + j * S::T, cg = at % CG, kg = at / CG;
          if (S::BLOCKS % S::T != 0 && at >= S::BLOCKS) continue;
          const int run = 2 * (kg >> 2) + (kg & 1), half = 4 * (kg >> 1 & 1);
          uint32_t x[4][2];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint2 kw = __builtin_bit_cast(uint2, kr[j][i]), vw = __builtin_bit_cast(uint2, vr[j][i]);
            *(uint2*)&mem.k[0][(4 * kg + i) * KS + 4 * cg] = kw;
            x[i][0] = vw.x, x[i][1] = vw.y;
            const h2 v0 = __builtin_bit_cast(h2, vw.x), v1 = __builtin_bit_cast(h2, vw.y);
            v_sq = __builtin_amdgcn_fdot2(v1, v1, __builtin_amdgcn_fdot2(v0, v0, v_sq, false), false);
          }
          asm volatile("" : "+v"(v_sq));     // now: later it would hold these values beside the next tile's (16 spilled)
#pragma unroll
          for (int c = 0; c < 4; ++c) {      // 4 x 4 two-byte values turned by byte permutations
            const uint32_t sel = c % 2 ? 0x07060302u : 0x05040100u;
            *(uint2*)&mem.v[0][S::v_at(4 * cg + c, run) + half] = make_uint2(__builtin_amdgcn_perm(x[1][c / 2], x[0][c / 2], sel),
                                                                     __builtin_amdgcn_perm(x[3][c / 2], x[2][c / 2], sel));
          }
        }
      }
      if (!C::SCALED && t + 1 == t1) {
        const float x = wave_most(v_sq);
        if (lane == 0) mem.mx[wv][1] = x;
      }
      place(id, in);
      __syncthreads();                 // the tile is there
      if (t + 1 < t1) {
        fetch();
        lookup(t + 2, id, in);
      }
      asm volatile("" : "+v"(v_first));      // the places that follow from it are found anew, rather than held
      const int k0 = t * KT;
      if (k0 >= w_hi || k0 + KT <= w_lo) continue;
      if constexpr (C::SCALED) {
        up_least = min(up_least, up), broken = broken || endless;
        if (o_up != v_up) {
          const float f = ldexpf(1.f, v_up - o_up);
          o_up = v_up;
          v_sum *= f;
#pragma unroll
          for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] *= f;
        }
        v_sum = fmaf(v_most, power_of(v_up), v_sum);
      }

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
        const int hi = hi_now(), b0 = max(Item::lo_of(a, hi) - k0, 0), b1 = min(hi - k0, KT);
        uint64_t m = b1 > b0 ? now & (~(uint64_t)0 >> (64 - b1)) & (~(uint64_t)0 << b0) : 0;
        there = there || m != 0;
        m >>= 4 * g;
#pragma unroll
        for (int u = 0; u < KT / 32; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int keep = (int)((uint32_t)(m >> 32 * u) << (31 - (8 * (r / 4) + r % 4))) >> 31;
            sc[u][r] = __int_as_float((keep & __float_as_int(sc[u][r])) | (~keep & (int)0xff800000));
          }
      }
      const float c = factor * down;
      // Half by half, 32 keys: weights against the reference so far, whose sum of positive numbers shows whether one of
      // them is too large for float16.  Only then, and for rows that have met no key before, the largest score is found
      // and the reference moved.  The products of one half run beside the weights of the next.
#pragma unroll
      for (int w = 0; w < KT / 32; ++w) {
        float p[16], part_sum, most;
        auto weigh = [&]() {
          const float ref = (top == -INFINITY ? 0.f : top) - kRef;
          float x[2];
#pragma unroll
          for (int r = 0; r < 16; r += 2) {
            p[r] = exp2_fast(fmaf(sc[w][r], c, -ref)), p[r + 1] = exp2_fast(fmaf(sc[w][r + 1], c, -ref));
            x[r / 8] = r % 8 == 0 ? p[r] + p[r + 1] : x[r / 8] + (p[r] + p[r + 1]);
          }
          most = fmaxf(x[0], x[1]);
          part_sum = x[0] + x[1];
        };
        weigh();
        if (__any(!(most <= kMost / kHold) || top == -INFINITY)) {
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
        h8 ph[2], pl[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if constexpr (ND > 2 && KT == 64) __builtin_amdgcn_sched_barrier(0);     // moved further up, planes spill
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float p0 = p[8 * u + e], p1 = p[8 * u + e + 1];
            h2 h = half2_of(p0, p1);
            if constexpr (kHold != 1.f) h *= (_Float16)kHold;
            const h2 l = rest2_of(p0, p1, kHold, h);
            ph[u][e] = h[0], ph[u][e + 1] = h[1];
            pl[u][e] = l[0], pl[u][e + 1] = l[1];
          }
          settled(pl[u]);
          // products of one accumulator are kept apart, as above
          h8 vx8[N][ND];
#pragma unroll
          for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) vx8[j][i] = *(const h8*)&mem.v[j][S::v_at(v_first, i, 4 * w + 2 * u)];
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

  // What the row's scores are off by at most where small planes end, in units of 2^-25 c: its own ends, those of numbers of up
  // to 2^-18 of the largest, times the largest keys, and the keys' ends times its numbers.
  auto ends_of = [&]() {
    const int r = valid ? row_now() : 0;
    const float* q = a.q + (int64_t)token_of(r) * a.ldq + (int64_t)head_of(r) * d + 8 * g;
    float big = 0.f, ends = 0.f, all = 0.f;
#pragma unroll 1
    for (int c = 0; c + 8 * g < d; c += 16)
#pragma unroll
      for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(q[c + e]));
    big = fmaxf(big, __shfl_xor(big, 32, kWave));
    const float unit = ldexpf(1.f, up_of(big));
#pragma unroll 1
    for (int c = 0; c + 8 * g < d; c += 16)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = fabsf(q[c + e] * unit);
        if (x != 0.f && x < 0x1p-3f) ends += C::SCALED ? 0x1p15f : 0x1p16f;
        if (C::SCALED) all += x;
      }
    ends += all;
    return ends + __shfl_xor(ends, 32, kWave);
  };

  // register r of o[i]: channel 32 i + 8 (r / 4) + 4 g + r % 4
  sum += __shfl_xor(sum, 32, kWave);
  const float inv = 1.f / (sum * kHold);
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
  // Each key's weight is off by up to 2^-25 of 2^12 where the small planes end.  That is 2^-18 of the outputs together, or
  // less, if the outputs before the division are above 2^-7 of the keys' |v| of a channel summed.  For that stands the largest of
  // every tile, as often as it has keys; for float16 values, which are not scaled and whose largest is not known, the root of
  // keys times their squares' sum, the largest of a thread's, which has four channels of some of the keys.
  float all = KT * v_sum;
  if constexpr (!C::SCALED) {
    constexpr int kShare = S::T % CG == 0 ? S::T / CG : KT / 4;        // threads that a channel lies with
    const int hi = hi_now(), met = min(hi, t1 * KT) - max(Item::lo_of(a, hi), t0 * KT);
    uint32_t bits = 0;
    if (t0 < t1)
#pragma unroll
      for (int w = 0; w < W; ++w) bits = max(bits, __float_as_uint(mem.mx[w][1]));
    all = sqrtf((float)met * (float)kShare * __uint_as_float(bits));  // or NaN
  }
  const bool lost = all != 0.f && ((C::SCALED && big < 1.f) || !(big * sum * kHold >= 0x1p-7f * all));
  // A score's terms are up to 2^30 c_most (2^31 of float16 keys, which are not scaled), and off by 2^-10 of that where a small
  // plane ends.  As long as that is 2^-20 of the largest score, or of 1, in every channel at once, the row is as good as
  // float32's; else its channels are looked at.
  const float c_most = factor * (C::SCALED ? power_of(-up_least) : 1.f), most = 0x1p-20f * fmaxf(1.f, fabsf(top));
  bool coarse = ends && !(c_most * (float)d * 0x1p-9f <= most);
  if (__any(valid && there && coarse)) {
    coarse = coarse && !(c_most * 0x1p-25f * ends_of() <= most);
    if constexpr (!C::SCALED) {        // 2^16 stands for keys that are seldom near it: a row's own
      uint64_t left = __ballot(valid && there && coarse && g == 0);
      while (left) {
        const int r = uniform(__ffsll((unsigned long long)left) - 1);
        left &= left - 1;
        const int row_hi = it.hi_of(a, wv * kWaveRows + r);
        const float at = key_ends<E>(a, it.b, it.kvh, a.q + (int64_t)token_of(wv * kWaveRows + r) * a.ldq +
                                                          (int64_t)head_of(wv * kWaveRows + r) * d,
                                     max(Item::lo_of(a, row_hi), t0 * KT), min(row_hi, t1 * KT));
        if (n == r) coarse = !(c_most * 0x1p-25f * at <= most);
      }
    }
  }
  odd = odd || broken || coarse || !(sum > 0.f && sum < INFINITY) || lost;
  odd = __shfl_xor((int)odd, 32, kWave) || odd;
  const bool again = valid && there && odd;
  const float unit = C::SCALED ? ldexpf(1.f, -o_up) : 1.f;
  if (valid && !again) {
    const int r = row_now();
    float* dst = whole ? a.out + (int64_t)token_of(r) * a.ldo + (int64_t)head_of(r) * d : part + (int64_t)r * d;
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
    if (!whole && g == 0) part_ml[r] = make_float2(there ? top : -INFINITY, there ? sum : 0.f);
  }
  uint64_t rest = __ballot(again && g == 0);
  while (rest) {
    const int r = uniform(__ffsll((unsigned long long)rest) - 1);
    rest &= rest - 1;
    const int r_tok = token_of(wv * kWaveRows + r), r_head = head_of(wv * kWaveRows + r);
    const int row_hi = it.hi_of(a, wv * kWaveRows + r), r_hi = min(row_hi, t1 * KT), r_lo = max(Item::lo_of(a, row_hi), t0 * KT);
    RowSum<E> x;
    x.run(a, it.b, it.kvh, a.q + (int64_t)r_tok * a.ldq + (int64_t)r_head * d, r_lo, r_hi);
    const bool none = x.there && x.top == -INFINITY;       // scores of -inf alone
    float* to = whole ? a.out + (int64_t)r_tok * a.ldo + (int64_t)r_head * d : part + (int64_t)(wv * kWaveRows + r) * d;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (64 * i + lane < d) to[64 * i + lane] = !x.there || (none && !whole) ? 0.f : x.o[i];
    if (!whole && lane == 0) part_ml[wv * kWaveRows + r] = make_float2(none ? kNoScore : x.top, x.sum * (0x1p12f / kHold));
  }
}

// Waves a SIMD that the registers are held to: a third one, where it fits, works while the others wait at their barriers
// (float16, 14 on 2 heads of 64, 8 x 800 queries over 5800 keys: 339 -> 284 us; with float32 the spills cost more).
template <typename E, int ND>
constexpr int simd_waves() {
  return ND > 4 ? 1 : ND == 2 && Cell<E>::N == 1 && !Cell<E>::SCALED ? 3 : 2;
}

// One workgroup a (tile of rows, kv head).  12 prompts of up to 900 tokens (14 on 2 heads of 64, float32) 49 us, where the
// 15 tiles of the longest, 1.5 us each in a workgroup that has its CU alone, take half of it.
template <typename E, int ND, bool FULL, int W>
__global__ __launch_bounds__(64 * W, (simd_waves<E, ND>())) void k_extend_whole(ExtArgs a, bool by_keys) {
  __shared__ typename Shape<E, ND, W>::Mem mem;
  Item it;
  // what sees the most keys goes first, or at least the last tiles of each sequence
  const int at = (int)(blockIdx.x / (unsigned)a.kv_heads);
  if (!(by_keys ? find_by_keys<Shape<E, ND, W>::KT, W>(a, at, it) : find_item<W>(a, a.slots - 1 - at, it))) return;
  it.kvh = (int)(blockIdx.x % (unsigned)a.kv_heads);
  int t0, t1;
  tiles_of<Shape<E, ND, W>::KT>(a, it, t0, t1);
  attend<E, ND, FULL, W>(a, it, t0, t1, true, nullptr, nullptr, mem);
}

// A workgroup's part of an item (slot, kv head): `part` of `parts` equal runs of its key tiles.  Parts of one item have
// places that follow each other; parts 0: nothing to do.
struct Piece {
  int b, kvh, tile, part, parts, place, pad[2];
};

// The last i of [0, n) with v[i] <= x; v[0] <= x.
__device__ __forceinline__ int last_at(const int32_t* v, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// The keys of long items shared out by what the device holds, so that a long cache with few rows, a ragged batch and a
// causal triangle all fill the machine and a captured launch serves every length.  Items are cut into equal parts of at
// most `most` key tiles, a workgroup each.  `most` is the size with the least estimate of: no cut; the least of a few
// sizes whose parts all run at once (`groups` do); half a workgroup's mean load.  A part is charged kPartCost tiles for
// its start and end, and kCutCost more where it has to be joined (some 2 us a tile); what runs in several rounds half of
// the largest part for the last.  A tile takes kAlone of its time in a workgroup that shares its CU with none, which is how
// long items end.  Where nothing is cut, and items are more than run at once or the largest kUneven of their mean, they go by
// size, the largest first in kSizes steps: 12 ragged slices of up to 800 queries over 5800 keys (32 on 8 heads of 128,
// bfloat16) 710 us with the larger items cut in half, 655 so; the same of float16, 14 on 2 heads of 64, 188 and 176, but 248
// uncut by slots.  4 slices of 500 over 2500 (20 on 4 heads of 80, float32), nearly alike, lose by it: 200 and 219.
//
// One workgroup, a thread a slot: 8 - 13 us, the chain of its loads, searches and sums.  (Done by every workgroup of
// k_extend_split for itself it took 4 - 9 us of each, and registers of the products.)
constexpr int kPlanThreads = kSplitSlots, kTries = 9, kPartCost = 2, kCutCost = 3, kSizes = 8;
constexpr float kAlone = 0.55f, kUneven = 1.25f;
template <int KT, int W>
__global__ __launch_bounds__(kPlanThreads) void k_extend_plan(ExtArgs a) {
  constexpr int kRows = kWaveRows * W, kWaves = kPlanThreads / 64, kSums = kTries + 1;
  __shared__ int32_t s_slot[kSplitSlots];           // a sequence's first slot
  __shared__ int32_t s_pieces[kSplitSlots];         // parts of the slots ahead
  __shared__ int32_t s_places[kSplitSlots];         // of them those of cut items
  __shared__ int32_t s_cuts[kSplitSlots];           // items that are cut, of the slots ahead
  __shared__ int32_t s_parts[kSplitSlots];
  __shared__ uint32_t s_red[kWaves][kSums];
  __shared__ uint64_t s_up[kWaves];
  __shared__ int32_t s_tile[kSplitSlots];           // slots in their order
  __shared__ int32_t s_size[kWaves][kSizes];
  __shared__ float s_load, s_items, s_inv;
  __shared__ uint32_t s_top;
  __shared__ bool s_sort;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, slots = a.slots, hk = a.kv_heads;
  for (int b = tid; b < a.batch; b += kPlanThreads) s_slot[b] = first_slot<W>(a, b);
  __syncthreads();
  const int s = slots - 1 - tid;                    // the last slots first: they see the most keys
  int mine = 0;                                     // key tiles of this thread's slot, for one kv head
  if (s >= 0 && s_slot[0] <= s) {
    const int b = last_at(s_slot, a.batch, s);
    const Seq q = seq_of(a, b);
    const int64_t row0 = (int64_t)(s - s_slot[b]) * kRows, rows = min((int64_t)q.count * a.group - row0, (int64_t)kRows);
    if (row0 >= 0 && rows > 0) {
      Item one{b, 0, q.first, q.base, q.len, (int)row0, (int)rows};
      int u0, u1;
      tiles_of<KT>(a, one, u0, u1);
      mine = max(u1 - u0, 1);          // rows with no key to see are written too: a part with nothing in it
    }
  }
  {
    const uint32_t lo = wave_sum_u32((uint32_t)mine & 0xffff), hi = wave_sum_u32((uint32_t)mine >> 16), n = __popcll(__ballot(mine > 0));
    const uint32_t top = wave_fold((uint32_t)mine, [](uint32_t x, uint32_t y) { return max(x, y); });
    if (lane == 0) s_red[wv][0] = lo, s_red[wv][1] = hi, s_red[wv][2] = n, s_red[wv][3] = top;
  }
  __syncthreads();
  if (tid == 0) {
    float units = 0.f, n = 0.f;
    uint32_t top = 1;
    for (int w = 0; w < kWaves; ++w) {
      units += (float)s_red[w][0] + 65536.f * (float)s_red[w][1];
      n += (float)s_red[w][2];
      top = max(top, s_red[w][3]);
    }
    s_load = units * (float)hk / (float)a.groups, s_items = n * (float)hk, s_top = top;
  }
  __syncthreads();
  const float load = s_load, least = fmaxf(ceilf(load), 1.f);
  auto size_of = [&](int k) { return k < kTries ? ceilf(least * (1.f + (float)k / (kTries - 1))) : fmaxf(ceilf(0.5f * load), 1.f); };
  auto parts_of = [](int n, float inv) { return n > 0 ? 1 + (int)((float)(n - 1) * inv) : 0; };
#pragma unroll
  for (int k = 0; k < kSums; ++k) {
    const uint32_t need = wave_sum_u32((uint32_t)parts_of(mine, 1.f / size_of(k)));
    if (lane == 0) s_red[wv][k] = need;
  }
  __syncthreads();
  if (wv == 0) {
    // a candidate a lane; the last lane: no cut
    const float groups = (float)a.groups, top = (float)s_top, whole = s_items, cost = kPartCost + kCutCost;
    float est = INFINITY, size = top;
    if (lane < kSums) {
      uint32_t need = 0;
      for (int w = 0; w < kWaves; ++w) need += s_red[w][lane];
      const float n = (float)need * (float)hk;
      size = size_of(lane);
      est = n <= groups ? size + cost : lane < kTries ? INFINITY : load + cost * n / groups + 0.5f * size;
      if (size >= top) est = INFINITY;
    } else if (lane == kSums) {
      est = fmaxf(kAlone * top, whole <= groups ? load : load + top / kSizes) + kPartCost * fmaxf(whole / groups, 1.f);
    }
    const float best = -wave_max_dpp(-est);
    const int pick = __ffsll((unsigned long long)__ballot(est == best)) - 1;
    size = __shfl(size, pick, kWave);
    if (lane == 0) s_inv = 1.f / size, s_sort = pick == kSums && (whole > groups || top * whole > kUneven * load * groups);
  }
  __syncthreads();
  int parts = parts_of(mine, s_inv), slot = s;
  if (s_sort) {
    const int of = mine > 0 ? (int)((uint32_t)(s_top - mine) * (uint64_t)kSizes / s_top) : kSizes - 1;
    int rank = 0;
#pragma unroll
    for (int i = 0; i < kSizes; ++i) {
      const uint64_t m = __ballot(of == i);
      if (lane == 0) s_size[wv][i] = __popcll(m);
      if (of == i) rank = __popcll(m & (((uint64_t)1 << lane) - 1));
    }
    __syncthreads();
    for (int w = 0; w < kWaves; ++w)
#pragma unroll
      for (int i = 0; i < kSizes; ++i)
        if (i < of || (i == of && w < wv)) rank += s_size[w][i];
    s_tile[rank] = s;
    s_parts[rank] = parts;
    __syncthreads();
    slot = s_tile[tid], parts = s_parts[tid];
    __syncthreads();
  }
  s_tile[tid] = slot;
  // parts, parts of cut items, and cut items of the slots ahead, 21 bits each: there are at most 2^10 and 3 groups
  const uint64_t n = parts > 1 ? (uint64_t)parts | (uint64_t)parts << 21 | (uint64_t)1 << 42 : (uint64_t)parts;
  uint64_t up = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t u = __shfl_up((unsigned long long)up, o, kWave);
    if (lane >= o) up += u;
  }
  if (lane == 63) s_up[wv] = up;
  __syncthreads();
  uint64_t all = 0;
  up -= n;
  for (int w = 0; w < kWaves; ++w) {
    if (w < wv) up += s_up[w];
    all += s_up[w];
  }
  constexpr uint64_t kField = (1 << 21) - 1;
  s_pieces[tid] = (int)(up & kField) * hk, s_places[tid] = (int)(up >> 21 & kField) * hk, s_cuts[tid] = (int)(up >> 42) * hk;
  s_parts[tid] = parts;
  __syncthreads();
  const int count = min((int)(all & kField) * hk, a.pieces_most);
  if (tid == 0) a.counts[0] = min((int)(all >> 42) * hk, a.cuts_most), a.counts[1] = count, a.counts[2] = s_sort;
  for (int w = tid; w < count; w += kPlanThreads) {
    const int at = last_at(s_pieces, min(slots, kSplitSlots), w), slot = s_tile[at], b = last_at(s_slot, a.batch, slot);
    const int of = s_parts[at], in = w - s_pieces[at], kvh = in / of, part = in - kvh * of, place = s_places[at] + in;
    const int cut = s_cuts[at] + kvh;
    Piece one{b, kvh, slot - s_slot[b], part, of, place, {0, 0}};
    if (of > 1 && (place >= a.places || cut >= a.cuts_most)) one.parts = 0;      // starts that do not rise
    a.pieces[w] = one;
    if (one.parts > 1 && part == 0) a.cuts[cut] = one;
  }
}

// Of a cut item each workgroup leaves its rows' outputs, maxima and sums (`part`, `part_ml`).  The two cases named at
// `attend`: 283 and 726 us in the median of a trace (265 and 688 at least), beside them the plan and 9 and 5 us of joins.
template <typename E, int ND, bool FULL, int W>
__global__ __launch_bounds__(64 * W, (simd_waves<E, ND>())) void k_extend_split(ExtArgs a) {
  typedef Shape<E, ND, W> S;
  __shared__ typename S::Mem mem;
  // pieces that follow each other share keys: they go to one XCD's L2 where all run at once and are alike
  const int count = a.counts[1], eighth = (count + 7) / 8, in_eighth = (int)(blockIdx.x / 8);
  const bool runs = count <= a.groups && !a.counts[2];
  const int w = runs ? (int)(blockIdx.x % 8) * eighth + in_eighth : (int)blockIdx.x;
  if (w >= count || (runs && in_eighth >= eighth)) return;
  const Piece p = a.pieces[w];
  Item it;
  const int parts = uniform(p.parts), part = uniform(p.part);
  if (parts < 1 || !item_of<W>(a, uniform(p.b), uniform(p.tile), it)) return;
  it.kvh = uniform(p.kvh);
  int t0, t1;
  tiles_of<S::KT>(a, it, t0, t1);
  const int64_t place = uniform(p.place);
  const int from = t0 + (int)((int64_t)(t1 - t0) * part / parts), to = t0 + (int)((int64_t)(t1 - t0) * (part + 1) / parts);
  attend<E, ND, FULL, W>(a, it, from, to, parts == 1, a.part + place * a.part_rows * a.d, a.part_ml + place * a.part_rows, mem);
}

// Few rows a sequence: a wave each has 32 rows and one of `parts` runs of every item's keys, cut alike whatever their
// lengths (the host knows no more), so that no plan has to come first.  4 queries over 504 keys (14 on 2 heads of 64, float32) 8.0 us
// and 4.1 of joining: launches and memory latencies.
template <typename E, int ND, bool FULL>
__global__ __launch_bounds__(64, (simd_waves<E, ND>())) void k_extend_few(ExtArgs a, int parts) {
  typedef Shape<E, ND, 1> S;
  __shared__ typename S::Mem mem;
  const int item = (int)(blockIdx.x / (unsigned)parts), part = (int)(blockIdx.x % (unsigned)parts);
  Item it;
  if (!find_item<1>(a, item / a.kv_heads, it)) return;
  it.kvh = item % a.kv_heads;
  int t0, t1;
  tiles_of<S::KT>(a, it, t0, t1);
  const int from = t0 + (int)((int64_t)(t1 - t0) * part / parts), to = t0 + (int)((int64_t)(t1 - t0) * (part + 1) / parts);
  attend<E, ND, FULL, 1>(a, it, from, to, parts == 1, a.part + (int64_t)blockIdx.x * a.part_rows * a.d,
                         a.part_ml + (int64_t)blockIdx.x * a.part_rows, mem);
}

// The parts of an item's rows.  A wave reads four channels a lane, so several parts at a time, then joins its lanes; with
// many parts the waves share them, with few each takes rows of its own.  parts 0: the items are those of `cuts`.  Bound by
// the parts' bytes: 38 us for some 100 MB, 8 for 500 queries in 14 heads over 60501 keys, 4.3 for 4.
constexpr int kJoinAhead = 4, kJoinFew = 32, kJoinGroups = 2048;
template <int LP, int W>                         // lanes of a part: a power of two with 4 LP >= d
__global__ __launch_bounds__(256) void k_extend_join(ExtArgs a, int parts, int rows) {
  constexpr int PP = 64 / LP;                    // parts of one load
  __shared__ float s_o[4][256], s_ml[4][2];
  const int lane = threadIdx.x & 63, wv = uniform((int)threadIdx.x >> 6), c4 = 4 * (lane % LP), sub = lane / LP;
  const int row_groups = (a.part_rows + rows - 1) / rows;        // `rows` at a time
  const int tasks = (parts ? a.slots * a.kv_heads : a.counts[0]) * row_groups;
  for (int task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int item = task / row_groups;
    Item it;
    int64_t first;
    int count;
    if (parts) {
      if (!find_item<W, 4>(a, item / a.kv_heads, it)) continue;
      it.kvh = item % a.kv_heads;
      first = (int64_t)item * parts;
      count = parts;
    } else {
      const Piece cut = a.cuts[item];
      if (!item_of<W>(a, uniform(cut.b), uniform(cut.tile), it)) continue;
      it.kvh = uniform(cut.kvh);
      first = uniform(cut.place);
      count = uniform(cut.parts);
    }
    const int row0 = task % row_groups * rows, end = min(row0 + rows, it.rows);
    const bool few = count <= kJoinFew;
    const int step = few ? PP : 4 * PP;
    for (int r = few ? row0 + wv : row0; r < end; r += few ? 4 : 1) {
      f32x4u x{};
      float top = -INFINITY, sum = 0.f;
      for (int i = (few ? 0 : wv * PP) + sub; __any(i < count); i += step * kJoinAhead) {
        f32x4u y[kJoinAhead];
        float2 ml[kJoinAhead];
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u) {
          const int m = i + u * step;
          const int64_t at = (first + min(m, count - 1)) * a.part_rows + r;
          ml[u] = a.part_ml[at];
          y[u] = f32x4u{};
          if (c4 < a.d) y[u] = *(const f32x4u*)(a.part + at * a.d + c4);
          if (m >= count) ml[u].x = -INFINITY;
        }
        float now = top;
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u) now = fmaxf(now, ml[u].x);
        // x is a mean, so that values near the largest float stay in its range
        const float f = weight_of(top, now) * sum;
        float g[kJoinAhead];
        sum = f;
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u) {
          g[u] = ml[u].x != -INFINITY ? weight_of(ml[u].x, now) * ml[u].y : 0.f;
          sum += g[u];
        }
        const float one = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int j = 0; j < 4; ++j) x.v[j] *= f * one;
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u)
          if (ml[u].x != -INFINITY) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x.v[j] += g[u] * one * y[u].v[j];
          }
        top = now;
      }
      auto join = [&](float t, float l, const f32x4u& o) {
        const float now = fmaxf(top, t), f = weight_of(top, now) * sum, g = weight_of(t, now) * l;
        sum = f + g;
        const float one = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int j = 0; j < 4; ++j) x.v[j] = f * one * x.v[j] + g * one * o.v[j];
        top = now;
      };
#pragma unroll
      for (int o = LP; o < 64; o <<= 1) {
        f32x4u y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y.v[j] = __shfl_xor(x.v[j], o, kWave);
        join(__shfl_xor(top, o, kWave), __shfl_xor(sum, o, kWave), y);
      }
      const int flat = it.row0 + r, head = it.kvh * a.group + flat % a.group;
      float* out = a.out + (int64_t)(it.first + flat / a.group) * a.ldo + (int64_t)head * a.d;
      if (!few) {
        __syncthreads();
        if (sub == 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) s_o[wv][c4 + j] = x.v[j];
        }
        if (lane == 0) s_ml[wv][0] = top, s_ml[wv][1] = sum;
        __syncthreads();
        if (wv != 0) continue;
#pragma unroll
        for (int u = 1; u < 4; ++u) {
          f32x4u y;
#pragma unroll
          for (int j = 0; j < 4; ++j) y.v[j] = s_o[u][c4 + j];
          join(s_ml[u][0], s_ml[u][1], y);
        }
      }
      if (sub == 0 && c4 < a.d) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x.v[j] = top == -INFINITY ? 0.f : sum == 0.f ? NAN : x.v[j];
        *(f32x4u*)(out + c4) = x;
      }
    }
  }
}

template <int ND, int W>
void launch_join(const ExtArgs& a, int64_t items, int parts, hipStream_t st) {
  const int rows = parts > kJoinFew ? 1 : 4;
  const dim3 grid((unsigned)std::min<int64_t>(items * ceil_div(a.part_rows, rows), kJoinGroups)), block(256);
  if (ND == 2) hipLaunchKernelGGL((k_extend_join<16, W>), grid, block, 0, st, a, parts, rows);
  else if (ND <= 4) hipLaunchKernelGGL((k_extend_join<32, W>), grid, block, 0, st, a, parts, rows);
  else hipLaunchKernelGGL((k_extend_join<64, W>), grid, block, 0, st, a, parts, rows);
}

// Scratch for `rows` rows of parts and `more` bytes behind them; CV3_ENOMEM, which callers live without: there is none.
int part_scratch(ExtArgs& a, int64_t rows, size_t more, void** work, void** behind, hipStream_t st) {
  const int rc = scratch_alloc(work, (size_t)rows * (a.d * 4 + 8) + more, st);
  if (rc) {
    *work = nullptr;
    return rc;
  }
  a.part = (float*)*work;
  a.part_ml = (float2*)(a.part + rows * a.d);
  *behind = a.part_ml + rows;
  return CV3_OK;
}

template <typename E, int ND, bool FULL>
int run_tiles(ExtArgs a, hipStream_t st) {
  constexpr int W = 4, kAtOnce = 256 * simd_waves<E, ND>() * 4;     // waves that the registers let run at once
  const int64_t cap = a.blocks * a.page, rows = a.n * a.group;
  void *work = nullptr, *behind;
  int rc = CV3_OK;
  const bool few = rows <= kFewRows * a.batch;
  if (few && ND == 2) {
    constexpr int KT = Shape<E, ND, 1>::KT;
    a.slots = (int)(rows / kWaveRows + a.batch);
    a.part_rows = (int)std::min<int64_t>(kWaveRows, rows);
    const int64_t items = (int64_t)a.slots * a.kv_heads;
    // enough waves to fill the machine twice, but parts of 8 tiles where there would be more than 16 of them
    const int64_t tiles = ceil_div(cap, KT), most = tiles <= 16 ? tiles : std::max<int64_t>(16, tiles / 8);
    int64_t parts = std::max<int64_t>(1, std::min(ceil_div(2 * kAtOnce, items), most));
    if (parts > 1) {
      rc = part_scratch(a, items * parts * a.part_rows, 0, &work, &behind, st);
      if (rc && rc != CV3_ENOMEM) return rc;
      if (rc) parts = 1;               // without memory: one wave an item
    }
    if constexpr (ND == 2)
      hipLaunchKernelGGL((k_extend_few<E, ND, FULL>), dim3((unsigned)(items * parts)), dim3(64), 0, st, a, (int)parts);
    if (work) launch_join<ND, 1>(a, items, (int)parts, st);
  } else {
    a.slots = (int)(rows / (kWaveRows * W) + a.batch);
    const int64_t items = (int64_t)a.slots * a.kv_heads;
    a.groups = kAtOnce / W;
    const bool ordered = a.batch <= 64;
    const int64_t whole = few ? kWholeKeys / 4 : ordered && 4 * items >= 3 * a.groups ? kOrderKeys : kWholeKeys;
    if (a.slots <= kSplitSlots && cap > whole) {
      a.part_rows = (int)std::min<int64_t>(kWaveRows * W, rows);
      // parts of no more than half a mean load: items and 2 groups of them, 4 groups of those in cut items
      a.pieces_most = (int)items + 2 * a.groups;
      a.places = 4 * a.groups;
      a.cuts_most = (int)std::min<int64_t>(items, 2 * a.groups);
      const size_t lists = (size_t)(a.pieces_most + a.cuts_most) * sizeof(Piece) + 16;
      rc = part_scratch(a, (int64_t)a.places * a.part_rows, lists, &work, &behind, st);
      if (rc && rc != CV3_ENOMEM) return rc;
      a.pieces = (Piece*)behind;
      a.cuts = a.pieces + a.pieces_most;
      a.counts = (int*)(a.cuts + a.cuts_most);
    }
    if (work) {
      hipLaunchKernelGGL((k_extend_plan<Shape<E, ND, W>::KT, W>), dim3(1), dim3(kPlanThreads), 0, st, a);
      hipLaunchKernelGGL((k_extend_split<E, ND, FULL, W>), dim3((unsigned)a.pieces_most), dim3(64 * W), 0, st, a);
      launch_join<ND, W>(a, a.cuts_most, 0, st);
    } else {                           // short tables, very many tiles, or no memory: one workgroup an item
      hipLaunchKernelGGL((k_extend_whole<E, ND, FULL, W>), dim3((unsigned)items), dim3(64 * W), 0, st, a,
                         ordered && a.batch > 1 && items > kOrderItems);
    }
  }
  const hipError_t err = hipGetLastError();
  rc = work ? scratch_free(work, st) : CV3_OK;
  CV3_REQUIRE(err == hipSuccess, CV3_EHIP, "kernel launch failed: %s", hipGetErrorString(err));
  return rc;
}

template <typename E>
int extend_for(const ExtArgs& a, hipStream_t st) {
  switch ((a.d + 31) / 32) {
    case 1:
    case 2: return a.d == 64 ? run_tiles<E, 2, true>(a, st) : run_tiles<E, 2, false>(a, st);
    case 3: return run_tiles<E, 3, false>(a, st);
    case 4: return a.d == 128 ? run_tiles<E, 4, true>(a, st) : run_tiles<E, 4, false>(a, st);
    case 5:
    case 6: return run_tiles<E, 6, false>(a, st);
    default: return run_tiles<E, 8, false>(a, st);
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
            0, scale * 1.4426950408889634f};
  hipStream_t st = stream_of(s);
  if (cache_type == CV3_F32) return extend_for<float>(a, st);
  if (cache_type == CV3_F16) return extend_for<_Float16>(a, st);
  return extend_for<__bf16>(a, st);
}

}  // extern "C"
