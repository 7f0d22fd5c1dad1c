// Attention of several new tokens per sequence over the paged INT8 cache: every
// row of a ragged batch (a drafted tree, or a chunk of a prompt) against the
// cached tokens of its sequence and the new tokens that its mask names.
//
//   s = (q . kc) * ks / sqrt(D),   out = sum_t p_t vs_t vc_t / sum_t p_t,
//   p_t = exp(s_t - max s)
//
// with the INT8 codes kc, vc and the FP32 scales ks, vs of (token, KV head).
//
// One pass over the keys with the running maximum and sum of the softmax. A
// workgroup takes a tile of the (new token, head of the group) rows of one sequence
// and KV head and a chunk of its keys; where there are several chunks their FP32 sums
// meet in a second kernel. How long the chunks are is found on the GPU, from lengths
// that the host does not know. Tiles of keys come from the pages to LDS by DMA while
// the tile before is worked on. Two kernels: one for few rows, bound by memory, and
// one for many, bound by the vector ALU that turns scores into probabilities beside
// the matrix cores. 8 sequences of 8 K to 32 K tokens, 4 KV heads of 128 channels, 8
// query heads each: one token each 47 us (the cache at 4.5 TB/s but for 10 us before
// the first and after the last keys), trees of 16 70 us, of 64 201 us (628 TFLOP/s).
//
// Scores are exact sums of FP32-scaled products of the stored codes but for the FP32
// rounding; the rounding to fewer bits that there is: a probability times its value
// scale to the 11 bits of FP16, the second product's operand (an eighth of the BF16
// output's half step; for products far below the row's largest see TreeScales), and
// query values that are more than 2^6 below their row's largest (few rows) or 2^12 (many).
// Maxima, sums and all accumulators are FP32, and so are scores, which have to be in its
// range: a row with one past it is NaN, and it alone.
#include <atomic>
#include <type_traits>

#include "q6moe_api.h"
#include "q6moe_device.h"

#define LDS_PTR(p) ((__attribute__((address_space(3))) void*)(uint32_t)(uintptr_t)(p))

namespace q6moe {

typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr int kTreeThreads = 256;
constexpr int kTreeCus = 256;
constexpr int kTreeMaxHeads = 65535;
constexpr float kTreeFloor = -0x1p126f;  // running maximum before the first seen key
constexpr float kTreeSlack = 8.f;        // a score may pass the running maximum by 2^8 before that is raised

struct TreeParams {
  const uint16_t* q;
  int64_t q_stride;
  const int8_t* kc;
  const int8_t* vc;
  const void* ks;
  const void* vs;
  int scale_bf16;
  const int32_t* table;
  const int32_t* len;
  const int32_t* starts;
  const uint64_t* masks;
  int words;
  int batch, rows, max_count;
  int kvh, hq, r;
  int pool_pages, pps, page, cap;
  uint32_t page_magic;  // t / page = t * page_magic >> page_shift for 0 <= t < 2^31
  int page_shift;
  int slots;       // workgroups that the work is split for
  int whole;       // no split over keys
  int grid;        // workgroups of the launch
  int parts;       // places for partial sums
  float to_log2;   // log2(e) / sqrt(D)
  float* part;     // [item of a split sequence][row of the tile][D] partial sums
  float* stat;     // [item of a split sequence][row of the tile][2]: maximum (log2) and sum
  int32_t* info;   // [2 batch + 2]: first place of each sequence's sums; the keys per item; the items; and
                   // with ``whose`` the first item of each sequence
  int32_t* whose;  // [workgroup] each item's sequence, where tree_plan_kernel finds the items; else null
  uint16_t* out;
};

// Calls of few rows per KV head: 32 rows per workgroup, every wave all of them
// with keys of its own. Bound by memory.
template <int D>
struct TreeThin {
  static constexpr int kRows = 32;    // (new token, head of the group) rows per workgroup
  static constexpr int kTile = 32;    // keys per tile of a wave
  static constexpr int kStep = 128;   // keys per turn of the workgroup
  static constexpr int kPerCu = D > 128 ? 1 : 2;  // workgroups per CU
  static constexpr int kHalf = kTile * D;         // bytes of a tile's keys, and of its values
  static constexpr int kScale = 2 * 32 * 4 + 16;  // per wave: a tile's key and value scales, value factor
  static constexpr int kRing = 4 * 2 * 2 * kHalf;  // per wave a tile in work and one on its way
  static constexpr int kLds = kRing + 4 * kScale + 32 + 16;  // and four words of masks, four flags
  static_assert(kPerCu * kLds <= 160 * 1024, "tile");
};

// Calls of many rows: 128 rows per workgroup, 32 per wave, which share the keys.
template <int D>
struct TreeWide {
  static constexpr int kRows = 128;
  static constexpr int kTile = D == 256 ? 32 : 64;
  static constexpr int kStep = kTile;
  static constexpr int kPerCu = D == 64 ? 4 : (D == 128 ? 3 : 2);
  static constexpr int kHalf = kTile * D;
  static constexpr int kScale = 2 * kTile * 4 + 16;
  // Of a wave's 2 D / 32 operands of queries, those in LDS. (With all of them in
  // registers some spilled, and their reload waited for the DMA just issued: 8 x
  // 64-token trees over 32 K tokens 261 us against 236.)
  static constexpr int kQueries = D == 256 ? 2 : 0;
  // a tile's codes, the same in FP16, scales, masks, queries, four flags
  static constexpr int kLds = 2 * kHalf + 4 * kHalf + 4 * kScale + 32 + 4096 * kQueries + 16;
  static_assert(kPerCu * kLds <= 160 * 1024, "tile");
};

// The wave's loads and DMA have landed.
__device__ __forceinline__ void tree_landed() {
  __builtin_amdgcn_s_waitcnt(15 << 8 | 7 << 4);  // vmcnt(0)
  asm volatile("" ::: "memory");
}

// A value that the compiler knows nothing of: what is formed from it in a loop is
// formed anew each time, instead of being held in registers across the loop.
__device__ __forceinline__ uint32_t tree_opaque(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}

// The kernel's arguments read again, and with them all that a chunk begun anew needs: what
// it uses is not held in registers through the pass before.
__device__ __forceinline__ TreeParams tree_again() {
  auto args = (__attribute__((address_space(4))) const uint64_t*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  uint64_t word[sizeof(TreeParams) / 8];
#pragma unroll
  for (int i = 0; i < (int)(sizeof word / 8); ++i) word[i] = args[i];
  return __builtin_bit_cast(TreeParams, word);
}

// Whether a pass was left. The compiler is not to know it where it ends: it put the pass
// after it in between, with the sums of the first in scratch memory (one token over
// 16 K, 256-wide heads, 28.8 us became 33.5).
__device__ __forceinline__ bool tree_left(bool whole) {
  int v = __builtin_amdgcn_readfirstlane(whole);
  asm volatile("" : "+s"(v));
  return !v;
}

// What the rows of a sequence need: cached tokens, new tokens with rows, keys in reach.
struct TreeSeq {
  int start, count, len, n;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams& p, int b) {
  TreeSeq s;
  const int a = p.starts[b], e = p.starts[b + 1], n = p.len[b];
  s.start = a < 0 ? 0 : (a < p.rows ? a : p.rows);
  const int end = e < p.rows ? e : p.rows;
  int c = end - s.start;
  c = c < 0 ? 0 : c;
  s.count = c < p.max_count ? c : p.max_count;
  s.len = n < 0 ? 0 : (n < p.cap ? n : p.cap);
  s.n = s.len + s.count < p.cap ? s.len + s.count : p.cap;
  return s;
}
__device__ __forceinline__ int tree_tiles(const TreeParams& p, const TreeSeq& s, int rows) {
  return (s.count * p.r + rows - 1) / rows;
}
__device__ __forceinline__ int tree_chunks(int n, int keys) { return n <= keys ? 1 : (n + keys - 1) / keys; }
// Keys per chunk, in whole steps: alike, and never more than ``keys`` of tree_chunks,
// as that is whole steps too; then no chunk is empty either. (Full chunks and a rest:
// a chunk of 1024 tokens over 1000 cached ones 89 us against 78, over 8 K 240 and 225.)
__device__ __forceinline__ int tree_span(int n, int chunks, int step) {
  const int steps = (n + step - 1) / step;
  return (steps + chunks - 1) / chunks * step;
}
// Keys that the rows of one tile reach, and those that all of them see.
__device__ __forceinline__ void tree_reach(const TreeParams& p, const TreeSeq& s, int tile, int rows, int* n,
                                           int* all) {
  if (p.masks) {
    *n = s.n;
    *all = s.len;
    return;
  }
  const int first = tile * rows / p.r, last = (tile * rows + rows - 1) / p.r;
  const int to = s.len + (last < s.count ? last + 1 : s.count), seen = s.len + first + 1;
  *n = to < p.cap ? to : p.cap;
  *all = seen < p.cap ? seen : p.cap;
}

// The priority of a wave in turn ``turn``: the N workgroups of a CU, which start
// with different turns, take the first place in turn. With equal priorities the
// oldest of three ran ahead (6500 cycles a turn, the youngest 9300) and the last
// ended alone: 64-token trees over 32 K tokens 243 us, with turns 230; 16-token
// trees in the thin kernel 74.7 and 73.3.
template <int N>
__device__ __forceinline__ void tree_priority(int turn) {
  const int k = turn % N;
  if (k == 0)
    __builtin_amdgcn_s_setprio(0);
  else if (k == 1)
    __builtin_amdgcn_s_setprio(1);
  else if (k == 2)
    __builtin_amdgcn_s_setprio(2);
  else
    __builtin_amdgcn_s_setprio(3);
}

struct TreeItem {
  int place, b, tile, kh, chunk, keys;  // place: of its partial sums
  TreeSeq seq;
};

template <typename T, typename F>
__device__ __forceinline__ T tree_wave_reduce(T v, F f) {
  const auto step = [&](auto ctrl) {
    const int w = __builtin_bit_cast(int, v);
    v = f(v, __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(w, w, decltype(ctrl)::value, 0xf, 0xf, true)));
  };
  step(std::integral_constant<int, 0xb1>{});   // quad_perm [1,0,3,2]
  step(std::integral_constant<int, 0x4e>{});   // quad_perm [2,3,0,1]
  step(std::integral_constant<int, 0x124>{});  // row_ror:4
  step(std::integral_constant<int, 0x128>{});  // row_ror:8
  const auto swap = [&](auto r) {
    v = f(__builtin_bit_cast(T, (uint32_t)r[0]), __builtin_bit_cast(T, (uint32_t)r[1]));
  };
  uint32_t w = __builtin_bit_cast(uint32_t, v);
  swap(__builtin_amdgcn_permlane16_swap(w, w, false, false));
  w = __builtin_bit_cast(uint32_t, v);
  swap(__builtin_amdgcn_permlane32_swap(w, w, false, false));
  return v;
}

// Sum of v over the lanes up to this one: shifts within rows of 16, then the rows'
// last lanes spread over the rows after them.
__device__ __forceinline__ int tree_wave_scan(int v) {
  const auto add = [&](auto ctrl, auto rows) {
    v += __builtin_amdgcn_update_dpp(0, v, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});  // row_shr:1
  add(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});  // row_shr:2
  add(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});  // row_shr:4
  add(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});  // row_shr:8
  add(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // row_bcast:15 into rows 1 and 3
  add(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});  // row_bcast:31 into rows 2 and 3
  return v;
}

// The call's work, sum over sequences of tiles x heads x keys, is cut into chunks of
// at most ``keys`` keys: the least number that gives no more chunks than the chip
// holds workgroups, so that all run at once and, whatever the lengths, end together.
// Only the GPU knows the lengths. (Cut at the mean instead, 64-token trees made 640
// chunks for then 512 places: 321 us against 236.) Where the tiles themselves fill
// half of the places or more, the chunks are half as long as the mean share and run
// in turns. ``sum(zero, f)`` is the sum of f over the sequences.
template <int ROWS, int STEP, typename S>
__device__ __forceinline__ int tree_keys(const TreeParams& p, S&& sum) {
  if (p.whole) return 1 << 30;
  const auto units = [&](const TreeSeq& s) { return tree_tiles(p, s, ROWS) * p.kvh; };
  const float total = sum(0.f, [&](const TreeSeq& s) { return (float)units(s) * (float)s.n; });
  const int tiles = sum(0, units);
  const bool once = 2 * tiles <= p.slots;
  constexpr int kMost = (1 << 30) / STEP - 1;  // with one more a chunk holds any sequence
  const float share = total / (float)(once ? p.slots : 2 * p.slots) * (1.f / STEP);
  int lo = share < (float)kMost ? (int)share : kMost;
  lo = lo < 1 ? 1 : lo;
  // in steps; hi gives few enough chunks: each tile has at most one that is not full
  const float sure = total / (float)(p.slots - tiles) * (1.00001f / STEP);
  int hi = once ? (sure < (float)kMost ? (int)sure : kMost) + 1 : lo + 1;
  // few tiles: hi is within an eighth of the least
  if (once && 8 * tiles > p.slots)
    for (int i = 0; i < 5 && lo < hi; ++i) {
      const int mid = (lo + hi) >> 1;
      // at least the number of chunks: a rounded quotient, raised by 2^-20
      const float per = 1.000001f / (float)(mid * STEP);
      const int n = sum(0, [&](const TreeSeq& s) { return units(s) * ((int)((float)s.n * per) + 1); });
      if (n <= p.slots)
        hi = mid;
      else
        lo = mid + 1;
    }
  return hi * STEP;
}

// Items of a sequence: chunks x KV heads x tiles, tiles fastest.
template <int ROWS>
__device__ __forceinline__ int tree_items(const TreeParams& p, const TreeSeq& s, int keys) {
  return tree_tiles(p, s, ROWS) * p.kvh * tree_chunks(s.n, keys);
}

// More sequences than a wave has lanes: one workgroup finds the items for all others
// in one launch more, 4.3 us. One token each, every wave for itself and so: 65
// sequences of up to 4 K tokens 45.0 and 47.1 us, 256 of 1000 58.0 and 52.8, 600 of
// 300 71 and 52, 2000 of 200 358 and 132.
constexpr int kTreeLanes = 64, kTreePlan = 1024;
template <int ROWS, int STEP>
__global__ void __launch_bounds__(kTreePlan) tree_plan_kernel(TreeParams p) {
  __shared__ int lds[kTreePlan / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const auto sum = [&](auto zero, auto of) {
    auto v = zero;
    for (int b = threadIdx.x; b < p.batch; b += kTreePlan) v += of(tree_seq(p, b));
    v = tree_wave_reduce(v, [](auto x, auto y) { return x + y; });
    __syncthreads();  // lds may still be read
    if (lane == 0) lds[wave] = __builtin_bit_cast(int, v);
    __syncthreads();
    v = zero;
    for (int w = 0; w < kTreePlan / 64; ++w) v += __builtin_bit_cast(decltype(v), lds[w]);
    return v;
  };
  const int keys = tree_keys<ROWS, STEP>(p, sum);
  const auto before = [&](int n, int& base) {  // of the threads before; base grows by all
    const int upto = tree_wave_scan(n);
    __syncthreads();
    if (lane == 63) lds[wave] = upto;
    __syncthreads();
    int first = base + upto - n;
    for (int w = 0; w < kTreePlan / 64; ++w) {
      first += w < wave ? lds[w] : 0;
      base += lds[w];
    }
    return first;
  };
  int items = 0, places = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kTreePlan) {
    const int b = b0 + (int)threadIdx.x;
    const TreeSeq s = b < p.batch ? tree_seq(p, b) : TreeSeq{0, 0, 0, 0};
    const int n = tree_items<ROWS>(p, s, keys);
    const int first = before(n, items), place = before(s.n > keys ? n : 0, places);
    if (b < p.batch) {
      p.info[b] = place;
      p.info[p.batch + 2 + b] = first;
      for (int i = first < 0 ? 0 : first; i < first + n && i < p.grid; ++i) p.whose[i] = b;
    }
  }
  if (threadIdx.x == 0) {
    p.info[p.batch] = keys;
    p.info[p.batch + 1] = items;
  }
}

// The workgroup's item, from tree_plan_kernel or, of up to 64 sequences, found by each
// wave for itself, a lane for each.
template <int ROWS, int STEP>
__device__ __forceinline__ bool tree_item(const TreeParams& p, TreeItem& it) {
  const int lane = threadIdx.x & 63;
  TreeSeq mine{0, 0, 0, 0};
  int upto = 0, n = 0, total;  // items of the lane's sequence and up to it
  if (p.whose) {
    it.keys = p.info[p.batch];
    total = p.info[p.batch + 1];
  } else {
    if (lane < p.batch) mine = tree_seq(p, lane);
    it.keys = tree_keys<ROWS, STEP>(p, [&](auto zero, auto of) {
      auto v = of(mine);
      v = tree_wave_reduce(v, [](auto x, auto y) { return x + y; });
      return __builtin_bit_cast(decltype(v), __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
    });
    n = tree_items<ROWS>(p, mine, it.keys);
    upto = tree_wave_scan(n);
    total = __builtin_amdgcn_readlane(upto, 63);
  }
  // Workgroup i runs on XCD i % 8: each XCD takes a contiguous run of the items, so
  // that the tiles that share a chunk's keys share its L2; the runs are alike.
  // (Starts that do not ascend can name more items than there are workgroups.)
  const int most = (int)(gridDim.x >> 3), run = (total + 7) >> 3 < most ? (total + 7) >> 3 : most;
  const int place = (int)(blockIdx.x >> 3);
  const int id = (int)(blockIdx.x & 7) * run + place;
  if (place >= run || id >= total) return false;
  int first, sums;  // first item of the sequence, and place of its sums
  if (p.whose) {
    const int b = p.whose[id];
    it.b = b < 0 || b >= p.batch ? 0 : b;  // as for the items that no workgroup has
    it.seq = tree_seq(p, it.b);
    sums = p.info[it.b];
    first = p.info[p.batch + 2 + it.b];
  } else {
    it.b = __builtin_ctzll(__ballot(id < upto));
    it.seq.start = __builtin_amdgcn_readlane(mine.start, it.b);
    it.seq.count = __builtin_amdgcn_readlane(mine.count, it.b);
    it.seq.len = __builtin_amdgcn_readlane(mine.len, it.b);
    it.seq.n = __builtin_amdgcn_readlane(mine.n, it.b);
    first = __builtin_amdgcn_readlane(upto - n, it.b);
    const int split = mine.n > it.keys ? n : 0;
    sums = __builtin_amdgcn_readlane(tree_wave_scan(split) - split, it.b);
    if (threadIdx.x == 0 && id == first) p.info[it.b] = sums;
    if (threadIdx.x == 0 && id == 0) p.info[p.batch] = it.keys;
  }
  const int in = id - first, tiles = tree_tiles(p, it.seq, ROWS);
  it.place = sums + in;
  if (in < 0 || tiles < 1 || (it.seq.n > it.keys && (it.place < 0 || it.place >= p.parts))) return false;
  const int row = in / tiles;
  it.tile = in - row * tiles;
  it.chunk = row / p.kvh;
  it.kh = row - it.chunk * p.kvh;
  return true;
}

// A tile's rows in LDS: key t lies in row tree_row(t), bits 0 and 2 of t exchanged,
// so that the two half waves, which read the values of keys 4 apart, meet
// different halves of the banks. Chunk c of a row's key lies in slot c ^
// tree_swizzle(row), so that the 16 lanes that read one column of 16 keys meet 16
// different bank groups; values, read by rows, lie as they are.
__device__ __forceinline__ uint32_t tree_row(uint32_t key) { return (key & ~5u) | (key & 1) << 2 | (key >> 2 & 1); }
template <int D>
__device__ __forceinline__ uint32_t tree_swizzle(uint32_t row) {
  constexpr uint32_t CH = D / 16;
  return (row / (16 / CH)) & (CH - 1);
}

// The channel of accumulator element v of channel block c, for a lane of half
// wave h: each lane's loads of D / 32 consecutive channels of a key serve all
// blocks (for D = 64, of 4 channels, of which the upper 16 rows take the last two).
template <int D>
__device__ __forceinline__ int tree_channel(int c, int v, int h) {
  const int i = 8 * (v >> 2) + 4 * h + (v & 3);
  return D == 64 ? 4 * (i & 15) + 2 * (i >> 4) + c : D / 32 * i + c;
}

// New tokens that some row of the sequence sees. What the cache holds at the
// others' places (they may never have been written) is not read. One wave's work.
__device__ __forceinline__ void tree_wanted(const TreeParams& p, const TreeSeq& s, uint64_t* wanted) {
  const int lane = threadIdx.x & 63;
  for (int w = 0; w < p.words; ++w) {
    uint64_t some = 0;
    for (int i = lane; i < s.count; i += 64) some |= p.masks[(int64_t)(s.start + i) * p.words + w];
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) some |= __shfl_xor((unsigned long long)some, off);
    if (lane == 0) wanted[w] = some;
  }
}

// Bit i: a row's token j sees key k0 + i; moved to the keys of half wave h.
__device__ __forceinline__ uint32_t tree_visible(const TreeParams& p, const TreeSeq& s, int j, int k0, int c1, int h) {
  const int jj = k0 - s.len;
  uint32_t on;
  if (p.masks) {
    const uint64_t* w = p.masks + (int64_t)(s.start + j) * p.words;
    if (jj >= 0) {
      const int at = jj >> 6, sh = jj & 63;
      const uint64_t a = at < p.words ? w[at] : 0, b = at + 1 < p.words ? w[at + 1] : 0;
      on = (uint32_t)(a >> sh | (b << 1) << (63 - sh));
    } else if (jj > -32) {
      on = (uint32_t)(w[0] << -jj) | ((1u << -jj) - 1);
    } else {
      on = ~0u;
    }
  } else {
    const int seen = j + 1 - jj;  // keys of the block up to the row's own
    on = seen >= 32 ? ~0u : (seen <= 0 ? 0u : (1u << seen) - 1);
  }
  const int left = c1 - k0;
  if (left < 32) on &= left <= 0 ? 0u : (1u << left) - 1;
  return on >> (4 * h);
}

// The way from a tile's keys to the cache: the lane looks up key ``lane`` of the
// tile (of 32: lanes 0-31 for its key scale, the others for its value scale).
template <int T>
struct TreeLookup {
  const int32_t* table;
  const uint64_t* wanted;
  int c1, len, kh, lane;
  bool pick;
  int entry;        // page-table entry of the next tile's key
  uint32_t rk, rv;  // scales on their way, as they lie in the cache
  bool seen, on;    // whether some row sees the key, and whether it has any

  __device__ __forceinline__ int page_of(const TreeParams& p, int t) const {
    return (int)((uint64_t)(uint32_t)t * p.page_magic >> p.page_shift);
  }
  __device__ __forceinline__ int clamp(int t) const { return t < c1 ? t : (c1 > 0 ? c1 - 1 : 0); }
  __device__ __forceinline__ void ask(const TreeParams& p, int t0) {
    entry = table[page_of(p, clamp(t0 + (lane & (T - 1))))];
  }
  static __device__ __forceinline__ uint32_t bits(const TreeParams& p, const void* s, int64_t i) {
    return p.scale_bf16 ? (uint32_t)reinterpret_cast<const uint16_t*>(s)[i] : reinterpret_cast<const uint32_t*>(s)[i];
  }
  // Pool row of the lane's key of the tile at t0 (0 where nothing is read), its
  // scales' loads, and the entry for the tile at t1.
  __device__ __forceinline__ int row(const TreeParams& p, int t0, int t1) {
    const int t = t0 + (lane & (T - 1)), tc = clamp(t);
    seen = t < c1;
    if (pick && t0 + T > len) {  // uniform over the wave
      const int jj = t - len;
      if (t < c1 && jj >= 0) seen = wanted[jj >> 6] >> (jj & 63) & 1;
    }
    on = seen && entry >= 0 && entry < p.pool_pages;
    const int r = on ? entry * p.page + (tc - page_of(p, tc) * p.page) : 0;
    ask(p, t1);
    const int64_t at = (int64_t)r * p.kvh + kh;
    if (T == 32) {
      rk = bits(p, lane < 32 ? p.ks : p.vs, at);
    } else {
      rk = bits(p, p.ks, at);
      rv = bits(p, p.vs, at);
    }
    return r;
  }
};

// Scales of a tile into the wave's LDS. Probability x value scale is an FP16 operand,
// which has 11 bits from 2^-14 on and a step of 2^-24 below. The value scales are
// brought to at most 2^6 by a power of two that falls as larger ones are met. While
// none is below 2^-5 then, a row, whose largest probability is at least 1, keeps 11
// bits of products down to 2^-9 of its largest, and the others to 2^-20 of that.
// Scales further apart (one that a row does not see, or that hardly counts in it, would
// take the others' bits: below some 2^-5 or past 2^3 to 2^6 times the largest of the chunk's
// first keys), of 0, beyond 2^100 and unmapped pages make the chunk ``odd``, and so do key
// scales beyond 2^20, of which a score could leave the range of FP32 on the way.
// It is begun anew with the scales as they are, and each row finds a factor of its own
// from the products that it sees (tree_any_scales), so that products keep 11 bits down
// to 2^-17 of its largest and the others to 2^-28 of that. With a maximum and a factor
// for each 32 keys, that is slower: with scales of 0 in every chunk one token each over
// 32 K tokens 51 us against 41, trees of 16 97 against 75, of 64 364 against 203.
template <int T, bool kAny>
struct TreeScales {
  float factor = 1.f, limit = -1.f;  // of the newest tile
  float low = -1.f;                  // the smallest scale that is not odd
  bool odd = false;
  // The key scales times ``unit`` 2^e.
  __device__ __forceinline__ void put(const TreeParams& p, const TreeLookup<T>& at, float* sc, float unit = 1.f,
                                      int e = 0) {
    const auto value = [&](uint32_t bits) {
      return at.on ? __builtin_bit_cast(float, p.scale_bf16 ? bits << 16 : bits) : 0.f;
    };
    const float k = value(at.rk), v = T == 32 ? k : value(at.rv);
    if constexpr (!kAny) {
      // of 32 keys a lane holds a key scale or a value scale
      const bool keys = T == 32 && at.lane < 32;
      const float a = fabsf(v), most = keys ? 0x1p20f : limit, least = keys ? -1.f : low;
      bool out = (a > most) | (a < least);
      if (T == 64) out |= fabsf(k) > 0x1p20f;
      if (__any(out & at.seen)) {
        const bool mine = !keys & at.seen, far = (T == 64 || keys) & at.seen & (fabsf(k) > 0x1p20f);
        const bool finite = a < __builtin_inff();
        const float x = tree_wave_reduce(mine && finite ? a : 0.f, [](float c, float d) { return fmaxf(c, d); });
        int ve = __builtin_amdgcn_readfirstlane((int)(__builtin_bit_cast(uint32_t, x) >> 23)) - 127;
        ve = ve < -124 ? -124 : ve;
        if (low < 0.f) low = ve < -121 ? 0x1p-126f : __builtin_bit_cast(float, (uint32_t)(127 + ve - 5) << 23);
        factor = __builtin_bit_cast(float, (uint32_t)(127 + 3 - ve) << 23);  // 2^(3-ve): at most 2^4 now
        limit = __builtin_bit_cast(float, (uint32_t)(127 + ve + 3 > 254 ? 254 : 127 + ve + 3) << 23);
        odd = __any((mine & ((a < low) | !finite)) | far) || limit > low * 0x1p11f || limit > 0x1p100f;
      }
    }
    if (T == 32) {
      sc[at.lane] = at.lane < 32 ? __builtin_ldexpf(k * unit, e) : v * factor;
    } else {
      sc[at.lane] = __builtin_ldexpf(k * unit, e);
      sc[T + at.lane] = v * factor;
    }
    if (at.lane == 0) sc[2 * T] = factor;
  }
};

// A row's softmax so far: maximum (log2), sum over the lane's keys, value factor.
// A score less its maximum is formed by one FMA, of a maximum that is rounded. Beyond 2^13
// (kTreeHuge) half a step of that is more than the 2^-11 by which a probability is
// rounded, and from 2^27 on one could overflow: such maxima, too, make the chunk odd.
constexpr float kTreeHuge = 0x1p13f;
struct TreeState {
  float m = kTreeFloor, l = 0.f, factor = 1.f;
  bool huge = false;  // of some row of the wave
};

// The maximum of 32 keys' scores, ``top``, and their value factor, taken into the
// state; calls fade(f) where what was summed up to now is to be multiplied by f.
// The maximum is raised only where a score passes it by 2^8, for the whole wave.
template <typename F>
__device__ __forceinline__ void tree_raise(TreeState& st, float top, float factor, F&& fade) {
  factor = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, factor)));
  if (__any(top > st.m + kTreeSlack) || factor != st.factor) {  // uniform over the wave
    const float to = fmaxf(st.m, fmaxf(top, __shfl_xor(top, 32)));
    const float f = __builtin_amdgcn_exp2f(st.m - to);
    fade(f * (factor / st.factor));
    st.huge |= __any((fabsf(to) > kTreeHuge) & (to != kTreeFloor));
    st.factor = factor;
    st.m = to;
    st.l *= f;
  }
}

// The same where scores come less the row's maximum so far (``t``): the maximum is
// raised where one is beyond 2^8, and set by the row's first seen keys.
struct TreeLevel {
  float m = 0.f, l = 0.f, factor = 1.f;
  float limit = -3.4028235e38f;  // kTreeSlack once m is set
  bool huge = false;
};
template <typename F>
__device__ __forceinline__ void tree_level(TreeLevel& st, float* t, float top, float factor, F&& fade) {
  factor = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, factor)));
  if (__any(top > st.limit) || factor != st.factor) {  // uniform over the wave
    const float both = fmaxf(top, __shfl_xor(top, 32));
    const bool on = both > st.limit;
    const float to = on ? st.m + both : st.m, by = on ? to - st.m : 0.f;
    const float f = st.limit < 0.f ? 1.f : __builtin_amdgcn_exp2f(-by);
    fade(f * (factor / st.factor));
    st.huge |= __any(fabsf(to) > kTreeHuge);
    st.factor = factor;
    st.m = to;
    st.l *= f;
    st.limit = on ? kTreeSlack : st.limit;
#pragma unroll
    for (int v = 0; v < 16; ++v) t[v] -= by;
  }
}

// The same for scales of any size: the scores ``t`` (log2, -inf where not seen) become
// probability x value scale x the row's factor, which brings the largest product so
// far, ``most``, to between 2^3 and 2^4. vs(g): the scales of keys 4 g + [0, 4).
template <typename V, typename F>
__device__ __forceinline__ void tree_any_scales(TreeState& st, float& most, float* t, V&& vs, F&& fade) {
  float top = t[0];
#pragma unroll
  for (int v = 1; v < 16; ++v) top = fmaxf(top, t[v]);
  const float to = fmaxf(st.m, fmaxf(top, __shfl_xor(top, 32)));
  const float f = __builtin_amdgcn_exp2f(st.m - to);
  st.m = to;
  st.l *= f;
  float x = 0.f;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 by = vs(g);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int v = 4 * g + u;
      const bool on = t[v] != -__builtin_inff();
      const float e = __builtin_amdgcn_exp2f(t[v] - to);
      st.l += on ? e : 0.f;
      t[v] = on ? e * by[u] : 0.f;
      x = fmaxf(x, fabsf(t[v]));
    }
  }
  most = fmaxf(most * f, fmaxf(x, __shfl_xor(x, 32)));
  float factor = st.factor;
  int up = 0;
  if (most > 0.f) {
    const int e = (int)(__builtin_bit_cast(uint32_t, most) >> 23);
    factor = __builtin_bit_cast(float, (uint32_t)(257 - (e < 3 ? 3 : e)) << 23);
    up = (int)(__builtin_bit_cast(uint32_t, factor) >> 23) - (int)(__builtin_bit_cast(uint32_t, st.factor) >> 23);
  }
  fade(__builtin_ldexpf(f, up < 126 ? up : 126));  // more only where nothing was summed up
  st.factor = factor;
#pragma unroll
  for (int v = 0; v < 16; ++v) t[v] *= factor;
}

// A score is sum x key scale x unit 2^e, of which the last two may leave the range of
// FP32 where the score does not: a 2^e below 1 goes first.
struct TreeBy {
  float pre, post;
  __device__ __forceinline__ TreeBy(float unit, int e)
      : pre(__builtin_ldexpf(1.f, e < 0 ? e : 0)), post(__builtin_ldexpf(unit, e < 0 ? 0 : e)) {}
  __device__ __forceinline__ float operator()(float sum, float scale) const { return sum * pre * scale * post; }
};

// The rows of a workgroup: which query, and the bits of its channels.
template <int D>
struct TreeRow {
  bool live;
  int j, hh;
  int e;      // exponent of the row's largest magnitude
  bool bad;   // an infinite or NaN query: NaN scores
  u32x4 raw[D / 32][2];
  // raw[s][i] of half wave h: channels 32 s + 16 h + 8 i + [0, 8), the order of INT8
  // operands, or 32 s + 16 i + 8 h + [0, 8), that of FP16 ones. The loads, and then
  // what needs them.
  template <bool kBytes>
  __device__ __forceinline__ void ask(const TreeParams& p, const TreeItem& it, int row, int h) {
    live = row < it.seq.count * p.r;
    j = live ? row / p.r : 0;
    hh = live ? row - j * p.r : 0;
    const uint16_t* src = p.q + (int64_t)(it.seq.start + j) * p.q_stride + (int64_t)(it.kh * p.r + hh) * D;
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = kBytes ? 32 * s + 16 * h + 8 * i : 32 * s + 16 * i + 8 * h;
        raw[s][i] = live ? *reinterpret_cast<const u32x4*>(src + c) : u32x4{0u, 0u, 0u, 0u};
      }
  }
  __device__ __forceinline__ void scale() {
    u16x2 tops = {0, 0};  // the largest magnitudes' bits
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w)
          tops = __builtin_elementwise_max(tops, __builtin_bit_cast(u16x2, raw[s][i][w] & 0x7fff7fffu));
    const uint32_t mine = tops[0] > tops[1] ? tops[0] : tops[1], other = __shfl_xor(mine, 32);
    const uint32_t top = mine > other ? mine : other;
    bad = top >= 0x7f80u;
    // the largest stays below 127 * 256 + 128 in steps of 2^(e-14)
    e = (int)(top >> 7) - 127 + ((top & 0x7f) == 0x7f);
    e = e < -112 ? -112 : e;  // smaller queries lose bits: what is left is off by 2^-127 at most
  }
  __device__ __forceinline__ float value(int s, int i, int k) const {  // k of 8
    const uint32_t x = raw[s][i][k >> 1];
    return __builtin_bit_cast(float, k & 1 ? x & 0xffff0000u : x << 16);
  }
};

// Runs of a lane's sums whose channels lie together: each four become f(first channel, them).
template <int D, typename A, typename F>
__device__ __forceinline__ void tree_runs(A& acc, int h, F&& f) {
  constexpr int kRun = D == 64 ? 4 : D / 32, kRuns = D / 2 / kRun;
#pragma unroll
  for (int q = 0; q < kRuns; ++q)
#pragma unroll
    for (int u = 0; u < kRun; u += 4) {
      const int c = tree_channel<D>(0, q, h) + u;
      if constexpr (D == 64) {
        const f32x4 v = f(c, f32x4{acc[0][q], acc[1][q], acc[0][q + 8], acc[1][q + 8]});
        acc[0][q] = v[0], acc[1][q] = v[1], acc[0][q + 8] = v[2], acc[1][q + 8] = v[3];
      } else {
        const f32x4 v = f(c, f32x4{acc[u][q], acc[u + 1][q], acc[u + 2][q], acc[u + 3][q]});
        acc[u][q] = v[0], acc[u + 1][q] = v[1], acc[u + 2][q] = v[2], acc[u + 3][q] = v[3];
      }
    }
}

// A row's sums (of the values times the state's factor) to the workspace, or its output.
template <int D, typename A>
__device__ __forceinline__ void tree_result(const TreeParams& p, const TreeItem& it, A& acc, bool split, float m,
                                            float l, int j, int hh, int64_t place, int h) {
  if (split) {
    float* dst = p.part + place * D;
    tree_runs<D>(acc, h, [&](int c, f32x4 v) { return *reinterpret_cast<f32x4*>(dst + c) = v; });
    if (h == 0) *reinterpret_cast<f32x2*>(p.stat + 2 * place) = f32x2{m, l};
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* dst = p.out + ((int64_t)(it.seq.start + j) * p.hq + it.kh * p.r + hh) * D;
  tree_runs<D>(acc, h, [&](int c, f32x4 v) {
    const u32x2 y = {pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv)};
    *reinterpret_cast<u32x2*>(dst + c) = y;
    return v;
  });
}

// ---------------------------------------------------------------------------
// Few rows. The waves have keys of their own and do not wait for each other; a turn
// of 32 keys costs some 300 vector instructions, 16 exponentials and 16 MFMAs (128
// channels). Queries are 16-bit integers in two INT8 operands, q = (256 hi + lo)
// 2^(e-14): exact for values down to 2^-6 of the row's largest. So the INT8 codes
// of the keys are matrix operands as they lie, and the sums are exact. The values'
// codes + 128 enter the second product as FP16 subnormals, (code + 128) 2^-24, one
// byte permutation per two of them; the 128 is taken back at the end with the sum
// of the rounded probabilities.
// ---------------------------------------------------------------------------
template <int D, bool kAny>
__device__ __forceinline__ bool tree_thin_pass(const TreeParams& p) {
  using C = TreeThin<D>;
  constexpr int KS = D / 32;  // channel blocks of 32
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  TreeItem it;
  if (!tree_item<C::kRows, C::kStep>(p, it)) return true;  // uniform over the workgroup
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, h = lane >> 5;
  const TreeSeq seq = it.seq;
  int n, n_all;
  tree_reach(p, seq, it.tile, C::kRows, &n, &n_all);
  const int chunks = tree_chunks(n, it.keys);
  if (it.chunk >= chunks) return true;
  const int span = tree_span(n, chunks, C::kStep), c0 = it.chunk * span;
  const int c1 = n - c0 < span ? n : c0 + span;
  const int turns = (c1 - c0 + C::kStep - 1) / C::kStep;

  uint8_t* ring = smem + wave * (4 * C::kHalf);
  float* scales = reinterpret_cast<float*>(smem + C::kRing + wave * C::kScale);
  uint64_t* wanted = reinterpret_cast<uint64_t*>(smem + C::kRing + 4 * C::kScale);
  TreeLookup<C::kTile> keys{p.table + (int64_t)it.b * p.pps, wanted, c1, seq.len, it.kh, lane,
                            p.masks && c1 > seq.len, 0, 0, 0, false, false};
  TreeScales<C::kTile, kAny> put;
  const auto tile_at = [&](int i) { return c0 + (wave + 4 * i) * C::kTile; };
  keys.ask(p, tile_at(0));
  TreeRow<D> row;
  row.template ask<true>(p, it, it.tile * C::kRows + col, h);
  if (keys.pick) {
    if (wave == 0) tree_wanted(p, seq, wanted);
    __syncthreads();
  }
  const uint32_t row_bytes = (uint32_t)p.kvh * D;
  const int8_t* kbase = p.kc + (int64_t)it.kh * D;
  const int8_t* vbase = p.vc + (int64_t)it.kh * D;
  const auto issue = [&](int i, int stage) {
    const int r = keys.row(p, tile_at(i), tile_at(i + 1));
    uint8_t* st = ring + stage * 2 * C::kHalf;
#pragma unroll
    for (int d = 0; d < KS; ++d) {  // 64 chunks of 16 bytes each
      const uint32_t line = 64 * d / (D / 16) + (uint32_t)lane / (D / 16), slot = (uint32_t)lane % (D / 16);
      const uint32_t rr = __builtin_amdgcn_ds_bpermute(4 * tree_row(line), r);
      const int8_t* k = kbase + (uint64_t)rr * row_bytes + 16 * (slot ^ tree_swizzle<D>(line));
      const int8_t* v = vbase + (uint64_t)rr * row_bytes + 16 * slot;
      __builtin_amdgcn_global_load_lds(k, LDS_PTR(st + 1024 * d), 16, 0, 0);
      __builtin_amdgcn_global_load_lds(v, LDS_PTR(st + C::kHalf + 1024 * d), 16, 0, 0);
    }
  };
  issue(0, 0);

  row.scale();
  i32x4 qhi[KS], qlo[KS];
  {
    // v = q 2^(14-e) rounded into the low bits of 1.5 * 2^23 + v; its low byte is lo,
    // the second byte of v + 128 is hi
    const float up = __builtin_ldexpf(1.f, 14 - row.e);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[i] = __builtin_bit_cast(uint32_t, __builtin_fmaf(row.value(s, w >> 1, 4 * (w & 1) + i), up, 12582912.f));
        const uint32_t l01 = __builtin_amdgcn_perm(v[1], v[0], 0x0c0c0400u);
        const uint32_t l23 = __builtin_amdgcn_perm(v[3], v[2], 0x04000c0cu);
        const uint32_t h01 = __builtin_amdgcn_perm(v[1] + 128, v[0] + 128, 0x0c0c0501u);
        const uint32_t h23 = __builtin_amdgcn_perm(v[3] + 128, v[2] + 128, 0x05010c0cu);
        qhi[s][w] = (int)(h01 | h23);
        qlo[s][w] = (int)(l01 | l23);
      }
  }
  const float qf = row.bad ? __builtin_nanf("") : __builtin_ldexpf(p.to_log2, row.e - 14);

  const TreeBy score(row.bad ? __builtin_nanf("") : p.to_log2, row.e - 14);

  f32x16 acc[KS];
#pragma unroll
  for (int c = 0; c < KS; ++c)
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[c][v] = 0.f;
  TreeState st;
  float psum = 0.f;  // of the rounded probabilities times the value scales
  float most = 0.f;  // see tree_any_scales

  const int krow = tree_row(col);
  const uint32_t koff = krow * D, ksw = tree_swizzle<D>(krow);
  const uint32_t voff = h * D + (D == 64 ? 4 * (col & 15) : D / 32 * col);
  const uint32_t vsel = D == 64 ? (uint32_t)(col >> 4) * 0x00020002u : 0u;  // the lane's channels of its 4
  // The wave's 32 keys of a turn: scores, probabilities, values.
  const auto compute = [&](auto slow, int t0, int stage) {
    const uint8_t* kt = ring + stage * 2 * C::kHalf + koff;
    const uint8_t* vt = ring + stage * 2 * C::kHalf + C::kHalf + voff;
    const float* sc = scales + 4 * h;
    i32x16 hi, lo;
#pragma unroll
    for (int v = 0; v < 16; ++v) hi[v] = lo[v] = 0;
    i32x4 a[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) a[s] = *reinterpret_cast<const i32x4*>(kt + 16 * ((2 * s + h) ^ ksw));
    __builtin_amdgcn_sched_barrier(0);  // all on their way before the first product
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      hi = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[s], qhi[s], hi, 0, 0, 0);
      lo = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[s], qlo[s], lo, 0, 0, 0);
    }
    uint32_t vis = 0;
    if constexpr (slow) vis = row.live ? tree_visible(p, seq, row.j, t0, c1, h) : 0u;
    float t[16], top = -__builtin_inff();
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 ksv = *reinterpret_cast<const f32x4*>(sc + 8 * g);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int v = 4 * g + u;
        const float sum = (float)((hi[v] << 8) + lo[v]);
        t[v] = kAny ? score(sum, ksv[u]) : sum * ksv[u];
        if constexpr (slow) t[v] = vis >> (8 * g + u) & 1 ? t[v] : -__builtin_inff();
        top = fmaxf(top, t[v]);
      }
    }
    const auto fade = [&](float f) {
      psum *= f;
#pragma unroll
      for (int c = 0; c < KS; ++c)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[c][v] *= f;
    };
    if constexpr (kAny)
      tree_any_scales(st, most, t, [&](int g) { return *reinterpret_cast<const f32x4*>(sc + 32 + 8 * g); }, fade);
    else
      tree_raise(st, top * qf, sc[64 - 4 * h], fade);
#pragma unroll
    for (int mm = 0; mm < 2; ++mm) {  // 16 keys: 8 of each half wave
      // the lane's channels of its half wave's 8 keys; byte b of two keys makes one
      // operand word
      constexpr int W = D == 256 ? 2 : 1;
      uint32_t x[8][W];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint8_t* src = vt + (16 * mm + tree_row(8 * (i >> 2) + (i & 3))) * D;
        if constexpr (W == 2) {
          const u32x2 y = *reinterpret_cast<const u32x2*>(src);
          x[i][0] = y[0];
          x[i][1] = y[1];
        } else {
          x[i][0] = *reinterpret_cast<const uint32_t*>(src);
        }
      }
      f32x4 vsv[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) vsv[g] = *reinterpret_cast<const f32x4*>(sc + 32 + 16 * mm + 8 * g);
      __builtin_amdgcn_sched_barrier(0);  // the same: 16-token trees over 32 K tokens 72.3 us, 70.6 so
      f16x8 pv;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if constexpr (kAny) {
            pv[4 * g + u] = (_Float16)t[8 * mm + 4 * g + u];
            continue;
          }
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(t[8 * mm + 4 * g + u], qf, -st.m));
          float w = e * vsv[g][u];
          if constexpr (slow) {
            const bool on = vis >> (16 * mm + 8 * g + u) & 1;
            st.l += on ? e : 0.f;
            w = on ? w : 0.f;
          } else {
            st.l += e;
          }
          pv[4 * g + u] = (_Float16)w;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const f16x2 one = {(_Float16)1.f, (_Float16)1.f}, pair = {pv[2 * u], pv[2 * u + 1]};
        psum = __builtin_amdgcn_fdot2(pair, one, psum, false);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int w = 0; w < W; ++w) x[i][w] ^= 0x80808080u;
#pragma unroll
      for (int c = 0; c < KS; ++c) {
        u32x4 a;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          a[q] = __builtin_amdgcn_perm(x[2 * q + 1][c >> 2], x[2 * q][c >> 2],
                                       0x0c040c00u + (uint32_t)(c & 3) * 0x00010001u + vsel);
        acc[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), pv, acc[c], 0, 0, 0);
      }
    }
  };

  // Turn i: its tile has landed; the next is issued into the other half of the ring,
  // whose reads are done. The waves work apart. (A third stage: at 64 channels 13.1 us
  // against 12.5 for 24 trees of 5 over 3000 tokens, one token over 32 K 12.5 and 11.7.)
  int stage = 0;
  const int place = (int)(blockIdx.x >> 3) / (kTreeCus / 8);  // 32 CUs per XCD
  const auto advance = [&](int i) {
    if (C::kPerCu > 1) tree_priority<C::kPerCu>(place + i);
    tree_landed();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // and reads of the scales
    put.put(p, keys, scales);
    issue(i + 1, stage ^ 1);
  };
  // first the turns whose tile every row sees whole
  const int open = (n_all < c1 ? n_all : c1) - tile_at(0);
  int fast = open >= C::kTile ? (open / C::kTile - 1) / 4 + 1 : 0;
  fast = fast < turns ? fast : turns;
  int i = 0;
  if constexpr (!kAny)
    for (; i < fast; ++i) {
      advance(i);
      if (put.odd) break;
      compute(std::false_type{}, 0, stage);
      stage ^= 1;
    }
  for (; i < turns && !put.odd; ++i) {
    advance(i);
    if (put.odd) break;
    compute(std::true_type{}, tile_at(i), stage);
    stage ^= 1;
  }
  tree_landed();
  int* odd = reinterpret_cast<int*>(smem + C::kLds - 16);  // of each wave
  if (!kAny && lane == 0) odd[wave] = put.odd || st.huge;

  // Both half waves hold half of a row's keys in l and psum.
  float l = st.l + __shfl_xor(st.l, 32), m = st.m;
  psum += __shfl_xor(psum, 32);
  // The waves' sums meet in LDS, each brought to the common maximum; then every
  // thread adds four channels of a row in wave order. A row's 16-byte runs are
  // swizzled by the row, so that the 32 rows of a store meet all banks.
  float* sum = reinterpret_cast<float*>(smem);  // [wave][row][D]
  float* stats = reinterpret_cast<float*>(smem + 4 * C::kRows * D * 4);  // [wave][row]: maximum, sum
  static_assert(4 * C::kRows * (D * 4 + 8) <= C::kLds, "merge");
  __syncthreads();
  if constexpr (!kAny)
    if (odd[0] | odd[1] | odd[2] | odd[3]) return false;
  if (h == 0) *reinterpret_cast<f32x2*>(stats + 2 * (wave * C::kRows + col)) = f32x2{m, l};
  __syncthreads();
  const auto joint = [&](int row, float* all) {
    f32x2 st[4];
    float to = kTreeFloor;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      st[g] = *reinterpret_cast<const f32x2*>(stats + 2 * (g * C::kRows + row));
      to = fmaxf(to, st[g][0]);
    }
    *all = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g) *all += st[g][1] * __builtin_amdgcn_exp2f(st[g][0] - to);
    return to;
  };
  float all;
  // 2^24 / factor may leave the range of FP32 where the sums do not: two steps there
  const float up = __builtin_amdgcn_exp2f(m - joint(col, &all)) * ((kAny ? 1.f : 0x1p24f) / st.factor);
  const float shift = 128.f * psum * 0x1p-24f;
  if (row.live)
    tree_runs<D>(acc, h, [&](int c, f32x4 v) {
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = kAny ? (v[u] - shift) * 0x1p24f * up : (v[u] - shift) * up;
      return *reinterpret_cast<f32x4*>(sum + (wave * C::kRows + col) * D + 4 * ((c / 4) ^ (col & (D / 4 - 1)))) = v;
    });
  __syncthreads();
  const int first = it.tile * C::kRows, left = seq.count * p.r - first;
  const int live = left < C::kRows ? left : C::kRows;
  const bool split = chunks > 1;
  for (int i = threadIdx.x; i < live * (D / 4); i += kTreeThreads) {
    const int rr = i / (D / 4), c = i % (D / 4);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < 4; ++g)
      v += *reinterpret_cast<const f32x4*>(sum + (g * C::kRows + rr) * D + 4 * (c ^ (rr & (D / 4 - 1))));
    const float to = joint(rr, &all);
    const int64_t place = (int64_t)it.place * C::kRows + rr;
    if (split) {
      *reinterpret_cast<f32x4*>(p.part + place * D + 4 * c) = v;
      if (c == 0) *reinterpret_cast<f32x2*>(p.stat + 2 * place) = f32x2{to, all};
    } else {
      const float inv = all == 0.f ? 0.f : 1.f / all;
      const int j = (first + rr) / p.r, hh = first + rr - j * p.r;
      *reinterpret_cast<u32x2*>(p.out + ((int64_t)(seq.start + j) * p.hq + it.kh * p.r + hh) * D + 4 * c) =
          u32x2{pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv)};
    }
  }
  return true;
}

template <int D>
__global__ void __launch_bounds__(kTreeThreads, TreeThin<D>::kPerCu) tree_thin_kernel(TreeParams p) {
  if (tree_left(tree_thin_pass<D, false>(p))) {
    __syncthreads();  // all have read the flags
    tree_thin_pass<D, true>(tree_again());
  }
}

// ---------------------------------------------------------------------------
// Many rows. The four waves bring a tile's codes to FP16 together, (code) 2^-24,
// exact, in the order of the matrix operands; each then works on its 32 rows. Queries
// are FP16 too, scaled by a power of two that the wave's rows share, so that it and 1
// / sqrt(D) go into the keys' scales and one FMA gives a score less its row's maximum
// (221 us against 228 for 64-token trees over 32 K tokens): exact for values down to
// 2^-28 of the largest of the 32 rows, below that off by 2^-39 of it. Rows that lie
// further apart than 2^16 take the pass for odd scales, where each has its own power, so
// that a row's values are exact down to 2^-12 of its largest at least, and the others
// off by 2^-23 of that. (A chunk of 1024 tokens over 8 K, 256-wide heads: 300 us in the
// kernel for few rows, 235 here; with three workgroups per CU in place of two at 128
// channels, 64-token trees over 32 K 238 and 220.)
// With 128 channels, 64 keys cost a wave some 350 vector instructions
// and 32 MFMAs, 1024 cycles of the matrix cores; a vector instruction issues in 61 %
// of a SIMD's cycles and the matrix cores work in 33 %. Measured and left: 64 rows per wave,
// which share the operands from LDS (registers spill at 128 channels: 347 us against
// 247; at 64, two waves per SIMD, 294 against 293); addresses within the tile held in
// registers (1 % faster at 128 channels, 4 % slower at 256).
// ---------------------------------------------------------------------------
template <int D, bool kAny>
__device__ __forceinline__ bool tree_wide_pass(const TreeParams& p) {
  using C = TreeWide<D>;
  constexpr int KS = D / 32, T = C::kTile;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  TreeItem it;
  if (!tree_item<C::kRows, C::kStep>(p, it)) return true;  // uniform over the workgroup
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, h = lane >> 5;
  const TreeSeq seq = it.seq;
  int n, n_all;
  tree_reach(p, seq, it.tile, C::kRows, &n, &n_all);
  const int chunks = tree_chunks(n, it.keys);
  if (it.chunk >= chunks) return true;
  const int span = tree_span(n, chunks, C::kStep), c0 = it.chunk * span;
  const int c1 = n - c0 < span ? n : c0 + span;
  const int turns = (c1 - c0 + T - 1) / T;

  uint8_t* kr = smem;                  // the codes as they lie in the cache
  uint8_t* vr = kr + C::kHalf;
  uint8_t* kf = vr + C::kHalf;         // [16-channel step][half][key] x 8 channels
  uint8_t* vf = kf + 2 * C::kHalf;     // [16 keys][half][channel block][row] x 8 keys
  float* scales = reinterpret_cast<float*>(vf + 2 * C::kHalf + wave * C::kScale);
  uint64_t* wanted = reinterpret_cast<uint64_t*>(vf + 2 * C::kHalf + 4 * C::kScale);
  uint8_t* ql = vf + 2 * C::kHalf + 4 * C::kScale + 32 + 1024 * C::kQueries * wave + 16 * lane;
  TreeLookup<T> keys{p.table + (int64_t)it.b * p.pps, wanted, c1, seq.len, it.kh, lane, p.masks && c1 > seq.len,
                     0, 0, 0, false, false};
  TreeScales<T, kAny> put;  // the waves look at the same scales, and find the same ones odd
  const auto tile_at = [&](int i) { return c0 + i * T; };
  keys.ask(p, tile_at(0));
  TreeRow<D> row;
  row.template ask<false>(p, it, it.tile * C::kRows + wave * 32 + col, h);
  if (keys.pick) {
    if (wave == 0) tree_wanted(p, seq, wanted);
    __syncthreads();
  }
  const uint32_t row_bytes = (uint32_t)p.kvh * D;
  const int8_t* kbase = p.kc + (int64_t)it.kh * D;
  const int8_t* vbase = p.vc + (int64_t)it.kh * D;
  constexpr int kDma = C::kHalf / 4096;  // DMA instructions per wave for keys, and for values
  const auto issue = [&](int i) {
    const int r = keys.row(p, tile_at(i), tile_at(i + 1));
    const uint32_t at = tree_opaque(lane);
#pragma unroll
    for (int d = 0; d < kDma; ++d) {
      const uint32_t first = 64 * (wave * kDma + d);  // chunks of 16 bytes
      const uint32_t line = first / (D / 16) + at / (D / 16), slot = at % (D / 16);
      const uint32_t rr = __builtin_amdgcn_ds_bpermute(4 * tree_row(line), r);
      const int8_t* k = kbase + (uint64_t)rr * row_bytes + 16 * (slot ^ tree_swizzle<D>(line));
      const int8_t* v = vbase + (uint64_t)rr * row_bytes + 16 * slot;
      __builtin_amdgcn_global_load_lds(k, LDS_PTR(kr + 16 * first), 16, 0, 0);
      __builtin_amdgcn_global_load_lds(v, LDS_PTR(vr + 16 * first), 16, 0, 0);
    }
  };
  issue(0);

  row.scale();
  // the largest of the wave's rows; each row's own where scales are odd
  const int e = kAny ? row.e
                     : __builtin_amdgcn_readfirstlane(
                           tree_wave_reduce(row.bad ? -112 : row.e, [](int a, int b) { return a > b ? a : b; }));
  const TreeBy score(1.f, e + 10);
  // Rows whose largest is below 2^-16 of that lose bits, and scores of queries past 2^60 may
  // leave the range of FP32 on the way: then each row by itself (rows of zeros, and of
  // 2^-112 and less, whose scores are as good as 0 with key scales that are not odd, do
  // not count).
  const bool far = !kAny && (__any(!row.bad & (row.e > -112) & (e - row.e > 16)) || e > 60);
  f16x8 q[KS][2];
  {
    const float up = row.bad ? __builtin_nanf("") : __builtin_ldexpf(1.f, 14 - e);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) q[s][i][k] = (_Float16)(row.value(s, i, k) * up);
#pragma unroll
    for (int k = 0; k < C::kQueries; ++k) *reinterpret_cast<f16x8*>(ql + 1024 * k) = q[k >> 1][k & 1];
  }
  // the lane's row, formed anew where registers are short: at 128 channels two more
  // made a query operand spill, and its reload wait for the DMA (210 us became 230)
  const auto which = [&] {
    return it.tile * C::kRows + wave * 32 + (int)((D == 128 ? tree_opaque(lane) : (uint32_t)lane) & 31);
  };
  const bool rows = it.tile * C::kRows + wave * 32 < seq.count * p.r;  // the wave has any

  f32x16 acc[KS];
#pragma unroll
  for (int c = 0; c < KS; ++c)
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[c][v] = 0.f;
  std::conditional_t<kAny, TreeState, TreeLevel> st;
  float most = 0.f;  // see tree_any_scales

  // The tile's codes into FP16: a key's 16 channels per thread and turn, then four
  // keys' D / 32 channels (of D = 64: 4). Code + 128 as a subnormal, less 128.
  const f16x2 bias = __builtin_bit_cast(f16x2, 0x80808080u);  // -128 2^-24 each
  const auto half2 = [&](uint32_t hi, uint32_t lo, uint32_t sel) {
    return __builtin_bit_cast(uint32_t, (f16x2)(__builtin_bit_cast(f16x2, __builtin_amdgcn_perm(hi, lo, sel)) + bias));
  };
  const auto convert = [&]() {
    const uint32_t tid = tree_opaque(threadIdx.x);
#pragma unroll
    for (int i = 0; i < C::kHalf / 4096; ++i) {
      const uint32_t key = tid % T, chunk = tid / T + i * (kTreeThreads / T), line = tree_row(key);
      u32x4 x = *reinterpret_cast<const u32x4*>(kr + line * D + 16 * (chunk ^ tree_swizzle<D>(line)));
      u32x4 y[2];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t u = x[w] ^ 0x80808080u;
        y[w >> 1][2 * (w & 1)] = half2(u, u, 0x0c010c00u);
        y[w >> 1][2 * (w & 1) + 1] = half2(u, u, 0x0c030c02u);
      }
      *reinterpret_cast<u32x4*>(kf + 16 * ((2 * chunk) * T + key)) = y[0];
      *reinterpret_cast<u32x4*>(kf + 16 * ((2 * chunk + 1) * T + key)) = y[1];
    }
    constexpr int kLanes = D == 64 ? 16 : 32, W = D == 256 ? 2 : 1;
    const uint32_t quad = tid % kLanes;
#pragma unroll
    for (int k = 0; k < T / 4 * kLanes / kTreeThreads; ++k) {
      const uint32_t four = tid / kLanes + k * (kTreeThreads / kLanes);  // keys 4 four + [0, 4)
      uint32_t x[4][W];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* src = vr + tree_row(4 * four + i) * D + 4 * W * quad;
        if constexpr (W == 2) {
          const u32x2 y = *reinterpret_cast<const u32x2*>(src);
          x[i][0] = y[0] ^ 0x80808080u;
          x[i][1] = y[1] ^ 0x80808080u;
        } else {
          x[i][0] = *reinterpret_cast<const uint32_t*>(src) ^ 0x80808080u;
        }
      }
      // keys 4 four + i: 16 keys' block four / 4, half wave four & 1, operand place 4
      // (four / 2 & 1) + i
      uint8_t* dst = vf + 16 * ((four >> 2) * 2 + (four & 1)) * KS * 32 + 8 * (four >> 1 & 1);
#pragma unroll
      for (int b = 0; b < 4 * W; ++b) {
        const uint32_t sel = 0x0c040c00u + (uint32_t)(b & 3) * 0x00010001u;
        const u32x2 y = {half2(x[1][b >> 2], x[0][b >> 2], sel), half2(x[3][b >> 2], x[2][b >> 2], sel)};
        const uint32_t c = D == 64 ? b & 1 : b, r = D == 64 ? quad + 16 * (b >> 1) : quad;
        *reinterpret_cast<u32x2*>(dst + 16 * (c * 32 + r)) = y;
      }
    }
  };
  const auto compute = [&](auto slow, int t0) {
    const uint8_t* kt = kf + 16 * (h * T + col);
    const uint8_t* vt = vf + 16 * (h * KS * 32 + col);
    const float* sc = scales + 4 * h;
#pragma unroll
    for (int nb = 0; nb < T / 32; ++nb) {
      f32x16 s;
#pragma unroll
      for (int v = 0; v < 16; ++v) s[v] = 0.f;
      const auto key = [&](int k) { return *reinterpret_cast<const f16x8*>(kt + 16 * (2 * k * T + 32 * nb)); };
      f16x8 a[2 * KS];
      a[0] = key(0);
      a[1] = key(1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < 2 * KS; ++k) {
        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(
            a[k], k < C::kQueries ? *reinterpret_cast<const f16x8*>(ql + 1024 * k) : q[k >> 1][k & 1], s, 0, 0, 0);
        if (k + 2 < 2 * KS) a[k + 2] = key(k + 2);
      }
      uint32_t vis = 0;
      if constexpr (slow) {
        const int i = which();
        vis = i < seq.count * p.r ? tree_visible(p, seq, i / p.r, t0 + 32 * nb, c1, h) : 0u;
      }
      float t[16], top = -__builtin_inff();
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 ksv = *reinterpret_cast<const f32x4*>(sc + 32 * nb + 8 * g);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int v = 4 * g + u;
          t[v] = kAny ? score(s[v], ksv[u]) : __builtin_fmaf(s[v], ksv[u], -st.m);
          if constexpr (slow) t[v] = vis >> (8 * g + u) & 1 ? t[v] : -__builtin_inff();
          top = fmaxf(top, t[v]);
        }
      }
      const auto fade = [&](float f) {
#pragma unroll
        for (int c = 0; c < KS; ++c)
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[c][v] *= f;
      };
      if constexpr (kAny)
        tree_any_scales(st, most, t, [&](int g) { return *reinterpret_cast<const f32x4*>(sc + T + 32 * nb + 8 * g); },
                        fade);
      else
        tree_level(st, t, top, sc[2 * T - 4 * h], fade);
      // Two operands of each sixteen keys' values are on their way before their
      // probabilities are formed, and nothing is moved across: left to itself the
      // scheduler read them one by one, each product waiting for LDS (64-token trees
      // over 32 K tokens 221 us against 210; with four of them registers spill, 232).
#pragma unroll
      for (int mm = 0; mm < 2; ++mm) {
        const auto value = [&](int c) {
          return *reinterpret_cast<const f16x8*>(vt + 16 * (((2 * nb + mm) * 2 * KS + c) * 32));
        };
        const f16x8 x[2] = {value(0), value(1)};
        f16x8 pv;
        f32x4 vsv[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) vsv[g] = *reinterpret_cast<const f32x4*>(sc + T + 32 * nb + 16 * mm + 8 * g);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if constexpr (kAny) {
              pv[4 * g + u] = (_Float16)t[8 * mm + 4 * g + u];
              continue;
            }
            const float y = __builtin_amdgcn_exp2f(t[8 * mm + 4 * g + u]);
            float w = y * vsv[g][u];
            if constexpr (slow) {
              const bool on = vis >> (16 * mm + 8 * g + u) & 1;
              st.l += on ? y : 0.f;
              w = on ? w : 0.f;
            } else {
              st.l += y;
            }
            pv[4 * g + u] = (_Float16)w;
          }
        }
#pragma unroll
        for (int c = 0; c < KS; ++c)
          acc[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(c < 2 ? x[c & 1] : value(c), pv, acc[c], 0, 0, 0);
      }
    }
  };

  // Turn i: the tile's DMA has landed; all waves convert it, issue the next tile
  // into its place, and compute.
  const int place = (int)(blockIdx.x >> 3) / (kTreeCus / 8);  // 32 CUs per XCD
  const auto advance = [&](int i) {
    tree_priority<C::kPerCu>(place + i);
    tree_landed();
    put.put(p, keys, scales, p.to_log2, kAny ? 0 : e + 10);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    convert();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    issue(i + 1);
  };
  const int open = (n_all < c1 ? n_all : c1) - c0;
  const int fast = open >= T ? (open / T < turns ? open / T : turns) : 0;
  int i = 0;
  if constexpr (!kAny)
    for (; i < fast; ++i) {
      advance(i);
      if (put.odd) break;
      if (rows) compute(std::false_type{}, 0);
    }
  for (; i < turns && !put.odd; ++i) {
    advance(i);
    if (put.odd) break;
    if (rows) compute(std::true_type{}, tile_at(i));
  }
  tree_landed();
  if (put.odd) return false;
  if constexpr (!kAny) {
    int* again = reinterpret_cast<int*>(smem + C::kLds - 16);  // of each wave
    if (lane == 0) again[wave] = far || st.huge;
    __syncthreads();
    if (again[0] | again[1] | again[2] | again[3]) return false;
  }
  const float l = st.l + __shfl_xor(st.l, 32), up = (kAny ? 1.f : 0x1p24f) / st.factor;
#pragma unroll
  for (int c = 0; c < KS; ++c)
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[c][v] = kAny ? acc[c][v] * 0x1p24f * up : acc[c][v] * up;  // as in the thin kernel
  const int at = which();
  float m = st.m;
  if constexpr (!kAny) m = st.limit < 0.f ? kTreeFloor : m;
  if (at < seq.count * p.r)
    tree_result<D>(p, it, acc, chunks > 1, m, l, at / p.r, at % p.r, (int64_t)it.place * C::kRows + wave * 32 + col, h);
  return true;
}

template <int D>
__global__ void __launch_bounds__(kTreeThreads, TreeWide<D>::kPerCu) tree_wide_kernel(TreeParams p) {
  if (tree_left(tree_wide_pass<D, false>(p))) {
    __syncthreads();  // all are done with the masks
    tree_wide_pass<D, true>(tree_again());
  }
}

// The chunks' sums of a row and head joined in chunk order, D / 4 lanes of four
// channels each. ``parts`` groups of lanes take a head's chunks between them, in
// runs, and meet in LDS. Eight chunks' sums are loaded at a time; lane i of the
// group holds the weight of chunk i.
template <int D, bool kJoin>
__global__ void __launch_bounds__(kTreeThreads) tree_combine_kernel(TreeParams p, int tile_rows, int log_parts) {
  constexpr int W = D / 4, kGroups = kTreeThreads / W;
  if (!kJoin) log_parts = 0;
  __shared__ f32x4 sums[kTreeThreads];
  __shared__ f32x2 stats[kGroups];
  const int row = blockIdx.x, lane = threadIdx.x & 63;
  const int keys = p.info[p.batch];
  TreeSeq s{0, 0, 0, 0};
  int b = -1, from = 0;  // the row's sequence: the first that ends behind it
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const int mine = b0 + lane < p.batch ? b0 + lane : p.batch - 1;
    const TreeSeq t = tree_seq(p, mine);
    const int at = p.info[mine];
    const uint64_t has = __ballot(b0 + lane < p.batch && p.starts[mine + 1] > row);
    if (has) {
      const int on = __builtin_ctzll(has);
      b = b0 + on;
      s.start = __builtin_amdgcn_readlane(t.start, on);
      s.count = __builtin_amdgcn_readlane(t.count, on);
      s.len = __builtin_amdgcn_readlane(t.len, on);
      s.n = __builtin_amdgcn_readlane(t.n, on);
      from = __builtin_amdgcn_readlane(at, on);
      break;
    }
  }
  const int j = row - s.start;
  if (b < 0 || j < 0 || j >= s.count || s.n <= keys) return;  // the whole workgroup; not split
  const int parts = 1 << log_parts, group = threadIdx.x / W, part = group & (parts - 1), in = lane & (W - 1);
  // one turn where the groups meet (kJoin)
  for (unsigned y = blockIdx.y; y * kGroups < (unsigned)p.hq << log_parts; y += gridDim.y) {
    const int head = (int)(y * kGroups + group) >> log_parts, c = 4 * in;
    const int kh = head / p.r, rr = j * p.r + head - kh * p.r;
    const int tile = rr / tile_rows, tiles = tree_tiles(p, s, tile_rows);
    int n, n_all;
    tree_reach(p, s, tile, tile_rows, &n, &n_all);
    int chunks = tree_chunks(n, keys);
    const int64_t first = ((int64_t)from + (int64_t)kh * tiles + tile) * tile_rows + rr - tile * tile_rows;
    const int64_t step = (int64_t)p.kvh * tiles * tile_rows;
    // starts that do not ascend can name more items than the workspace has places for
    const bool live =
        head < p.hq && chunks > 1 && from >= 0 && first + (chunks - 1) * step < (int64_t)p.parts * tile_rows;
    const int run = (chunks + parts - 1) >> log_parts, end_run = (part + 1) * run;
    const int to_chunk = live ? (end_run < chunks ? end_run : chunks) : 0;
    float m = kTreeFloor, l = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = part * run; i0 < to_chunk; i0 += W) {
      const bool on = i0 + in < to_chunk;
      const f32x2* from = reinterpret_cast<const f32x2*>(p.stat + 2 * (first + (i0 + in) * step));
      const f32x2 st = on ? *from : f32x2{kTreeFloor, 0.f};
      float to = st[0];
#pragma unroll
      for (int off = 1; off < W; off <<= 1) to = fmaxf(to, __shfl_xor(to, off));
      to = fmaxf(to, m);
      const float fade = __builtin_amdgcn_exp2f(m - to), weight = __builtin_amdgcn_exp2f(st[0] - to);
      m = to;
      float some = st[1] * weight;
#pragma unroll
      for (int off = 1; off < W; off <<= 1) some += __shfl_xor(some, off);
      l = l * fade + some;
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] *= fade;
      const int end = to_chunk - i0 < W ? to_chunk - i0 : W;
      for (int i = 0; i < end; i += 8) {
        f32x4 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int ii = i + k < end ? i + k : end - 1;
          x[k] = *reinterpret_cast<const f32x4*>(p.part + (first + (i0 + ii) * step) * D + c);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float f = __shfl(weight, i + k, W);
          if (i + k < end)
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = __builtin_fmaf(x[k][u], f, v[u]);
        }
      }
    }
    if constexpr (kJoin) {
      sums[threadIdx.x] = v;
      if (in == 0) stats[group] = f32x2{m, l};
      __syncthreads();
      if (part) continue;
      float to = m;
      for (int g = 1; g < parts; ++g) to = fmaxf(to, stats[group + g][0]);
      const float fade = __builtin_amdgcn_exp2f(m - to);
      l *= fade;
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] *= fade;
      for (int g = 1; g < parts; ++g) {
        const f32x2 st = stats[group + g];
        const f32x4 x = sums[threadIdx.x + g * W];
        const float weight = __builtin_amdgcn_exp2f(st[0] - to);
        l = __builtin_fmaf(st[1], weight, l);
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = __builtin_fmaf(x[u], weight, v[u]);
      }
    }
    if (!live) continue;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<u32x2*>(p.out + ((int64_t)row * p.hq + head) * D + c) =
        u32x2{pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv)};
  }
}


// The sizes that 32-bit indexes of tiles and tokens hold.
static bool tree_holds(int64_t rows, int64_t hq, int64_t kvh, int64_t batch, int64_t max_count) {
  return rows >= 1 && rows < (1 << 24) && max_count >= 1 && max_count < (1 << 24) && batch >= 1 && batch <= 65535 &&
         kvh >= 1 && kvh <= kTreeMaxHeads && hq >= 1 && hq <= kTreeMaxHeads && hq % kvh == 0 &&
         rows * (hq / kvh) < (1 << 30);
}

struct TreeLayout {
  int wide;
  int slots, whole;
  int64_t units;  // row tiles x KV heads, at most
  int64_t parts;  // places for partial sums
  int64_t grid;   // at most so many workgroups have work
  size_t info, whose, stat, part, total;
};

static size_t tree_align(size_t v) { return (v + 255) & ~(size_t)255; }

template <int D>
static int tree_per_cu(bool wide) { return wide ? TreeWide<D>::kPerCu : TreeThin<D>::kPerCu; }

static TreeLayout tree_layout(int64_t batch, int64_t rows, int64_t max_count, int64_t hq, int64_t kvh, int64_t dim,
                              int64_t cap) {
  TreeLayout L;
  const int64_t r = hq / kvh;
  // row tiles of all sequences together, at most: each sequence ends with one that
  // is not full
  const auto tiles = [&](int64_t tile) {
    const int64_t by_batch = batch * cdiv(max_count * r, tile), by_rows = rows * r / tile + batch;
    return kvh * (by_batch < by_rows ? by_batch : by_rows);
  };
  const auto slots = [&](bool wide) {
    return kTreeCus *
           (dim == 64 ? tree_per_cu<64>(wide) : (dim == 128 ? tree_per_cu<128>(wide) : tree_per_cu<256>(wide)));
  };
  // The wide kernel has the higher rate, but its workgroups' partial sums are four
  // times as many bytes: some 25 us more for writing and joining them. It is taken for
  // more than three thin tiles per sequence and KV head where those would fill the
  // chip (then they run in turns; 8 sequences of 64 tokens x 8 heads over 500 tokens
  // 38 us against 44, over 32 K 239 against 335) or where the work, at the sequences'
  // capacity (only the GPU knows the lengths), is beyond 2^36 operations, 2^35 with D
  // = 64, whose exponentials weigh more. With D = 128, thin against wide, in us with
  // the join: 2 x 16 tokens over 2000 18 and 34, 4 x 32 over 8000 35 and 47, 2 x 64
  // over 32 K (2^36) 87 and 90, 4 x 64 over 32 K (2^37) 184 and 145; 64 rows per head
  // over 32 K 48 and 60, 96 rows 61 and 70. With D = 64, 8 KV heads, 1 x 64 over 8000
  // 31 and 40, 4 x 16 over 32 K (2^35) 66 and 58; with D = 256, 2 KV heads, 4 x 16
  // over 32 K (2^35) 64 and 72, 4 x 32 (2^36) 110 and 96. Short contexts under a wide
  // table pay for it: in one of 128 K tokens 4 x 16 over 1000 21.3 us against 16.9 in a
  // table of their own width, 4 x 32 over 8000 45.4 and 34.2.
  const int64_t thin = TreeThin<128>::kRows;
  L.wide = max_count * r > 3 * thin &&
           (2 * tiles(thin) > slots(false) || (double)rows * hq * cap * dim * 4. > (dim == 64 ? 0x1p35 : 0x1p36));
  const int64_t tile = L.wide ? TreeWide<128>::kRows : thin, units = tiles(tile);
  L.slots = slots(L.wide);
  L.units = units;
  // Many short sequences fill the chip without a split, and a launch less; one long
  // one among them (its capacity tells) has to be split all the same: 600 of 300
  // tokens and one of 30 K, one token each, 286 us without and 87 with.
  const int64_t step = L.wide ? (dim == 256 ? TreeWide<256>::kStep : TreeWide<128>::kStep) : TreeThin<128>::kStep;
  L.whole = units >= 4 * L.slots && cap <= 32 * step;
  const bool once = 2 * units <= L.slots;
  L.grid = L.whole ? units : (once ? L.slots : units + 2 * L.slots);
  L.grid = cdiv(L.grid, 8) * 8;  // whole runs per XCD
  // In turns a chunk has more keys than a half of a place's share, and a split
  // sequence less than twice its keys' share of chunks (64: of the sum's rounding).
  L.parts = L.whole ? 0 : (once ? L.grid : 4 * L.slots + 64);
  L.info = 0;
  L.whose = tree_align(L.info + (size_t)(2 * batch + 2) * 4);
  L.stat = tree_align(L.whose + (batch > kTreeLanes ? (size_t)L.grid * 4 : 0));
  L.part = tree_align(L.stat + (size_t)(L.parts * tile) * 8);
  L.total = tree_align(L.part + (size_t)(L.parts * tile) * dim * 4);
  return L;
}

template <typename C, typename K>
static void tree_run(K kernel, std::atomic<uint64_t>& done, const TreeParams& p, const TreeLayout& L, hipStream_t s) {
  once_per_device(done, [&] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                              C::kLds);
  });
  if (p.whose) hipLaunchKernelGGL((tree_plan_kernel<C::kRows, C::kStep>), dim3(1), dim3(kTreePlan), 0, s, p);
  hipLaunchKernelGGL(kernel, dim3((unsigned)L.grid), dim3(kTreeThreads), C::kLds, s, p);
}

template <int D>
static int tree_launch(const TreeParams& p, const TreeLayout& L, hipStream_t s) {
  static std::atomic<uint64_t> thin{0}, wide{0};
  if (L.wide)
    tree_run<TreeWide<D>>(tree_wide_kernel<D>, wide, p, L, s);
  else
    tree_run<TreeThin<D>>(tree_thin_kernel<D>, thin, p, L, s);
  if (!L.whole) {
    constexpr int kGroups = 4 * kTreeThreads / D;
    // A group of lanes for every 8 of the chunks that a row is expected to have: one
    // sequence's token over 32 K tokens 14.3 us with one group, 5.8 with eight; its
    // tree of 16 26.6 and 11.0. (For every 4: 8 chunks 4.0 us against 3.7.)
    const int64_t share = L.slots / L.units, most = cdiv(p.cap, L.wide ? TreeWide<D>::kStep : TreeThin<D>::kStep);
    const int64_t chunks = share < most ? share : most;
    int log_parts = 0;
    while ((1 << log_parts) < kGroups && (16 << log_parts) <= chunks) ++log_parts;
    const auto kernel = log_parts ? tree_combine_kernel<D, true> : tree_combine_kernel<D, false>;
    // Many rows are one workgroup each: where few are split, finding that out counts
    // (16384 rows of 32 heads, none split, 46 us, 6.5 so).
    const int64_t heads = log_parts || p.rows <= 4096 ? cdiv((int64_t)p.hq << log_parts, kGroups) : 1;
    hipLaunchKernelGGL(kernel, dim3((unsigned)p.rows, (unsigned)heads), dim3(kTreeThreads), 0, s, p,
                       L.wide ? TreeWide<D>::kRows : TreeThin<D>::kRows, log_parts);
  }
  return check_launch("tree_attention");
}

}  // namespace q6moe

using namespace q6moe;

extern "C" size_t q6moe_tree_attn_workspace_size(int64_t batch, int64_t rows, int64_t max_count, int64_t query_heads,
                                                 int64_t kv_heads, int64_t head_dim, int64_t pages_per_seq,
                                                 int64_t page_size) {
  if (!tree_holds(rows, query_heads, kv_heads, batch, max_count) || pages_per_seq < 1 || page_size < 1 ||
      pages_per_seq >= (1 << 30) || page_size >= (1 << 30) || pages_per_seq * page_size > (1 << 30))
    return 0;
  return tree_layout(batch, rows, max_count, query_heads, kv_heads, head_dim,
                     pages_per_seq * page_size).total;
}

extern "C" int q6moe_kv_tree_attention(const q6moe_tree_attn_args* a, void* stream) {
  Q6MOE_REQUIRE(a, "tree_attention: null args");
  Q6MOE_REQUIRE(a->q && a->k_codes && a->v_codes && a->k_scales && a->v_scales && a->page_table && a->lengths &&
                    a->starts && a->out,
                "tree_attention: null pointer");
  Q6MOE_REQUIRE(a->head_dim == 64 || a->head_dim == 128 || a->head_dim == 256,
                "tree_attention: head_dim must be 64, 128 or 256");
  Q6MOE_REQUIRE(a->batch >= 1 && a->batch <= 65535 && a->kv_heads >= 1 && a->kv_heads <= kTreeMaxHeads &&
                    a->query_heads >= 1 && a->query_heads <= kTreeMaxHeads && a->query_heads % a->kv_heads == 0,
                "tree_attention: query_heads must be a multiple of kv_heads, batch and heads at most 65535");
  Q6MOE_REQUIRE(a->rows >= 1 && a->rows < (1 << 24) && a->max_count >= 1 && a->max_count < (1 << 24),
                "tree_attention: rows and max_count must be positive and below 2^24");
  Q6MOE_REQUIRE(tree_holds(a->rows, a->query_heads, a->kv_heads, a->batch, a->max_count),
                "tree_attention: rows x query heads per KV head must be below 2^30");
  Q6MOE_REQUIRE(a->page_size >= 1 && a->pages_per_seq >= 1 && a->pool_pages >= 1 && a->page_size < (1 << 30) &&
                    a->pages_per_seq < (1 << 30) && a->pool_pages < (1ll << 31) &&
                    a->pages_per_seq * a->page_size <= (1 << 30) && a->pool_pages * a->page_size < (1ll << 31),
                "tree_attention: page_size, pages_per_seq and pool_pages must be positive, a sequence's capacity at "
                "most 2^30 and the pool below 2^31 tokens");
  Q6MOE_REQUIRE(a->scale_dtype == Q6MOE_BF16 || a->scale_dtype == Q6MOE_F32, "tree_attention: scale dtype");
  Q6MOE_REQUIRE(!a->masks || (a->mask_words >= 1 && a->mask_words <= 4 && a->max_count <= 64 * a->mask_words),
                "tree_attention: masks hold max_count bits in at most 4 words");
  Q6MOE_REQUIRE(a->q_stride >= 0 && a->q_stride % 8 == 0, "tree_attention: q_stride must be a multiple of 8");
  Q6MOE_REQUIRE(a->workspace, "tree_attention: null pointer (workspace)");
  Q6MOE_REQUIRE(aligned(a->q, 16) && aligned(a->k_codes, 16) && aligned(a->v_codes, 16) && aligned(a->out, 16) &&
                    aligned(a->workspace, 256),
                "tree_attention: q, codes and out need 16-byte and workspace 256-byte alignment");
  const TreeLayout L = tree_layout(a->batch, a->rows, a->max_count, a->query_heads, a->kv_heads, a->head_dim,
                                   a->pages_per_seq * a->page_size);
  Q6MOE_REQUIRE(L.grid < (1ll << 31), "tree_attention: too many rows");
  if (a->workspace_bytes < L.total) {
    set_error("tree_attention: workspace too small (need " + std::to_string(L.total) + " bytes)");
    return Q6MOE_ERR_INVALID;
  }
  TreeParams p;
  p.q = a->q;
  p.q_stride = a->q_stride;
  p.kc = a->k_codes;
  p.vc = a->v_codes;
  p.ks = a->k_scales;
  p.vs = a->v_scales;
  p.scale_bf16 = a->scale_dtype == Q6MOE_BF16;
  p.table = a->page_table;
  p.len = a->lengths;
  p.starts = a->starts;
  p.masks = reinterpret_cast<const uint64_t*>(a->masks);
  p.words = (int)a->mask_words;
  p.batch = (int)a->batch;
  p.rows = (int)a->rows;
  p.max_count = (int)a->max_count;
  p.kvh = (int)a->kv_heads;
  p.hq = (int)a->query_heads;
  p.r = p.hq / p.kvh;
  p.pool_pages = (int)a->pool_pages;
  p.pps = (int)a->pages_per_seq;
  p.page = (int)a->page_size;
  p.cap = (int)(a->pages_per_seq * a->page_size);
  int lg = 0;
  while ((1ll << lg) < a->page_size) ++lg;
  p.page_magic = (uint32_t)(((1ull << (31 + lg)) + a->page_size - 1) / a->page_size);
  p.page_shift = 31 + lg;
  p.slots = L.slots;
  p.whole = L.whole;
  p.grid = (int)L.grid;
  p.parts = (int)L.parts;
  p.to_log2 = 1.4426950408889634f / sqrtf((float)a->head_dim);
  uint8_t* w = reinterpret_cast<uint8_t*>(a->workspace);
  p.info = reinterpret_cast<int32_t*>(w + L.info);
  p.whose = a->batch > kTreeLanes ? reinterpret_cast<int32_t*>(w + L.whose) : nullptr;
  p.stat = reinterpret_cast<float*>(w + L.stat);
  p.part = reinterpret_cast<float*>(w + L.part);
  p.out = a->out;
  hipStream_t s = (hipStream_t)stream;
  return a->head_dim == 64 ? tree_launch<64>(p, L, s)
                           : (a->head_dim == 128 ? tree_launch<128>(p, L, s) : tree_launch<256>(p, L, s));
}
