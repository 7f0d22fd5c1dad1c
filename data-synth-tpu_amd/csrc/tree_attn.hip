// Attention of several new tokens per sequence over the paged INT8 cache: every
// row of a ragged batch (a drafted tree, or a chunk of a prompt) against the
// cached tokens of its sequence and the new tokens that its mask names.
//
//   s = (q . kc) * ks / sqrt(D),   out = sum_t p_t vs_t vc_t / sum_t p_t,
//   p_t = exp(s_t - max s)
//
// with the INT8 codes kc, vc and the FP32 scales ks, vs of (token, KV head).
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

constexpr int kTreeThreads = 256;
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
  float to_log2;   // log2(e) / sqrt(D)
  float* part;     // [workgroup][row of the tile][D] partial sums
  float* stat;     // [workgroup][row of the tile][2]: maximum (log2) and sum
  int32_t* info;   // [batch + 1]: first workgroup of each sequence; at [batch] the keys per workgroup
  uint16_t* out;
};

template <int D, int RW>
struct TreeCfg {
  static constexpr int kRows = 32 * RW;          // (new token, head of the group) rows per workgroup
  static constexpr int kGroups = 4 / RW;         // waves that share rows take different keys
  static constexpr int kTile = RW == 1 ? 32 : 64;  // keys per tile of a group
  static constexpr int kBlocks = kTile / 32;
  static constexpr int kStep = kTile * kGroups;  // keys per turn of the workgroup
  // Stages: two workgroups share a CU's LDS, one of 256-channel heads
  static constexpr int kStages = D > 64 && RW < 4 ? 2 : 3;
  static constexpr int kPerCu = D == 256 ? 1 : 2;  // workgroups per CU
  static constexpr int kHalf = kTile * D;        // bytes of a tile's keys, and of its values
  static constexpr int kDma = kHalf / 1024 / RW;  // DMA instructions per wave for each
  static constexpr int kChunks = D / 16;         // 16-byte chunks of a key
  static constexpr int kRing = kGroups * kStages * 2 * kHalf;
  static constexpr int kScale = 2 * 64 * 4 + 16;  // per wave and stage: key and value scales, value factor
  static constexpr int kLds = kRing + 4 * kStages * kScale + 32;  // and four words of masks
  static_assert(kHalf % (1024 * RW) == 0 && kPerCu * kLds <= 160 * 1024, "tile");
};

template <int N>
__device__ __forceinline__ void tree_wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
  asm volatile("" ::: "memory");
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

struct TreeItem {
  int b, tile, kh, chunk, keys;
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
  v = f(v, __shfl_xor(v, 16));
  return f(v, __shfl_xor(v, 32));
}

// The workgroup's item, found by each wave for itself (lane t takes the sequences
// t, t + 64, ..). The call's work, sum over sequences of tiles x heads x keys, is
// cut into chunks of at most ``keys`` keys: the least number that gives no more
// chunks than the chip holds workgroups, so that all run at once and, whatever the
// lengths, end together. Only the GPU knows the lengths. (Cut at the mean instead,
// 64-token trees made 640 chunks for 512 places: 321 us against 236.) Where the
// tiles themselves fill half of the places or more, the chunks are half as long as
// the mean share and run in turns.
template <int ROWS, int STEP>
__device__ __forceinline__ bool tree_item(const TreeParams& p, TreeItem& it) {
  const int lane = threadIdx.x & 63;
  const TreeSeq none{0, 0, 0, 0}, mine = lane < p.batch ? tree_seq(p, lane) : none;
  const auto units = [&](const TreeSeq& s) { return tree_tiles(p, s, ROWS) * p.kvh; };
  const auto sum = [&](auto zero, auto of) {
    auto v = lane < p.batch ? of(mine) : zero;
    for (int b = lane + 64; b < p.batch; b += 64) v += of(tree_seq(p, b));
    return tree_wave_reduce(v, [](auto x, auto y) { return x + y; });
  };
  int keys = 1 << 30;
  if (!p.whole) {
    const float total = sum(0.f, [&](const TreeSeq& s) { return (float)units(s) * (float)s.n; });
    const int tiles = sum(0, units);
    const bool once = 2 * tiles <= p.slots;
    int lo = (int)(total / (float)(once ? p.slots : 2 * p.slots) * (1.f / STEP));
    lo = lo < 1 ? 1 : (lo < (1 << 30) / STEP / 2 - 1 ? lo : (1 << 30) / STEP / 2 - 1);
    int hi = once ? 2 * lo + 2 : lo + 1;  // in steps; hi gives few enough chunks
    if (once && p.batch <= 256)
      for (int i = 0; i < 5 && lo < hi; ++i) {
        const int mid = (lo + hi) >> 1;
        const int n = sum(0, [&](const TreeSeq& s) { return units(s) * tree_chunks(s.n, mid * STEP); });
        if (n <= p.slots)
          hi = mid;
        else
          lo = mid + 1;
      }
    keys = hi * STEP;
  }
  const int id = blockIdx.x;
  int base = 0;
  it.b = -1;
  it.keys = keys;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {  // 64 sequences at a time
    const TreeSeq s = b0 == 0 ? mine : (b0 + lane < p.batch ? tree_seq(p, b0 + lane) : none);
    const int n = units(s) * tree_chunks(s.n, keys);
    int upto = n;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(upto, off);
      if (lane >= off) upto += v;
    }
    upto += base;
    const uint64_t has = __ballot(id < upto);
    if (has) {
      const int at = __builtin_ctzll(has);
      it.b = b0 + at;
      it.seq.start = __builtin_amdgcn_readlane(s.start, at);
      it.seq.count = __builtin_amdgcn_readlane(s.count, at);
      it.seq.len = __builtin_amdgcn_readlane(s.len, at);
      it.seq.n = __builtin_amdgcn_readlane(s.n, at);
      const int first = __builtin_amdgcn_readlane(upto - n, at), in = id - first;
      const int tiles = tree_tiles(p, it.seq, ROWS), row = in / tiles;
      it.tile = in - row * tiles;
      it.chunk = row / p.kvh;
      it.kh = row - it.chunk * p.kvh;
      if (threadIdx.x == 0 && in == 0) p.info[it.b] = first;
      break;
    }
    base = __builtin_amdgcn_readlane(upto, 63);
  }
  if (threadIdx.x == 0 && id == 0) p.info[p.batch] = keys;
  return it.b >= 0;
}

// A tile's rows in LDS: key t lies in row tree_row(t), bits 0 and 2 of t exchanged,
// so that the two half waves, which read the values of keys 4 apart, meet
// different halves of the banks. Chunk c of a row's key lies in slot c ^
// tree_swizzle(row), so that the 16 lanes that read one column of 16 keys meet 16
// different bank groups; values, read by rows, lie as they are.
__device__ __forceinline__ int tree_row(int key) { return (key & ~5) | (key & 1) << 2 | (key >> 2 & 1); }
template <int CH>
__device__ __forceinline__ int tree_swizzle(int row) {
  return (row / (16 / CH)) & (CH - 1);
}

// The channel of accumulator element v (of channel block c), for a lane of half
// wave h: each lane's loads of D / 32 consecutive channels of a key serve all
// blocks (for D = 64, of 4 channels, of which the upper 16 rows take the last two).
template <int D>
__device__ __forceinline__ int tree_channel(int c, int v, int h) {
  const int i = 8 * (v >> 2) + 4 * h + (v & 3);
  return D == 64 ? 4 * (i & 15) + 2 * (i >> 4) + c : D / 32 * i + c;
}

template <int D, int RW>
__global__ void __launch_bounds__(kTreeThreads, D == 256 ? 1 : 2) tree_attn_kernel(TreeParams p) {
  using C = TreeCfg<D, RW>;
  constexpr int KS = D / 32;  // channel blocks of 32
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  TreeItem it;
  if (!tree_item<C::kRows, C::kStep>(p, it)) return;  // uniform over the workgroup
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = wave / RW, rw = wave % RW;
  const int col = lane & 31, h = lane >> 5;
  const TreeSeq seq = it.seq;
  int n, n_all;
  tree_reach(p, seq, it.tile, C::kRows, &n, &n_all);
  const int c0 = it.chunk * it.keys;
  if (c0 > 0 && c0 >= n) return;
  const int c1 = n - c0 < it.keys ? n : c0 + it.keys;
  const bool split = tree_chunks(n, it.keys) > 1;

  // New tokens that some row of the sequence sees. What the cache holds at the
  // others' places (they may never have been written) is not read.
  uint64_t* wanted = reinterpret_cast<uint64_t*>(smem + C::kRing + 4 * C::kStages * C::kScale);
  const bool pick = p.masks && c1 > seq.len;
  if (pick) {
    if (wave == 0)
      for (int w = 0; w < p.words; ++w) {
        uint64_t some = 0;
        for (int i = lane; i < seq.count; i += 64) some |= p.masks[(int64_t)(seq.start + i) * p.words + w];
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) some |= __shfl_xor((unsigned long long)some, off);
        if (lane == 0) wanted[w] = some;
      }
    __syncthreads();
  }

  // ---- the stream of key and value tiles --------------------------------
  uint8_t* ring = smem + group * (C::kStages * 2 * C::kHalf);
  float* scales = reinterpret_cast<float*>(smem + C::kRing + wave * (C::kStages * C::kScale));
  const int turns = (c1 - c0 + C::kStep - 1) / C::kStep;
  const int64_t row_bytes = (int64_t)p.kvh * D;
  const int8_t* kbase = p.kc + (int64_t)it.kh * D;
  const int8_t* vbase = p.vc + (int64_t)it.kh * D;
  const int32_t* trow = p.table + (int64_t)it.b * p.pps;
  const int last = c1 > c0 ? c1 - 1 : 0;
  const int tkey = lane & (C::kTile - 1);  // the key of a tile that this lane looks up
  auto tile_at = [&](int i) { return c0 + (group + C::kGroups * i) * C::kTile; };
  auto page_of = [&](int t) { return (int)((uint64_t)(uint32_t)t * p.page_magic >> p.page_shift); };
  auto entry = [&](int i) {  // page-table entry of the lane's key in turn i's tile
    const int t = tile_at(i) + tkey;
    return trow[page_of(t < c1 ? t : last)];
  };
  int pg = entry(0);
  uint32_t rk = 0, rv = 0;  // scales on their way, as they lie in the cache
  bool ron = false;         // and whether there are any
  auto scale_bits = [&](const void* s, int64_t i) {
    return p.scale_bf16 ? (uint32_t)reinterpret_cast<const uint16_t*>(s)[i] : reinterpret_cast<const uint32_t*>(s)[i];
  };
  auto issue = [&](int i, int stage) {
    const int t0 = tile_at(i), t = t0 + tkey;
    ron = t < c1 && pg >= 0 && pg < p.pool_pages;
    if (pick && t0 + C::kTile > seq.len) {  // uniform over the wave
      const int jj = t - seq.len;
      if (t < c1 && jj >= 0) ron = ron && (wanted[jj >> 6] >> (jj & 63) & 1);
    }
    const int tc = t < c1 ? t : last;
    const int r = ron ? pg * p.page + (tc - page_of(tc) * p.page) : 0;
    pg = entry(i + 1);
    const int64_t at = (int64_t)r * p.kvh + it.kh;
    if (C::kTile == 32) {  // lanes 0-31 load key scales, the others value scales
      rk = scale_bits(h ? p.vs : p.ks, at);
    } else {
      rk = scale_bits(p.ks, at);
      rv = scale_bits(p.vs, at);
    }
    uint8_t* st = ring + stage * 2 * C::kHalf;
#pragma unroll
    for (int d = 0; d < C::kDma; ++d) {
      const int first = (rw * C::kDma + d) * 64;  // first 16-byte slot
      const int line = (first + lane) / C::kChunks, slot = (first + lane) % C::kChunks;
      const int64_t off = (int64_t)__shfl(r, tree_row(line)) * row_bytes;
      const int8_t* k = kbase + off + 16 * (slot ^ tree_swizzle<C::kChunks>(line));
      const int8_t* v = vbase + off + 16 * slot;
      __builtin_amdgcn_global_load_lds(k, LDS_PTR(st + first * 16), 16, 0, 0);
      __builtin_amdgcn_global_load_lds(v, LDS_PTR(st + C::kHalf + first * 16), 16, 0, 0);
    }
  };
  issue(0, 0);

  // The lane's row of the tile: query (new token j, head hh of the group), held
  // as 16-bit integers in two INT8 operands q = (256 hi + lo) 2^(e-14), e the
  // exponent of the row's largest value: exact for values down to 2^-6 of it.
  const int row = it.tile * C::kRows + rw * 32 + col;
  const bool live = row < seq.count * p.r;
  const int j = live ? row / p.r : 0, hh = live ? row - j * p.r : 0;
  i32x4 qhi[KS], qlo[KS];
  float qf;
  {
    const uint16_t* src = p.q + (int64_t)(seq.start + j) * p.q_stride + (int64_t)(it.kh * p.r + hh) * D + 16 * h;
    uint32_t top = 0;  // the largest magnitude's bits
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const u32x4 x = live ? *reinterpret_cast<const u32x4*>(src + 32 * s + 8 * e) : u32x4{0u, 0u, 0u, 0u};
        i32x4& keep = e ? qlo[s] : qhi[s];
        keep = __builtin_bit_cast(i32x4, x);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t a = x[w] & 0x7fffu, b = (x[w] >> 16) & 0x7fffu;
          top = top > a ? top : a;
          top = top > b ? top : b;
        }
      }
    const uint32_t other = __shfl_xor(top, 32);
    top = top > other ? top : other;
    int e = (int)(top >> 7) - 127 + ((top & 0x7f) == 0x7f);  // the largest stays below 127 * 256 + 128
    e = e < -110 ? -110 : e;  // smaller queries lose bits: scores below 2^-90
    // v = q 2^(14-e) rounded into the low bits of 1.5 * 2^23 + v; its low byte is lo,
    // the second byte of v + 128 is hi
    const float up = __builtin_ldexpf(1.f, 14 - e);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const i32x4 raw[2] = {qhi[s], qlo[s]};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t x = (uint32_t)raw[w >> 1][(2 * w + (i >> 1)) & 3];
          const float f = __builtin_bit_cast(float, i & 1 ? x & 0xffff0000u : x << 16);
          v[i] = __builtin_bit_cast(uint32_t, __builtin_fmaf(f, up, 12582912.f));
        }
        const uint32_t l01 = __builtin_amdgcn_perm(v[1], v[0], 0x0c0c0400u);
        const uint32_t l23 = __builtin_amdgcn_perm(v[3], v[2], 0x04000c0cu);
        const uint32_t h01 = __builtin_amdgcn_perm(v[1] + 128, v[0] + 128, 0x0c0c0501u);
        const uint32_t h23 = __builtin_amdgcn_perm(v[3] + 128, v[2] + 128, 0x05010c0cu);
        qhi[s][w] = (int)(h01 | h23);
        qlo[s][w] = (int)(l01 | l23);
      }
    }
    qf = __builtin_ldexpf(p.to_log2, e - 14);
    if (top >= 0x7f80u) qf = __builtin_nanf("");  // an infinite or NaN query: NaN scores
  }

  f32x16 acc[KS];
#pragma unroll
  for (int c = 0; c < KS; ++c)
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[c][v] = 0.f;
  float m = kTreeFloor, l = 0.f, psum = 0.f;
  float vfac = 1.f, vfac_new = 1.f, vtop = -1.f;  // value factor in use, of the newest tile, and its limit

  // Scales of the tile issued a turn ago into the wave's LDS. The value scales are
  // brought to at most 2^6 by a power of two that falls as larger ones are met, so
  // that probability x scale keeps its 11 bits in FP16.
  auto put_scales = [&](int stage) {
    float* sc = scales + stage * (C::kScale / 4);
    auto value = [&](uint32_t bits) {
      return ron ? __builtin_bit_cast(float, p.scale_bf16 ? bits << 16 : bits) : 0.f;
    };
    const float k = value(rk), v = C::kTile == 32 ? k : value(rv);
    const float a = (C::kTile == 64 || h) && fabsf(v) < __builtin_inff() ? fabsf(v) : 0.f;
    if (__any(a > vtop)) {
      float x = a;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) x = fmaxf(x, __shfl_xor(x, off));
      int e = (int)(__builtin_bit_cast(uint32_t, x) >> 23) - 127;
      e = e < -110 ? -110 : e;
      vfac_new = __builtin_bit_cast(float, (uint32_t)(127 + 3 - e) << 23);  // 2^(3-e): at most 2^4 now
      vtop = __builtin_bit_cast(float, (uint32_t)(127 + e + 3 > 254 ? 254 : 127 + e + 3) << 23);
    }
    if (C::kTile == 32) {
      sc[lane] = h ? v * vfac_new : k;
    } else {
      sc[lane] = k;
      sc[64 + lane] = v * vfac_new;
    }
    if (lane == 0) sc[128] = vfac_new;
  };

  const int krow = tree_row(col);
  const uint32_t koff = krow * D, ksw = tree_swizzle<C::kChunks>(krow);
  const uint32_t voff = h * D + (D == 64 ? 4 * (col & 15) : D / 32 * col);
  const uint32_t vsel = D == 64 ? (uint32_t)(col >> 4) * 0x00020002u : 0u;  // the lane's channels of its 4
  auto compute = [&](auto slow, int t0, int stage) {
    const uint8_t* kt = ring + stage * 2 * C::kHalf;
    const uint8_t* vt = kt + C::kHalf + voff;
    const float* sc = scales + stage * (C::kScale / 4) + 4 * h;
    float t[C::kBlocks][16];
    float top = -__builtin_inff();
    uint32_t vis[C::kBlocks];
#pragma unroll
    for (int nb = 0; nb < C::kBlocks; ++nb) {
      i32x16 hi, lo;
#pragma unroll
      for (int v = 0; v < 16; ++v) hi[v] = lo[v] = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const i32x4 a = *reinterpret_cast<const i32x4*>(kt + 32 * nb * D + koff + 16 * ((2 * s + h) ^ ksw));
        hi = __builtin_amdgcn_mfma_i32_32x32x32_i8(a, qhi[s], hi, 0, 0, 0);
        lo = __builtin_amdgcn_mfma_i32_32x32x32_i8(a, qlo[s], lo, 0, 0, 0);
      }
      if constexpr (slow) {
        // bit i: the lane's row sees key t0 + 32 nb + i; then moved to the half wave's keys
        const int k0 = t0 + 32 * nb, jj = k0 - seq.len;
        uint32_t on = 0;
        if (p.masks) {
          const uint64_t* w = p.masks + (int64_t)(seq.start + j) * p.words;
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
        vis[nb] = live ? on >> (4 * h) : 0u;
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 ksv = *reinterpret_cast<const f32x4*>(sc + 32 * nb + 8 * g);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int v = 4 * g + u;
          t[nb][v] = (float)((hi[v] << 8) + lo[v]) * ksv[u];
          if constexpr (slow) t[nb][v] = vis[nb] >> (8 * g + u) & 1 ? t[nb][v] : -__builtin_inff();
          top = fmaxf(top, t[nb][v]);
        }
      }
    }
    top *= qf;
    const float vf = __builtin_bit_cast(
        float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, sc[128 - 4 * h])));
    if (__any(top > m + kTreeSlack) || vf != vfac) {  // uniform over the wave
      const float to = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)));
      const float fade_l = __builtin_amdgcn_exp2f(m - to), fade = fade_l * (vf / vfac);
      vfac = vf;
      m = to;
      l *= fade_l;
      psum *= fade;
#pragma unroll
      for (int c = 0; c < KS; ++c)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[c][v] *= fade;
    }
#pragma unroll
    for (int nb = 0; nb < C::kBlocks; ++nb)
#pragma unroll
      for (int mm = 0; mm < 2; ++mm) {  // 16 keys: 8 of each half wave
        f16x8 pv;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const f32x4 vsv = *reinterpret_cast<const f32x4*>(sc + (C::kTile == 32 ? 32 : 64) + 32 * nb + 16 * mm + 8 * g);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int v = 8 * mm + 4 * g + u;
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(t[nb][v], qf, -m));
            float w = e * vsv[u];
            if constexpr (slow) {
              const bool on = vis[nb] >> (16 * mm + 8 * g + u) & 1;
              l += on ? e : 0.f;
              w = on ? w : 0.f;
            } else {
              l += e;
            }
            pv[4 * g + u] = (_Float16)w;
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const f16x2 one = {(_Float16)1.f, (_Float16)1.f}, pair = {pv[2 * u], pv[2 * u + 1]};
          psum = __builtin_amdgcn_fdot2(pair, one, psum, false);
        }
        // Values: the lane's channels of its half wave's 8 keys; byte b of two keys
        // makes one operand word. Code + 128 enters as an FP16 subnormal, (code + 128)
        // 2^-24: the 128 is taken back at the end with the sum of the rounded
        // probabilities.
        constexpr int W = D == 256 ? 2 : 1;
        uint32_t x[8][W];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint8_t* src = vt + (32 * nb + 16 * mm + tree_row(8 * (i >> 2) + (i & 3))) * D;
          if constexpr (W == 2) {
            const u32x2 y = *reinterpret_cast<const u32x2*>(src);
            x[i][0] = y[0] ^ 0x80808080u;
            x[i][1] = y[1] ^ 0x80808080u;
          } else {
            x[i][0] = *reinterpret_cast<const uint32_t*>(src) ^ 0x80808080u;
          }
        }
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

  // Turn i issues the tile of turn i + kStages - 1; its scales reach LDS a turn
  // later. Waits count DMA instructions: those of the tiles after this one may
  // still be in flight.
#pragma unroll
  for (int i = 1; i < C::kStages - 1; ++i) {
    put_scales(i - 1);
    issue(i, i);
  }
  int stage = 0;
  auto advance = [&](int i) {
    tree_wait_vm<(C::kStages - 2) * 2 * C::kDma>();
    // the wave's reads of the stage that is written next have returned
    if (RW > 1)
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const int next = stage == 0 ? C::kStages - 1 : stage - 1;
    put_scales(C::kStages == 2 ? stage : (stage + 1 == C::kStages ? 0 : stage + 1));
    issue(i + C::kStages - 1, next);
  };
  // first the turns whose tile every row sees whole
  const int open = (n_all < c1 ? n_all : c1) - tile_at(0);
  int fast = open / C::kTile > 0 ? (open / C::kTile - 1) / C::kGroups + 1 : 0;
  fast = fast < turns ? fast : turns;
  int i = 0;
  for (; i < fast; ++i) {
    advance(i);
    compute(std::false_type{}, 0, stage);
    stage = stage + 1 == C::kStages ? 0 : stage + 1;
  }
  for (; i < turns; ++i) {
    advance(i);
    compute(std::true_type{}, tile_at(i), stage);
    stage = stage + 1 == C::kStages ? 0 : stage + 1;
  }
  tree_wait_vm<0>();

  // ---- the row's result -------------------------------------------------
  // Both half waves hold half of a row's keys in l and psum.
  l += __shfl_xor(l, 32);
  psum += __shfl_xor(psum, 32);
  const float up = 0x1p24f / vfac, shift = 128.f * psum * 0x1p-24f;
#pragma unroll
  for (int c = 0; c < KS; ++c)
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[c][v] = (acc[c][v] - shift) * up;
  // Channels q * kRun + [0, kRun) of a lane's sums lie together.
  constexpr int kRun = D == 64 ? 4 : KS, kRuns = KS * 16 / kRun;
  auto at_run = [&](int q) { return tree_channel<D>(0, q, h); };
  auto of_run = [&](int q, int u) { return D == 64 ? acc[u & 1][q + 8 * (u >> 1)] : acc[D == 64 ? 0 : u][q]; };
  auto set_run = [&](int q, int u, float v) {
    if constexpr (D == 64)
      acc[u & 1][q + 8 * (u >> 1)] = v;
    else
      acc[u][q] = v;
  };
  if constexpr (C::kGroups > 1) {
    // the groups' sums meet in LDS, in group order
    __syncthreads();
    float* st = reinterpret_cast<float*>(smem);   // [group][row]: maximum, sum
    float* sum = st + 2 * C::kGroups * C::kRows;  // [row][D], one group at a time
    const int rr = rw * 32 + col;
    if (h == 0) {
      st[2 * (group * C::kRows + rr)] = m;
      st[2 * (group * C::kRows + rr) + 1] = l;
    }
    __syncthreads();
    float to = kTreeFloor, all = 0.f;
#pragma unroll
    for (int g = 0; g < C::kGroups; ++g) to = fmaxf(to, st[2 * (g * C::kRows + rr)]);
#pragma unroll
    for (int g = 0; g < C::kGroups; ++g)
      all += st[2 * (g * C::kRows + rr) + 1] * __builtin_amdgcn_exp2f(st[2 * (g * C::kRows + rr)] - to);
    const float fade = __builtin_amdgcn_exp2f(m - to);
#pragma unroll
    for (int c = 0; c < KS; ++c)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[c][v] *= fade;
    for (int g = C::kGroups - 1; g >= 0; --g) {
      if (group == g) {
#pragma unroll
        for (int q = 0; q < kRuns; ++q)
#pragma unroll
          for (int u = 0; u < kRun; u += 4) {
            f32x4* at = reinterpret_cast<f32x4*>(sum + rr * (D + 4) + at_run(q) + u);
            f32x4 v = {of_run(q, u), of_run(q, u + 1), of_run(q, u + 2), of_run(q, u + 3)};
            if (g < C::kGroups - 1) v += *at;
            *at = v;
          }
      }
      __syncthreads();
    }
    if (group > 0) return;
#pragma unroll
    for (int q = 0; q < kRuns; ++q)
#pragma unroll
      for (int u = 0; u < kRun; u += 4) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(sum + rr * (D + 4) + at_run(q) + u);
#pragma unroll
        for (int w = 0; w < 4; ++w) set_run(q, u + w, v[w]);
      }
    m = to;
    l = all;
  }
  if (!live) return;
  if (split) {
    const int64_t at = (int64_t)blockIdx.x * C::kRows + rw * 32 + col;
    float* dst = p.part + at * D;
#pragma unroll
    for (int q = 0; q < kRuns; ++q)
#pragma unroll
      for (int u = 0; u < kRun; u += 4)
        *reinterpret_cast<f32x4*>(dst + at_run(q) + u) =
            f32x4{of_run(q, u), of_run(q, u + 1), of_run(q, u + 2), of_run(q, u + 3)};
    if (h == 0) *reinterpret_cast<f32x2*>(p.stat + 2 * at) = f32x2{m, l};
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* dst = p.out + ((int64_t)(seq.start + j) * p.hq + it.kh * p.r + hh) * D;
#pragma unroll
  for (int q = 0; q < kRuns; ++q)
#pragma unroll
    for (int u = 0; u < kRun; u += 4)
      *reinterpret_cast<u32x2*>(dst + at_run(q) + u) =
          u32x2{pack_bf16x2(of_run(q, u) * inv, of_run(q, u + 1) * inv),
                pack_bf16x2(of_run(q, u + 2) * inv, of_run(q, u + 3) * inv)};
}

// The chunks' sums of a row and head joined in chunk order, D / 4 lanes of four
// channels each. Eight chunks' sums are loaded at a time; lane i of the head holds
// the weight of chunk i.
template <int D>
__global__ void __launch_bounds__(kTreeThreads) tree_combine_kernel(TreeParams p, int tile_rows) {
  constexpr int W = D / 4;  // lanes per head
  const int row = blockIdx.x, lane = threadIdx.x & 63;
  const int at = (blockIdx.y * kTreeThreads + threadIdx.x) * 4;  // within the row's heads
  int b = 0;  // the sequences that end before the row
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const uint64_t before = __ballot(b0 + lane < p.batch && p.starts[b0 + lane + 1] <= row);
    b += __popcll(before);
    if (!(before >> 63)) break;
  }
  if (b >= p.batch) return;
  const TreeSeq s = tree_seq(p, b);
  const int keys = p.info[p.batch], from = p.info[b];
  const int j = row - s.start;
  if (j < 0 || j >= s.count || at >= p.hq * D) return;  // whole heads
  const int head = at / D, c = at - head * D, kh = head / p.r, rr = j * p.r + head - kh * p.r;
  const int tile = rr / tile_rows, tiles = tree_tiles(p, s, tile_rows);
  int n, n_all;
  tree_reach(p, s, tile, tile_rows, &n, &n_all);
  const int chunks = tree_chunks(n, keys);
  if (chunks == 1) return;
  const int64_t first = ((int64_t)from + (int64_t)kh * tiles + tile) * tile_rows + rr - tile * tile_rows;
  const int64_t step = (int64_t)p.kvh * tiles * tile_rows;
  const int in = lane & (W - 1);
  float m = kTreeFloor, l = 0.f;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < chunks; i0 += W) {
    const bool on = i0 + in < chunks;
    const f32x2 st = on ? *reinterpret_cast<const f32x2*>(p.stat + 2 * (first + (i0 + in) * step)) : f32x2{kTreeFloor, 0.f};
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
    const int end = chunks - i0 < W ? chunks - i0 : W;
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
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<u32x2*>(p.out + (int64_t)row * p.hq * D + at) =
      u32x2{pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv)};
}

constexpr int kTreeCus = 256;

struct TreeLayout {
  int row_waves;  // waves of a workgroup with rows of their own
  int slots, whole;
  int64_t grid;   // at most so many workgroups have work
  size_t info, stat, part, total;
};

static size_t tree_align(size_t v) { return (v + 255) & ~(size_t)255; }

static TreeLayout tree_layout(int64_t batch, int64_t rows, int64_t max_count, int64_t hq, int64_t kvh, int64_t dim) {
  TreeLayout L;
  const int64_t r = hq / kvh;
  L.row_waves = max_count * r <= 32 ? 1 : (max_count * r <= 64 ? 2 : 4);
  const int64_t tile = 32 * L.row_waves;
  // row tiles of all sequences together: each ends with one that is not full
  const int64_t by_batch = batch * cdiv(max_count * r, tile), by_rows = rows * r / tile + batch;
  const int64_t units = kvh * (by_batch < by_rows ? by_batch : by_rows);
  L.slots = kTreeCus * (dim == 256 ? TreeCfg<256, 1>::kPerCu : TreeCfg<128, 1>::kPerCu);
  L.whole = units >= 4 * L.slots;
  L.grid = L.whole ? units : (2 * units <= L.slots ? L.slots : units + 2 * L.slots);
  const int64_t parts = L.whole ? 0 : L.grid * tile;
  L.info = 0;
  L.stat = tree_align(L.info + (size_t)(batch + 1) * 4);
  L.part = tree_align(L.stat + (size_t)parts * 8);
  L.total = tree_align(L.part + (size_t)parts * dim * 4);
  return L;
}

template <int D, int RW>
static int tree_launch(const TreeParams& p, const TreeLayout& L, hipStream_t s) {
  using C = TreeCfg<D, RW>;
  static std::atomic<uint64_t> done{0};
  once_per_device(done, [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&tree_attn_kernel<D, RW>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, C::kLds);
  });
  hipLaunchKernelGGL((tree_attn_kernel<D, RW>), dim3((unsigned)L.grid), dim3(kTreeThreads), C::kLds, s, p);
  if (!L.whole)
    hipLaunchKernelGGL(tree_combine_kernel<D>, dim3((unsigned)p.rows, (unsigned)cdiv(p.hq * D, 4 * kTreeThreads)),
                       dim3(kTreeThreads), 0, s, p, C::kRows);
  return check_launch("tree_attention");
}

template <int D>
static int tree_launch(const TreeParams& p, const TreeLayout& L, hipStream_t s) {
  return L.row_waves == 1 ? tree_launch<D, 1>(p, L, s)
                          : (L.row_waves == 2 ? tree_launch<D, 2>(p, L, s) : tree_launch<D, 4>(p, L, s));
}

}  // namespace q6moe

using namespace q6moe;

extern "C" size_t q6moe_tree_attn_workspace_size(int64_t batch, int64_t rows, int64_t max_count, int64_t query_heads,
                                                 int64_t kv_heads, int64_t head_dim, int64_t pages_per_seq,
                                                 int64_t page_size) {
  if (batch < 1 || rows < 1 || max_count < 1 || query_heads < 1 || kv_heads < 1 || pages_per_seq < 1 || page_size < 1)
    return 0;
  if (query_heads % kv_heads || batch > 65535 || rows >= (1 << 24) || max_count >= (1 << 24)) return 0;
  return tree_layout(batch, rows, max_count, query_heads, kv_heads, head_dim).total;
}

extern "C" int q6moe_kv_tree_attention(const q6moe_tree_attn_args* a, void* stream) {
  Q6MOE_REQUIRE(a, "tree_attention: null args");
  Q6MOE_REQUIRE(a->q && a->k_codes && a->v_codes && a->k_scales && a->v_scales && a->page_table && a->lengths &&
                    a->starts && a->out && a->workspace,
                "tree_attention: null pointer");
  Q6MOE_REQUIRE(a->head_dim == 64 || a->head_dim == 128 || a->head_dim == 256,
                "tree_attention: head_dim must be 64, 128 or 256");
  Q6MOE_REQUIRE(a->batch >= 1 && a->batch <= 65535 && a->kv_heads >= 1 && a->kv_heads <= kTreeMaxHeads &&
                    a->query_heads >= 1 && a->query_heads <= kTreeMaxHeads && a->query_heads % a->kv_heads == 0,
                "tree_attention: query_heads must be a multiple of kv_heads, batch and heads at most 65535");
  Q6MOE_REQUIRE(a->rows >= 1 && a->rows < (1 << 24) && a->max_count >= 1 && a->max_count < (1 << 24),
                "tree_attention: rows and max_count must be positive and below 2^24");
  Q6MOE_REQUIRE(a->page_size >= 1 && a->pages_per_seq >= 1 && a->pool_pages >= 1 && a->page_size < (1 << 30) &&
                    a->pages_per_seq < (1 << 30) && a->pool_pages < (1ll << 31) &&
                    a->pages_per_seq * a->page_size <= (1 << 30) && a->pool_pages * a->page_size < (1ll << 31),
                "tree_attention: page_size, pages_per_seq and pool_pages must be positive, a sequence's capacity at "
                "most 2^30 and the pool below 2^31 tokens");
  Q6MOE_REQUIRE(a->scale_dtype == Q6MOE_BF16 || a->scale_dtype == Q6MOE_F32, "tree_attention: scale dtype");
  Q6MOE_REQUIRE(!a->masks || (a->mask_words >= 1 && a->mask_words <= 4 && a->max_count <= 64 * a->mask_words),
                "tree_attention: masks hold max_count bits in at most 4 words");
  Q6MOE_REQUIRE(a->q_stride >= 0 && a->q_stride % 8 == 0, "tree_attention: q_stride must be a multiple of 8");
  Q6MOE_REQUIRE(aligned(a->q, 16) && aligned(a->k_codes, 16) && aligned(a->v_codes, 16) && aligned(a->out, 16) &&
                    aligned(a->workspace, 256),
                "tree_attention: q, codes and out need 16-byte and workspace 256-byte alignment");
  const TreeLayout L =
      tree_layout(a->batch, a->rows, a->max_count, a->query_heads, a->kv_heads, a->head_dim);
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
  p.to_log2 = 1.4426950408889634f / sqrtf((float)a->head_dim);
  uint8_t* w = reinterpret_cast<uint8_t*>(a->workspace);
  p.info = reinterpret_cast<int32_t*>(w + L.info);
  p.stat = reinterpret_cast<float*>(w + L.stat);
  p.part = reinterpret_cast<float*>(w + L.part);
  p.out = a->out;
  hipStream_t s = (hipStream_t)stream;
  return a->head_dim == 64 ? tree_launch<64>(p, L, s)
                           : (a->head_dim == 128 ? tree_launch<128>(p, L, s) : tree_launch<256>(p, L, s));
}
