// The bookkeeping of a step that takes several new tokens per sequence over the
// paged KV cache: pages and slots for the new tokens (q6moe_kv_plan), pages
// given back (q6moe_kv_release), accepted tokens moved together (q6moe_kv_keep).
// No counterpart in the reference, whose cache is dense and whose steps take one
// token per sequence.
//
// A sequence b holds lengths[b] cached tokens; its new token j lies at position
// lengths[b] + j, row starts[b] + j of the ragged batch, starts the running sum of
// the counts. The free pages are a stack, taken from and given back at its end in
// the order of (sequence, page index), so all results are deterministic.
//
// Latency-bound: a few kilobytes for a decode step. A step's calls are one launch of
// one workgroup each (a plan and its release of 8 sequences with 16-token trees: 5
// launches 20 us of kernels, 2 launches 11 us); larger ones take two or three, in
// which every workgroup forms the sums over earlier sequences for itself, from one
// load per 256 of them, instead of waiting for a launch more.
#include "q6moe_api.h"
#include "q6moe_device.h"

namespace q6moe {

constexpr int kStepThreads = 256;
constexpr int kStepWaves = kStepThreads / 64;
constexpr int kMaxTree = 256;  // new tokens per sequence that masks tell apart
constexpr int64_t kStepMaxBatch = 65535;

// Sum of v over the workgroup, known to every thread.
__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* lds) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off);
  __syncthreads();  // lds may still be read
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  int64_t s = 0;
#pragma unroll
  for (int w = 0; w < kStepWaves; ++w) s += lds[w];
  return s;
}

// Number of flagged threads before this one in the workgroup; *total: all of them.
__device__ __forceinline__ int block_rank(bool flag, int64_t* lds, int* total) {
  const uint64_t m = __ballot(flag);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = __popcll(m);
  __syncthreads();
  int before = __popcll(m & ((1ull << (threadIdx.x & 63)) - 1)), all = 0;
#pragma unroll
  for (int w = 0; w < kStepWaves; ++w) {
    if (w < (int)(threadIdx.x >> 6)) before += (int)lds[w];
    all += (int)lds[w];
  }
  *total = all;
  return before;
}

struct PlanParams {
  int32_t* table;
  const int32_t* lengths;
  const int32_t* counts;
  const int32_t* free_pages;
  int64_t free_capacity;
  int32_t* free_count;
  const int32_t* parents;
  int64_t batch, pps, page, rows, max_count;  // max_count: most new tokens per sequence that are placed
  int words;
  int most_lost;  // that a sequence adds to ``missing``: with all rows no more than 2^31 - 1 for all of them
  int32_t* starts;
  int64_t* slots;
  int32_t* positions;
  uint64_t* masks;
  int32_t* missing;
  int32_t* need;  // workspace: pages that sequence b needs; at [batch] the free pages before the call
};

__device__ __forceinline__ int64_t plan_len(const PlanParams& p, int64_t b) {
  const int64_t n = p.lengths[b];
  return n < 0 ? 0 : n;
}
__device__ __forceinline__ int64_t plan_asked(const PlanParams& p, int64_t b) {
  const int64_t c = p.counts[b];
  return c < 0 ? 0 : c;
}
__device__ __forceinline__ int64_t plan_count(const PlanParams& p, int64_t b) {
  const int64_t c = plan_asked(p, b);
  return c < p.max_count ? c : p.max_count;
}
// New tokens of sequence b that have rows, where ``before`` rows belong to earlier ones.
__device__ __forceinline__ int64_t plan_fit(const PlanParams& p, int64_t count, int64_t before) {
  const int64_t left = p.rows - before;
  return left <= 0 ? 0 : (count < left ? count : left);
}
// What a sequence adds to ``missing`` for tokens past max_count and rows.
__device__ __forceinline__ int plan_lost(const PlanParams& p, int64_t lost) {
  return lost < p.most_lost ? (int)lost : p.most_lost;
}
// Page indexes [first, end) that the new tokens of sequence b lie in.
__device__ __forceinline__ void plan_pages(const PlanParams& p, int64_t len, int64_t count, int64_t* first,
                                           int64_t* end) {
  *first = len / p.page;
  const int64_t e = (len + count + p.page - 1) / p.page;
  *end = count == 0 ? *first : (e < p.pps ? e : p.pps);
}
// Rows of the sequences before b.
__device__ __forceinline__ int64_t plan_before(const PlanParams& p, int64_t b, int64_t* lds) {
  int64_t s = 0;
  for (int64_t i = threadIdx.x; i < b; i += kStepThreads) s += plan_count(p, i);
  return block_sum(s, lds);
}

// Pages that each sequence needs: its unmapped entries under the new tokens.
__global__ void __launch_bounds__(kStepThreads) plan_need_kernel(PlanParams p) {
  __shared__ int64_t lds[kStepWaves];
  const int64_t b = blockIdx.x;
  const int64_t before = plan_before(p, b, lds);
  int64_t first, end;
  plan_pages(p, plan_len(p, b), plan_fit(p, plan_count(p, b), before), &first, &end);
  int64_t n = 0;
  for (int64_t e = first + threadIdx.x; e < end; e += kStepThreads) n += p.table[b * p.pps + e] < 0;
  n = block_sum(n, lds);
  if (threadIdx.x == 0) {
    p.need[b] = (int32_t)n;
    if (b == 0) {
      p.missing[0] = 0;
      const int64_t have = p.free_count[0];
      p.need[p.batch] = (int32_t)(have < 0 ? 0 : (have < p.free_capacity ? have : p.free_capacity));
    }
  }
}

// Slot of the token at position t of sequence b, -1 without a page.
__device__ __forceinline__ int64_t plan_slot(const PlanParams& p, int64_t b, int64_t t) {
  if (t >= p.pps * p.page) return -1;  // below 2^31, so that 32-bit divisions serve
  const uint32_t page = (uint32_t)p.page, e = (uint32_t)t / page;
  const int64_t pg = p.table[b * p.pps + e];
  return pg < 0 ? -1 : pg * p.page + ((uint32_t)t - e * page);
}

constexpr int kTakeRows = 4096;  // rows of a sequence that its workgroup writes
__device__ __forceinline__ void plan_behind(const PlanParams& p, int64_t row) {
  p.slots[row] = -1;
  p.positions[row] = 0;
  if (p.masks)
    for (int w = 0; w < p.words; ++w) p.masks[row * p.words + w] = 0;
}

// Takes sequence b's pages from the stack, then (kRows) writes its rows, and the
// last workgroup those behind the last sequence. The rows of a tree, at most
// kMaxTree, lie one per thread: the ancestors by pointer doubling in LDS, each round
// adds those 1, 2, 4, ... levels further up.
template <bool kRows>
__global__ void __launch_bounds__(kStepThreads) plan_take_kernel(PlanParams p) {
  __shared__ int64_t lds[kStepWaves];
  const int64_t b = blockIdx.x;
  int64_t rows = 0, need = 0;
  for (int64_t i = threadIdx.x; i < b; i += kStepThreads) {
    rows += plan_count(p, i);
    need += p.need[i];
  }
  const int64_t before = block_sum(rows, lds);
  int64_t rank = block_sum(need, lds);  // pages that earlier sequences need
  const int64_t have = p.need[p.batch];
  const int64_t len = plan_len(p, b), count = plan_fit(p, plan_count(p, b), before);
  int64_t first, end;
  plan_pages(p, len, count, &first, &end);
  for (int64_t e0 = first; e0 < end; e0 += kStepThreads) {
    const int64_t e = e0 + threadIdx.x;
    const bool want = e < end && p.table[b * p.pps + e] < 0;
    int all;
    const int64_t at = rank + block_rank(want, lds, &all);
    if (want && at < have) p.table[b * p.pps + e] = p.free_pages[have - 1 - at];
    rank += all;
  }
  const int64_t start = before < p.rows ? before : p.rows;
  if (threadIdx.x == 0) {
    p.starts[b] = (int32_t)start;
    if (b == p.batch - 1) {
      p.starts[p.batch] = (int32_t)(start + count);
      p.free_count[0] = (int32_t)(have - (rank < have ? rank : have));
    }
  }
  const int64_t lost = plan_asked(p, b) - count;
  if (threadIdx.x == 0 && lost) atomicAdd(p.missing, plan_lost(p, lost));
  if constexpr (!kRows) return;
  __syncthreads();  // the table entries above
  if (b == p.batch - 1)
    for (int64_t row = start + count + threadIdx.x; row < p.rows; row += kStepThreads) plan_behind(p, row);
  if (!p.parents) {
    int none = 0;
    for (int64_t j = threadIdx.x; j < count; j += kStepThreads) {
      const int64_t slot = plan_slot(p, b, len + j);
      p.slots[start + j] = slot;
      p.positions[start + j] = (int32_t)(len + j);
      none += slot < 0;
    }
    if (none) atomicAdd(p.missing, none);
    return;
  }
  __shared__ uint64_t sees[kMaxTree][kMaxTree / 64];
  __shared__ int up[kMaxTree], depth[kMaxTree];
  const int j = threadIdx.x;
  if (j < count) {
    const int64_t parent = p.parents[start + j];
    up[j] = parent >= 0 && parent < j ? (int)parent : -1;
    depth[j] = up[j] >= 0;
    for (int w = 0; w < p.words; ++w) sees[j][w] = w == j >> 6 ? 1ull << (j & 63) : 0;
  }
  for (int64_t reach = 1; reach < count; reach *= 2) {
    __syncthreads();
    uint64_t more[kMaxTree / 64] = {};
    int to = -1, deeper = 0;
    if (j < count && up[j] >= 0) {
      const int u = up[j];
#pragma unroll
      for (int w = 0; w < kMaxTree / 64; ++w)
        if (w < p.words) more[w] = sees[u][w];
      to = up[u];
      deeper = depth[u];
    }
    __syncthreads();
    if (j < count) {
#pragma unroll
      for (int w = 0; w < kMaxTree / 64; ++w)
        if (w < p.words) sees[j][w] |= more[w];
      depth[j] += deeper;
      up[j] = to;
    }
  }
  if (j < count) {
    const int64_t slot = plan_slot(p, b, len + j), row = start + j;
    p.slots[row] = slot;
    p.positions[row] = (int32_t)(len + depth[j]);
    for (int w = 0; w < p.words; ++w) p.masks[row * p.words + w] = sees[j][w];
    if (slot < 0) atomicAdd(p.missing, 1);
  }
}

// Rows of the ragged batch where a sequence has more of them than one workgroup
// should write: slots and positions, and the rows behind the last sequence. Four rows
// per thread, whose table entries are on their way together.
constexpr int kPlanRows = 4;
__global__ void __launch_bounds__(kStepThreads) plan_rows_kernel(PlanParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t row0 = ((int64_t)blockIdx.x * kStepThreads + (threadIdx.x & ~63)) * kPlanRows;  // of the wave
  const int64_t used = p.starts[p.batch];
  // The last sequence with starts[b] <= row: for the wave's first row by 64 probes at
  // a time, then on from there.
  int b = 0, n = (int)p.batch;  // the sequence is one of b .. b + n - 1
  while (n > 1) {
    const int step = (n + 63) / 64, at = b + lane * step;
    const int below = __popcll(__ballot(lane * step < n && p.starts[at] <= row0));
    const int skip = (below - 1) * step;
    b += skip;
    n = n - skip < step ? n - skip : step;
  }
  int lost = 0;
#pragma unroll
  for (int k = 0; k < kPlanRows; ++k) {
    const int64_t row = row0 + 64 * k + lane;
    if (row >= used) {
      if (row < p.rows) plan_behind(p, row);
      continue;
    }
    while (b + 1 < p.batch && p.starts[b + 1] <= row) ++b;
    const int64_t t = plan_len(p, b) + row - p.starts[b];
    const int64_t slot = plan_slot(p, b, t);
    p.slots[row] = slot;
    p.positions[row] = (int32_t)t;
    lost += slot < 0;
  }
  if (lost) atomicAdd(p.missing, lost);
}

// ---- one workgroup for a step's plan ---------------------------------------
constexpr int kSmallThreads = 1024;
constexpr int kSmallWaves = kSmallThreads / 64;
constexpr int kSmallRows = 4096;     // rows, and words of masks, that one workgroup takes
constexpr int kSmallTreeRows = 2048;
constexpr int kSmallPages = 32;      // pages per sequence that its thread looks through

// Sum of v over the threads before this one; *total: over all of them.
__device__ __forceinline__ int small_before(int v, int* lds, int* total) {
  int upto = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int x = __shfl_up(upto, off);
    if ((int)(threadIdx.x & 63) >= off) upto += x;
  }
  __syncthreads();  // lds may still be read
  if ((threadIdx.x & 63) == 63) lds[threadIdx.x >> 6] = upto;
  __syncthreads();
  int before = upto - v, all = 0;
#pragma unroll
  for (int w = 0; w < kSmallWaves; ++w) {
    if (w < (int)(threadIdx.x >> 6)) before += lds[w];
    all += lds[w];
  }
  *total = all;
  return before;
}

// At most 1024 sequences, one per thread, and few rows: the steps of the three
// kernels above in turn. The trees of all sequences are resolved together.
template <bool kTree>
__global__ void __launch_bounds__(kSmallThreads) plan_small_kernel(PlanParams p) {
  __shared__ int lds[kSmallWaves];
  __shared__ int s_start[kSmallThreads + 1], s_len[kSmallThreads];
  __shared__ uint64_t sees[kTree ? kSmallRows : 1];
  __shared__ int up[kTree ? kSmallTreeRows : 1], depth[kTree ? kSmallTreeRows : 1];
  const int t = threadIdx.x, batch = (int)p.batch, rows = (int)p.rows;
  int64_t len = 0, asked = 0, first = 0, end = 0;
  int count = 0, all, need = 0;
  if (t < batch) {
    len = plan_len(p, t);
    asked = plan_asked(p, t);
    count = (int)(asked < p.max_count ? (asked < rows ? asked : rows) : (p.max_count < rows ? p.max_count : rows));
  }
  const int64_t have0 = p.free_count[0];
  const int have = (int)(have0 < 0 ? 0 : (have0 < p.free_capacity ? have0 : p.free_capacity));
  const int before = small_before(count, lds, &all);
  const int used = all < rows ? all : rows;
  int32_t* table = p.table + t * p.pps;
  if (t < batch) {
    count = (int)plan_fit(p, count, before);
    plan_pages(p, len, count, &first, &end);
    for (int64_t e = first; e < end; ++e) need += table[e] < 0;
    s_start[t] = before < rows ? before : rows;
    s_len[t] = (int)len;
    p.starts[t] = s_start[t];
  }
  if (t == 0) p.starts[batch] = used;
  int taken;
  int rank = small_before(need, lds, &taken);
  if (need)
    for (int64_t e = first; e < end; ++e)
      if (table[e] < 0) {
        if (rank < have) table[e] = p.free_pages[have - 1 - rank];
        ++rank;
      }
  if (t == 0) p.free_count[0] = have - (taken < have ? taken : have);
  int missing = t < batch ? plan_lost(p, asked - count) : 0;
  __syncthreads();  // the entries and sums above
  const auto sequence = [&](int row) {  // the last one with s_start[b] <= row
    int b = 0, hi = batch - 1;
    while (b < hi) {
      const int mid = (b + hi + 1) >> 1;
      if (s_start[mid] <= row)
        b = mid;
      else
        hi = mid - 1;
    }
    return b;
  };
  if constexpr (kTree) {
    const int words = p.words;
    for (int row = t; row < used; row += kSmallThreads) {
      const int b = sequence(row), j = row - s_start[b], parent = p.parents[row];
      up[row] = parent >= 0 && parent < j ? s_start[b] + parent : -1;
      depth[row] = up[row] >= 0;
      for (int w = 0; w < words; ++w) sees[row * words + w] = w == j >> 6 ? 1ull << (j & 63) : 0;
    }
    for (int reach = 1; reach < p.max_count; reach *= 2) {
      uint64_t more[kSmallTreeRows / kSmallThreads][kMaxTree / 64];
      int to[kSmallTreeRows / kSmallThreads], deeper[kSmallTreeRows / kSmallThreads];
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kSmallTreeRows / kSmallThreads; ++k) {
        const int row = t + k * kSmallThreads, u = row < used ? up[row] : -1;
        to[k] = -1;
        deeper[k] = 0;
        if (u >= 0) {
          to[k] = up[u];
          deeper[k] = depth[u];
        }
#pragma unroll
        for (int w = 0; w < kMaxTree / 64; ++w) more[k][w] = u >= 0 && w < words ? sees[u * words + w] : 0;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kSmallTreeRows / kSmallThreads; ++k) {
        const int row = t + k * kSmallThreads;
        if (row >= used) continue;
        up[row] = to[k];
        depth[row] += deeper[k];
#pragma unroll
        for (int w = 0; w < kMaxTree / 64; ++w)
          if (w < words) sees[row * words + w] |= more[k][w];
      }
    }
    __syncthreads();
  }
  for (int row = t; row < rows; row += kSmallThreads) {
    int64_t slot = -1;
    int position = 0;
    if (row < used) {
      const int b = sequence(row), j = row - s_start[b];
      slot = plan_slot(p, b, (int64_t)s_len[b] + j);
      position = (int)((int64_t)s_len[b] + (kTree ? depth[row] : j));
      missing += slot < 0;
    }
    p.slots[row] = slot;
    p.positions[row] = position;
    if constexpr (kTree)
      for (int w = 0; w < p.words; ++w) p.masks[(int64_t)row * p.words + w] = row < used ? sees[row * p.words + w] : 0;
  }
  small_before(missing, lds, &all);
  if (t == 0) p.missing[0] = all;
}

struct ReleaseParams {
  int32_t* table;
  const int32_t* lengths;
  int32_t* free_pages;
  int64_t free_capacity;
  int32_t* free_count;
  int64_t batch, pps, page;
  int32_t* back;  // workspace: pages that sequence b gives back; at [batch] the free pages before the call
};

__device__ __forceinline__ int64_t release_first(const ReleaseParams& p, int64_t b) {
  const int64_t n = p.lengths[b];
  return n <= 0 ? 0 : (n + p.page - 1) / p.page;
}

__global__ void __launch_bounds__(kStepThreads) release_count_kernel(ReleaseParams p) {
  __shared__ int64_t lds[kStepWaves];
  const int64_t b = blockIdx.x;
  int64_t n = 0;
  for (int64_t e = release_first(p, b) + threadIdx.x; e < p.pps; e += kStepThreads)
    n += p.table[b * p.pps + e] >= 0;
  n = block_sum(n, lds);
  if (threadIdx.x == 0) {
    p.back[b] = (int32_t)n;
    if (b == 0) {
      const int64_t have = p.free_count[0];
      p.back[p.batch] = (int32_t)(have < 0 ? 0 : (have < p.free_capacity ? have : p.free_capacity));
    }
  }
}

// Page i of the ``total`` that go back lies at have + total - 1 - i, where taking
// pages in the same order found it. Pages that the stack has no room for (the
// first ones, then) stay mapped.
__global__ void __launch_bounds__(kStepThreads) release_put_kernel(ReleaseParams p) {
  __shared__ int64_t lds[kStepWaves];
  const int64_t b = blockIdx.x;
  int64_t mine = 0, all = 0;
  for (int64_t i = threadIdx.x; i < p.batch; i += kStepThreads) {
    const int64_t n = p.back[i];
    mine += i < b ? n : 0;
    all += n;
  }
  int64_t rank = block_sum(mine, lds);
  const int64_t total = block_sum(all, lds);
  const int64_t have = p.back[p.batch];
  for (int64_t e0 = release_first(p, b); e0 < p.pps; e0 += kStepThreads) {
    const int64_t e = e0 + threadIdx.x;
    const int32_t pg = e < p.pps ? p.table[b * p.pps + e] : -1;
    int n;
    const int64_t at = have + total - 1 - (rank + block_rank(pg >= 0, lds, &n));
    if (pg >= 0 && at < p.free_capacity) {
      p.free_pages[at] = pg;
      p.table[b * p.pps + e] = -1;
    }
    rank += n;
  }
  if (b == 0 && threadIdx.x == 0) {
    const int64_t now = have + total;
    p.free_count[0] = (int32_t)(now < p.free_capacity ? now : p.free_capacity);
  }
}

// At most 1024 sequences and 4096 entries, a run of them per thread. (16384 entries
// took one workgroup 22 us, the two launches above 7.7.)
constexpr int kSmallEntries = 4;
__global__ void __launch_bounds__(kSmallThreads) release_small_kernel(ReleaseParams p) {
  __shared__ int lds[kSmallWaves];
  __shared__ int s_first[kSmallThreads];
  const int t = threadIdx.x, pps = (int)p.pps, entries = (int)p.batch * pps;
  const int per = (entries + kSmallThreads - 1) / kSmallThreads, i0 = t * per;
  if (t < p.batch) s_first[t] = (int)release_first(p, t);
  const int64_t have0 = p.free_count[0];
  const int64_t have = have0 < 0 ? 0 : (have0 < p.free_capacity ? have0 : p.free_capacity);
  int32_t pg[kSmallEntries];
#pragma unroll
  for (int k = 0; k < kSmallEntries; ++k) pg[k] = k < per && i0 + k < entries ? p.table[i0 + k] : -1;
  __syncthreads();
  int b = i0 / pps, e = i0 - b * pps, n = 0, total;
#pragma unroll
  for (int k = 0; k < kSmallEntries; ++k) {
    if (pg[k] >= 0 && e < s_first[b]) pg[k] = -1;
    n += pg[k] >= 0;
    if (++e == pps) {
      e = 0;
      ++b;
    }
  }
  int rank = small_before(n, lds, &total);
#pragma unroll
  for (int k = 0; k < kSmallEntries; ++k)
    if (pg[k] >= 0) {
      const int64_t at = have + total - 1 - rank++;
      if (at < p.free_capacity) {
        p.free_pages[at] = pg[k];
        p.table[i0 + k] = -1;
      }
    }
  if (t == 0) p.free_count[0] = (int32_t)(have + total < p.free_capacity ? have + total : p.free_capacity);
}

// ---------------------------------------------------------------------------
// Accepted tokens of a tree moved to the front of its places, in the caches of
// all layers: row of position len + path[i] -> row of position len + i. A
// workgroup takes one sequence, one pool and a column of its rows; every thread
// holds what it moves in registers and all of a workgroup's reads come before its
// writes, so a path may cross itself. Bound by its chain of round trips: accepted,
// path, two page-table entries, the row.
// ---------------------------------------------------------------------------
constexpr int kKeepPools = 128;  // pools per launch: their pointers are kernel arguments
constexpr int kKeepRows = 256;   // most accepted tokens of a sequence
constexpr int kKeepTurns = 8;    // units (16, 4 or 1 bytes) that a thread holds
// Units of a row per workgroup: 32, which covers 512 bytes of codes, for up to 64
// accepted tokens, else 8.
constexpr int kKeepWide = 32, kKeepNarrow = kKeepTurns * kStepThreads / kKeepRows;

struct KeepParams {
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* path;
  const int32_t* accepted;
  int64_t pps, page, pool_pages, most;
  int64_t units[2];  // per row of the codes, and of the scales
  int blocks;        // workgroups over a row of codes; further ones take the scales
  void* pool[kKeepPools][2];
};

__device__ __forceinline__ int64_t keep_row(const KeepParams& p, int64_t b, int64_t t) {
  if (t < 0 || t >= p.pps * p.page) return -1;  // below 2^31, so that 32-bit divisions serve
  const uint32_t page = (uint32_t)p.page, e = (uint32_t)t / page;
  const int64_t pg = p.table[b * p.pps + e];
  return pg < 0 || pg >= p.pool_pages ? -1 : pg * p.page + ((uint32_t)t - e * page);
}

template <int kUnits, typename Unit>
__device__ __forceinline__ void keep_move(const KeepParams& p, int what, int64_t block, int n) {
  const int64_t b = blockIdx.y, units = p.units[what];
  const int64_t u = block * kUnits + threadIdx.x % kUnits;
  const int64_t len = p.lengths[b] < 0 ? 0 : p.lengths[b];
  Unit* pool = reinterpret_cast<Unit*>(p.pool[blockIdx.z][what]);
  Unit held[kKeepTurns];
  int64_t to[kKeepTurns];
#pragma unroll
  for (int k = 0; k < kKeepTurns; ++k) {
    const int i = k * (kStepThreads / kUnits) + (int)threadIdx.x / kUnits;
    to[k] = -1;
    if (i < n && u < units) {
      const int64_t step = p.path[b * p.most + i];
      const int64_t from = step < 0 ? -1 : keep_row(p, b, len + step);
      to[k] = from < 0 || step == i ? -1 : keep_row(p, b, len + i);
      if (to[k] >= 0) held[k] = pool[from * units + u];
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kKeepTurns; ++k)
    if (to[k] >= 0) pool[to[k] * units + u] = held[k];
}

template <int kUnits, typename Codes, typename Scales>
__global__ void __launch_bounds__(kStepThreads) keep_kernel(KeepParams p) {
  const int64_t asked = p.accepted[blockIdx.y];
  const int n = (int)(asked < p.most ? asked : p.most);
  if (n <= 0) return;
  if ((int)blockIdx.x < p.blocks)
    keep_move<kUnits, Codes>(p, 0, blockIdx.x, n);
  else
    keep_move<kUnits, Scales>(p, 1, blockIdx.x - p.blocks, n);
}

// The largest unit of 16, 4 and 1 bytes that rows and pools are multiples of.
static int keep_unit(int64_t bits) { return bits % 16 == 0 ? 16 : (bits % 4 == 0 ? 4 : 1); }

template <int kUnits, typename Codes>
static void keep_launch(const KeepParams& p, int scale_unit, dim3 grid, hipStream_t s) {
  if (scale_unit == 16)
    hipLaunchKernelGGL((keep_kernel<kUnits, Codes, u32x4>), grid, dim3(kStepThreads), 0, s, p);
  else if (scale_unit == 4)
    hipLaunchKernelGGL((keep_kernel<kUnits, Codes, uint32_t>), grid, dim3(kStepThreads), 0, s, p);
  else
    hipLaunchKernelGGL((keep_kernel<kUnits, Codes, uint8_t>), grid, dim3(kStepThreads), 0, s, p);
}

template <int kUnits>
static void keep_width(const KeepParams& p, const int* unit, dim3 grid, hipStream_t s) {
  if (unit[0] == 16)
    keep_launch<kUnits, u32x4>(p, unit[1], grid, s);
  else if (unit[0] == 4)
    keep_launch<kUnits, uint32_t>(p, unit[1], grid, s);
  else
    keep_launch<kUnits, uint8_t>(p, unit[1], grid, s);
}

// The caller's pools, as many per launch as its arguments hold.
static int keep_pools(KeepParams p, const q6moe_kv_keep_args* a, hipStream_t s) {
  const int64_t rows = a->pool_pages * a->page_size, bytes[2] = {a->code_bytes, a->scale_bytes};
  int64_t cache = 0, place = 0;  // the next pool: number ``place`` of its cache's
  while (cache < a->count) {
    int64_t bits[2] = {bytes[0], bytes[1]};
    int n = 0;
    while (n < kKeepPools && cache < a->count) {
      for (int w = 0; w < 2; ++w) {
        p.pool[n][w] = reinterpret_cast<uint8_t*>(a->pools[2 * cache + w]) + place * rows * bytes[w];
        bits[w] |= (int64_t)reinterpret_cast<uintptr_t>(p.pool[n][w]);
      }
      ++n;
      if (++place == (a->stacked ? a->stacked[cache] : 1)) {
        place = 0;
        ++cache;
      }
    }
    const int unit[2] = {keep_unit(bits[0]), keep_unit(bits[1])};
    p.units[0] = bytes[0] / unit[0];
    p.units[1] = bytes[1] / unit[1];
    const bool wide = p.most <= kKeepTurns * kStepThreads / kKeepWide;
    const int per = wide ? kKeepWide : kKeepNarrow;
    p.blocks = (int)cdiv(p.units[0], per);
    const dim3 grid((unsigned)(p.blocks + cdiv(p.units[1], per)), (unsigned)a->batch, (unsigned)n);
    if (wide)
      keep_width<kKeepWide>(p, unit, grid, s);
    else
      keep_width<kKeepNarrow>(p, unit, grid, s);
    if (const int rc = check_launch("kv_keep")) return rc;
  }
  return Q6MOE_OK;
}

}  // namespace q6moe

using namespace q6moe;

extern "C" size_t q6moe_kv_plan_workspace_size(int64_t batch) { return batch < 1 ? 0 : (size_t)(batch + 1) * 4; }

extern "C" int q6moe_kv_plan(const q6moe_kv_plan_args* a, void* stream) {
  Q6MOE_REQUIRE(a, "kv_plan: null args");
  Q6MOE_REQUIRE(a->page_table && a->lengths && a->counts && a->free_pages && a->free_count && a->starts && a->slots &&
                    a->positions && a->missing && a->workspace,
                "kv_plan: null pointer");
  Q6MOE_REQUIRE(a->batch >= 1 && a->batch <= kStepMaxBatch && a->pages_per_seq >= 1 && a->page_size >= 1 &&
                    a->free_capacity >= 1 && a->rows >= 1 && a->rows < (1ll << 31) && a->max_count >= 1,
                "kv_plan: batch, pages_per_seq, page_size, free_capacity, rows and max_count must be positive "
                "(batch at most 65535, rows below 2^31)");
  Q6MOE_REQUIRE(a->pages_per_seq < (1ll << 31) && a->page_size < (1ll << 31) &&
                    a->pages_per_seq * a->page_size < (1ll << 31) && a->free_capacity < (1ll << 31),
                "kv_plan: a sequence's capacity and the free stack must be below 2^31");
  if (a->parents) {
    Q6MOE_REQUIRE(a->masks && a->max_count <= kMaxTree, "kv_plan: trees need masks and a max_count of at most 256");
  } else {
    Q6MOE_REQUIRE(!a->masks, "kv_plan: masks need parents");
  }
  if (a->workspace_bytes < q6moe_kv_plan_workspace_size(a->batch)) {
    set_error("kv_plan: workspace too small (need " + std::to_string(q6moe_kv_plan_workspace_size(a->batch)) +
              " bytes)");
    return Q6MOE_ERR_INVALID;
  }
  PlanParams p;
  p.table = a->page_table;
  p.lengths = a->lengths;
  p.counts = a->counts;
  p.free_pages = a->free_pages;
  p.free_capacity = a->free_capacity;
  p.free_count = a->free_count;
  p.parents = a->parents;
  p.batch = a->batch;
  p.pps = a->pages_per_seq;
  p.page = a->page_size;
  p.rows = a->rows;
  p.max_count = a->max_count;
  p.words = a->parents ? (int)cdiv(a->max_count, 64) : 0;
  const int64_t lost = (0x7fffffff - a->rows) / a->batch;
  p.most_lost = lost > 1 ? (int)lost : 1;
  p.starts = a->starts;
  p.slots = a->slots;
  p.positions = a->positions;
  p.masks = reinterpret_cast<uint64_t*>(a->masks);
  p.missing = a->missing;
  p.need = reinterpret_cast<int32_t*>(a->workspace);
  hipStream_t s = (hipStream_t)stream;
  // One launch where a thread can take a sequence's pages and one workgroup the rows.
  const int64_t most = p.max_count < p.rows ? p.max_count : p.rows;
  if (p.batch <= kSmallThreads && p.rows <= kSmallRows && most / p.page + 2 <= kSmallPages &&
      (!p.parents || (p.rows <= kSmallTreeRows && p.rows * p.words <= kSmallRows))) {
    if (p.parents)
      hipLaunchKernelGGL(plan_small_kernel<true>, dim3(1), dim3(kSmallThreads), 0, s, p);
    else
      hipLaunchKernelGGL(plan_small_kernel<false>, dim3(1), dim3(kSmallThreads), 0, s, p);
    return check_launch("kv_plan kernel");
  }
  hipLaunchKernelGGL(plan_need_kernel, dim3((unsigned)p.batch), dim3(kStepThreads), 0, s, p);
  // Sequences of up to 4096 new tokens by their own workgroups: 638 K rows of 256
  // sequences in two launches 14.0 us, in three 17.0.
  if (most <= kTakeRows) {
    hipLaunchKernelGGL(plan_take_kernel<true>, dim3((unsigned)p.batch), dim3(kStepThreads), 0, s, p);
  } else {
    hipLaunchKernelGGL(plan_take_kernel<false>, dim3((unsigned)p.batch), dim3(kStepThreads), 0, s, p);
    hipLaunchKernelGGL(plan_rows_kernel, dim3((unsigned)cdiv(p.rows, kStepThreads * kPlanRows)),
                       dim3(kStepThreads), 0, s, p);
  }
  return check_launch("kv_plan kernels");
}

extern "C" int q6moe_kv_release(int32_t* page_table, const int32_t* lengths, int32_t* free_pages,
                                int64_t free_capacity, int32_t* free_count, int64_t batch, int64_t pages_per_seq,
                                int64_t page_size, void* workspace, size_t workspace_bytes, void* stream) {
  Q6MOE_REQUIRE(page_table && lengths && free_pages && free_count && workspace, "kv_release: null pointer");
  Q6MOE_REQUIRE(batch >= 1 && batch <= kStepMaxBatch && pages_per_seq >= 1 && page_size >= 1 && free_capacity >= 1,
                "kv_release: batch (at most 65535), pages_per_seq, page_size and free_capacity must be positive");
  Q6MOE_REQUIRE(pages_per_seq < (1ll << 31) && page_size < (1ll << 31) && free_capacity < (1ll << 31),
                "kv_release: sizes must be below 2^31");
  if (workspace_bytes < q6moe_kv_plan_workspace_size(batch)) {
    set_error("kv_release: workspace too small (need " + std::to_string(q6moe_kv_plan_workspace_size(batch)) +
              " bytes)");
    return Q6MOE_ERR_INVALID;
  }
  ReleaseParams p{page_table, lengths, free_pages, free_capacity, free_count, batch, pages_per_seq, page_size,
                  reinterpret_cast<int32_t*>(workspace)};
  hipStream_t s = (hipStream_t)stream;
  if (batch <= kSmallThreads && batch * pages_per_seq <= kSmallThreads * kSmallEntries) {
    hipLaunchKernelGGL(release_small_kernel, dim3(1), dim3(kSmallThreads), 0, s, p);
    return check_launch("kv_release kernel");
  }
  hipLaunchKernelGGL(release_count_kernel, dim3((unsigned)batch), dim3(kStepThreads), 0, s, p);
  hipLaunchKernelGGL(release_put_kernel, dim3((unsigned)batch), dim3(kStepThreads), 0, s, p);
  return check_launch("kv_release kernels");
}

extern "C" int q6moe_kv_keep(const q6moe_kv_keep_args* a, void* stream) {
  Q6MOE_REQUIRE(a, "kv_keep: null args");
  Q6MOE_REQUIRE(a->pools && a->page_table && a->lengths && a->path && a->accepted, "kv_keep: null pointer");
  Q6MOE_REQUIRE(a->count >= 1 && a->count <= (1 << 20) && a->batch >= 1 && a->batch <= kStepMaxBatch,
                "kv_keep: count and batch (at most 65535) must be positive");
  Q6MOE_REQUIRE(a->code_bytes >= 1 && a->scale_bytes >= 1 && a->code_bytes < (1 << 24) && a->scale_bytes < (1 << 24),
                "kv_keep: row sizes must be positive and below 2^24 bytes");
  Q6MOE_REQUIRE(a->pool_pages >= 1 && a->pages_per_seq >= 1 && a->page_size >= 1 && a->pool_pages < (1ll << 31) &&
                    a->pages_per_seq < (1ll << 31) && a->page_size < (1ll << 31) &&
                    a->pages_per_seq * a->page_size < (1ll << 31),
                "kv_keep: pool_pages, pages_per_seq and page_size must be positive, a sequence's capacity below 2^31");
  Q6MOE_REQUIRE(a->path_len >= 1 && a->path_len <= kKeepRows, "kv_keep: a path holds 1 to 256 tokens");
  for (int64_t i = 0; i < 2 * a->count; ++i) Q6MOE_REQUIRE(a->pools[i], "kv_keep: null pool");
  if (a->stacked)
    for (int64_t i = 0; i < a->count; ++i)
      Q6MOE_REQUIRE(a->stacked[i] >= 1 && a->stacked[i] <= (1 << 20), "kv_keep: a cache stacks 1 to 2^20 pools");
  KeepParams p;
  p.table = a->page_table;
  p.lengths = a->lengths;
  p.path = a->path;
  p.accepted = a->accepted;
  p.pps = a->pages_per_seq;
  p.page = a->page_size;
  p.pool_pages = a->pool_pages;
  p.most = a->path_len;
  hipStream_t s = (hipStream_t)stream;
  return keep_pools(p, a, s);
}
