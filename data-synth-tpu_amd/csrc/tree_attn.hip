// Attention of several new tokens per sequence over the paged INT8 cache: every
// row of a ragged batch (a drafted tree, or a chunk of a prompt) against the
// cached tokens of its sequence and the new tokens that its mask names.
//
//   s = (q . kc) * ks / sqrt(D),   out = sum_t p_t vs_t vc_t / sum_t p_t,
//   p_t = exp(s_t - max s)
//
// with the INT8 codes kc, vc and the FP32 scales ks, vs of (token, KV head).
#include "q6moe_api.h"
#include "q6moe_device.h"

namespace q6moe {

constexpr int kTreeThreads = 256;
constexpr int kTreeMaxHeads = 65535;

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
  int64_t batch, rows, max_count;
  int kvh, hq, r;
  int64_t pool_pages, pps, page, cap;
  uint16_t* out;
};

__device__ __forceinline__ float tree_scale(const TreeParams& p, const void* s, int64_t i) {
  return p.scale_bf16 ? bf16_to_float(reinterpret_cast<const uint16_t*>(s)[i]) : reinterpret_cast<const float*>(s)[i];
}

// One workgroup per (row, query head): 256 keys at a time, one per thread for
// the scores, then one channel per thread (and key group) for the sum of values.
template <int D>
__global__ void __launch_bounds__(kTreeThreads) tree_attn_simple_kernel(TreeParams p) {
  __shared__ float qs[D], pr[kTreeThreads], red[kTreeThreads];
  __shared__ int64_t at[kTreeThreads];
  const int64_t row = blockIdx.x;
  const int h = blockIdx.y, kh = h / p.r, t = threadIdx.x;
  int64_t b = 0, hi = p.batch - 1;  // the last sequence with starts[b] <= row
  while (b < hi) {
    const int64_t mid = (b + hi + 1) / 2;
    if (p.starts[mid] <= row)
      b = mid;
    else
      hi = mid - 1;
  }
  const int64_t j = row - p.starts[b];
  if (j < 0 || row >= p.starts[b + 1] || j >= p.max_count) return;
  int64_t count = p.starts[b + 1] - p.starts[b];
  count = count < p.max_count ? count : p.max_count;
  const int64_t len = p.len[b] < 0 ? 0 : p.len[b];
  const int64_t seen = p.masks ? count : j + 1;
  const int64_t n = len + seen < p.cap ? len + seen : p.cap;
  if (t < D) qs[t] = bf16_to_float(p.q[row * p.q_stride + (int64_t)h * D + t]);
  float m = -__builtin_inff(), l = 0.f, acc = 0.f;
  constexpr int kParts = kTreeThreads / D;  // key groups of the value sum
  const int c = t % D, part = t / D;
  const float inv = 1.f / sqrtf((float)D);
  for (int64_t t0 = 0; t0 < n; t0 += kTreeThreads) {
    __syncthreads();
    const int64_t key = t0 + t;
    bool on = key < n;
    if (on && key >= len && p.masks) {
      const int64_t jj = key - len;
      on = (p.masks[row * p.words + (jj >> 6)] >> (jj & 63)) & 1;
    }
    int64_t r = -1;
    if (on) {
      const int64_t pg = p.table[b * p.pps + key / p.page];
      if (pg >= 0 && pg < p.pool_pages) r = pg * p.page + key % p.page;
    }
    float s = -__builtin_inff();
    if (on) {
      float dot = 0.f;
      if (r >= 0) {
        const int8_t* k = p.kc + (r * p.kvh + kh) * D;
        for (int d = 0; d < D; ++d) dot += qs[d] * (float)k[d];
        dot *= tree_scale(p, p.ks, r * p.kvh + kh);
      }
      s = dot * inv;
    }
    red[t] = s;
    at[t] = r;
    __syncthreads();
    float top = m;
    for (int i = 0; i < kTreeThreads; ++i) top = fmaxf(top, red[i]);
    const float shift = top == -__builtin_inff() ? 0.f : top;
    const float e = on ? expf(s - shift) : 0.f;
    pr[t] = e;
    __syncthreads();
    const float fade = expf(m - shift);
    l *= fade;
    acc *= fade;
    for (int i = 0; i < kTreeThreads; ++i) l += pr[i];
    for (int i = part; i < kTreeThreads; i += kParts) {
      const int64_t rr = at[i];
      if (pr[i] != 0.f && rr >= 0)
        acc += pr[i] * tree_scale(p, p.vs, rr * p.kvh + kh) * (float)p.vc[(rr * p.kvh + kh) * D + c];
    }
    m = top;
  }
  __syncthreads();
  red[t] = acc;
  __syncthreads();
  if (t < D) {
    float v = 0.f;
    for (int i = 0; i < kParts; ++i) v += red[i * D + t];
    p.out[(row * p.hq + h) * D + t] = bf16_bits(l == 0.f ? 0.f : v / l);
  }
}

}  // namespace q6moe

using namespace q6moe;

extern "C" size_t q6moe_tree_attn_workspace_size(int64_t batch, int64_t rows, int64_t max_count, int64_t query_heads,
                                                 int64_t kv_heads, int64_t head_dim, int64_t pages_per_seq,
                                                 int64_t page_size) {
  if (batch < 1 || rows < 1 || max_count < 1 || query_heads < 1 || kv_heads < 1 || pages_per_seq < 1 || page_size < 1)
    return 0;
  return 256;
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
                    a->pages_per_seq * a->page_size <= (1 << 30),
                "tree_attention: page_size, pages_per_seq and pool_pages must be positive, a sequence's capacity at "
                "most 2^30");
  Q6MOE_REQUIRE(a->scale_dtype == Q6MOE_BF16 || a->scale_dtype == Q6MOE_F32, "tree_attention: scale dtype");
  Q6MOE_REQUIRE(!a->masks || (a->mask_words >= 1 && a->mask_words <= 4 && a->max_count <= 64 * a->mask_words),
                "tree_attention: masks hold max_count bits in at most 4 words");
  Q6MOE_REQUIRE(a->q_stride >= 0 && a->q_stride % 8 == 0, "tree_attention: q_stride must be a multiple of 8");
  Q6MOE_REQUIRE(aligned(a->q, 16) && aligned(a->k_codes, 16) && aligned(a->v_codes, 16) && aligned(a->out, 16) &&
                    aligned(a->workspace, 256),
                "tree_attention: q, codes and out need 16-byte and workspace 256-byte alignment");
  const size_t need = q6moe_tree_attn_workspace_size(a->batch, a->rows, a->max_count, a->query_heads, a->kv_heads,
                                                     a->head_dim, a->pages_per_seq, a->page_size);
  if (a->workspace_bytes < need) {
    set_error("tree_attention: workspace too small (need " + std::to_string(need) + " bytes)");
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
  p.batch = a->batch;
  p.rows = a->rows;
  p.max_count = a->max_count;
  p.kvh = (int)a->kv_heads;
  p.hq = (int)a->query_heads;
  p.r = p.hq / p.kvh;
  p.pool_pages = a->pool_pages;
  p.pps = a->pages_per_seq;
  p.page = a->page_size;
  p.cap = a->pages_per_seq * a->page_size;
  p.out = a->out;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)p.rows, (unsigned)p.hq);
  if (a->head_dim == 64)
    hipLaunchKernelGGL(tree_attn_simple_kernel<64>, grid, dim3(kTreeThreads), 0, s, p);
  else if (a->head_dim == 128)
    hipLaunchKernelGGL(tree_attn_simple_kernel<128>, grid, dim3(kTreeThreads), 0, s, p);
  else
    hipLaunchKernelGGL(tree_attn_simple_kernel<256>, grid, dim3(kTreeThreads), 0, s, p);
  return check_launch("tree_attention");
}
