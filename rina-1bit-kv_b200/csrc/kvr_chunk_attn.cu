// Attention of packed query tokens over their requests' keys: pages
// (kvr_paged_attn) or packed K/V (kvr_prompt_attn), causal, grouped heads,
// driven by a plan (kvr_attn_plan.cuh).
//
// out = softmax(q k^T / scale) v over the keys a row sees, and lse =
// log(sum exp(q k^T / scale)); a row that sees no key gives zeros and -inf.
//
// A warp per query row walks the row's keys once with a running maximum and
// sum; lane l holds channels 4l .. 4l+3 of q, k, v and the output.
#include "kvr_attn_plan.cuh"

namespace kvr {

struct ChunkArgs {
  const void *q, *k, *v;
  int64_t q_stride;
  int64_t n_tokens, n_keys;         // packed K/V: tokens; pages: unused
  int64_t tok_stride, page_stride;  // elements
  int64_t k_tok_stride, v_tok_stride;
  int n_q, n_kv, batch;
  int paged, page;
  int64_t n_pages;
  const int *table;
  int64_t table_stride;
  int table_width;
  const PlanHeader *hdr;
  float inv_scale;
  void *out;
  float *lse;
  unsigned *err;
};

template <int DT>
__global__ void __launch_bounds__(256) chunk_attn_kernel(ChunkArgs a) {
  const PlanHeader &h = *a.hdr;
  if (h.magic != kPlanMagic || h.n_tokens != a.n_tokens || h.n_q != a.n_q || h.n_kv != a.n_kv || h.batch != a.batch) {
    if (threadIdx.x == 0) atomicOr(a.err, kWsErrPlan);
    return;
  }
  const PlanPiece *pieces = reinterpret_cast<const PlanPiece *>(a.hdr + 1);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = a.n_q / a.n_kv;
  for (int64_t w = blockIdx.x; w < (int64_t)h.n_pieces * a.n_kv; w += gridDim.x) {
    const PlanPiece p = pieces[w / a.n_kv];
    const int head = (int)(w % a.n_kv);
    for (int r = warp; r < p.n_tok * g; r += 8) {
      const int64_t t = p.q_start + r / g;
      const int hq = head * g + r % g;
      if (t < 0 || t >= a.n_tokens) continue;
      const int end = h.causal ? min(p.kv_len, p.first_end + r / g) : p.kv_len;
      const int begin = h.window > 0 ? max(0, p.first_end + r / g - h.window) : 0;
      float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.0f;
      load4<DT>(a.q, t * a.q_stride + (int64_t)hq * kD + lane * 4, q);
      for (int j = begin; j < end; ++j) {
        int64_t ki, vi;
        float k[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
        bool there;
        if (a.paged) {
          const int pj = j / a.page;
          const int page = pj < a.table_width ? a.table[p.k_start * a.table_stride + pj] : -1;
          there = page >= 0 && page < a.n_pages;
          ki = vi = page * a.page_stride + (int64_t)(j % a.page) * a.tok_stride;
        } else {
          there = (int64_t)p.k_start + j < a.n_keys;
          ki = ((int64_t)p.k_start + j) * a.k_tok_stride;
          vi = ((int64_t)p.k_start + j) * a.v_tok_stride;
        }
        if (there) {
          load4<DT>(a.k, ki + (int64_t)head * kD + lane * 4, k);
          load4<DT>(a.v, vi + (int64_t)head * kD + lane * 4, v);
        }
        const float s = warp_sum(q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3]) * a.inv_scale;
        const float mn = fmaxf(m, s), f = m == -INFINITY ? 0.0f : expf(m - mn), e = expf(s - mn);
        l = l * f + e;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] = o[c] * f + e * v[c];
        m = mn;
      }
      const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
      const int64_t oi = (t * a.n_q + hq) * kD + lane * 4;
#pragma unroll
      for (int c = 0; c < 4; ++c) store_elem<DT>(a.out, oi + c, l == 0.0f ? 0.0f : o[c] * inv);
      if (a.lse && lane == 0) a.lse[t * a.n_q + hq] = l == 0.0f ? -INFINITY : m + logf(l);
    }
  }
}

static int chunk_check(const char *fn, ChunkArgs &a, int dtype, int d, float scale, const void *plan,
                       size_t plan_bytes, void *workspace, size_t workspace_bytes) {
  KVR_REQUIRE(a.q && a.k && a.v && a.out && plan && workspace, "%s: null pointer", fn);
  if (d != kD) return set_error(KVR_ENOTSUP, "%s: head_dim must be 128", fn);
  if (dtype != KVR_F16 && dtype != KVR_BF16) return set_error(KVR_ENOTSUP, "%s: fp16 or bf16", fn);
  KVR_REQUIRE(a.n_kv > 0 && a.n_q > 0 && a.n_q % a.n_kv == 0, "%s: n_q must be a multiple of n_kv", fn);
  if (a.n_q / a.n_kv > kPlanRows)
    return set_error(KVR_ENOTSUP, "%s: more than %d query heads per KV head", fn, kPlanRows);
  KVR_REQUIRE(a.batch >= 1 && a.batch <= kPlanMaxBatch, "%s: batch must be in [1, %d]", fn, kPlanMaxBatch);
  KVR_REQUIRE(a.n_tokens >= 0 && a.n_tokens <= kPlanMaxTokens, "%s: bad token count", fn);
  KVR_REQUIRE(a.q_stride >= (int64_t)a.n_q * d && a.q_stride % 8 == 0,
              "%s: a token's heads must be contiguous, rows 16-byte aligned", fn);
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) |
                         reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.out) |
                         reinterpret_cast<uintptr_t>(plan);
  KVR_REQUIRE((ptrs & 15) == 0, "%s: pointers must be 16-byte aligned", fn);
  KVR_REQUIRE(plan_bytes >= kvr_attn_plan_bytes(a.n_tokens, a.batch, a.n_q, a.n_kv), "%s: plan too small", fn);
  KVR_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "%s: workspace alignment", fn);
  const size_t need = kvr_attn_workspace_bytes(a.n_q, a.n_kv);
  KVR_REQUIRE(workspace_bytes >= need, "%s: workspace %zu < %zu bytes", fn, workspace_bytes, need);
  KVR_REQUIRE(scale == scale && scale <= 3.0e38f, "%s: bad scale", fn);
  a.inv_scale = 1.0f / (scale > 0.0f ? scale : sqrtf((float)d));
  a.hdr = static_cast<const PlanHeader *>(plan);
  a.err = static_cast<unsigned *>(workspace);
  return KVR_OK;
}

static int chunk_launch(const char *fn, const ChunkArgs &a, int dtype, kvr_stream_t stream) {
  if (dtype == KVR_F16) chunk_attn_kernel<KVR_F16><<<148 * 8, 256, 0, as_cuda(stream)>>>(a);
  else chunk_attn_kernel<KVR_BF16><<<148 * 8, 256, 0, as_cuda(stream)>>>(a);
  return check_launch(fn);
}

}  // namespace kvr

using namespace kvr;

extern "C" size_t kvr_attn_workspace_bytes(int n_q, int n_kv) {
  (void)n_q;
  (void)n_kv;
  return kWsHeader;
}

extern "C" int kvr_paged_attn(const void *q, int dtype, int64_t n_tokens, int batch, int n_q, int n_kv, int d,
                              int64_t q_stride, const void *k_pages, const void *v_pages, int64_t n_pages, int page,
                              int64_t page_stride, int64_t tok_stride, const int32_t *block_table,
                              int64_t table_stride, int table_width, const void *plan, size_t plan_bytes, float scale,
                              void *out, float *lse, void *workspace, size_t workspace_bytes, kvr_stream_t stream) {
  clear_error();
  if (n_tokens == 0) return KVR_OK;
  ChunkArgs a{};
  a.q = q; a.k = k_pages; a.v = v_pages;
  a.q_stride = q_stride;
  a.n_tokens = n_tokens;
  a.tok_stride = tok_stride; a.page_stride = page_stride;
  a.n_q = n_q; a.n_kv = n_kv; a.batch = batch;
  a.paged = 1; a.page = page; a.n_pages = n_pages;
  a.table = block_table; a.table_stride = table_stride; a.table_width = table_width;
  a.out = out; a.lse = lse;
  const int rc = chunk_check("kvr_paged_attn", a, dtype, d, scale, plan, plan_bytes, workspace, workspace_bytes);
  if (rc) return rc;
  KVR_REQUIRE(block_table && table_width >= 1 && table_stride >= table_width, "kvr_paged_attn: bad block table");
  KVR_REQUIRE(n_pages > 0 && n_pages <= INT_MAX, "kvr_paged_attn: bad page pool");
  if (page < 8 || page % 8 != 0 || page > (1 << 20))
    return set_error(KVR_ENOTSUP, "kvr_paged_attn: the page size must be a multiple of 8 tokens");
  KVR_REQUIRE(tok_stride >= (int64_t)n_kv * d && tok_stride % 8 == 0 && page_stride >= 0 && page_stride % 8 == 0,
              "kvr_paged_attn: a token's heads must be contiguous, rows 16-byte aligned");
  return chunk_launch("kvr_paged_attn", a, dtype, stream);
}

extern "C" int kvr_prompt_attn(const void *q, const void *k, const void *v, int dtype, int64_t n_tokens,
                               int64_t n_keys, int batch, int n_q, int n_kv, int d, int64_t q_stride, int64_t k_stride,
                               int64_t v_stride, const void *plan, size_t plan_bytes, float scale, void *out,
                               float *lse, void *workspace, size_t workspace_bytes, kvr_stream_t stream) {
  clear_error();
  if (n_tokens == 0) return KVR_OK;
  ChunkArgs a{};
  a.q = q; a.k = k; a.v = v;
  a.q_stride = q_stride;
  a.n_tokens = n_tokens; a.n_keys = n_keys;
  a.k_tok_stride = k_stride; a.v_tok_stride = v_stride;
  a.n_q = n_q; a.n_kv = n_kv; a.batch = batch;
  a.out = out; a.lse = lse;
  const int rc = chunk_check("kvr_prompt_attn", a, dtype, d, scale, plan, plan_bytes, workspace, workspace_bytes);
  if (rc) return rc;
  KVR_REQUIRE(n_keys > 0 && n_keys <= kPlanMaxLen, "kvr_prompt_attn: bad key count");
  KVR_REQUIRE(k_stride >= (int64_t)n_kv * d && v_stride >= (int64_t)n_kv * d && (k_stride | v_stride) % 8 == 0,
              "kvr_prompt_attn: a token's heads must be contiguous, rows 16-byte aligned");
  return chunk_launch("kvr_prompt_attn", a, dtype, stream);
}
