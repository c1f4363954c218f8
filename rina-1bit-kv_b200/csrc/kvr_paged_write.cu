// RoPE of a step's new q and k, and the write of k and v into their pages.
//
// y_c = x_c cos_c - x_{c+64} sin_c, y_{c+64} = x_{c+64} cos_{c+64} + x_c sin_{c+64}
// (rotate_half convention) in fp32, rounded once to the tensors' type; k and v
// of token t go to cache slot slots[t] (page slots[t] / page), q to q_out.
//
// The bytes bound it (32/8 heads: 24.6 KB a token): 16384 tokens in 72 us, 5.8
// TB/s of the 6.5 that a plain copy measures; in a graph 2047 (64/8 heads) in 15
// us, part of them kept in L2, and one token in 2 us, the time of a launch (both 17
// us as calls from the host).  Eight lanes own a row:
// lane c holds channels 8c.. and 64+8c.., so a channel and its partner sit in
// the same thread and a warp's loads and stores are whole 128-byte lines.  A
// warp stays with one token and walks its rows four at a time with the
// token's table entries in registers; `parts` warps share a token so that a
// single token still spreads over enough warps to hide one round trip.
#include "kvr_attn_plan.cuh"

namespace kvr {

constexpr int kPwThreads = 128;

struct PagedWriteArgs {
  const void *q, *k, *v;
  int64_t n_tokens;
  int n_q, n_kv;
  int64_t q_stride, k_stride, v_stride;  // elements per token
  const float *cos_tbl, *sin_tbl;
  int64_t rope_stride, max_pos;
  const int *positions;
  const int64_t *slots;
  void *q_out;
  uint16_t *k_pages, *v_pages;
  int64_t n_slots;
  int page;
  int64_t page_stride, tok_stride;
  int parts;
};

template <int DT>
__global__ void __launch_bounds__(kPwThreads) paged_write_kernel(PagedWriteArgs a) {
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31;
  const int64_t unit = ((int64_t)blockIdx.x * kPwThreads + threadIdx.x) >> 5;
  const int64_t t = unit / a.parts;
  if (t >= a.n_tokens) return;
  const int part = (int)(unit - t * a.parts);
  const int c = (lane & 7) * 8, sub = lane >> 3;
  const int64_t slot = a.slots[t];
  const int64_t pos = a.positions ? a.positions[t] : 0;
  const bool live = slot >= 0 && slot < a.n_slots && (!a.cos_tbl || (pos >= 0 && pos < a.max_pos));
  float cl[8], ch[8], sl[8], sh[8];
  if (a.cos_tbl && live) {
    load8<KVR_F32>(a.cos_tbl, pos * a.rope_stride + c, cl);
    load8<KVR_F32>(a.cos_tbl, pos * a.rope_stride + 64 + c, ch);
    load8<KVR_F32>(a.sin_tbl, pos * a.rope_stride + c, sl);
    load8<KVR_F32>(a.sin_tbl, pos * a.rope_stride + 64 + c, sh);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      cl[e] = ch[e] = 1.0f;
      sl[e] = sh[e] = 0.0f;
    }
  }
  const int64_t at = live ? slot / a.page * a.page_stride + slot % a.page * a.tok_stride : 0;
  const int n_rot = a.q ? a.n_q : 0, rows = n_rot + 2 * a.n_kv;
  for (int r = part * 4 + sub; r < rows; r += a.parts * 4) {
    if (r < n_rot) {
      float x[8], y[8];
      void *o = a.q_out;
      const int64_t oi = (t * a.n_q + r) * kD + c;
      if (live) {
        load8<DT>(a.q, t * a.q_stride + (int64_t)r * kD + c, x);
        load8<DT>(a.q, t * a.q_stride + (int64_t)r * kD + 64 + c, y);
      } else {  // a padding token: zeros
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = y[e] = 0.0f;
      }
      float lo[8], hi[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo[e] = x[e] * cl[e] - y[e] * sl[e];
        hi[e] = y[e] * ch[e] + x[e] * sh[e];
      }
      store8<DT>(o, oi, lo);
      store8<DT>(o, oi + 64, hi);
    } else if (live && r < n_rot + a.n_kv) {
      const int h = r - n_rot;
      float x[8], y[8], lo[8], hi[8];
      load8<DT>(a.k, t * a.k_stride + (int64_t)h * kD + c, x);
      load8<DT>(a.k, t * a.k_stride + (int64_t)h * kD + 64 + c, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo[e] = x[e] * cl[e] - y[e] * sl[e];
        hi[e] = y[e] * ch[e] + x[e] * sh[e];
      }
      store8<DT>(a.k_pages, at + (int64_t)h * kD + c, lo);
      store8<DT>(a.k_pages, at + (int64_t)h * kD + 64 + c, hi);
    } else if (live) {
      const int h = r - n_rot - a.n_kv;
      const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.v) + t * a.v_stride +
                                                         (int64_t)h * kD + c);
      uint4 *dst = reinterpret_cast<uint4 *>(a.v_pages + at + (int64_t)h * kD + c);
      const uint4 u = src[0], w = src[8];
      dst[0] = u;
      dst[8] = w;
    }
  }
}

}  // namespace kvr

using namespace kvr;

extern "C" int kvr_paged_write(const void *q, const void *k, const void *v, int dtype, int64_t n_tokens, int n_q,
                               int n_kv, int d, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                               const float *cos_tbl, const float *sin_tbl, int64_t rope_stride, int64_t max_pos,
                               const int32_t *positions, const int64_t *slots, void *q_out, void *k_pages,
                               void *v_pages, int64_t n_pages, int page, int64_t page_stride, int64_t tok_stride,
                               kvr_stream_t stream) {
  clear_error();
  if (n_tokens == 0) return KVR_OK;
  KVR_REQUIRE(k && v && slots && k_pages && v_pages, "kvr_paged_write: null pointer");
  KVR_REQUIRE(!q == !q_out, "kvr_paged_write: q and q_out come together");
  KVR_REQUIRE(!cos_tbl == !sin_tbl && (!cos_tbl || positions), "kvr_paged_write: RoPE needs both tables and positions");
  KVR_REQUIRE(n_tokens > 0 && n_kv > 0 && (!q || n_q > 0), "kvr_paged_write: bad shape");
  if (d != kD) return set_error(KVR_ENOTSUP, "kvr_paged_write: head_dim must be 128");
  if (dtype != KVR_F16 && dtype != KVR_BF16)
    return set_error(KVR_ENOTSUP, "kvr_paged_write: the cache holds fp16 or bf16");
  KVR_REQUIRE(n_pages > 0 && page > 0, "kvr_paged_write: bad page pool");
  KVR_REQUIRE((!q || q_stride >= (int64_t)n_q * d) && k_stride >= (int64_t)n_kv * d && v_stride >= (int64_t)n_kv * d &&
                  tok_stride >= (int64_t)n_kv * d && page_stride >= 0,
              "kvr_paged_write: a token's heads must be contiguous");
  KVR_REQUIRE(((q ? q_stride : 0) | k_stride | v_stride | tok_stride | page_stride) % 8 == 0 &&
                  (!cos_tbl || (rope_stride % 4 == 0 && rope_stride >= d && max_pos > 0)),
              "kvr_paged_write: strides must keep rows 16-byte aligned");
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                         reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(q_out) |
                         reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages) |
                         reinterpret_cast<uintptr_t>(cos_tbl) | reinterpret_cast<uintptr_t>(sin_tbl);
  KVR_REQUIRE((ptrs & 15) == 0, "kvr_paged_write: pointers must be 16-byte aligned");
  // q_out may be q itself, row by row; nothing else that a call writes may lie in what it reads
  auto span = [](int64_t rows, int64_t stride, int64_t heads) { return ((rows - 1) * stride + heads * kD) * 2; };
  auto meet = [](const void *p, int64_t n, const void *o, int64_t m) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(o);
    return x < y + (uintptr_t)m && y < x + (uintptr_t)n;
  };
  if (q) {
    const int64_t n = span(n_tokens, (int64_t)n_q * d, n_q), pool = span(n_pages, page_stride, 0) + span(page, tok_stride, n_kv);
    KVR_REQUIRE((q_out == q && (n_tokens == 1 || q_stride == (int64_t)n_q * d)) || !meet(q_out, n, q, span(n_tokens, q_stride, n_q)),
                "kvr_paged_write: q_out must be q itself, laid out alike, or apart from it");
    KVR_REQUIRE(!meet(q_out, n, k, span(n_tokens, k_stride, n_kv)) && !meet(q_out, n, v, span(n_tokens, v_stride, n_kv)) &&
                    !meet(q_out, n, k_pages, pool) && !meet(q_out, n, v_pages, pool),
                "kvr_paged_write: q_out must not lie in k, v or the pages");
  }
  PagedWriteArgs a{q, k, v, n_tokens, n_q, n_kv, q_stride, k_stride, v_stride, cos_tbl, sin_tbl, rope_stride, max_pos,
                   positions, slots, q_out, static_cast<uint16_t *>(k_pages), static_cast<uint16_t *>(v_pages),
                   n_pages * page, page, page_stride, tok_stride, 1};
  const int rows = (q ? n_q : 0) + 2 * n_kv;
  while (a.parts * 4 < rows && n_tokens * a.parts < 148 * 16) a.parts *= 2;
  const int64_t ctas = (n_tokens * a.parts * 32 + kPwThreads - 1) / kPwThreads;
  KVR_REQUIRE(ctas <= INT_MAX, "kvr_paged_write: too many tokens");
  const cudaError_t e = launch_dependent(dtype == KVR_F16 ? paged_write_kernel<KVR_F16> : paged_write_kernel<KVR_BF16>,
                                         (unsigned)ctas, kPwThreads, 0, as_cuda(stream), a);
  if (e != cudaSuccess) return set_error(KVR_ECUDA, "kvr_paged_write: %s", cudaGetErrorString(e));
  return check_launch("kvr_paged_write");
}
