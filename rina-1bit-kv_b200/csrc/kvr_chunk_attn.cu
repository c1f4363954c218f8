// Attention of packed query tokens over their requests' keys: pages
// (kvr_paged_attn) or packed K/V (kvr_prompt_attn), causal, grouped heads,
// driven by a plan (kvr_attn_plan.cuh).
//
// out = softmax(q k^T / scale) v over the keys a row sees, and lse =
// log(sum exp(q k^T / scale)); a row that sees no key gives zeros and -inf.
//
// One pass over the keys with a running maximum and sum.  A CTA (one per SM)
// walks the plan's pieces: up to two 128-row query tiles against K/V tiles of
// 128 keys.  Packing the g query heads of a KV head into the rows (row = token
// * g + j) lets one K/V tile serve all of them, for one token as for many.
//   warp 9   copies: Q tiles, then K, V, K, V, ... by TMA (128-byte swizzle)
//            into rings of two and three 32 KB stages; a paged tile is a box per page
//            (or per gcd(page, 128) rows), a missing page an out-of-range box,
//            which the TMA fills with zeros;
//   warp 8   one lane issues tcgen05.mma: S = Q_t K^T (128 x 128 x 128,
//            operands in shared memory);
//   warp 10  likewise O_t += P_t V, P_t in tensor memory, V read column-wise
//            from shared memory; a warp of its own, so that neither kind waits
//            in the other's issue order;
//   warps 0-3 and 4-7   a warpgroup per query tile, a row per thread: S from
//            tensor memory into registers, mask, maximum, exp2, sum; the
//            weights P_t, rounded to the tensors' 16-bit type, back to tensor
//            memory.
// Tensor memory: S, P_0 | P_1 (64 columns each), O_0, O_1, 128 columns each.
// One S serves both tiles: a warpgroup copies it to registers at once and
// frees it, so the tensor core computes the next S while the weights of this
// one are formed, and a tile's chain is its softmax, not softmax + two MMAs.
// (An S per tile with P over it and S of the next keys after P V, one issuing
// warp: 328 us for a chunk of 512 at 32256, 32/8 heads, in a graph of 12 calls;
// this way 236 us.  Call after call, at the clock of a longer load, 275 us.)
//
// What binds a long prompt: a warpgroup's chain of a K/V tile, about 2900
// cycles beside the other warpgroup's, and 500 more until the next S is seen,
// against 2048 cycles of MMA for both tiles.  (Prompt of 16384: 1.88 ms call after
// call, 1171 TFLOP/s, 0.71 of the burst and 0.85 of the sustained matmul rate; 1.64
// to 1.72 ms in a graph of 12.)  Tensor pipe and special function
// unit (16 exponentials a cycle) are 70 % active each.  With the MMAs reduced to
// one step in eight a chunk of 512 at 32256 takes 3 % less, without the
// exponentials 7 %, without both 33 %: what is left is the issue of some 560
// instructions a tile by one warp per scheduler and tile.  So the slow paths
// (a wait that has to poll, the rescaling, the masks) are kept small and out of
// the way: 72 KB of code to 54 KB gained 10 % on windowed and packed prompts.
// Exponentials on the FMA pipe (a polynomial for 1/8 to 1/2 of them) lost 3 to
// 30 % by their instructions; four warpgroups with half of a tile's keys each
// lost 60 % (104 registers a thread, maxima met through shared memory).
//
// The output accumulator is rescaled only when a row's maximum has grown by
// more than 2^kLazy since its last rescale (the weights stay below 2^(kLazy +
// kShift), the sums are exact either way), so the read-modify-write of O is
// rare after the first tiles.  Weights carry a factor 2^kShift that cancels in
// the division: it keeps fp16 weights of 2^-18 out of the subnormals.
//
// What is held in fewer than 32 bits: the weights P, rounded to the tensors'
// type because both operands of an MMA are of one 16-bit type; the sum that
// divides them is of the unrounded ones, in fp32.  That makes the error against
// 64 bits 1.1 to 1.4 times that of rounding the output alone (2.3e-3 for 1.7e-3
// in bf16, 2.5e-4 for 2.0e-4 in fp16, relative in the 2-norm).
//
// Keys past a request's end, or before every row's window, are masked in S,
// and their V rows are zeroed in shared memory, because 0 times a NaN of a
// neighbour would still be a NaN.  (Not so a request's own keys that some rows of
// an item see and others do not: an infinity or NaN in such a V row reaches both.)
//
// Rows without a query (a decode step has g of them in 128) are kept at zero,
// in Q and in P: the MMAs over them cost no time that the memory does not, but
// with other requests' queries in them they cost power, and with it clock
// (decode of 32 x 16384 back to back: 418 -> 387 us).  For the same reason a
// piece of at most 16 rows is multiplied as M = 64: its rows 0 .. 15 lie in the
// same lanes of tensor memory (row r in lane r / 16 * 32 + r % 16), half the
// rows are computed (back to back 2000 times 396 -> 363 us; a plain copy of as
// many bytes takes 333 us then).
//
// Every wait is bounded; one that gives up sets the error word, lets the
// copies and MMAs in flight drain and frees the tensor memory.  A warp's lanes
// give up together: by a vote at the wait, or, where a vote costs time (the
// issuing warps), by going on to the piece's end (tc_wait_on).
#include "kvr_attn_plan.cuh"
#include "kvr_tcgen05.cuh"

namespace kvr {

constexpr int kCaThreads = 384;  // two softmax warpgroups; MMA, copies and two idle warps
// A ring of K tiles and one of V tiles.  (One ring for both would not do: K and V have different consumers,
// and a stage's barrier tells its phases apart by parity only, so each phase must be seen by the same waiter.)
constexpr int kCaStagesK = 2, kCaStagesV = 3, kCaStages = kCaStagesK + kCaStagesV;
constexpr uint32_t kCaTile = 128 * kD * 2;      // 32 KB: 128 rows of K, V or Q
constexpr uint32_t kCaHalf = kCaTile / 2;       // 64 channels of them
constexpr uint32_t kCaOffKv = 2 * kCaTile;
constexpr uint32_t kCaOffBar = kCaOffKv + kCaStages * kCaTile;
constexpr int kCaBars = 2 * kCaStages + 15;
constexpr int kCaRecords = 64;                  // pieces of a CTA kept in shared memory
constexpr uint32_t kCaOffRec = (kCaOffBar + kCaBars * 8 + 16 + 31) / 32 * 32;
constexpr uint32_t kCaSmem = kCaOffRec + kCaRecords * 32;
constexpr uint32_t kCaTmemCols = 512;
constexpr int kCaFewTokens = 8;  // a query tile with at most so many tokens is loaded token by token
constexpr int kCaFewRows = 16;   // a piece with at most so many rows is multiplied as M = 64
constexpr float kLazy = 6.0f, kShift = 4.0f;
constexpr float kLowest = -3e38f;  // maximum of a row that has seen nothing: finite, so that -inf - it is -inf
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;


struct ChunkArgs {
  int64_t n_tokens;
  int n_q, n_kv, batch;
  int page, box;                // paged: tokens per page, rows per copy (gcd(page, 128))
  int n_pages;
  const int *table;
  int64_t table_stride;
  int table_width;
  const PlanHeader *hdr;
  float to_log2;                // log2(e) / scale
  void *out;
  float *lse;
  float *part_o, *part_ml;      // partial rows: 128 values; maximum (log2 units) and sum
  unsigned *err;
};

// ------------------------------------------------------- tcgen05 and TMA ----

// N x K with N contiguous (V, N = channels): atoms of 64 channels x 8 keys; 16
// KB to the other 64 channels (low word), 1 KB to the next 8 keys.
__device__ __forceinline__ uint32_t ca_desc_mn(uint32_t saddr) { return (saddr >> 4) | ((kCaHalf >> 4) << 16); }
// kind::f16, fp32 accumulator, M 128 or 64, N 128.
template <int DT>
__host__ __device__ constexpr uint32_t ca_idesc(bool b_mn, uint32_t m = 128) {
  return (1u << 4) | ((DT == KVR_BF16 ? 1u : 0u) << 7) | ((DT == KVR_BF16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
         ((128u >> 3) << 17) | ((m >> 4) << 24);
}

__device__ __forceinline__ void ca_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void ca_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void ca_st16(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}

// 32 bytes to global memory: a whole sector per lane (a row per lane makes
// 16-byte stores write half sectors, twice as many).
__device__ __forceinline__ void ca_store32(void *p, const uint32_t *w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

__device__ __forceinline__ void ca_tma4(uint32_t dst, const CUtensorMap *m, int c1, int c2, int c3, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(m), "r"(0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void ca_tma5(uint32_t dst, const CUtensorMap *m, int c1, int c2, int c3, int c4,
                                        uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
      "%6}], [%7];" ::"r"(dst),
      "l"(m), "r"(0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_u32(bar))
      : "memory");
}

// ---------------------------------------------------------------- waiting ----

// Whether the phase is complete by now (never waits).
__device__ __forceinline__ bool ca_test(uint64_t *bar, unsigned phase) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(phase)
      : "memory");
  return done != 0;
}
// Stage of the n-th K (or V) tile.
__device__ __forceinline__ int ca_stage(bool v, int n) { return v ? kCaStagesK + n % kCaStagesV : n % kCaStagesK; }

// ------------------------------------------------------------ the pieces ----

// Piece number r of CTA c (see kvr_attn_plan.cuh), or false past the last.
struct CaPiece {
  PlanPiece p;
  int head, n, two;  // KV head, K/V tiles, whether the second query tile has rows
};
// (a call's pieces number less than 2^31: 2^24 tokens in items of 256 rows)
__device__ __forceinline__ unsigned ca_index(int r) {
  return r * gridDim.x + ((r & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}
__device__ __forceinline__ bool ca_piece(const ChunkArgs &a, const unsigned char *rec, unsigned total, unsigned heads,
                                         int per, int r, CaPiece &o) {
  const unsigned i = ca_index(r);
  if (i >= total) return false;
  const unsigned e = i / heads;
  o.p = r < kCaRecords ? reinterpret_cast<const PlanPiece *>(rec)[r] : reinterpret_cast<const PlanPiece *>(a.hdr + 1)[e];
  o.head = (int)(i - e * heads) + (o.p.n_tok >> 16);
  o.p.n_tok &= 0xffff;
  o.p.n_tok = min(max(o.p.n_tok, 0), per);
  o.n = o.p.n_tok > 0 ? max(o.p.kt1 - o.p.kt0, 0) : 0;
  o.two = o.p.n_tok > (per >> 1);
  return true;
}

__device__ __forceinline__ float ca_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float ca_max3(float x, float y, float z) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
// Pairs of floats for the packed fp32 instructions.
__device__ __forceinline__ uint64_t ca_pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float ca_lo(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float ca_hi(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint64_t ca_fma2(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}
__device__ __forceinline__ uint64_t ca_add2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ uint64_t ca_exp2_sfu(uint64_t x) { return ca_pair(ca_exp2(ca_lo(x)), ca_exp2(ca_hi(x))); }
// Bits 0 .. n - 1 (none for n <= 0, all for n >= 32).
__device__ __forceinline__ uint32_t ca_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
template <int DT>
__device__ __forceinline__ uint32_t ca_pack(float lo, float hi) {
  uint32_t r;
  if constexpr (DT == KVR_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Whether the plan is one for this call, with all of its items.
__device__ __forceinline__ bool ca_plan_fits(const PlanHeader &h, const ChunkArgs &a) {
  return h.magic == kPlanMagic && h.n_tokens == a.n_tokens && h.n_q == a.n_q && h.n_kv == a.n_kv && h.batch == a.batch &&
         !h.dropped;
}

template <int DT, bool PAGED>
__global__ void __launch_bounds__(kCaThreads, 1)
    chunk_attn_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mq1,
                      const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                      const ChunkArgs a) {
  extern __shared__ __align__(1024) unsigned char sm[];
  uint64_t *kv_full = reinterpret_cast<uint64_t *>(sm + kCaOffBar);
  uint64_t *kv_empty = kv_full + kCaStages;
  uint64_t *q_full = kv_empty + kCaStages;
  uint64_t *q_empty = q_full + 2;
  uint64_t *s_full = q_empty + 2;
  uint64_t *p_full = s_full + 2;
  uint64_t *pv_done = p_full + 4;  // p_full: two halves per tile
  uint64_t *s_free = pv_done + 2;
  uint64_t *drained = s_free + 1;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drained + 2);
  volatile int *abort_s = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kCaTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (tid == 9 * 32) {
    *abort_s = 0;
    for (int s = 0; s < kCaStages; ++s) {
      tc_bar_init(&kv_full[s], 1);
      tc_bar_init(&kv_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      tc_bar_init(&q_full[t], 1);
      tc_bar_init(&q_empty[t], 1);
      tc_bar_init(&s_full[t], 1);
      tc_bar_init(&p_full[2 * t], 4);
      tc_bar_init(&p_full[2 * t + 1], 4);
      tc_bar_init(&drained[t], 1);
      tc_bar_init(&pv_done[t], 1);
    }
    tc_bar_init(s_free, 4);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // barriers: for the copies and commits
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();  // what follows reads the plan, q and the cache
  griddep_launch();  // the joining kernel waits for this grid's end

  // (the CTA's first pieces go to shared memory: every role reads each of them)
  const PlanHeader &h = *a.hdr;
  const bool fits = ca_plan_fits(h, a);
  if (!fits && tid == 0) atomicOr(a.err, kWsErrPlan);
  const unsigned heads = h.even ? 1u : (unsigned)a.n_kv;  // KV heads that a list entry stands for
  const unsigned total = fits ? (unsigned)h.n_pieces * heads : 0;
  const int causal = h.causal, window = h.window;
  if (tid < kCaRecords && ca_index(tid) < total)
    reinterpret_cast<PlanPiece *>(sm + kCaOffRec)[tid] =
        reinterpret_cast<const PlanPiece *>(a.hdr + 1)[ca_index(tid) / heads];
  __syncthreads();
  const int g = a.n_q / a.n_kv, tpt = kPlanRows / g, per = 2 * tpt;

  // registers: 384 threads x 168 at launch = (208 + 208 + 88) x 128
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == 11) {
    __syncthreads();
  } else if (warp == 9) {
    // ---- copies
    int fill[2] = {0, 0}, uses[2] = {0, 0};  // K and V stages, Q tiles filled so far
    int zero_from[2] = {128, 128};           // rows of the Q tiles that hold zeros
    CaPiece c;
    bool ok = true;
    for (int r = 0; ok && ca_piece(a, sm + kCaOffRec, total, heads, per, r, c); ++r) {
      const int64_t row = PAGED ? (int64_t)c.p.k_start * a.table_stride : 0;
      const bool known = PAGED && c.p.k_start >= 0 && c.p.k_start < a.batch;
      int id = 0, off = 0;  // paged: this lane's page and row in it, of the next K/V tile
      auto look = [&](int kt) {
        if (PAGED && lane * a.box < 128) {
          const int key = kt * 128 + lane * a.box, pj = key / a.page;
          off = key - pj * a.page;
          id = known && key < c.p.kv_len && pj < a.table_width ? a.table[row + pj] : -1;
          if (id < 0 || id >= a.n_pages) id = a.n_pages;  // out of range: zeros
        }
      };
      auto load = [&](const CUtensorMap *m, bool v, int kt) {
        const int n = fill[v], depth = v ? kCaStagesV : kCaStagesK, s = ca_stage(v, n);
        if (n >= depth && !tc_wait_warp(&kv_empty[s], (unsigned)((n / depth - 1) & 1), abort_s)) return false;
        ++fill[v];
        const uint32_t dst = smem_u32(sm) + kCaOffKv + s * kCaTile;
        if (lane == 0) mbar_expect_tx(&kv_full[s], kCaTile);
        __syncwarp();
        if (PAGED) {
          if (lane * a.box < 128) {
            const uint32_t d = dst + lane * a.box * 128;
            ca_tma5(d, m, off, 0, c.head, id, &kv_full[s]);
            ca_tma5(d + kCaHalf, m, off, 1, c.head, id, &kv_full[s]);
          }
        } else if (lane == 0) {
          ca_tma4(dst, m, c.p.k_start + kt * 128, 0, c.head, &kv_full[s]);
        }
        return true;
      };
      auto load_q = [&](int t) {
        if (uses[t] > 0 && !tc_wait_warp(&q_empty[t], (unsigned)((uses[t] - 1) & 1), abort_s)) return false;
        const uint32_t dst = smem_u32(sm) + t * kCaTile;
        const int n_tok = min(tpt, c.p.n_tok - t * tpt);
        if (n_tok <= kCaFewTokens) {  // token by token, zeros below
          unsigned char *qs = sm + t * kCaTile;
          const int from = n_tok * g * 8;  // 16-byte pieces of a half row
          for (int e = from + lane; e < zero_from[t] * 8; e += 32) {
            *reinterpret_cast<uint4 *>(qs + e * 16) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4 *>(qs + kCaHalf + e * 16) = make_uint4(0, 0, 0, 0);
          }
          zero_from[t] = n_tok * g;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          if (lane == 0) mbar_expect_tx(&q_full[t], 2u * 128u * n_tok * g);
          __syncwarp();
          if (lane < 2 * n_tok) {
            const int k = lane >> 1, half = lane & 1;
            ca_tma5(dst + half * kCaHalf + k * g * 128, &mq1, 0, c.p.q_start + t * tpt + k, half, c.head, &q_full[t]);
          }
        } else {
          zero_from[t] = 128;
          if (lane == 0) {
            mbar_expect_tx(&q_full[t], 2u * 128u * tpt * g);
            ca_tma5(dst, &mq, 0, c.p.q_start + t * tpt, 0, c.head, &q_full[t]);
            ca_tma5(dst + kCaHalf, &mq, 0, c.p.q_start + t * tpt, 1, c.head, &q_full[t]);
          }
        }
        ++uses[t];
        return true;
      };
      if (c.n == 0) continue;
      look(c.p.kt0);
      ok = load_q(0) && load(&mk, false, c.p.kt0) && (!c.two || load_q(1));
      for (int i = 0; ok && i < c.n; ++i) {
        ok = load(&mv, true, c.p.kt0 + i);
        if (ok && i + 1 < c.n) {
          look(c.p.kt0 + i + 1);
          ok = load(&mk, false, c.p.kt0 + i + 1);
        }
      }
      ok = __all_sync(~0u, ok && !*abort_s);
    }
    if (!ok && lane == 0) {
      if (!*abort_s) atomicOr(a.err, 1u);
      *abort_s = 1;
    }
    __syncthreads();  // end of work
    if (*abort_s) {   // copies in flight must land before the CTA exits
      for (int v = 0; v < 2; ++v) {
        const int depth = v ? kCaStagesV : kCaStagesK;
        for (int k = max(0, fill[v] - depth); k < fill[v]; ++k)
          for (uint32_t it = 0; it < kSpinLimit && !mbar_try_wait(&kv_full[ca_stage(v, k)], (unsigned)((k / depth) & 1));)
            ++it;
      }
      for (int t = 0; t < 2; ++t)
        for (uint32_t it = 0; uses[t] && it < kSpinLimit && !mbar_try_wait(&q_full[t], (unsigned)((uses[t] - 1) & 1));)
          ++it;
    }
  } else {
    // ---- MMAs: warp 8 the products S, warp 10 the products P V
    const uint32_t q_base = smem_u32(sm), kv_base = q_base + kCaOffKv;
    const bool scores = warp == 8;
    const uint32_t tmem_u = tc_uniform(tmem);
    const int depth = scores ? kCaStagesK : kCaStagesV;
    int j = 0;               // K or V tiles consumed so far
    int seen[2] = {0, 0};    // warp 8: Q tiles, warp 10: P tiles consumed so far
    int si = 0;
    CaPiece c;
    for (int r = 0; ca_piece(a, sm + kCaOffRec, total, heads, per, r, c); ++r) {
      if (__any_sync(~0u, *abort_s)) break;
      const int tiles = c.two ? 2 : 1;
      const uint32_t idesc = tc_uniform(ca_idesc<DT>(!scores, c.p.n_tok * g <= kCaFewRows ? 64 : 128));
      // rows of V that no query row of the piece may see
      const int before = window > 0 ? c.p.first_end - window : 0;
      for (int i = 0; i < c.n; ++i, ++j) {
        const int s = ca_stage(!scores, j);
        tc_wait_on(&kv_full[s], (unsigned)((j / depth) & 1), abort_s, a.err);
        if (scores) {
          for (int t = 0; t < tiles; ++t) {
            if (i == 0) tc_wait_on(&q_full[t], (unsigned)(seen[t]++ & 1), abort_s, a.err);
            if (si > 0) tc_wait_on(s_free, (unsigned)((si - 1) & 1), abort_s, a.err);
            ++si;
            tc_fence_after();
            const uint32_t qa = tc_uniform(tc_desc_k(q_base + t * kCaTile));
            const uint32_t kb = tc_uniform(tc_desc_k(kv_base + s * kCaTile));
            const uint32_t full = tc_uniform(smem_u32(&s_full[t]));
            if (tc_elect()) {
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const uint32_t o = ((k >> 2) * kCaHalf + (k & 3) * 32) >> 4;
                tc_mma_ss(tmem_u, tc_desc(qa + o), tc_desc(kb + o), idesc, k > 0);
              }
              tc_commit(full);
              if (i + 1 == c.n) tc_commit(smem_u32(&q_empty[t]));
            }
          }
        } else {
          const int key0 = (c.p.kt0 + i) * 128, hi = min(128, c.p.kv_len - key0), lo = min(128, max(0, before - key0));
          if (hi < 128 || lo > 0) {
            unsigned char *vs = sm + kCaOffKv + s * kCaTile;
            for (int e = lane; e < 128 * 16; e += 32) {
              const int row = e >> 4;
              if (row < lo || row >= hi)
                *reinterpret_cast<uint4 *>(vs + (e & 8 ? kCaHalf : 0) + row * 128 + (e & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
          for (int t = 0; t < tiles; ++t) {
            const uint32_t vb = tc_uniform(ca_desc_mn(kv_base + s * kCaTile)), add = tc_uniform(i > 0 ? 1u : 0u);
            const uint32_t pa = tc_uniform(tmem + 128 + t * 64), oa = tc_uniform(tmem + 256 + t * 128);
            const uint32_t done = tc_uniform(smem_u32(&pv_done[t]));
            // in two halves of the keys: the first weights are multiplied while the others are formed
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              tc_wait_on(&p_full[2 * t + half], (unsigned)(seen[t] & 1), abort_s, a.err);
              tc_fence_after();
              if (tc_elect()) {
#pragma unroll
                for (int k = 4 * half; k < 4 * half + 4; ++k)
                  ca_mma_ts(oa, pa + k * 8, tc_desc(vb + k * (2048 >> 4)), idesc, k > 0 ? 1u : add);
                if (half) tc_commit(done);
              }
            }
            ++seen[t];
          }
        }
        __syncwarp();
        if (tc_elect()) tc_commit(smem_u32(&kv_empty[s]));
      }
    }
    // every MMA, and the arrivals that its commits owe, before the tensor memory is freed and the CTA ends
    uint64_t *bar = &drained[scores ? 0 : 1];
    __syncwarp();
    if (tc_elect()) tc_commit(smem_u32(bar));
    for (uint32_t it = 0; it < kSpinLimit && !mbar_try_wait(bar, 0);) ++it;
    __syncthreads();
  }
  } else {
    // ---- softmax: warpgroup t, a row per thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int t = warp >> 2, wrow = (warp & 3) * 32, row = wrow + lane;
    const uint32_t s_addr = tmem + ((uint32_t)wrow << 16), p_addr = s_addr + 128 + t * 64, o_addr = s_addr + 256 + t * 128;
    const int tok_in = row / g;               // token of the row within its tile
    const int tok = t * tpt + tok_in;         // ... within the item
    const int tok_a = t * tpt + wrow / g, tok_b = t * tpt + min(tpt - 1, (wrow + 31) / g);
    int sn = 0, on = 0;                       // S tiles and P V products seen so far
    const uint64_t to2 = ca_pair(a.to_log2, a.to_log2);
    bool ok = true;
    CaPiece c;
    for (int r = 0; ok && ca_piece(a, sm + kCaOffRec, total, heads, per, r, c); ++r) {
      const int n_tok = min(tpt, c.p.n_tok - t * tpt);  // tokens of this tile
      if (n_tok <= 0) continue;
      const bool live = tok_in < n_tok, busy = wrow < n_tok * g;  // the row / the warp has something to do
      const int end = causal ? min(c.p.kv_len, c.p.first_end + tok) : c.p.kv_len;
      const int begin = window > 0 ? max(0, c.p.first_end + tok - window) : 0;
      const int end_a = causal ? min(c.p.kv_len, c.p.first_end + tok_a) : c.p.kv_len;
      const int begin_b = window > 0 ? max(0, c.p.first_end + tok_b - window) : 0;
      float mc = live ? kLowest : INFINITY, l = 0.0f;  // running maximum in log2 units (rows without a query: weights 0), sum
      for (int i = 0; i < c.n; ++i, ++sn) {
        ok = tc_wait_warp(&s_full[t], (unsigned)(sn & 1), abort_s);
        if (!ok) break;
        if (busy) {
          tc_fence_after();
          float s[128];
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_ld32(s_addr + k * 32, s + k * 32);
          tc_wait_ld();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) tc_arrive(s_free);
          const int k0 = (c.p.kt0 + i) * 128;
          if (__builtin_expect(k0 + 128 > end_a || k0 < begin_b, 0)) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t sees = ca_below(end - k0 - 32 * w) & ~ca_below(begin - k0 - 32 * w);
#pragma unroll
              for (int k = 0; k < 32; ++k) s[w * 32 + k] = sees & (1u << k) ? s[w * 32 + k] : -INFINITY;
            }
          }
          float mx[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) mx[u] = ca_max3(s[u], s[8 + u], s[16 + u]);
#pragma unroll
          for (int k = 24; k < 120; k += 16) {
#pragma unroll
            for (int u = 0; u < 8; ++u) mx[u] = ca_max3(mx[u], s[k + u], s[k + 8 + u]);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) mx[u] = ca_max3(mx[u], s[120 + u], s[124 + u]);
          mx[0] = ca_max3(mx[0], mx[4], mx[5]);
          mx[1] = ca_max3(mx[1], mx[6], mx[7]);
          // The maximum moves only in steps above 2^kLazy (and at the first key the row sees).  A NaN score makes
          // it NaN and with it the whole row; so does a score of +inf, by inf - inf.
          const float top = ca_max3(ca_max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * a.to_log2;
          // (Of a piece multiplied as M = 64 the other rows' S is left over from anything.)
          const bool grow = live && !(top <= mc + kLazy);
          // P V of the tile before: whether it is through is asked ahead of the place that needs to know
          bool before = i > 0, seen_pv = !before || ca_test(&pv_done[t], (unsigned)(on & 1));
          if (__builtin_expect(i > 0 && __any_sync(~0u, grow), 0)) {
            ok = tc_wait_warp(&pv_done[t], (unsigned)(on & 1), abort_s);
            if (!ok) break;
            ++on;
            before = false;
            seen_pv = true;
            tc_fence_after();
            const float f = grow ? ca_exp2(mc - top) : 1.0f;
            l *= f;
#pragma unroll 1
            for (int k = 0; k < 8; ++k) {
              float o[16];
              tc_ld16(o_addr + k * 16, o);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = f == 0.0f ? 0.0f : o[e] * f;
              ca_st16(o_addr + k * 16, reinterpret_cast<const uint32_t *>(o));
            }
          }
          if (grow) mc = top;
          const uint64_t add2 = ca_pair(kShift - mc, kShift - mc);
          // A pair of weights per step: scale and shift kAhead pairs ahead of the exponentials, rounding
          // and sum kBehind pairs after them, so that the special function unit is fed without a pause.
          constexpr int kAhead = 4, kBehind = 4;
          uint64_t x[64];
          uint64_t sums[4] = {0, 0, 0, 0};
          uint32_t pk[64];
#pragma unroll
          for (int e = -kAhead; e < 64 + kBehind; ++e) {
            const int f = e + kAhead, b = e - kBehind;
            if (f >= 0 && f < 64) x[f] = ca_fma2(ca_pair(s[2 * f], s[2 * f + 1]), to2, add2);
            if (e >= 0 && e < 64) x[e] = ca_exp2_sfu(x[e]);
            if (b >= 0) {
              pk[b] = ca_pack<DT>(ca_lo(x[b]), ca_hi(x[b]));
              sums[b & 3] = ca_add2(sums[b & 3], x[b]);
            }
            if (b == 31) {
              // P is free once P V of the tile before has read it
              if (!__all_sync(~0u, seen_pv)) {
                ok = tc_wait_warp(&pv_done[t], (unsigned)(on & 1), abort_s);
                if (!ok) break;
              }
              on += before;
              tc_fence_after();
              ca_st16(p_addr, pk);
              ca_st16(p_addr + 16, pk + 16);
            }
            if (b == 47) {  // the first half's stores have had 16 pairs to land
              ca_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) tc_arrive(&p_full[2 * t]);
              ca_st16(p_addr + 32, pk + 32);
            }
            if (b == 63) ca_st16(p_addr + 48, pk + 48);
          }
          if (!ok) break;
          const uint64_t sum = ca_add2(ca_add2(sums[0], sums[1]), ca_add2(sums[2], sums[3]));
          l += ca_lo(sum) + ca_hi(sum);
          ca_wait_st();
          tc_fence_before();
        } else {
          if (lane == 0) tc_arrive(s_free);
          if (i == 0) {  // no query in the warp's rows: weights 0
            const uint32_t zero[16] = {};
#pragma unroll 1
            for (int k = 0; k < 4; ++k) ca_st16(p_addr + k * 16, zero);
            ca_wait_st();
            tc_fence_before();
          }
          if (i > 0) {
            ok = tc_wait_warp(&pv_done[t], (unsigned)(on & 1), abort_s);
            if (!ok) break;
            ++on;
          }
          if (lane == 0) tc_arrive(&p_full[2 * t]);
        }
        __syncwarp();
        if (lane == 0) tc_arrive(&p_full[2 * t + 1]);
      }
      if (!ok) break;
      // ---- the piece's rows
      if (c.n > 0) {
        ok = tc_wait_warp(&pv_done[t], (unsigned)(on & 1), abort_s);
        if (!ok) break;
        ++on;
      }
      if (!busy) continue;
      // a row that saw a key has a weight of 2^kShift at least
      const bool none = l < 1.0f;
      tc_fence_after();
      const int64_t token = (int64_t)c.p.q_start + tok;
      const int hq = c.head * g + row - tok_in * g;
      const bool store = live && token >= 0 && token < a.n_tokens;
      if (c.p.part >= 0) {
        const int64_t pr = (int64_t)c.head * h.part_rows + c.p.part + t * tpt * g + row;
#pragma unroll 1
        for (int k = 0; k < 4; ++k) {
          float o[32];
          tc_ld32(o_addr + k * 32, o);
          tc_wait_ld();
          if (live) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              ca_store32(a.part_o + pr * kD + k * 32 + e * 8, reinterpret_cast<const uint32_t *>(o + e * 8));
          }
        }
        if (live) *reinterpret_cast<float2 *>(a.part_ml + pr * 2) = make_float2(mc - kShift, none ? 0.0f : l);
      } else {
        const float inv = 1.0f / l;
        uint16_t *dst = static_cast<uint16_t *>(a.out) + (token * a.n_q + hq) * kD;
#pragma unroll 1
        for (int k = 0; k < 4; ++k) {
          float o[32];
          if (c.n > 0) {
            tc_ld32(o_addr + k * 32, o);
            tc_wait_ld();
          }
          if (store) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t w[8];
#pragma unroll
              for (int u = 0; u < 8; ++u) {
                const float x = o[e * 16 + 2 * u], y = o[e * 16 + 2 * u + 1];
                w[u] = none ? 0u : ca_pack<DT>(x * inv, y * inv);
              }
              ca_store32(dst + k * 32 + e * 16, w);
            }
          }
        }
        if (store && a.lse) a.lse[token * a.n_q + hq] = none ? -INFINITY : (mc - kShift + log2f(l)) * kLn2;
      }
      // the next piece's first P V overwrites O: it waits for p_full, which this warp arrives at later
      tc_fence_before();
    }
    if (!ok && lane == 0) {
      if (!*abort_s) atomicOr(a.err, 1u);
      *abort_s = 1;
    }
    __syncthreads();
  }
  // every role is past its last access to the tensor memory (or drained after an abort)
  tc_fence_after();
  __syncwarp();
  if (warp == 8)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCaTmemCols));
}

// Joins the partial rows of cut items in the order of their pieces: a warp per
// row.  Lane k first fetches maximum and sum of piece k (and k + 32, ...), so
// that all weights exist before a value is needed; then lane l adds up channels
// 4l .. 4l + 3, eight pieces' loads at a time.  (One piece after the other, each
// waiting for its maximum and then its values: 15 us for 8 rows x 16 pieces.)
template <int DT>
__global__ void __launch_bounds__(256) chunk_join_kernel(const ChunkArgs a) {
  griddep_wait();
  griddep_launch();
  const PlanHeader &h = *a.hdr;
  if (!ca_plan_fits(h, a)) return;
  const PlanSplit *splits = plan_splits(a.hdr, a.n_tokens, a.batch, a.n_q, a.n_kv);
  const int lane = threadIdx.x & 31, g = a.n_q / a.n_kv, rows = 2 * (kPlanRows / g) * g;
  const int heads = h.even ? 1 : a.n_kv;  // KV heads that a split stands for
  const int units = h.n_splits * heads * rows;  // (splits have workspace rows each, of which there are 75776)
  for (int u = blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += gridDim.x * 8) {
    const int sh = u / rows, row = u - sh * rows, e = sh / heads;
    PlanSplit sp = splits[e];
    const int head = sh - e * heads + (sp.n_tok >> 16);
    sp.n_tok &= 0xffff;
    if (row >= sp.n_tok * g) continue;
    const int64_t r0 = h.even ? sp.part + row : (int64_t)head * h.part_rows + sp.part + row;
    const int64_t r1 = (h.even ? plan_even_row(sp.part, 1) + row : r0 + sp.n_tok * g);  // piece 1; then equal steps
    const int64_t step = h.even ? 4 * kPlanRows : sp.n_tok * g;
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < sp.n_pieces; k0 += 32) {
      const int k = k0 + lane;
      const int64_t r = k == 0 ? r0 : r1 + (k - 1) * step;
      const float2 ml = k < sp.n_pieces ? *reinterpret_cast<const float2 *>(a.part_ml + r * 2) : make_float2(0.0f, 0.0f);
      // (a piece in which the row sees nothing has the sum 0)
      const float mn = fmaxf(m, warp_max(ml.y != 0.0f ? ml.x : -INFINITY));
      const float f = ml.y != 0.0f ? exp2f(ml.x - mn) : 0.0f;
      const float old = m == -INFINITY ? 0.0f : exp2f(m - mn);
      m = mn;
      l = l * old + warp_sum(f * ml.y);
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] *= old;
      const int n = min(32, sp.n_pieces - k0);
#pragma unroll 8
      for (int j = 0; j < n; ++j) {
        const float w = __shfl_sync(0xffffffffu, f, j);
        const int64_t rj = k0 + j == 0 ? r0 : r1 + (k0 + j - 1) * step;
        const float4 x = *reinterpret_cast<const float4 *>(a.part_o + rj * kD + lane * 4);
        o[0] += w != 0.0f ? w * x.x : 0.0f;
        o[1] += w != 0.0f ? w * x.y : 0.0f;
        o[2] += w != 0.0f ? w * x.z : 0.0f;
        o[3] += w != 0.0f ? w * x.w : 0.0f;
      }
    }
    const int64_t token = (int64_t)sp.q_start + row / g;
    const int hq = head * g + row % g;
    if (token < 0 || token >= a.n_tokens) continue;
    const float inv = 1.0f / l;
    uint2 w = make_uint2(ca_pack<DT>(o[0] * inv, o[1] * inv), ca_pack<DT>(o[2] * inv, o[3] * inv));
    if (l == 0.0f) w = make_uint2(0u, 0u);
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + (token * a.n_q + hq) * kD + lane * 4) = w;
    if (a.lse && lane == 0) a.lse[token * a.n_q + hq] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
  }
}

// ------------------------------------------------------------------- host ----

struct ChunkCall {
  const void *q, *k, *v;
  int64_t q_stride;
  ChunkArgs a;
  CUtensorMap mq, mq1, mk, mv;  // mq1: q one token at a time
};

static int chunk_check(const char *fn, ChunkCall &c, int dtype, int d, float scale, const void *plan,
                       size_t plan_bytes, void *workspace, size_t workspace_bytes) {
  ChunkArgs &a = c.a;
  KVR_REQUIRE(c.q && c.k && c.v && a.out && plan && workspace, "%s: null pointer", fn);
  if (d != kD) return set_error(KVR_ENOTSUP, "%s: head_dim must be 128", fn);
  if (dtype != KVR_F16 && dtype != KVR_BF16) return set_error(KVR_ENOTSUP, "%s: fp16 or bf16", fn);
  KVR_REQUIRE(a.n_kv > 0 && a.n_q > 0 && a.n_q % a.n_kv == 0, "%s: n_q must be a multiple of n_kv", fn);
  if (a.n_q / a.n_kv > kPlanRows)
    return set_error(KVR_ENOTSUP, "%s: more than %d query heads per KV head", fn, kPlanRows);
  KVR_REQUIRE(a.batch >= 1 && a.batch <= kPlanMaxBatch, "%s: batch must be in [1, %d]", fn, kPlanMaxBatch);
  KVR_REQUIRE(a.n_tokens >= 0 && a.n_tokens <= kPlanMaxTokens, "%s: bad token count", fn);
  KVR_REQUIRE(c.q_stride >= (int64_t)a.n_q * d && c.q_stride % 8 == 0,
              "%s: a token's heads must be contiguous, rows 16-byte aligned", fn);
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(c.q) | reinterpret_cast<uintptr_t>(c.k) |
                         reinterpret_cast<uintptr_t>(c.v) | reinterpret_cast<uintptr_t>(a.out) |
                         reinterpret_cast<uintptr_t>(plan);
  KVR_REQUIRE((ptrs & 15) == 0, "%s: pointers must be 16-byte aligned", fn);
  KVR_REQUIRE((reinterpret_cast<uintptr_t>(a.out) & 31) == 0, "%s: out must be 32-byte aligned", fn);
  KVR_REQUIRE(plan_bytes >= kvr_attn_plan_bytes(a.n_tokens, a.batch, a.n_q, a.n_kv), "%s: plan too small", fn);
  KVR_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "%s: workspace alignment", fn);
  const size_t need = kvr_attn_workspace_bytes();
  KVR_REQUIRE(workspace_bytes >= need, "%s: workspace %zu < %zu bytes", fn, workspace_bytes, need);
  KVR_REQUIRE(scale == scale && scale <= 3.0e38f, "%s: bad scale", fn);
  a.to_log2 = kLog2e / (scale > 0.0f ? scale : sqrtf((float)d));
  a.hdr = static_cast<const PlanHeader *>(plan);
  a.err = static_cast<unsigned *>(workspace);
  a.part_o = reinterpret_cast<float *>(static_cast<char *>(workspace) + kWsHeader);
  a.part_ml = a.part_o + kD * (size_t)kPartRows;
  return KVR_OK;
}

// Bytes of `rows` rows of n_kv or n_q heads, `stride` elements apart.
static int64_t row_span(int64_t rows, int64_t stride, int64_t heads) { return ((rows - 1) * stride + heads * kD) * 2; }

// What a call writes must not lie in what it reads: rows are finished, and stored, while other CTAs still read.
static int chunk_check_out(const char *fn, const ChunkCall &c, int64_t k_bytes, int64_t v_bytes) {
  const ChunkArgs &a = c.a;
  auto meet = [](const void *p, int64_t n, const void *q, int64_t m) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q);
    return x < y + (uintptr_t)m && y < x + (uintptr_t)n;
  };
  const struct { const void *p; int64_t n; } w[2] = {{a.out, row_span(a.n_tokens, (int64_t)a.n_q * kD, a.n_q)},
                                                     {a.lse, a.n_tokens * a.n_q * 4}};
  for (const auto &o : w) {
    if (!o.p) continue;
    const char *name = o.p == a.out ? "out" : "lse";
    KVR_REQUIRE(!meet(o.p, o.n, c.q, row_span(a.n_tokens, c.q_stride, a.n_q)), "%s: %s must not be q or lie in it", fn, name);
    KVR_REQUIRE(!meet(o.p, o.n, c.k, k_bytes) && !meet(o.p, o.n, c.v, v_bytes), "%s: %s must not lie in the keys or values",
                fn, name);
  }
  KVR_REQUIRE(!a.lse || !meet(w[0].p, w[0].n, w[1].p, w[1].n), "%s: out and lse overlap", fn);
  return KVR_OK;
}

template <int DT, bool PAGED>
static cudaError_t chunk_kernels(const ChunkCall &c, int dev, cudaStream_t st) {
  static thread_local int set_dev = -1;
  if (set_dev != dev) {
    const cudaError_t e = cudaFuncSetAttribute(chunk_attn_kernel<DT, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               kCaSmem);
    if (e != cudaSuccess) return e;
    set_dev = dev;
  }
  const cudaError_t e = launch_dependent(chunk_attn_kernel<DT, PAGED>, kPlanCtas, kCaThreads, kCaSmem, st, c.mq, c.mq1,
                                         c.mk, c.mv, c.a);
  if (e != cudaSuccess) return e;
  return launch_dependent(chunk_join_kernel<DT>, kPlanCtas * 4, 256, 0, st, c.a);
}

static int chunk_launch(const char *fn, ChunkCall &c, int dtype, bool paged, kvr_stream_t stream) {
  const ChunkArgs &a = c.a;
  if (!encode_tiled()) return set_error(KVR_ECUDA, "%s: the driver has no cuTensorMapEncodeTiled", fn);
  const int g = a.n_q / a.n_kv, tpt = kPlanRows / g;
  // q as (64 channels, head of the group, token, channel half, KV head)
  const cuuint64_t qd[5] = {64, (cuuint64_t)g, (cuuint64_t)a.n_tokens, 2, (cuuint64_t)a.n_kv};
  const cuuint64_t qs[4] = {kD * 2, (cuuint64_t)c.q_stride * 2, 128, (cuuint64_t)g * kD * 2};
  const cuuint32_t qb[5] = {64, (cuuint32_t)g, (cuuint32_t)tpt, 1, 1};
  const cuuint32_t qb1[5] = {64, (cuuint32_t)g, 1, 1, 1};
  if (!make_map(&c.mq, dtype, c.q, 5, qd, qs, qb) || !make_map(&c.mq1, dtype, c.q, 5, qd, qs, qb1)) return set_error(KVR_EINVAL, "%s: q has a layout TMA cannot read", fn);
  int dev = 0;
  cudaGetDevice(&dev);
  cudaError_t e;
  cudaStream_t st = as_cuda(stream);
  if (dtype == KVR_F16) e = paged ? chunk_kernels<KVR_F16, true>(c, dev, st) : chunk_kernels<KVR_F16, false>(c, dev, st);
  else e = paged ? chunk_kernels<KVR_BF16, true>(c, dev, st) : chunk_kernels<KVR_BF16, false>(c, dev, st);
  if (e != cudaSuccess) return set_error(KVR_ECUDA, "%s: %s", fn, cudaGetErrorString(e));
  return check_launch(fn);
}

}  // namespace kvr

using namespace kvr;

extern "C" size_t kvr_attn_workspace_bytes(void) {
  return kWsHeader + (size_t)kPartRows * (kD + 2) * sizeof(float);
}

extern "C" int kvr_paged_attn(const void *q, int dtype, int64_t n_tokens, int batch, int n_q, int n_kv, int d,
                              int64_t q_stride, const void *k_pages, const void *v_pages, int64_t n_pages, int page,
                              int64_t page_stride, int64_t tok_stride, const int32_t *block_table,
                              int64_t table_stride, int table_width, const void *plan, size_t plan_bytes, float scale,
                              void *out, float *lse, void *workspace, size_t workspace_bytes, kvr_stream_t stream) {
  clear_error();
  if (n_tokens == 0) return KVR_OK;
  ChunkCall c{};
  c.q = q; c.k = k_pages; c.v = v_pages;
  c.q_stride = q_stride;
  ChunkArgs &a = c.a;
  a.n_tokens = n_tokens;
  a.n_q = n_q; a.n_kv = n_kv; a.batch = batch;
  a.page = page; a.n_pages = (int)n_pages;
  a.table = block_table; a.table_stride = table_stride; a.table_width = table_width;
  a.out = out; a.lse = lse;
  const int rc = chunk_check("kvr_paged_attn", c, dtype, d, scale, plan, plan_bytes, workspace, workspace_bytes);
  if (rc) return rc;
  KVR_REQUIRE(block_table && table_width >= 1 && table_stride >= table_width, "kvr_paged_attn: bad block table");
  KVR_REQUIRE(n_pages > 0 && n_pages < INT_MAX, "kvr_paged_attn: bad page pool");
  if (page < 8 || page % 8 != 0 || page > (1 << 20))
    return set_error(KVR_ENOTSUP, "kvr_paged_attn: the page size must be a multiple of 8 tokens");
  KVR_REQUIRE(tok_stride >= (int64_t)n_kv * d && tok_stride % 8 == 0 && page_stride >= 0 && page_stride % 8 == 0,
              "kvr_paged_attn: a token's heads must be contiguous, rows 16-byte aligned");
  const int64_t pool = row_span(n_pages, page_stride, 0) + row_span(page, tok_stride, n_kv);
  const int bad = chunk_check_out("kvr_paged_attn", c, pool, pool);
  if (bad) return bad;
  bind_context();
  a.box = 128;
  while (page % a.box) a.box /= 2;
  // the pool as (64 channels, row of the page, channel half, KV head, page)
  const cuuint64_t kd[5] = {64, (cuuint64_t)page, 2, (cuuint64_t)n_kv, (cuuint64_t)n_pages};
  const cuuint64_t ks[4] = {(cuuint64_t)tok_stride * 2, 128, kD * 2, (cuuint64_t)page_stride * 2};
  const cuuint32_t kb[5] = {64, (cuuint32_t)a.box, 1, 1, 1};
  if (!encode_tiled() || !make_map(&c.mk, dtype, k_pages, 5, kd, ks, kb) || !make_map(&c.mv, dtype, v_pages, 5, kd, ks, kb))
    return set_error(KVR_EINVAL, "kvr_paged_attn: the pool has a layout TMA cannot read");
  return chunk_launch("kvr_paged_attn", c, dtype, true, stream);
}

extern "C" int kvr_prompt_attn(const void *q, const void *k, const void *v, int dtype, int64_t n_tokens,
                               int64_t n_keys, int batch, int n_q, int n_kv, int d, int64_t q_stride, int64_t k_stride,
                               int64_t v_stride, const void *plan, size_t plan_bytes, float scale, void *out,
                               float *lse, void *workspace, size_t workspace_bytes, kvr_stream_t stream) {
  clear_error();
  if (n_tokens == 0) return KVR_OK;
  ChunkCall c{};
  c.q = q; c.k = k; c.v = v;
  c.q_stride = q_stride;
  ChunkArgs &a = c.a;
  a.n_tokens = n_tokens;
  a.n_q = n_q; a.n_kv = n_kv; a.batch = batch;
  a.out = out; a.lse = lse;
  const int rc = chunk_check("kvr_prompt_attn", c, dtype, d, scale, plan, plan_bytes, workspace, workspace_bytes);
  if (rc) return rc;
  KVR_REQUIRE(n_keys > 0 && n_keys <= kPlanMaxLen, "kvr_prompt_attn: bad key count");
  KVR_REQUIRE(k_stride >= (int64_t)n_kv * d && v_stride >= (int64_t)n_kv * d && (k_stride | v_stride) % 8 == 0,
              "kvr_prompt_attn: a token's heads must be contiguous, rows 16-byte aligned");
  const int bad = chunk_check_out("kvr_prompt_attn", c, row_span(n_keys, k_stride, n_kv), row_span(n_keys, v_stride, n_kv));
  if (bad) return bad;
  bind_context();
  // k and v as (64 channels, token, channel half, KV head)
  const cuuint64_t kd[4] = {64, (cuuint64_t)n_keys, 2, (cuuint64_t)n_kv};
  const cuuint64_t ks[3] = {(cuuint64_t)k_stride * 2, 128, kD * 2}, vs[3] = {(cuuint64_t)v_stride * 2, 128, kD * 2};
  const cuuint32_t kb[4] = {64, 128, 2, 1};
  if (!encode_tiled() || !make_map(&c.mk, dtype, k, 4, kd, ks, kb) || !make_map(&c.mv, dtype, v, 4, kd, vs, kb))
    return set_error(KVR_EINVAL, "kvr_prompt_attn: k or v has a layout TMA cannot read");
  return chunk_launch("kvr_prompt_attn", c, dtype, false, stream);
}
