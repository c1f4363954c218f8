// A sparse MLP ("mixture of experts") of a few tokens.
//
//   z = x Wr^T (E logits a token), p = softmax(z), the top_k largest p_e with
//   weights w_e = scale p_e (or scale p_e / sum of the chosen p),
//   y = sum_e w_e Wd_e (silu(Wg_e x) * (Wu_e x)).
//
// With up to 128 tokens the weights of the chosen experts, 6 H I bytes each, are
// what has to be read; a token's share of the arithmetic is small.  So the weights
// are streamed once, and the tokens ride along.  Two kernels:
//
// moe_route_kernel: clusters of 8 CTAs take 1 to 8 tokens; a CTA forms the logits of an
// eighth of the experts, the cluster exchanges them over distributed shared memory,
// and CTA r ranks token r's.  Logits are sums of exact products, 32-bit partial sums
// per lane joined in 64 bits: the last expert chosen and the first left out can lie
// close together.
//
// moe_experts_kernel: one CTA per SM, with the experts' weights as the M side of
// tcgen05.mma (rows of a weight tile) and the tokens as the N side, so that an MMA costs
// little more than its weights' bytes and a few tokens leave no rows empty that memory
// would have to fill.  Segments are an expert's tokens, at most `cols` of them.
// Work units, taken in order from one ticket counter:
//   gate/up  R1 rows (16 of gate, 16 of up, ...) of a segment's expert over x: h, in two
//            16-bit parts
//   down     R2 rows of Wd over a share of both parts of h: partial rows (token, choice,
//            share) in 32 bits
//   sum      128 columns of y of some tokens: choices and shares of each token in order
// A unit waits only for units with lower tickets, which run already: no CTA has to
// be resident for another to end.  Weights of a down unit stream in while its h is
// still being formed, so the memory does not idle between the phases.
//   warp 0  tickets, weight tiles by TMA (128-byte swizzle) into a ring of stages
//   warps 1, 3  token rows into the same stages, 16 bytes a lane, swizzled by hand
//   warp 2  tcgen05.mma, accumulators of two units in tensor memory
//   warps 4-7  epilogues of 32 rows each; sums
//
// Both operands of an MMA are of one 16-bit type, so h has to be rounded for the
// second product.  It goes in as two columns, h rounded and what the rounding left:
// 16 bits of it in bf16, in fp16 22 of an h from 1/8 up, and below that what is left to
// the smallest step, 2^-24 (18 bits at 0.01), for copies and columns that the few tokens leave room for.  (Rounded once, y was 1.4 to 1.6 times as far from 64 bits as its own
// rounding makes it.)  Sums, router weights and partial rows are fp32.
//
// What binds: HBM where the weights are many.  128 tokens over 128 experts of 4096 x 1408
// (4.4 GB): 664 us in a graph, 6.7 TB/s, a plain copy's rate (708 back to back for seconds, under the
// power cap); 32 over 8 experts of 4096 x 14336 443.  One token, 8 of 128 experts of 2048 x 768 (75
// MB, 12 us of reading): 27 us, the rest a chain of round trips: logits and ranks (4), lists
// (1), a first tile's way from memory (2), h through a counter and L2 (3), last products, partial
// rows and sums (6).  With many tokens an expert their rows cross L2 as often as the weights: 69 tokens over 4 of
// 4 experts of 1128 x 13776 110 us, of which 57 are the weights'; 128 over 6 of 8 of 720 x 888 63, of 5.
//
// Waits are bounded; one that gives up sets the status word, lets copies and MMAs in
// flight end and frees the tensor memory.
#include "kvr_tcgen05.cuh"

namespace kvr {

constexpr int kMoMaxTokens = 128, kMoMaxExperts = 512, kMoMaxTopK = 16;
constexpr int kMoMaxPicks = kMoMaxTokens * kMoMaxTopK;
constexpr int kMoSms = 148;

// ------------------------------------------------------------------ router ----

constexpr int kMrThreads = 256, kMrCluster = 8, kMrMaxTokens = 8, kMrExperts = 4;

struct RouteArgs {
  const void *x, *router;
  int64_t x_stride, router_stride;
  int tokens, hidden, experts, top_k, norm;
  float scale;
  int *ids;
  float *weights;
  int *counters;  // cleared for the second kernel
  int n_counters;
};

__device__ __forceinline__ void mo_cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ double mo_peer_double(const double *p, unsigned rank) {
  uint32_t a;
  double v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(a) : "memory");
  return v;
}
// Order-preserving map double -> uint64; NaN below everything, never 0.
__device__ __forceinline__ uint64_t mo_key(double z) {
  if (z != z) return 1;
  const uint64_t u = (uint64_t)__double_as_longlong(z == 0.0 ? 0.0 : z);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

template <int DT>
__device__ __forceinline__ void mo_widen(const uint4 &u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (DT == KVR_BF16) {
      x[2 * j] = __uint_as_float(w[j] << 16);
      x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
      x[2 * j] = f.x;
      x[2 * j + 1] = f.y;
    }
  }
}

// NT tokens a cluster: as few as the SMs have clusters for, since a CTA's time is its tokens' products.  (From four on,
// registers for two CTAs an SM: 16 clusters of 8 do not fit the GPCs one CTA an SM, and the last one came 13 us late.)
template <int DT, int NT>
__global__ void __cluster_dims__(kMrCluster, 1, 1) __launch_bounds__(kMrThreads, NT < 4 ? 1 : 2) moe_route_kernel(RouteArgs a) {
  constexpr int kWarps = kMrThreads / 32;
  __shared__ double part[NT][kMoMaxExperts / kMrCluster];  // logits of this CTA's experts
  __shared__ double slice[kWarps][NT][kMrExperts];         // of a warp's channels
  __shared__ double all_s[kMoMaxExperts];                  // of this CTA's token
  __shared__ __align__(16) uint64_t key_s[kMoMaxExperts];
  __shared__ int chosen[kMoMaxTopK];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = blockIdx.x % kMrCluster, t0 = blockIdx.x / kMrCluster * NT;
  const int n_tok = min(NT, a.tokens - t0);
  griddep_wait();
  griddep_launch();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < a.n_counters; i += kMrThreads) a.counters[i] = 0;
  const int per = (a.experts + kMrCluster - 1) / kMrCluster, e0 = rank * per, n_exp = max(0, min(a.experts - e0, per));
  // A warp takes four experts over a part of the channels: what it loads of x serves four, of the router NT.
  const int groups = (n_exp + kMrExperts - 1) / kMrExperts, parts = groups > 0 && groups < kWarps ? kWarps / groups : 1;
  for (int g = warp / parts; g < groups; g += kWarps / parts) {
    float s[NT][kMrExperts] = {};
    const int c0 = warp % parts * 256 + lane * 8, dc = parts * 256;
    const uint16_t *w_row = static_cast<const uint16_t *>(a.router) + (e0 + g * kMrExperts) * a.router_stride;
    const uint16_t *x_row = static_cast<const uint16_t *>(a.x) + t0 * a.x_stride;
    int64_t w_off[kMrExperts], x_off[NT];  // (experts and tokens past the last: the last again, to no use)
#pragma unroll
    for (int e = 0; e < kMrExperts; ++e) w_off[e] = min(e, n_exp - 1 - g * kMrExperts) * a.router_stride;
#pragma unroll
    for (int t = 0; t < NT; ++t) x_off[t] = min(t, n_tok - 1) * a.x_stride;
#pragma unroll(NT == 1 ? 4 : 2)
    for (int c = c0; c < a.hidden; c += dc) {
      uint4 w[kMrExperts], x[NT];
#pragma unroll
      for (int e = 0; e < kMrExperts; ++e) w[e] = __ldg(reinterpret_cast<const uint4 *>(w_row + w_off[e] + c));
#pragma unroll
      for (int t = 0; t < NT; ++t) x[t] = __ldg(reinterpret_cast<const uint4 *>(x_row + x_off[t] + c));
      float wf[kMrExperts][8];
#pragma unroll
      for (int e = 0; e < kMrExperts; ++e) mo_widen<DT>(w[e], wf[e]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float xf[8];
        mo_widen<DT>(x[t], xf);
#pragma unroll
        for (int e = 0; e < kMrExperts; ++e)
#pragma unroll
          for (int j = 0; j < 8; ++j) s[t][e] = fmaf(xf[j], wf[e][j], s[t][e]);
      }
    }
    // The lanes' sums, in 64 bits: at each step a lane hands half of its values on and adds up the other half, so that
    // in the end it has one (or, of the last steps, all lanes the same).
    constexpr int kValues = NT * kMrExperts;
    double v[kValues];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < kMrExperts; ++e) v[t * kMrExperts + e] = s[t][e];
    int which = 0, n = kValues;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const bool upper = lane & o;
      if (n > 1) {
        n >>= 1;
        which = which * 2 + upper;
#pragma unroll
        for (int j = 0; j < kValues / 2; ++j)
          if (j < n) {
            const double send = upper ? v[j] : v[j + n];
            v[j] = (upper ? v[j + n] : v[j]) + __shfl_xor_sync(0xffffffffu, send, o);
          }
      } else {
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
      }
    }
    if ((lane & (32 / kValues - 1)) == 0) {
      const int t = which / kMrExperts, e = which % kMrExperts;
      if (parts > 1) slice[warp][t][e] = v[0];
      else if (g * kMrExperts + e < n_exp) part[t][g * kMrExperts + e] = v[0];
    }
  }
  if (parts > 1) {  // in the order of the channels
    __syncthreads();
    for (int i = threadIdx.x; i < NT * n_exp; i += kMrThreads) {
      const int t = i / n_exp, e = i - t * n_exp;
      double d = 0.0;
      for (int q = 0; q < parts; ++q) d += slice[e / kMrExperts * parts + q][t][e % kMrExperts];
      part[t][e] = d;
    }
  }
  mo_cluster_sync();
  // CTA r: token r.  An expert's rank is the number of those above it: larger logits, lower experts among equal ones.
  if (rank < n_tok) {
    const int even = (a.experts + 1) / 2 * 2;
    for (int e = threadIdx.x; e < even; e += kMrThreads) {
      const double z = e < a.experts ? mo_peer_double(&part[rank][e % per], e / per) : 0.0;
      all_s[e] = z;
      key_s[e] = e < a.experts ? mo_key(z) : 0;
    }
    __syncthreads();
    int each = 1;  // threads that share an expert's count
    while (each < 32 && a.experts * each * 2 <= kMrThreads) each *= 2;
    for (int e0 = 0; e0 < a.experts; e0 += kMrThreads / each) {
      const int e = e0 + threadIdx.x / each;
      const uint64_t mine = e < a.experts ? key_s[e] : 0;
      int above = 0;
#pragma unroll 4
      for (int o = threadIdx.x % each * 2; o < even; o += 2 * each) {
        const ulonglong2 k = *reinterpret_cast<const ulonglong2 *>(&key_s[o]);
        above += (k.x > mine || (k.x == mine && o < e)) + (k.y > mine || (k.y == mine && o + 1 < e));
      }
      for (int o = 1; o < each; o <<= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
      if (e < a.experts && threadIdx.x % each == 0 && above < a.top_k) chosen[above] = e;
    }
    __syncthreads();
    if (warp == 0) {
      const double m = all_s[chosen[0]];  // (a NaN only where all are)
      float all = 0.0f;
      for (int e = lane; e < a.experts; e += 32) all += expf((float)(all_s[e] - m));
      all = warp_sum(all);
      const float w = lane < a.top_k ? expf((float)(all_s[chosen[lane]] - m)) : 0.0f, sum = warp_sum(w);
      if (lane < a.top_k) {
        const int64_t o = (int64_t)(t0 + rank) * a.top_k + lane;
        a.ids[o] = chosen[lane];
        // a logit that is no number, or infinite, leaves no weight that means anything
        a.weights[o] = all < INFINITY ? a.scale * w / (a.norm ? sum : all) : NAN;
      }
    }
  }
  mo_cluster_sync();  // the other CTAs' logits stay until they are read
}

// ----------------------------------------------------------------- experts ----

constexpr int kMoThreads = 256;
constexpr int kMoMaxStages = 16, kMoSched = 4;
constexpr uint32_t kMoRing = 204 * 1024;   // stages, and what an MMA reads past the last: 128 rows from a tile's start
constexpr uint32_t kMoTmemCols = 512;      // two accumulators of up to 256 columns
constexpr int kMoMinCols = 16;
constexpr int kMoMaxSegs = kMoMaxExperts + kMoMaxPicks / kMoMinCols;
constexpr int kMoSumCols = 128;            // columns of y of a sum unit

struct ExpertArgs {
  int tokens, hidden, inter, experts, top_k;
  int rows1, rows2;      // rows of a gate/up and of a down unit
  int kb1, kb2;          // 64-column blocks of a stage
  int cols, cols2;       // columns of a gate/up unit (most tokens of a segment) and of a down unit, multiples of 16
  int shares;            // of an expert's inner channels in down units
  int sum_tokens;        // tokens of a sum unit
  int stages;
  uint32_t stage_bytes, a_bytes;  // of a stage; its weights' part
  const void *x;
  int64_t x_stride;
  const int *ids;
  const float *weights;
  void *h;               // (tokens * top_k, 2, inter): rounded, rest
  float *part;           // (tokens * top_k, shares, hidden)
  void *y;
  int *counters;         // ticket; warps' parts of segments' gate/up units done; segments done of 32-row strips of y
  unsigned *err;
};

struct MoShared {
  uint64_t full_a[kMoMaxStages], full_b[kMoMaxStages], empty[kMoMaxStages];
  uint64_t acc_full[2], acc_empty[2], sched_full[kMoSched], sched_empty[kMoSched], drained;
  uint32_t tmem;
  int abort_s;
  int sched[kMoSched];
  int n_segs;
  int warp_sums[2][kMoThreads / 32];
  int seg_expert[kMoMaxSegs];
  short seg_first[kMoMaxSegs], seg_n[kMoMaxSegs];
  short first[kMoMaxExperts];
  short picks[kMoMaxPicks];  // token * top_k + choice, by expert
  float weights[kMoMaxPicks];
  uint32_t rows[2][2 * kMoMaxTokens];  // where x's or h's are, in 16 bytes, of the unit that a copying warp is at
};

__device__ __forceinline__ void mo_tma4(uint32_t dst, const CUtensorMap *m, int c0, int c1, int c2, int c3, uint32_t bar,
                                        uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, "
      "%4, %5}], [%6], %7;" ::"r"(dst),
      "l"(m), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void mo_tma3(uint32_t dst, const CUtensorMap *m, int c0, int c1, int c2, uint32_t bar,
                                        uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, "
      "%4}], [%5], %6;" ::"r"(dst),
      "l"(m), "r"(c0), "r"(c1), "r"(c2), "r"(bar), "l"(policy)
      : "memory");
}
// 16 bytes (zeros where !there) past L1.
__device__ __forceinline__ void mo_copy16(uint32_t dst, const char *src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void mo_ld4(uint32_t taddr, float *f) {
  uint32_t *r = reinterpret_cast<uint32_t *>(f);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr));
}
__device__ __forceinline__ int mo_acquire(const int *p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
// After an abort: waits (not for long) for the copies of the last `filled` stages before stage `st`.
__device__ __forceinline__ void mo_drain(uint64_t *full, int st, unsigned parity, int filled, int stages) {
  for (; filled > 0; --filled) {
    if (--st < 0) {
      st = stages - 1;
      parity ^= 1;
    }
    mbar_wait_bounded(&full[st], parity ^ 1, 1u << 14);
  }
}
template <int DT>
__host__ __device__ constexpr uint32_t mo_idesc(uint32_t n) {  // kind::f16, fp32 accumulator, M 128
  return (1u << 4) | ((DT == KVR_BF16 ? 1u : 0u) << 7) | ((DT == KVR_BF16 ? 1u : 0u) << 10) | ((n >> 3) << 17) |
         ((128u >> 4) << 24);
}

// Work unit u: phase (0: gate/up, 1: down, 2: sum), segment (2: columns of y), tile of rows (2: tokens), and the
// 64-column blocks [b0, b1) of the weights.
struct MoUnit {
  int phase, seg, tile, share, b0, b1;
};
struct MoPlan {
  int segs, tiles1, tiles2, sums;  // sums: units of a column block
  int first2, first3, units;       // first down unit, first sum unit, all
  int blocks1, blocks2, shares;
};
__device__ __forceinline__ MoUnit mo_unit(const MoPlan &p, int u) {
  MoUnit w;
  w.share = w.b0 = w.b1 = 0;
  if (u < p.first2) {
    w.phase = 0;
    w.seg = u / p.tiles1;
    w.tile = u - w.seg * p.tiles1;
    w.b1 = p.blocks1;
  } else if (u < p.first3) {
    u -= p.first2;
    w.phase = 1;
    const int t = u / p.shares;
    w.share = u - t * p.shares;
    w.seg = t / p.tiles2;
    w.tile = t - w.seg * p.tiles2;
    w.b0 = p.blocks2 * w.share / p.shares;
    w.b1 = p.blocks2 * (w.share + 1) / p.shares;
  } else {
    u -= p.first3;
    w.phase = 2;
    w.seg = u / p.sums;
    w.tile = u - w.seg * p.sums;
  }
  return w;
}
// The part of a 16-bit type that a value rounds to, kept finite (the rest then holds up to as much again).
template <int DT>
__device__ __forceinline__ float mo_rounded(float x) {
  const float most = DT == KVR_F16 ? 65504.0f : 3.3895313892515355e38f;
  const float r = round_dt<DT>(x);
  return r > most ? most : r < -most ? -most : r;
}

template <int DT>
__global__ void __launch_bounds__(kMoThreads, 1)
    moe_experts_kernel(const __grid_constant__ CUtensorMap mw1, const __grid_constant__ CUtensorMap mw2, const ExpertArgs a) {
  extern __shared__ __align__(1024) unsigned char sm[];
  MoShared &s = *reinterpret_cast<MoShared *>(sm + kMoRing);
  volatile int *abort_s = &s.abort_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem)),
                 "r"(kMoTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (tid == 32) {
    for (const CUtensorMap *m : {&mw1, &mw2}) asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
  }
  if (tid == 0) {
    s.abort_s = 0;
    for (int i = 0; i < a.stages; ++i) {
      tc_bar_init(&s.full_a[i], 1);
      tc_bar_init(&s.full_b[i], 32);  // a copying warp's lanes
      tc_bar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc_bar_init(&s.acc_full[i], 1);
      tc_bar_init(&s.acc_empty[i], 4);
    }
    for (int i = 0; i < kMoSched; ++i) {
      tc_bar_init(&s.sched_full[i], 1);
      tc_bar_init(&s.sched_empty[i], 7);  // two copying warps, MMA, four epilogue warps
    }
    tc_bar_init(&s.drained, 1);
  }
  // tokens of each expert, a bit each; where the stages will be
  unsigned (*mask)[kMoMaxTokens / 32] = reinterpret_cast<unsigned (*)[kMoMaxTokens / 32]>(sm);
  for (int i = tid; i < kMoMaxExperts * (kMoMaxTokens / 32); i += kMoThreads) (&mask[0][0])[i] = 0;
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // barriers: for the copies and commits
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem;
  griddep_wait();  // what follows reads the routing
  griddep_launch();
  int *ticket = a.counters, *seg_done = a.counters + 1, *strip_done = seg_done + kMoMaxSegs;
  int next = 0;  // (the first ticket, asked for while the lists are made)
  if (tid == 0) next = atomicAdd(ticket, 1);

  // picks by expert, and segments.  Every CTA makes the same lists.
  const int picks = a.tokens * a.top_k;
  if (picks <= 32) {  // by one warp, a pick per lane: no bits, no meetings (a token of 128 experts 28.2 -> 27.4 us)
    if (warp == 0) {
      const int id = lane < picks ? a.ids[lane] : -1;
      if (lane < picks) s.weights[lane] = a.weights[lane];
      const unsigned same = __match_any_sync(0xffffffffu, id);  // picks of the lane's expert
      const int lead = __ffs(same) - 1, n = id >= 0 && lead == lane ? __popc(same) : 0, n_s = (n + a.cols - 1) / a.cols;
      int at_n = n, at_s = n_s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int yn = __shfl_up_sync(0xffffffffu, at_n, o), ys = __shfl_up_sync(0xffffffffu, at_s, o);
        if (lane >= o) {
          at_n += yn;
          at_s += ys;
        }
      }
      if (lane == 31) s.n_segs = at_s;
      at_n -= n;
      at_s -= n_s;
      for (int c = 0; c < n; c += a.cols, ++at_s) {
        s.seg_expert[at_s] = id;
        s.seg_first[at_s] = (short)(at_n + c);
        s.seg_n[at_s] = (short)min(a.cols, n - c);
      }
      const int first = __shfl_sync(0xffffffffu, at_n, lead);
      if (id >= 0) s.picks[first + __popc(same & ((1u << lane) - 1))] = (short)lane;
    }
  } else {  // a bit per (expert, token), counts and prefix sums
    constexpr int kIds = kMoMaxPicks / kMoThreads;
    int id[kIds];
#pragma unroll
    for (int j = 0; j < kIds; ++j) {
      const int i = tid + j * kMoThreads;
      id[j] = i < picks ? a.ids[i] : -1;
      if (i < picks) s.weights[i] = a.weights[i];
    }
#pragma unroll
    for (int j = 0; j < kIds; ++j)
      if (id[j] >= 0) {
        const int t = (tid + j * kMoThreads) / a.top_k;
        atomicOr(&mask[id[j]][t >> 5], 1u << (t & 31));
      }
    __syncthreads();
    {
      constexpr int kEach = kMoMaxExperts / kMoThreads;
      int n[kEach], sum_n = 0, sum_s = 0;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const int e = tid * kEach + j;
        n[j] = 0;
#pragma unroll
        for (int w = 0; w < kMoMaxTokens / 32; ++w) n[j] += __popc(mask[e][w]);
        sum_n += n[j];
        sum_s += (n[j] + a.cols - 1) / a.cols;
      }
      int at_n = sum_n, at_s = sum_s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int yn = __shfl_up_sync(0xffffffffu, at_n, o), ys = __shfl_up_sync(0xffffffffu, at_s, o);
        if (lane >= o) {
          at_n += yn;
          at_s += ys;
        }
      }
      if (lane == 31) {
        s.warp_sums[0][warp] = at_n;
        s.warp_sums[1][warp] = at_s;
      }
      __syncthreads();
      at_n -= sum_n;
      at_s -= sum_s;
      for (int w = 0; w < warp; ++w) {
        at_n += s.warp_sums[0][w];
        at_s += s.warp_sums[1][w];
      }
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const int e = tid * kEach + j;
        s.first[e] = (short)at_n;
        for (int c = 0; c < n[j]; c += a.cols) {
          s.seg_expert[at_s] = e;
          s.seg_first[at_s] = (short)(at_n + c);
          s.seg_n[at_s] = (short)min(a.cols, n[j] - c);
          ++at_s;
        }
        at_n += n[j];
      }
      if (tid == kMoThreads - 1) s.n_segs = at_s;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kIds; ++j)
      if (id[j] >= 0) {
        const int i = tid + j * kMoThreads, t = i / a.top_k, e = id[j];
        int before = __popc(mask[e][t >> 5] & ((1u << (t & 31)) - 1));
        for (int w = 0; w < (t >> 5); ++w) before += __popc(mask[e][w]);
        s.picks[s.first[e] + before] = (short)i;
      }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // copies will write where the bits were
  __syncthreads();
  MoPlan p;
  p.segs = s.n_segs;
  p.tiles1 = (a.inter + a.rows1 / 2 - 1) / (a.rows1 / 2);
  p.tiles2 = (a.hidden + a.rows2 - 1) / a.rows2;
  p.sums = (a.tokens + a.sum_tokens - 1) / a.sum_tokens;
  p.first2 = p.segs * p.tiles1;
  p.blocks1 = (a.hidden + 63) / 64;
  p.blocks2 = (a.inter + 63) / 64;
  p.shares = a.shares;
  p.first3 = p.first2 + p.segs * p.tiles2 * a.shares;
  p.units = p.first3 + (a.hidden + kMoSumCols - 1) / kMoSumCols * p.sums;
  const uint32_t ring = smem_u32(sm);

  if (warp == 0) {
    // ---- tickets and weights.  The whole warp walks, one lane issues: a copy's operands lie in uniform registers, and
    // only of values that come from a shuffle or from the launch does the compiler know that they may (copies issued by
    // lane 0 alone, with its own ticket's numbers: 320 cycles each, not 60).  Stage and phase are counted up: divisions
    // made a stage cost more than its bytes take to arrive.  Weights are read once: first to leave L2, which h and the
    // partial rows need.
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    int st = 0, filled = 0;
    unsigned parity = 1;
    bool ok = true;
    for (int q = 0; ok; ++q) {
      const int u = (int)tc_uniform(next);
      if (lane == 0 && u < p.units) next = atomicAdd(ticket, 1);  // asked for ahead: its answer is due a unit later
      ok = tc_wait_warp(&s.sched_empty[q % kMoSched], ((q / kMoSched) & 1) ^ 1, abort_s);
      if (!ok) break;
      if (lane == 0) {
        s.sched[q % kMoSched] = u < p.units ? u : -1;
        tc_arrive(&s.sched_full[q % kMoSched]);
      }
      __syncwarp();
      if (u >= p.units) break;
      const MoUnit w = mo_unit(p, u);
      if (w.phase == 2) continue;
      const bool down = w.phase == 1;
      const int e = (int)tc_uniform(s.seg_expert[w.seg]);
      const int kb = down ? a.kb2 : a.kb1, rows = down ? a.rows2 : a.rows1;
      const int row = down ? w.tile * rows : w.tile * rows / 2;
      for (int b0 = w.b0; b0 < w.b1; b0 += kb) {
        const int nb = min(kb, w.b1 - b0);
        tc_wait_on(&s.empty[st], parity, abort_s, a.err);
        uint32_t dst = tc_uniform(ring + st * a.stage_bytes);
        const uint32_t full = tc_uniform(smem_u32(&s.full_a[st]));
        if (tc_elect()) {
          mbar_expect_tx(&s.full_a[st], nb * rows * 128);
          for (int c = b0 * 64; c < (b0 + nb) * 64; c += 64) {
            if (down) {
              mo_tma3(dst, &mw2, c, row, e, full, policy);
              dst += rows * 128;
            } else {
              for (int r = 0; r < rows; r += 32, dst += 32 * 128)  // 16 rows of gate, the same 16 of up
                mo_tma4(dst, &mw1, c, row + r / 2, 0, e, full, policy);
            }
          }
        }
        __syncwarp();
        filled = min(filled + 1, a.stages);
        if (++st == a.stages) {
          st = 0;
          parity ^= 1;
        }
      }
      ok = __all_sync(0xffffffffu, !*abort_s);
    }
    if (!ok && lane == 0) {
      if (!*abort_s) atomicOr(a.err, 1u);
      *abort_s = 1;
    }
    __syncwarp();
    // nothing may be in flight to this CTA's memory when it ends; after an abort the last stages were not seen full
    if (*abort_s) mo_drain(s.full_a, st, parity, filled, a.stages);
  } else if (warp == 1 || warp == 3) {
    // ---- rows of the tokens: the warps take stages by turns, a lane 16 bytes of a row at a time.  A lane's arrival follows
    // its copies, so neither warp waits for them.  (TMA gathers of four rows, a lane each: 100 cycles a gather, which 16
    // tokens an expert already notice.  Both warps at every stage, handing it on when its copies are there: their work
    // on a stage took longer than its weights.)
    const int half = warp >> 1, chunk = lane & 7, sub = lane >> 3;
    uint32_t *from = s.rows[half];
    int st = 0, turn = half, known = -1;
    unsigned parity = 1, done = 0;  // segments 32 known .. whose h is there, a bit each
    bool ok = true;
    // places of rows 8 i + sub and 8 i + 4 + sub, swizzled
    const uint32_t at0 = a.a_bytes + sub * 128 + ((chunk ^ sub) << 4), at1 = a.a_bytes + (sub + 4) * 128 + ((chunk ^ (sub + 4)) << 4);
    for (int q = 0; ok; ++q) {
      ok = tc_wait_warp(&s.sched_full[q % kMoSched], (q / kMoSched) & 1, abort_s);
      if (!ok) break;
      const int u = s.sched[q % kMoSched];
      __syncwarp();
      if (lane == 0) tc_arrive(&s.sched_empty[q % kMoSched]);
      if (u < 0) break;
      const MoUnit w = mo_unit(p, u);
      if (w.phase == 2) continue;
      const bool down = w.phase == 1;
      // columns: tokens; or, of h, rounded parts and rests in turn
      const int first = s.seg_first[w.seg], n = s.seg_n[w.seg] * (down ? 2 : 1), quads = (n + 3) / 4;
      const int kb = down ? a.kb2 : a.kb1, cols = down ? a.cols2 : a.cols, width = down ? a.inter : a.hidden;
      const char *base = static_cast<const char *>(down ? a.h : a.x) + chunk * 16;
      const uint32_t pitch = (down ? a.inter : (int)a.x_stride) / 8;
      for (int i = lane; i < quads * 4; i += 32) {
        const int c = min(i, n - 1);  // (past the last: its row again, to no use)
        const int pick = s.picks[first + (down ? c >> 1 : c)];
        from[i] = (down ? pick * 2 + (c & 1) : pick / a.top_k) * pitch;
      }
      if (down && (w.seg / 32 != known || !((done >> (w.seg & 31)) & 1))) {
        // until its gate/up units are done: a lane looks at a segment, so that the next units' need not be asked for again
        known = w.seg / 32;
        const int look = known * 32 + lane;
        for (uint32_t i = 0;; ++i) {
          done = __ballot_sync(0xffffffffu, look < p.segs && mo_acquire(seg_done + look) >= p.tiles1 * (a.rows1 / 32));
          if ((done >> (w.seg & 31)) & 1) break;
          if (__any_sync(0xffffffffu, i >= kSpinLimit || *abort_s)) {
            ok = false;
            break;
          }
          __nanosleep(32);
        }
        if (!ok) break;
      }
      __syncwarp();
      for (int b0 = w.b0; b0 < w.b1; b0 += kb) {
        if (turn == 0) {
          const int nb = min(kb, w.b1 - b0);
          tc_wait_on(&s.empty[st], parity, abort_s, a.err);
          for (int b = 0; b < nb; ++b) {
            const int col = (b0 + b) * 64;
            const bool there = col + chunk * 8 < width;
            const char *src = base + (there ? col * 2 : 0);
            uint32_t dst = ring + st * a.stage_bytes + b * cols * 128;
            const uint32_t *f = from + sub;
            int i = 0;
            for (; i + 4 <= quads; i += 4, f += 16, dst += 2048) {
              uint32_t o[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) o[j] = f[j * 4];
#pragma unroll
              for (int j = 0; j < 4; ++j) mo_copy16(dst + (j & 1 ? at1 : at0) + j / 2 * 1024, src + (uint64_t)o[j] * 16, there);
            }
            for (; i < quads; ++i, f += 4)
              mo_copy16(dst + (i & 1 ? at1 : at0) + (i & 3) / 2 * 1024, src + (uint64_t)*f * 16, there);
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&s.full_b[st])) : "memory");
        }
        turn ^= 1;
        if (++st == a.stages) {
          st = 0;
          parity ^= 1;
        }
      }
      __syncwarp();
      ok = __all_sync(0xffffffffu, !*abort_s);
    }
    if (!ok && lane == 0) {
      if (!*abort_s) atomicOr(a.err, 1u);
      *abort_s = 1;
    }
    cp_async_wait<0>();
  } else if (warp == 2) {
    // ---- MMA
    int st = 0, n_acc = 0;
    unsigned parity = 0;
    bool ok = true;
    for (int q = 0; ok; ++q) {
      ok = tc_wait_warp(&s.sched_full[q % kMoSched], (q / kMoSched) & 1, abort_s);
      if (!ok) break;
      const int u = (int)tc_uniform(s.sched[q % kMoSched]);
      __syncwarp();
      if (lane == 0) tc_arrive(&s.sched_empty[q % kMoSched]);
      if (u < 0) break;
      const MoUnit w = mo_unit(p, u);
      if (w.phase == 2) continue;
      const bool down = w.phase == 1;
      const int n = (s.seg_n[w.seg] * (down ? 2 : 1) + 15) / 16 * 16, rows = down ? a.rows2 : a.rows1;
      const int kb = down ? a.kb2 : a.kb1, cols = down ? a.cols2 : a.cols;
      const int buf = n_acc & 1;
      const uint32_t idesc = tc_uniform(mo_idesc<DT>(n)), acc = tc_uniform(tmem + buf * 256);
      const uint32_t a_step = tc_uniform(rows * 128 >> 4), b_step = tc_uniform(cols * 128 >> 4);
      tc_wait_on(&s.acc_empty[buf], ((n_acc >> 1) & 1) ^ 1, abort_s, a.err);
      ++n_acc;
      for (int b0 = w.b0; b0 < w.b1; b0 += kb) {
        const int nb = min(kb, w.b1 - b0);
        tc_wait_on(&s.full_b[st], parity, abort_s, a.err);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // rows stored by lanes' copies, read by MMAs
        tc_wait_on(&s.full_a[st], parity, abort_s, a.err);
        tc_fence_after();
        const uint32_t wa = tc_uniform(tc_desc_k(ring + st * a.stage_bytes));
        const uint32_t xb = tc_uniform(tc_desc_k(ring + st * a.stage_bytes + a.a_bytes));
        const uint32_t done = tc_uniform(smem_u32(&s.empty[st])), go = tc_uniform(b0 > w.b0 ? 1u : 0u);
        if (tc_elect()) {
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if (b < nb) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                tc_mma_ss(acc, tc_desc(wa + b * a_step + k * 2), tc_desc(xb + b * b_step + k * 2), idesc, b + k > 0 ? 1u : go);
            }
          tc_commit(done);
        }
        __syncwarp();
        if (++st == a.stages) {
          st = 0;
          parity ^= 1;
        }
      }
      const uint32_t full = tc_uniform(smem_u32(&s.acc_full[buf]));
      if (tc_elect()) tc_commit(full);
      __syncwarp();
      ok = __all_sync(0xffffffffu, !*abort_s);
    }
    if (!ok && lane == 0) {
      if (!*abort_s) atomicOr(a.err, 1u);
      *abort_s = 1;
    }
    // MMAs end before the tensor memory goes
    if (tc_elect()) tc_commit(smem_u32(&s.drained));
    mbar_wait_bounded(&s.drained, 0);
  } else if (warp >= 4) {
    // ---- epilogues: warp w has rows 32 (w - 4) .. of a unit
    const int mine = warp - 4, row0 = mine * 32;
    const uint32_t lanes = tmem + ((uint32_t)row0 << 16);
    int n_acc = 0;
    bool ok = true;
    for (int q = 0; ok; ++q) {
      ok = tc_wait_warp(&s.sched_full[q % kMoSched], (q / kMoSched) & 1, abort_s);
      if (!ok) break;
      const int u = s.sched[q % kMoSched];
      __syncwarp();
      if (lane == 0) tc_arrive(&s.sched_empty[q % kMoSched]);
      if (u < 0) break;
      const MoUnit w = mo_unit(p, u);
      if (w.phase == 2) {
        // 128 columns of y, four a lane, a token at a time: when all segments' rows are there
        const int col0 = w.seg * kMoSumCols, col = col0 + lane * 4;
        if (lane < kMoSumCols / 32 && col0 + lane * 32 < a.hidden)
          for (uint32_t i = 0; mo_acquire(strip_done + col0 / 32 + lane) < p.segs * p.shares; ++i) {
            if (i >= kSpinLimit || *abort_s) {
              ok = false;
              break;
            }
            __nanosleep(32);
          }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        __syncwarp();
        if (col >= a.hidden) continue;
        const int parts = a.top_k * p.shares, t1 = min(a.tokens, (w.tile + 1) * a.sum_tokens);
        for (int t = w.tile * a.sum_tokens + mine * 2; t < t1; t += 8) {  // two tokens, for the loads in flight
          float4 sum[2] = {};
          const float *rows = a.part + (int64_t)t * parts * a.hidden + col;
          const int64_t other = t + 1 < t1 ? (int64_t)parts * a.hidden : 0;
#pragma unroll 8
          for (int k = 0; k < parts; ++k, rows += a.hidden) {
            const float4 v[2] = {__ldcg(reinterpret_cast<const float4 *>(rows)), __ldcg(reinterpret_cast<const float4 *>(rows + other))};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              sum[i].x += v[i].x;
              sum[i].y += v[i].y;
              sum[i].z += v[i].z;
              sum[i].w += v[i].w;
            }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t lo = (uint32_t)bits_dt<DT>(sum[i].x) | ((uint32_t)bits_dt<DT>(sum[i].y) << 16);
            const uint32_t hi = (uint32_t)bits_dt<DT>(sum[i].z) | ((uint32_t)bits_dt<DT>(sum[i].w) << 16);
            if (t + i < t1)
              *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.y) + (int64_t)(t + i) * a.hidden + col) = make_uint2(lo, hi);
          }
        }
        continue;
      }
      const bool down = w.phase == 1;
      const int first = s.seg_first[w.seg], n = s.seg_n[w.seg], rows = down ? a.rows2 : a.rows1, buf = n_acc & 1;
      ok = tc_wait_warp(&s.acc_full[buf], (n_acc >> 1) & 1, abort_s);
      ++n_acc;
      if (!ok) break;
      tc_fence_after();
      if (row0 < rows) {
        // four columns at a time, rolled: a launch meets this code cold, and 16 at a time took 2 us longer to fetch
#pragma unroll 1
        for (int c0 = 0; c0 < n * (down ? 2 : 1); c0 += 4) {
          float v[4];
          mo_ld4(lanes + buf * 256 + c0, v);
          tc_wait_ld();
          if (down) {
            const int row = w.tile * rows + row0 + lane;
            if (row < a.hidden) {
#pragma unroll
              for (int c = 0; c < 4; c += 2)
                if (c0 + c < 2 * n) {
                  const int pick = s.picks[first + (c0 + c) / 2];
                  a.part[((int64_t)pick * p.shares + w.share) * a.hidden + row] = s.weights[pick] * (v[c] + v[c + 1]);
                }
            }
          } else {
            // lane l < 16 has gate row l, lane l + 16 up row l: the lower lanes take the even tokens, the upper the odd
            const int row = (w.tile * rows + row0) / 2 + (lane & 15);
            const bool upper = lane >= 16;
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
              const float got = __shfl_xor_sync(0xffffffffu, upper ? v[c] : v[c + 1], 16);
              const float gate = upper ? got : v[c], up = upper ? v[c + 1] : got;
              const int col = c0 + c + (upper ? 1 : 0);
              if (col < n && row < a.inter) {
                const float h = gate / (1.0f + expf(-gate)) * up, most = mo_rounded<DT>(h);
                const int64_t o = (int64_t)s.picks[first + col] * 2 * a.inter + row;
                store_elem<DT>(a.h, o, most);
                store_elem<DT>(a.h, o + a.inter, h - most);
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        tc_arrive(&s.acc_empty[buf]);
        __threadfence();  // the warp's rows, before they are counted
        const int strip = (w.tile * rows + row0) / 32;
        if (row0 < rows) {
          if (!down) atomicAdd(seg_done + w.seg, 1);
          else if (strip * 32 < a.hidden) atomicAdd(strip_done + strip, 1);
        }
      }
    }
    if (!ok && lane == 0) {
      if (!*abort_s) atomicOr(a.err, 1u);
      *abort_s = 1;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kMoTmemCols));
}

// -------------------------------------------------------------------- host ----

// How a call's experts are cut, from its sizes.
struct MoeCut {
  int rows1, rows2, kb1, kb2, cols, cols2, shares, sum_tokens, stages;
  uint32_t stage_bytes, a_bytes;
};

// Rows of a gate/up unit: the least time of the fullest SM, by whole units.  A unit's time is that of its bytes, but not
// below that of 64 rows: issuing a stage of 32 takes as long.
static int moe_rows(int64_t segs, int64_t rows) {
  int best = 32;
  int64_t least = INT64_MAX;
  for (int r = 32; r <= 128; r += 32) {
    const int64_t units = segs * ((rows + r - 1) / r), t = (units + kMoSms - 1) / kMoSms * ((r < 64 ? 64 : r) + 4);
    if (t < least) {
      least = t;
      best = r;
    }
  }
  return best;
}

static MoeCut moe_cut(int64_t tokens, int hidden, int inter, int experts, int top_k) {
  MoeCut c;
  const int64_t picks = tokens * top_k, segs = picks < experts ? picks : experts;
  // twice an expert's mean share and 16, where all its tokens are not fewer
  int64_t cols = (2 * picks / experts + 16 + 15) / 16 * 16;
  if (cols > (tokens + 15) / 16 * 16) cols = (tokens + 15) / 16 * 16;
  c.cols = (int)cols;
  c.cols2 = (int)(2 * cols < (2 * tokens + 15) / 16 * 16 ? 2 * cols : (2 * tokens + 15) / 16 * 16);  // h in two parts
  c.rows1 = moe_rows(segs, 2 * (int64_t)inter);
  // Down units are of 128 rows and a share of the inner channels, since partial rows are summed in any case: as many
  // shares as make the fullest SM's time least, a unit costing about two 64-column blocks besides its own.
  c.rows2 = hidden > 96 ? 128 : (hidden + 31) / 32 * 32;
  const int64_t tiles2 = segs * ((hidden + c.rows2 - 1) / c.rows2), blocks2 = (inter + 63) / 64;
  c.shares = 1;
  int64_t least = INT64_MAX;
  for (int n = 1; n <= 8 && n <= blocks2; ++n) {
    const int64_t t = (tiles2 * n + kMoSms - 1) / kMoSms * ((blocks2 + n - 1) / n + 2);
    if (t < least) {
      least = t;
      c.shares = n;
    }
  }
  // a stage of 16 to 40 KB: a stage costs its issuing warps some hundred cycles, whatever it holds
  auto blocks = [](int rows, int cols) {
    int kb = 4;
    while (kb > 1 && kb * (rows + cols) * 128 > 40 * 1024) kb /= 2;
    return kb;
  };
  c.kb1 = blocks(c.rows1, c.cols);
  c.kb2 = blocks(c.rows2, c.cols2);
  const int a1 = c.kb1 * c.rows1, a2 = c.kb2 * c.rows2, b1 = c.kb1 * c.cols, b2 = c.kb2 * c.cols2;
  c.a_bytes = (uint32_t)(a1 > a2 ? a1 : a2) * 128;
  c.stage_bytes = c.a_bytes + (uint32_t)(b1 > b2 ? b1 : b2) * 128;
  // an MMA reads 128 rows, however few of them a tile has: past its stage, where the tile is short
  auto past = [&](int kb, int rows) {
    const uint32_t end = (uint32_t)(kb - 1) * rows * 128 + 128 * 128;
    return end > c.stage_bytes ? end - c.stage_bytes : 0u;
  };
  const uint32_t p1 = past(c.kb1, c.rows1), p2 = past(c.kb2, c.rows2);
  c.stages = (int)((kMoRing - (p1 > p2 ? p1 : p2)) / c.stage_bytes);
  if (c.stages > kMoMaxStages) c.stages = kMoMaxStages;
  // sum units for every SM where there are as many tokens
  const int64_t strips = (hidden + kMoSumCols - 1) / kMoSumCols;
  c.sum_tokens = 8;
  while (c.sum_tokens < 16 && strips * ((tokens + c.sum_tokens - 1) / c.sum_tokens) > 2 * kMoSms) c.sum_tokens *= 2;
  return c;
}

static size_t moe_counters(int hidden) { return 1 + kMoMaxSegs + (size_t)(hidden + 31) / 32; }

template <int DT>
static cudaError_t moe_launch(const RouteArgs &r, const ExpertArgs &x, const CUtensorMap (&m)[2], cudaStream_t st) {
  constexpr int kSmem = kMoRing + (int)sizeof(MoShared);
  static_assert(kSmem <= 227 * 1024, "shared memory of a CTA");
  static thread_local int set_dev = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (set_dev != dev) {
    const cudaError_t e = cudaFuncSetAttribute(moe_experts_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    set_dev = dev;
  }
  int nt = 1;
  while (nt < kMrMaxTokens && (r.tokens + nt - 1) / nt * kMrCluster > kMoSms) nt *= 2;
  auto route = nt == 1 ? moe_route_kernel<DT, 1> : nt == 2 ? moe_route_kernel<DT, 2> : nt == 4 ? moe_route_kernel<DT, 4> : moe_route_kernel<DT, 8>;
  const cudaError_t e = launch_dependent(route, (unsigned)((r.tokens + nt - 1) / nt * kMrCluster), kMrThreads, 0, st, r);
  if (e != cudaSuccess) return e;
  return launch_dependent(moe_experts_kernel<DT>, kMoSms, kMoThreads, kSmem, st, m[0], m[1], x);
}

}  // namespace kvr

using namespace kvr;

extern "C" size_t kvr_moe_workspace_bytes(int64_t n_tokens, int hidden, int inter, int experts, int top_k) {
  if (n_tokens < 1 || n_tokens > kMoMaxTokens || hidden < 1 || inter < 1 || experts < 1 || top_k < 1 || top_k > kMoMaxTopK)
    return 0;
  const size_t picks = (size_t)n_tokens * top_k;
  return align_up(moe_counters(hidden) * 4, 256) + align_up(picks * inter * 4, 256) +
         picks * moe_cut(n_tokens, hidden, inter, experts, top_k).shares * hidden * 4;
}

extern "C" int kvr_moe_layer(const void *x, int dtype, int64_t n_tokens, int hidden, int64_t x_stride, const void *router,
                             int64_t router_stride, const void *gate_up, int64_t gu_expert_stride, int64_t gu_row_stride,
                             const void *down, int64_t down_expert_stride, int64_t down_row_stride, int experts, int inter,
                             int top_k, int norm, float scale, void *y, int32_t *ids, float *weights, void *workspace,
                             size_t workspace_bytes, void *status, kvr_stream_t stream) {
  clear_error();
  KVR_REQUIRE(n_tokens >= 0 && hidden >= 1 && inter >= 1 && experts >= 1 && top_k >= 1 && top_k <= experts,
              "kvr_moe_layer: bad shape");
  if (n_tokens > kMoMaxTokens || experts > kMoMaxExperts || top_k > kMoMaxTopK)
    return set_error(KVR_ENOTSUP, "kvr_moe_layer: at most %d tokens, %d experts and %d of them a token", kMoMaxTokens,
                     kMoMaxExperts, kMoMaxTopK);
  if (dtype != KVR_F16 && dtype != KVR_BF16) return set_error(KVR_ENOTSUP, "kvr_moe_layer: fp16 or bf16");
  if (hidden % 8 || inter % 8) return set_error(KVR_ENOTSUP, "kvr_moe_layer: hidden and inter must be multiples of 8");
  if (hidden > 1 << 16 || inter > 1 << 20) return set_error(KVR_ENOTSUP, "kvr_moe_layer: hidden or inter too large");
  if (n_tokens > 1 && x_stride > 1 << 28) return set_error(KVR_ENOTSUP, "kvr_moe_layer: x's rows lie too far apart");
  if (n_tokens == 0) return KVR_OK;
  KVR_REQUIRE(x && router && gate_up && down && y && ids && weights && workspace && status, "kvr_moe_layer: null pointer");
  KVR_REQUIRE((x_stride >= hidden || n_tokens == 1) && router_stride >= hidden && gu_row_stride >= hidden &&
                  down_row_stride >= inter && gu_expert_stride >= 2 * (int64_t)inter * gu_row_stride - (gu_row_stride - hidden) &&
                  down_expert_stride >= (int64_t)hidden * down_row_stride - (down_row_stride - inter),
              "kvr_moe_layer: rows must not share memory");
  KVR_REQUIRE((x_stride | router_stride | gu_row_stride | gu_expert_stride | down_row_stride | down_expert_stride) % 8 == 0,
              "kvr_moe_layer: strides must keep rows 16-byte aligned");
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(router) |
                         reinterpret_cast<uintptr_t>(gate_up) | reinterpret_cast<uintptr_t>(down) |
                         reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(status);
  KVR_REQUIRE((ptrs & 15) == 0 && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
              "kvr_moe_layer: pointers must be 16-byte aligned, the workspace 256-byte");
  KVR_REQUIRE(workspace_bytes >= kvr_moe_workspace_bytes(n_tokens, hidden, inter, experts, top_k),
              "kvr_moe_layer: workspace too small");
  // rows of y are stored while other CTAs still read
  auto meets = [&](const void *in, int64_t elements) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(in), q = reinterpret_cast<uintptr_t>(y);
    return p < q + (uintptr_t)n_tokens * hidden * 2 && q < p + (uintptr_t)elements * 2;
  };
  KVR_REQUIRE(!meets(x, (n_tokens - 1) * x_stride + hidden), "kvr_moe_layer: y must not lie in x");
  KVR_REQUIRE(!meets(router, (experts - 1) * router_stride + hidden) &&
                  !meets(gate_up, (experts - 1) * gu_expert_stride + (2 * (int64_t)inter - 1) * gu_row_stride + hidden) &&
                  !meets(down, (experts - 1) * down_expert_stride + (hidden - 1) * down_row_stride + inter),
              "kvr_moe_layer: y must not lie in the weights");
  if (!encode_tiled()) return set_error(KVR_ECUDA, "kvr_moe_layer: the driver has no cuTensorMapEncodeTiled");
  bind_context();
  const MoeCut c = moe_cut(n_tokens, hidden, inter, experts, top_k);
  const int64_t picks = n_tokens * top_k;
  char *ws = static_cast<char *>(workspace);
  RouteArgs r{};
  r.x = x; r.router = router; r.x_stride = x_stride; r.router_stride = router_stride;
  r.tokens = (int)n_tokens; r.hidden = hidden; r.experts = experts; r.top_k = top_k; r.norm = norm;
  r.scale = scale; r.ids = ids; r.weights = weights;
  r.counters = reinterpret_cast<int *>(ws); r.n_counters = (int)moe_counters(hidden);
  ExpertArgs a{};
  a.tokens = (int)n_tokens; a.hidden = hidden; a.inter = inter; a.experts = experts; a.top_k = top_k;
  a.rows1 = c.rows1; a.rows2 = c.rows2; a.kb1 = c.kb1; a.kb2 = c.kb2; a.cols = c.cols; a.cols2 = c.cols2;
  a.shares = c.shares; a.sum_tokens = c.sum_tokens; a.stages = c.stages;
  a.stage_bytes = c.stage_bytes; a.a_bytes = c.a_bytes;
  a.x = x; a.x_stride = n_tokens > 1 ? x_stride : hidden;
  a.ids = ids; a.weights = weights;
  a.h = ws + align_up(moe_counters(hidden) * 4, 256);
  a.part = reinterpret_cast<float *>(static_cast<char *>(a.h) + align_up((size_t)picks * inter * 4, 256));
  a.y = y;
  a.counters = r.counters; a.err = static_cast<unsigned *>(status);
  CUtensorMap m[2];
  const cuuint64_t gd[4] = {(cuuint64_t)hidden, (cuuint64_t)inter, 2, (cuuint64_t)experts};
  const cuuint64_t gs[3] = {(cuuint64_t)gu_row_stride * 2, (cuuint64_t)gu_row_stride * inter * 2, (cuuint64_t)gu_expert_stride * 2};
  const cuuint64_t dd[3] = {(cuuint64_t)inter, (cuuint64_t)hidden, (cuuint64_t)experts};
  const cuuint64_t ds[2] = {(cuuint64_t)down_row_stride * 2, (cuuint64_t)down_expert_stride * 2};
  const cuuint32_t gb[4] = {64, 16, 2, 1}, db[3] = {64, (cuuint32_t)c.rows2, 1};
  if (!make_map(&m[0], dtype, gate_up, 4, gd, gs, gb) || !make_map(&m[1], dtype, down, 3, dd, ds, db))
    return set_error(KVR_EINVAL, "kvr_moe_layer: a layout that TMA cannot read");
  const cudaError_t e = dtype == KVR_F16 ? moe_launch<KVR_F16>(r, a, m, as_cuda(stream)) : moe_launch<KVR_BF16>(r, a, m, as_cuda(stream));
  if (e != cudaSuccess) return set_error(KVR_ECUDA, "kvr_moe_layer: %s", cudaGetErrorString(e));
  return check_launch("kvr_moe_layer");
}
