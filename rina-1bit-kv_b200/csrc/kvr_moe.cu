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
// moe_route_kernel: clusters of 8 CTAs take 8 tokens; a CTA forms the logits of an
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
//   gate/up  R1 rows (16 of gate, 16 of up, ...) of a segment's expert over x: h, in 16 bits
//   down     R2 rows of Wd over h: partial rows (token, choice) in 32 bits
// A unit waits only for units with lower tickets, which run already: no CTA has to
// be resident for another to end.  Weights of a down unit stream in while its h is
// still being formed, so the memory does not idle between the phases.
//   warp 0  tickets, weight tiles by TMA (128-byte swizzle) into a ring of stages
//   warp 1  token rows by TMA gather into the same stages
//   warp 2  tcgen05.mma, accumulators of two units in tensor memory
//   warps 4-7  epilogues of 32 rows each; the warp that finishes the last segment of
//           32 rows of y adds up the choices of each token, in their order: no atomics
//           on values.
//
// What is held in fewer than 32 bits: h, rounded to the tensors' type because
// both operands of an MMA are of one 16-bit type.  Sums, router weights and
// partial rows are fp32.  The error against 64 bits is that of two roundings, of h and of
// y: sqrt(2) times that of rounding y alone.
//
// Waits are bounded; one that gives up sets the status word, lets copies and MMAs in
// flight end and frees the tensor memory.
#include "kvr_tcgen05.cuh"

namespace kvr {

constexpr int kMoMaxTokens = 128, kMoMaxExperts = 512, kMoMaxTopK = 16;
constexpr int kMoMaxPicks = kMoMaxTokens * kMoMaxTopK;
constexpr int kMoSms = 148;

// ------------------------------------------------------------------ router ----

constexpr int kMrThreads = 256, kMrCluster = 8, kMrTokens = 8;

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
// Larger first; NaN below everything.
__device__ __forceinline__ bool mo_above(double x, int i, double y, int j) {
  return x > y || (x == y && i < j) || (y != y && (x == x || i < j));
}

template <int DT>
__global__ void __cluster_dims__(kMrCluster, 1, 1) __launch_bounds__(kMrThreads) moe_route_kernel(RouteArgs a) {
  __shared__ double part[kMrTokens][kMoMaxExperts / kMrCluster];  // logits of this CTA's experts
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = blockIdx.x % kMrCluster, t0 = blockIdx.x / kMrCluster * kMrTokens;
  const int n_tok = min(kMrTokens, a.tokens - t0);
  griddep_wait();
  griddep_launch();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < a.n_counters; i += kMrThreads) a.counters[i] = 0;
  const int per = (a.experts + kMrCluster - 1) / kMrCluster, e0 = rank * per, e1 = min(a.experts, e0 + per);
  for (int e = e0 + warp; e < e1; e += kMrThreads / 32) {
    float s[kMrTokens] = {};
    for (int c = lane * 8; c < a.hidden; c += 256) {
      float w[8];
      load8<DT>(a.router, e * a.router_stride + c, w);
#pragma unroll
      for (int t = 0; t < kMrTokens; ++t) {
        if (t < n_tok) {
          float x[8];
          load8<DT>(a.x, (t0 + t) * a.x_stride + c, x);
#pragma unroll
          for (int j = 0; j < 8; ++j) s[t] = fmaf(x[j], w[j], s[t]);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < kMrTokens; ++t) {
      double d = s[t];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
      if (lane == t && t < n_tok) part[t][e - e0] = d;
    }
  }
  mo_cluster_sync();
  // CTA r: token r, by one warp; lane l holds experts l, l + 32, ...
  if (rank < n_tok && warp == 0) {
    constexpr int kEach = kMoMaxExperts / 32;
    const int64_t t = t0 + rank;
    double z[kEach];
    float e[kEach], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int x = i * 32 + lane;
      z[i] = 0.0;
      if (x < a.experts) {
        z[i] = mo_peer_double(&part[rank][x % per], x / per);
        m = fmaxf(m, (float)z[i]);
      }
    }
    m = warp_max(m);
    float all = 0.0f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      e[i] = i * 32 + lane < a.experts ? expf((float)(z[i] - (double)m)) : 0.0f;
      all += e[i];
    }
    all = warp_sum(all);
    unsigned taken = 0;
    float sum = 0.0f, mine = 0.0f;
    int my_id = 0;
    for (int k = 0; k < a.top_k; ++k) {
      double best = NAN;
      int at = INT_MAX;
      float v = 0.0f;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int x = i * 32 + lane;
        if (x < a.experts && !((taken >> i) & 1) && (at == INT_MAX || mo_above(z[i], x, best, at))) {
          best = z[i];
          at = x;
          v = e[i];
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double ob = __shfl_xor_sync(0xffffffffu, best, o);
        const int oa = __shfl_xor_sync(0xffffffffu, at, o);
        const float ov = __shfl_xor_sync(0xffffffffu, v, o);
        if (oa != INT_MAX && (at == INT_MAX || mo_above(ob, oa, best, at))) {
          best = ob;
          at = oa;
          v = ov;
        }
      }
      if ((at & 31) == lane) taken |= 1u << (at >> 5);
      sum += v;
      if (lane == k) {
        mine = v;
        my_id = at;
      }
    }
    if (lane < a.top_k) {
      // a logit that is no number, or infinite, leaves no weight that means anything
      const float w = all < INFINITY ? a.scale * mine / (a.norm ? sum : all) : NAN;
      a.ids[t * a.top_k + lane] = my_id;
      a.weights[t * a.top_k + lane] = w;
    }
  }
  mo_cluster_sync();  // the other CTAs' logits stay until they are read
}

// ----------------------------------------------------------------- experts ----

constexpr int kMoThreads = 256;
constexpr int kMoMaxStages = 16, kMoSched = 4;
constexpr uint32_t kMoRing = 192 * 1024;   // stages
constexpr uint32_t kMoPad = 16 * 1024;     // an MMA reads 128 rows from a tile's start, however few of them it uses
constexpr uint32_t kMoTmemCols = 256;      // two accumulators of 128 columns
constexpr int kMoMinCols = 16;
constexpr int kMoMaxSegs = kMoMaxExperts + kMoMaxPicks / kMoMinCols;

struct ExpertArgs {
  int tokens, hidden, inter, experts, top_k;
  int rows1, rows2;      // rows of a gate/up and of a down unit
  int kb1, kb2;          // 64-column blocks of a stage
  int cols;              // most tokens of a segment, a multiple of 16
  int stages;
  uint32_t stage_bytes, a_bytes;  // of a stage; its weights' part
  const int *ids;
  const float *weights;
  void *h;               // (tokens * top_k, inter)
  float *part;           // (tokens * top_k, hidden)
  void *y;
  int64_t y_stride;
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
  unsigned mask[kMoMaxExperts][kMoMaxTokens / 32];  // tokens of each expert
  short first[kMoMaxExperts];
  short picks[kMoMaxPicks];  // token * top_k + choice, by expert
};

__device__ __forceinline__ void mo_tma4(uint32_t dst, const CUtensorMap *m, int c0, int c1, int c2, int c3, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(m), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void mo_tma3(uint32_t dst, const CUtensorMap *m, int c0, int c1, int c2, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(dst),
      "l"(m), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}
// 64 columns of four rows.
__device__ __forceinline__ void mo_gather4(uint32_t dst, const CUtensorMap *m, int c0, int r0, int r1, int r2, int r3,
                                           uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
      "%4, %5, %6}], [%7];" ::"r"(dst),
      "l"(m), "r"(c0), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ int mo_acquire(const int *p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
template <int DT>
__host__ __device__ constexpr uint32_t mo_idesc(uint32_t n) {  // kind::f16, fp32 accumulator, M 128
  return (1u << 4) | ((DT == KVR_BF16 ? 1u : 0u) << 7) | ((DT == KVR_BF16 ? 1u : 0u) << 10) | ((n >> 3) << 17) |
         ((128u >> 4) << 24);
}

// Work unit u: phase (0: gate/up, 1: down), segment, tile of rows.
struct MoUnit {
  int down, seg, tile;
};
__device__ __forceinline__ MoUnit mo_unit(const ExpertArgs &a, int u, int segs, int tiles1) {
  const int n1 = segs * tiles1;
  MoUnit w;
  w.down = u >= n1;
  if (!w.down) {
    w.seg = u / tiles1;
    w.tile = u - w.seg * tiles1;
  } else {  // tile by tile, so that choices are added up while others are still multiplied
    u -= n1;
    w.tile = u / segs;
    w.seg = u - w.tile * segs;
  }
  return w;
}

template <int DT>
__global__ void __launch_bounds__(kMoThreads, 1)
    moe_experts_kernel(const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mw1,
                       const __grid_constant__ CUtensorMap mh, const __grid_constant__ CUtensorMap mw2, const ExpertArgs a) {
  extern __shared__ __align__(1024) unsigned char sm[];
  MoShared &s = *reinterpret_cast<MoShared *>(sm + kMoRing + kMoPad);
  volatile int *abort_s = &s.abort_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem)),
                 "r"(kMoTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (tid == 0) {
    s.abort_s = 0;
    for (int i = 0; i < a.stages; ++i) {
      tc_bar_init(&s.full_a[i], 1);
      tc_bar_init(&s.full_b[i], 1);
      tc_bar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc_bar_init(&s.acc_full[i], 1);
      tc_bar_init(&s.acc_empty[i], 4);
    }
    for (int i = 0; i < kMoSched; ++i) {
      tc_bar_init(&s.sched_full[i], 1);
      tc_bar_init(&s.sched_empty[i], 6);  // copies of tokens, MMA, four epilogue warps
    }
    tc_bar_init(&s.drained, 1);
  }
  for (int i = tid; i < kMoMaxExperts * (kMoMaxTokens / 32); i += kMoThreads) (&s.mask[0][0])[i] = 0;
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // barriers: for the copies and commits
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem;
  griddep_wait();  // what follows reads the routing
  griddep_launch();

  // picks by expert, and segments.  Every CTA makes the same lists: a bit per (expert, token), counts and prefix sums.
  const int picks = a.tokens * a.top_k;
  for (int i = tid; i < picks; i += kMoThreads) {
    const int t = i / a.top_k;
    atomicOr(&s.mask[a.ids[i]][t >> 5], 1u << (t & 31));
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
      for (int w = 0; w < kMoMaxTokens / 32; ++w) n[j] += __popc(s.mask[e][w]);
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
  for (int i = tid; i < picks; i += kMoThreads) {
    const int t = i / a.top_k, e = a.ids[i];
    int before = 0;
    for (int w = 0; w < (t >> 5); ++w) before += __popc(s.mask[e][w]);
    before += __popc(s.mask[e][t >> 5] & ((1u << (t & 31)) - 1));
    s.picks[s.first[e] + before] = (short)i;
  }
  __syncthreads();
  const int segs = s.n_segs;
  const int tiles1 = (a.inter + a.rows1 / 2 - 1) / (a.rows1 / 2), tiles2 = (a.hidden + a.rows2 - 1) / a.rows2;
  const int units = segs * (tiles1 + tiles2);
  int *ticket = a.counters, *seg_done = a.counters + 1, *strip_done = seg_done + kMoMaxSegs;
  const int blocks1 = (a.hidden + 63) / 64, blocks2 = (a.inter + 63) / 64;
  const uint32_t ring = smem_u32(sm);

  if (warp == 0) {
    // ---- tickets and weights: one lane
    if (lane == 0) {
      int it = 0, q = 0;
      int next = atomicAdd(ticket, 1);
      bool ok = true;
      while (ok) {
        const int u = next;
        if (u < units) next = atomicAdd(ticket, 1);  // asked for ahead: its answer is due a unit later
        ok = tc_wait(&s.sched_empty[q % kMoSched], ((q / kMoSched) & 1) ^ 1, abort_s);
        if (!ok) break;
        s.sched[q % kMoSched] = u < units ? u : -1;
        tc_arrive(&s.sched_full[q % kMoSched]);
        ++q;
        if (u >= units) break;
        const MoUnit w = mo_unit(a, u, segs, tiles1);
        const int e = s.seg_expert[w.seg];
        const int blocks = w.down ? blocks2 : blocks1, kb = w.down ? a.kb2 : a.kb1, rows = w.down ? a.rows2 : a.rows1;
        for (int b0 = 0; b0 < blocks; b0 += kb, ++it) {
          const int st = it % a.stages, nb = min(kb, blocks - b0);
          if (!(ok = tc_wait(&s.empty[st], ((it / a.stages) & 1) ^ 1, abort_s))) break;
          mbar_expect_tx(&s.full_a[st], nb * rows * 128);
          uint32_t dst = ring + st * a.stage_bytes;
          for (int b = b0; b < b0 + nb; ++b) {
            if (w.down) {
              mo_tma3(dst, &mw2, b * 64, w.tile * rows, e, &s.full_a[st]);
              dst += rows * 128;
            } else {
              for (int r = 0; r < rows; r += 32, dst += 32 * 128)  // 16 rows of gate, the same 16 of up
                mo_tma4(dst, &mw1, b * 64, (w.tile * rows + r) / 2, 0, e, &s.full_a[st]);
            }
          }
        }
      }
      if (!ok) {
        if (!*abort_s) atomicOr(a.err, 1u);
        *abort_s = 1;
      }
      // nothing may be in flight to this CTA's memory when it ends; after an abort the last stages were not seen full
      if (*abort_s)
        for (int i = max(0, it - a.stages); i < it; ++i)
          mbar_wait_bounded(&s.full_a[i % a.stages], (i / a.stages) & 1, 1u << 14);
    }
  } else if (warp == 1) {
    // ---- rows of the tokens, four a copy
    int it = 0;
    bool ok = true;
    for (int q = 0; ok; ++q) {
      ok = tc_wait_warp(&s.sched_full[q % kMoSched], (q / kMoSched) & 1, abort_s);
      if (!ok) break;
      const int u = s.sched[q % kMoSched];
      __syncwarp();
      if (lane == 0) tc_arrive(&s.sched_empty[q % kMoSched]);
      if (u < 0) break;
      const MoUnit w = mo_unit(a, u, segs, tiles1);
      const int first = s.seg_first[w.seg], n = s.seg_n[w.seg], quads = (n + 3) / 4;
      if (w.down) {  // until its gate/up units are done
        if (lane == 0)
          for (uint32_t i = 0; mo_acquire(seg_done + w.seg) < tiles1 * (a.rows1 / 32); ++i) {
            if (i >= kSpinLimit || *abort_s) {
              ok = false;
              break;
            }
            __nanosleep(32);
          }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        __syncwarp();
        asm volatile("fence.proxy.async;" ::: "memory");  // h was stored, and is read by copies
      }
      const int blocks = w.down ? blocks2 : blocks1, kb = w.down ? a.kb2 : a.kb1;
      for (int b0 = 0; b0 < blocks; b0 += kb, ++it) {
        const int st = it % a.stages, nb = min(kb, blocks - b0);
        if (!(ok = tc_wait_warp(&s.empty[st], ((it / a.stages) & 1) ^ 1, abort_s))) break;
        if (lane == 0) mbar_expect_tx(&s.full_b[st], nb * quads * 512);
        __syncwarp();
        for (int i = lane; i < nb * quads; i += 32) {
          const int b = i / quads, g = i - b * quads;
          int r[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int pick = s.picks[first + min(g * 4 + j, n - 1)];  // (past the last: its row again, to no use)
            r[j] = w.down ? pick : pick / a.top_k;
          }
          mo_gather4(ring + st * a.stage_bytes + a.a_bytes + (b * a.cols + g * 4) * 128, w.down ? &mh : &mx, (b0 + b) * 64,
                     r[0], r[1], r[2], r[3], &s.full_b[st]);
        }
        __syncwarp();
      }
    }
    if (lane == 0) {
      if (!ok) {
        if (!*abort_s) atomicOr(a.err, 1u);
        *abort_s = 1;
      }
      if (*abort_s)
        for (int i = max(0, it - a.stages); i < it; ++i)
          mbar_wait_bounded(&s.full_b[i % a.stages], (i / a.stages) & 1, 1u << 14);
    }
    __syncwarp();
  } else if (warp == 2) {
    // ---- MMA
    int it = 0;
    bool ok = true;
    for (int q = 0; ok; ++q) {
      ok = tc_wait_warp(&s.sched_full[q % kMoSched], (q / kMoSched) & 1, abort_s);
      if (!ok) break;
      const int u = s.sched[q % kMoSched];
      __syncwarp();
      if (lane == 0) tc_arrive(&s.sched_empty[q % kMoSched]);
      if (u < 0) break;
      const MoUnit w = mo_unit(a, u, segs, tiles1);
      const int n = (s.seg_n[w.seg] + 15) / 16 * 16, rows = w.down ? a.rows2 : a.rows1;
      const int blocks = w.down ? blocks2 : blocks1, kb = w.down ? a.kb2 : a.kb1, buf = q & 1;
      const uint32_t idesc = tc_uniform(mo_idesc<DT>(n)), acc = tc_uniform(tmem + buf * 128);
      tc_wait_on(&s.acc_empty[buf], ((q >> 1) & 1) ^ 1, abort_s, a.err);
      for (int b0 = 0; b0 < blocks; b0 += kb, ++it) {
        const int st = it % a.stages, nb = min(kb, blocks - b0);
        tc_wait_on(&s.full_b[st], (it / a.stages) & 1, abort_s, a.err);
        tc_wait_on(&s.full_a[st], (it / a.stages) & 1, abort_s, a.err);
        tc_fence_after();
        const uint32_t wa = tc_uniform(tc_desc_k(ring + st * a.stage_bytes));
        const uint32_t xb = tc_uniform(tc_desc_k(ring + st * a.stage_bytes + a.a_bytes));
        const uint32_t done = tc_uniform(smem_u32(&s.empty[st]));
        if (tc_elect()) {
          for (int b = 0; b < nb; ++b) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              tc_mma_ss(acc, tc_desc(wa + b * (rows * 128 >> 4) + k * 2), tc_desc(xb + b * (a.cols * 128 >> 4) + k * 2), idesc,
                        b0 + b + k > 0);
          }
          tc_commit(done);
        }
        __syncwarp();
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
    const int part = warp - 4, row0 = part * 32;
    const uint32_t lanes = tmem + ((uint32_t)row0 << 16);
    bool ok = true;
    for (int q = 0; ok; ++q) {
      ok = tc_wait_warp(&s.sched_full[q % kMoSched], (q / kMoSched) & 1, abort_s);
      if (!ok) break;
      const int u = s.sched[q % kMoSched], buf = q & 1;
      __syncwarp();
      if (lane == 0) tc_arrive(&s.sched_empty[q % kMoSched]);
      if (u < 0) break;
      const MoUnit w = mo_unit(a, u, segs, tiles1);
      const int first = s.seg_first[w.seg], n = s.seg_n[w.seg], rows = w.down ? a.rows2 : a.rows1;
      ok = tc_wait_warp(&s.acc_full[buf], (q >> 1) & 1, abort_s);
      if (!ok) break;
      tc_fence_after();
      if (row0 < rows) {
        for (int c0 = 0; c0 < n; c0 += 16) {
          float v[16];
          tc_ld16(lanes + buf * 128 + c0, v);
          tc_wait_ld();
          if (w.down) {
            const int row = w.tile * rows + row0 + lane;
            if (row < a.hidden) {
#pragma unroll
              for (int c = 0; c < 16; ++c)
                if (c0 + c < n) a.part[(int64_t)s.picks[first + c0 + c] * a.hidden + row] = v[c];
            }
          } else {
            // lane l < 16 has gate row l, lane l + 16 up row l: the lower lanes take the even tokens, the upper the odd
            const int row = (w.tile * rows + row0) / 2 + (lane & 15);
            const bool upper = lane >= 16;
#pragma unroll
            for (int c = 0; c < 16; c += 2) {
              const float got = __shfl_xor_sync(0xffffffffu, upper ? v[c] : v[c + 1], 16);
              const float gate = upper ? got : v[c], up = upper ? v[c + 1] : got;
              const int col = c0 + c + (upper ? 1 : 0);
              if (col < n && row < a.inter)
                store_elem<DT>(a.h, (int64_t)s.picks[first + col] * a.inter + row, gate / (1.0f + expf(-gate)) * up);
            }
          }
        }
      }
      tc_fence_before();
      if (!w.down) asm volatile("fence.proxy.async;" ::: "memory");  // h is read by copies
      __threadfence();
      __syncwarp();
      if (lane == 0) tc_arrive(&s.acc_empty[buf]);
      if (row0 >= rows) continue;
      if (!w.down) {
        if (lane == 0) atomicAdd(seg_done + w.seg, 1);
        continue;
      }
      const int strip = (w.tile * rows + row0) / 32;
      int done = 0;
      if (strip * 32 < a.hidden && lane == 0) done = atomicAdd(strip_done + strip, 1) + 1;
      if (__shfl_sync(0xffffffffu, done, 0) != segs) continue;
      __threadfence();
      // the last segment's 32 rows: y, the choices of each token in their order, four rows a lane
      const int row = strip * 32 + (lane & 7) * 4;
      if (row < a.hidden) {
#pragma unroll 2
        for (int t = lane >> 3; t < a.tokens; t += 4) {
          float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
          for (int k = 0; k < a.top_k; ++k) {
            const float wk = __ldg(a.weights + t * a.top_k + k);
            const float4 p = __ldcg(reinterpret_cast<const float4 *>(a.part + (int64_t)(t * a.top_k + k) * a.hidden + row));
            sum.x = fmaf(wk, p.x, sum.x);
            sum.y = fmaf(wk, p.y, sum.y);
            sum.z = fmaf(wk, p.z, sum.z);
            sum.w = fmaf(wk, p.w, sum.w);
          }
          const uint32_t lo = (uint32_t)bits_dt<DT>(sum.x) | ((uint32_t)bits_dt<DT>(sum.y) << 16);
          const uint32_t hi = (uint32_t)bits_dt<DT>(sum.z) | ((uint32_t)bits_dt<DT>(sum.w) << 16);
          *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.y) + t * a.y_stride + row) = make_uint2(lo, hi);
        }
      }
      __syncwarp();
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
  int rows1, rows2, kb1, kb2, cols, stages;
  uint32_t stage_bytes, a_bytes;
};

// Rows of a unit: as many as leave every SM several units, so that none waits long for the last.
static int moe_rows(int64_t segs, int64_t rows) {
  for (int r = 128; r > 32; r /= 2)
    if (segs * ((rows + r - 1) / r) >= kMoSms * 6) return r;
  return 32;
}

static MoeCut moe_cut(int64_t tokens, int hidden, int inter, int experts, int top_k) {
  MoeCut c;
  const int64_t picks = tokens * top_k, segs = picks < experts ? picks : experts;
  // twice an expert's mean share and 16, where all its tokens are not fewer
  int64_t cols = (2 * picks / experts + 16 + 15) / 16 * 16;
  if (cols > (tokens + 15) / 16 * 16) cols = (tokens + 15) / 16 * 16;
  c.cols = (int)cols;
  c.rows1 = moe_rows(segs, 2 * (int64_t)inter);
  c.rows2 = moe_rows(segs, hidden);
  auto blocks = [&](int rows) { return rows + c.cols <= 48 ? 4 : rows + c.cols <= 96 ? 2 : 1; };
  c.kb1 = blocks(c.rows1);
  c.kb2 = blocks(c.rows2);
  const int a1 = c.kb1 * c.rows1, a2 = c.kb2 * c.rows2, kb = c.kb1 > c.kb2 ? c.kb1 : c.kb2;
  c.a_bytes = (uint32_t)(a1 > a2 ? a1 : a2) * 128;
  c.stage_bytes = c.a_bytes + (uint32_t)kb * c.cols * 128;
  c.stages = (int)(kMoRing / c.stage_bytes);
  if (c.stages > kMoMaxStages) c.stages = kMoMaxStages;
  return c;
}

static size_t moe_counters(int hidden) { return 1 + kMoMaxSegs + (size_t)(hidden + 31) / 32; }

template <int DT>
static cudaError_t moe_launch(const RouteArgs &r, const ExpertArgs &x, const CUtensorMap (&m)[4], cudaStream_t st) {
  constexpr int kSmem = kMoRing + kMoPad + (int)sizeof(MoShared);
  static_assert(kSmem <= 227 * 1024, "shared memory of a CTA");
  static thread_local int set_dev = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (set_dev != dev) {
    const cudaError_t e = cudaFuncSetAttribute(moe_experts_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    set_dev = dev;
  }
  const unsigned groups = (unsigned)((r.tokens + kMrTokens - 1) / kMrTokens);
  const cudaError_t e = launch_dependent(moe_route_kernel<DT>, groups * kMrCluster, kMrThreads, 0, st, r);
  if (e != cudaSuccess) return e;
  return launch_dependent(moe_experts_kernel<DT>, kMoSms, kMoThreads, kSmem, st, m[0], m[1], m[2], m[3], x);
}

}  // namespace kvr

using namespace kvr;

extern "C" size_t kvr_moe_workspace_bytes(int64_t n_tokens, int hidden, int inter, int top_k) {
  if (n_tokens < 1 || n_tokens > kMoMaxTokens || hidden < 1 || inter < 1 || top_k < 1 || top_k > kMoMaxTopK) return 0;
  const size_t picks = (size_t)n_tokens * top_k;
  return align_up(moe_counters(hidden) * 4, 256) + align_up(picks * inter * 2, 256) + picks * hidden * 4;
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
  KVR_REQUIRE(workspace_bytes >= kvr_moe_workspace_bytes(n_tokens, hidden, inter, top_k), "kvr_moe_layer: workspace too small");
  {  // rows of y are stored while other CTAs still read x
    const uintptr_t p = reinterpret_cast<uintptr_t>(x), q = reinterpret_cast<uintptr_t>(y);
    const uintptr_t n = ((n_tokens - 1) * x_stride + hidden) * 2, m = n_tokens * (uintptr_t)hidden * 2;
    KVR_REQUIRE(p + n <= q || q + m <= p, "kvr_moe_layer: y must not lie in x");
  }
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
  a.rows1 = c.rows1; a.rows2 = c.rows2; a.kb1 = c.kb1; a.kb2 = c.kb2; a.cols = c.cols; a.stages = c.stages;
  a.stage_bytes = c.stage_bytes; a.a_bytes = c.a_bytes;
  a.ids = ids; a.weights = weights;
  a.h = ws + align_up(moe_counters(hidden) * 4, 256);
  a.part = reinterpret_cast<float *>(static_cast<char *>(a.h) + align_up((size_t)picks * inter * 2, 256));
  a.y = y; a.y_stride = hidden;
  a.counters = r.counters; a.err = static_cast<unsigned *>(status);
  CUtensorMap m[4];
  const cuuint64_t xd[2] = {(cuuint64_t)hidden, (cuuint64_t)n_tokens}, xs[1] = {(cuuint64_t)(n_tokens > 1 ? x_stride : hidden) * 2};
  const cuuint64_t hd[2] = {(cuuint64_t)inter, (cuuint64_t)picks}, hs[1] = {(cuuint64_t)inter * 2};
  const cuuint64_t gd[4] = {(cuuint64_t)hidden, (cuuint64_t)inter, 2, (cuuint64_t)experts};
  const cuuint64_t gs[3] = {(cuuint64_t)gu_row_stride * 2, (cuuint64_t)gu_row_stride * inter * 2, (cuuint64_t)gu_expert_stride * 2};
  const cuuint64_t dd[3] = {(cuuint64_t)inter, (cuuint64_t)hidden, (cuuint64_t)experts};
  const cuuint64_t ds[2] = {(cuuint64_t)down_row_stride * 2, (cuuint64_t)down_expert_stride * 2};
  const cuuint32_t row[2] = {64, 1}, gb[4] = {64, 16, 2, 1}, db[3] = {64, (cuuint32_t)c.rows2, 1};
  if (!make_map(&m[0], dtype, x, 2, xd, xs, row) || !make_map(&m[1], dtype, gate_up, 4, gd, gs, gb) ||
      !make_map(&m[2], dtype, a.h, 2, hd, hs, row) || !make_map(&m[3], dtype, down, 3, dd, ds, db))
    return set_error(KVR_EINVAL, "kvr_moe_layer: a layout that TMA cannot read");
  const cudaError_t e = dtype == KVR_F16 ? moe_launch<KVR_F16>(r, a, m, as_cuda(stream)) : moe_launch<KVR_BF16>(r, a, m, as_cuda(stream));
  if (e != cudaSuccess) return set_error(KVR_ECUDA, "kvr_moe_layer: %s", cudaGetErrorString(e));
  return check_launch("kvr_moe_layer");
}
