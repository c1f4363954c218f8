// Beam search's choice of continuations.
//
// Request b has K beams with running scores c_k and a row of V logits each:
// score(k, t) = c_k + x_kt - lse_k, lse_k = log sum_t exp(x_kt).  The n best of
// its K V continuations come out in order, equal scores by beam and token.
//
// One pass over the logits.  beam_rows_kernel: a CTA takes a segment of a row,
// holds a running maximum and sum of exponentials per thread and, for the CTA, a
// list of the segment's best logits.  The list's n-th is a threshold that few logits
// pass: 16 a tile at first, then n times the logarithm of the tiles in all.  Threads
// add what passes without waiting for one another; all warps meet only to cut the
// list to n.  The first threshold comes from the threads' own maxima over the first
// tile.  Within a row the order of the logits is the order of the scores, so no
// normaliser is needed yet.  beam_merge_kernel: a CTA per request joins the sums,
// scores the K S n listed logits and picks the n best.
//
// Scores are compared in 64 bits: c_k + (x - lse_k) in 32 would make different
// logits equal and order them by token.  Sums are in 32 bits per thread (at most
// some thousand exponentials <= 1) and joined in 64 by the second kernel.  (Which logits a
// thread adds up depends on where a row lies within 16 bytes, so equal rows may have
// sums of other last bits, and ties between their beams no order but theirs.)
//
// What binds: 512 rows of 128256 in fp32, 51.5 us (5.1 TB/s; a kernel that only
// reads them with as many CTAs takes 47): some 200 instructions a warp and tile of 512
// logits, and 3 us at either end of a segment when nothing streams.  Rows in several
// segments fill the SMs where rows are few, and pay those ends each (1184 CTAs for 512
// rows: 9 us more).  Tried: words of all rows in equal shares, 6 us more; copies two tiles
// ahead, 8 us more (fewer CTAs have room).  One request of 4 beams and 32000 tokens: 7.8 us,
// a chain of two launches and their barriers; the second kernel is 4 to 5 us of it.  That one is slow where very many
// candidates pass its threshold: 32 beams of equal scores with n = 64, 4.2 ms (spread over 12 units: 38 us).
#include <cfloat>

#include "kvr_common.cuh"

namespace kvr {

constexpr int kBsThreads = 256, kBsRowThreads = 256;  // of the second kernel, of the first
constexpr int kBsTile = 16;       // logits of a thread in a tile
constexpr int kBsMaxN = 128, kBsMaxBeams = 32, kBsMaxEos = 8;
constexpr int kBsSlack = 32;      // entries beyond n that a list holds before it is cut
constexpr int kBsList = kBsMaxN + kBsSlack + kBsTile * kBsRowThreads;  // and all of a tile
constexpr int kBsMaxCands = 8192; // of a request in the second kernel
constexpr int kBsPicked = 1024;   // candidates that it ranks from shared memory

struct BeamArgs {
  const void *logits;
  int64_t row_stride;  // elements
  int rows, beams, n, splits;
  int vocab;
  const float *cum;
  float2 *ml;          // (rows, splits) maximum and sum
  uint64_t *cands;     // (rows, splits, n) keys, 0: none
  float *scores, *next_scores;
  int *out_beams, *tokens, *next_beams, *next_tokens;
  int n_eos;
  int eos[kBsMaxEos];
};

__device__ __forceinline__ float bs_max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
__device__ __forceinline__ float bs_exp(float x) {  // e^x for x <= 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}
// Larger logits first, lower tokens first among equal ones; 0 is below every key.
__device__ __forceinline__ uint64_t bs_key(float x, int token) {
  return ((uint64_t)float_key(x) << 32) | (uint32_t)(0xffffffffu - (uint32_t)token);
}
__device__ __forceinline__ float bs_value(uint64_t key) { return key_float((uint32_t)(key >> 32)); }
__device__ __forceinline__ int bs_token(uint64_t key) { return (int)(0xffffffffu - (uint32_t)key); }

struct __align__(16) BeamShared {
  uint64_t list[kBsList];
  uint64_t best[kBsRowThreads];
  uint64_t nth;
  int count;
  float m[kBsRowThreads / 32], s[kBsRowThreads / 32];
};

// How many maxima the n-th largest is taken of, for a threshold that n values at least are not below: four times n (of
// fewer, more values lie above it), all threads' at most.
__device__ __forceinline__ int bs_groups(int n) {
  int m = 32;
  while (m < 4 * n && m < kBsThreads) m *= 2;
  return m;
}

// The n-th largest of one key per thread (distinct unless 0), to all of the CTA's.
__device__ __forceinline__ uint64_t bs_nth(BeamShared &sh, uint64_t mine, int n) {
  const int tid = threadIdx.x;
  sh.best[tid] = mine;
  if (tid == 0) sh.nth = 0;
  __syncthreads();
  int above = 0;
#pragma unroll 4
  for (int i = 0; i < kBsRowThreads; i += 2) {
    const ulonglong2 o = *reinterpret_cast<const ulonglong2 *>(&sh.best[i]);
    above += (o.x > mine) + (o.y > mine);
  }
  if (mine && above == n - 1) sh.nth = mine;
  __syncthreads();
  return sh.nth;
}

// Cuts the list to its n best, in order.  All threads, between barriers.
__device__ __noinline__ void bs_cut(BeamShared &sh, int n) {
  const int tid = threadIdx.x;
  int c = sh.count;
  if (c > kBsRowThreads) {  // first to those not below the n-th of the threads' own, moved to the front
    uint64_t mine = 0;
    for (int i = tid; i < c; i += kBsRowThreads) mine = max(mine, sh.list[i]);
    const uint64_t low = bs_nth(sh, mine, n);
    if (tid == 0) sh.count = 0;
    for (int i0 = 0; i0 < c; i0 += kBsRowThreads) {
      const uint64_t key = i0 + tid < c ? sh.list[i0 + tid] : 0;
      __syncthreads();  // a place is written when it has been read
      if (key && key >= low) sh.list[atomicAdd(&sh.count, 1)] = key;
    }
    __syncthreads();
    c = sh.count;
  }
  // ranks among the rest; the sorted ones go through `best`, n of which have room
  for (int i = tid; i < c; i += kBsRowThreads) {
    const uint64_t mine = sh.list[i];
    int above = 0;
#pragma unroll 4
    for (int j = 0; j + 1 < c; j += 2) {
      const ulonglong2 o = *reinterpret_cast<const ulonglong2 *>(&sh.list[j]);
      above += (o.x > mine) + (o.y > mine);
    }
    if (c & 1) above += sh.list[c - 1] > mine;
    if (above < n) sh.best[above] = mine;
  }
  __syncthreads();
  if (tid < min(c, n)) sh.list[tid] = sh.best[tid];
  if (tid == 0) sh.count = min(c, n);
  __syncthreads();
}

template <int DT>
__device__ __forceinline__ void bs_widen(const uint4 &u, float *x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (DT == KVR_F32) {
      x[j] = __uint_as_float(w[j]);
    } else if constexpr (DT == KVR_BF16) {
      x[2 * j] = __uint_as_float(w[j] << 16);
      x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
      x[2 * j] = f.x;
      x[2 * j + 1] = f.y;
    }
  }
}

// Sum of e^(x - from), two at a time in the packed instructions.
__device__ __forceinline__ float bs_sum(const float (&x)[kBsTile], float from) {
  uint64_t acc = 0, neg, log2e;
  asm("mov.b64 %0, {%1, %1};" : "=l"(neg) : "f"(-from));
  asm("mov.b64 %0, {%1, %1};" : "=l"(log2e) : "f"(1.4426950408889634f));
#pragma unroll
  for (int i = 0; i < kBsTile; i += 2) {
    uint64_t d;
    float lo, hi;
    // the difference first: as one fma of x, log2(e) and the scaled maximum, the maximum's rounding would be an error of
    // every term
    asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tadd.rn.f32x2 t, t, %3;\n\tmul.rn.f32x2 %0, t, %4;\n\t}"
        : "=l"(d)
        : "f"(x[i]), "f"(x[i + 1]), "l"(neg), "l"(log2e));
    asm("{\n\t.reg .f32 a, b;\n\tmov.b64 {a, b}, %2;\n\tex2.approx.ftz.f32 %0, a;\n\tex2.approx.ftz.f32 %1, b;\n\t}"
        : "=f"(lo), "=f"(hi)
        : "l"(d));
    asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tadd.rn.f32x2 %0, %0, t;\n\t}" : "+l"(acc) : "f"(lo), "f"(hi));
  }
  return __uint_as_float((uint32_t)acc) + __uint_as_float((uint32_t)(acc >> 32));
}

// A value that n logits of the tile's are not below, of the threads' maxima: the least of what the warps' k-th largest are,
// k warps' worth of n.  (The n-th largest of all threads' maxima is nearer, and takes a microsecond more.)
__device__ __forceinline__ float bs_first_limit(BeamShared &sh, float top, int n, int full_warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int k = (n + full_warps - 1) / full_warps;
  unsigned key = top > -INFINITY ? float_key(top) : 0, kth = 0;
  for (int i = 0; i < k && k <= 32; ++i) {
    kth = __reduce_max_sync(0xffffffffu, key);
    if (lane == __ffs(__ballot_sync(0xffffffffu, key == kth)) - 1) key = 0;
  }
  if (lane == 0) sh.m[warp] = kth ? key_float(kth) : -INFINITY;
  __syncthreads();
  float low = sh.m[0];
  for (int w = 1; w < full_warps; ++w) low = fminf(low, sh.m[w]);
  return fmaxf(low, -FLT_MAX);
}

template <int DT>
__global__ void __launch_bounds__(kBsRowThreads, 1024 / kBsRowThreads) beam_rows_kernel(BeamArgs a) {
  constexpr int kPer = DT == KVR_F32 ? 4 : 8, kSize = 16 / kPer;  // logits of a 16-byte granule, bytes of one
  constexpr int kVecs = kBsTile / kPer, kTile = kVecs * kBsRowThreads;
  __shared__ BeamShared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n;
  const int row = blockIdx.x / a.splits, split = blockIdx.x - row * a.splits;
  // The row's granules: rows need not start on one, so its first and last may hold logits of others, masked below.
  // (Every granule read holds one of the row's at least.)
  const char *base = static_cast<const char *>(a.logits) + (int64_t)row * a.row_stride * kSize;
  const int head = (int)((reinterpret_cast<uintptr_t>(base) & 15) / kSize);
  const uint4 *src = reinterpret_cast<const uint4 *>(base - head * kSize);
  const int granules = (int)(((int64_t)head + a.vocab + kPer - 1) / kPer);
  const int g0 = (int)((int64_t)granules * split / a.splits), g1 = (int)((int64_t)granules * (split + 1) / a.splits);
  if (tid == 0) sh.count = 0;
  griddep_wait();
  griddep_launch();
  uint64_t *out = a.cands + ((int64_t)row * a.splits + split) * n;
  // A beam that there is not (a first step has one of K, a request that has ended none): its row is not read.  (24 requests
  // of 8 beams, one each, 128256 logits in fp16: 22.5 -> 13.7 us.)
  if (!isfinite(a.cum[row])) {
    for (int i = tid; i < n; i += kBsRowThreads) out[i] = 0;
    if (tid == 0) a.ml[(int64_t)row * a.splits + split] = make_float2(0.0f, 1.0f);
    return;
  }
  const uint32_t pad = DT == KVR_F32 ? 0xff800000u : DT == KVR_BF16 ? 0xff80ff80u : 0xfc00fc00u;  // -inf
  // (fp32: the next tile's words; 16 bits: two tiles', as many)
  constexpr int kAhead = 4 / kVecs;
  uint4 next[kAhead][kVecs];
  auto fetch = [&](uint4 (&to)[kVecs], int at) {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      const int g = at + v * kBsRowThreads + tid;
      to[v] = g < g1 ? __ldcs(src + g) : make_uint4(pad, pad, pad, pad);
    }
  };
  float m = -INFINITY, s = 0.0f;
  // what a logit has to be above, or equal to with a lower token (warps are not at the same tile: a list's last entry may
  // be of a later one)
  float limit = -FLT_MAX;  // (so that -inf is below it)
  int limit_token = INT_MAX;
  // All warps cut the list and take over its limit; true when all of them are done.  They meet only for that: a warp that
  // starts a tile with too many entries in the list comes here, and so does one that is done, so each of the others adds
  // one tile at most, for which the list has room.  (A barrier a tile: 6 us more for 512 rows of 128256, and most of a warp's
  // time at it.)
  auto meet = [&](bool done) {
    const bool all = __syncthreads_and(done);
    bs_cut(sh, n);
    if (sh.count == n) {
      limit = bs_value(sh.list[n - 1]);
      limit_token = bs_token(sh.list[n - 1]);
    }
    __syncthreads();  // the count is read before any warp adds to it
    return all;
  };
  auto tile = [&](uint4 (&from)[kVecs], int at, bool first) {
    float x[kBsTile], tops[kBsTile / 4], top;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) bs_widen<DT>(from[v], x + v * kPer);
    auto token = [&](int i) { return (at + i / kPer * kBsRowThreads + tid) * kPer - head + i % kPer; };
    if (first || at + kTile >= g1) {
#pragma unroll
      for (int i = 0; i < kBsTile; ++i)
        if (token(i) < 0 || token(i) >= a.vocab) x[i] = -INFINITY;
    }
    if (at + kAhead * kTile < g1) fetch(from, at + kAhead * kTile);
#pragma unroll
    for (int q = 0; q < kBsTile / 4; ++q) {  // (a NaN is passed over here, not in the sum)
      tops[q] = bs_max3(x[4 * q], x[4 * q + 1], fmaxf(x[4 * q + 2], x[4 * q + 3]));
    }
    top = bs_max3(tops[0], tops[1], fmaxf(tops[2], tops[3]));
    if (top > m) {  // (rare after the first tiles)
      s *= bs_exp(m - top);
      m = top;
    }
    s += bs_sum(x, m == -INFINITY ? 0.0f : m);
    if (first) {
      limit = bs_first_limit(sh, top, n, max(1, min(kBsRowThreads, g1 - g0) / 32));
    }
    if (top >= limit) {
      unsigned which = 0;
#pragma unroll
      for (int i = 0; i < kBsTile; ++i) which |= (x[i] >= limit ? 1u : 0u) << i;
#pragma unroll 1
      for (; which; which &= which - 1) {
        const int i = __ffs(which) - 1, t = token(i);
        float y[kBsTile];
#pragma unroll
        for (int j = 0; j < kBsTile; ++j) y[j] = x[j];
#pragma unroll
        for (int o = kBsTile / 2; o > 0; o >>= 1)
#pragma unroll
          for (int j = 0; j < o; ++j) y[j] = i & o ? y[j + o] : y[j];
        if (y[0] > limit || t < limit_token) sh.list[atomicAdd(&sh.count, 1)] = bs_key(y[0], t);
      }
    }
    __syncwarp();
  };
#pragma unroll
  for (int d = 0; d < kAhead; ++d)
    if (g0 + d * kTile < g1) fetch(next[d], g0 + d * kTile);
  tile(next[0], g0, true);
  meet(false);
  if (g0 + kTile < g1) {
    for (int at = g0 + kTile; at < g1; at += kAhead * kTile) {
#pragma unroll
      for (int d = 0; d < kAhead; ++d)
        if (at + d * kTile < g1) {
          if (__any_sync(0xffffffffu, *static_cast<volatile int *>(&sh.count) > n + kBsSlack)) meet(false);
          tile(next[(d + 1) % kAhead], at + d * kTile, false);
        }
    }
    __syncwarp();
    while (!meet(true)) {
    }
  }
  for (int i = tid; i < n; i += kBsRowThreads) out[i] = i < sh.count ? sh.list[i] : 0;
  const float wm = warp_max(m);
  s *= bs_exp(m - (wm == -INFINITY ? 0.0f : wm));
  s = warp_sum(s);
  if (lane == 0) {
    sh.m[warp] = wm;
    sh.s[warp] = s;
  }
  __syncthreads();
  if (tid == 0) {
    float bm = -INFINITY, bs = 0.0f;
    for (int w = 0; w < kBsRowThreads / 32; ++w) bm = fmaxf(bm, sh.m[w]);
    for (int w = 0; w < kBsRowThreads / 32; ++w) bs += sh.s[w] * bs_exp(sh.m[w] - (bm == -INFINITY ? 0.0f : bm));
    a.ml[(int64_t)row * a.splits + split] = make_float2(bm, bs);
  }
}

// Order of scores: a 64-bit key of the score (0: no candidate), then beam and token.
struct __align__(16) BeamRank {
  uint64_t key, id;
};
// (Both halves in any case: a branch between them made a step of the ranking loops 100 cycles.)
__device__ __forceinline__ bool bs_above(const BeamRank &x, const BeamRank &y) {
  return (x.key > y.key) | ((x.key == y.key) & (x.id < y.id));
}
__device__ __forceinline__ uint64_t bs_double_key(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x == 0.0 ? 0.0 : x);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double bs_key_double(uint64_t k) {
  return __longlong_as_double((long long)((k >> 63) ? (k & 0x7fffffffffffffffull) : ~k));
}

__global__ void __launch_bounds__(kBsThreads) beam_merge_kernel(BeamArgs a) {
  extern __shared__ BeamRank all[];  // (beams, splits, n)
  __shared__ double lse[kBsMaxBeams];
  __shared__ float cum[kBsMaxBeams];
  __shared__ BeamRank best[kBsThreads], picked[kBsPicked], sorted[kBsMaxN], nth;
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x, n = a.n, K = a.beams;
  const int per_beam = a.splits * n, total = K * per_beam, groups = bs_groups(n);
  if (tid == 0) {
    count = 0;
    nth = BeamRank{0, 0};
  }
  if (tid < n) sorted[tid] = BeamRank{0, 0};
  griddep_wait();
  griddep_launch();
  constexpr int kAhead = 4;  // candidates that a thread asks for while the sums are joined
  const uint64_t *cands = a.cands + (int64_t)b * total;
  uint64_t ahead[kAhead];
#pragma unroll
  for (int r = 0; r < kAhead; ++r) ahead[r] = tid + r * kBsThreads < total ? cands[tid + r * kBsThreads] : 0;
  for (int k = warp; k < K; k += kBsThreads / 32) {  // a beam's sums, in 64 bits
    const float2 *ml = a.ml + ((int64_t)b * K + k) * a.splits;
    const float c = a.cum[(int64_t)b * K + k];
    float m = -INFINITY;
    for (int i = lane; i < a.splits; i += 32) m = fmaxf(m, ml[i].x);
    m = warp_max(m);
    const float from = m == -INFINITY ? 0.0f : m;
    double s = 0.0;
    for (int i = lane; i < a.splits; i += 32) s += (double)ml[i].y * (double)expf(ml[i].x - from);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) {
      lse[k] = (double)m + log(s);
      cum[k] = c;
    }
  }
  __syncthreads();
  BeamRank mine{0, 0};
  auto enter = [&](int i, uint64_t c) {
    const int k = i / per_beam;
    BeamRank r{0, 0};
    if (c) {
      const double score = (double)cum[k] + ((double)bs_value(c) - lse[k]);
      if (isfinite((float)score)) r = BeamRank{bs_double_key(score), (uint64_t)k << 32 | (uint32_t)bs_token(c)};
    }
    all[i] = r;
    if (r.key && bs_above(r, mine)) mine = r;
  };
#pragma unroll
  for (int r = 0; r < kAhead; ++r)
    if (tid + r * kBsThreads < total) enter(tid + r * kBsThreads, ahead[r]);
  for (int i = tid + kAhead * kBsThreads; i < total; i += kBsThreads) enter(i, cands[i]);
  // a threshold, where there are many: the n-th largest of groups' maxima
  if (total > kBsThreads / 2) {
    const int each = kBsThreads / groups;
    for (int o = 1; o < each; o <<= 1) {
      const BeamRank r{__shfl_xor_sync(0xffffffffu, mine.key, o), __shfl_xor_sync(0xffffffffu, mine.id, o)};
      if (r.key && (!mine.key || bs_above(r, mine))) mine = r;
    }
    if (tid % each == 0) best[tid / each] = mine;
    __syncthreads();
    if (tid < groups) {
      mine = best[tid];
      int above = 0;
#pragma unroll 8
      for (int i = 0; i < groups; ++i) above += bs_above(best[i], mine);
      if (mine.key && above == n - 1) nth = mine;
    }
    __syncthreads();
    const BeamRank low = nth;
    for (int i = tid; i < total; i += kBsThreads) {
      const BeamRank r = all[i];
      if (r.key && !bs_above(low, r)) {
        const int at = atomicAdd(&count, 1);
        if (at < kBsPicked) picked[at] = r;
      }
    }
  }
  __syncthreads();
  const BeamRank low = nth;
  // ranks: among those picked or, where they are too many for the list, among all
  const bool few = total > kBsThreads / 2 && count <= kBsPicked;
  const BeamRank *from = few ? picked : all;
  const int m = few ? count : total;
  for (int i = tid; i < m; i += kBsThreads) {
    const BeamRank r = from[i];
    if (!r.key || bs_above(low, r)) continue;
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < m; ++j) above += bs_above(from[j], r);
    if (above < n) sorted[above] = r;
  }
  __syncthreads();
  if (tid < n) {
    const BeamRank r = sorted[tid];
    const int64_t o = (int64_t)b * n + tid;
    a.scores[o] = r.key ? (float)bs_key_double(r.key) : -INFINITY;
    a.out_beams[o] = r.key ? (int)(r.id >> 32) : -1;
    a.tokens[o] = r.key ? (int)(uint32_t)r.id : -1;
  }
  // the first K that do not end a sequence go on
  if (warp == 0) {
    int taken = 0;
    for (int i0 = 0; i0 < n && taken < K; i0 += 32) {
      const int i = i0 + lane;
      const BeamRank r = i < n ? sorted[i] : BeamRank{0, 0};
      bool on = r.key != 0;
      for (int e = 0; e < a.n_eos; ++e) on = on && (int)(uint32_t)r.id != a.eos[e];
      const unsigned who = __ballot_sync(0xffffffffu, on);
      const int to = taken + __popc(who & ((1u << lane) - 1));
      if (on && to < K) {
        a.next_scores[(int64_t)b * K + to] = (float)bs_key_double(r.key);
        a.next_beams[(int64_t)b * K + to] = (int)(r.id >> 32);
        a.next_tokens[(int64_t)b * K + to] = (int)(uint32_t)r.id;
      }
      taken += __popc(who);
    }
    for (int k = taken + lane; k < K; k += 32) {
      a.next_scores[(int64_t)b * K + k] = -INFINITY;
      a.next_beams[(int64_t)b * K + k] = -1;
      a.next_tokens[(int64_t)b * K + k] = -1;
    }
  }
}

// Segments of a row: enough CTAs for every SM to hold several at a time, none below a tile's worth of 16-byte
// granules / 2, and no more candidates than the second kernel has room for.
int beam_splits(int64_t rows, int beams, int n, int64_t vocab, int dtype) {
  const int64_t granules = (vocab * (int64_t)dtype_size(dtype) + 15) / 16;
  int64_t s = (148 * 3 + rows - 1) / rows;
  if (s > (granules + 511) / 512) s = (granules + 511) / 512;
  if (s > kBsMaxCands / (beams * n)) s = kBsMaxCands / (beams * n);
  return (int)(s < 1 ? 1 : s);
}

}  // namespace kvr

using namespace kvr;

extern "C" size_t kvr_beam_select_workspace_bytes(int batch, int n_beams, int64_t vocab, int dtype, int n) {
  if (batch < 1 || n_beams < 1 || n_beams > kBsMaxBeams || n < 1 || n > kBsMaxN || vocab < 1 || !valid_dtype(dtype)) return 0;
  const int64_t rows = (int64_t)batch * n_beams;
  return (size_t)rows * beam_splits(rows, n_beams, n, vocab, dtype) * (n + 1) * 8;
}

extern "C" int kvr_beam_select(const void *logits, int dtype, int64_t row_stride, int batch, int n_beams, int64_t vocab,
                               const float *cum, int n, const int32_t *eos_host, int n_eos, float *scores, int32_t *beams,
                               int32_t *tokens, float *next_scores, int32_t *next_beams, int32_t *next_tokens,
                               void *workspace, size_t workspace_bytes, kvr_stream_t stream) {
  clear_error();
  KVR_REQUIRE(batch >= 0 && n_beams >= 1 && n >= n_beams && vocab >= 1 && vocab <= INT_MAX / 2 && n_eos >= 0,
              "kvr_beam_select: bad shape");
  if (n_beams > kBsMaxBeams || n > kBsMaxN || n_eos > kBsMaxEos)
    return set_error(KVR_ENOTSUP, "kvr_beam_select: at most %d beams, %d candidates, %d ends of sequence", kBsMaxBeams,
                     kBsMaxN, kBsMaxEos);
  KVR_REQUIRE(valid_dtype(dtype), "kvr_beam_select: bad dtype");
  if (batch == 0) return KVR_OK;
  KVR_REQUIRE(logits && cum && scores && beams && tokens && next_scores && next_beams && next_tokens && workspace &&
                  (!n_eos || eos_host),
              "kvr_beam_select: null pointer");
  const int64_t rows = (int64_t)batch * n_beams;
  KVR_REQUIRE(row_stride >= 0 || rows == 1, "kvr_beam_select: bad row stride");
  KVR_REQUIRE(reinterpret_cast<uintptr_t>(logits) % dtype_size(dtype) == 0 && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
              "kvr_beam_select: pointers must be aligned");
  const int splits = beam_splits(rows, n_beams, n, vocab, dtype);
  KVR_REQUIRE(workspace_bytes >= kvr_beam_select_workspace_bytes(batch, n_beams, vocab, dtype, n),
              "kvr_beam_select: workspace too small");
  KVR_REQUIRE(rows * splits <= INT_MAX, "kvr_beam_select: too many rows");
  BeamArgs a{};
  a.logits = logits; a.row_stride = row_stride;
  a.rows = (int)rows; a.beams = n_beams; a.n = n; a.splits = splits; a.vocab = (int)vocab;
  a.cum = cum;
  a.cands = static_cast<uint64_t *>(workspace);
  a.ml = reinterpret_cast<float2 *>(a.cands + rows * splits * n);
  a.scores = scores; a.out_beams = beams; a.tokens = tokens;
  a.next_scores = next_scores; a.next_beams = next_beams; a.next_tokens = next_tokens;
  a.n_eos = n_eos;
  for (int e = 0; e < n_eos; ++e) a.eos[e] = eos_host[e];
  const unsigned grid = (unsigned)(rows * splits);
  cudaError_t e = launch_dependent(dtype == KVR_F32   ? beam_rows_kernel<KVR_F32>
                                   : dtype == KVR_F16 ? beam_rows_kernel<KVR_F16>
                                                      : beam_rows_kernel<KVR_BF16>,
                                   grid, kBsRowThreads, 0, as_cuda(stream), a);
  if (e != cudaSuccess) return set_error(KVR_ECUDA, "kvr_beam_select: %s", cudaGetErrorString(e));
  const size_t smem = (size_t)n_beams * splits * n * sizeof(BeamRank);
  if (smem > 8 * 1024) {
    // 48 KB without asking, of which the fixed arrays take 23
    e = cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBsMaxCands * (int)sizeof(BeamRank));
    if (e != cudaSuccess) return set_error(KVR_ECUDA, "kvr_beam_select: %s", cudaGetErrorString(e));
  }
  e = launch_dependent(beam_merge_kernel, (unsigned)batch, kBsThreads, smem, as_cuda(stream), a);
  if (e != cudaSuccess) return set_error(KVR_ECUDA, "kvr_beam_select: %s", cudaGetErrorString(e));
  return check_launch("kvr_beam_select");
}
