// Block tables, slot maps and attention plans from request lengths.
//
// A serving step appends new_len[b] tokens to request b, which has ctx_len[b]
// in the cache.  With pages of P tokens the request holds ceil(ctx/P) pages
// and needs ceil((ctx+new)/P); the fresh ones come off the end of the free
// list in request order, so page k of the step (exclusive sum of the needs
// plus its index) is free[n_free - 1 - k] and no page needs an atomic.  Token
// i lies at position p = ctx + i - cu[b] and in slot table[b][p/P] * P + p%P.
// A request takes no page that its table row has no entry for, and its tokens
// without a page are its last ones, so the keys it has after the step are the
// first kv_len: ctx + new, or as many as its pages hold.
//
// One launch does all of it.  Every CTA forms the two prefix sums (tokens,
// fresh pages) of all requests in shared memory by itself: two words per
// request from L2 are cheaper than a second kernel that waits for a first.
// CTA 0 then writes the per-request outputs and the attention plan, the others
// take the tokens and fresh pages.  Tokens in fresh pages read the free list,
// not the table that other CTAs are filling.  The work is a few hundred bytes
// to a few MB: launch and dependent-load latency bound it (32 decode requests, in
// a graph: 4.8 us, 12 with their plan; a call from the host takes 21).
#include "kvr_attn_plan.cuh"

namespace kvr {

// Exclusive sum over the CTA of one value per thread; `total` is the sum.
__device__ __forceinline__ int64_t block_exclusive(int64_t v, int64_t *warp_sums, int64_t &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int64_t s = lane < nw ? warp_sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  total = warp_sums[31];
  return x - v + (warp ? warp_sums[warp - 1] : 0);
}

// Largest i in [0, n) with a[i] <= x (a ascending, a[0] <= x).
__device__ __forceinline__ int last_not_above(const int *a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One request as the plan sees it; b == batch stands for the tokens past the
// last request (padding: no keys, their rows come out as zeros).
struct PlanRequest {
  int q0, q_len, kv_len, k_start;
  int first;  // keys before its first query
};
__device__ __forceinline__ PlanRequest plan_request(const PlanArgs &a, int b) {
  PlanRequest r;
  const int lo = min(max(a.cu_q[b], 0), a.n_tokens);
  const int hi = b < a.batch ? min(max(a.cu_q[b + 1], lo), a.n_tokens) : a.n_tokens;
  r.q0 = lo;
  r.q_len = hi - lo;
  if (b == a.batch) {
    r.kv_len = 0;
    r.k_start = 0;
  } else if (a.kv_len) {
    r.kv_len = min(max(a.kv_len[b], 0), 2 * kPlanMaxLen);
    r.k_start = b;
  } else if (a.cu_k) {
    r.k_start = max(a.cu_k[b], 0);
    r.kv_len = min(max(a.cu_k[b + 1] - r.k_start, 0), 2 * kPlanMaxLen);
  } else {
    r.k_start = lo;
    r.kv_len = r.q_len;
  }
  r.first = a.ctx && b < a.batch ? min(max(a.ctx[b], 0), kPlanMaxLen) : r.kv_len - r.q_len;
  return r;
}

// Item i of request r: its piece record over all the K/V tiles it needs.
__device__ __forceinline__ PlanPiece plan_item(const PlanArgs &a, const PlanRequest &r, int i) {
  const int per = 2 * plan_tpt(a.n_q, a.n_kv);
  PlanPiece p;
  p.q_start = r.q0 + i * per;
  p.n_tok = max(0, min(per, r.q_len - i * per));
  p.kv_len = r.kv_len;
  p.k_start = r.k_start;
  p.part = -1;
  p.first_end = a.causal ? r.first + i * per + 1 : r.kv_len;
  const int64_t end = a.causal ? min((int64_t)r.kv_len, (int64_t)p.first_end + p.n_tok - 1) : r.kv_len;
  const int64_t begin = a.window > 0 ? max((int64_t)0, (int64_t)p.first_end - a.window) : 0;
  p.kt0 = (int)(begin / kPlanKeys);
  p.kt1 = end > begin ? (int)((end + kPlanKeys - 1) / kPlanKeys) : p.kt0;
  return p;
}

constexpr int kPlanBins = 1024;
constexpr int kPlanCands = 32;

struct PlanShared {
  int first[kPlanMaxBatch + 2];  // exclusive sum of the requests' items
  int hist[kPlanBins];           // items of each length
  int rows[kPlanBins];           // their query rows
  int place[kPlanBins];          // next list entry of each piece length
  int64_t warp_sums[32];
  float time[kPlanCands];        // estimate of each candidate
  int longest_kv, longest, n_splits, n_rows;
  int ahead[kPlanCtas + 1];      // even plan: exclusive sum of the items' K/V tiles
};

// Candidate lengths of the longest piece: the longest item in k parts.
__device__ __constant__ short kPlanParts[kPlanCands] = {1,  2,  3,  4,  5,  6,  7,  8,  9,  10, 11, 12, 14, 16, 18, 20,
                                                        22, 24, 28, 32, 36, 42, 48, 56, 64, 74, 84, 96, 112, 128, 148, 296};

// Estimated time, in K/V tiles, with `count` pieces of at most `len` tiles per
// head and `rows` partial rows: a piece costs about one tile to fill and drain,
// a partial tile of 256 rows about two more to write and join, joining at all
// about three (a second launch).  Pieces beyond a full round of the SMs leave
// the last round partly empty; the more unequal the pieces are, the better the
// short ones fill it, which the fourth power of mean / longest stands for.
__device__ __forceinline__ float plan_estimate(float work, float count, float rows, int len, int n_kv) {
  const float pieces = count * n_kv, top = len + 1.0f;
  const float total = (work + count + rows * (2.0f / 256.0f)) * n_kv;
  const float joined = rows > 0.0f ? 3.0f : 0.0f;
  if (pieces <= kPlanCtas) return top + joined + (rows > 0.0f ? 2.0f * fminf(1.0f, rows / (256.0f * count)) : 0.0f);
  const float rounds = pieces / kPlanCtas, mean = total / pieces, u = fminf(1.0f, mean / top);
  return joined + fmaxf(top, total / kPlanCtas + (ceilf(rounds) - rounds) * mean * u * u * u * u);
}

__device__ __forceinline__ void plan_header(const PlanArgs &a, int n_pieces, int n_splits, int part_rows, int dropped,
                                            int even) {
  PlanHeader &h = *a.hdr;
  h.magic = kPlanMagic;
  h.n_tokens = a.n_tokens;
  h.batch = a.batch;
  h.n_q = a.n_q;
  h.n_kv = a.n_kv;
  h.causal = a.causal;
  h.window = a.window;
  h.n_pieces = n_pieces;
  h.n_splits = n_splits;
  h.part_rows = part_rows;
  h.dropped = dropped;
  h.even = even;
}

// The even plan for n items (at most one per CTA and head, item tid in `mine`);
// false, with nothing written, where the best of the candidates is as good.
__device__ bool plan_even(const PlanArgs &a, PlanShared &s, int n, const PlanPiece &mine, int longest) {
  const int tid = threadIdx.x, lane = tid & 31;
  const int len = tid < n ? mine.kt1 - mine.kt0 : 0;
  int64_t sum;
  const int at = (int)min(block_exclusive(len, s.warp_sums, sum), (int64_t)(INT_MAX / 1024));
  if (tid <= n) s.ahead[tid] = at;  // thread n: the sum of all
  __syncthreads();
  const int64_t work = sum * a.n_kv;
  float best = s.time[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = fminf(best, __shfl_xor_sync(0xffffffffu, best, o));
  // a CTA has two pieces more often than not: a tile each to fill and drain, two for partial rows, three to join
  const float even = (float)((work + kPlanCtas - 1) / kPlanCtas) + 2.0f + 2.0f + 3.0f;
  if (work > INT_MAX / 2 || !(even < best)) return false;
  // CTA c: tiles [lo, hi) of the row of all items, heads innermost; at most kRounds pieces
  constexpr int kRounds = (kPlanExtra + 2) / kPlanCtas;
  const int c = tid;
  int lo = 0, hi = 0, item = 0, head = 0, rounds = 0;
  if (c < kPlanCtas) {
    lo = (int)(work * c / kPlanCtas);
    hi = (int)(work * (c + 1) / kPlanCtas);
    // an item's heads follow one another, len tiles each, from n_kv * ahead on
    item = last_not_above(s.ahead, n, lo / a.n_kv);
    while (item + 1 < n && s.ahead[item + 1] * a.n_kv <= lo) ++item;
    const int il = s.ahead[item + 1] - s.ahead[item];
    head = il > 0 ? (lo - s.ahead[item] * a.n_kv) / il : 0;
    // how many pieces that makes
    int pos = lo, it = item, hd = head;
    while (pos < hi) {
      const int l1 = s.ahead[it + 1] - s.ahead[it], end = s.ahead[it] * a.n_kv + (hd + 1) * l1;
      if (l1 > 0) {
        pos = min(hi, end);
        ++rounds;
      }
      if (l1 == 0 || pos == end) {
        if (l1 == 0 || ++hd == a.n_kv) {
          hd = 0;
          ++it;
        }
      }
    }
  }
  // items without tiles still need their zero rows: leave those calls, and ranges of many items, to the candidates
  const int empty = tid < n && len == 0;
  const int most = (int)__reduce_max_sync(0xffffffffu, empty ? kRounds + 1 : rounds);
  if (tid == 0) s.n_rows = 0;
  __syncthreads();
  if (lane == 0) atomicMax(&s.n_rows, most);
  __syncthreads();
  const int n_rounds = s.n_rows;
  __syncthreads();
  if (tid == 0) s.n_rows = 0;
  if (n_rounds > kRounds) return false;
  if (c < kPlanCtas) {
    int pos = lo;
    for (int r = 0; r < n_rounds; ++r) {
      PlanPiece p{};
      if (pos < hi) {
        while (s.ahead[item + 1] == s.ahead[item]) ++item;
        const int l1 = s.ahead[item + 1] - s.ahead[item], begin = s.ahead[item] * a.n_kv + head * l1, end = begin + l1;
        const int to = min(hi, end);
        const int b = last_not_above(s.first, a.batch + 1, item);
        p = plan_item(a, plan_request(a, b), item - s.first[b]);
        const int kt0 = p.kt0, slot = 2 * c + (pos > lo ? 1 : 0);
        const bool cut = pos > begin || to < end;
        p.n_tok |= head << 16;
        p.kt0 = kt0 + pos - begin;
        p.kt1 = kt0 + to - begin;
        p.part = cut ? slot * 2 * kPlanRows : -1;
        if (cut && pos == begin) {  // the CTA with an item's first piece enters the item
          // its last tile, end - 1, is CTA l's for the l with work * l / G <= end - 1 < work * (l + 1) / G
          int l = (int)((int64_t)(end - 1) * kPlanCtas / work);
          while ((int)(work * (l + 1) / kPlanCtas) <= end - 1) ++l;
          while ((int)(work * l / kPlanCtas) > end - 1) --l;
          a.splits[atomicAdd(&s.n_splits, 1)] = PlanSplit{p.q_start, p.n_tok, p.part, l - c + 1};
        }
        pos = to;
        if (to == end && ++head == a.n_kv) {
          head = 0;
          ++item;
        }
      }
      a.pieces[r * kPlanCtas + ((r & 1) ? kPlanCtas - 1 - c : c)] = p;
    }
  }
  __syncthreads();
  if (tid == 0) plan_header(a, n_rounds * kPlanCtas, s.n_splits, 0, 0, 1);
  return true;
}

// One CTA.  Two passes over the items (their lengths; their places), an item
// per thread; in between a warp per candidate length goes over the histogram of
// lengths, not over the items.  Atomics on shared counters are made once per
// warp and value: 700 items of one length on one counter cost more than all of
// the rest (map of 48 prompts in a graph: 50 us with an atomic per item and
// candidate sums over the items, 14.7 us this way).
__device__ void plan_build(const PlanArgs &a, PlanShared &s) {
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int g = a.n_q / a.n_kv, per = 2 * plan_tpt(a.n_q, a.n_kv);
  const int nb = a.batch + 1;
  s.hist[tid] = s.rows[tid] = s.place[tid] = 0;
  if (tid == 0) s.longest_kv = s.longest = s.n_splits = s.n_rows = 0;
  // requests -> first item of each (a contiguous run of requests per thread)
  const int each = (nb + nt - 1) / nt;
  int64_t sum = 0, total;  // 64 bits: offsets that overlap can add up to more than 2^31 items
  int most = 0;
  for (int k = 0; k < each; ++k) {
    const int b = tid * each + k;
    if (b < nb) {
      const PlanRequest r = plan_request(a, b);
      sum += (r.q_len + per - 1) / per;
      if (r.q_len > 0) most = max(most, r.kv_len);
    }
  }
  int64_t at = block_exclusive(sum, s.warp_sums, total);
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) atomicMax(&s.longest_kv, most);
  for (int k = 0; k < each; ++k) {
    const int b = tid * each + k;
    if (b < nb) {
      s.first[b] = (int)min(at, (int64_t)INT_MAX);
      if (each > 1) at += (plan_request(a, b).q_len + per - 1) / per;
    }
  }
  __syncthreads();
  const int n = (int)min(total, (int64_t)a.max_items);
  const int dropped = total > n ? 1 : 0;
  int shift = 0;  // lengths of 2^shift share a bin and count as the longest of them
  while (((s.longest_kv / kPlanKeys + 1) >> shift) >= kPlanBins) ++shift;
  auto item = [&](int i) {
    const int b = last_not_above(s.first, nb, i);
    return plan_item(a, plan_request(a, b), i - s.first[b]);
  };
  const PlanPiece mine = tid < n ? item(tid) : PlanPiece{};
  for (int i0 = 0; i0 < n; i0 += nt) {
    const int i = i0 + tid;
    int len = 0;
    if (i < n) {
      const PlanPiece p = i0 ? item(i) : mine;
      len = p.kt1 - p.kt0;
      const unsigned same = __match_any_sync(__activemask(), len >> shift);
      const int rows = (int)__reduce_add_sync(same, (unsigned)(p.n_tok * g));
      if (lane == __ffs(same) - 1) {
        atomicAdd(&s.hist[len >> shift], __popc(same));
        atomicAdd(&s.rows[len >> shift], rows);
      }
    }
    len = __reduce_max_sync(0xffffffffu, len);
    if (lane == 0) atomicMax(&s.longest, len);
  }
  __syncthreads();
  const int longest = s.longest, low = (1 << shift) - 1;
  // the length an item counts as: the longest of its bin, but none longer than the longest item (which the first
  // candidate has to leave whole: only so does its list always fit)
  auto counted = [&](int len) { return min(len | low, longest); };
  {  // warp c: candidate c
    const int top = max(1, (longest + kPlanParts[warp] - 1) / kPlanParts[warp]);
    float work = 0.0f, count = 0.0f, rows = 0.0f;
    for (int bin = lane; bin <= longest >> shift; bin += 32) {
      const int items = s.hist[bin], len = counted(bin << shift);
      if (items == 0) continue;
      const int np = max(1, (len + top - 1) / top);
      work += (float)items * len;
      count += (float)items * np;
      if (np > 1) rows += (float)s.rows[bin] * np;
    }
    work = warp_sum(work);
    count = warp_sum(count);
    rows = warp_sum(rows);
    // a list too long for the plan or rows too many for the workspace (with a margin for the fp32 sums) are refused
    const bool fits = warp == 0 || (count - n <= kPlanExtra - 1 && rows * a.n_kv <= kPartRows * 0.999f);
    if (lane == 0) s.time[warp] = fits ? plan_estimate(work, count, rows, top, a.n_kv) : INFINITY;
  }
  __syncthreads();
  if ((int64_t)n * a.n_kv <= kPlanCtas && plan_even(a, s, n, mine, longest)) return;
  float best = s.time[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = fminf(best, __shfl_xor_sync(0xffffffffu, best, o));
  const int parts = kPlanParts[__ffs(__ballot_sync(0xffffffffu, s.time[lane] == best)) - 1];
  const int top = max(1, (longest + parts - 1) / parts);
  // longest pieces first: counting sort by the pieces' length (thread = bin of item lengths here)
  auto pieces_of = [&](int len) { return max(1, (counted(len) + top - 1) / top); };
  auto place_of = [&](int len, int np) { return kPlanBins - 1 - (((counted(len) + np - 1) / np) >> shift); };
  if (s.hist[tid]) {
    const int len = tid << shift, np = pieces_of(len);
    atomicAdd(&s.place[place_of(len, np)], s.hist[tid] * np);
  }
  __syncthreads();
  const int start = (int)block_exclusive(s.place[tid], s.warp_sums, total);
  s.place[tid] = start;
  __syncthreads();
  for (int i = tid; i < n; i += nt) {
    PlanPiece p = i == tid ? mine : item(i);
    const int len = p.kt1 - p.kt0, np = pieces_of(len), to_bin = place_of(len, np), kt0 = p.kt0;
    if (np == 1 && parts == 1) {
      const unsigned same = __match_any_sync(__activemask(), to_bin);
      int to = 0;
      if (lane == __ffs(same) - 1) to = atomicAdd(&s.place[to_bin], __popc(same));
      to = __shfl_sync(same, to, __ffs(same) - 1) + __popc(same & ((1u << lane) - 1));
      a.pieces[to] = p;
      continue;
    }
    const int to = atomicAdd(&s.place[to_bin], np);
    int part = -1;
    if (np > 1) {
      part = atomicAdd(&s.n_rows, np * p.n_tok * g);
      a.splits[atomicAdd(&s.n_splits, 1)] = PlanSplit{p.q_start, p.n_tok, part, np};
    }
    for (int k = 0; k < np; ++k) {
      p.kt0 = kt0 + (int)((int64_t)len * k / np);
      p.kt1 = kt0 + (int)((int64_t)len * (k + 1) / np);
      p.part = part < 0 ? -1 : part + k * p.n_tok * g;
      a.pieces[to + k] = p;
    }
  }
  __syncthreads();
  if (tid == 0) plan_header(a, (int)total, s.n_splits, s.n_rows, dropped, 0);
}
static_assert(kPlanCands == kPlanThreads / 32, "one candidate per warp");
static_assert(kPlanBins == kPlanThreads, "one bin per thread in the scan");

__global__ void __launch_bounds__(kPlanThreads, 1) attn_plan_kernel(PlanArgs a) {
  __shared__ PlanShared s;
  griddep_wait();
  griddep_launch();
  plan_build(a, s);
}

struct MapArgs {
  const int *ctx_len, *new_len;
  int batch, n_tokens, page;
  int *table;
  int64_t table_stride;
  int table_width;
  const int *free_pages, *n_free;
  int n_free_cap;  // entries of free_pages
  int *cu, *kv_len, *positions;
  int64_t *slots;
  int *n_free_out, *info;
  PlanArgs plan;
  int with_plan;
};

// Cached tokens of request b (a length that no cache can have counts as its bound).
__device__ __forceinline__ int map_ctx(const MapArgs &a, int b) { return min(max(a.ctx_len[b], 0), kPlanMaxLen); }
// Fresh pages of a request that goes from ctx to kv tokens: those that its table row has entries for.
__device__ __forceinline__ int map_fresh(const MapArgs &a, int ctx, int kv) {
  const int P = a.page, W = a.table_width;
  return min((kv + P - 1) / P, W) - min((ctx + P - 1) / P, W);
}

__global__ void __launch_bounds__(kPlanThreads, 1) paged_map_kernel(MapArgs a) {
  __shared__ int cu[kPlanMaxBatch + 1];
  __shared__ union {
    int fresh[kPlanMaxBatch + 1];  // exclusive sum of the fresh pages
    PlanShared plan;
  } s;
  __shared__ int64_t warp_sums[32];
  __shared__ int n_cut, n_over, n_beyond;
  int *fresh = s.fresh;
  const int tid = threadIdx.x, nt = blockDim.x, P = a.page;
  griddep_wait();
  griddep_launch();
  if (tid == 0) n_cut = n_over = n_beyond = 0;
  const int each = (a.batch + nt - 1) / nt;
  // tokens first: requests are cut where the step's n_tokens end
  int64_t sum = 0, total;
  for (int k = 0; k < each; ++k) {
    const int b = tid * each + k;
    if (b < a.batch) sum += max(a.new_len[b], 0);
  }
  int64_t at = block_exclusive(sum, warp_sums, total);
  for (int k = 0; k < each; ++k) {
    const int b = tid * each + k;
    if (b < a.batch) {
      cu[b] = (int)min(at, (int64_t)a.n_tokens);
      at += max(a.new_len[b], 0);
    }
  }
  if (tid == 0) cu[a.batch] = (int)min(total, (int64_t)a.n_tokens);
  __syncthreads();
  sum = 0;
  for (int k = 0; k < each; ++k) {
    const int b = tid * each + k;
    if (b < a.batch) {
      const int ctx = map_ctx(a, b), kv = ctx + cu[b + 1] - cu[b];
      sum += map_fresh(a, ctx, kv);
    }
  }
  at = block_exclusive(sum, warp_sums, total);
  const int need = (int)total;
  for (int k = 0; k < each; ++k) {
    const int b = tid * each + k;
    if (b < a.batch) {
      const int ctx = map_ctx(a, b), kv = ctx + cu[b + 1] - cu[b];
      fresh[b] = (int)at;
      at += map_fresh(a, ctx, kv);
    }
  }
  if (tid == 0) fresh[a.batch] = need;
  __syncthreads();
  const int n_free = min(max(*a.n_free, 0), a.n_free_cap);
  if (blockIdx.x == 0) {
    for (int b = tid; b < a.batch; b += nt) {
      const int ctx = map_ctx(a, b), now = cu[b + 1] - cu[b], had = (ctx + P - 1) / P, pages = (ctx + now + P - 1) / P;
      a.cu[b] = cu[b];
      if (max(a.new_len[b], 0) > now) atomicAdd(&n_cut, 1);
      if (pages > a.table_width) {
        atomicAdd(&n_over, 1);
        atomicAdd(&n_beyond, pages - max(had, a.table_width));
      }
      const int want = map_fresh(a, ctx, ctx + now), got = min(want, max(n_free - fresh[b], 0));
      int kv = ctx + now;
      if (got < want || pages > a.table_width)
        kv = (int)min((int64_t)kv, max((int64_t)ctx, (int64_t)(min(had, a.table_width) + got) * P));
      a.kv_len[b] = kv;
    }
    __syncthreads();  // cu and kv_len are in place for the plan as well
    if (tid == 0) {
      a.cu[a.batch] = cu[a.batch];
      *a.n_free_out = max(n_free - need, 0);
      a.info[0] = max(need + n_beyond - n_free, 0);
      a.info[1] = n_cut;
      a.info[2] = n_over;
      a.info[3] = 0;
    }
    __syncthreads();
    if (a.with_plan) plan_build(a.plan, s.plan);
    return;
  }
  const int64_t step = (int64_t)(gridDim.x - 1) * nt, me = (int64_t)(blockIdx.x - 1) * nt + tid;
  for (int64_t i = me; i < a.n_tokens; i += step) {
    int pos = 0;
    int64_t slot = -1;
    if (i < cu[a.batch]) {
      // the last request that starts at or before token i and is not empty owns it
      const int b = last_not_above(cu, a.batch, (int)i);
      const int ctx = map_ctx(a, b), had = (ctx + P - 1) / P;
      pos = ctx + (int)i - cu[b];
      const int j = pos / P;
      if (j < a.table_width) {
        int page = -1;
        if (j < had) {
          page = a.table[b * a.table_stride + j];
        } else {
          const int k = fresh[b] + j - had;
          if (k < n_free) page = a.free_pages[n_free - 1 - k];
        }
        if (page >= 0) slot = (int64_t)page * P + pos % P;
      }
    }
    a.positions[i] = pos;
    a.slots[i] = slot;
  }
  for (int64_t k = me; k < need; k += step) {
    const int b = last_not_above(fresh, a.batch, (int)k);
    const int ctx = map_ctx(a, b);
    const int j = (ctx + P - 1) / P + (int)k - fresh[b];
    if (j < a.table_width) a.table[b * a.table_stride + j] = k < n_free ? a.free_pages[n_free - 1 - k] : -1;
  }
}

int plan_check(const char *fn, PlanArgs &a, int64_t n_tokens, int64_t window, void *plan, size_t plan_bytes) {
  KVR_REQUIRE(a.batch >= 1 && a.batch <= kPlanMaxBatch, "%s: batch must be in [1, %d]", fn, kPlanMaxBatch);
  KVR_REQUIRE(n_tokens >= 0 && n_tokens <= kPlanMaxTokens, "%s: bad token count", fn);
  KVR_REQUIRE(a.n_kv > 0 && a.n_q > 0 && a.n_q % a.n_kv == 0, "%s: n_q must be a multiple of n_kv", fn);
  if (a.n_q / a.n_kv > kPlanRows)
    return set_error(KVR_ENOTSUP, "%s: more than %d query heads per KV head", fn, kPlanRows);
  KVR_REQUIRE(window >= 0, "%s: window must be >= 0 (0: none)", fn);
  KVR_REQUIRE(a.causal || window == 0, "%s: a window needs causal", fn);
  KVR_REQUIRE(plan && (reinterpret_cast<uintptr_t>(plan) & 15) == 0, "%s: plan must be 16-byte aligned", fn);
  const size_t want = kvr_attn_plan_bytes(n_tokens, a.batch, a.n_q, a.n_kv);
  KVR_REQUIRE(plan_bytes >= want, "%s: plan %zu < %zu bytes", fn, plan_bytes, want);
  a.n_tokens = (int)n_tokens;
  a.window = (int)(window > INT_MAX / 2 ? 0 : window);
  a.hdr = reinterpret_cast<PlanHeader *>(plan);
  a.pieces = reinterpret_cast<PlanPiece *>(a.hdr + 1);
  a.max_items = (int)plan_max_items(n_tokens, a.batch, a.n_q, a.n_kv);
  a.splits = const_cast<PlanSplit *>(plan_splits(a.hdr, n_tokens, a.batch, a.n_q, a.n_kv));
  return KVR_OK;
}

}  // namespace kvr

using namespace kvr;

extern "C" size_t kvr_attn_plan_bytes(int64_t n_tokens, int batch, int n_q, int n_kv) {
  if (n_tokens < 0 || batch < 1 || n_kv < 1 || n_q < n_kv || n_q / n_kv > kPlanRows) return 0;
  return sizeof(PlanHeader) + (size_t)(plan_max_items(n_tokens, batch, n_q, n_kv) + kPlanExtra) * sizeof(PlanPiece) +
         kPlanExtra * sizeof(PlanSplit);
}

extern "C" int kvr_attn_plan(const int32_t *cu_q, const int32_t *kv_len, const int32_t *cu_k, int batch,
                             int64_t n_tokens, int n_q, int n_kv, int causal, int64_t window, void *plan,
                             size_t plan_bytes, kvr_stream_t stream) {
  clear_error();
  KVR_REQUIRE(cu_q, "kvr_attn_plan: null pointer");
  KVR_REQUIRE(!(kv_len && cu_k), "kvr_attn_plan: give kv_len (pages) or cu_k (packed keys), not both");
  PlanArgs a{cu_q, kv_len, cu_k, nullptr, batch, 0, n_q, n_kv, causal ? 1 : 0, 0, nullptr, nullptr, nullptr, 0};
  const int rc = plan_check("kvr_attn_plan", a, n_tokens, window, plan, plan_bytes);
  if (rc) return rc;
  const cudaError_t e = launch_dependent(attn_plan_kernel, 1, kPlanThreads, 0, as_cuda(stream), a);
  if (e != cudaSuccess) return set_error(KVR_ECUDA, "kvr_attn_plan: %s", cudaGetErrorString(e));
  return check_launch("kvr_attn_plan");
}

extern "C" int kvr_paged_map(const int32_t *ctx_len, const int32_t *new_len, int batch, int64_t n_tokens, int page,
                             int32_t *block_table, int64_t table_stride, int table_width, const int32_t *free_pages,
                             int64_t n_free_cap, const int32_t *n_free, int32_t *cu_q, int32_t *kv_len,
                             int32_t *positions, int64_t *slots, int32_t *n_free_out, int32_t *info, int n_q, int n_kv,
                             int64_t window, void *plan, size_t plan_bytes, kvr_stream_t stream) {
  clear_error();
  KVR_REQUIRE(ctx_len && new_len && block_table && n_free && cu_q && kv_len && n_free_out && info,
              "kvr_paged_map: null pointer");
  KVR_REQUIRE(n_tokens == 0 || (positions && slots), "kvr_paged_map: null pointer");
  KVR_REQUIRE(n_free_cap >= 0 && n_free_cap <= INT_MAX / 2 && (n_free_cap == 0 || free_pages),
              "kvr_paged_map: bad free list");
  KVR_REQUIRE(batch >= 1 && batch <= kPlanMaxBatch, "kvr_paged_map: batch must be in [1, %d]", kPlanMaxBatch);
  KVR_REQUIRE(n_tokens >= 0 && n_tokens <= kPlanMaxTokens, "kvr_paged_map: bad token count");
  KVR_REQUIRE(page >= 1 && page <= (1 << 20), "kvr_paged_map: bad page size");
  KVR_REQUIRE(table_width >= 1 && table_stride >= table_width, "kvr_paged_map: bad block table shape");
  KVR_REQUIRE(n_free != n_free_out, "kvr_paged_map: n_free_out must not be n_free");
  MapArgs m{};
  if (plan) {
    m.plan = PlanArgs{cu_q, kv_len, nullptr, ctx_len, batch, 0, n_q, n_kv, 1, 0, nullptr, nullptr, nullptr, 0};
    const int rc = plan_check("kvr_paged_map", m.plan, n_tokens, window, plan, plan_bytes);
    if (rc) return rc;
    m.with_plan = 1;
  }
  m.ctx_len = ctx_len; m.new_len = new_len;
  m.batch = batch; m.n_tokens = (int)n_tokens; m.page = page;
  m.table = block_table; m.table_stride = table_stride; m.table_width = table_width;
  m.free_pages = free_pages; m.n_free = n_free; m.n_free_cap = (int)n_free_cap;
  m.cu = cu_q; m.kv_len = kv_len; m.positions = positions; m.slots = slots;
  m.n_free_out = n_free_out; m.info = info;
  // CTA 0 and one CTA per 1024 tokens, at most one per SM
  int64_t ctas = (n_tokens + kPlanThreads - 1) / kPlanThreads;
  ctas = ctas < 1 ? 1 : (ctas > kPlanCtas - 1 ? kPlanCtas - 1 : ctas);
  const cudaError_t e = launch_dependent(paged_map_kernel, (unsigned)ctas + 1, kPlanThreads, 0, as_cuda(stream), m);
  if (e != cudaSuccess) return set_error(KVR_ECUDA, "kvr_paged_map: %s", cudaGetErrorString(e));
  return check_launch("kvr_paged_map");
}
