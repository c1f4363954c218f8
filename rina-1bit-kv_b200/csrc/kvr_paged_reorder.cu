// Reordering of a paged cache's rows: after a beam search step, row i of a
// group becomes what row parents[i] of the group was.
//
// Pages are shared, not copied.  `shared[p]` counts the rows that hold page p
// beyond the first, so a page that only one row holds, or none, has 0, and pages
// that come off or go to the free list need no entry of their own.  A row's last page,
// where it is not full, is written by the row's next token: the first row of the
// call that it falls to keeps it (none, where a row outside of the call holds it), every other one
// gets a fresh page with a copy of its tokens.
//
// A page holds tokens [j P, (j + 1) P) of a sequence, so it stands in column j
// of every row that holds it, and columns do not meet.  paged_reorder_kernel: one
// cluster of 8 CTAs; a warp takes 32 columns of a group, a column per lane:
//   1  the column's pages: holders in the group before and after.  Where the group
//      has all of a page's holders, its new count, or that it is free, is settled
//      at once.  Counts of pages with holders outside go up and down by atomics, with a
//      mark, so that another group does not take what is left for all there was;
//   -  only if there were such pages: the marks go, and a page without a holder is
//      claimed by the lowest place (row, column) that gave it up, by a minimum;
//   2  (after the cluster has met) free pages counted per row, their prefix sums, the
//      pages to the end of the free list in order of rows and columns, new entries;
//   3  (after it has met again; CTA 0, a thread per row) last pages: who copies, fresh
//      pages off the end of the list, lengths.
// No result depends on the order of atomics.  copy_pages_kernel then copies the
// tokens of the listed pages in all layers, K and V, 16 bytes a lane.
//
// What binds: tables and counts are small and lie in L2, so the first kernel is a
// chain of dependent loads and two meetings; HBM binds the copies.  Both kernels in a graph: a
// prompt of 1000 tokens forked 4 ways in 32 layers 17 us, 8 groups of 8 rows of 1300 to 2000 pages, little
// to copy, 25; 16 groups of 4 in 32 layers, 67 MB read and as many written, 36 us (the
// copies alone at a plain copy's rate: 20).
#include "kvr_attn_plan.cuh"

namespace kvr {

constexpr int kPrCluster = 8, kPrThreads = 1024, kPrWarps = kPrThreads / 32;
constexpr int kPrMaxBeams = 32, kPrMaxRows = 4096;
constexpr int kPrCopyWords = 256;    // of 16 bytes, that a warp copies at a time
constexpr int kPrMark = 1 << 18;     // on counts of pages with holders outside of a group: above all counts
constexpr int kPrMaxTable = 1 << 16; // rows of a table
constexpr int kPrSmem = 216 * 1024;  // places of the rows, and entries of as many units as fit

struct ReorderArgs {
  int *table;
  int64_t table_stride;
  int table_rows, width;
  int *ctx;
  int page;
  int *shared;
  int n_pages;
  int *free_pages;
  int n_free_cap;
  int *n_free;
  const int *rows, *parents;
  int groups, beams;
  int slots;    // units of a warp whose entries stay in shared memory
  int *info;
  int *counts;  // (groups * beams, blocks of 32 columns) scratch: pages given back
  unsigned *given;  // (units, 32) scratch: places of the group whose page a lane gives back, a bit each
  int4 *copies; // (groups * beams) scratch: from page, to page, tokens
  int *n_copies;
};

// What is known of a place (a row of a group) before the call.
struct PrPlace {
  int row, parent;  // table row; place of its parent in the group; -1: none
  int len, last;    // its tokens; the page that its parent's last tokens lie in, -1: none, or a full one
};

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int pr_peer(const int *p, unsigned rank) {
  uint32_t a;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// Sum of v over the CTA's lower threads; `total` over all.
__device__ __forceinline__ int pr_exclusive(int v, int *warp_sums, int &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  total = warp_sums[31];
  return x - v + (warp ? warp_sums[warp - 1] : 0);
}
static_assert(kPrWarps == 32, "one sum per lane");

__global__ void __cluster_dims__(kPrCluster, 1, 1) __launch_bounds__(kPrThreads, 1) paged_reorder_kernel(ReorderArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int warp_sums[32], longest, disputed;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.beams, n = a.groups * K;
  PrPlace *place = reinterpret_cast<PrPlace *>(smem);  // (n)
  int *ahead = reinterpret_cast<int *>(place + n);     // (n) pages given back by the places before; at last, who copies
  int *entries = ahead + n;                            // (warps, slots, K, 32)
  if (tid == 0) longest = disputed = 0;
  griddep_wait();
  griddep_launch();
  __syncthreads();
  int most = 0;
  for (int i = tid; i < n; i += kPrThreads) {
    const int r = a.rows[i], p = a.parents[i];
    PrPlace x;
    x.row = r >= 0 && r < a.table_rows ? r : -1;
    x.parent = x.row >= 0 && p >= 0 && p < K ? p : -1;
    x.len = x.row < 0 ? 0 : (int)min((int64_t)max(__ldcg(a.ctx + x.row), 0), (int64_t)a.width * a.page);
    x.last = -1;
    place[i] = x;
    most = max(most, (x.len + a.page - 1) / a.page);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0 && most > 0) atomicMax(&longest, most);
  __syncthreads();
  const int blocks = (longest + 31) / 32, units = a.groups * blocks, all_warps = kPrCluster * kPrWarps;
  // unit u of this warp: group, 32 columns.  CTA first, so that few units spread over the cluster's SMs
  const int me = warp * kPrCluster + (int)blockIdx.x;
  const bool kept = units <= all_warps * a.slots;  // all units' entries stay in shared memory
  struct Place {
    int row, parent, held;
  };
  auto place_of = [&](int u) {  // lane i: place i of the unit's group, and its pages
    Place x{-1, -1, 0};
    if (lane < K) {
      const PrPlace p = place[u / blocks * K + lane];
      x = Place{p.row, p.parent, (p.len + a.page - 1) / a.page};
    }
    return x;
  };
  auto load = [&](int u, int nth, bool again) {
    int *old = entries + (warp * a.slots + (kept ? nth : 0)) * K * 32 + lane;
    if (kept && again) return old;
    const int j = (u - u / blocks * blocks) * 32 + lane;
    const Place x = place_of(u);
#pragma unroll 8
    for (int i = 0; i < K; ++i) {  // (a lane reads back only what it wrote)
      const int r = __shfl_sync(0xffffffffu, x.row, i), h = __shfl_sync(0xffffffffu, x.held, i);
      int e = -1;
      if (j < h) e = a.table[r * a.table_stride + j];
      old[i * 32] = e >= 0 && e < a.n_pages ? e : -1;
    }
    return old;
  };
  // places of entries; the claims lie below every count
  auto claim = [&](int u, int i) {
    const int g = u / blocks;
    return INT_MIN + (g * K + i) * (blocks * 32) + (u - g * blocks) * 32 + lane;
  };
  auto count = [&](int u, unsigned given) {
    const int g = u / blocks;
    for (int i = 0; i < K; ++i) {
      const unsigned who = __ballot_sync(0xffffffffu, (given >> i) & 1);
      if (lane == 0) a.counts[(int64_t)(g * K + i) * blocks + u - g * blocks] = __popc(who);
    }
  };
  // Of the column's page at place i: whether the group's holders change and i is the first of them; how many they are.
  // All lanes together (the parents come from the lanes).
  auto changes = [&](const int *old, int parent, int i, int &before, int &after) {
    const int page = old[i * 32];
    bool first = page >= 0;
    before = after = 0;
#pragma unroll 4
    for (int o = 0; o < K; ++o) {
      const bool same = old[o * 32] == page;
      first &= !(same && o < i);
      before += same;
      const int p = __shfl_sync(0xffffffffu, parent, o);
      after += p >= 0 && old[p * 32] == page;
    }
    return first && before != after;
  };
  for (int u = me, nth = 0; u < units; u += all_warps, ++nth) {
    const int *old = load(u, nth, false);
    const int parent = place_of(u).parent;
    bool differs = false;
    for (int i = 0; i < K; ++i) {
      const int p = __shfl_sync(0xffffffffu, parent, i);
      differs |= old[i * 32] != (p < 0 ? -1 : old[p * 32]);
    }
    unsigned given = 0;
    if (__any_sync(0xffffffffu, differs)) {
      for (int i0 = 0; i0 < K; i0 += 4) {  // four counts' loads at a time
        int before[4], after[4], c[4];
        bool is[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          is[q] = i0 + q < K && changes(old, parent, i0 + q, before[q], after[q]);
          c[q] = is[q] ? __ldcg(a.shared + old[(i0 + q) * 32]) : 0;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (!is[q]) continue;
          int *to = a.shared + old[(i0 + q) * 32];
          if (c[q] < before[q]) {  // (no holder but this group's)
            *to = max(after[q] - 1, 0);
            if (after[q] == 0) given |= 1u << (i0 + q);
          } else {
            atomicAdd(to, after[q] - before[q] + kPrMark);
            disputed = 1;
          }
        }
      }
      __syncwarp();
    }
    a.given[u * 32 + lane] = given;
    count(u, given);
  }
  if (blockIdx.x == 0)  // before any entry is written: the pages that rows will have to copy
    for (int i = tid; i < n; i += kPrThreads) {
      const int p = place[i].parent;
      if (p < 0) continue;
      const int from = i / K * K + p, len = place[from].len;
      if (len % a.page == 0) continue;
      const int page = a.table[place[from].row * a.table_stride + (len - 1) / a.page];
      if (page >= 0 && page < a.n_pages) place[i].last = page;
    }
  cluster_sync();
  int any = 0;
  for (int c = 0; c < kPrCluster; ++c) any |= pr_peer(&disputed, c);
  if (any) {
    // what the first pass did with atomics, again: pass 0 takes the marks off, 1 claims, 2 sees whose claim it was
    for (int pass = 0; pass < 3; ++pass) {
      for (int u = me, nth = 0; u < units; u += all_warps, ++nth) {
        const int *old = load(u, nth, true);
        const int parent = place_of(u).parent;
        unsigned given = a.given[u * 32 + lane];
        for (int i = 0; i < K; ++i) {
          int before, after;
          const bool is = changes(old, parent, i, before, after);
          int *c = a.shared + max(old[i * 32], 0);
          if (is && pass == 0 && __ldcg(c) >= kPrMark / 2) atomicSub(c, kPrMark);
          if (is && pass == 1 && after == 0 && __ldcg(c) < 0) atomicMin(c, claim(u, i));
          if (is && pass == 2 && after == 0 && __ldcg(c) == claim(u, i)) {
            given |= 1u << i;
            *c = 0;
          }
        }
        a.given[u * 32 + lane] = given;
        if (pass == 2) count(u, given);
      }
      cluster_sync();
    }
  }
  // pages given back by each row, and by those before it
  for (int i = warp; i < n; i += kPrWarps) {
    int sum = 0;
    for (int b = lane; b < blocks; b += 32) sum += __ldcg(a.counts + (int64_t)i * blocks + b);
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == 0) ahead[i] = sum;
  }
  __syncthreads();
  int gone;
  {
    const int each = (n + kPrThreads - 1) / kPrThreads;
    int sum = 0;
    for (int i = tid * each; i < min((tid + 1) * each, n); ++i) sum += ahead[i];
    int at = pr_exclusive(sum, warp_sums, gone);
    for (int i = tid * each; i < min((tid + 1) * each, n); ++i) {
      const int c = ahead[i];
      ahead[i] = at;
      at += c;
    }
  }
  const int n_free = min(max(__ldcg(a.n_free), 0), a.n_free_cap);
  __syncthreads();
  for (int u = me, nth = 0; u < units; u += all_warps, ++nth) {
    const int *old = load(u, nth, true);
    const int g = u / blocks, b = u - g * blocks, j = b * 32 + lane;
    const Place x = place_of(u);
    const unsigned given = a.given[u * 32 + lane], anyone = __reduce_or_sync(0xffffffffu, given);
    for (int i = 0; i < K; ++i) {
      if ((anyone >> i) & 1) {
        const int64_t at_i = g * K + i;
        int before = 0;  // the row's in columns before this unit's
        for (int c = lane; c < b; c += 32) before += __ldcg(a.counts + at_i * blocks + c);
        before = __reduce_add_sync(0xffffffffu, before);
        const unsigned who = __ballot_sync(0xffffffffu, (given >> i) & 1);
        const int64_t at = (int64_t)n_free + ahead[at_i] + before + __popc(who & ((1u << lane) - 1));
        if (((given >> i) & 1) && at < a.n_free_cap) a.free_pages[at] = old[i * 32];
      }
      const int r = __shfl_sync(0xffffffffu, x.row, i), p = __shfl_sync(0xffffffffu, x.parent, i);
      const int had_n = __shfl_sync(0xffffffffu, x.held, i), gets_n = __shfl_sync(0xffffffffu, x.held, max(p, 0));
      const int gets = p < 0 ? -1 : old[p * 32];
      if (r >= 0 && old[i * 32] != gets && j < max(had_n, p < 0 ? 0 : gets_n)) a.table[r * a.table_stride + j] = gets;
    }
  }
  cluster_sync();
  if (blockIdx.x != 0) return;
  // last pages, a thread per row: first who copies, by counts that no place has changed yet.  The first place of the call that
  // a page falls to keeps it, unless a row outside of the call holds it too
  for (int i = tid; i < n; i += kPrThreads) {
    const int last = place[i].last;
    int copy = 0;
    if (last >= 0) {
      const int holders = __ldcg(a.shared + last) + 1;
      int before, same;
      auto look = [&](int from, int to) {
        before = same = 0;
        for (int o = from; o < to; ++o) {
          const int is = place[o].last == last;
          same += is;
          before += is && o < i;
        }
      };
      look(i / K * K, i / K * K + K);
      if (same < holders) look(0, n);  // (never so after a beam search's step: the group has all holders)
      copy = before > 0 || holders > same;
    }
    ahead[i] = copy;
  }
  __syncthreads();
  const int left = (int)min((int64_t)n_free + gone, (int64_t)a.n_free_cap);
  int done = 0, missing = 0;
  for (int i0 = 0; i0 < n; i0 += kPrThreads) {
    const int i = i0 + tid;
    const PrPlace x = i < n ? place[i] : PrPlace{-1, -1, 0, -1};
    const int now = x.parent >= 0 ? place[i / K * K + x.parent].len : 0, copy = i < n ? ahead[i] : 0;
    int sum;
    const int k = done + pr_exclusive(copy, warp_sums, sum);
    done += sum;
    if (copy) {
      const int to = k < left ? __ldcg(a.free_pages + left - 1 - k) : -1, col = (now - 1) / a.page;
      atomicSub(a.shared + x.last, 1);
      a.table[x.row * a.table_stride + col] = to;
      if (to >= 0) a.copies[k] = make_int4(x.last, to, now % a.page, 0);
      else ++missing;
    }
    if (x.row >= 0) a.ctx[x.row] = copy && k >= left ? now / a.page * a.page : now;
  }
  int all_missing;
  pr_exclusive(missing, warp_sums, all_missing);
  if (tid == 0) {
    a.info[0] = all_missing;
    a.info[1] = *a.n_copies = done - all_missing;
    a.info[2] = gone;
    a.info[3] = 0;
    *a.n_free = max(left - done, 0);
  }
}

struct CopyArgs {
  uint16_t *k, *v;
  int layers, page, n_kv;
  int64_t layer_stride, page_stride, tok_stride;  // elements
  const int4 *copies;
  const int *n_copies;
};

// A warp takes 256 words of 16 bytes of a page at a time, eight a lane on their way.  (Eight tokens at a time, with a
// division a word: 450 instructions in place of 130, 1 to 2 us more a call.)
__global__ void __launch_bounds__(256) copy_pages_kernel(CopyArgs a) {
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31, row = a.n_kv * 16;  // words of a token: 128 channels of 2 bytes a head
  const unsigned chunks = ((unsigned)a.page * row + kPrCopyWords - 1) / kPrCopyWords, inv = 0xffffffffu / row + 1;
  // (a page is larger than 512 bytes, so that all of a GPU's memory is fewer chunks than 2^31)
  const unsigned n = (unsigned)*a.n_copies * a.layers * 2 * chunks;
  for (unsigned w = blockIdx.x * 8 + (threadIdx.x >> 5); w < n; w += gridDim.x * 8) {
    // chunks innermost: the copies of a page follow one another
    unsigned rest = w / chunks;
    const int first = (w - rest * chunks) * kPrCopyWords + lane;
    const unsigned pair = rest / a.layers, layer = rest - pair * a.layers;
    const int4 c = a.copies[pair >> 1];
    const int words = c.z * row;
    uint16_t *pool = (pair & 1 ? a.v : a.k) + layer * a.layer_stride;
    const uint16_t *src = pool + c.x * a.page_stride;
    uint16_t *dst = pool + c.y * a.page_stride;
    uint4 x[kPrCopyWords / 32];
    auto at = [&](int i) {
      int t = __umulhi(i, inv);  // i / row, or one more
      t -= t * row > i;
      return t * a.tok_stride + (i - t * row) * 8;
    };
#pragma unroll
    for (int u = 0; u < kPrCopyWords / 32; ++u)
      if (first + u * 32 < words) x[u] = __ldcs(reinterpret_cast<const uint4 *>(src + at(first + u * 32)));
#pragma unroll
    for (int u = 0; u < kPrCopyWords / 32; ++u)
      if (first + u * 32 < words) *reinterpret_cast<uint4 *>(dst + at(first + u * 32)) = x[u];
  }
}

}  // namespace kvr

using namespace kvr;

extern "C" size_t kvr_paged_reorder_workspace_bytes(int groups, int beams, int table_width) {
  if (groups < 1 || beams < 1 || beams > kPrMaxBeams || table_width < 1) return 0;
  const size_t n = (size_t)groups * beams, blocks = (table_width + 31) / 32;
  return n * sizeof(int4) + 16 + (n * blocks + (size_t)groups * blocks * 32) * sizeof(int);
}

extern "C" int kvr_paged_reorder(int32_t *block_table, int64_t table_stride, int table_rows, int table_width,
                                 int32_t *ctx_len, int page, int32_t *shared, int64_t n_pages, int32_t *free_pages,
                                 int64_t n_free_cap, int32_t *n_free, const int32_t *rows, const int32_t *parents,
                                 int groups, int beams, void *k_pages, void *v_pages, int dtype, int layers, int n_kv,
                                 int d, int64_t layer_stride, int64_t page_stride, int64_t tok_stride, int32_t *info,
                                 void *workspace, size_t workspace_bytes, kvr_stream_t stream) {
  clear_error();
  KVR_REQUIRE(groups >= 0 && beams >= 1, "kvr_paged_reorder: bad groups");
  if (beams > kPrMaxBeams || (int64_t)groups * beams > kPrMaxRows)
    return set_error(KVR_ENOTSUP, "kvr_paged_reorder: at most %d beams and %d rows", kPrMaxBeams, kPrMaxRows);
  KVR_REQUIRE(info && n_free, "kvr_paged_reorder: null pointer");
  KVR_REQUIRE(block_table && ctx_len && shared && (rows || !groups) && (parents || !groups) && workspace,
              "kvr_paged_reorder: null pointer");
  KVR_REQUIRE(page >= 1 && page <= (1 << 20), "kvr_paged_reorder: bad page size");
  if (table_rows > kPrMaxTable) return set_error(KVR_ENOTSUP, "kvr_paged_reorder: at most %d table rows", kPrMaxTable);
  KVR_REQUIRE(table_rows >= 1 && table_width >= 1 && (table_stride >= table_width || table_rows == 1),
              "kvr_paged_reorder: bad block table shape");
  KVR_REQUIRE((int64_t)groups * beams * align_up(table_width, 32) < (1 << 30), "kvr_paged_reorder: the rows are too long");
  KVR_REQUIRE(n_pages >= 1 && n_pages <= INT_MAX / 2 && n_free_cap >= 0 && n_free_cap <= INT_MAX / 2 &&
                  (n_free_cap == 0 || free_pages),
              "kvr_paged_reorder: bad page pool or free list");
  if (d != kD) return set_error(KVR_ENOTSUP, "kvr_paged_reorder: head_dim must be 128");
  if (dtype != KVR_F16 && dtype != KVR_BF16)
    return set_error(KVR_ENOTSUP, "kvr_paged_reorder: the cache holds fp16 or bf16");
  KVR_REQUIRE(k_pages && v_pages, "kvr_paged_reorder: null pointer");
  KVR_REQUIRE(layers >= 1 && n_kv >= 1 && tok_stride >= (int64_t)n_kv * d && page_stride >= 0 && layer_stride >= 0,
              "kvr_paged_reorder: a token's heads must be contiguous");
  if ((int64_t)page * n_kv >= 1 << 27) return set_error(KVR_ENOTSUP, "kvr_paged_reorder: pages of 32 GB");
  KVR_REQUIRE((layer_stride | page_stride | tok_stride) % 8 == 0 &&
                  ((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages) |
                    reinterpret_cast<uintptr_t>(workspace)) & 15) == 0,
              "kvr_paged_reorder: pointers and strides must keep rows 16-byte aligned");
  KVR_REQUIRE(groups == 0 || workspace_bytes >= kvr_paged_reorder_workspace_bytes(groups, beams, table_width),
              "kvr_paged_reorder: workspace too small");
  ReorderArgs a{};
  a.table = block_table; a.table_stride = table_stride; a.table_rows = table_rows; a.width = table_width;
  a.ctx = ctx_len; a.page = page;
  a.shared = shared; a.n_pages = (int)n_pages;
  a.free_pages = free_pages; a.n_free_cap = (int)n_free_cap; a.n_free = n_free;
  a.rows = rows; a.parents = parents; a.groups = groups; a.beams = beams;
  a.info = info;
  a.copies = static_cast<int4 *>(workspace);
  a.n_copies = reinterpret_cast<int *>(a.copies + (size_t)groups * beams);
  a.counts = a.n_copies + 4;
  a.given = reinterpret_cast<unsigned *>(a.counts + (size_t)groups * beams * ((table_width + 31) / 32));
  if (groups == 0) {
    const cudaError_t z = cudaMemsetAsync(info, 0, 16, as_cuda(stream));
    return z == cudaSuccess ? KVR_OK : set_error(KVR_ECUDA, "kvr_paged_reorder: %s", cudaGetErrorString(z));
  }
  // entries of as many units as a row of the table can make, where they fit
  const size_t places = (size_t)groups * beams * (sizeof(PrPlace) + sizeof(int)), unit = (size_t)kPrWarps * beams * 32 * sizeof(int);
  const int64_t warps = kPrCluster * kPrWarps, most = ((int64_t)groups * ((table_width + 31) / 32) + warps - 1) / warps;
  a.slots = (int)((kPrSmem - places) / unit);
  if (a.slots > most) a.slots = (int)most;
  static_assert((size_t)kPrMaxRows * (sizeof(PrPlace) + sizeof(int)) + (size_t)kPrWarps * 32 * kPrMaxBeams * sizeof(int) <= kPrSmem,
                "a unit of a warp at least");
  const size_t smem = places + a.slots * unit;
  if (smem > 40 * 1024) {
    const cudaError_t s = cudaFuncSetAttribute(paged_reorder_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPrSmem);
    if (s != cudaSuccess) return set_error(KVR_ECUDA, "kvr_paged_reorder: %s", cudaGetErrorString(s));
  }
  cudaError_t e = launch_dependent(paged_reorder_kernel, kPrCluster, kPrThreads, smem, as_cuda(stream), a);
  if (e != cudaSuccess) return set_error(KVR_ECUDA, "kvr_paged_reorder: %s", cudaGetErrorString(e));
  CopyArgs c{static_cast<uint16_t *>(k_pages), static_cast<uint16_t *>(v_pages), layers, page, n_kv,
             layer_stride, page_stride, tok_stride, a.copies, a.n_copies};
  // at most as many warps as there can be chunks
  const int64_t chunks = (int64_t)groups * beams * layers * 2 * (((int64_t)page * n_kv * 16 + kPrCopyWords - 1) / kPrCopyWords);
  const int64_t ctas = (chunks + 7) / 8;
  e = launch_dependent(copy_pages_kernel, (unsigned)(ctas > 148 * 8 ? 148 * 8 : ctas), 256, 0, as_cuda(stream), c);
  if (e != cudaSuccess) return set_error(KVR_ECUDA, "kvr_paged_reorder: %s", cudaGetErrorString(e));
  return check_launch("kvr_paged_reorder");
}
