// Reordering of a paged cache's rows: after a beam search step, row i of a
// group becomes what row parents[i] of the group was.
//
// Pages are shared, not copied.  `shared[p]` counts the rows that hold page p
// beyond the first, so a page that only one row holds, or none, has 0, and pages
// that come off or go to the free list need no entry of their own.  A row's last page,
// where it is not full, is written by the row's next token: the parent's first
// child keeps it, every other child gets a fresh page with a copy of its tokens.
//
// A page holds tokens [j P, (j + 1) P) of a sequence, so it stands in column j
// of every row that holds it, and columns do not meet.  paged_reorder_kernel: one
// cluster of 8 CTAs; a warp takes 32 columns of a group, a column per lane:
//   1  counts: + for the page that a row gets, - for the one that it loses;
//   2  a page with a count below 0 has no holder left.  Rows of several groups may
//      have lost it: the lowest place (row, column) claims it, by a minimum;
//   3  claims won per row and 32 columns, their prefix sums;
//   4  claimed pages to the end of the free list, in order of rows and columns,
//      and the rows' new entries;
//   5  (CTA 0, a thread per row) last pages: who copies, fresh pages off the end
//      of the list, lengths.
// No result depends on the order of atomics.  Tables and counts are small and lie
// in L2: the chain of phases bounds it.  copy_pages_kernel then copies the tokens
// of the listed pages in all layers, K and V, 16 bytes a lane; HBM bounds that.
#include "kvr_attn_plan.cuh"

namespace kvr {

constexpr int kPrCluster = 8, kPrThreads = 512, kPrWarps = kPrThreads / 32;
constexpr int kPrMaxBeams = 32, kPrMaxRows = 4096;
constexpr int kPrStepTokens = 8;  // tokens that a warp copies at a time

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
  int *info;
  int *counts;  // (groups * beams, blocks of 32 columns) scratch
  int4 *copies; // (groups * beams) scratch: from page, to page, tokens
  int *n_copies;
};

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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
    int s = lane < kPrWarps ? warp_sums[lane] : 0;
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

__device__ __forceinline__ int pr_row(const ReorderArgs &a, int i) {  // table row of place i, -1: none
  const int r = a.rows[i];
  return r >= 0 && r < a.table_rows ? r : -1;
}
__device__ __forceinline__ int pr_len(const ReorderArgs &a, int i) {  // its tokens before the call
  const int r = pr_row(a, i);
  return r < 0 ? 0 : (int)min((int64_t)max(__ldcg(a.ctx + r), 0), (int64_t)a.width * a.page);
}
__device__ __forceinline__ int pr_parent(const ReorderArgs &a, int i) {  // place of its parent, -1: none
  const int p = a.parents[i];
  return p >= 0 && p < a.beams ? i / a.beams * a.beams + p : -1;
}

__global__ void __cluster_dims__(kPrCluster, 1, 1) __launch_bounds__(kPrThreads) paged_reorder_kernel(ReorderArgs a) {
  extern __shared__ int old_s[];  // (warps, beams, 32): a unit's old entries
  __shared__ int parent_s[kPrWarps][kPrMaxBeams], row_s[kPrWarps][kPrMaxBeams], held_s[kPrWarps][kPrMaxBeams];
  __shared__ int warp_sums[32], longest;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.beams, n = a.groups * K;
  griddep_wait();
  griddep_launch();
  if (tid == 0) longest = 0;
  __syncthreads();
  int most = 0;
  for (int i = tid; i < n; i += kPrThreads) most = max(most, (pr_len(a, i) + a.page - 1) / a.page);
  most = warp_max_int(most);
  if (lane == 0) atomicMax(&longest, most);
  __syncthreads();
  const int blocks = (longest + 31) / 32, units = a.groups * blocks, all_warps = kPrCluster * kPrWarps;
  // unit u of this warp: group, columns.  CTA first, so that few units spread over the cluster's SMs
  const int me = warp * kPrCluster + (int)blockIdx.x;
  int *old = old_s + warp * K * 32;
  auto load = [&](int u) {
    const int g = u / blocks, j = (u - g * blocks) * 32 + lane;
    __syncwarp();
    if (lane < K) {
      const int i = g * K + lane;
      const int r = pr_row(a, i), p = pr_parent(a, i);
      row_s[warp][lane] = r;
      held_s[warp][lane] = (pr_len(a, i) + a.page - 1) / a.page;
      parent_s[warp][lane] = r < 0 || p < 0 ? -1 : p - g * K;
    }
    __syncwarp();
#pragma unroll 8
    for (int i = 0; i < K; ++i) {
      int e = -1;
      if (j < held_s[warp][i]) e = a.table[row_s[warp][i] * a.table_stride + j];
      old[i * 32 + lane] = e >= 0 && e < a.n_pages ? e : -1;
    }
    // (a lane reads back only what it wrote)
  };
  auto fresh = [&](int i) {  // what place i of the unit gets
    const int p = parent_s[warp][i];
    return p < 0 ? -1 : old[p * 32 + lane];
  };
  const bool once = units <= all_warps;  // a warp's only unit stays in shared memory
  for (int u = me; u < units; u += all_warps) {
    load(u);
    for (int i = 0; i < K; ++i) {
      const int had = old[i * 32 + lane], gets = fresh(i);
      if (had == gets) continue;
      if (gets >= 0) atomicAdd(a.shared + gets, 1);
      if (had >= 0) atomicSub(a.shared + had, 1);
    }
  }
  cluster_sync();
  // place of an entry; the claims lie below every count
  auto claim = [&](int u, int i) {
    const int g = u / blocks;
    return INT_MIN + (g * K + i) * (blocks * 32) + (u - g * blocks) * 32 + lane;
  };
  for (int u = me; u < units; u += all_warps) {
    if (!once) load(u);
    for (int i = 0; i < K; ++i) {
      const int had = old[i * 32 + lane];
      if (had >= 0 && had != fresh(i) && __ldcg(a.shared + had) < 0) atomicMin(a.shared + had, claim(u, i));
    }
  }
  cluster_sync();
  for (int u = me; u < units; u += all_warps) {
    if (!once) load(u);
    const int g = u / blocks;
    for (int i = 0; i < K; ++i) {
      const int had = old[i * 32 + lane];
      const bool won = had >= 0 && had != fresh(i) && __ldcg(a.shared + had) == claim(u, i);
      const unsigned who = __ballot_sync(0xffffffffu, won);
      if (lane == 0) a.counts[(int64_t)(g * K + i) * blocks + u - g * blocks] = __popc(who);
    }
  }
  cluster_sync();
  const int n_free = min(max(*a.n_free, 0), a.n_free_cap);
  int gone = 0;
  if (blockIdx.x == 0) {  // prefix sums of the counts, in place
    const int64_t entries = (int64_t)n * blocks, each = (entries + kPrThreads - 1) / kPrThreads;
    int sum = 0;
    for (int64_t k = tid * each; k < min((tid + 1) * each, entries); ++k) sum += __ldcg(a.counts + k);
    int at = pr_exclusive(sum, warp_sums, gone);
    for (int64_t k = tid * each; k < min((tid + 1) * each, entries); ++k) {
      const int c = __ldcg(a.counts + k);
      a.counts[k] = at;
      at += c;
    }
  }
  cluster_sync();
  for (int u = me; u < units; u += all_warps) {
    if (!once) load(u);
    const int g = u / blocks, j = (u - g * blocks) * 32 + lane;
    for (int i = 0; i < K; ++i) {
      const int had = old[i * 32 + lane], gets = fresh(i);
      const bool won = had >= 0 && had != gets && __ldcg(a.shared + had) == claim(u, i);
      const unsigned who = __ballot_sync(0xffffffffu, won);
      if (won) {
        const int64_t at = (int64_t)n_free + __ldcg(a.counts + (int64_t)(g * K + i) * blocks + u - g * blocks) +
                           __popc(who & ((1u << lane) - 1));
        if (at < a.n_free_cap) a.free_pages[at] = had;
        a.shared[had] = 0;
      }
      const int r = row_s[warp][i], p = parent_s[warp][i];
      if (r >= 0 && had != gets && j < max(held_s[warp][i], p < 0 ? 0 : held_s[warp][p]))
        a.table[r * a.table_stride + j] = gets;
    }
  }
  cluster_sync();
  if (blockIdx.x != 0) return;
  // last pages, a thread per row
  const int left = (int)min((int64_t)n_free + gone, (int64_t)a.n_free_cap);
  int done = 0, missing = 0;
  const int step = kPrThreads / K * K;  // whole groups: lengths are read before any of the group is written
  for (int i0 = 0; i0 < n; i0 += step) {
    const int i = i0 + tid;
    const bool in = tid < step && i < n;
    const int parent = in ? pr_parent(a, i) : -1, r = in ? pr_row(a, i) : -1;
    const int now = parent >= 0 && r >= 0 ? pr_len(a, parent) : 0;
    const int col = (now - 1) / a.page;
    int copy = 0, page = -1;
    if (now % a.page) {
      page = __ldcg(a.table + r * a.table_stride + col);
      if (page >= 0 && page < a.n_pages) {
        int before = 0, same = 0;  // children of the parent
        const int g = i / K * K;
        for (int o = g; o < g + K; ++o) {
          const int is = pr_parent(a, o) == parent && pr_row(a, o) >= 0;
          same += is;
          before += is && o < i;
        }
        copy = before > 0 || __ldcg(a.shared + page) + 1 > same;  // (or a row outside of the group holds it)
      }
    }
    int sum;
    const int k = done + pr_exclusive(copy, warp_sums, sum);
    done += sum;
    __syncthreads();  // lengths, counts and entries of these rows are read
    if (copy) {
      const int to = k < left ? a.free_pages[left - 1 - k] : -1;
      atomicSub(a.shared + page, 1);
      a.table[r * a.table_stride + col] = to;
      if (to >= 0) a.copies[k] = make_int4(page, to, now % a.page, 0);
      if (to < 0) {
        ++missing;
        a.ctx[r] = col * a.page;
      }
    }
    if (r >= 0 && !(copy && k >= left)) a.ctx[r] = now;
    __syncthreads();
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

__global__ void __launch_bounds__(256) copy_pages_kernel(CopyArgs a) {
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31, steps = (a.page + kPrStepTokens - 1) / kPrStepTokens;
  const int64_t warps = (int64_t)gridDim.x * 8, n = (int64_t)*a.n_copies * a.layers * 2 * steps;
  const int row = a.n_kv * 16;  // 16-byte words of a token: 128 channels of 2 bytes a head
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < n; w += warps) {
    // steps innermost: the copies of a page follow one another
    const int step = (int)(w % steps);
    int64_t rest = w / steps;
    const int layer = (int)(rest % a.layers);
    rest /= a.layers;
    const bool v = rest & 1;
    const int4 c = a.copies[rest >> 1];
    const int t0 = step * kPrStepTokens, tokens = min(kPrStepTokens, c.z - t0);
    if (tokens <= 0) continue;
    uint16_t *pool = (v ? a.v : a.k) + layer * a.layer_stride + t0 * a.tok_stride;
    const uint16_t *src = pool + c.x * a.page_stride;
    uint16_t *dst = pool + c.y * a.page_stride;
    const int words = tokens * row;
    for (int at = lane; at < words; at += 32 * 8) {
      uint4 x[8];
      int64_t off[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = at + u * 32, t = i / row;
        off[u] = t * a.tok_stride + (i - t * row) * 8;
        if (i < words) x[u] = __ldcs(reinterpret_cast<const uint4 *>(src + off[u]));
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (at + u * 32 < words) *reinterpret_cast<uint4 *>(dst + off[u]) = x[u];
    }
  }
}

}  // namespace kvr

using namespace kvr;

extern "C" size_t kvr_paged_reorder_workspace_bytes(int groups, int beams, int table_width) {
  if (groups < 1 || beams < 1 || beams > kPrMaxBeams || table_width < 1) return 0;
  const size_t n = (size_t)groups * beams;
  return n * sizeof(int4) + 16 + n * ((table_width + 31) / 32) * sizeof(int);
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
  if (groups == 0) {
    const cudaError_t z = cudaMemsetAsync(info, 0, 16, as_cuda(stream));
    return z == cudaSuccess ? KVR_OK : set_error(KVR_ECUDA, "kvr_paged_reorder: %s", cudaGetErrorString(z));
  }
  const size_t smem = (size_t)kPrWarps * beams * 32 * sizeof(int);
  if (smem > 40 * 1024) {
    const cudaError_t s = cudaFuncSetAttribute(paged_reorder_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               kPrWarps * kPrMaxBeams * 32 * (int)sizeof(int));
    if (s != cudaSuccess) return set_error(KVR_ECUDA, "kvr_paged_reorder: %s", cudaGetErrorString(s));
  }
  cudaError_t e = launch_dependent(paged_reorder_kernel, kPrCluster, kPrThreads, smem, as_cuda(stream), a);
  if (e != cudaSuccess) return set_error(KVR_ECUDA, "kvr_paged_reorder: %s", cudaGetErrorString(e));
  CopyArgs c{static_cast<uint16_t *>(k_pages), static_cast<uint16_t *>(v_pages), layers, page, n_kv,
             layer_stride, page_stride, tok_stride, a.copies, a.n_copies};
  // at most as many warps as there can be steps of work
  const int64_t steps = (int64_t)groups * beams * layers * 2 * ((page + kPrStepTokens - 1) / kPrStepTokens);
  const int64_t ctas = (steps + 7) / 8;
  e = launch_dependent(copy_pages_kernel, (unsigned)(ctas > 148 * 8 ? 148 * 8 : ctas), 256, 0, as_cuda(stream), c);
  if (e != cudaSuccess) return set_error(KVR_ECUDA, "kvr_paged_reorder: %s", cudaGetErrorString(e));
  return check_launch("kvr_paged_reorder");
}
