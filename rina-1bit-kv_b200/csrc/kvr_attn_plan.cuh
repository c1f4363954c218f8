// The work list of an attention call over requests of different lengths
// (kvr_paged_attn, kvr_prompt_attn), built on the device from the lengths.
//
// The query rows of a request and KV head are its (token, head of the group)
// pairs, row = token * g + j, g = n_q / n_kv.  An item is the rows of up to
// 2 * tpt consecutive tokens, tpt = floor(128 / g): two 128-row tiles that
// share every K/V tile of 128 keys they read.  A piece is a range of an
// item's K/V tiles; the list holds the pieces of ONE head, longest first, and
// serves every KV head: entry p stands for pieces p * n_kv + h.  CTA c of G
// takes pieces c, 2G-1-c, 2G+c, 4G-1-c, ...: with the list sorted the long and
// the short ones even out, and no counter has to be shared or reset.
//
// Items are cut into pieces only where whole items would leave SMs idle: the
// length of the longest piece is the one of 32 candidates for which the
// estimated time is least (plan_estimate).  Where there are fewer items than
// SMs, a second way to cut is weighed against these: all items of all heads in
// a row, and every CTA takes the same number of K/V tiles of that row (an
// `even` plan; its list holds the pieces of all heads, round by round).  A
// chunk of 512 at 32256 (64 items of about 254 tiles) has 110 tiles for each of
// 148 CTAs then; equal pieces give 127 to 128 of them.  The pieces of a cut item
// leave unnormalised partial rows in the workspace, which a second kernel joins
// in the order of the pieces.
#pragma once

#include "kvr_common.cuh"

namespace kvr {

constexpr int kPlanMagic = 0x4b565031;
constexpr int kPlanThreads = 1024;
constexpr int kPlanMaxBatch = 4096;
constexpr int kPlanMaxTokens = 1 << 24;  // query tokens of a call
constexpr int kPlanMaxLen = 1 << 29;     // keys of a request: leaves room for sums in 32 bits
constexpr int kD = 128;          // head_dim
constexpr int kPlanRows = 128;   // rows of a query tile
constexpr int kPlanKeys = 128;   // keys of a K/V tile
constexpr int kPlanCtas = 148;   // SMs the work is spread over

struct PlanHeader {  // 64 words
  int magic, n_tokens, batch, n_q, n_kv, causal, window;
  int n_pieces;      // per head
  int n_splits;      // items cut into pieces, per head
  int part_rows;     // rows of partial results, per head
  int dropped;       // 1: items did not fit the list (offsets that overlap): no call runs the plan
  int even;          // 1: pieces and splits name their head
  int pad[52];
};

struct PlanPiece {   // 8 words
  int q_start;       // first token of the item, in the packed batch
  int n_tok;         // its tokens (in an even plan: head << 16 | tokens; 0: no piece)
  int first_end;     // keys its first token may see: kv_len - q_len (or ctx) + offset + 1 (causal), can be <= 0
  int kv_len;        // keys of the request
  int k_start;       // first key of the request in packed K/V (prompt), or the request's index (pages)
  int kt0, kt1;      // K/V tiles [kt0, kt1) of the piece
  int part;          // row base of its partial results, -1: the piece is the whole item
};
static_assert(sizeof(PlanPiece) == 32, "piece record");

struct PlanSplit {   // an item cut into pieces
  int q_start, n_tok;  // as in its pieces
  int part;          // row base of its first piece; the others follow, n_tok * g rows each (even: see plan_even_row)
  int n_pieces;
};

constexpr int kPlanExtra = 512;                   // pieces per head beyond one per item
constexpr int kPartRows = 2 * kPlanCtas * 2 * kPlanRows;  // partial rows the workspace holds

__host__ __device__ inline int plan_tpt(int n_q, int n_kv) { return kPlanRows / (n_q / n_kv); }
__host__ __device__ inline int64_t plan_max_items(int64_t n_tokens, int batch, int n_q, int n_kv) {
  return n_tokens / (2 * plan_tpt(n_q, n_kv)) + batch + 2;
}

// Rows of partial results in an even plan: CTA c has room for two pieces, its
// first and its last, at 2c and 2c + 1; an item's pieces after its first are
// the first ones of the CTAs that follow.
__host__ __device__ inline int plan_even_row(int part, int k) {
  const int slot = 2 * kPlanRows;
  return k == 0 ? part : (part / (2 * slot) + k) * 2 * slot;
}

struct PlanArgs {
  const int *cu_q;    // (batch + 1)
  const int *kv_len;  // (batch) or NULL
  const int *cu_k;    // (batch + 1) or NULL; both NULL: the keys are the queries' tokens
  const int *ctx;     // (batch) keys before each request's queries, or NULL: the queries are its last tokens
  int batch, n_tokens, n_q, n_kv, causal, window;
  PlanHeader *hdr;
  PlanPiece *pieces;
  PlanSplit *splits;
  int max_items;
};

__host__ __device__ inline const PlanSplit *plan_splits(const PlanHeader *h, int64_t n_tokens, int batch, int n_q,
                                                        int n_kv) {
  const PlanPiece *p = reinterpret_cast<const PlanPiece *>(h + 1);
  return reinterpret_cast<const PlanSplit *>(p + plan_max_items(n_tokens, batch, n_q, n_kv) + kPlanExtra);
}

// Checks of the arguments every plan-building entry point shares; fills the
// pointers into the plan buffer.  Returns a status.
int plan_check(const char *fn, PlanArgs &a, int64_t n_tokens, int64_t window, void *plan, size_t plan_bytes);

}  // namespace kvr
