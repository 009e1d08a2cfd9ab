// Parameters of the kernels around a paged key / value cache (paged.cu, paged_attn.cu).
//
// A pool holds pages of `page_size` rows for every K / V head. Row p of sequence b is row
// p % page_size of page table[b][p / page_size]; a page number outside the pool is never followed.
#pragma once
#include "common.cuh"

namespace dab {

// codes of the error word, next to those of bounded waits
enum PagedError : int {
  ERR_PAGE = 0x601,       // a page number is outside the pool
  ERR_LENGTH = 0x602,     // a sequence is longer than its row of the page table
  ERR_POSITION = 0x603,   // a position is past the rotation tables
  ERR_STARTS = 0x604,     // a sequence begins or ends outside the tokens
};

struct PagedAppend {
  const void* k; const void* v; int64_t k_t, k_h, v_t, v_h;      // new rows [T, H, D], strides in elements
  const void* q; void* q_out; int64_t q_t, q_h, qo_t, qo_h;      // queries [T, Hq, D] and rotated queries
  void* kp; void* vp; int64_t p_p, p_h, p_r;                     // pool: strides over page, head, row
  const int32_t* table; int64_t table_stride;                    // [B, max_pages]
  const int32_t* lengths;                                        // [B], the new rows counted
  const int32_t* cu;                                             // [B + 1], null: token b is sequence b's only one
  const void* cos; const void* sin; int64_t cs_r;                // [table_rows, D], null: rows go in as they are
  int* err;
  int T, B, H, Hq, max_pages, num_pages, ps_shift, table_rows;
};

// How the CTAs of a decode step are shared between the prefixes and the sequences' own rows: CTAs and first CTA of
// each, and what each costs.
struct Ctas {
  int n[2], from[2];
  int64_t cost[2];
};

struct PagedAttn {
  // maps of the queries (a tile of tokens, and one token) and of the K / V rows, made at the launch
  CUtensorMap tm_q, tm_q1, tm_k, tm_v;
  const void* q; void* out; int64_t q_t, q_h, o_t, o_h;          // [T, Hq, D]
  const void* k; const void* v; int64_t k_p, k_h, k_r, v_p, v_h, v_r;  // pool, or (table null) rows [T, H, D]
  const int32_t* table; int64_t table_stride;
  const int32_t* lengths;                                        // [B], null: as many rows as queries
  const int32_t* cu;                                             // [B + 1], null: query b is sequence b's only one
  const int32_t* prefix_cu; const int32_t* prefix_len;           // groups of sequences and what each shares
  int* err;
  float scale_log2;                                              // sm_scale * log2(e)
  int T, B, H, G, max_pages, num_pages, ps_shift, groups, causal;
  int decode;     // one token per sequence, the work cut into even ranges of key tiles
  int may_split;  // prompts: the units may be too few for the SMs
  int num_ctas;
  int w_start, w_pair, w_thin;  // decode: costs of beginning a unit, and of its key tiles
  // workspace: piece counter and finished CTAs, records of sequences and groups, partial results
  unsigned* counter;
  int64_t* rec_cost; int64_t* rec_row; Ctas* rec_ctas; float* part_o; float2* part_s;
};

// Records a wrong argument that only the device sees; the first one stays.
__device__ __forceinline__ void paged_error(int* err, int code) {
  if (err) atomicCAS(err, 0, code);
}

// Rows that sequence b's page table can hold of its length.
__device__ __forceinline__ int paged_length(int len, int max_pages, int ps_shift, int* err) {
  if (len <= 0) return 0;
  if (((len - 1) >> ps_shift) < max_pages) return len;
  paged_error(err, ERR_LENGTH);
  return max_pages << ps_shift;
}

// Tokens [c0, c1) of sequence b, kept inside [0, T]; returns whether its start lies behind its end.
__device__ __forceinline__ bool paged_tokens(const int32_t* cu, int b, int T, int* err, int& c0, int& c1) {
  if (!cu) {
    c0 = b;
    c1 = b + 1;
    return false;
  }
  c0 = cu[b];
  c1 = cu[b + 1];
  const bool falls = c1 < c0;
  if (c0 < 0 || c1 > T || c1 < c0) {
    paged_error(err, ERR_STARTS);
    c0 = min(max(c0, 0), T);
    c1 = min(max(c1, c0), T);
  }
  return falls;
}

// The last b in [0, B) with cu[b] <= t, for t in [cu[0], cu[B]); -1 for other tokens. The whole warp
// calls it: 32 entries are looked at in one step.
__device__ __forceinline__ int paged_sequence(const int32_t* cu, int B, int t) {
  const int lane = lane_id();
  int lo = 0, hi = B;  // cu[lo] <= t < cu[hi]
  if (cu[0] > t || cu[B] <= t) return -1;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5;
    const int i = lo + (lane + 1) * step;
    const unsigned above = __ballot_sync(0xFFFFFFFFu, i >= hi || cu[i] > t);
    const int n = __ffs(above) - 1;  // entries lo + step .. lo + n * step are at most t
    const int at = lo + n * step;
    hi = min(hi, at + step);
    lo = at;
  }
  return lo;
}

}  // namespace dab
