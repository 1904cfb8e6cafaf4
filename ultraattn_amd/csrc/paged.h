// What the paged cache's kernels share.
//
// A cache's rows lie in pages: pools [n_pages, page, heads, head_dim]; row r of sequence b is slot r % page of page table[b, r / page].  A page outside the
// pool is not there: nothing is written to it, and what it would hold is not seen.
//
// A call's new tokens: n_new[b] of n_tokens are real, token t is at row base + t, base = lens[b] - n_new[b].  They are a chain or a tree: parents[b, t] is the
// token before token t, anything but 0 .. t - 1 says that it follows row base - 1.  Its depth counts the tokens before it in its branch, and
// base + depth is its position.
#pragma once
#include "ua_common.h"

namespace ua {

constexpr int kPagedMost = 1 << 29;                   // lengths are clamped to it: no sum of two rows leaves 32 bits
constexpr int kTreeMost = UA_PAGED_MAX_TREE;
constexpr int kTreeThreads = 256;                     // of the workgroups that walk trees
static_assert(kTreeMost == kTreeThreads, "a token a thread");

struct PagedSteps {                                   // the new tokens of all sequences
  const int32_t *lens, *n_new, *parents;
  int64_t parents_stride;                             // 0: one tree for all
  int n_tokens;
};
struct PagedTable {
  const int32_t* table;
  int64_t stride;
  int n_pages, page, room;                            // room: rows that the table has entries for, at most kPagedMost
  Div by_page;
};
struct StepOf { int len, n, base; };                  // one sequence's
__device__ __forceinline__ StepOf step_of(const PagedSteps& p, int b) {
  const int n = p.n_new ? min(max(p.n_new[b], 0), p.n_tokens) : p.n_tokens, len = min(max(p.lens[b], 0), kPagedMost);
  return {len, n, len - n};
}
__device__ __forceinline__ int parent_of(const PagedSteps& p, int b, int t) {
  const int parent = t < p.n_tokens ? p.parents[b * p.parents_stride + t] : -1;
  return parent < t ? max(parent, -1) : -1;
}

// Depths of a sequence's tokens, by a workgroup of kTreeThreads: every token's distance to a token before it, and that one, doubled until all have
// reached the first of their branch, as many times as the deepest branch's logarithm.  Up to 64 tokens every wave does this for itself, a lane a token, and
// writes what the others write; more meet at two barriers a round.  `parent`: of the token that tree_token names.
__device__ __forceinline__ int tree_token(const PagedSteps& p) { return p.n_tokens <= 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x; }
__device__ __forceinline__ void tree_depths(const PagedSteps& p, int parent, int (&depth)[kTreeMost], int (&before)[kTreeMost]) {
  const int t = tree_token(p);
  int d = parent >= 0;
  if (p.n_tokens <= 64) {
    while (__builtin_amdgcn_ballot_w64(parent >= 0) != 0) {
      const int from = max(parent, 0), far = __shfl(d, from), next = __shfl(parent, from);
      if (parent >= 0) {
        d += far;
        parent = next;
      }
    }
    depth[t] = d;
    return;
  }
  while (true) {
    depth[t] = d;
    before[t] = parent;
    if (!__syncthreads_or(parent >= 0)) return;
    if (parent >= 0) {
      d += depth[parent];
      parent = before[parent];
    }
    __syncthreads();
  }
}

inline int paged_room(int page, int max_pages) {
  const int64_t room = (int64_t)page * max_pages;
  return room < kPagedMost ? (int)room : kPagedMost;
}
// Sizes that every entry point of the paged cache checks alike.
inline int paged_check(int batch, int n_tokens, int n_kv_heads, int n_pages, int page, int max_pages, int64_t table_stride, const int32_t* parents,
                       int64_t parents_stride) {
  if (batch < 0 || n_tokens < 0 || n_kv_heads <= 0 || n_pages < 0 || page <= 0 || max_pages < 0 || table_stride < 0 || parents_stride < 0) return UA_ERR_SHAPE;
  if (page > kPagedMost || n_tokens > kPagedMost / 2) return UA_ERR_SHAPE;
  if (parents && n_tokens > kTreeMost) return UA_ERR_SHAPE;
  return UA_OK;
}

}  // namespace ua
