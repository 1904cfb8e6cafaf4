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

// Trees are resolved by waves, a lane a token of 64: within them a token takes up the branch of the token 2^k before it, round by round, as many times as the
// deepest branch's logarithm, without a barrier.  Up to 64 tokens every wave does all of it for itself and writes what the others write; of more, wave w has tokens 64 w ..,
// and a branch goes on where the tokens before have it: one barrier, and a step for every earlier 64.  (Round by round over all tokens, with two barriers each: 26
// tokens 4400 cycles, now 860.)
__device__ __forceinline__ int tree_token(const PagedSteps& p) { return p.n_tokens <= 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x; }
struct TreePart {
  uint32_t bits[2];       // the branch's tokens among the wave's 64, the token itself included
  int exit;               // the last of its tokens before those, or -1
};
// t: the lane's token; parent: as parent_of gives it.
__device__ __forceinline__ TreePart tree_part(int t, int parent) {
  const int lane = t & 63, first = t - lane;
  TreePart x{{lane < 32 ? 1u << lane : 0u, lane < 32 ? 0u : 1u << (lane & 31)}, parent < first ? parent : -1};
  int before = parent - first;                        // in the wave, or below 0
  while (__builtin_amdgcn_ballot_w64(before >= 0) != 0) {
    const int from = max(before, 0);
    const uint32_t lo = __shfl(x.bits[0], from), hi = __shfl(x.bits[1], from);
    const int exit = __shfl(x.exit, from), next = __shfl(before, from);
    if (before >= 0) {
      x.bits[0] |= lo;
      x.bits[1] |= hi;
      x.exit = exit;
      before = next;
    }
  }
  return x;
}
// Depths of a sequence's tokens, by a workgroup of kTreeThreads; `parent`: of the token that tree_token names.
__device__ __forceinline__ void tree_depths(const PagedSteps& p, int parent, int (&depth)[kTreeMost], int (&exit)[kTreeMost]) {
  const int t = tree_token(p);
  const TreePart x = tree_part(t, parent);
  int d = __popc(x.bits[0]) + __popc(x.bits[1]) - 1;
  if (p.n_tokens <= 64) {
    depth[t] = d;
    return;
  }
  depth[t] = d;
  exit[t] = x.exit;
  __syncthreads();
  for (int at = x.exit; at >= 0; at = exit[at]) d += depth[at] + 1;
  __syncthreads();
  depth[t] = d;
  __syncthreads();
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
