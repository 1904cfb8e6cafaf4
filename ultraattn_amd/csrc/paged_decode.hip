// Attention of the new tokens of every sequence, a chain or a tree, against a paged cache that holds them already.
//
// The rows of a key head are the new tokens of each of the query heads that share it, row = token * group + head of the group.  Two kernels:
//   few rows (up to 32 of a key head): as against a contiguous cache, four waves of a workgroup go through blocks of 32 keys of their own, rows are the columns
//     of 16x16x32 products, and the waves' rows are merged at the end.  Bound: HBM, the visible keys and values once.
//   many rows: tiles of 128, 32 a wave as two times 16 columns of the same products, go through blocks of 64 keys together (two LDS stages).  Bound: the products,
//     or HBM where the tiles are few.  (With 32x32x16 products, half as many instructions, 2048 tokens of 8 x 4 heads after 6144 keys took 247 us, with these 235, on one card;
//     as it is now, 225 to 231 on four.)
// The keys of long caches are cut into parts, workgroups of their own, that leave fp32 rows for a merge.
//
// Pages: a lane's copy names its own address, so a block's keys may lie on any pages and start anywhere.  The table's entries come into LDS two blocks ahead, by
// the same asynchronous copies; one lane a key turns them into addresses of its key and its value, which the copies' lanes take from LDS.  Keys
// that nothing in the workgroup sees (behind the last, on a page that is not there) are read from a row of zeros.
//
// What a row sees of 32 keys is one word: up to its own position, from its window's first key on or among the sinks, on pages that are there, and of
// the new tokens those of its branch.
//
// P is rounded to the operands' type, which the matrix instruction asks for: independent errors of half a step, which the sum over the keys averages, beside the one
// of O (relative error against 64 bits, bf16 2.3e-3 where O's alone is 1.7e-3).  A second product of what the rounding leaves would double V's.  Sums,
// statistics and parts' rows stay in 32 bits.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include "paged.h"
#include "swa.h"

namespace ua {

constexpr int kPagedWaves = 4, kPagedMaxParts = 64;
__device__ __attribute__((aligned(256))) const uint32_t kZeroRow[64] = {};

// P is held times 2^bits of the largest score's (as in the other kernels of these types).
template <class T> constexpr float kFewBits = 0.f;
template <> constexpr float kFewBits<fp16> = 14.f;
template <class T> struct ManyRaise;
template <> struct ManyRaise<bf16> { static constexpr float kSum = 16777216.f, kBits = 0.f; };
template <> struct ManyRaise<fp16> { static constexpr float kSum = 32768.f, kBits = 7.f; };

struct PagedRows { const char* rows; int64_t page, slot, head; };       // strides in bytes
struct PagedParams {
  const void* q;
  PagedRows k, v;
  void* o;
  float* lse;
  PagedSteps steps;
  PagedTable pages;
  Strides3 qs, os;
  int n_heads, n_kv_heads, group, left, sinks, rows, n_tiles, n_parts, least;       // left: kFar = no bound; rows: of a key head; least: blocks of a part
  float scale_log2;
  float *part_o, *part_lse;
  int64_t o_part, lse_part;
  Div by_kv_heads, by_group, by_tiles, by_walks;      // by_walks: parts and key heads of a sequence
  int batch, n_groups, sorted, eight_shift;
};

// The kernel's parameters read again: those that only a walk's end needs do not occupy scalar registers during the walk.
__device__ __forceinline__ const PagedParams& parameters() {
  typedef const __attribute__((address_space(4))) PagedParams* kernarg;
  kernarg at = (kernarg)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  return *(const PagedParams*)at;
}

// A lane's 16 bytes (4 bytes) from its own address into LDS, lane l at +16 l (+4 l) of the wave-uniform `lds`; see dma16_abs.
__device__ __forceinline__ void dma16_at(uint64_t from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(lds), "v"(from) : "m0");
}
__device__ __forceinline__ void dma4_at(uint64_t from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" :: "s"(lds), "v"(from) : "m0");
}

// The r-th longest of up to 64 sequences (the first of equal ones first), a lane a sequence: launches of many workgroups take the longest walks first, so that
// they do not end alone.
__device__ __forceinline__ StepOf ranked(const PagedParams& p, int r, int& b) {
  const int lane = fresh_lane();
  const StepOf mine = step_of(p.steps, min(lane, p.batch - 1));
  int rank = 0;
  for (int i = 0; i < p.batch; ++i) {
    const int len = __builtin_amdgcn_readlane(mine.len, i);
    rank += len > mine.len || (len == mine.len && i < lane);
  }
  b = __ffsll((unsigned long long)__builtin_amdgcn_ballot_w64(rank == r && lane < p.batch)) - 1;
  return {__builtin_amdgcn_readlane(mine.len, b), __builtin_amdgcn_readlane(mine.n, b), __builtin_amdgcn_readlane(mine.base, b)};
}

// Blocks of kKeys keys that a tile's tokens t0 .. t1 see: the sinks before the window, then the window's first key on.
template <int kKeys>
struct PagedWalk {
  int n_sink, n, start, sinks_end, last;              // keys that a row sees: before sinks_end, and start .. last
  __device__ __forceinline__ PagedWalk(const PagedParams& p, const StepOf& of, int t0, int t1) {
    const bool any = t0 < of.n;
    last = any ? min(of.base + min(t1, of.n - 1), p.pages.room - 1) : -1;
    start = max(of.base + (p.steps.parents ? 0 : t0) - p.left, 0);
    sinks_end = max(min(min(p.sinks, start), last + 1), 0);
    n_sink = (sinks_end + kKeys - 1) / kKeys;
    n = n_sink + (last >= start ? (last - start) / kKeys + 1 : 0);
  }
  // Parts that the walk is cut into: all of p.n_parts, but no more than its blocks in runs of p.least, a last shorter run included.  A part takes every so many-th
  // block, so that parts differ by one, and may have fewer than p.least.
  __device__ __forceinline__ int parts(const PagedParams& p) const { return min(p.n_parts, max((n + p.least - 1) / p.least, 1)); }
  __device__ __forceinline__ int at(int i) const { return i < n_sink ? i * kKeys : start + (i - n_sink) * kKeys; }
  __device__ __forceinline__ int end_of(int i) const { return i < n_sink ? sinks_end : last + 1; }
};

// How a wave gets at kRows keys of a block: lane l stands for key row_of(l % kRows), its K (l / kRows even) or its V.
template <int kRows>
struct PagedLane {
  uint64_t base;
  int64_t page, slot;
  __device__ __forceinline__ PagedLane(const PagedParams& p, int hk, int lane) {
    const bool second = (lane / kRows) & 1;
    base = reinterpret_cast<uint64_t>(second ? p.v.rows + hk * p.v.head : p.k.rows + hk * p.k.head);
    page = second ? p.v.page : p.k.page;
    slot = second ? p.v.slot : p.k.slot;
  }
  // The key's entry on its way into LDS (of keys behind the last: the last one's).
  static __device__ __forceinline__ void fetch(const PagedParams& p, const int32_t* line, int key, int last, uint32_t lds) {
    dma4_at(reinterpret_cast<uint64_t>(line + quotient(min(max(key, 0), last), p.pages.by_page)), lds);
  }
  // The key's address, or zeros', from its entry; whether it is there.
  __device__ __forceinline__ uint64_t address(const PagedParams& p, int key, int end, int entry, bool& there) const {
    const int k = min(key, end - 1), i = quotient(max(k, 0), p.pages.by_page), in_page = k - i * p.pages.page;
    there = key < end && (uint32_t)entry < (uint32_t)p.pages.n_pages;
    return there ? base + (uint64_t)((int64_t)entry * page) + (uint64_t)((int64_t)in_page * slot) : reinterpret_cast<uint64_t>(kZeroRow);
  }
};

// The branches of a sequence's tokens: bit j of a token's 256 is set if it is token j or comes behind it.  Words 1 .. 8 of a token's line hold them, word 0
// stands for the cache's rows before (all seen); word 9, which is shifted in behind the last bit, no row gets to.
constexpr int kDepth = 9, kExit = 10, kBranchPitch = 11;       // (words; odd, so that 32 tokens' lines meet 32 banks)
struct Branches { uint32_t line[kTreeMost * kBranchPitch]; };
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }
// (see tree_part.)  A window cuts what is further behind and not among the sinks.  Of up to 64 tokens every wave stores all lines, with no barrier behind: each word
// once, as it is read, so that no wave puts back what another reads already; what is cut is cut in registers.  kMost: tokens that the kernel takes at the most.
template <int kMost>
__device__ __forceinline__ void tree_branches(const PagedParams& p, const StepOf& of, int parent, Branches& out) {
  const int t = tree_token(p.steps), words = 2 * (t >> 6);
  const bool alone = kMost <= 64 || p.steps.n_tokens <= 64, cut = p.left < p.steps.n_tokens;
  const TreePart x = tree_part(t, parent);
  uint32_t* const line = out.line + t * kBranchPitch;
  int depth = __popc(x.bits[0]) + __popc(x.bits[1]) - 1;
  line[0] = ~0u;
  if (alone) {
    uint64_t bits = (uint64_t)x.bits[1] << 32 | x.bits[0];
    if (cut)
      for (int j = 0; j < p.steps.n_tokens; ++j) {        // (the wave's lanes are the tokens)
        const int theirs = __builtin_amdgcn_readlane(depth, j);
        if (depth - theirs > p.left && of.base + theirs >= p.sinks) bits &= ~(1ull << j);
      }
    line[1] = (uint32_t)bits;
    line[2] = (uint32_t)(bits >> 32);
    line[3] = 0u;
    line[kDepth] = depth;
  } else {
    line[1 + words] = x.bits[0];
    line[2 + words] = x.bits[1];
    line[kExit] = x.exit;
    for (int w = 0; w < kTreeMost / 32; ++w)
      if (w < words || w > words + 1) line[1 + w] = 0u;
    __syncthreads();
    for (int at = x.exit; at >= 0;) {                     // (of another token's line only what it wrote before the barrier is read)
      const uint32_t* const theirs = out.line + at * kBranchPitch;
      const int there = 2 * (at >> 6);
      const uint32_t lo = theirs[1 + there], hi = theirs[2 + there];
      line[1 + there] = lo;
      line[2 + there] = hi;
      depth += __popc(lo) + __popc(hi);
      at = (int)theirs[kExit];
    }
    line[kDepth] = depth;
    __syncthreads();
    if (cut) {                                            // (of its own line, by its one thread; of the others only the depths are read)
      asm volatile("" ::: "memory");
      for (int w = 0; w <= words + 1; ++w) {
        const uint32_t all = line[1 + w];
        uint32_t kept = all;
        for (uint32_t rest = all; rest; rest &= rest - 1) {
          const int theirs = (int)out.line[(32 * w + __ffs(rest) - 1) * kBranchPitch + kDepth];
          if (depth - theirs > p.left && of.base + theirs >= p.sinks) kept &= ~(rest & -rest);
        }
        line[1 + w] = kept;
      }
      __syncthreads();
    }
  }
  asm volatile("" ::: "memory");
}

// What a row sees.
struct RowSees {
  int hi, lo, sinks, base;                              // keys lo .. hi and those before `sinks`, up to hi
  const uint32_t* bits;                                 // its token's branch
  template <bool kTree>
  __device__ __forceinline__ void of(const PagedParams& p, const StepOf& step, int token, const Branches& branches) {
    const bool real = token < step.n;
    const int pos = step.base + (kTree ? (int)branches.line[token * kBranchPitch + kDepth] : token);
    hi = real ? min(step.base + token, p.pages.room - 1) : -1;
    lo = kTree ? min(pos - p.left, step.base) : pos - p.left;
    sinks = p.sinks;
    base = step.base;
    bits = branches.line + token * kBranchPitch;
  }
  // of keys key .. key + 31
  template <bool kTree>
  __device__ __forceinline__ uint32_t word(int key) const {
    uint32_t w = below(hi + 1 - key) & (~below(lo - key) | below(sinks - key));
    if (kTree) {
      const int s = min(max(key - base, -32), 255), i = (s >> 5) + 1;
      w &= __builtin_amdgcn_alignbit(bits[i + 1], bits[i], s & 31);
    }
    return w;
  }
};

// A workgroup of a part that a short walk does not have: rows that saw nothing.  (No copy may still be on its way into LDS.)
__device__ __forceinline__ void leave_part(const PagedParams& p, int part, int b, int hk, int row0, int row1) {
  for (int row = row0 + threadIdx.x; row <= row1; row += blockDim.x) {
    const int token = quotient(row, p.by_group);
    p.part_lse[part * p.lse_part + ((int64_t)b * p.n_heads + hk * p.group + row - token * p.group) * p.steps.n_tokens + token] = -INFINITY;
  }
  wait_vmem_all();
}

template <int kD>
struct FewHead {
  static constexpr int kKeys = 32, kRow = 2 * kD, kChunks = kD / 8, kCopyRows = 1024 / kRow, kUnits = kKeys / kCopyRows, kTile = kUnits * 1024;
  static constexpr int kStage = 2 * kTile, kWave = 2 * kStage, kSteps = kD / 32, kBlocks = kD / 16;
  static constexpr int kEntries = 256, kTable = 2 * kEntries + 512;       // of a wave: two blocks' entries, a block's addresses
  // K: 16 rows are read at one chunk.  V is read transposed: 8 rows at two chunks that start at a multiple of two.
  static __device__ __forceinline__ int slot_k(int r, int c) { return kD == 128 ? c ^ (r & 15) : c ^ (r >> 1 & 7); }
  static __device__ __forceinline__ int slot_v(int r, int c) { return kD == 128 ? c ^ ((r & 3) << 2) ^ ((r >> 2 & 1) << 1) : c ^ ((r >> 1 & 3) << 1); }
};
struct NoBranches { uint32_t line[1]; };

template <class T, int kD, int kTiles, bool kTree>
__global__ __launch_bounds__(64 * kPagedWaves, 2) void paged_few_kernel(const PagedParams p) {
  using H = FewHead<kD>;
  using V = SwaVec<T>;
  typedef typename V::x8 x8;
  constexpr int kRows = 16 * kTiles, kOutPitch = 4 * kD + 16;             // (bytes of a row of fp32 at the merge)
  static_assert(kRows * kOutPitch + 8 * kRows <= H::kWave, "a wave's rows and statistics fit its stages");
  __shared__ __attribute__((aligned(1024))) unsigned char smem[kPagedWaves * H::kWave];
  __shared__ __attribute__((aligned(256))) unsigned char tables[kPagedWaves * H::kTable];
  __shared__ std::conditional_t<kTree, Branches, NoBranches> branch_store;
  Branches& branches = reinterpret_cast<Branches&>(branch_store);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_byte*)smem;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, quad = lane >> 4;
  const int r = quotient(blockIdx.x, p.by_walks), of_r = blockIdx.x - r * p.by_walks.d, part = quotient(of_r, p.by_kv_heads), hk = of_r - part * p.n_kv_heads;
  int b = r;
  const StepOf step = p.sorted ? ranked(p, r, b) : step_of(p.steps, r);
  constexpr int row0 = 0;
  const int row1 = p.rows - 1;
  const int32_t* const line = p.pages.table + b * p.pages.stride;
  const uint32_t mine = lds0 + wave * H::kWave, entries = (uint32_t)(uintptr_t)(lds_byte*)tables + wave * H::kTable, places = entries + 2 * H::kEntries;
  const int key_row = lane & 31, copy_row = lane / H::kChunks, chunk = lane % H::kChunks;
  // What does not depend on the length is on its way before it has come: the first two blocks' entries where there is no window (if the walk then turns out to
  // be cut into fewer parts, the second's again), the tree, Q.
  int i = part * kPagedWaves + wave;
  const bool early = p.left == kFar && p.pages.room > 0;
  if (early) {
    PagedLane<32>::fetch(p, line, 32 * i + key_row, p.pages.room - 1, entries);
    PagedLane<32>::fetch(p, line, 32 * (i + kPagedWaves * p.n_parts) + key_row, p.pages.room - 1, entries + H::kEntries);
  }
  int parent = kTree ? parent_of(p.steps, b, tree_token(p.steps)) : -1;
  // Q as B operands: row col of the tile, columns 32 s + 8 quad ..
  x8 qf[kTiles][H::kSteps];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const int row = min(row0 + 16 * t + col, p.rows - 1), token = quotient(row, p.by_group), h = hk * p.group + row - token * p.group;
    const T* q = (const T*)p.q + b * p.qs.b + token * p.qs.s + h * p.qs.h + 8 * quad;
#pragma unroll
    for (int s = 0; s < H::kSteps; ++s) qf[t][s] = *reinterpret_cast<const x8*>(q + 32 * s);
  }
  const PagedLane<32> from(p, hk, lane);
  const PagedWalk<H::kKeys> walk(p, step, quotient(row0, p.by_group), quotient(row1, p.by_group));
  const int parts = walk.parts(p), stride = kPagedWaves * parts, i1 = walk.n;
  auto fetch = [&](int i, uint32_t to) { from.fetch(p, line, walk.at(i) + key_row, walk.last, to); };
  // The block's addresses into LDS; which of its keys are there.
  auto locate = [&](int i, uint32_t entry_at) {
    bool there;
    const uint64_t a = from.address(p, walk.at(i) + key_row, walk.end_of(i), lds_get<int>(entry_at + 4 * lane), there);
    lds_put(places + 8 * lane, a);
    return (uint32_t)__builtin_amdgcn_ballot_w64(there);
  };
  // (all addresses are read before the first copy: read one by one, with a wait each, 16 copies took 2000 cycles)
  auto copy_in = [&](uint32_t stage) {
    uint64_t k[H::kUnits], v[H::kUnits];
#pragma unroll
    for (int u = 0; u < H::kUnits; ++u) {
      k[u] = lds_get<uint64_t>(places + 8 * (H::kCopyRows * u + copy_row));
      v[u] = lds_get<uint64_t>(places + 256 + 8 * (H::kCopyRows * u + copy_row));
    }
    asm volatile("" ::: "memory");
#pragma unroll
    for (int u = 0; u < H::kUnits; ++u) {
      const int r = H::kCopyRows * u + copy_row;
      dma16_at(k[u] + 16 * H::slot_k(r, chunk), stage + 1024 * u);
      dma16_at(v[u] + 16 * H::slot_v(r, chunk), stage + H::kTile + 1024 * u);
    }
  };
  constexpr int kCopies = 2 * H::kUnits;
  if (part >= parts) {
    leave_part(p, part, b, hk, row0, row1);
    return;
  }
  if (!early && i < i1) fetch(i, entries);
  if ((!early || parts != p.n_parts) && i + stride < i1) {
    if (early) wait_vmem_all();                            // (the same place in LDS)
    fetch(i + stride, entries + H::kEntries);
  }
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int s = 0; s < H::kSteps; ++s) asm volatile("" : "+v"(qf[t][s]));     // arrived before the walk counts its copies
  asm volatile("" : "+v"(parent));
  wait_vmem_all();
  uint32_t there = 0, there_next = 0;
  // (Nothing is copied of blocks that are none: a CU's four waves bring 64 bytes a cycle, so a block of each is 1000 cycles.)
  if (i < i1) {
    there = locate(i, entries);
    copy_in(mine);
    if (i + stride < i1) {
      there_next = locate(i + stride, entries + H::kEntries);
      if (i + 2 * stride < i1) fetch(i + 2 * stride, entries);
      copy_in(mine + H::kStage);
    }
  }
  if constexpr (kTree) tree_branches<kRows>(p, step, parent, branches);
  RowSees sees[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) sees[t].template of<kTree>(p, step, quotient(min(row0 + 16 * t + col, p.rows - 1), p.by_group), branches);
  f32x4 o[kTiles][H::kBlocks];
  float m_run[kTiles], m_use[kTiles], l_run[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    m_run[t] = -INFINITY;
    m_use[t] = l_run[t] = 0.f;
#pragma unroll
    for (int d = 0; d < H::kBlocks; ++d) o[t][d] = f32x4{0};
  }
  uint32_t stage = mine, other = mine + H::kStage, entry_now = entries, entry_next = entries + H::kEntries;
  for (; i < i1; i += stride) {
    // (in flight: this block, the entries two blocks on, the next block)
    if (i + stride < i1) asm volatile("s_waitcnt vmcnt(%0)" :: "n"(kCopies) : "memory");
    else                 wait_vmem_all();
    const bool copies = i + 2 * stride < i1;
    const uint32_t there_after = copies ? locate(i + 2 * stride, entry_now) : 0;
    const int key0 = walk.at(i);
    x8 kf[2][H::kSteps];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int s = 0; s < H::kSteps; ++s) {
        const int r = 16 * n + col;
        kf[n][s] = lds_get<x8>(stage + r * H::kRow + (H::slot_k(r, 4 * s + quad) << 4));
      }
    x8 vf[H::kBlocks];
#pragma unroll
    for (int d = 0; d < H::kBlocks; ++d) {
      const int r = 4 * quad + (col >> 2), c = 2 * d + ((col & 3) >> 1);
      const uint32_t at = stage + H::kTile + r * H::kRow + (H::slot_v(r, c) << 4) + (col & 1) * 8;        // (row + 16: the same slot)
      vf[d] = lds_tr_pair<T>(at, at + 16 * H::kRow);
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      f32x4 s[2] = {f32x4{0}, f32x4{0}};
#pragma unroll
      for (int k = 0; k < H::kSteps; ++k)
#pragma unroll
        for (int n = 0; n < 2; ++n) s[n] = V::mfma16(kf[n][k], qf[t][k], s[n]);
      const uint32_t seen = (sees[t].template word<kTree>(key0) & there) >> (4 * quad);
      float mx = -INFINITY, a, c;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (!(seen >> (16 * n + j) & 1)) s[n][j] = -INFINITY;
          mx = fmaxf(mx, s[n][j]);
        }
      swap_lanes<16>(mx, a, c);
      swap_lanes<32>(fmaxf(a, c), a, c);
      mx = fmaxf(a, c) * p.scale_log2;
      if (__builtin_amdgcn_ballot_w64(mx > m_run[t]) != 0) {
        const float m_new = fmaxf(m_run[t], mx);
        m_use[t] = m_new == -INFINITY ? 0.f : m_new - kFewBits<T>;
        const float alpha = m_new == m_run[t] ? 1.f : fast_exp2(m_run[t] - m_new);
        m_run[t] = m_new;
        l_run[t] *= alpha;
#pragma unroll
        for (int d = 0; d < H::kBlocks; ++d) o[t][d] *= alpha;
      }
      x8 pf;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float e = fast_exp2(fmaf(s[n][j], p.scale_log2, -m_use[t]));
          l_run[t] += e;
          pf[4 * n + j] = (T)e;
        }
#pragma unroll
      for (int d = 0; d < H::kBlocks; ++d) o[t][d] = V::mfma16(vf[d], pf, o[t][d]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                    // everything of this stage is in registers
    if (copies) {
      if (i + 3 * stride < i1) fetch(i + 3 * stride, entry_next);
      copy_in(stage);
    }
    there = there_next;
    there_next = there_after;
    const uint32_t x = stage, y = entry_now;
    stage = other;
    other = x;
    entry_now = entry_next;
    entry_next = y;
  }
  wait_vmem_all();
  // ---- the waves' rows: O as fp32, then the reference and the sum of each
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    float a, c;
    swap_lanes<16>(l_run[t], a, c);
    swap_lanes<32>(a + c, a, c);
#pragma unroll
    for (int d = 0; d < H::kBlocks; ++d) lds_put(mine + (16 * t + col) * kOutPitch + (16 * d + 4 * quad) * 4, o[t][d]);
    if (quad == 0) {
      lds_put(mine + kRows * kOutPitch + 8 * (16 * t + col), m_run[t]);
      lds_put(mine + kRows * kOutPitch + 8 * (16 * t + col) + 4, a + c);
    }
  }
  __syncthreads();
  constexpr int kPer = kD / 16;
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const int r = 16 * t + (threadIdx.x >> 4), c = threadIdx.x & 15, row = row0 + r;
    if (row >= p.rows) continue;
    float m = -INFINITY, l = 0.f, acc[kPer] = {};
#pragma unroll
    for (int w = 0; w < kPagedWaves; ++w) m = fmaxf(m, lds_get<float>(lds0 + w * H::kWave + kRows * kOutPitch + 8 * r));
    const float at = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kPagedWaves; ++w) {
      const uint32_t rows = lds0 + w * H::kWave;
      const float f = fast_exp2(lds_get<float>(rows + kRows * kOutPitch + 8 * r) - at);
      l += f * lds_get<float>(rows + kRows * kOutPitch + 8 * r + 4);
#pragma unroll
      for (int j = 0; j < kPer; j += 4) {
        const f32x4 x = lds_get<f32x4>(rows + r * kOutPitch + (c * kPer + j) * 4);
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[j + n] += f * x[n];
      }
    }
    const bool any = l > 0.f || l != l;                                  // (NaN stays)
    const float inv = any ? 1.f / l : 0.f, lse = any ? (m - kFewBits<T> + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
    const int token = quotient(row, p.by_group), h = hk * p.group + row - token * p.group;
    const int64_t out_row = ((int64_t)b * p.n_heads + h) * p.steps.n_tokens + token;
    if (p.n_parts > 1) {
      if (c == 0) p.part_lse[part * p.lse_part + out_row] = lse;
      if (any) {
        float* to = p.part_o + part * p.o_part + out_row * kD + c * kPer;
#pragma unroll
        for (int j = 0; j < kPer; j += 4) *reinterpret_cast<f32x4*>(to + j) = f32x4{acc[j] * inv, acc[j + 1] * inv, acc[j + 2] * inv, acc[j + 3] * inv};
      }
    } else {
      typedef __attribute__((ext_vector_type(kPer))) T vec;
      vec w;
#pragma unroll
      for (int j = 0; j < kPer; ++j) w[j] = any ? (T)(acc[j] * inv) : (T)0.f;
      *reinterpret_cast<vec*>((T*)p.o + b * p.os.b + token * p.os.s + h * p.os.h + c * kPer) = w;
      if (c == 0) p.lse[out_row] = lse;
    }
  }
}

// ---- many rows ------------------------------------------------------------------------------------------------------------
// Row of a tile's wave (of 32) -> token, query head.
struct RowPlace { int token, head; };
__device__ __forceinline__ RowPlace row_place(const PagedParams& p, int hk, int row) {
  const int token = quotient(row, p.by_group);
  return {token, hk * p.group + row - token * p.group};
}

// Three workgroups of heads of 64 share a CU (two: 4 prompts of 2048 tokens of 8 x 4 heads 119 us where they take 108; 16 trees of 64 tokens after 2048 to 8192 keys
// 85 and 77; one prompt of 2048 after 6144, which more parts than two a CU do not help, 152 and 160).
template <class T, int kD, bool kTree>
__global__ __launch_bounds__(256, kD == 64 ? 3 : 2) void paged_many_kernel(const PagedParams p) {
  using H = SwaHead<kD>;
  using V = SwaVec<T>;
  typedef typename V::x8 x8;
  using F = FewHead<kD>;                    // (the products' fragments and LDS layout are those of few rows, two tiles of 16 a wave)
  constexpr int kPieces = 2 * H::kCopies, kSecond = H::kTile, kMine = kSwaBlock / kPagedWaves;        // kMine: keys of a block that a wave copies
  static_assert(kMine == 16 && H::kCopies * H::kCopyRows == kMine, "a wave's keys");
  __shared__ __attribute__((aligned(1024))) unsigned char stage_a[2 * H::kTile];
  __shared__ __attribute__((aligned(1024))) unsigned char stage_b[2 * H::kTile];
  __shared__ __attribute__((aligned(256))) unsigned char tables[kPagedWaves * 1024];                  // of a wave: three blocks' entries, a block's addresses
  __shared__ std::conditional_t<kTree, Branches, NoBranches> branch_store;
  Branches& branches = reinterpret_cast<Branches&>(branch_store);
  const uint32_t lds[2] = {(uint32_t)(uintptr_t)(lds_byte*)stage_a, (uint32_t)(uintptr_t)(lds_byte*)stage_b};
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Tiles that read the same keys beside each other, on one XCD if there are whole eights of parts and key heads; then key heads, parts, sequences.  Of one to two
  // workgroups a CU the second ones in reverse, so that long and short walks share a CU.
  const int at = p.n_groups > kCus && p.n_groups <= 2 * kCus && (int)blockIdx.x >= kCus ? p.n_groups - 1 - ((int)blockIdx.x - kCus) : (int)blockIdx.x;
  const int eighth = at >> p.eight_shift, rest = quotient(eighth, p.by_tiles), tile = eighth - rest * p.n_tiles;
  const int walk_at = (rest << p.eight_shift) + (at & ((1 << p.eight_shift) - 1));
  const int r = quotient(walk_at, p.by_walks), of_r = walk_at - r * p.by_walks.d, part = quotient(of_r, p.by_kv_heads), hk = of_r - part * p.n_kv_heads;
  int b = r;
  const StepOf step = p.sorted ? ranked(p, r, b) : step_of(p.steps, r);
  const int r0 = tile * kSwaRows, row0 = r0 + 32 * wave, n_rows = p.rows - row0;      // rows of this wave that exist (may be <= 0)
  const int32_t* const line = p.pages.table + b * p.pages.stride;
  const uint32_t entries = (uint32_t)(uintptr_t)(lds_byte*)tables + wave * 1024, entries_first = entries + 512, places = entries + 768;
  const int m = lane & (kMine - 1), key_row = H::kCopyRows * (kPagedWaves * (m / H::kCopyRows) + wave) + m % H::kCopyRows;
  const int copy_row = lane / H::kChunks, slot_row = H::kCopyRows * wave + copy_row, chunk = lane % H::kChunks;
  const uint32_t k_chunk = 16 * F::slot_k(slot_row, chunk), v_chunk = 16 * F::slot_v(slot_row, chunk);
  // (as with few rows: what does not depend on the length first)
  const bool early = p.left == kFar && p.pages.room > 0;
  if (early) {
    PagedLane<kMine>::fetch(p, line, kSwaBlock * part + lane, p.pages.room - 1, entries_first);
    PagedLane<kMine>::fetch(p, line, kSwaBlock * (part + p.n_parts) + lane, p.pages.room - 1, entries + 256);
    PagedLane<kMine>::fetch(p, line, kSwaBlock * (part + 2 * p.n_parts) + lane, p.pages.room - 1, entries);
  }
  int parent = kTree ? parent_of(p.steps, b, tree_token(p.steps)) : -1;
  const int col = lane & 15, quad = lane >> 4;
  x8 qf[2][F::kSteps];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const RowPlace r = row_place(p, hk, min(row0 + 16 * t + col, p.rows - 1));
    const T* q = (const T*)p.q + b * p.qs.b + r.token * p.qs.s + r.head * p.qs.h + 8 * quad;
#pragma unroll
    for (int k = 0; k < F::kSteps; ++k) qf[t][k] = *reinterpret_cast<const x8*>(q + 32 * k);
  }
  const PagedLane<kMine> from(p, hk, lane);
  const PagedWalk<kSwaBlock> walk(p, step, quotient(r0, p.by_group), quotient(min(r0 + kSwaRows, p.rows) - 1, p.by_group));
  const int parts = walk.parts(p), i0 = part, i1 = walk.n;
  auto fetch = [&](int i, uint32_t at) { from.fetch(p, line, walk.at(i) + lane, walk.last, at); };
  // Of the block after the next: the addresses into LDS, and which keys are there.
  uint64_t there = 0, there_next = 0, there_after = 0;
  auto locate = [&](int i, int entry_mine, int entry_lane) {
    bool is;
    const int key0 = walk.at(i), end = i < i1 ? walk.end_of(i) : 0;
    const uint64_t a = from.address(p, key0 + key_row, end, entry_mine, is);
    if (lane < 2 * kMine) lds_put(places + 8 * lane, a);
    there_after = __builtin_amdgcn_ballot_w64(key0 + lane < end && (uint32_t)entry_lane < (uint32_t)p.pages.n_pages);
  };
  const uint32_t mine_at = entries + 4 * key_row, lane_at = entries + 4 * lane;
  auto place = [&](int n) { return lds_get<uint64_t>(places + 128 * (n & 1) + 8 * (H::kCopyRows * (n >> 1) + copy_row)) + (n & 1 ? v_chunk : k_chunk); };
  auto copy = [&](int n, uint64_t a, uint32_t stage) {
    dma16_at(a, stage + (n & 1 ? kSecond : 0) + (kPagedWaves * (n >> 1) + wave) * 1024);
  };
  if (part >= parts) {
    leave_part(p, part, b, hk, r0, min(r0 + kSwaRows, p.rows) - 1);
    return;
  }
  if (i0 < i1 && (!early || parts != p.n_parts)) {
    if (early) wait_vmem_all();                            // (the same places in LDS)
    else       fetch(i0, entries_first);
    fetch(i0 + parts, entries + 256);
    fetch(i0 + 2 * parts, entries);
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int k = 0; k < F::kSteps; ++k) asm volatile("" : "+v"(qf[t][k]));
  asm volatile("" : "+v"(parent));
  wait_vmem_all();
  if (i0 < i1) {
    locate(i0, lds_get<int>(mine_at + 512), lds_get<int>(lane_at + 512));
    there = there_after;
    uint64_t at[kPieces];
#pragma unroll
    for (int n = 0; n < kPieces; ++n) at[n] = place(n);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int n = 0; n < kPieces; ++n) copy(n, at[n], lds[0]);
    locate(i0 + parts, lds_get<int>(mine_at + 256), lds_get<int>(lane_at + 256));
    there_next = there_after;
  }
  if (kTree && i0 < i1) tree_branches<kTreeMost>(p, step, parent, branches);
  RowSees sees[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) sees[t].template of<kTree>(p, step, quotient(min(row0 + 16 * t + col, p.rows - 1), p.by_group), branches);
  // Keys that every real row of the wave sees: from .. to - 1, and those before `sinks` up to there.
  const int t_first = quotient(min(row0, p.rows - 1), p.by_group), t_last = min(quotient(min(row0 + 31, p.rows - 1), p.by_group), step.n - 1);
  const int all_to = min(kTree ? step.base : step.base + t_first + 1, p.pages.room), all_from = step.base + (kTree ? step.n - 1 : t_last) - p.left;
  const int some_to = t_first >= step.n ? 0 : kTree ? walk.last + 1 : step.base + t_last + 1, some_from = step.base + (kTree ? 0 : t_first) - p.left;
  f32x4 o[2][F::kBlocks];
  float m_run[2], m_use[2], l_run[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    m_run[t] = -INFINITY;
    m_use[t] = l_run[t] = 0.f;
#pragma unroll
    for (int d = 0; d < F::kBlocks; ++d) o[t][d] = f32x4{0};
  }
  uint32_t nat[F::kSteps], tr[F::kBlocks];
#pragma unroll
  for (int k = 0; k < F::kSteps; ++k) nat[k] = col * F::kRow + (F::slot_k(col, 4 * k + quad) << 4);
#pragma unroll
  for (int d = 0; d < F::kBlocks; ++d) {
    const int r = 4 * quad + (col >> 2);
    tr[d] = kSecond + r * F::kRow + (F::slot_v(r, 2 * d + ((col & 3) >> 1)) << 4) + (col & 1) * 8;
  }

  auto walk_step = [&](int i, auto stage_tag) {
    constexpr int kStage = decltype(stage_tag)::value;
    const uint32_t here = lds[kStage], other = lds[kStage ^ 1];
    const int key0 = walk.at(i);
    wait_vmem_all();
    __syncthreads();                        // this block and the entries two blocks on have landed, and everyone has left the other stage
    // Addresses of the next block, made a step ago; entries of the one after it, to make its addresses of beside the products.
    uint64_t at[kPieces];
#pragma unroll
    for (int n = 0; n < kPieces; ++n) at[n] = place(n);
    asm volatile("" ::: "memory");          // (read at once, not one by one before its copy)
    const int mine_after = lds_get<int>(mine_at + 256 * kStage), lane_after = lds_get<int>(lane_at + 256 * kStage);
    fetch(i + 3 * parts, entries + 256 * (kStage ^ 1));
    auto turn_over = [&]() {
      locate(i + 2 * parts, mine_after, lane_after);
      there = there_next;
      there_next = there_after;
    };
    const bool hidden = n_rows <= 0 || key0 >= some_to || (key0 + kSwaBlock <= some_from && key0 >= p.sinks);
    if (hidden) {
#pragma unroll
      for (int n = 0; n < kPieces; ++n) copy(n, at[n], other);
      turn_over();
      return;
    }
    // S^T: four blocks of 16 keys in turn, either of the wave's tiles.  From here through the exponentials the wave goes before the SIMD's other one, so that
    // the two take turns, one's K products beside the other's V products: 2048 tokens of 8 x 4 heads after 6144 keys 245 -> 229 us (one card, in turn),
    // D = 64 157 -> 150; first through K's products alone 228 and 159, through V's products too 245 and 154, exponentials alone 242 and 152.
    __builtin_amdgcn_s_setprio(1);
    f32x4 s[2][4];
    {
      constexpr int kAhead = 4, kAll = 4 * F::kSteps;
      x8 kf[kAll];
      auto rd = [&](int n) { return lds_get<x8>(here + nat[n >> 2] + 16 * F::kRow * (n & 3)); };
#pragma unroll
      for (int n = 0; n < kAhead; ++n) kf[n] = rd(n);
      __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
      for (int n = 0; n < kAll; ++n) {
        if (n + kAhead < kAll) kf[n + kAhead] = rd(n + kAhead);
#pragma unroll
        for (int t = 0; t < 2; ++t) s[t][n & 3] = V::mfma16(kf[n], qf[t][n >> 2], n < 4 ? f32x4{0} : s[t][n & 3]);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (n & 1) copy(n >> 1, at[n >> 1], other);
      }
      static_assert(kAll / 2 == kPieces, "a copy after every other fragment");
    }
    const bool whole = key0 + kSwaBlock <= all_to && (key0 >= all_from || key0 + kSwaBlock <= p.sinks) && there == ~0ull;
    if (!whole) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t seen = (sees[t].template word<kTree>(key0 + 32 * half) & (uint32_t)(there >> (32 * half))) >> (4 * quad);
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (!(seen >> (16 * n + j) & 1)) s[t][2 * half + n][j] = -INFINITY;
        }
    }
    constexpr int kVAhead = kD == 64 ? 2 : 3, kVAll = 2 * F::kBlocks;
    x8 vf[4];
    auto rd_v = [&](int n) {                // fragment n % kBlocks of 32 keys
      const uint32_t a = here + tr[n % F::kBlocks] + 32 * F::kRow * (n / F::kBlocks);
      return lds_tr_pair<T>(a, a + 16 * F::kRow);
    };
#pragma unroll
    for (int n = 0; n < kVAhead; ++n) vf[n] = rd_v(n);
    float rs[2];
    x8 pf[2][2];
    auto exponentials = [&]() {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        rs[t] = 0.f;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float e = fast_exp2(fmaf(s[t][n][j], p.scale_log2, -m_use[t]));
            rs[t] += e;
            pf[t][n >> 1][4 * (n & 1) + j] = (T)e;
          }
      }
    };
    exponentials();
    __builtin_amdgcn_s_setprio(0);
    if (__builtin_amdgcn_ballot_w64(!(rs[0] < ManyRaise<T>::kSum) || !(rs[1] < ManyRaise<T>::kSum) || m_run[0] == -INFINITY || m_run[1] == -INFINITY) != 0) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {         // wave-uniform, rare
        float mx = s[t][0][0], a, c;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) mx = fmaxf(mx, s[t][n][j]);
        swap_lanes<16>(mx, a, c);
        swap_lanes<32>(fmaxf(a, c), a, c);
        const float m_new = fmaxf(m_run[t], fmaxf(a, c) * p.scale_log2);
        m_use[t] = m_new == -INFINITY ? 0.f : m_new - ManyRaise<T>::kBits;
        const float alpha = m_new == m_run[t] ? 1.f : fast_exp2(m_run[t] - m_new);      // m_run = -inf -> 0
        m_run[t] = m_new;
        l_run[t] *= alpha;
#pragma unroll
        for (int d = 0; d < F::kBlocks; ++d) o[t][d] *= alpha;
      }
      exponentials();
    }
    l_run[0] += rs[0];
    l_run[1] += rs[1];
    turn_over();
#pragma unroll
    for (int n = 0; n < kVAll; ++n) {
      if (n + kVAhead < kVAll) vf[(n + kVAhead) & 3] = rd_v(n + kVAhead);
#pragma unroll
      for (int t = 0; t < 2; ++t) o[t][n % F::kBlocks] = V::mfma16(vf[n & 3], pf[t][n / F::kBlocks], o[t][n % F::kBlocks]);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
  };
  for (int i = i0; i < i1; i += 2 * parts) {
    walk_step(i, std::integral_constant<int, 0>{});
    if (i + parts < i1) walk_step(i + parts, std::integral_constant<int, 1>{});
  }
  wait_vmem_all();                          // the last step's copies filled a stage with zeros
  __syncthreads();
  if (n_rows <= 0) return;
  const PagedParams& e = parameters();
  const uint32_t turn = lds[0] + wave * 32 * H::kRow;
  const int out_lane = fresh_lane(), out_col = out_lane & 15, out_quad = out_lane >> 4;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    float a, c;
    swap_lanes<16>(l_run[t], a, c);
    swap_lanes<32>(a + c, a, c);
    const float l = a + c;
    const int row = row0 + 16 * t + out_col;
    const RowPlace mine = row_place(e, hk, min(row, e.rows - 1));
    const bool any = (l > 0.f || l != l) && mine.token < step.n;         // (NaN stays; a token that is none saw keys beside the others)
    const float inv = any ? 1.f / l : 0.f, lse = any ? (m_use[t] + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
    const int64_t out_row = ((int64_t)b * e.n_heads + mine.head) * e.steps.n_tokens + mine.token;
    if (e.n_parts > 1) {
      if (row < e.rows && any) {
        float* to = e.part_o + part * e.o_part + out_row * kD + 4 * out_quad;
#pragma unroll
        for (int d = 0; d < F::kBlocks; ++d) *reinterpret_cast<f32x4*>(to + 16 * d) = o[t][d] * inv;
      }
      if (row < e.rows && out_quad == 0) e.part_lse[part * e.lse_part + out_row] = lse;
    } else {
      if (row < e.rows && out_quad == 0) e.lse[out_row] = lse;
#pragma unroll
      for (int d = 0; d < F::kBlocks; ++d) {
        typename V::x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = any ? (T)(o[t][d][j] * inv) : (T)0.f;
        lds_put(turn + H::at_n(16 * t + out_col, 2 * d + (out_quad >> 1)) + 8 * (out_quad & 1), w);
      }
    }
  }
  if (e.n_parts > 1) return;
#pragma unroll
  for (int i = 0; i < H::kSteps; ++i) {
    const int r = H::kCopyRows * i + out_lane / H::kChunks, ch = out_lane % H::kChunks;
    const u32x4 x = lds_get<u32x4>(turn + H::at_n(r, ch));
    if (row0 + r < e.rows) {
      const RowPlace at = row_place(e, hk, row0 + r);
      *reinterpret_cast<u32x4*>((T*)e.o + b * e.os.b + at.token * e.os.s + at.head * e.os.h + ch * 8) = x;
    }
  }
}

// ---- parts joined, few rows --------------------------------------------------------------------------------------------------
// As in swa_merge, by a workgroup a row: 16 groups of 16 lanes take the parts' rows side by side, so that all of them are on their way at once and are added
// up through LDS (32 rows of 128 in 32 parts: 5.4 us with the 64 lanes a row of swa_merge, and 3.7 this way).
template <class T, int kD>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedParams p, Div by_heads, Div by_tokens) {
  constexpr int kPer = kD / 16, kMost = kPagedMaxParts / 16;
  __shared__ __attribute__((aligned(16))) float sums[16][kD + 4];
  const int row = blockIdx.x, group = threadIdx.x >> 4, c = threadIdx.x & 15, lane = threadIdx.x & 63;
  const float l = lane < p.n_parts ? p.part_lse[lane * p.lse_part + row] : -INFINITY;
  float top = l;
#pragma unroll
  for (int d = 32; d; d /= 2) top = fmaxf(top, __shfl_xor(top, d));
  const float ref = top == -INFINITY ? 0.f : top, w = l == -INFINITY ? 0.f : fast_exp2((l - ref) * kLog2e);
  float total = w, acc[kPer] = {};
#pragma unroll
  for (int d = 32; d; d /= 2) total += __shfl_xor(total, d);
#pragma unroll
  for (int n = 0; n < kMost; ++n) {
    const int i = 16 * n + group;
    const float f = __shfl(w, i);
    if (i < p.n_parts && f != 0.f) {                     // (a part that saw nothing left no row)
      const float* x = p.part_o + i * p.o_part + (int64_t)row * kD + c * kPer;
#pragma unroll
      for (int j = 0; j < kPer; j += 4) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(x + j);
#pragma unroll
        for (int m = 0; m < 4; ++m) acc[j + m] += f * y[m];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kPer; j += 4) *reinterpret_cast<f32x4*>(&sums[group][c * kPer + j]) = f32x4{acc[j], acc[j + 1], acc[j + 2], acc[j + 3]};
  __syncthreads();
  const bool any = total > 0.f || total != total;        // (NaN stays)
  const int bh = quotient(row, by_tokens), token = row - bh * p.steps.n_tokens, b = quotient(bh, by_heads), h = bh - b * p.n_heads;
  if (threadIdx.x < kD) {
    float x = 0.f;
#pragma unroll
    for (int g = 0; g < 16; ++g) x += sums[g][threadIdx.x];
    ((T*)p.o)[b * p.os.b + token * p.os.s + h * p.os.h + threadIdx.x] = any ? (T)(x / total) : (T)0.f;
  }
  if (threadIdx.x == 0) p.lse[row] = any ? ref + __builtin_amdgcn_logf(total) * kLn2 : -INFINITY;
}

// ---- host -----------------------------------------------------------------------------------------------------------------
// tiles: 16-row tiles of a workgroup of few rows; row_tiles: workgroups of a key head's rows; least: blocks of a part
struct PagedShape { bool many; int tiles, row_tiles, parts, least; };
// Parts of a key head's keys: what an estimate in microseconds says of the longest walks that the call allows (lengths are on the device; shorter walks make fewer
// parts).  Fitted to 2166 (few rows) and 4612 (many) drawn calls of 1 to 64 sequences, 1 to 256 tokens, 60 to 33000 rows, each timed in up to 12 numbers of
// parts: what it takes is 1.3 and 1.8 % slower than the best of them on average, 8 and 10 % at the 95th percentile.  The tables of all
// these calls were as wide as their longest sequence.  Wider ones are cut for the walks that they allow: 26 tokens of 8 x 4 heads after 2751 rows 17.7 us in a table of 2784
// rows, 20.0 of 8192, 23.4 of 32768 and more; 64 x 8 of 8192 to 16384, one token, 555 in 16384 and 584 in 131072.  us in 1, 2, 4, 8, 16 and 32 parts:
//     few    1 x 8, 4000 rows, 128 columns             38.7   25.0   17.3   13.2   11.3   11.2
//            3 x 8, 6007 to 21353                     237    127     72.3   45.9   36.7   40.6
//            64 x 8, 8192 to 16384                    549    560    571    594
//     many   1 x 8, 2777 rows, 26 tokens of 4 heads    58.3   36.1   24.4   19.3   17.8   19.9
//            16 x 8, 2048 to 8192, 64 tokens of 4     171    122    123    155    213    374
//            3 x 8, 700 to 6000, 256 tokens           118     67.5   41.9   32.2   38.6   48.4
static PagedShape paged_shape(int batch, int n_tokens, int n_heads, int n_kv_heads, int room, int head_dim, int64_t left, int64_t sinks) {
  PagedShape s;
  const int64_t rows = (int64_t)n_tokens * (n_heads / n_kv_heads);
  s.many = rows > 32;
  s.tiles = rows <= 16 ? 1 : 2;
  const int tile_rows = s.many ? kSwaRows : 16 * s.tiles, keys = s.many ? kSwaBlock : 32, waves = s.many ? 1 : kPagedWaves;
  s.row_tiles = (int)((rows + tile_rows - 1) / tile_rows);
  s.least = waves;
  int64_t seen = ((int64_t)room + keys - 1) / keys;
  if (left >= 0)
    seen = std::min(seen, (std::min<int64_t>(left, kFar) + n_tokens + 2 * keys - 2) / keys + (std::min<int64_t>(sinks, room) + keys - 1) / keys);
  const double walks = (double)batch * n_kv_heads, groups = walks * s.row_tiles, entries = (double)batch * n_tokens * n_heads * head_dim;
  auto few_us = [&](int parts) {
    const double step = head_dim == 64 ? 0.83 : 1.41, slots = head_dim == 64 ? 2 * kCus : kCus;         // a block of 32 keys a wave
    const double n = groups * parts, steps = std::ceil((double)seen / (waves * parts)), rounds = n <= slots ? 1 : n / slots + 0.66;
    const double memory = walks * seen * keys * head_dim * 4 / 8.1e6 + (batch > 1 ? 0.11 * steps : 0);
    return 2.4 + std::max(rounds * steps * step, memory) + (parts > 1 ? 4.1 + 0.024 * parts + entries * parts * 6e-7 : 0);
  };
  auto many_us = [&](int parts) {
    // a block of 64 keys by a workgroup that has its CU, and by one of two (heads of 64: three) that fill it
    const double alone = head_dim == 64 ? 0.98 : 1.31, shared = head_dim == 64 ? 1.3 : 1.5, slots = (head_dim == 64 ? 3 : 2) * kCus;
    const double n = groups * parts, steps = std::ceil((double)seen / parts), beside = std::min(std::max((n - kCus) / (slots - kCus), 0.0), 1.0);
    double walk = std::max(steps * (alone + (shared - alone) * beside), groups * seen / slots * shared);
    if (n > slots) walk = std::max(walk, (n / slots + 0.43) * steps * shared);
    return 11.9 + walk + (parts > 1 ? 3.3 + entries * parts * 1.84e-6 : 0);
  };
  s.parts = 1;
  double best_us = 1e30;
  // (every number up to 8, then every second, fourth and eighth one: 20 of them, twice a call)
  for (int parts = 1; parts <= kPagedMaxParts && (parts == 1 || waves * (parts - 1) < seen); parts += parts < 8 ? 1 : parts < 16 ? 2 : parts < 32 ? 4 : 8) {
    const double us = s.many ? many_us(parts) : few_us(parts);
    if (us < 0.98 * best_us) { best_us = us; s.parts = parts; }
  }
  return s;
}
constexpr int kJoinRows = 2048;                       // rows up to which a workgroup joins one
static int paged_decode_check(int batch, int n_tokens, int n_heads, int n_kv_heads, int n_pages, int page, int max_pages, int head_dim, int dtype,
                              int64_t table_stride, const int32_t* parents, int64_t parents_stride, int64_t left, int64_t sinks, float scale) {
  const int rc = paged_check(batch, n_tokens, n_kv_heads, n_pages, page, max_pages, table_stride, parents, parents_stride);
  if (rc != UA_OK) return rc;
  if (n_heads <= 0 || n_heads % n_kv_heads || left < -1 || sinks < 0) return UA_ERR_SHAPE;
  if (n_tokens > kSwaMaxLen || (int64_t)n_tokens * (n_heads / n_kv_heads) > kSwaMaxLen || (int64_t)batch * n_tokens * n_heads > INT32_MAX / kPagedMaxParts)
    return UA_ERR_SHAPE;
  if ((head_dim != 64 && head_dim != 128) || (dtype != UA_BF16 && dtype != UA_FP16) || !swa_scale_ok(scale)) return UA_ERR_UNSUPPORTED;
  return UA_OK;
}
template <class T, int kD, bool kTree>
static void paged_launch(const PagedParams& p, const PagedShape& s, unsigned n, hipStream_t st) {
  if (s.many)            paged_many_kernel<T, kD, kTree><<<n, 256, 0, st>>>(p);
  else if (s.tiles == 1) paged_few_kernel<T, kD, 1, kTree><<<n, 64 * kPagedWaves, 0, st>>>(p);
  else                   paged_few_kernel<T, kD, 2, kTree><<<n, 64 * kPagedWaves, 0, st>>>(p);
}

}  // namespace ua

extern "C" int64_t ua_paged_decode_workspace_bytes(int batch, int n_tokens, int n_heads, int n_kv_heads, int page, int max_pages, int head_dim, int64_t left,
                                                   int64_t sinks) {
  using namespace ua;
  if (paged_decode_check(batch, n_tokens, n_heads, n_kv_heads, 1, page, max_pages, head_dim, UA_BF16, 0, nullptr, 0, left, sinks, 1.f) != UA_OK) return 0;
  const int parts = paged_shape(batch, n_tokens, n_heads, n_kv_heads, paged_room(page, max_pages), head_dim, left, sinks).parts;
  const int64_t rows = (int64_t)batch * n_tokens * n_heads;
  return parts > 1 ? parts * (align256(rows * head_dim * 4) + align256(rows * 4)) : 0;
}

extern "C" int ua_paged_decode(const void* q, const void* k_pages, const void* v_pages, void* o, float* lse, const int32_t* table, const int32_t* lens,
                               const int32_t* n_new, const int32_t* parents, int batch, int n_tokens, int n_heads, int n_kv_heads, int n_pages, int page,
                               int max_pages, int head_dim, int dtype, int64_t table_stride, int64_t parents_stride, const int64_t* q_strides,
                               const int64_t* k_page_strides, const int64_t* v_page_strides, const int64_t* o_strides, int64_t left, int64_t sinks,
                               float softmax_scale, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace ua;
  int rc = paged_decode_check(batch, n_tokens, n_heads, n_kv_heads, n_pages, page, max_pages, head_dim, dtype, table_stride, parents, parents_stride, left,
                              sinks, softmax_scale);
  if (rc != UA_OK) return rc;
  if ((int64_t)batch * n_tokens == 0) return UA_OK;
  const bool none = n_pages == 0 || max_pages == 0;        // (the pools and the table may be NULL)
  if (!q || !o || !lse || !lens || !q_strides || !k_page_strides || !v_page_strides || !o_strides || (!none && (!k_pages || !v_pages || !table)))
    return UA_ERR_NULL;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(o) || !aligned4(table) || !aligned4(lens) || !aligned4(n_new) ||
      !aligned4(parents) || !swa_strides_ok(q_strides, false) || !swa_strides_ok(k_page_strides, false) || !swa_strides_ok(v_page_strides, false) ||
      !swa_strides_ok(o_strides, true))
    return UA_ERR_ALIGN;
  rc = check_device();
  if (rc != UA_OK) return rc;
  PagedParams p{};
  p.pages = {table, table_stride, n_pages, page, none ? 0 : paged_room(page, max_pages), make_div(page)};
  const PagedShape s = paged_shape(batch, n_tokens, n_heads, n_kv_heads, paged_room(page, max_pages), head_dim, left, sinks);
  p.q = q; p.o = o; p.lse = lse;
  p.k = {(const char*)k_pages, 2 * k_page_strides[0], 2 * k_page_strides[1], 2 * k_page_strides[2]};
  p.v = {(const char*)v_pages, 2 * v_page_strides[0], 2 * v_page_strides[1], 2 * v_page_strides[2]};
  p.steps = {lens, n_new, parents, parents_stride, n_tokens};
  p.qs = {q_strides[0], q_strides[1], q_strides[2]};
  p.os = {o_strides[0], o_strides[1], o_strides[2]};
  p.n_heads = n_heads; p.n_kv_heads = n_kv_heads; p.group = n_heads / n_kv_heads;
  p.left = left < 0 ? kFar : (int)std::min<int64_t>(left, kFar);
  p.sinks = left < 0 ? 0 : (int)std::min<int64_t>(sinks, kFar);
  p.rows = n_tokens * p.group;
  p.n_tiles = s.row_tiles;
  p.least = s.least;
  p.scale_log2 = softmax_scale * kLog2e;
  p.n_parts = 1;
  const int64_t rows = (int64_t)batch * n_tokens * n_heads, o_bytes = align256(rows * head_dim * 4), lse_bytes = align256(rows * 4);
  if (s.parts > 1 && workspace && aligned16(workspace) && workspace_bytes >= s.parts * (o_bytes + lse_bytes)) {
    p.n_parts = s.parts;
    p.part_o = (float*)workspace;
    p.part_lse = (float*)((char*)workspace + s.parts * o_bytes);
    p.o_part = o_bytes / 4;
    p.lse_part = lse_bytes / 4;
  }
  p.by_kv_heads = make_div(n_kv_heads);
  p.by_group = make_div(p.group);
  p.by_tiles = make_div(p.n_tiles);
  p.by_walks = make_div(p.n_parts * n_kv_heads);
  const hipStream_t st = (hipStream_t)stream;
  const int64_t n = (int64_t)batch * n_kv_heads * p.n_tiles * p.n_parts;
  if (n > kSwaMaxGroups) return UA_ERR_SHAPE;
  p.batch = batch;
  p.n_groups = (int)n;
  p.sorted = batch > 1 && batch <= 64 && n > kCus;
  p.eight_shift = n / p.n_tiles % 8 ? 0 : 3;
  auto by_tree = [&](auto element, auto dim) {
    typedef decltype(element) T;
    constexpr int kD = decltype(dim)::value;
    if (parents) paged_launch<T, kD, true>(p, s, (unsigned)n, st); else paged_launch<T, kD, false>(p, s, (unsigned)n, st);
  };
  auto by_dim = [&](auto element) {
    if (head_dim == 64) by_tree(element, std::integral_constant<int, 64>{}); else by_tree(element, std::integral_constant<int, 128>{});
  };
  if (dtype == UA_FP16) by_dim(fp16(0)); else by_dim(bf16(0.f));
  if (hipGetLastError() != hipSuccess) return UA_ERR_LAUNCH;
  if (p.n_parts == 1) return UA_OK;
  if (rows <= kJoinRows && p.n_parts > 4) {
    auto join = [&](auto element, auto dim) {
      paged_join_kernel<decltype(element), decltype(dim)::value><<<(unsigned)rows, 256, 0, st>>>(p, make_div(n_heads), make_div(n_tokens));
    };
    auto join_dim = [&](auto element) {
      if (head_dim == 64) join(element, std::integral_constant<int, 64>{}); else join(element, std::integral_constant<int, 128>{});
    };
    if (dtype == UA_FP16) join_dim(fp16(0)); else join_dim(bf16(0.f));
    return hipGetLastError() == hipSuccess ? UA_OK : UA_ERR_LAUNCH;
  }
  return swa_merge(p.part_o, p.o_part, p.part_lse, p.lse_part, p.n_parts, o, p.os, lse, batch, n_heads, n_tokens, head_dim, dtype, st);
}
