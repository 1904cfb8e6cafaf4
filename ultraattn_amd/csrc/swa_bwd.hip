// Sliding-window attention with sinks, backward: P is made again from the rows' LSE, nothing is added atomically.
//
//   columns: a workgroup (4 waves of 32 keys) per (128 keys, key head) holds K and V and walks the blocks of 64 query rows that see
//            it, of all query heads that share it:  S = Q K^T, dP = dO V^T - delta, dV^T += dO^T P, dK^T += Q^T dS;
//   rows:    a workgroup per (128 queries, head) holds Q and dO and walks the blocks of 64 keys (SwaWalk):
//            S^T = K Q^T, dP^T = V dO^T - delta, dQ^T += K^T dS^T.
// P = exp2(scale log2(e) S - log2(e) LSE), dS = P dP; dK and dQ are multiplied by the scale at their end.  In the accumulators a lane holds
// one key (query), so that P and dS, rounded, are operands of the next products.  Both sides are one launch: neither leaves the device partly
// empty at its end.
//
// P and dS are rounded to the operands' type for the products that sum them, as P is in the forward; everything else stays in fp32.
//
// A column of the sinks is seen by every later query: its walk is cut into parts of about the others' length, which leave fp32 dK and
// dV that a last launch adds in their order.  So are all walks where there are few of them.
#include <algorithm>
#include <cmath>
#include "swa.h"

namespace ua {

// P <= 1 in fp16 is below its normal range from 6e-5 on, where long rows are: it is held times 2^14, dV is divided by that.  So is dS = P (dP - delta):
// times 2^(14 - k), where a wave's k begins at 4 and grows with the largest |dP - delta| that it meets, below 2^(k + 1); the gradient summed so far shrinks by as
// much and is multiplied by 2^(k - 14) at its end.  So dS down to 2^-29 of the largest dP - delta has all bits, whatever the size of dO.  (bf16 has
// fp32's range.)  It costs 2 of 66 us (2 x 10 heads of 64, 1333 x 2048), 3 of 185 (16 of 128, 4096): the largest
// one is known late.  Found beside dV's products, which then come before dK's, it cost no less, and registers.
template <class T> constexpr int kSwaBits = 0;
template <> constexpr int kSwaBits<fp16> = 14;
template <class T> constexpr int kSwaFirst = kSwaBits<T> ? 4 : 0;
__device__ __forceinline__ float power2(int n) { return __int_as_float((127 + n) << 23); }
// How much k has to grow by, seldom anything, with the gradient so far.  (Infinities stay; they say nothing of the others.  2^60 is beyond any other.)
template <int kN>
__device__ __forceinline__ int swa_grow(const f32x16& dp, int k, f32x16 (&acc)[kN]) {
  float half[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 16; i += 2) half[i >> 1 & 1] = fmaxf(fmaxf(half[i >> 1 & 1], fabsf(dp[i])), fabsf(dp[i + 1]));
  const float most = fmaxf(half[0], half[1]);
  if (__builtin_amdgcn_ballot_w64(most >= power2(1 + k)) == 0) return 0;
  int more = 0;
  while (k + more < 60 && __builtin_amdgcn_ballot_w64(most >= power2(1 + k + more) && most < INFINITY) != 0) more += 2;
#pragma unroll
  for (int m = 0; m < kN; ++m)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[m][i] *= power2(-more);
  return more;
}

template <int kD> using BwdStream = SwaStream<kD, kB, kB>;
template <int kD> struct BwdLds {
  static constexpr int kStage = BwdStream<kD>::kBytes, kStat = 2 * kStage, kStatBytes = 2 * kSwaBlock * 4, kBytes = kStat + 2 * kStatBytes;
};
// Addresses, within a stage, of 128-bit reads of 32 rows and of transposing reads.
template <class T, int kD>
struct BwdAddr {
  using H = SwaHead<kD>;
  typedef typename SwaVec<T>::x8 x8;
  static constexpr int kNat = 4, kTr = 4;
  uint32_t nat[kNat], tr[kTr];
  __device__ __forceinline__ explicit BwdAddr(uint32_t lds) {
    const int lane = fresh_lane();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (of 128 columns the chunks 2 i and 2 i + 1 of 16 lie 32 bytes apart; so do rows 8 apart, at a constant)
      nat[i] = lds + H::at_b(lane & 31, (kD == 128 ? 4 : 2) * i + (lane >> 5));
      tr[i] = lds + (kD == 128 ? H::tr_offset_b(lane, i, 0) : H::tr_offset_b(lane, i >> 1, i & 1));
      asm volatile("" : "+v"(nat[i]), "+v"(tr[i]));
    }
  }
  static constexpr int kRows32 = 32 / H::kCopyRows * H::kPitchB, kRows16 = kRows32 / 2, kRows8 = kRows32 / 4;
  template <int kOff> __device__ __forceinline__ x8 row(int i) const {                 // columns 16 i ..
    return lds_get<x8>(kD == 128 ? nat[i >> 1] + (kOff + 32 * (i & 1)) : nat[i] + kOff);
  }
  template <int kOff> __device__ __forceinline__ x8 column(int i) const {              // columns 32 (i % kBlocks), 16 rows from 16 (i / kBlocks) on
    constexpr int kB = H::kBlocks;
    const int rows = kOff + kRows16 * (i / kB);
    return kD == 128 ? lds_tr_pair<T>(tr[i % kB] + rows, tr[i % kB] + (rows + kRows8)) : lds_tr_pair<T>(tr[2 * (i % kB)] + rows, tr[2 * (i % kB) + 1] + rows);
  }
};

// The kernel's parameters read again from the kernel-argument segment: each walk's behind the branch that leads to it, and its end's behind the
// walk.  All at once ask for more scalar registers than there are, and live in vector lanes then.
__device__ __forceinline__ const SwaParams& params_again() {
  typedef const __attribute__((address_space(4))) SwaParams* Late;
  Late p = (Late)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const SwaParams*)p;
}

// ---- columns ------------------------------------------------------------------------------------------------------
// 32 query rows at kOff of a stage, their statistics at `stat`.  first, seen: the rows row0 + quad that a lane's key is visible to, if `mask`.
template <class T, int kD, int kOff, int kCopies, class Copy>
__device__ __forceinline__ void dkdv_rows(const BwdAddr<T, kD>& ad, uint32_t stat, const typename SwaVec<T>::x8 (&kf)[kD / 16],
                                          const typename SwaVec<T>::x8 (&vf)[kD / 16], f32x16 (&dk)[kD / 32], f32x16 (&dv)[kD / 32], float scale_log2,
                                          int& ds_k, bool mask, int row0, int first, uint32_t seen, Copy copy) {
  using V = SwaVec<T>;
  using H = SwaHead<kD>;
  typedef typename V::x8 x8;
  constexpr int kY = BwdStream<kD>::kSecond;
  f32x16 s, dp;
  const uint32_t mine = stat + 16 * (fresh_lane() >> 5);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 a = lds_get<f32x4>(mine + 32 * g), c = lds_get<f32x4>(mine + kSwaBlock * 4 + 32 * g);
#pragma unroll
    for (int j = 0; j < 4; ++j) { s[4 * g + j] = a[j]; dp[4 * g + j] = c[j]; }
  }
  __builtin_amdgcn_sched_barrier(0);
  {
    constexpr int kAhead = 2, kAll = 2 * H::kSteps;
    x8 fr[kAll];
    auto rd = [&](int i) { return (i & 1) ? ad.template row<kOff + kY>(i >> 1) : ad.template row<kOff>(i >> 1); };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fr[i] = rd(i);
    __builtin_amdgcn_sched_group_barrier(0x100, 8 + kAhead, 0);
#pragma unroll
    for (int i = 0; i < kAll; ++i) {
      if (i + kAhead < kAll) fr[i + kAhead] = rd(i + kAhead);
      if (i & 1) dp = V::mfma(fr[i], vf[i >> 1], dp);
      else       s = V::mfma(fr[i], kf[i >> 1], s);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      if ((i + 1) * kCopies / kAll != i * kCopies / kAll) copy(i * kCopies / kAll);
    }
  }
  constexpr int kTAhead = 2, kTAll = 4 * H::kBlocks;
  auto rd_tr = [&](int i) { return (i & 1) ? ad.template column<kOff>(i >> 1) : ad.template column<kOff + kY>(i >> 1); };
  x8 ft[kTAll];
#pragma unroll
  for (int i = 0; i < kTAhead; ++i) ft[i] = rd_tr(i);
  if (mask) {
    const int row = row0 + 4 * (fresh_lane() >> 5) - first;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if ((uint32_t)(row + 8 * (i >> 2) + (i & 3)) >= seen) { s[i] = -INFINITY; dp[i] = 0.f; }      // (dp: NaN of a row not seen stays out)
  }
  if constexpr (kSwaBits<T> != 0) ds_k += swa_grow(dp, ds_k, dk);
  x8 pb[2], dsb[2];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float e = fast_exp2(kSwaBits<T> ? fmaf(s[i], scale_log2, kSwaBits<T>) : s[i] * scale_log2);
    pb[i >> 3][i & 7] = (T)e;
    dsb[i >> 3][i & 7] = (T)(kSwaBits<T> ? e * dp[i] * power2(-ds_k) : e * dp[i]);
  }
#pragma unroll
  for (int i = 0; i < kTAll; ++i) {
    if (i + kTAhead < kTAll) ft[i + kTAhead] = rd_tr(i + kTAhead);
    const int n = i >> 1, m = n % H::kBlocks, t = n / H::kBlocks;
    if (i & 1) dk[m] = V::mfma(ft[i], dsb[t], dk[m]);
    else       dv[m] = V::mfma(ft[i], pb[t], dv[m]);
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
  }
}

template <class T, int kD>
__device__ __forceinline__ void columns_walk(uint32_t lds, int block) {
  const SwaParams& p = params_again();
  using H = SwaHead<kD>;
  using L = BwdLds<kD>;
  typedef typename SwaVec<T>::x8 x8;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int run = block < p.cols[0].n_blocks ? 0 : 1;
  const SwaColumns& c = p.cols[run];
  int pos, bh;
  map_block(block - (run ? p.cols[0].n_blocks : 0), c.map, pos, bh);
  const int tile = quotient(pos, c.by_parts), part = pos - tile * c.n_parts, kt = c.first + tile;
  const int b = quotient(bh, p.by_kv_heads), hk = bh - b * p.n_kv_heads, k0 = kt * kSwaRows;
  const SwaColumn col(k0, min(k0 + kSwaRows, p.seq_k) - 1, p.hi, p.lo, p.sinks, p.seq_q);
  const int total = col.n * p.group, part_len = (total + c.n_parts - 1) / c.n_parts;
  const int i0 = min(part * part_len, total), i1 = min(i0 + part_len, total);

  // a step's place: query head (of the group) and block of 64 rows
  int g = __builtin_amdgcn_readfirstlane(col.n ? i0 / col.n : 0), at = i0 - g * col.n;
  BwdStream<kD> in(p.qs.s, p.ds.s, wave, lane);
  auto base = [&](int head) {
    const int h = hk * p.group + head;
    in.of((const T*)p.q + b * p.qs.b + h * p.qs.h, (const T*)p.dout + b * p.ds.b + h * p.ds.h);
  };
  // -lse / scale (rows that see nothing, and rows that are not there: -inf, so that P = 0) and -delta, from which S and dP start; two waves bring either
  auto load_stat = [&](int head, int row0) {
    const int row = row0 + 32 * (wave & 1) + (fresh_lane() & 31);
    const float* rows = (wave >= 2 ? p.delta : p.lse) + ((int64_t)b * p.n_heads + hk * p.group + head) * p.seq_q;
    return row < p.seq_q ? rows[row] : wave >= 2 ? 0.f : -INFINITY;
  };
  const float scale_log2 = p.scale_log2;
  auto put_stat = [&](int stage, float x) {
    const float y = wave >= 2 ? -x : x == -INFINITY ? x : x * (-kLog2e / scale_log2);
    lds_put(lds + L::kStat + stage * L::kStatBytes + 128 * wave + 4 * (fresh_lane() & 31), y);
  };
  float stat = 0.f;
  if (i0 < i1) {
    base(g);
    in.block((col.first + at) * kSwaBlock, col.end, true);
#pragma unroll
    for (int n = 0; n < in.kPieces; ++n) in.copy(n, lds);
    stat = load_stat(g, (col.first + at) * kSwaBlock);
  }
  const int key0 = k0 + 32 * wave, from = min(key0, p.seq_k - 1);
  x8 kf[H::kSteps], vf[H::kSteps];
  {
    u32x4 kraw[H::kSteps], vraw[H::kSteps];
    swa_load_rows<kD>(kraw, (const T*)p.k + b * p.ks.b + from * p.ks.s + hk * p.ks.h, p.ks.s, p.seq_k - from);
    swa_load_rows<kD>(vraw, (const T*)p.v + b * p.vs.b + from * p.vs.s + hk * p.vs.h, p.vs.s, p.seq_k - from);
    const uint32_t turn = lds + L::kStage + wave * 32 * H::kRow;       // the stage that the first step fills
    swa_put_rows<kD>(kraw, turn);
    swa_frags<T, kD>(kf, turn);
    swa_put_rows<kD>(vraw, turn);
    swa_frags<T, kD>(vf, turn);
  }
  f32x16 dk[H::kBlocks], dv[H::kBlocks];
#pragma unroll
  for (int m = 0; m < H::kBlocks; ++m) { dk[m] = f32x16{0}; dv[m] = f32x16{0}; }
  int ds_k = kSwaFirst<T>;
  const BwdAddr<T, kD> ad(lds);
  if (i0 < i1) put_stat(0, stat);
#pragma unroll
  for (int i = 0; i < H::kSteps; ++i) asm volatile("" : "+v"(kf[i]), "+v"(vf[i]));      // arrived before the walk
  // the rows that this lane's key is visible to: first .. first + seen - 1
  const int key = key0 + (lane & 31);
  wait_vmem_all();
  __syncthreads();

  auto step = [&](int i, auto stage_tag) {
    constexpr int kStage = decltype(stage_tag)::value;
    const int row0 = (col.first + at) * kSwaBlock;
    if (++at == col.n) { at = 0; base(++g < p.group ? g : 0); }
    const int next0 = (col.first + at) * kSwaBlock;
    in.block(next0, col.end, i + 1 < i1);
    if (i + 1 < i1) stat = load_stat(g, next0);
    if (row0 < col.start) lds_clear_rows<kD, H::kPitchB, BwdStream<kD>::kSecond>(lds + kStage * L::kStage, 0, col.start - row0);
    const uint32_t other = lds + (kStage ^ 1) * L::kStage;
    auto rows = [&](auto mb_tag) {
      constexpr int kMb = decltype(mb_tag)::value, kCopies = BwdStream<kD>::kPieces / 2;
      const int r0 = row0 + 32 * kMb;
      auto copy = [&](int n) { in.copy(kMb * kCopies + n, other); };
      // beyond the rows, before what they see, or behind it and no sink
      int hidden = __builtin_amdgcn_readfirstlane(max(max(r0 - p.seq_q + 1, key0 - r0 - 31 - p.hi), min(r0 + p.lo - key0 - 31, key0 - p.sinks + 1)));
      if (hidden > 0)
#pragma unroll
        for (int n = 0; n < kCopies; ++n) copy(n);
      asm volatile("" : "+s"(hidden));       // (as two sides of one branch the products do not stay in the same registers)
      if (hidden > 0) return;
      const bool whole = key0 + 31 <= r0 + p.hi && (key0 >= r0 + 31 + p.lo || key0 + 31 < p.sinks);
      int first = 0;
      uint32_t seen = 0;
      if (!whole) {
        first = key - p.hi;
        const int last = min(key < p.sinks ? kFar : key - p.lo, col.end - 1);      // (a row that is not there: 0 times NaN of the key)
        seen = last >= first ? (uint32_t)last - (uint32_t)first + 1u : 0u;
      }
      dkdv_rows<T, kD, kStage * L::kStage + kMb * BwdAddr<T, kD>::kRows32, kCopies>(
          ad, lds + L::kStat + kStage * L::kStatBytes + kMb * 128, kf, vf, dk, dv, scale_log2, ds_k, !whole, r0, first, seen, copy);
    };
    rows(std::integral_constant<int, 0>{});
    rows(std::integral_constant<int, 1>{});
    wait_vmem_all();
    if (i + 1 < i1) put_stat(kStage ^ 1, stat);
    __syncthreads();                        // the next block has landed, and everyone has left this one
  };
  for (int i = i0; i < i1; i += 2) {
    step(i, std::integral_constant<int, 0>{});
    if (i + 1 < i1) step(i + 1, std::integral_constant<int, 1>{});
  }
  const SwaParams& e = params_again();
  const int n_rows = e.seq_k - key0;
  if (n_rows <= 0) return;
  const SwaColumns& ec = e.cols[run];
  const float dk_scale = e.scale * power2(ds_k - kSwaBits<T>);
  if (ec.n_parts > 1) {
    const int64_t row = part * ec.part + ((int64_t)bh * ec.tiles * kSwaRows + key0 - ec.first * kSwaRows) * kD;
    swa_store_f32<kD>(ec.dk + row, kD, n_rows, dk, dk_scale);
    swa_store_f32<kD>(ec.dv + row, kD, n_rows, dv, power2(-kSwaBits<T>));
  } else {
    const uint32_t turn = lds + wave * 32 * H::kRow;
    swa_store_rows<T, kD>((T*)e.dk + b * e.dks.b + (int64_t)key0 * e.dks.s + hk * e.dks.h, e.dks.s, n_rows, dk, dk_scale, turn);
    swa_store_rows<T, kD>((T*)e.dv + b * e.dvs.b + (int64_t)key0 * e.dvs.s + hk * e.dvs.h, e.dvs.s, n_rows, dv, power2(-kSwaBits<T>), turn);
  }
}

// ---- rows ---------------------------------------------------------------------------------------------------------
template <class T, int kD, int kOff, int kCopies, class Copy>
__device__ __forceinline__ void dq_keys(const BwdAddr<T, kD>& ad, const typename SwaVec<T>::x8 (&qf)[kD / 16], const typename SwaVec<T>::x8 (&dof)[kD / 16],
                                        const f32x16& neg_delta, f32x16 (&dq)[kD / 32], float scale_log2, float& lse2, int& ds_k, bool mask, int key0, int first,
                                        uint32_t seen, int sinks, Copy copy) {
  using V = SwaVec<T>;
  using H = SwaHead<kD>;
  typedef typename V::x8 x8;
  constexpr int kY = BwdStream<kD>::kSecond;
  f32x16 s, dp;
  {
    constexpr int kAhead = 4, kAll = 2 * H::kSteps;
    x8 fr[kAll];
    auto rd = [&](int i) { return (i & 1) ? ad.template row<kOff + kY>(i >> 1) : ad.template row<kOff>(i >> 1); };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fr[i] = rd(i);
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
    for (int i = 0; i < kAll; ++i) {
      if (i + kAhead < kAll) fr[i + kAhead] = rd(i + kAhead);
      if (i & 1) dp = V::mfma(fr[i], dof[i >> 1], i == 1 ? neg_delta : dp);
      else       s = V::mfma(fr[i], qf[i >> 1], i == 0 ? f32x16{0} : s);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      if ((i + 1) * kCopies / kAll != i * kCopies / kAll) copy(i * kCopies / kAll);
    }
  }
  constexpr int kTAhead = 3, kTAll = 2 * H::kBlocks;
  x8 ft[kTAll];
#pragma unroll
  for (int i = 0; i < kTAhead; ++i) ft[i] = ad.template column<kOff>(i);
  if (mask) {
    const int key = key0 + 4 * (fresh_lane() >> 5);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int k = key + 8 * (i >> 2) + (i & 3);
      if ((uint32_t)(k - first) >= seen && k >= sinks) { s[i] = -INFINITY; dp[i] = 0.f; }
    }
  }
  if constexpr (kSwaBits<T> != 0) {
    const int more = swa_grow(dp, ds_k, dq);
    ds_k += more;
    lse2 += more;                           // 2^(14 - k) is in the exponent
  }
  x8 dsb[2];
#pragma unroll
  for (int i = 0; i < 16; ++i) dsb[i >> 3][i & 7] = (T)(fast_exp2(fmaf(s[i], scale_log2, -lse2)) * dp[i]);
#pragma unroll
  for (int i = 0; i < kTAll; ++i) {
    if (i + kTAhead < kTAll) ft[i + kTAhead] = ad.template column<kOff>(i + kTAhead);
    dq[i % H::kBlocks] = V::mfma(ft[i], dsb[i / H::kBlocks], dq[i % H::kBlocks]);
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
  }
}

template <class T, int kD>
__device__ __forceinline__ void rows_walk(uint32_t lds, int block) {
  const SwaParams& p = params_again();
  using H = SwaHead<kD>;
  using L = BwdLds<kD>;
  typedef typename SwaVec<T>::x8 x8;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int pos, bh;
  map_block(block, p.map, pos, bh);
  const int line = quotient(pos, p.by_parts), part = pos - line * p.n_parts, qt = p.n_qtiles - 1 - line;
  const int b = quotient(bh, p.by_heads), h = bh - b * p.n_heads, hk = quotient(h, p.by_group);
  const int r0 = qt * kSwaRows, row0 = r0 + 32 * wave, n_rows = p.seq_q - row0;
  const SwaWalk walk(r0, min(r0 + kSwaRows, p.seq_q) - 1, p.hi, p.lo, p.sinks, p.seq_k);
  const int part_len = (walk.n + p.n_parts - 1) / p.n_parts, i0 = min(part * part_len, walk.n), i1 = min(i0 + part_len, walk.n);
  BwdStream<kD> in(p.ks.s, p.vs.s, wave, lane);
  in.of((const T*)p.k + b * p.ks.b + hk * p.ks.h, (const T*)p.v + b * p.vs.b + hk * p.vs.h);
  if (i0 < i1) {
    in.block(walk.at(i0) * kSwaBlock, walk.end_of(walk.at(i0)), true);
#pragma unroll
    for (int n = 0; n < in.kPieces; ++n) in.copy(n, lds);
  }
  const int from = min(row0, p.seq_q - 1);
  x8 qf[H::kSteps], dof[H::kSteps];
  float lse_raw, neg_delta;
  {
    u32x4 qraw[H::kSteps], doraw[H::kSteps];
    swa_load_rows<kD>(qraw, (const T*)p.q + b * p.qs.b + from * p.qs.s + h * p.qs.h, p.qs.s, p.seq_q - from);
    swa_load_rows<kD>(doraw, (const T*)p.dout + b * p.ds.b + from * p.ds.s + h * p.ds.h, p.ds.s, p.seq_q - from);
    const int64_t row = (int64_t)bh * p.seq_q + min(row0 + (lane & 31), p.seq_q - 1);
    lse_raw = p.lse[row];
    neg_delta = -p.delta[row];
    const uint32_t turn = lds + L::kStage + wave * 32 * H::kRow;
    swa_put_rows<kD>(qraw, turn);
    swa_frags<T, kD>(qf, turn);
    swa_put_rows<kD>(doraw, turn);
    swa_frags<T, kD>(dof, turn);
  }
  float lse2 = lse_raw == -INFINITY ? INFINITY : lse_raw * kLog2e - (kSwaBits<T> - kSwaFirst<T>);        // (P = 0 in rows that see nothing)
  int ds_k = kSwaFirst<T>;
  f32x16 nd, dq[H::kBlocks];
#pragma unroll
  for (int i = 0; i < 16; ++i) nd[i] = neg_delta;
  asm volatile("" : "+v"(nd));              // registers, not one value moved into an accumulator again and again
#pragma unroll
  for (int m = 0; m < H::kBlocks; ++m) dq[m] = f32x16{0};
  const BwdAddr<T, kD> ad(lds);
#pragma unroll
  for (int i = 0; i < H::kSteps; ++i) asm volatile("" : "+v"(qf[i]), "+v"(dof[i]));

  auto step = [&](int i, auto stage_tag) {
    constexpr int kStage = decltype(stage_tag)::value;
    const int block0 = walk.at(i) * kSwaBlock;
    in.block(walk.at(i + 1) * kSwaBlock, walk.end_of(walk.at(i + 1)), i + 1 < i1);
    wait_vmem_all();
    __syncthreads();                        // this block has landed, and everyone has left the other stage
    if (block0 < walk.start && block0 + kSwaBlock > walk.start)
      lds_clear_rows<kD, H::kPitchB>(lds + kStage * L::kStage, max(p.sinks - block0, 0), walk.start - block0);
    const uint32_t other = lds + (kStage ^ 1) * L::kStage;
    auto keys = [&](auto mb_tag) {
      constexpr int kMb = decltype(mb_tag)::value, kCopies = BwdStream<kD>::kPieces / 2;
      const int key0 = block0 + 32 * kMb;
      auto copy = [&](int n) { in.copy(kMb * kCopies + n, other); };
      int hidden = __builtin_amdgcn_readfirstlane(max(max(key0 - p.seq_k + 1, key0 - row0 - 31 - p.hi), min(row0 + p.lo - key0 - 31, key0 - p.sinks + 1)));
      if (hidden > 0)
#pragma unroll
        for (int n = 0; n < kCopies; ++n) copy(n);
      asm volatile("" : "+s"(hidden));       // (see columns_walk)
      if (hidden > 0) return;
      const bool whole = key0 + 31 <= min(row0 + p.hi, p.seq_k - 1) && (key0 >= row0 + 31 + p.lo || key0 + 31 < p.sinks);
      int first = 0, sinks = 0;
      uint32_t seen = 0;
      if (!whole) {
        const int row = row0 + (fresh_lane() & 31), last = min(row + p.hi, p.seq_k - 1);
        first = row + p.lo;
        seen = (uint32_t)max(last - first + 1, 0);
        sinks = min(p.sinks, last + 1);
      }
      dq_keys<T, kD, kStage * L::kStage + kMb * BwdAddr<T, kD>::kRows32, kCopies>(ad, qf, dof, nd, dq, p.scale_log2, lse2, ds_k, !whole, key0, first, seen, sinks,
                                                                                  copy);
    };
    keys(std::integral_constant<int, 0>{});
    keys(std::integral_constant<int, 1>{});
  };
  for (int i = i0; i < i1; i += 2) {
    step(i, std::integral_constant<int, 0>{});
    if (i + 1 < i1) step(i + 1, std::integral_constant<int, 1>{});
  }
  wait_vmem_all();                          // the last step's copies filled a stage with zeros
  __syncthreads();
  if (n_rows <= 0) return;
  const SwaParams& e = params_again();
  const float dq_scale = e.scale * power2(ds_k - kSwaBits<T>);
  if (e.n_parts > 1)
    swa_store_f32<kD>(e.part_o + part * e.o_part + ((int64_t)bh * e.seq_q + row0) * kD, kD, n_rows, dq, dq_scale);
  else
    swa_store_rows<T, kD>((T*)e.dq + b * e.dqs.b + (int64_t)row0 * e.dqs.s + h * e.dqs.h, e.dqs.s, n_rows, dq, dq_scale, lds + wave * 32 * H::kRow);
}

template <class T, int kD>
__global__ __launch_bounds__(256, 2) void swa_bwd_kernel(const SwaParams p) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[BwdLds<kD>::kBytes];
  const uint32_t lds = (uint32_t)(uintptr_t)(lds_byte*)smem;
  if ((int)blockIdx.x < p.n_col_blocks) columns_walk<T, kD>(lds, blockIdx.x);
  else                                  rows_walk<T, kD>(lds, blockIdx.x - p.n_col_blocks);
}

// delta = rowsum(dO * O).  16 tokens of 4 heads a workgroup: memory sees rows of 4 heads, and 64 bytes of each head's result.
//
// O was rounded by half a step, u.  In a row of n keys that moves delta by about u |dO| / sqrt(n), while dP - delta is about |dO|: for
// few keys as much as the rounding of dS, and such rows have the largest gradients (1333 queries that run out of their keys, fp16: dQ off by
// 3.1e-4, 3.0e-4 without it).  So rows of up to kFewKeys keys make their O again, unrounded, if their LSE is that of these keys alone (of a shard it
// is not).  All keys' loads are in flight at once, and a thread has one row: such rows one after the other, in four iterations of four keys, took 15 us.
constexpr int kFewKeys = 8;
// The sum over the 8 or 16 lanes of a row, in each of them.
template <int kLanes>
__device__ __forceinline__ float row_sum(float x) {
  auto from = [](float y, auto ctrl) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(y), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  x += from(x, std::integral_constant<int, 0xb1>{});         // neighbours
  x += from(x, std::integral_constant<int, 0x4e>{});         // pairs
  x += from(x, std::integral_constant<int, 0x141>{});        // mirrored in 8 lanes
  if (kLanes == 16) x += from(x, std::integral_constant<int, 0x140>{});        // in 16
  return x;
}
template <class T, int kD>
__global__ __launch_bounds__(8 * kD) void swa_delta_kernel(const SwaParams p) {
  constexpr int kLanes = kD / 8;
  typedef typename SwaVec<T>::x8 x8;
  __shared__ float sums[16][4];
  const int th = quotient(blockIdx.x, p.by_kv_heads), hb = blockIdx.x - th * p.by_kv_heads.d, b = quotient(th, p.by_parts), t0 = (th - b * p.by_parts.d) * 16, h0 = 4 * hb;
  const int lane = threadIdx.x % kLanes, r = threadIdx.x / kLanes, t = min(t0 + r / 4, p.seq_q - 1), h = min(h0 + r % 4, p.n_heads - 1);
  const x8 x = *reinterpret_cast<const x8*>((const T*)p.o + b * p.os.b + t * p.os.s + h * p.os.h + 8 * lane);
  const x8 y = *reinterpret_cast<const x8*>((const T*)p.dout + b * p.ds.b + t * p.ds.s + h * p.ds.h + 8 * lane);
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) sum = fmaf((float)x[j], (float)y[j], sum);
  sum = row_sum<kLanes>(sum);
  const int last = min(t + p.hi, p.seq_k - 1), first = max(t + p.lo, 0), sinks = max(min(min(p.sinks, last + 1), first), 0);
  const int n = max(last - first + 1, 0) + sinks;
  if (n > 0 && n <= kFewKeys) {                            // the same for all lanes of a row
    const int hk = quotient(h, p.by_group);
    const T* k = (const T*)p.k + b * p.ks.b + hk * p.ks.h + 8 * lane;
    const T* v = (const T*)p.v + b * p.vs.b + hk * p.vs.h + 8 * lane;
    x8 kr[kFewKeys], vr[kFewKeys];
#pragma unroll
    for (int m = 0; m < kFewKeys; ++m) {
      const int j = min(m, n - 1);
      const int64_t key = j < sinks ? j : first + j - sinks;
      kr[m] = *reinterpret_cast<const x8*>(k + key * p.ks.s);
      vr[m] = *reinterpret_cast<const x8*>(v + key * p.vs.s);
    }
    const x8 q = *reinterpret_cast<const x8*>((const T*)p.q + b * p.qs.b + t * p.qs.s + h * p.qs.h + 8 * lane);
    const float lse2 = p.lse[((int64_t)b * p.n_heads + h) * p.seq_q + t] * kLog2e;
    float mass = 0.f, again = 0.f;
#pragma unroll
    for (int m = 0; m < kFewKeys; ++m) {
      float s = 0.f, dp = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s = fmaf((float)q[j], (float)kr[m][j], s);
        dp = fmaf((float)y[j], (float)vr[m][j], dp);
      }
      s = row_sum<kLanes>(s);
      dp = row_sum<kLanes>(dp);
      if (m < n) {
        const float e = fast_exp2(fmaf(s, p.scale_log2, -lse2));
        mass += e;
        again = fmaf(e, dp, again);
      }
    }
    if (fabsf(mass - 1.f) < 1.f / 16384.f) sum = again;
  }
  if (lane == 0) sums[r / 4][r % 4] = sum;
  __syncthreads();
  if (threadIdx.x < 64) {
    const int ts = t0 + threadIdx.x % 16, hs = h0 + threadIdx.x / 16;
    if (ts < p.seq_q && hs < p.n_heads) p.delta[((int64_t)b * p.n_heads + hs) * p.seq_q + ts] = sums[threadIdx.x % 16][threadIdx.x / 16];
  }
}

// Sums of fp32 parts, part i at parts + i * part, contiguous [batch * heads, tokens, kD], into the first `tokens` rows of a strided result.
struct SwaSum {
  const float* parts; void* out;
  int64_t part;
  Strides3 os;
  int n_parts, tokens, part_tokens, heads, n_rows, n_groups;     // part_tokens: rows of a head in the parts
  Div by_tokens, by_heads;
};
constexpr int kMaxSums = 5;                          // dK and dV of either run of columns, dQ
struct SwaSums { SwaSum s[kMaxSums]; };
template <class T, int kD>
__global__ __launch_bounds__(256) void swa_sum_kernel(const SwaSums all) {
  int block = blockIdx.x, which = 0;
  while (which < kMaxSums - 1 && block >= all.s[which].n_groups) block -= all.s[which++].n_groups;
  const SwaSum& x = all.s[which];
  constexpr int kPer = kD / 16;
  const int row = block * 16 + (threadIdx.x >> 4), c = threadIdx.x & 15;
  if (row >= x.n_rows) return;
  const int bh = quotient(row, x.by_tokens), t = row - bh * x.tokens, b = quotient(bh, x.by_heads), h = bh - b * x.heads;
  const float* from = x.parts + ((int64_t)bh * x.part_tokens + t) * kD + c * kPer;
  float acc[kPer] = {};
  for (int i = 0; i < x.n_parts; ++i)
#pragma unroll
    for (int j = 0; j < kPer; j += 4) {
      const f32x4 y = *reinterpret_cast<const f32x4*>(from + i * x.part + j);
#pragma unroll
      for (int n = 0; n < 4; ++n) acc[j + n] += y[n];
    }
  typedef __attribute__((ext_vector_type(kPer))) T vec;
  vec w;
#pragma unroll
  for (int j = 0; j < kPer; ++j) w[j] = (T)acc[j];
  *reinterpret_cast<vec*>((T*)x.out + b * x.os.b + t * x.os.s + h * x.os.h + c * kPer) = w;
}

// How a backward is cut, and where its parts lie in the workspace (bytes).
struct BwdCut {
  int row_parts, n_sink, col_parts[2];            // n_sink: tiles of the first run of columns
  int64_t dq_bytes, col_bytes[2], total;          // of a part; of a part's dK
};
// Walks are cut to about what a workgroup has on average with two of them on every CU (of heads of 64 as well, of which three fit), `each`, where the time
// that the longest take beyond that is well above what the parts cost: their rows' way through memory and the launch that adds them.  Lengths are counted in
// products of 64 rows (0.8 us where two workgroups share every CU, 0.5 where they hardly do); a column's step has four of them and a row's three.
// us, whole and cut as taken here:
//     128 columns   16 heads, 4096, window 1024, 4 sinks      154   116        64 columns   14 heads on 2, 3000, window 464       102    39
//                   4, 2048 causal                           62.0  44.3                     2, 8192, window 2048, 70 sinks        191    54
//                   32 on 8, 100 x 16384                      380   131                     2 x 10 on 5, 1333 x 2048, window 700  49.5  44.7
//                   8 on 2, 16384, window 4096, 16 sinks     2136   721
// Against a cut of every walk of more than 1.5 each + 24 products, forward and backward in one, both rules in turn, 22 drawn shapes on which they differ (of
// 147): 5 to 20 % faster in fourteen (16 heads on 2 of 64, 1332 and 1924 causal, 65 -> 59 and 91 -> 81; 8 on 2, 956, window 110, 60 -> 48), up to 3 % in three, slower
// in five (4 x 32 on 8, 290 causal, 58 -> 66; 2 x 32 on 4 of 64, 3781, window 234, 139 -> 147).  Slower too where only a little is left beyond `each`, which
// runs on alone faster than is counted here: 8 on 2, 16384, window 4096, 971 -> 981; 16 on 4, 8192, window 2048, 523 -> 529.
static BwdCut bwd_cut(const SwaParams& p, int head_dim, bool cut) {
  BwdCut c{1, 0, {1, 1}, 0, {0, 0}, 0};
  const double cols = (double)p.batch * p.n_kv_heads, rows = (double)p.batch * p.n_heads * p.n_qtiles;
  if (!cut || cols * p.n_ktiles == 0 || rows == 0) return c;
  auto column = [&](int t) { return SwaColumn(t * kSwaRows, imin((t + 1) * kSwaRows, p.seq_k) - 1, p.hi, p.lo, p.sinks, p.seq_q).n * p.group; };
  const int sink_tiles = std::min((p.sinks + kSwaRows - 1) / kSwaRows, p.n_ktiles), other_tiles = p.n_ktiles - sink_tiles;
  const SwaSteps row = swa_row_steps(p), sink = swa_steps(0, sink_tiles, column), col = swa_steps(sink_tiles, other_tiles, column);
  const double work = 3 * rows * row.mean + 4 * cols * (sink_tiles * sink.mean + other_tiles * col.mean);
  const double each = std::max(work / (2 * kCus), 32.0), product_us = each > 64 ? 0.8 : 0.5, row_bytes = head_dim * 4;
  auto parts = [&](double products, double part_bytes) {
    const int n = (int)std::min(std::ceil(products / each), (double)UA_MAX_PARTS);
    const double gain = product_us * (products - std::max(products / n, each)), cost = 6 + 2 * n * part_bytes / 5e6;
    return gain > 1.3 * cost ? n : 1;
  };
  c.row_parts = parts(3.0 * row.most, rows * kSwaRows * row_bytes);
  c.col_parts[0] = parts(4.0 * sink.most, 2 * cols * sink_tiles * kSwaRows * row_bytes);
  c.col_parts[1] = parts(4.0 * col.most, 2 * cols * other_tiles * kSwaRows * row_bytes);
  if (c.col_parts[0] == c.col_parts[1]) c.col_parts[0] = 1;
  else c.n_sink = sink_tiles;
  if (c.row_parts > 1) c.dq_bytes = align256((int64_t)p.batch * p.n_heads * p.seq_q * head_dim * 4);
  const int tiles[2] = {c.n_sink, p.n_ktiles - c.n_sink};
  for (int i = 0; i < 2; ++i) {
    if (c.col_parts[i] > 1) c.col_bytes[i] = align256((int64_t)p.batch * p.n_kv_heads * tiles[i] * kSwaRows * head_dim * 4);
    c.total += 2 * c.col_parts[i] * c.col_bytes[i];
  }
  c.total += c.row_parts * c.dq_bytes;
  return c;
}

template <class T, int kD>
static int bwd_run(const SwaParams& p, unsigned n, const SwaSums& sums, hipStream_t st) {
  if (n) swa_bwd_kernel<T, kD><<<n, 256, 0, st>>>(p);
  if (hipGetLastError() != hipSuccess) return UA_ERR_LAUNCH;
  int groups = 0;
  for (const SwaSum& x : sums.s) groups += x.n_groups;
  if (groups) swa_sum_kernel<T, kD><<<groups, 256, 0, st>>>(sums);
  return hipGetLastError() == hipSuccess ? UA_OK : UA_ERR_LAUNCH;
}
}  // namespace ua

extern "C" int ua_swa_bwd_delta(const void* o, const void* dout, const void* q, const void* k, const void* v, const float* lse, float* delta, int batch,
                                int n_heads, int n_kv_heads, int seqlen_q, int seqlen_k, int head_dim, int dtype, const int64_t* o_strides,
                                const int64_t* do_strides, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides, int64_t q_start,
                                int64_t k_start, int64_t left, int64_t right, int64_t sinks, float softmax_scale, void* stream) {
  using namespace ua;
  SwaParams p{};
  int rc = swa_fill(p, batch, n_heads, n_kv_heads, seqlen_q, seqlen_k, head_dim, dtype, q_start, k_start, left, right, sinks, softmax_scale);
  if (rc != UA_OK) return rc;
  const int64_t tokens = (seqlen_q + 15) / 16, heads = (n_heads + 3) / 4;
  if (batch * tokens * heads > (int64_t)UINT32_MAX / (8 * head_dim)) return UA_ERR_SHAPE;
  if ((int64_t)batch * seqlen_q == 0) return UA_OK;
  if (!o || !dout || !q || !lse || !delta || (seqlen_k > 0 && (!k || !v))) return UA_ERR_NULL;
  for (const int64_t* s : {o_strides, do_strides, q_strides, k_strides, v_strides}) {
    if (!s) return UA_ERR_NULL;
    if (!swa_strides_ok(s, false)) return UA_ERR_ALIGN;
  }
  for (const void* x : {o, dout, q, k, v})
    if (!aligned16(x)) return UA_ERR_ALIGN;
  rc = check_device();
  if (rc != UA_OK) return rc;
  auto three = [](const int64_t* s) { return Strides3{s[0], s[1], s[2]}; };
  p.o = const_cast<void*>(o); p.dout = dout; p.q = q; p.k = k; p.v = v; p.lse = const_cast<float*>(lse); p.delta = delta;
  p.os = three(o_strides); p.ds = three(do_strides); p.qs = three(q_strides); p.ks = three(k_strides); p.vs = three(v_strides);
  p.by_kv_heads = make_div((uint32_t)heads);             // (of this launch: groups of four heads, and of 16 tokens)
  p.by_parts = make_div((uint32_t)tokens);
  const unsigned n = (unsigned)(batch * tokens * heads);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == UA_FP16) {
    if (head_dim == 64) swa_delta_kernel<fp16, 64><<<n, 8 * 64, 0, st>>>(p);
    else                swa_delta_kernel<fp16, 128><<<n, 8 * 128, 0, st>>>(p);
  } else {
    if (head_dim == 64) swa_delta_kernel<bf16, 64><<<n, 8 * 64, 0, st>>>(p);
    else                swa_delta_kernel<bf16, 128><<<n, 8 * 128, 0, st>>>(p);
  }
  return hipGetLastError() == hipSuccess ? UA_OK : UA_ERR_LAUNCH;
}

extern "C" int64_t ua_swa_bwd_workspace_bytes(int batch, int n_heads, int n_kv_heads, int seqlen_q, int seqlen_k, int head_dim, int64_t q_start,
                                              int64_t k_start, int64_t left, int64_t right, int64_t sinks) {
  using namespace ua;
  SwaParams p{};
  if (swa_fill(p, batch, n_heads, n_kv_heads, seqlen_q, seqlen_k, head_dim, UA_BF16, q_start, k_start, left, right, sinks, 1.f) != UA_OK) return 0;
  return bwd_cut(p, head_dim, true).total;
}

extern "C" int ua_swa_bwd(const void* dout, const void* q, const void* k, const void* v, const float* lse, const float* delta, void* dq, void* dk, void* dv,
                          int batch, int n_heads, int n_kv_heads, int seqlen_q, int seqlen_k, int head_dim, int dtype, const int64_t* do_strides,
                          const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides, const int64_t* dq_strides,
                          const int64_t* dk_strides, const int64_t* dv_strides, int64_t q_start, int64_t k_start, int64_t left, int64_t right, int64_t sinks,
                          float softmax_scale, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace ua;
  SwaParams p{};
  int rc = swa_fill(p, batch, n_heads, n_kv_heads, seqlen_q, seqlen_k, head_dim, dtype, q_start, k_start, left, right, sinks, softmax_scale);
  if (rc != UA_OK) return rc;
  const bool some_q = (int64_t)batch * seqlen_q > 0, some_k = (int64_t)batch * seqlen_k > 0;
  if (!some_q && !some_k) return UA_OK;
  for (const int64_t* s : {do_strides, q_strides, k_strides, v_strides, dq_strides, dk_strides, dv_strides})
    if (!s) return UA_ERR_NULL;
  if ((some_q && (!dout || !q || !lse || !delta || !dq)) || (some_k && (!k || !v || !dk || !dv))) return UA_ERR_NULL;
  for (const void* x : {dout, q, k, v, (const void*)dq, (const void*)dk, (const void*)dv})
    if (!aligned16(x)) return UA_ERR_ALIGN;
  for (const int64_t* s : {do_strides, q_strides, k_strides, v_strides})
    if (!swa_strides_ok(s, false)) return UA_ERR_ALIGN;
  for (const int64_t* s : {dq_strides, dk_strides, dv_strides})
    if (!swa_strides_ok(s, true)) return UA_ERR_ALIGN;
  for (const int64_t* s : {do_strides, q_strides, k_strides, v_strides})
    if (s[1] > UA_SWA_MAX_TOKEN_STRIDE) return UA_ERR_SHAPE;
  rc = check_device();
  if (rc != UA_OK) return rc;
  auto three = [](const int64_t* s) { return Strides3{s[0], s[1], s[2]}; };
  p.dout = dout; p.q = q; p.k = k; p.v = v; p.lse = const_cast<float*>(lse); p.delta = const_cast<float*>(delta);
  p.dq = dq; p.dk = dk; p.dv = dv;
  p.ds = three(do_strides); p.qs = three(q_strides); p.ks = three(k_strides); p.vs = three(v_strides);
  p.dqs = three(dq_strides); p.dks = three(dk_strides); p.dvs = three(dv_strides);
  BwdCut cut = bwd_cut(p, head_dim, workspace && aligned16(workspace));
  if (workspace_bytes < cut.total) cut = bwd_cut(p, head_dim, false);
  p.n_parts = cut.row_parts;
  p.by_parts = make_div(p.n_parts);
  const int key_heads = batch * n_kv_heads;
  char* at = (char*)workspace;
  SwaSums sums{};
  int n_sums = 0;
  auto sum = [&](const float* parts, int64_t part, int n_parts, void* out, const Strides3& os, int tokens, int part_tokens, int heads) {
    const int rows = batch * heads * tokens;
    sums.s[n_sums++] = {parts, out, part, os, n_parts, tokens, part_tokens, heads, rows, (rows + 15) / 16, make_div(std::max(tokens, 1)), make_div(heads)};
  };
  const int size = 2;                                     // bytes of an element
  for (int i = 0; i < 2; ++i) {
    SwaColumns& c = p.cols[i];
    c.first = i ? cut.n_sink : 0;
    c.tiles = i ? p.n_ktiles - cut.n_sink : cut.n_sink;
    c.n_parts = cut.col_parts[i];
    c.by_parts = make_div(c.n_parts);
    c.n_blocks = key_heads * c.tiles * c.n_parts;
    c.map = block_map(std::max(key_heads, 1), std::max(c.tiles * c.n_parts, 1));
    p.n_col_blocks += c.n_blocks;
    if (c.n_parts == 1 || c.tiles == 0) continue;
    c.part = cut.col_bytes[i] / 4;
    c.dk = (float*)at;
    c.dv = (float*)(at + c.n_parts * cut.col_bytes[i]);
    at += 2 * c.n_parts * cut.col_bytes[i];
    const int row = c.first * kSwaRows, tokens = std::min(c.tiles * kSwaRows, seqlen_k - row);
    sum(c.dk, c.part, c.n_parts, (char*)dk + row * p.dks.s * size, p.dks, tokens, c.tiles * kSwaRows, n_kv_heads);
    sum(c.dv, c.part, c.n_parts, (char*)dv + row * p.dvs.s * size, p.dvs, tokens, c.tiles * kSwaRows, n_kv_heads);
  }
  if (p.n_parts > 1) {
    p.part_o = (float*)at;
    p.o_part = cut.dq_bytes / 4;
    sum(p.part_o, p.o_part, p.n_parts, dq, p.dqs, seqlen_q, seqlen_q, n_heads);
  }
  p.map = block_map(std::max(batch * n_heads, 1), std::max(p.n_qtiles * p.n_parts, 1));
  const unsigned n = (unsigned)(p.n_col_blocks + batch * n_heads * p.n_qtiles * p.n_parts);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == UA_FP16) return head_dim == 64 ? bwd_run<fp16, 64>(p, n, sums, st) : bwd_run<fp16, 128>(p, n, sums, st);
  return head_dim == 64 ? bwd_run<bf16, 64>(p, n, sums, st) : bwd_run<bf16, 128>(p, n, sums, st);
}
