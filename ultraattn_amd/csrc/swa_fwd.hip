// Sliding-window attention with sinks, forward.
//
// One workgroup (4 waves of 32 query rows) per (128 rows, head) walks the 64-key blocks that its rows see (SwaWalk): the sinks' blocks, then the
// window's.  Transposed products, as in the block-sparse forward: S^T = K Q^T, O^T += V^T P^T, so that a lane holds one query's column and
// exp2(S^T), rounded, is the next product's B operand.  Only blocks at the window's edges compare positions; blocks that a wave's 32 rows do not see
// are skipped by it.  K and V come in through two LDS stages, the next block's copies between this one's matrix instructions.
//
// The running maximum is raised only where a block's sums show a score far above it, or where a row has not seen a key yet.
//
// P is rounded to the operands' type, which the matrix instruction asks for: independent errors of half a step, which the sum over the keys averages,
// beside the output's own (error against 64 bits: bf16 1.9e-3, with P in 32 bits 1.6e-3).  Scores, the row sums and O stay in fp32.
#include <algorithm>
#include <type_traits>
#include "swa.h"

namespace ua {

// kSum: sums of a lane's 32 exponentials from which the reference is raised; kBits: P is held times 2^kBits of the largest score's.  fp16 holds P up
// to 65504 and, times 2^7, down to 2^-31 of the largest: without that, 70000 keys at 2^-26 of it, a thousandth of the row, vanished.
// (32 equal keys leave the sum 8 times below the bound.)
template <class T> struct SwaRaise;
template <> struct SwaRaise<bf16> { static constexpr float kSum = 16777216.f, kBits = 0.f; };
template <> struct SwaRaise<fp16> { static constexpr float kSum = 32768.f, kBits = 7.f; };

template <class T, int kD>
__global__ __launch_bounds__(256, 2) void swa_fwd_kernel(const SwaParams p) {
  using H = SwaHead<kD>;
  using V = SwaVec<T>;
  typedef typename V::x8 x8;
  __shared__ __attribute__((aligned(1024))) unsigned char stage_a[2 * H::kTile];
  __shared__ __attribute__((aligned(1024))) unsigned char stage_b[2 * H::kTile];
  const uint32_t lds[2] = {(uint32_t)(uintptr_t)(lds_byte*)stage_a, (uint32_t)(uintptr_t)(lds_byte*)stage_b};
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int pos, bh;
  map_block(blockIdx.x, p.map, pos, bh);
  const int line = quotient(pos, p.by_parts), part = pos - line * p.n_parts;
  const int qt = p.n_qtiles - 1 - line;                   // (the longest walks of a causal window first)
  const int b = quotient(bh, p.by_heads), h = bh - b * p.n_heads, hk = quotient(h, p.by_group);
  const int r0 = qt * kSwaRows, row0 = r0 + 32 * wave, n_rows = p.seq_q - row0;      // rows of this wave that exist (may be <= 0)

  const SwaWalk walk(r0, min(r0 + kSwaRows, p.seq_q) - 1, p.hi, p.lo, p.sinks, p.seq_k);
  const int part_len = (walk.n + p.n_parts - 1) / p.n_parts, i0 = min(part * part_len, walk.n), i1 = min(i0 + part_len, walk.n);
  typedef SwaStream<kD, kN, kT> Stream;
  Stream in(p.ks.s, p.vs.s, wave, lane);
  in.of((const T*)p.k + b * p.ks.b + hk * p.ks.h, (const T*)p.v + b * p.vs.b + hk * p.vs.h);
  if (i0 < i1) {
    in.block(walk.at(i0) * kSwaBlock, walk.end_of(walk.at(i0)), true);
#pragma unroll
    for (int n = 0; n < in.kPieces; ++n) in.copy(n, lds[0]);
  }
  x8 qf[H::kSteps];
  {
    u32x4 raw[H::kSteps];
    const int first = min(row0, p.seq_q - 1);
    swa_load_rows<kD>(raw, (const T*)p.q + b * p.qs.b + first * p.qs.s + h * p.qs.h, p.qs.s, p.seq_q - first);
    const uint32_t turn = lds[1] + wave * 32 * H::kRow;   // the stage that the first step fills
    swa_put_rows<kD>(raw, turn);
    swa_frags<T, kD>(qf, turn);
#pragma unroll
    for (int i = 0; i < H::kSteps; ++i) asm volatile("" : "+v"(qf[i]));      // read before the walk
  }
  f32x16 o[H::kBlocks];
#pragma unroll
  for (int m = 0; m < H::kBlocks; ++m) o[m] = f32x16{0};
  float m_run = -INFINITY, m_use = 0.f, l_run = 0.f;
  uint32_t nat[H::kSteps], tr[H::kBlocks];
#pragma unroll
  for (int i = 0; i < H::kSteps; ++i) nat[i] = H::at_n(lane & 31, 2 * i + (lane >> 5));
#pragma unroll
  for (int m = 0; m < H::kBlocks; ++m) tr[m] = Stream::kSecond + H::tr_offset(lane, m);

  auto step = [&](int i, auto stage_tag) {
    constexpr int kStage = decltype(stage_tag)::value;
    const uint32_t here = lds[kStage], other = lds[kStage ^ 1];
    const int key0 = walk.at(i) * kSwaBlock;
    in.block(walk.at(i + 1) * kSwaBlock, walk.end_of(walk.at(i + 1)), i + 1 < i1);
    wait_vmem_all();
    __syncthreads();                        // this block has landed, and everyone has left the other stage
    const bool hidden = key0 > row0 + 31 + p.hi || (key0 + kSwaBlock <= row0 + p.lo && key0 >= p.sinks);
    if (hidden) {
#pragma unroll
      for (int n = 0; n < in.kPieces; ++n) in.copy(n, other);
      return;
    }
    // S^T: two blocks of 32 keys in turn
    f32x16 s[2] = {f32x16{0}, f32x16{0}};
    {
      constexpr int kAhead = 4, kAll = 2 * H::kSteps;
      x8 kf[kAll];
      auto rd = [&](int n) { return lds_get<x8>(here + nat[n >> 1] + 32 * H::kRow * (n & 1)); };
#pragma unroll
      for (int n = 0; n < kAhead; ++n) kf[n] = rd(n);
      __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
      for (int n = 0; n < kAll; ++n) {
        if (n + kAhead < kAll) kf[n + kAhead] = rd(n + kAhead);
        s[n & 1] = V::mfma(kf[n], qf[n >> 1], s[n & 1]);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        if (n & 1) in.copy(n >> 1, other);
      }
      static_assert(kAll / 2 == Stream::kPieces, "a copy after every other product");
    }
    const bool whole = key0 + kSwaBlock - 1 <= min(row0 + p.hi, p.seq_k - 1) && (key0 >= row0 + 31 + p.lo || key0 + kSwaBlock <= p.sinks);
    if (!whole) {
      const int lane_now = fresh_lane(), row = row0 + (lane_now & 31), last = min(row + p.hi, p.seq_k - 1), first = row + p.lo;
      const uint32_t seen = (uint32_t)max(last - first + 1, 0);
      const int sinks = min(p.sinks, last + 1), key = key0 + 4 * (lane_now >> 5);
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int k = key + 32 * mb + 8 * (j >> 2) + (j & 3);
          if ((uint32_t)(k - first) >= seen && k >= sinks) s[mb][j] = -INFINITY;
        }
      if (key0 < walk.start && key0 + kSwaBlock > walk.start) lds_clear_rows<kD, 1024>(here + Stream::kSecond, max(p.sinks - key0, 0), walk.start - key0);
    }
    constexpr int kVAhead = 3, kVAll = 4 * H::kBlocks;
    x8 vf[4];
    auto rd_v = [&](int n) {                // fragment n % kBlocks of 16 keys
      const uint32_t at = here + tr[n % H::kBlocks] + 16 * H::kRow * (n / H::kBlocks);
      return lds_tr_pair<T>(at, at + 8 * H::kRow);
    };
#pragma unroll
    for (int n = 0; n < kVAhead; ++n) vf[n] = rd_v(n);
    float rs = 0.f;
    x8 pf[4];
    auto exponentials = [&]() {
      rs = 0.f;
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float e = fast_exp2(fmaf(s[mb][j], p.scale_log2, -m_use));
          rs += e;
          pf[2 * mb + (j >> 3)][j & 7] = (T)e;
        }
    };
    exponentials();
    if (__builtin_amdgcn_ballot_w64(!(rs < SwaRaise<T>::kSum) || m_run == -INFINITY) != 0) {        // wave-uniform, rare
      float mx = s[0][0], a, c;
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[mb][j]);
      swap_lanes<32>(mx, a, c);
      const float m_new = fmaxf(m_run, fmaxf(a, c) * p.scale_log2);
      m_use = m_new == -INFINITY ? 0.f : m_new - SwaRaise<T>::kBits;
      const float alpha = m_new == m_run ? 1.f : fast_exp2(m_run - m_new);      // m_run = -inf -> 0
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int m = 0; m < H::kBlocks; ++m)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[m][j] *= alpha;
      exponentials();
    }
    l_run += rs;
#pragma unroll
    for (int n = 0; n < kVAll; ++n) {
      if (n + kVAhead < kVAll) vf[(n + kVAhead) & 3] = rd_v(n + kVAhead);
      o[n % H::kBlocks] = V::mfma(vf[n & 3], pf[n / H::kBlocks], o[n % H::kBlocks]);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
  };
  for (int i = i0; i < i1; i += 2) {
    step(i, std::integral_constant<int, 0>{});
    if (i + 1 < i1) step(i + 1, std::integral_constant<int, 1>{});
  }
  wait_vmem_all();                          // the last step's copies filled a stage with zeros
  __syncthreads();
  if (n_rows <= 0) return;
  float a, c;
  swap_lanes<32>(l_run, a, c);
  const float l = a + c, inv = l > 0.f || l != l ? 1.f / l : 0.f;      // (NaN stays)
  const float lse = l > 0.f || l != l ? (m_use + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
  const int out_lane = fresh_lane();
  if (p.n_parts > 1) {
    const int64_t row = ((int64_t)bh * p.seq_q + row0);
    swa_store_f32<kD>(p.part_o + part * p.o_part + row * kD, kD, n_rows, o, inv);
    if (out_lane < min(n_rows, 32)) p.part_lse[part * p.lse_part + row + out_lane] = lse;
  } else {
    swa_store_rows<T, kD>((T*)p.o + b * p.os.b + (int64_t)row0 * p.os.s + h * p.os.h, p.os.s, n_rows, o, inv, lds[0] + wave * 32 * H::kRow);
    if (out_lane < min(n_rows, 32)) p.lse[(int64_t)bh * p.seq_q + row0 + out_lane] = lse;
  }
}

// Partial rows of fp32 and their lse, part i of row (b, h, s) at part_o + i * o_part + row * kD:
//   LSE = log sum_p exp(lse_p),  O = sum_p exp(lse_p - LSE) O_p.
// kLanes a row: a lane a part for the statistics, then groups of 16 lanes that take the parts' rows in turn.  Bound by the launch and by how many loads
// follow one another with many parts (a new token against 8000 keys in 31: 16 lanes a row 29.9 us, 64 13.1), by the rows with few (4 heads of 8192 in two:
// 16 lanes 53.2 us, 64 58.6).
template <class T, int kD, int kLanes>
__global__ __launch_bounds__(256) void merge_rows_kernel(const float* part_o, int64_t o_part, const float* part_lse, int64_t lse_part, int n_parts,
                                                         T* o, Strides3 os, float* lse, int n_rows, int n_heads, int seq, Div by_seq, Div by_heads) {
  constexpr int kPer = kD / 16;
  constexpr int kGroups = kLanes / 16;
  const int row = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes, lane = threadIdx.x % kLanes, c = lane & 15;
  if (row >= n_rows) return;
  const float l = lane < n_parts ? part_lse[lane * lse_part + row] : -INFINITY;
  float top = l;
#pragma unroll
  for (int d = kLanes / 2; d; d /= 2) top = fmaxf(top, __shfl_xor(top, d));
  const float at = top == -INFINITY ? 0.f : top, w = l == -INFINITY ? 0.f : fast_exp2((l - at) * kLog2e);
  float total = w, acc[kPer] = {};
#pragma unroll
  for (int d = kLanes / 2; d; d /= 2) total += __shfl_xor(total, d);
  for (int i0 = 0; i0 < n_parts; i0 += kGroups) {
    const int i = i0 + (lane >> 4);
    const float f = __shfl(w, i % kLanes, kLanes);
    if (i < n_parts && f != 0.f) {                       // (a part that saw nothing left no row)
      const float* x = part_o + i * o_part + (int64_t)row * kD + c * kPer;
#pragma unroll
      for (int j = 0; j < kPer; j += 4) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(x + j);
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[j + n] += f * y[n];
      }
    }
  }
  if constexpr (kGroups == 4)
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      acc[j] += __shfl_xor(acc[j], 16);
      acc[j] += __shfl_xor(acc[j], 32);
    }
  const bool any = total > 0.f || total != total;        // (NaN stays)
  const float inv = any ? 1.f / total : 0.f;
  const int bh = quotient(row, by_seq), s = row - bh * seq, b = quotient(bh, by_heads), h = bh - b * n_heads;
  if (lane < 16) {
    typedef __attribute__((ext_vector_type(kPer))) T vec;
    vec x;
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[j] = (T)(acc[j] * inv);
    *reinterpret_cast<vec*>(o + b * os.b + (int64_t)s * os.s + h * os.h + c * kPer) = x;
  }
  if (lane == 0) lse[row] = any ? at + __builtin_amdgcn_logf(total) * kLn2 : -INFINITY;
}

int swa_merge(const float* part_o, int64_t o_part, const float* part_lse, int64_t lse_part, int n_parts, void* o, const Strides3& os, float* lse,
              int batch, int n_heads, int seq, int head_dim, int dtype, hipStream_t st) {
  const int n_rows = batch * n_heads * seq;
  auto run = [&](auto kernel, int lanes, auto* out) {
    const int rows = 256 / lanes;
    kernel<<<(n_rows + rows - 1) / rows, 256, 0, st>>>(part_o, o_part, part_lse, lse_part, n_parts, out, os, lse, n_rows, n_heads, seq, make_div(seq),
                                                       make_div(n_heads));
  };
  auto by_lanes = [&](auto* out, auto dim) {
    typedef std::remove_pointer_t<decltype(out)> T;
    constexpr int kD = decltype(dim)::value;
    if (n_parts <= 4) run(merge_rows_kernel<T, kD, 16>, 16, out);
    else              run(merge_rows_kernel<T, kD, 64>, 64, out);
  };
  auto by_dim = [&](auto* out) {
    if (head_dim == 64) by_lanes(out, std::integral_constant<int, 64>{});
    else                by_lanes(out, std::integral_constant<int, 128>{});
  };
  if (dtype == UA_FP16) by_dim((fp16*)o); else by_dim((bf16*)o);
  return hipGetLastError() == hipSuccess ? UA_OK : UA_ERR_LAUNCH;
}

bool swa_strides_ok(const int64_t* s, bool written) {
  if (s[0] % 8 || s[1] % 8 || s[2] % 8 || s[0] < 0 || s[1] < 0 || s[2] < 0) return false;
  return !written || (s[1] > 0 && s[2] > 0);
}

int swa_fill(SwaParams& p, int batch, int n_heads, int n_kv_heads, int seq_q, int seq_k, int head_dim, int dtype, int64_t q_start, int64_t k_start,
             int64_t left, int64_t right, int64_t sinks, float softmax_scale) {
  constexpr int64_t kMost = int64_t(1) << 60;
  if (batch < 0 || n_heads <= 0 || n_kv_heads <= 0 || seq_q < 0 || seq_k < 0 || n_heads % n_kv_heads) return UA_ERR_SHAPE;
  const int64_t heads = (int64_t)batch * n_heads;
  if (seq_q > kSwaMaxLen || seq_k > kSwaMaxLen || heads > kSwaMaxGroups || heads * ((seq_q + kSwaRows - 1) / kSwaRows) > kSwaMaxGroups / 2 ||
      heads * ((seq_k + kSwaRows - 1) / kSwaRows) > kSwaMaxGroups / 2)
    return UA_ERR_SHAPE;
  if (q_start > kMost || q_start < -kMost || k_start > kMost || k_start < -kMost || left < -1 || right < -1 || left > kMost || right > kMost || sinks < 0 ||
      sinks > kMost)
    return UA_ERR_SHAPE;
  if ((head_dim != 64 && head_dim != 128) || (dtype != UA_BF16 && dtype != UA_FP16) || !swa_scale_ok(softmax_scale)) return UA_ERR_UNSUPPORTED;
  auto clamp = [](int64_t x) { return (int)std::min<int64_t>(std::max<int64_t>(x, -kFar), kFar); };
  p.batch = batch; p.n_heads = n_heads; p.n_kv_heads = n_kv_heads; p.group = n_heads / n_kv_heads; p.seq_q = seq_q; p.seq_k = seq_k;
  p.hi = right < 0 ? kFar : clamp(q_start - k_start + right);
  p.lo = left < 0 ? -kFar : clamp(q_start - k_start - left);
  p.sinks = left < 0 ? 0 : (int)std::min<int64_t>(std::max<int64_t>(sinks - k_start, 0), seq_k);
  p.scale = softmax_scale;
  p.scale_log2 = softmax_scale * kLog2e;
  p.n_qtiles = (seq_q + kSwaRows - 1) / kSwaRows;
  p.n_ktiles = (seq_k + kSwaRows - 1) / kSwaRows;
  p.n_parts = 1;
  p.by_heads = make_div(n_heads);
  p.by_kv_heads = make_div(n_kv_heads);
  p.by_group = make_div(p.group);
  return UA_OK;
}

// Parts that a forward's walks are cut into: what an estimate of the launch's time in microseconds says.  A step takes `alone` where a CU has one
// workgroup and `shared` where it has two; parts cost a launch for their merge, and each its rows' way through the caches.  (Of heads of 64 three fit a
// CU; the estimate counts two for them as well, and its constants were fitted that way.)  us, whole and in 2, 4, 8 and 16 parts (heads, queries x
// keys, window):
//     128 columns   4, 2048 causal     37.0   28.4   23.9   26.8   34.1          64 columns   8, 2048 causal       29.4  25.0  22.9  29.0  33.6
//                   8, 128 x 4096      66.6   41.1   27.0   19.8   18.4                       2, 8192, 2047        34.3  26.8  26.2  32.4  39.8
//                  32, 100 x 16384    255    135     74.1   46.5   45.5                       8, 512 causal        10.9  12.2  11.7  11.6  13.3
//                   4, 8192, 2047      44.3   52.5   58.3   82.6  136                         2 x 10, 1333 x 2048, 700  20.3  25.4  28.4  37.3  49.8
static int fwd_parts(const SwaParams& p, int head_dim) {
  const double lines = (double)p.batch * p.n_heads * p.n_qtiles;
  if (lines == 0 || lines >= 2 * kCus) return 1;
  const SwaSteps s = swa_row_steps(p);
  const double alone = head_dim == 64 ? 0.75 : 1.0, shared = head_dim == 64 ? 1.2 : 2.05;
  const double part_us = 0.15 + (double)p.batch * p.n_heads * p.seq_q * head_dim * 8e-7;      // written and read
  int best = 1;
  double best_us = 1e30;
  for (int parts = 1; parts <= UA_MAX_PARTS && (parts == 1 || 2 * parts <= s.most); ++parts) {
    const double busy = lines * parts * s.mean / std::max(s.most, 1), beside = std::min(std::max((busy - kCus) / kCus, 0.0), 1.0);
    const double walk = std::max((s.most + parts - 1) / parts * (alone + (shared - alone) * beside), lines * s.mean / (2 * kCus) * shared);
    const double us = 5 + walk + (parts > 1 ? 5 + part_us * parts : 0);
    if (us < 0.93 * best_us) { best_us = us; best = parts; }
  }
  return best;
}
static int64_t part_rows(const SwaParams& p) { return (int64_t)p.batch * p.n_heads * p.seq_q; }

}  // namespace ua

extern "C" int64_t ua_swa_workspace_bytes(int batch, int n_heads, int n_kv_heads, int seqlen_q, int seqlen_k, int head_dim, int64_t q_start,
                                          int64_t k_start, int64_t left, int64_t right, int64_t sinks) {
  using namespace ua;
  SwaParams p{};
  if (swa_fill(p, batch, n_heads, n_kv_heads, seqlen_q, seqlen_k, head_dim, UA_BF16, q_start, k_start, left, right, sinks, 1.f) != UA_OK) return 0;
  const int parts = fwd_parts(p, head_dim);
  return parts > 1 ? parts * (align256(part_rows(p) * head_dim * 4) + align256(part_rows(p) * 4)) : 0;
}

extern "C" int ua_swa_fwd(const void* q, const void* k, const void* v, void* o, float* lse, int batch, int n_heads, int n_kv_heads, int seqlen_q,
                          int seqlen_k, int head_dim, int dtype, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                          const int64_t* o_strides, int64_t q_start, int64_t k_start, int64_t left, int64_t right, int64_t sinks, float softmax_scale,
                          void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace ua;
  SwaParams p{};
  int rc = swa_fill(p, batch, n_heads, n_kv_heads, seqlen_q, seqlen_k, head_dim, dtype, q_start, k_start, left, right, sinks, softmax_scale);
  if (rc != UA_OK) return rc;
  if ((int64_t)batch * seqlen_q == 0) return UA_OK;
  if (!q || !o || !lse || !q_strides || !o_strides || !k_strides || !v_strides || (seqlen_k > 0 && (!k || !v))) return UA_ERR_NULL;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !swa_strides_ok(q_strides, false) || !swa_strides_ok(k_strides, false) ||
      !swa_strides_ok(v_strides, false) || !swa_strides_ok(o_strides, true))
    return UA_ERR_ALIGN;
  if (k_strides[1] > UA_SWA_MAX_TOKEN_STRIDE || v_strides[1] > UA_SWA_MAX_TOKEN_STRIDE) return UA_ERR_SHAPE;
  rc = check_device();
  if (rc != UA_OK) return rc;
  p.q = q; p.k = k; p.v = v; p.o = o; p.lse = lse;
  p.qs = {q_strides[0], q_strides[1], q_strides[2]};
  p.ks = {k_strides[0], k_strides[1], k_strides[2]};
  p.vs = {v_strides[0], v_strides[1], v_strides[2]};
  p.os = {o_strides[0], o_strides[1], o_strides[2]};
  const hipStream_t st = (hipStream_t)stream;
  const int parts = fwd_parts(p, head_dim);
  const int64_t o_bytes = align256(part_rows(p) * head_dim * 4), lse_bytes = align256(part_rows(p) * 4);
  if (parts > 1 && workspace && aligned16(workspace) && workspace_bytes >= parts * (o_bytes + lse_bytes)) {
    p.n_parts = parts;
    p.part_o = (float*)workspace;
    p.o_part = o_bytes / 4;
    p.part_lse = (float*)((char*)workspace + parts * o_bytes);
    p.lse_part = lse_bytes / 4;
  }
  p.by_parts = make_div(p.n_parts);
  p.map = block_map(batch * n_heads, p.n_qtiles * p.n_parts);
  const unsigned n = (unsigned)(batch * n_heads * p.n_qtiles * p.n_parts);
  if (dtype == UA_FP16) {
    if (head_dim == 64) swa_fwd_kernel<fp16, 64><<<n, 256, 0, st>>>(p);
    else                swa_fwd_kernel<fp16, 128><<<n, 256, 0, st>>>(p);
  } else {
    if (head_dim == 64) swa_fwd_kernel<bf16, 64><<<n, 256, 0, st>>>(p);
    else                swa_fwd_kernel<bf16, 128><<<n, 256, 0, st>>>(p);
  }
  if (hipGetLastError() != hipSuccess) return UA_ERR_LAUNCH;
  if (p.n_parts == 1) return UA_OK;
  return swa_merge(p.part_o, p.o_part, p.part_lse, p.lse_part, p.n_parts, o, p.os, lse, batch, n_heads, seqlen_q, head_dim, dtype, st);
}
