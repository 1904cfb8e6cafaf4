// Sliding-window attention of a few new tokens of every sequence against its cache.
//
// The rows of a key head, T tokens of each of the query heads that share it, are up to 16 (or 32) columns of 16x16x32 matrix instructions:
// S^T = K Q^T, O^T += V^T P^T.  A workgroup's four waves go through blocks of 32 keys of their own, each through its own two stages of LDS: no wave
// waits for another before the end, where their rows are merged.  The keys of long caches are cut into parts, workgroups of their own, that leave fp32 rows
// for a merge.
//
// Bound: HBM, the visible keys and values once per 32 rows of a key head: from 33 rows on (5 tokens of 7 heads, say) another workgroup reads them again, seldom
// from a cache (64 x 8 key heads of 8000: 32 rows 375 us, 35 to 64 rows 600).  Two stages of 16 KiB a wave keep 64 to 128 KiB in flight on every CU.
// P is rounded as in the forward.
#include <algorithm>
#include <cmath>
#include "swa.h"

namespace ua {

constexpr int kDecBlock = 32, kDecWaves = 4, kDecMaxParts = 64;

// P is held times 2^kDecBits of the largest score's, which no score exceeds here: fp16 then has it down to 2^-38 of that.
template <class T> constexpr float kDecBits = 0.f;
template <> constexpr float kDecBits<fp16> = 14.f;

struct DecParams {
  const void *q, *k, *v;
  void* o;
  float* lse;
  const int32_t* lens;
  Strides3 qs, ks, vs, os;
  int n_tokens, n_heads, n_kv_heads, group, room, left, sinks, rows, n_tiles, n_parts;       // left: kFar = no bound; rows: of a key head
  float scale_log2;
  float *part_o, *part_lse;
  int64_t o_part, lse_part;
  Div by_kv_heads, by_group, by_tiles, by_parts;
};

template <int kD>
struct DecHead {
  static constexpr int kRow = 2 * kD, kChunks = kD / 8, kCopyRows = 1024 / kRow, kUnits = kDecBlock / kCopyRows, kTile = kUnits * 1024;
  static constexpr int kStage = 2 * kTile, kWave = 2 * kStage, kSteps = kD / 32, kBlocks = kD / 16;
  // K: 16 rows are read at one chunk.  V is read transposed: 8 rows at two chunks that start at a multiple of two.
  static __device__ __forceinline__ int slot_k(int r, int c) { return kD == 128 ? c ^ (r & 15) : c ^ (r >> 1 & 7); }
  static __device__ __forceinline__ int slot_v(int r, int c) { return kD == 128 ? c ^ ((r & 3) << 2) ^ ((r >> 2 & 1) << 1) : c ^ ((r >> 1 & 3) << 1); }
};

template <class T, int kD, int kTiles>
__global__ __launch_bounds__(64 * kDecWaves) void swa_decode_kernel(const DecParams p) {
  using H = DecHead<kD>;
  using V = SwaVec<T>;
  typedef typename V::x8 x8;
  constexpr int kRows = 16 * kTiles, kOutPitch = 4 * kD + 16;             // (bytes of a row of fp32 at the merge)
  static_assert(kRows * kOutPitch + 8 * kRows <= H::kWave, "a wave's rows and statistics fit its stages");
  __shared__ __attribute__((aligned(1024))) unsigned char smem[kDecWaves * H::kWave];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_byte*)smem;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, quad = lane >> 4;
  const int rest = quotient(blockIdx.x, p.by_parts), part = blockIdx.x - rest * p.n_parts;
  const int bh = quotient(rest, p.by_tiles), tile = rest - bh * p.n_tiles, b = quotient(bh, p.by_kv_heads), hk = bh - b * p.n_kv_heads;
  const int next = min(max(p.lens[b], 0), kFar), len = min(next, p.room);      // (a length beyond the cache counts for the positions)
  const int row0 = tile * kRows, row1 = min(row0 + kRows, p.rows) - 1;
  const int pos0 = next - p.n_tokens + quotient(row0, p.by_group), pos1 = next - p.n_tokens + quotient(row1, p.by_group);
  const int last = min(pos1, len - 1), start = max(pos0 - p.left, 0);
  const int sinks_end = min(p.sinks, last + 1), n_sink = last >= 0 ? (sinks_end + kDecBlock - 1) / kDecBlock : 0, first = max(start / kDecBlock, n_sink);
  const int n_all = n_sink + (last >= start ? max(last / kDecBlock + 1 - first, 0) : 0);
  const int part_len = (n_all + p.n_parts - 1) / p.n_parts, i0 = min(part * part_len, n_all), i1 = min(i0 + part_len, n_all);
  auto key_of = [&](int i) { return (i < n_sink ? i : first + i - n_sink) * kDecBlock; };

  const char* const kbase = (const char*)((const T*)p.k + b * p.ks.b + hk * p.ks.h);
  const char* const vbase = (const char*)((const T*)p.v + b * p.vs.b + hk * p.vs.h);
  const int64_t k_row = 2 * p.ks.s, v_row = 2 * p.vs.s;
  const uint32_t mine = lds0 + wave * H::kWave;
  const int copy_row = lane / H::kChunks, chunk = lane % H::kChunks, k_off = copy_row * (int)k_row, v_off = copy_row * (int)v_row;
  auto copy_in = [&](int i, uint32_t stage) {
    const int key0 = key_of(i), n = i < i1 ? min((key0 + kDecBlock <= start ? sinks_end : last + 1) - key0, kDecBlock) : 0;       // (what no row sees is not read)
    const u32x4 rk = make_rsrc_words(kbase + key0 * k_row, n > 0 ? (uint32_t)((n - 1) * k_row + H::kRow) : 0);
    const u32x4 rv = make_rsrc_words(vbase + key0 * v_row, n > 0 ? (uint32_t)((n - 1) * v_row + H::kRow) : 0);
#pragma unroll
    for (int u = 0; u < H::kUnits; ++u) {
      const int r = H::kCopyRows * u + copy_row;
      dma16_abs(rk, stage + 1024 * u, k_off + 16 * H::slot_k(r, chunk), H::kCopyRows * u * (int)k_row);
      dma16_abs(rv, stage + H::kTile + 1024 * u, v_off + 16 * H::slot_v(r, chunk), H::kCopyRows * u * (int)v_row);
    }
  };
  int i = i0 + wave;
  copy_in(i, mine);
  copy_in(i + kDecWaves, mine + H::kStage);

  // Q as B operands: row col of the tile, columns 32 s + 8 quad ..
  x8 qf[kTiles][H::kSteps];
  int hi[kTiles], lo[kTiles];                 // the keys that the lane's row sees: lo .. hi, and the sinks up to hi
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const int row = min(row0 + 16 * t + col, p.rows - 1), token = quotient(row, p.by_group), h = hk * p.group + row - token * p.group;
    const T* q = (const T*)p.q + b * p.qs.b + token * p.qs.s + h * p.qs.h + 8 * quad;
#pragma unroll
    for (int s = 0; s < H::kSteps; ++s) qf[t][s] = *reinterpret_cast<const x8*>(q + 32 * s);
    const int pos = next - p.n_tokens + token;
    hi[t] = min(pos, len - 1);
    lo[t] = pos - p.left;
  }
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int s = 0; s < H::kSteps; ++s) asm volatile("" : "+v"(qf[t][s]));     // arrived before the walk counts its copies
  f32x4 o[kTiles][H::kBlocks];
  float m_run[kTiles], m_use[kTiles], l_run[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    m_run[t] = -INFINITY;
    m_use[t] = l_run[t] = 0.f;
#pragma unroll
    for (int d = 0; d < H::kBlocks; ++d) o[t][d] = f32x4{0};
  }
  uint32_t stage = mine, other = mine + H::kStage;
  constexpr int kCopies = 2 * H::kUnits;
  for (; i < i1; i += kDecWaves) {
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(kCopies) : "memory");       // the older stage has landed
    const int key0 = key_of(i);
    x8 kf[2][H::kSteps];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int s = 0; s < H::kSteps; ++s) {
        const int r = 16 * n + col;
        kf[n][s] = lds_get<x8>(stage + r * H::kRow + (H::slot_k(r, 4 * s + quad) << 4));
      }
    if (key0 < start && key0 + kDecBlock > start) lds_clear_rows<kD, 1024>(stage + H::kTile, max(p.sinks - key0, 0), start - key0);
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
      const uint32_t seen = (uint32_t)max(hi[t] - lo[t] + 1, 0);
      const int sinks = min(p.sinks, hi[t] + 1);
      float mx = -INFINITY, a, c;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = key0 + 16 * n + 4 * quad + j;
          if ((uint32_t)(k - lo[t]) >= seen && k >= sinks) s[n][j] = -INFINITY;
          mx = fmaxf(mx, s[n][j]);
        }
      swap_lanes<16>(mx, a, c);
      swap_lanes<32>(fmaxf(a, c), a, c);
      mx = fmaxf(a, c) * p.scale_log2;
      if (__builtin_amdgcn_ballot_w64(mx > m_run[t]) != 0) {
        const float m_new = fmaxf(m_run[t], mx);
        m_use[t] = m_new == -INFINITY ? 0.f : m_new - kDecBits<T>;
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
    copy_in(i + 2 * kDecWaves, stage);
    const uint32_t x = stage;
    stage = other;
    other = x;
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
    for (int w = 0; w < kDecWaves; ++w) m = fmaxf(m, lds_get<float>(lds0 + w * H::kWave + kRows * kOutPitch + 8 * r));
    const float at = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kDecWaves; ++w) {
      const uint32_t from = lds0 + w * H::kWave;
      const float f = fast_exp2(lds_get<float>(from + kRows * kOutPitch + 8 * r) - at);
      l += f * lds_get<float>(from + kRows * kOutPitch + 8 * r + 4);
#pragma unroll
      for (int j = 0; j < kPer; j += 4) {
        const f32x4 x = lds_get<f32x4>(from + r * kOutPitch + (c * kPer + j) * 4);
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[j + n] += f * x[n];
      }
    }
    const bool any = l > 0.f || l != l;
    const float inv = any ? 1.f / l : 0.f, lse = any ? (m - kDecBits<T> + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
    const int token = quotient(row, p.by_group), h = hk * p.group + row - token * p.group;
    const int64_t out_row = ((int64_t)b * p.n_heads + h) * p.n_tokens + token;
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
      for (int j = 0; j < kPer; ++j) w[j] = (T)(acc[j] * inv);
      *reinterpret_cast<vec*>((T*)p.o + b * p.os.b + token * p.os.s + h * p.os.h + c * kPer) = w;
      if (c == 0) p.lse[out_row] = lse;
    }
  }
}

struct DecShape { int tiles, row_tiles, parts; };        // 16-row tiles of a workgroup, workgroups of a key head's rows, parts of its keys
// Parts of a key head's keys: what an estimate in microseconds says of the longest caches that the call allows (lengths are on the device).  A round of
// workgroups on all CUs takes its start and its iterations, or what its keys take from memory; whole caches of a batch differ in length, and the longest
// ones end alone (64 x 8 of 8192 to 16384 keys, whole 582 us, in two or four parts 565); parts cost the launch that merges them.
// us in 1, 2, 4, 8, 16 and 32 parts (sequences x key heads, keys, columns):
//     1 x 8, 1027, 128    12.2  11.6  10.7  10.1   9.9  10.2        8 x 8, 4000, 128      33.3  27.1  26.9  29.2  36.6  45.5
//     1 x 8, 8000, 128    57.9  35.7  22.9  16.0  13.3  13.1        16 x 8, 1027, 128     15.8  17.7  23.5  30.3  39.7  65.2
//     4 x 1, 16000, 128  110.5  61.6  36.6  22.9  16.6  14.9        32 x 8, 2000, 64      24.1  26.0  27.0  29.3  35.8  55.4
static DecShape dec_shape(int batch, int n_tokens, int n_heads, int n_kv_heads, int room, int head_dim, int64_t left, int64_t sinks) {
  DecShape s;
  const int64_t rows = (int64_t)n_tokens * (n_heads / n_kv_heads);
  s.tiles = rows <= 16 ? 1 : 2;
  s.row_tiles = (int)((rows + 16 * s.tiles - 1) / (16 * s.tiles));
  const int64_t blocks = ((int64_t)room + kDecBlock - 1) / kDecBlock;
  const int64_t seen = left < 0 ? blocks : std::min(blocks, (std::min<int64_t>(left, kFar) + n_tokens + 2 * kDecBlock - 2) / kDecBlock +
                                                               (std::min<int64_t>(sinks, room) + kDecBlock - 1) / kDecBlock);
  const double groups = (double)batch * n_kv_heads * s.row_tiles, slots = head_dim == 64 ? 2 * kCus : kCus;
  const double memory_us = groups * seen * kDecBlock * head_dim * 4 / 7e6;
  s.parts = 1;
  double best_us = 1e30;
  for (int parts = 1; parts <= kDecMaxParts && (parts == 1 || kDecWaves * (parts - 1) < seen); ++parts) {
    const double rounds = std::ceil(groups * parts / slots), iterations = std::ceil((double)seen / (kDecWaves * parts));
    const double tail = batch > 1 && left < 0 ? 0.4 * iterations : 0;
    const double us = 2 * rounds + std::max(0.8 * rounds * iterations, memory_us) + tail + (parts > 1 ? 3.5 + 0.03 * parts : 0);
    if (us < 0.99 * best_us) { best_us = us; s.parts = parts; }
  }
  return s;
}
static int dec_check(int batch, int n_tokens, int n_heads, int n_kv_heads, int room, int head_dim, int dtype, int64_t left, int64_t sinks, float scale) {
  if (batch < 0 || n_tokens < 0 || n_heads <= 0 || n_kv_heads <= 0 || room < 0 || n_heads % n_kv_heads || left < -1 || sinks < 0) return UA_ERR_SHAPE;
  if (room > kSwaMaxLen || n_tokens > kSwaMaxLen || (int64_t)n_tokens * (n_heads / n_kv_heads) > kSwaMaxLen ||
      (int64_t)batch * n_tokens * n_heads > INT32_MAX / kDecMaxParts)
    return UA_ERR_SHAPE;
  if ((head_dim != 64 && head_dim != 128) || (dtype != UA_BF16 && dtype != UA_FP16) || !swa_scale_ok(scale)) return UA_ERR_UNSUPPORTED;
  return UA_OK;
}
template <class T, int kD>
static void dec_launch(const DecParams& p, int tiles, unsigned n, hipStream_t st) {
  if (tiles == 1) swa_decode_kernel<T, kD, 1><<<n, 64 * kDecWaves, 0, st>>>(p);
  else            swa_decode_kernel<T, kD, 2><<<n, 64 * kDecWaves, 0, st>>>(p);
}

}  // namespace ua

extern "C" int64_t ua_swa_decode_workspace_bytes(int batch, int n_tokens, int n_heads, int n_kv_heads, int room, int head_dim, int64_t left, int64_t sinks) {
  using namespace ua;
  if (dec_check(batch, n_tokens, n_heads, n_kv_heads, room, head_dim, UA_BF16, left, sinks, 1.f) != UA_OK) return 0;
  const int parts = dec_shape(batch, n_tokens, n_heads, n_kv_heads, room, head_dim, left, sinks).parts;
  const int64_t rows = (int64_t)batch * n_tokens * n_heads;
  return parts > 1 ? parts * (align256(rows * head_dim * 4) + align256(rows * 4)) : 0;
}

extern "C" int ua_swa_decode(const void* q, const void* k_cache, const void* v_cache, void* o, float* lse, const int32_t* lens, int batch, int n_tokens,
                             int n_heads, int n_kv_heads, int room, int head_dim, int dtype, const int64_t* q_strides, const int64_t* k_strides,
                             const int64_t* v_strides, const int64_t* o_strides, int64_t left, int64_t sinks, float softmax_scale, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  using namespace ua;
  int rc = dec_check(batch, n_tokens, n_heads, n_kv_heads, room, head_dim, dtype, left, sinks, softmax_scale);
  if (rc != UA_OK) return rc;
  if ((int64_t)batch * n_tokens == 0) return UA_OK;
  if (!q || !o || !lse || !lens || !q_strides || !k_strides || !v_strides || !o_strides || (room > 0 && (!k_cache || !v_cache))) return UA_ERR_NULL;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(o) || !aligned4(lens) || !swa_strides_ok(q_strides, false) ||
      !swa_strides_ok(k_strides, false) || !swa_strides_ok(v_strides, false) || !swa_strides_ok(o_strides, true))
    return UA_ERR_ALIGN;
  if (k_strides[1] > UA_SWA_MAX_TOKEN_STRIDE || v_strides[1] > UA_SWA_MAX_TOKEN_STRIDE) return UA_ERR_SHAPE;
  rc = check_device();
  if (rc != UA_OK) return rc;
  DecShape s = dec_shape(batch, n_tokens, n_heads, n_kv_heads, room, head_dim, left, sinks);
  DecParams p{};
  p.q = q; p.k = k_cache; p.v = v_cache; p.o = o; p.lse = lse; p.lens = lens;
  p.qs = {q_strides[0], q_strides[1], q_strides[2]};
  p.ks = {k_strides[0], k_strides[1], k_strides[2]};
  p.vs = {v_strides[0], v_strides[1], v_strides[2]};
  p.os = {o_strides[0], o_strides[1], o_strides[2]};
  p.n_tokens = n_tokens; p.n_heads = n_heads; p.n_kv_heads = n_kv_heads; p.group = n_heads / n_kv_heads; p.room = room;
  p.left = left < 0 ? kFar : (int)std::min<int64_t>(left, kFar);
  p.sinks = left < 0 ? 0 : (int)std::min<int64_t>(sinks, room);
  p.rows = n_tokens * p.group;
  p.n_tiles = s.row_tiles;
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
  p.by_parts = make_div(p.n_parts);
  const hipStream_t st = (hipStream_t)stream;
  const int64_t n = (int64_t)batch * n_kv_heads * p.n_tiles * p.n_parts;
  if (n > kSwaMaxGroups) return UA_ERR_SHAPE;
  if (dtype == UA_FP16) head_dim == 64 ? dec_launch<fp16, 64>(p, s.tiles, (unsigned)n, st) : dec_launch<fp16, 128>(p, s.tiles, (unsigned)n, st);
  else                  head_dim == 64 ? dec_launch<bf16, 64>(p, s.tiles, (unsigned)n, st) : dec_launch<bf16, 128>(p, s.tiles, (unsigned)n, st);
  if (hipGetLastError() != hipSuccess) return UA_ERR_LAUNCH;
  if (p.n_parts == 1) return UA_OK;
  return swa_merge(p.part_o, p.o_part, p.part_lse, p.lse_part, p.n_parts, o, p.os, lse, batch, n_heads, n_tokens, head_dim, dtype, st);
}
