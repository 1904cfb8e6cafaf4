// Rotary positions: pair i of the first `rotary_dim` entries of every head is turned by the angle position * freqs[i],
//   (a, b) -> scale * (a cos - b sin, b cos + a sin),
// with pairs (x[i], x[i + rotary_dim / 2]) or, interleaved, (x[2i], x[2i + 1]); the rest of the head passes through.  The
// gradient is the turn by the negative angle with the same scale.  The appending forms also send K, rotated, and V to
// their places in a cache, contiguous or in pages.
//
// Bound: HBM, each row in and out once.  The angles are not read from a table: a workgroup makes the cosines and sines of its tokens once, in
// LDS, and all heads of a token, of Q and of K, use them.
#include <algorithm>
#include <type_traits>
#include "paged.h"

namespace ua {

typedef _Float16 fp16;

constexpr int kRopeThreads = 256;
constexpr int kRopeAngles = 512;           // pairs of all of a workgroup's tokens (a head of 256 has up to 128)
constexpr int kRopeMaxTokens = 16;
constexpr int kRopeAhead = 4;              // items of a thread whose loads are in flight together

// One of the tensors that a call goes through: x [batch, tokens, heads, head_dim] to y, turned or (kRotate = 0) as it is.  An item is
// one or two vectors of a head: a pair of them that is turned, or two neighbours that pass through.
struct RopeTensor {
  const void* x; void* y;
  Strides3 xs, ys;
  int rotate, cached;        // cached: y's row is the token's position, [0, room), not its index (in pages: ys are the strides of page, slot and head)
  int items;                 // of a token, all heads
  Div by_head, by_token;     // items of a head, of a token
};
struct RopeParams {
  RopeTensor t[3];
  const double* freqs;
  const int32_t* pos32; const int64_t* pos64; const int32_t* lens;       // at most one of them
  int64_t pos_b, pos_s, start;
  int n_tokens, seqlen, tokens_per_group, n_half, head_vecs, room;
  float scale, sign;         // of the angle: -1 turns back
  Div by_seq;
};
struct PagedRopeParams : RopeParams {
  PagedSteps steps;
  PagedTable pages;
  Div by_lines;              // of trees: workgroups of a sequence
};

__device__ __forceinline__ int64_t rope_position(const RopeParams& p, int b, int s) {
  if (p.pos64) return p.pos64[b * p.pos_b + s * p.pos_s];
  if (p.pos32) return p.pos32[b * p.pos_b + s * p.pos_s];
  if (p.lens) return (int64_t)p.lens[b] - p.seqlen + s;
  return p.start + s;
}

// cos and sin of position * freq.  The angle in turns is a product in twice 64 bits, of which only the part behind the point is
// used: far positions, up to UA_ROPE_MAX_POSITION where 64 bits hold them, lose nothing (position 2^31 with one rounding in 64 bits is 5e-7 off, as much as a cosine in 32 bits has).
__device__ __forceinline__ void rope_angle(int64_t pos, double freq, float& c, float& s) {
#pragma clang fp contract(off)         // (turns - rint(turns) as one fma would count `rest` twice)
  constexpr double kHi = 0.15915494309189535, kLo = -9.839338337591e-18;       // 1 / (2 pi) = kHi + kLo
  const double f = freq * kHi, f_lo = fma(freq, kHi, -f) + freq * kLo;
  const double p = (double)pos, turns = p * f, rest = fma(p, f, -turns) + p * f_lo;
  const float half_turns = 2.f * (float)((turns - rint(turns)) + rest);
  sincospif(half_turns, &s, &c);
}

template <class T, int kV> __device__ __forceinline__ void rope_load(T (&d)[kV], const T* p) {
  typedef __attribute__((ext_vector_type(kV))) T vec;
  if constexpr (kV == 1) d[0] = *p;
  else {
    const vec x = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int j = 0; j < kV; ++j) d[j] = x[j];
  }
}
// kStream: results that are more than the caches hold go past them (2 x 8192 tokens, 40 heads of 128, 168 MB: 70.1 us, past them 54.5; 42 MB
// 16.5 either way).
constexpr int64_t kRopeStreamBytes = int64_t(128) << 20;
template <class T, int kV, bool kStream> __device__ __forceinline__ void rope_store(T* p, const T (&d)[kV]) {
  typedef __attribute__((ext_vector_type(kV))) T vec;
  if constexpr (kV == 1) *p = d[0];
  else {
    vec x;
#pragma unroll
    for (int j = 0; j < kV; ++j) x[j] = d[j];
    if constexpr (kStream) __builtin_nontemporal_store(x, reinterpret_cast<vec*>(p)); else *reinterpret_cast<vec*>(p) = x;
  }
}

// Two ways through a head, by what its layout allows:
//   kPairs   two vectors of kV entries and their partners, rotary_dim / 2 apart (kV divides that); interleaved only as single entries;
//   kBeside  interleaved: one vector holds kV / 2 pairs (2 x 8192 tokens, 16 heads of 128, 20 entries turned: as pairs of two vectors 31.5 us, so 23.5).
enum RopeWay { kPairs, kBeside };
// A workgroup goes through the tensors one after the other, or, where there are few tokens, takes one of them (blockIdx.y): which one is
// then a scalar either way.
template <class T, int kV, RopeWay kWay, bool kInterleaved, bool kStream, class Params>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(const Params p) {
  static_assert(kWay == kPairs ? !kInterleaved || kV == 1 : kInterleaved && kV > 1, "ways");
  constexpr bool kPaged = std::is_same_v<Params, PagedRopeParams>;
  __shared__ __attribute__((aligned(16))) float cosine[kRopeAngles], sine[kRopeAngles];
  __shared__ int64_t position[kRopeMaxTokens];             // in pages: of the cache's row, page * 2^32 + slot; -1 none, -2 no token
  __shared__ int depth[kPaged ? kTreeMost : 1], exits[kPaged ? kTreeMost : 1];
  int first = blockIdx.x * p.tokens_per_group, n_here = min(p.tokens_per_group, p.n_tokens - first), parent = -1;
  if constexpr (kPaged) {
    if (p.steps.parents) {                                 // a workgroup's tokens are of one sequence
      const int b = quotient(blockIdx.x, p.by_lines), s = (blockIdx.x - b * p.by_lines.d) * p.tokens_per_group;
      first = b * p.seqlen + s;
      n_here = min(p.tokens_per_group, p.seqlen - s);
      parent = parent_of(p.steps, b, tree_token(p.steps));
    }
  }
  const int begin = gridDim.y > 1 ? blockIdx.y : 0, end = gridDim.y > 1 ? begin + 1 : 3;
  bool made = false;
  for (int which = begin; which < end; ++which) {
    const RopeTensor& x = p.t[which];
    const int n = n_here * x.items, n_turned = x.rotate ? p.n_half / kV : 0, n_pairs = x.rotate ? p.n_half : 0;
    for (int i0 = 0; i0 < n; i0 += kRopeThreads * kRopeAhead) {
      T a[kRopeAhead][kV], b2[kRopeAhead][kV];
      T* to[kRopeAhead];
      int token[kRopeAhead], angle[kRopeAhead], second[kRopeAhead];    // kPairs: first angle, -1 passes through; entries to the second vector, 0 none
#pragma unroll
      for (int u = 0; u < kRopeAhead; ++u) {
        const int i = i0 + u * kRopeThreads + threadIdx.x;
        to[u] = nullptr;
        if (i >= n) continue;
        const int t = quotient(i, x.by_token), r = i - t * x.items, h = quotient(r, x.by_head), item = r - h * x.by_head.d;
        const int b = quotient(first + t, p.by_seq), s = first + t - b * p.seqlen;
        token[u] = t;
        const T* head = static_cast<const T*>(x.x) + b * x.xs.b + s * x.xs.s + h * x.xs.h;
        int at = item;                                      // the (first) vector
        if constexpr (kWay == kPairs) {
          if (item < n_turned) {
            angle[u] = t * p.n_half + item * kV;
            if (kInterleaved) at = 2 * item;
            second[u] = kInterleaved ? kV : p.n_half;
          } else {
            angle[u] = -1;
            at = 2 * item;                                  // (2 * n_turned vectors are turned)
            second[u] = at + 1 < p.head_vecs ? kV : 0;
          }
        } else {
          angle[u] = at * kV;                               // the first entry
        }
        to[u] = static_cast<T*>(x.y) + (kPaged && x.cached ? 0 : b * x.ys.b) + (x.cached ? 0 : s * x.ys.s) + h * x.ys.h + at * kV;
        rope_load<T, kV>(a[u], head + at * kV);
        if (kWay == kPairs && second[u]) rope_load<T, kV>(b2[u], head + at * kV + second[u]);
      }
      if (!made) {                                        // workgroup-uniform; the first loads are on their way meanwhile
        made = true;
        if constexpr (kPaged) {
          static_assert(kRopeThreads == kTreeThreads, "a token a thread");
          if (p.steps.parents) tree_depths(p.steps, parent, depth, exits);
        }
        for (int i = threadIdx.x; i < n_here * p.n_half; i += kRopeThreads) {
          const int t = i / p.n_half, b = quotient(first + t, p.by_seq), s = first + t - b * p.seqlen;
          float c, sn;
          int64_t pos;
          if constexpr (kPaged) pos = step_of(p.steps, b).base + (p.steps.parents ? depth[s] : s); else pos = rope_position(p, b, s);
          rope_angle(pos, p.freqs[i - t * p.n_half], c, sn);
          cosine[i] = c * p.scale;
          sine[i] = sn * p.scale * p.sign;
        }
        if (threadIdx.x < n_here) {
          const int b = quotient(first + threadIdx.x, p.by_seq), s = first + threadIdx.x - b * p.seqlen;
          if constexpr (kPaged) {
            const StepOf of = step_of(p.steps, b);
            const int row = of.base + s;
            int64_t at = s < of.n ? -1 : -2;
            if (s < of.n && row >= 0 && row < p.pages.room) {
              const int i = quotient(row, p.pages.by_page), page = p.pages.table[b * p.pages.stride + i];
              if (page >= 0 && page < p.pages.n_pages) at = (int64_t)page << 32 | (row - i * p.pages.page);
            }
            position[threadIdx.x] = at;
          } else {
            position[threadIdx.x] = rope_position(p, b, s);
          }
        }
        __syncthreads();
      }
#pragma unroll
      for (int u = 0; u < kRopeAhead; ++u) {
        if (!to[u]) continue;
        if (x.cached) {
          const int64_t row = position[token[u]];
          if constexpr (kPaged) {
            if (row < 0) continue;
            to[u] += (row >> 32) * x.ys.b + (uint32_t)row * x.ys.s;
          } else {
            if (row < 0 || row >= p.room) continue;
            to[u] += row * x.ys.s;
          }
        }
        if constexpr (kWay == kPairs) {
          if (angle[u] >= 0)
#pragma unroll
            for (int j = 0; j < kV; ++j) {
              const float c = cosine[angle[u] + j], s = sine[angle[u] + j], g = (float)a[u][j], e = (float)b2[u][j];
              a[u][j] = (T)(g * c - e * s);
              b2[u][j] = (T)(e * c + g * s);
            }
        } else {
          const int pair0 = angle[u] / 2, base = token[u] * p.n_half;
#pragma unroll
          for (int j = 0; j < kV / 2; ++j) {
            if (pair0 + j >= n_pairs) continue;
            const float c = cosine[base + pair0 + j], s = sine[base + pair0 + j], g = (float)a[u][2 * j], e = (float)a[u][2 * j + 1];
            a[u][2 * j] = (T)(g * c - e * s);
            a[u][2 * j + 1] = (T)(e * c + g * s);
          }
        }
        if constexpr (kPaged) {
          if (!x.cached && position[token[u]] == -2) {
#pragma unroll
            for (int j = 0; j < kV; ++j) a[u][j] = b2[u][j] = (T)0.f;
          }
        }
        rope_store<T, kV, kStream>(to[u], a[u]);
        if (kWay == kPairs && second[u]) rope_store<T, kV, kStream>(to[u] + second[u], b2[u]);
      }
    }
  }
}

template <class T, int kV, class P>
static void rope_launch(const P& p, bool interleaved, bool stream, dim3 groups, hipStream_t st) {
  constexpr bool kWide = kV * sizeof(T) == 16;
  auto run = [&](auto kernel) { kernel<<<groups, kRopeThreads, 0, st>>>(p); };
  if constexpr (kV == 1) interleaved ? run(rope_kernel<T, 1, kPairs, true, false, P>) : run(rope_kernel<T, 1, kPairs, false, false, P>);
  else if (interleaved)  kWide && stream ? run(rope_kernel<T, kV, kBeside, true, kWide, P>) : run(rope_kernel<T, kV, kBeside, true, false, P>);
  else                   kWide && stream ? run(rope_kernel<T, kV, kPairs, false, kWide, P>) : run(rope_kernel<T, kV, kPairs, false, false, P>);
}

struct RopeShape { int batch, seqlen, head_dim, rotary_dim, dtype; };

// The widest vector (in elements) that the tensors allow and that divides `unit` and the head.
static int rope_vector(const RopeShape& s, const RopeTensor* t, const int* heads, int n, int unit) {
  const int size = s.dtype == UA_FP32 ? 4 : 2;
  for (int v = 16 / size; v > 1; v /= 2) {
    bool ok = unit % v == 0 && s.head_dim % v == 0;
    for (int i = 0; i < n && ok; ++i) {
      if (!heads[i]) continue;
      const int64_t all[6] = {t[i].xs.b, t[i].xs.s, t[i].xs.h, t[i].ys.b, t[i].ys.s, t[i].ys.h};
      for (const int64_t x : all) ok = ok && x % v == 0;
      ok = ok && reinterpret_cast<uintptr_t>(t[i].x) % (v * size) == 0 && reinterpret_cast<uintptr_t>(t[i].y) % (v * size) == 0;
    }
    if (ok) return v;
  }
  return 1;
}

template <class P>
static int rope_run(P& p, const RopeShape& s, const int* heads, int n_tensors, int interleaved, hipStream_t st) {
  constexpr bool kPaged = std::is_same_v<P, PagedRopeParams>;
  const int size = s.dtype == UA_FP32 ? 4 : 2;
  p.n_half = s.rotary_dim / 2;
  const int v = rope_vector(s, p.t, heads, n_tensors, interleaved ? s.head_dim : p.n_half);
  const RopeWay way = interleaved && v > 1 ? kBeside : kPairs;
  p.head_vecs = s.head_dim / v;
  p.seqlen = s.seqlen;
  int64_t n_items = 0, bytes = 0;
  for (int i = 0; i < 3; ++i) {
    RopeTensor& t = p.t[i];
    if (i >= n_tensors || !heads[i]) { t.items = 0; t.by_head = t.by_token = make_div(1); continue; }
    // what passes through is there already (but not the zeros of tokens that are none)
    bool zeros = false;
    if constexpr (kPaged) zeros = p.steps.n_new != nullptr;
    const bool same = !zeros && t.rotate && !t.cached && t.x == t.y && t.xs.b == t.ys.b && t.xs.s == t.ys.s && t.xs.h == t.ys.h;
    const int turned = t.rotate ? p.n_half / v : 0;
    const int per_head = way == kPairs ? turned + (same ? 0 : (p.head_vecs - 2 * turned + 1) / 2) : same ? (s.rotary_dim + v - 1) / v : p.head_vecs;
    if ((int64_t)per_head * heads[i] * kRopeMaxTokens > INT32_MAX) return UA_ERR_SHAPE;
    t.items = per_head * heads[i];
    bytes += (int64_t)s.batch * s.seqlen * heads[i] * s.head_dim * size;
    t.by_head = make_div(per_head);
    t.by_token = make_div(t.items);
    n_items += t.items;
  }
  if ((int64_t)s.batch * s.seqlen > INT32_MAX) return UA_ERR_SHAPE;
  p.n_tokens = s.batch * s.seqlen;
  if (p.n_tokens == 0 || n_items == 0) return UA_OK;
  const bool stream = bytes > kRopeStreamBytes;
  p.by_seq = make_div(s.seqlen);
  // Tokens of a workgroup: as many as give each thread an angle, while that leaves four workgroups a CU; in pages, whose tokens' lengths, trees and table entries each
  // workgroup reads first, one, times the tensors (one token a workgroup and three or four, us: 32 trees of 25 tokens, 14 + 4 heads of 64, 8.2 and 6.4; 3
  // of 256, 8 + 16 of 128, 13.4 and 7.2; 16 chains of 64, 32 + 16 of 128, 11.4 and 8.8; 64 trees of 64 by tensors 21.8, all three 20.1).
  p.tokens_per_group = std::max(1, std::min({kRopeAngles / p.n_half, kRopeMaxTokens, (kRopeThreads + p.n_half - 1) / p.n_half,
                                             p.n_tokens / ((kPaged ? 1 : 4) * kCus)}));
  uint32_t lines = (uint32_t)(((int64_t)p.n_tokens + p.tokens_per_group - 1) / p.tokens_per_group);
  if constexpr (kPaged) {
    if (p.steps.parents) {
      const int of_one = (s.seqlen + p.tokens_per_group - 1) / p.tokens_per_group;
      if ((int64_t)s.batch * of_one > INT32_MAX) return UA_ERR_SHAPE;
      p.by_lines = make_div(of_one);
      lines = (uint32_t)(s.batch * of_one);
    }
  }
  if (lines > UINT32_MAX / kRopeThreads) return UA_ERR_SHAPE;              // (a launch counts its threads in 32 bits)
  const dim3 groups(lines, lines <= (kPaged ? 2 : 4) * kCus ? n_tensors : 1);
  const int rc = check_device();
  if (rc != UA_OK) return rc;
  auto launch = [&](auto element) {
    typedef decltype(element) T;
    if constexpr (sizeof(T) == 2) {
      if (v == 8) return rope_launch<T, 8>(p, interleaved, stream, groups, st);
    }
    if (v == 4) rope_launch<T, 4>(p, interleaved, stream, groups, st);
    else if (v == 2) rope_launch<T, 2>(p, interleaved, stream, groups, st);
    else rope_launch<T, 1>(p, interleaved, stream, groups, st);
  };
  if (s.dtype == UA_FP32) launch(0.f);
  else if (s.dtype == UA_FP16) launch(fp16(0));
  else launch(bf16(0.f));
  return hipGetLastError() == hipSuccess ? UA_OK : UA_ERR_LAUNCH;
}

static int rope_check(const RopeShape& s, int n_heads, int n_kv_heads, float scale) {
  if (s.batch < 0 || s.seqlen < 0 || n_heads < 0 || n_kv_heads < 0 || s.head_dim <= 0) return UA_ERR_SHAPE;
  if (s.rotary_dim <= 0 || s.rotary_dim % 2 || s.rotary_dim > s.head_dim) return UA_ERR_SHAPE;
  if (s.head_dim > UA_ROPE_MAX_DIM || s.dtype < UA_BF16 || s.dtype > UA_FP32 || !(scale > 0.f)) return UA_ERR_UNSUPPORTED;
  return UA_OK;
}
static_assert(UA_ROPE_MAX_DIM / 2 <= kRopeAngles, "the angles of one token fit");
static Strides3 strides_of(const int64_t* s) { return {s[0], s[1], s[2]}; }

}  // namespace ua

extern "C" int ua_rope(const void* q, const void* k, void* q_out, void* k_out, const double* freqs, const void* positions, int positions_64,
                       int64_t position_stride_b, int64_t position_stride_s, int64_t start, int batch, int seqlen, int n_heads, int n_kv_heads,
                       int head_dim, int rotary_dim, int dtype, int interleaved, int inverse, float scale, const int64_t* q_strides,
                       const int64_t* k_strides, const int64_t* q_out_strides, const int64_t* k_out_strides, void* stream) {
  using namespace ua;
  const RopeShape s{batch, seqlen, head_dim, rotary_dim, dtype};
  const int rc = rope_check(s, n_heads, n_kv_heads, scale);
  if (rc != UA_OK) return rc;
  if (!positions && (start > UA_ROPE_MAX_POSITION - seqlen || start < -UA_ROPE_MAX_POSITION)) return UA_ERR_SHAPE;
  if ((int64_t)batch * seqlen == 0) return UA_OK;
  if (!freqs || (n_heads && (!q || !q_out || !q_strides || !q_out_strides)) || (n_kv_heads && (!k || !k_out || !k_strides || !k_out_strides)))
    return UA_ERR_NULL;
  RopeParams p{};
  const int heads[2] = {n_heads, n_kv_heads};
  if (n_heads) { p.t[0] = {q, q_out, strides_of(q_strides), strides_of(q_out_strides), 1, 0, 0, {}, {}}; }
  if (n_kv_heads) { p.t[1] = {k, k_out, strides_of(k_strides), strides_of(k_out_strides), 1, 0, 0, {}, {}}; }
  p.freqs = freqs;
  p.pos64 = positions_64 ? (const int64_t*)positions : nullptr;
  p.pos32 = positions_64 ? nullptr : (const int32_t*)positions;
  p.pos_b = position_stride_b; p.pos_s = position_stride_s;
  p.start = start;
  p.scale = scale;
  p.sign = inverse ? -1.f : 1.f;
  return rope_run(p, s, heads, 2, interleaved, (hipStream_t)stream);
}

extern "C" int ua_rope_append(const void* q, const void* k, const void* v, void* q_out, void* k_cache, void* v_cache, const double* freqs,
                              const int32_t* lens, int batch, int n_new, int n_heads, int n_kv_heads, int room, int head_dim, int rotary_dim,
                              int dtype, int interleaved, float scale, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                              const int64_t* q_out_strides, const int64_t* k_cache_strides, const int64_t* v_cache_strides, void* stream) {
  using namespace ua;
  const RopeShape s{batch, n_new, head_dim, rotary_dim, dtype};
  const int rc = rope_check(s, n_heads, n_kv_heads, scale);
  if (rc != UA_OK) return rc;
  if (room < 0) return UA_ERR_SHAPE;
  if ((int64_t)batch * n_new == 0) return UA_OK;
  if (room == 0) n_kv_heads = 0;                     // (no row to write: the cache may be NULL)
  if (!freqs || !lens || (n_heads && (!q || !q_out || !q_strides || !q_out_strides)) ||
      (n_kv_heads && (!k || !v || !k_cache || !v_cache || !k_strides || !v_strides || !k_cache_strides || !v_cache_strides)))
    return UA_ERR_NULL;
  RopeParams p{};
  const int heads[3] = {n_heads, n_kv_heads, n_kv_heads};
  if (n_heads) p.t[0] = {q, q_out, strides_of(q_strides), strides_of(q_out_strides), 1, 0, 0, {}, {}};
  if (n_kv_heads) {
    p.t[1] = {k, k_cache, strides_of(k_strides), strides_of(k_cache_strides), 1, 1, 0, {}, {}};
    p.t[2] = {v, v_cache, strides_of(v_strides), strides_of(v_cache_strides), 0, 1, 0, {}, {}};
  }
  p.freqs = freqs;
  p.lens = lens;
  p.room = room;
  p.scale = scale;
  p.sign = 1.f;
  return rope_run(p, s, heads, 3, interleaved, (hipStream_t)stream);
}

extern "C" int ua_paged_append(const void* q, const void* k, const void* v, void* q_out, void* k_pages, void* v_pages, const double* freqs,
                               const int32_t* table, const int32_t* lens, const int32_t* n_new, const int32_t* parents, int batch, int n_tokens, int n_heads,
                               int n_kv_heads, int n_pages, int page, int max_pages, int head_dim, int rotary_dim, int dtype, int interleaved, float scale,
                               int64_t table_stride, int64_t parents_stride, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                               const int64_t* q_out_strides, const int64_t* k_page_strides, const int64_t* v_page_strides, void* stream) {
  using namespace ua;
  const RopeShape s{batch, n_tokens, head_dim, rotary_dim, dtype};
  int rc = rope_check(s, n_heads, n_kv_heads, scale);
  if (rc != UA_OK) return rc;
  rc = paged_check(batch, n_tokens, n_kv_heads, n_pages, page, max_pages, table_stride, parents, parents_stride);
  if (rc != UA_OK) return rc;
  if ((int64_t)batch * n_tokens == 0) return UA_OK;
  if (n_pages == 0 || max_pages == 0) n_kv_heads = 0;      // (no row to write: the pools may be NULL)
  if (!freqs || !lens || (n_heads && (!q || !q_out || !q_strides || !q_out_strides)) ||
      (n_kv_heads && (!table || !k || !v || !k_pages || !v_pages || !k_strides || !v_strides || !k_page_strides || !v_page_strides)))
    return UA_ERR_NULL;
  if (!aligned4(table) || !aligned4(lens) || !aligned4(n_new) || !aligned4(parents)) return UA_ERR_ALIGN;
  PagedRopeParams p{};
  const int heads[3] = {n_heads, n_kv_heads, n_kv_heads};
  if (n_heads) p.t[0] = {q, q_out, strides_of(q_strides), strides_of(q_out_strides), 1, 0, 0, {}, {}};
  if (n_kv_heads) {
    p.t[1] = {k, k_pages, strides_of(k_strides), strides_of(k_page_strides), 1, 1, 0, {}, {}};
    p.t[2] = {v, v_pages, strides_of(v_strides), strides_of(v_page_strides), 0, 1, 0, {}, {}};
  }
  p.freqs = freqs;
  p.scale = scale;
  p.sign = 1.f;
  p.steps = {lens, n_new, parents, parents_stride, n_tokens};
  p.pages = {table, table_stride, n_pages, page, n_kv_heads ? paged_room(page, max_pages) : 0, make_div(page)};
  return rope_run(p, s, heads, 3, interleaved, (hipStream_t)stream);
}
