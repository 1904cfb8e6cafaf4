// What joins results over shards of the keys, for the rows that sliding-window attention makes: bf16 and fp16, heads of 64 and 128.
// (merge.hip and reduce.hip do the same for bf16 heads of 128, in forms tuned to those.)
//
//   merge   LSE = log sum_p exp(lse_p),  O = sum_p exp(lse_p - LSE) O_p            contiguous parts
//   update  the same of two, strided, either of them fp32, the result too
//   sum     scale * sum_p G_p                                                      contiguous parts, or fp32 ones, into strided rows
//   delta   rowsum(dO O)
//
// 16 lanes a row, which read its statistics beside its data; sums in fp32, one rounding at the end; a part of weight 0 does not count, so that
// rows without keys may hold anything; NaN stays.  Bound: HBM, each row in and out once.  Measured, four parts of
// 268 MB in fp16: heads of 64, merge 279 us (4.8 TB/s), sum 244 (5.5), update in place 200 (4.0), delta 110 (4.9); heads of 128, 238, 231, 137 and 90.
#include <algorithm>
#include "swa.h"

namespace ua {

constexpr int kRowLanes = 16, kRowsGroup = 256 / kRowLanes;
template <int kD> struct RowPer { static constexpr int k = kD / kRowLanes; };        // elements of a lane: 8 or 4

template <class T, int kPer> __device__ __forceinline__ void row_load(float (&x)[kPer], const T* p) {
  typedef __attribute__((ext_vector_type(kPer))) T vec;
  const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
  for (int j = 0; j < kPer; ++j) x[j] = (float)v[j];
}
template <class T, int kPer> __device__ __forceinline__ void row_store(T* p, const float (&x)[kPer]) {
  typedef __attribute__((ext_vector_type(kPer))) T vec;
  vec v;
#pragma unroll
  for (int j = 0; j < kPer; ++j) v[j] = (T)x[j];
  *reinterpret_cast<vec*>(p) = v;
}
// of T or, wave-uniformly, of fp32
template <class T, int kPer> __device__ __forceinline__ void row_load(float (&x)[kPer], const void* base, int64_t at, bool f32) {
  if (f32) row_load(x, static_cast<const float*>(base) + at); else row_load(x, static_cast<const T*>(base) + at);
}
template <class T, int kPer> __device__ __forceinline__ void row_store(void* base, int64_t at, bool f32, const float (&x)[kPer]) {
  if (f32) row_store(static_cast<float*>(base) + at, x); else row_store(static_cast<T*>(base) + at, x);
}

struct RowsParams {
  const void* in[UA_MAX_PARTS];           // merge, sum: the parts; update: out, block; delta: o, dout
  const float* stat[UA_MAX_PARTS];        // merge: the parts' lse; update: lse, block lse
  void* out;
  float* out_stat;
  Strides3 is[2], ss[2], os, oss;         // update, delta: of `in` and `stat`; of the results
  int n_parts, n_rows, n_heads, seqlen;
  int in_f32[2], out_f32;
  float scale;
  Div by_heads, by_seq;
};
struct RowAt { int64_t b; int64_t s; int h; };
__device__ __forceinline__ int64_t offset(const RowAt& r, const Strides3& s) { return r.b * s.b + r.s * s.s + r.h * s.h; }
__device__ __forceinline__ RowAt row_at(const RowsParams& p, int row) {
  const int t = quotient(row, p.by_heads), b = quotient(t, p.by_seq);
  return {b, t - b * p.seqlen, row - t * p.n_heads};
}

template <class T, int kD>
__global__ __launch_bounds__(256) void rows_merge_kernel(const RowsParams p) {
  constexpr int kPer = RowPer<kD>::k;
  const int row = blockIdx.x * kRowsGroup + threadIdx.x / kRowLanes, lane = threadIdx.x % kRowLanes;
  if (row >= p.n_rows) return;
  const RowAt r = row_at(p, row);
  const int64_t at = (r.b * p.n_heads + r.h) * p.seqlen + r.s;
  static_assert(UA_MAX_PARTS <= kRowLanes, "a lane a part");
  float l = -INFINITY;
#pragma unroll
  for (int i = 0; i < UA_MAX_PARTS; ++i)                   // (the pointers are scalars: one after the other)
    if (i < p.n_parts && i == lane) l = p.stat[i][at];
  float top = l;
#pragma unroll
  for (int d = kRowLanes / 2; d; d /= 2) top = fmaxf(top, __shfl_xor(top, d));
  const float ref = top == -INFINITY ? 0.f : top, w = l == -INFINITY ? 0.f : fast_exp2((l - ref) * kLog2e);
  float total = w, acc[kPer] = {};
#pragma unroll
  for (int d = kRowLanes / 2; d; d /= 2) total += __shfl_xor(total, d);
  constexpr int kAhead = 4;                                // loads that follow one another (beyond the parts the last one again, at weight 0)
  for (int i0 = 0; i0 < p.n_parts; i0 += kAhead) {
    float x[kAhead][kPer];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) row_load(x[u], static_cast<const T*>(p.in[min(i0 + u, p.n_parts - 1)]) + (int64_t)row * kD + lane * kPer);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float f = __shfl(w, i0 + u, kRowLanes);        // (0 of lanes beyond the parts)
#pragma unroll
      for (int j = 0; j < kPer; ++j) acc[j] = f != 0.f ? fmaf(f, x[u][j], acc[j]) : acc[j];
    }
  }
  const bool any = total > 0.f || total != total;
  const float inv = any ? 1.f / total : 0.f;
#pragma unroll
  for (int j = 0; j < kPer; ++j) acc[j] *= inv;
  row_store(static_cast<T*>(p.out) + (int64_t)row * kD + lane * kPer, acc);
  if (lane == 0) p.out_stat[at] = any ? ref + __builtin_amdgcn_logf(total) * kLn2 : -INFINITY;
}

template <class T, int kD>
__global__ __launch_bounds__(256) void rows_update_kernel(const RowsParams p) {
  constexpr int kPer = RowPer<kD>::k;
  const int row = blockIdx.x * kRowsGroup + threadIdx.x / kRowLanes, lane = threadIdx.x % kRowLanes;
  if (row >= p.n_rows) return;
  const RowAt r = row_at(p, row);
  const float a = p.stat[0][offset(r, p.ss[0])], c = p.stat[1][offset(r, p.ss[1])];
  float x[kPer], y[kPer];
  row_load<T>(x, p.in[0], offset(r, p.is[0]) + lane * kPer, p.in_f32[0]);
  row_load<T>(y, p.in[1], offset(r, p.is[1]) + lane * kPer, p.in_f32[1]);
  const float top = fmaxf(a, c), ref = top == -INFINITY ? 0.f : top;
  const float ea = a == -INFINITY ? 0.f : fast_exp2((a - ref) * kLog2e), ec = c == -INFINITY ? 0.f : fast_exp2((c - ref) * kLog2e), total = ea + ec;
  const bool any = total > 0.f || total != total;
  const float inv = any ? 1.f / total : 0.f, wa = ea * inv, wc = ec * inv;
#pragma unroll
  for (int j = 0; j < kPer; ++j) x[j] = (wa != 0.f ? wa * x[j] : 0.f) + (wc != 0.f ? wc * y[j] : 0.f);
  row_store<T>(p.out, offset(r, p.os) + lane * kPer, p.out_f32, x);
  if (lane == 0) p.out_stat[offset(r, p.oss)] = any ? ref + __builtin_amdgcn_logf(total) * kLn2 : -INFINITY;
}

template <class T, int kD>
__global__ __launch_bounds__(256) void rows_sum_kernel(const RowsParams p) {
  constexpr int kPer = RowPer<kD>::k;
  const int row = blockIdx.x * kRowsGroup + threadIdx.x / kRowLanes, lane = threadIdx.x % kRowLanes;
  if (row >= p.n_rows) return;
  float acc[kPer] = {};
#pragma unroll 4
  for (int i = 0; i < p.n_parts; ++i) {
    float x[kPer];
    row_load<T>(x, p.in[i], (int64_t)row * kD + lane * kPer, p.in_f32[0]);
#pragma unroll
    for (int j = 0; j < kPer; ++j) acc[j] += x[j];
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) acc[j] *= p.scale;
  row_store(static_cast<T*>(p.out) + offset(row_at(p, row), p.os) + lane * kPer, acc);
}

template <class T, int kD>
__global__ __launch_bounds__(256) void rows_delta_kernel(const RowsParams p) {
  constexpr int kPer = RowPer<kD>::k;
  const int row = blockIdx.x * kRowsGroup + threadIdx.x / kRowLanes, lane = threadIdx.x % kRowLanes;
  if (row >= p.n_rows) return;
  const RowAt r = row_at(p, row);
  float x[kPer], y[kPer], sum = 0.f;
  row_load(x, static_cast<const T*>(p.in[0]) + offset(r, p.is[0]) + lane * kPer);
  row_load(y, static_cast<const T*>(p.in[1]) + offset(r, p.is[1]) + lane * kPer);
#pragma unroll
  for (int j = 0; j < kPer; ++j) sum = fmaf(x[j], y[j], sum);
#pragma unroll
  for (int d = kRowLanes / 2; d; d /= 2) sum += __shfl_xor(sum, d);
  if (lane == 0) p.out_stat[(r.b * p.n_heads + r.h) * p.seqlen + r.s] = sum;
}

static int rows_fill(RowsParams& p, int batch, int seqlen, int n_heads, int head_dim, int dtype) {
  if ((head_dim != 64 && head_dim != 128) || (dtype != UA_BF16 && dtype != UA_FP16)) return UA_ERR_UNSUPPORTED;
  if (batch < 0 || seqlen < 0 || n_heads <= 0) return UA_ERR_SHAPE;
  const int64_t tokens = (int64_t)batch * seqlen;
  if (tokens > INT32_MAX || tokens * n_heads > kSwaMaxGroups * kRowsGroup) return UA_ERR_SHAPE;         // (below 2^28: rows are counted in 32 bits)
  p.n_rows = (int)(tokens * n_heads); p.n_heads = n_heads; p.seqlen = seqlen;
  p.by_heads = make_div(n_heads);
  p.by_seq = make_div(std::max(seqlen, 1));
  return UA_OK;
}
// Rows of which every one begins on a boundary of a lane's vectors.
static bool rows_ok(const void* x, const int64_t* s, bool f32) {
  const int64_t q = f32 ? 4 : 8;
  return aligned16(x) && (!s || (s[0] % q == 0 && s[1] % q == 0 && s[2] % q == 0));
}
static Strides3 rows_strides(const int64_t* s) { return {s[0], s[1], s[2]}; }

template <class F>
static int rows_run(const RowsParams& p, int head_dim, int dtype, F kernel_of, void* stream) {
  const int rc = check_device();
  if (rc != UA_OK) return rc;
  auto go = [&](auto element, auto dim) {
    kernel_of(element, dim)<<<(p.n_rows + kRowsGroup - 1) / kRowsGroup, 256, 0, (hipStream_t)stream>>>(p);
  };
  auto by_dim = [&](auto element) {
    if (head_dim == 64) go(element, std::integral_constant<int, 64>{});
    else                go(element, std::integral_constant<int, 128>{});
  };
  if (dtype == UA_FP16) by_dim(fp16(0)); else by_dim(bf16(0.f));
  return hipGetLastError() == hipSuccess ? UA_OK : UA_ERR_LAUNCH;
}

}  // namespace ua

extern "C" int ua_rows_merge(const void* const* o_parts, const float* const* lse_parts, int n_parts, void* o, float* lse, int batch, int seqlen, int n_heads,
                             int head_dim, int dtype, void* stream) {
  using namespace ua;
  RowsParams p{};
  const int rc = rows_fill(p, batch, seqlen, n_heads, head_dim, dtype);
  if (rc != UA_OK) return rc;
  if (n_parts < 1 || n_parts > UA_MAX_PARTS) return UA_ERR_UNSUPPORTED;
  if (p.n_rows == 0) return UA_OK;
  if (!o_parts || !lse_parts || !o || !lse) return UA_ERR_NULL;
  if (!aligned16(o)) return UA_ERR_ALIGN;
  for (int i = 0; i < n_parts; ++i) {
    if (!o_parts[i] || !lse_parts[i]) return UA_ERR_NULL;
    if (!aligned16(o_parts[i])) return UA_ERR_ALIGN;
    p.in[i] = o_parts[i];
    p.stat[i] = lse_parts[i];
  }
  p.out = o; p.out_stat = lse; p.n_parts = n_parts;
  return rows_run(p, head_dim, dtype, [](auto e, auto d) { return rows_merge_kernel<decltype(e), decltype(d)::value>; }, stream);
}

extern "C" int ua_rows_update(const void* out, const float* lse, const void* block_out, const float* block_lse, void* new_out, float* new_lse, int batch,
                              int n_rows, int n_heads, int head_dim, int dtype, int out_is_fp32, int block_is_fp32, int new_is_fp32,
                              const int64_t* out_strides, const int64_t* lse_strides, const int64_t* block_out_strides, const int64_t* block_lse_strides,
                              const int64_t* new_out_strides, const int64_t* new_lse_strides, void* stream) {
  using namespace ua;
  RowsParams p{};
  const int rc = rows_fill(p, batch, n_rows, n_heads, head_dim, dtype);
  if (rc != UA_OK) return rc;
  if (p.n_rows == 0) return UA_OK;
  if (!out || !lse || !block_out || !block_lse || !new_out || !new_lse) return UA_ERR_NULL;
  for (const int64_t* s : {out_strides, lse_strides, block_out_strides, block_lse_strides, new_out_strides, new_lse_strides})
    if (!s) return UA_ERR_NULL;
  if (!rows_ok(out, out_strides, out_is_fp32) || !rows_ok(block_out, block_out_strides, block_is_fp32) || !rows_ok(new_out, new_out_strides, new_is_fp32))
    return UA_ERR_ALIGN;
  // in place only element for element: other lanes read their rows meanwhile
  if (new_out == out && (!out_is_fp32 != !new_is_fp32 || !std::equal(out_strides, out_strides + 3, new_out_strides))) return UA_ERR_SHAPE;
  if (new_lse == lse && !std::equal(lse_strides, lse_strides + 3, new_lse_strides)) return UA_ERR_SHAPE;
  p.in[0] = out; p.in[1] = block_out; p.stat[0] = lse; p.stat[1] = block_lse; p.out = new_out; p.out_stat = new_lse;
  p.is[0] = rows_strides(out_strides); p.is[1] = rows_strides(block_out_strides);
  p.ss[0] = rows_strides(lse_strides); p.ss[1] = rows_strides(block_lse_strides);
  p.os = rows_strides(new_out_strides); p.oss = rows_strides(new_lse_strides);
  p.in_f32[0] = out_is_fp32; p.in_f32[1] = block_is_fp32; p.out_f32 = new_is_fp32;
  return rows_run(p, head_dim, dtype, [](auto e, auto d) { return rows_update_kernel<decltype(e), decltype(d)::value>; }, stream);
}

extern "C" int ua_rows_sum(const void* const* parts, int n_parts, int parts_fp32, void* out, int batch, int seqlen, int n_heads, int head_dim, int dtype,
                           const int64_t* out_strides, float scale, void* stream) {
  using namespace ua;
  RowsParams p{};
  const int rc = rows_fill(p, batch, seqlen, n_heads, head_dim, dtype);
  if (rc != UA_OK) return rc;
  if (n_parts < 1 || n_parts > UA_MAX_PARTS) return UA_ERR_UNSUPPORTED;
  if (p.n_rows == 0) return UA_OK;
  if (!parts || !out || !out_strides) return UA_ERR_NULL;
  if (!rows_ok(out, out_strides, false)) return UA_ERR_ALIGN;
  for (int i = 0; i < n_parts; ++i) {
    if (!parts[i]) return UA_ERR_NULL;
    if (!aligned16(parts[i])) return UA_ERR_ALIGN;
    p.in[i] = parts[i];
  }
  p.out = out; p.os = rows_strides(out_strides); p.n_parts = n_parts; p.in_f32[0] = parts_fp32; p.scale = scale;
  return rows_run(p, head_dim, dtype, [](auto e, auto d) { return rows_sum_kernel<decltype(e), decltype(d)::value>; }, stream);
}

extern "C" int ua_rows_delta(const void* o, const void* dout, float* delta, int batch, int seqlen_q, int n_heads, int head_dim, int dtype,
                             const int64_t* o_strides, const int64_t* do_strides, void* stream) {
  using namespace ua;
  RowsParams p{};
  const int rc = rows_fill(p, batch, seqlen_q, n_heads, head_dim, dtype);
  if (rc != UA_OK) return rc;
  if (p.n_rows == 0) return UA_OK;
  if (!o || !dout || !delta || !o_strides || !do_strides) return UA_ERR_NULL;
  if (!rows_ok(o, o_strides, false) || !rows_ok(dout, do_strides, false)) return UA_ERR_ALIGN;
  p.in[0] = o; p.in[1] = dout; p.out_stat = delta;
  p.is[0] = rows_strides(o_strides); p.is[1] = rows_strides(do_strides);
  return rows_run(p, head_dim, dtype, [](auto e, auto d) { return rows_delta_kernel<decltype(e), decltype(d)::value>; }, stream);
}
