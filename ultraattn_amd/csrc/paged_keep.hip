// The rows of a tree's accepted branch moved together in a paged cache: row base + i of every layer's K and V takes what row base + path[i] holds, i < n_kept.
//
// A branch's tokens come in rising order, so path[i] >= i, and a row is read before it is written if rows are taken in order: a thread has one column of 16 bytes
// of one head and takes all rows of the branch, several of whose loads are in flight together, so that no thread waits for another and the move can be
// in place.  Bound: the launch, and two dependent reads (table, row); the rows, in and out once, are few.
#include <algorithm>
#include "paged.h"

namespace ua {

constexpr int kKeepThreads = 256, kKeepRows = 256, kKeepAhead = 8;       // rows of which places are held in LDS, and whose loads of a column are in flight

struct KeepPool { char* rows; int64_t layer, page, slot, head; };       // strides in bytes
struct KeepParams {
  KeepPool k, v;
  PagedSteps steps;
  PagedTable pages;
  const int32_t *path, *n_kept;
  int64_t path_stride;
  int n_path, n_heads, columns;                     // columns: of a head
  Div by_columns;
};

template <class Vec>
__global__ __launch_bounds__(kKeepThreads) void paged_keep_kernel(const KeepParams p) {
  __shared__ int from_page[kKeepRows], from_slot[kKeepRows], to_page[kKeepRows], to_slot[kKeepRows];
  const int b = blockIdx.y, layer = blockIdx.z, column = blockIdx.x * kKeepThreads + threadIdx.x;
  const StepOf of = step_of(p.steps, b);
  const int n = min(min(max(p.n_kept[b], 0), p.n_path), of.n);
  const int per_pool = p.n_heads * p.columns, at = column % per_pool, h = quotient(at, p.by_columns);
  const KeepPool& pool = column < per_pool ? p.k : p.v;
  char* const mine = pool.rows + layer * pool.layer + h * pool.head + (int64_t)(at - h * p.columns) * sizeof(Vec);
  for (int i0 = 0; i0 < n; i0 += kKeepRows) {
    const int rows = min(kKeepRows, n - i0);
    if (i0) __syncthreads();
    if (threadIdx.x < rows) {
      const int i = i0 + threadIdx.x, token = p.path[b * p.path_stride + i], to = of.base + i, from = of.base + min(max(token, 0), of.n);
      int page = -1, source = -1, slot = 0, source_slot = 0;
      if (token > i && token < of.n && to >= 0 && from < p.pages.room) {          // (token == i: it is there)
        const int32_t* const line = p.pages.table + b * p.pages.stride;
        const int x = quotient(to, p.pages.by_page), y = quotient(from, p.pages.by_page);
        page = line[x];
        source = line[y];
        slot = to - x * p.pages.page;
        source_slot = from - y * p.pages.page;
        if (page >= p.pages.n_pages || source < 0 || source >= p.pages.n_pages) page = -1;
      }
      from_page[threadIdx.x] = source;
      from_slot[threadIdx.x] = source_slot;
      to_page[threadIdx.x] = page;
      to_slot[threadIdx.x] = slot;
    }
    __syncthreads();
    if (column < 2 * per_pool) {
      for (int r0 = 0; r0 < rows; r0 += kKeepAhead) {
        Vec x[kKeepAhead];
#pragma unroll
        for (int u = 0; u < kKeepAhead; ++u) {
          const int r = r0 + u;
          if (r < rows && to_page[r] >= 0) x[u] = *reinterpret_cast<const Vec*>(mine + from_page[r] * pool.page + from_slot[r] * pool.slot);
        }
#pragma unroll
        for (int u = 0; u < kKeepAhead; ++u) {
          const int r = r0 + u;
          if (r < rows && to_page[r] >= 0) *reinterpret_cast<Vec*>(mine + to_page[r] * pool.page + to_slot[r] * pool.slot) = x[u];
        }
      }
    }
  }
}

}  // namespace ua

extern "C" int ua_paged_keep(void* k_pages, void* v_pages, const int32_t* table, const int32_t* lens, const int32_t* n_new, const int32_t* path,
                             const int32_t* n_kept, int layers, int batch, int n_tokens, int n_path, int n_kv_heads, int n_pages, int page, int max_pages,
                             int head_dim, int dtype, int64_t table_stride, int64_t path_stride, const int64_t* k_page_strides, const int64_t* v_page_strides,
                             void* stream) {
  using namespace ua;
  int rc = paged_check(batch, n_tokens, n_kv_heads, n_pages, page, max_pages, table_stride, nullptr, 0);
  if (rc != UA_OK) return rc;
  if (layers < 0 || n_path < 0 || head_dim <= 0 || path_stride < 0 || (int64_t)n_kv_heads * head_dim > INT32_MAX / 4) return UA_ERR_SHAPE;
  if (dtype < UA_BF16 || dtype > UA_FP32) return UA_ERR_UNSUPPORTED;
  if (layers > 65535 || batch > 65535) return UA_ERR_SHAPE;               // (a launch's y and z)
  if (!layers || !batch || !n_tokens || !n_path || !n_pages || !max_pages) return UA_OK;
  if (!k_pages || !v_pages || !table || !lens || !path || !n_kept || !k_page_strides || !v_page_strides) return UA_ERR_NULL;
  const int size = dtype == UA_FP32 ? 4 : 2;
  if (!aligned4(table) || !aligned4(lens) || !aligned4(n_new) || !aligned4(path) || !aligned4(n_kept)) return UA_ERR_ALIGN;
  KeepParams p{};
  uint64_t all = (uint64_t)head_dim * size | reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages);
  for (int i = 0; i < 4; ++i) all |= (uint64_t)(k_page_strides[i] * size) | (uint64_t)(v_page_strides[i] * size);
  if (all % size) return UA_ERR_ALIGN;
  auto pool = [&](void* rows, const int64_t* s) { return KeepPool{(char*)rows, s[0] * size, s[1] * size, s[2] * size, s[3] * size}; };
  p.k = pool(k_pages, k_page_strides);
  p.v = pool(v_pages, v_page_strides);
  p.steps = {lens, n_new, nullptr, 0, n_tokens};
  p.pages = {table, table_stride, n_pages, page, paged_room(page, max_pages), make_div(page)};
  p.path = path;
  p.n_kept = n_kept;
  p.path_stride = path_stride;
  p.n_path = n_path;
  p.n_heads = n_kv_heads;
  rc = check_device();
  if (rc != UA_OK) return rc;
  auto run = [&](auto vec) {
    p.columns = head_dim * size / (int)sizeof(vec);
    p.by_columns = make_div(p.columns);
    const int64_t groups = ((int64_t)2 * n_kv_heads * p.columns + kKeepThreads - 1) / kKeepThreads;
    paged_keep_kernel<decltype(vec)><<<dim3((unsigned)groups, batch, layers), kKeepThreads, 0, (hipStream_t)stream>>>(p);
  };
  // (heads that whole vectors of 16 bytes do not divide, or not on their boundaries, go entry by entry)
  if (all % 16 == 0) run(u32x4{}); else if (size == 4) run(uint32_t{}); else run(uint16_t{});
  return hipGetLastError() == hipSuccess ? UA_OK : UA_ERR_LAUNCH;
}
