// What the sliding-window attention kernels share: which keys a row sees, element types, LDS layouts for heads of 64 and 128, row tiles.
//
// Row r (query) of a call sees key j iff  j <= r + hi  and  (j >= r + lo  or  j < sinks);  hi and lo hold the window and the
// difference of the positions of query 0 and key 0, clamped to +-kFar, which is beyond any length.  What nothing in a workgroup's tile sees may be NaN.
#pragma once
#include "ua_common.h"

namespace ua {

typedef _Float16 fp16;
constexpr int kFar = 1 << 29;
constexpr int64_t kSwaMaxLen = 1 << 28;            // of queries and keys: no sum of a row and a bound leaves 32 bits
constexpr int64_t kSwaMaxGroups = UINT32_MAX / 256; // a launch counts its threads in 32 bits
constexpr int kSwaRows = 128;                      // of a workgroup's tile, 32 a wave
constexpr int kSwaBlock = 64;                      // rows of the other side that a step goes through

template <class T> struct SwaVec;
template <> struct SwaVec<bf16> {
  typedef bf16x8 x8;
  typedef bf16x4 x4;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct SwaVec<fp16> {
  typedef __attribute__((ext_vector_type(8))) _Float16 x8;
  typedef __attribute__((ext_vector_type(4))) _Float16 x4;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
// Two transposing reads (see lds_read_tr16_b64) as one operand: 4 rows from `a`, 4 from `b`.
template <class T>
__device__ __forceinline__ typename SwaVec<T>::x8 lds_tr_pair(uint32_t a, uint32_t b) {
  typedef __attribute__((ext_vector_type(4))) short s4;
  typedef __attribute__((address_space(3))) s4 lds_s4;
  const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4*>(a));
  const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4*>(b));
  return __builtin_bit_cast(typename SwaVec<T>::x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
}

// A head of kD elements in LDS.  One copy instruction of a wave fills 1 KiB: 4 rows of 256 bytes or 8 of 128.  The 16-byte chunk c of row r lies
// in slot c ^ f(r), so that the 16 or 32 lanes that LDS serves at a time meet different banks.
template <int kD>
struct SwaHead {
  static_assert(kD == 64 || kD == 128, "head sizes");
  static constexpr int kRow = 2 * kD, kChunks = kD / 8, kSteps = kD / 16, kBlocks = kD / 32;
  static constexpr int kCopyRows = 1024 / kRow, kCopies = kSwaBlock / kCopyRows / 4;      // of a wave and a block
  static constexpr int kUnits = kSwaBlock / kCopyRows;                                    // of a block
  // rows are read as they are: 16 rows at one chunk
  static __device__ __forceinline__ int slot_n(int r, int c) { return kD == 128 ? c ^ (r & 15) : c ^ (r >> 1 & 7); }
  // rows are read transposed: 4 rows at 4 chunks that start at a multiple of 4
  static __device__ __forceinline__ int slot_t(int r, int c) { return kD == 128 ? c ^ ((r & 3) << 2) : c ^ ((r >> 1 & 1) << 2); }
  // both: of 256 bytes as transposed, the fours of rows at a pitch of 1040 bytes, so that 16 rows meet 16 slots; of 128 bytes three bits of the row
  static __device__ __forceinline__ int slot_b(int r, int c) {
    return kD == 128 ? slot_t(r, c) : c ^ ((r >> 1 & 1) << 2) ^ ((r >> 2 & 1) << 1) ^ (r >> 3 & 1);
  }
  static constexpr int kPitchB = kD == 128 ? 1040 : 1024, kTile = kUnits * 1024, kTileB = kUnits * kPitchB;
  static __device__ __forceinline__ uint32_t at_n(int r, int c) { return r * kRow + (slot_n(r, c) << 4); }
  static __device__ __forceinline__ uint32_t at_b(int r, int c) { return r / kCopyRows * kPitchB + r % kCopyRows * kRow + (slot_b(r, c) << 4); }
  // transposing read m (of kBlocks): columns 32 m + lane % 32, rows 4 (lane / 32) .. + 3; of the `both` layout, rows + 8 * second
  static __device__ __forceinline__ uint32_t tr_offset(int lane, int m) {
    const int i = lane & 15, r = i >> 2, row = 4 * (lane >> 5) + r;
    return row * kRow + (slot_t(row, 4 * m + 2 * (lane >> 4 & 1) + ((i & 3) >> 1)) << 4) + (i & 1) * 8;
  }
  static __device__ __forceinline__ uint32_t tr_offset_b(int lane, int m, int second) {
    const int i = lane & 15, r = i >> 2, row = 4 * (lane >> 5) + r + 8 * second;
    return at_b(row, 4 * m + 2 * (lane >> 4 & 1) + ((i & 3) >> 1)) + (i & 1) * 8;
  }
};
// Zeros in rows from .. to - 1 of a tile in LDS, for a wave whose next reads are of them.  A walk's first block may hold rows before the first one that
// anything in the workgroup's tile sees: their weights are 0, which would make NaN of NaN or infinity.  (Rows behind the last one seen are not
// copied.)  Every wave that reads the block does this itself, so none waits for another; 16 writes at the most.
template <int kD, int kPitch, int kAlso = 0>                       // kAlso: bytes to a second tile of which the same rows are cleared
__device__ __forceinline__ void lds_clear_rows(uint32_t tile, int from, int to) {
  constexpr int kCopyRows = 1024 / (2 * kD);
  for (int u = from / kCopyRows; u * kCopyRows < to; ++u) {
    const int lane = fresh_lane(), r = u * kCopyRows + lane / (kD / 8);
    if (r >= from && r < to) {
      lds_put(tile + u * kPitch + 16 * lane, u32x4{0, 0, 0, 0});
      if (kAlso) lds_put(tile + u * kPitch + 16 * lane + kAlso, u32x4{0, 0, 0, 0});
    }
  }
  asm volatile("" ::: "memory");
}

// 32 rows between memory and a wave's own LDS (32 * kRow bytes): memory sees whole rows.  Rows from `n_rows` on are read as the last one
// and not written.
template <int kD>
__device__ __forceinline__ void swa_load_rows(u32x4 (&raw)[kD / 16], const void* rows, int64_t row_stride, int n_rows) {
  using H = SwaHead<kD>;
  const int lane = fresh_lane(), c = lane % H::kChunks;
#pragma unroll
  for (int i = 0; i < kD / 16; ++i) {
    const int r = min(H::kCopyRows * i + lane / H::kChunks, n_rows - 1);
    raw[i] = *reinterpret_cast<const u32x4*>(static_cast<const char*>(rows) + (r * row_stride + c * 8) * 2);
  }
}
template <int kD>
__device__ __forceinline__ void swa_put_rows(const u32x4 (&raw)[kD / 16], uint32_t lds) {
  using H = SwaHead<kD>;
  const int lane = fresh_lane();
#pragma unroll
  for (int i = 0; i < kD / 16; ++i) lds_put(lds + H::at_n(H::kCopyRows * i + lane / H::kChunks, lane % H::kChunks), raw[i]);
}
// B operands: row lane % 32, columns 16 i + 8 (lane / 32) ..
template <class T, int kD>
__device__ __forceinline__ void swa_frags(typename SwaVec<T>::x8 (&f)[kD / 16], uint32_t lds) {
  using H = SwaHead<kD>;
  const int lane = fresh_lane();
#pragma unroll
  for (int i = 0; i < kD / 16; ++i) f[i] = lds_get<typename SwaVec<T>::x8>(lds + H::at_n(lane & 31, 2 * i + (lane >> 5)));
}
// Accumulators of 32 rows, transposed (acc[m][4 g + j]: column 32 m + 8 g + 4 (lane / 32) + j of row lane % 32), times `mul`.
template <class T, int kD>
__device__ __forceinline__ void swa_store_rows(void* rows, int64_t row_stride, int n_rows, const f32x16 (&acc)[kD / 32], float mul, uint32_t lds) {
  using H = SwaHead<kD>;
  const int lane = fresh_lane();
#pragma unroll
  for (int m = 0; m < H::kBlocks; ++m)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      typename SwaVec<T>::x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = (T)(acc[m][4 * g + j] * mul);
      lds_put(lds + H::at_n(lane & 31, 4 * m + g) + 8 * (lane >> 5), w);
    }
#pragma unroll
  for (int i = 0; i < kD / 16; ++i) {
    const int r = H::kCopyRows * i + lane / H::kChunks, c = lane % H::kChunks;
    const u32x4 x = lds_get<u32x4>(lds + H::at_n(r, c));
    if (r < n_rows) *reinterpret_cast<u32x4*>(static_cast<char*>(rows) + (r * row_stride + c * 8) * 2) = x;
  }
}
// The same as fp32, straight from the registers (partial results, which stay in the caches): rows of kD floats.
template <int kD>
__device__ __forceinline__ void swa_store_f32(float* rows, int64_t row_stride, int n_rows, const f32x16 (&acc)[kD / 32], float mul) {
  const int lane = fresh_lane(), r = lane & 31;
  if (r < n_rows) {
    float* p = rows + r * row_stride + 4 * (lane >> 5);
#pragma unroll
    for (int m = 0; m < kD / 32; ++m)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(p + 32 * m + 8 * g) = f32x4{acc[m][4 * g] * mul, acc[m][4 * g + 1] * mul, acc[m][4 * g + 2] * mul, acc[m][4 * g + 3] * mul};
  }
}

// Two operands of 64 rows, copied asynchronously into a stage of LDS, x at 0, y behind it.  How either is read there: as it is (kN),
// transposed (kT), or both.
enum SwaRead { kN, kT, kB };
template <int kD, SwaRead kX, SwaRead kY>
struct SwaStream {
  using H = SwaHead<kD>;
  static constexpr int kPieces = 2 * H::kCopies;
  static constexpr int kPitchX = kX == kB ? H::kPitchB : 1024, kPitchY = kY == kB ? H::kPitchB : 1024, kSecond = H::kUnits * kPitchX;
  static constexpr int kBytes = kSecond + H::kUnits * kPitchY;
  const char *x, *y;
  int64_t xs, ys;                                  // bytes of a row
  int xoff, yoff;
  u32x4 rx, ry;
  uint32_t wave;
  template <SwaRead kRead>
  static __device__ __forceinline__ int offset(int row_stride, int wave, int lane) {       // of a copy's lane from the block's first row on
    const int r = H::kCopyRows * wave + lane / H::kChunks, s = lane % H::kChunks;
    return (r * row_stride + (kRead == kN ? H::slot_n(r, s) : kRead == kT ? H::slot_t(r, s) : H::slot_b(r, s)) * 8) * 2;
  }
  __device__ __forceinline__ SwaStream(int64_t xs_, int64_t ys_, int wave_, int lane) : xs(2 * xs_), ys(2 * ys_), wave(wave_) {
    xoff = offset<kX>((int)xs_, wave_, lane);
    yoff = offset<kY>((int)ys_, wave_, lane);
  }
  __device__ __forceinline__ void of(const void* x_, const void* y_) { x = (const char*)x_; y = (const char*)y_; }
  // Rows row0 .. row0 + 63 of n are next; those from n on read as zeros, and without `more` all of them.
  __device__ __forceinline__ void block(int row0, int n, bool more) {
    const int rows = more ? min(n - row0, kSwaBlock) : 0;
    rx = make_rsrc_words(x + row0 * xs, rows > 0 ? (uint32_t)((rows - 1) * xs + H::kRow) : 0);
    ry = make_rsrc_words(y + row0 * ys, rows > 0 ? (uint32_t)((rows - 1) * ys + H::kRow) : 0);
  }
  __device__ __forceinline__ void copy(int n, uint32_t stage) const {
    const int j = n >> 1, row = 4 * H::kCopyRows * j;
    if (n & 1) dma16_abs(ry, stage + kSecond + (4 * j + wave) * kPitchY, yoff, row * (int)ys);
    else       dma16_abs(rx, stage + (4 * j + wave) * kPitchX, xoff, row * (int)xs);
  }
};

#define UA_BOTH __host__ __device__ __forceinline__
UA_BOTH int imin(int a, int b) { return a < b ? a : b; }
UA_BOTH int imax(int a, int b) { return a > b ? a : b; }
// Blocks of 64 keys that a tile of rows r0 .. r1 walks: those of the sinks, then those of the window.
struct SwaWalk {
  int n_sink, first, n, start, sinks_end, end;     // of the keys that a row sees: start .. end - 1, and those before sinks_end
  UA_BOTH SwaWalk(int r0, int r1, int hi, int lo, int sinks, int n_keys) {
    const int last = imin(r1 + hi, n_keys - 1);
    start = imax(r0 + lo, 0);
    end = imax(last + 1, 0);
    sinks_end = imin(sinks, end);
    n_sink = last >= 0 ? (imin(sinks, last + 1) + kSwaBlock - 1) / kSwaBlock : 0;
    first = imax(start / kSwaBlock, n_sink);
    n = n_sink + (last >= start ? imax(last / kSwaBlock + 1 - first, 0) : 0);
  }
  __device__ __forceinline__ int at(int i) const { return i < n_sink ? i : first + i - n_sink; }
  // A block's keys from here on are not copied: nothing sees them.
  __device__ __forceinline__ int end_of(int block) const { return (block + 1) * kSwaBlock <= start ? sinks_end : end; }
};
// Blocks of 64 query rows, of one head, that see a tile of keys k0 .. k1.
struct SwaColumn {
  int first, n, start, end;                        // the rows that see a key: start .. end - 1
  UA_BOTH SwaColumn(int k0, int k1, int hi, int lo, int sinks, int n_rows) {
    start = imax(k0 - hi, 0);
    end = imax(k0 < sinks ? n_rows : imin(k1 - lo + 1, n_rows), 0);
    first = start / kSwaBlock;
    n = end > start ? (end - 1) / kSwaBlock + 1 - first : 0;
  }
};

// A run of a backward's columns, tiles first .. first + tiles - 1 of every key head, whose walks are cut into n_parts: with more than one part i
// leaves fp32 rows, contiguous [batch, key heads, 128 * tiles, head_dim], at dk + i * part and dv + i * part.
struct SwaColumns {
  int first, tiles, n_parts, n_blocks;
  float *dk, *dv;
  int64_t part;
  BlockMap map;
  Div by_parts;
};
struct SwaParams {
  const void *q, *k, *v, *dout;
  void *o, *dq, *dk, *dv;
  float *lse, *delta;
  Strides3 qs, ks, vs, os, ds, dqs, dks, dvs;
  int batch, n_heads, n_kv_heads, group, seq_q, seq_k, hi, lo, sinks;
  float scale, scale_log2;
  // The rows' walks are cut into n_parts; part i leaves fp32 rows (and, forward, their lse), contiguous [batch, heads, tokens, head_dim], at part_o +
  // i * o_part and part_lse + i * lse_part.  Backward: the columns of the sinks and the others are cut likewise, each into parts of their own.
  int n_parts;
  float *part_o, *part_lse;
  int64_t o_part, lse_part;
  SwaColumns cols[2];
  BlockMap map;
  Div by_heads, by_kv_heads, by_group, by_parts;
  int n_qtiles, n_ktiles, n_col_blocks;
};
// Steps of 64 rows that the walks of a side take, the mean and the most (of up to 33 of its tiles, evenly spread).
struct SwaSteps { double mean; int most; };
template <class Of> SwaSteps swa_steps(int first, int n, Of of) {
  SwaSteps s{0, 0};
  const int m = n < 33 ? n : 33;
  for (int i = 0; i < m; ++i) {
    const int x = of(first + (m > 1 ? (int)((int64_t)i * (n - 1) / (m - 1)) : 0));
    s.mean += (double)x / m;
    s.most = x > s.most ? x : s.most;
  }
  return s;
}
inline SwaSteps swa_row_steps(const SwaParams& p) {
  return swa_steps(0, p.n_qtiles, [&](int t) { return SwaWalk(t * kSwaRows, imin((t + 1) * kSwaRows, p.seq_q) - 1, p.hi, p.lo, p.sinks, p.seq_k).n; });
}

int swa_fill(SwaParams& p, int batch, int n_heads, int n_kv_heads, int seq_q, int seq_k, int head_dim, int dtype, int64_t q_start, int64_t k_start,
             int64_t left, int64_t right, int64_t sinks, float softmax_scale);
bool swa_strides_ok(const int64_t* s, bool written);
// The backward starts scores from -lse / scale, in 32 bits: both, and scale * log2(e), stay far from their ends.
inline bool swa_scale_ok(float scale) { return scale >= 0x1p-64f && scale <= 0x1p64f; }
// Merge of fp32 partial rows: see merge_rows_kernel.
int swa_merge(const float* part_o, int64_t o_part, const float* part_lse, int64_t lse_part, int n_parts, void* o, const Strides3& os, float* lse,
              int batch, int n_heads, int seq, int head_dim, int dtype, hipStream_t st);

}  // namespace ua
