// fa_paged.h - what the kernels on the paged 8-bit cache share.
//
// A value of a page is code 2^e, code an e4m3 number and 2^e the scale of its page and K/V head.
// e4m3 is a floating format, so a scale only has to bring the page's largest value into range; with
// powers of two it costs no rounding of its own, growing one moves the codes exactly (but for
// subnormals), and both products below take it in exponent arithmetic.
//
// Attention over the pages.
//
//   s'_ij = (q_i . code_j) c 2^ke(page) + ve(page),  c = log2(e) / sqrt(D)
//   p'_ij = 2^(s'_ij - m'),  acc_i = sum_j p'_ij vcode_j,  l_i = sum_j 2^-ve p'_ij,  o = acc / l
//
// The V scale sits in the exponent: p' is measured by what its key adds to the output, so its
// rounding to 16 bits (fp16: 2^-11 relative, next to the largest contribution) is safe for any mix of
// scales, one accumulator serves all pages, and l, in fp32, takes the scales out again.  (|ve| <= 40 keeps
// 2^-ve p' of every key that counts inside fp32's normal range.)  The codes go into the products
// unscaled, exact in both 16-bit types: QK in the queries' type, PV in fp16.  m' is lazy and low: it
// moves, to 7 below the largest score, when a score passes it by more than 15.  So p' <= 2^15, and
// the many small weights of a long flat tail stay above fp16's subnormals down to 2^-21 of the largest.
#pragma once

#include "fa_device.h"
#include "fa_launch.h"

namespace fa {

constexpr int kScaleMin = -40, kScaleMax = 40;   // l needs their spread to stay far inside fp32's (above)
constexpr float kCodeMax = 448.f;

__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }

// Exponent of a stored scale (kept within the range that the append writes).
__device__ __forceinline__ int scale_of(const void* scales, long long i) {
  return min(max((int)static_cast<const uint8_t*>(scales)[i] - 127, kScaleMin), kScaleMax);
}

// The page that the table names for column `col` of sequence b; -1: none.
__device__ __forceinline__ int page_of(const fa_paged_cache& c, int b, int col) {
  if (col >= c.table_width) return -1;
  const int p = c.block_table[b * c.table_stride + col];
  return p >= 0 && p < c.num_pages ? p : -1;
}

// Lengths as the kernels use them: nothing negative, no sum past 31 bits.
__device__ __forceinline__ int past_of(const int* past, int b) { return min(max(past[b], 0), 0x3FFFFFFF); }
__device__ __forceinline__ int fresh_of(const int* fresh, int b, int N) { return fresh ? min(max(fresh[b], 0), N) : N; }

constexpr int kMaxSplit = 128;                  // parts that a row's keys are split into at most
constexpr float kLazy = 15.f, kBelow = 7.f;     // m' moves to kBelow under the largest score, when one passes it by kLazy

__device__ __forceinline__ uint32_t cvt_f16(uint32_t w, bool hi) {
  const f16x2 r = hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false);
  return __builtin_bit_cast(uint32_t, r);
}

template <typename E>
__device__ __forceinline__ u32x4 codes8(uint32_t w0, uint32_t w1) {
  if constexpr (std::is_same<E, F16>::value) {
    return u32x4{cvt_f16(w0, false), cvt_f16(w0, true), cvt_f16(w1, false), cvt_f16(w1, true)};
  } else {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.f, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.f, true))};
  }
}

// A NaN of V behind a row's last key must not reach the row, and 0 NaN would: in the tiles where rows end,
// NaN codes are added as zeros, and where one was met the tiles are read again behind the loop, to make
// NaN of what sees one: counts = seen (1 or 0) x is NaN (1 or 0).
//
// 0x80 in each byte of w that is a NaN code (0x7F, 0xFF), 0 in the others.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint32_t without_nan(uint32_t w, uint32_t nan) { return w & ~((nan >> 7) * 0xFFu); }
__device__ __forceinline__ uint32_t nan_as_one(uint32_t w) { return (nan_bytes(w) >> 7) * 0x38u; }   // e4m3 1 or 0

// Keys of a split of a row block: `keys` keys that some row sees in at most nsplit parts, each a multiple
// of `step`.
__device__ __forceinline__ int split_keys(int keys, int nsplit, int step) {
  const int per = (keys + nsplit - 1) / nsplit;
  return max((per + step - 1) / step * step, step);
}

// Token range of a row block, and how many keys its rows see.
struct Block {
  int past, fresh, r0, rows, lmin, keys;
};

__device__ __forceinline__ Block block_of(const PagedArgs& a, int b, int rb, int G, int block_rows) {
  Block x;
  x.past = past_of(a.past, b);
  x.fresh = fresh_of(a.fresh, b, a.N);
  x.r0 = rb * block_rows;
  x.rows = a.N * G;
  const int tok0 = x.r0 / G, tok1 = min(min((x.r0 + block_rows - 1) / G, a.N - 1), x.fresh - 1);
  x.lmin = x.past + tok0;                              // the last key that the first live row sees
  // (a length past the table: its first key without a page makes the rows NaN, the rest need not be walked)
  const long long named = (long long)a.cache.table_width * a.cache.page_size;
  x.keys = tok0 < x.fresh ? (int)min((long long)(x.past + tok1 + 1), named + 1) : 0;
  return x;
}

// A split leaves, for each row, D unnormalised sums, m' and l.
template <int D>
__device__ __forceinline__ float* part_row(const PagedArgs& a, long long block, int split, int row, int block_rows) {
  return a.part + ((block * a.nsplit + split) * block_rows + row) * (D + 4);
}

// (fa_paged_rows.hip) blocks of 128 or 256 rows, keys in tiles of kBlockKeys
constexpr int kBlockKeys = 64;
int paged_rows(int dtype, const PagedArgs& a, int row_blocks, int block_rows);

}  // namespace fa
