// Eight consecutive elements of a row in one thread, at any alignment.
//
// Rows of odd widths start off 16 bytes.  The hardware loads and stores 16 bytes at any address,
// so such rows move in the same wide accesses.  FULL: the vector is whole -- no thread branches on
// `left` (the elements from here to the row's end), and the loads of a batch are issued without a
// wait between them.  Otherwise a row's last, partial vector goes element by element.
#pragma once
#include "common.h"

namespace smpk {

constexpr int kCols = 8;

typedef uint32_t Word4 __attribute__((ext_vector_type(4), aligned(2)));

template <typename T>
union Raw8 {
  Word4 w[kCols * sizeof(T) / 16];
  T v[kCols];
};

template <bool FULL, typename T>
__device__ __forceinline__ void read8(const T* p, int left, Raw8<T>& r) {
  constexpr int M = 16 / sizeof(T);
  if (FULL || left >= kCols) {
#pragma unroll
    for (int k = 0; k < kCols / M; ++k) r.w[k] = *reinterpret_cast<const Word4*>(p + k * M);
  } else {
#pragma unroll
    for (int j = 0; j < kCols; ++j) r.v[j] = j < left ? p[j] : from_f32<T>(0.f);
  }
}

template <typename T>
__device__ __forceinline__ float at8(const Raw8<T>& r, int j) {
  return to_f32(r.v[j]);
}

template <bool FULL, typename T>
__device__ __forceinline__ void read8(const T* p, int left, float (&o)[kCols]) {
  Raw8<T> r;
  read8<FULL>(p, left, r);
#pragma unroll
  for (int j = 0; j < kCols; ++j) o[j] = at8(r, j);
}

// STREAM: past the caches, for outputs that are written once, in whole lines, and that no kernel
// finds there later.  Stored normally and so: the gradient of a 50257 x 1600 bf16 table 132 and
// 118 us; block norms of 16384 rows forward, 1600 bf16 44 and 43 us, 4096 bf16 107 and 94 us, 1600 fp32 91 and
// 70 us, backward, 1600 bf16 82 and 72 us.  Not where a table's reads want the memory too (65536 gathered
// rows of a cold table: 76 and 82 us; 65 and 52 us of one that was read just before), where what is written is
// what was just read (clip of 1.4 GB: 837 and 926 us with the norm), nor for rows of fp32 in the backward,
// whose lanes write half lines.
template <bool FULL, bool STREAM, typename T>
__device__ __forceinline__ void write8(T* p, int left, const float (&o)[kCols]) {
  constexpr int M = 16 / sizeof(T);
  if (FULL || left >= kCols) {
    Raw8<T> r;
#pragma unroll
    for (int j = 0; j < kCols; ++j) r.v[j] = from_f32<T>(o[j]);
#pragma unroll
    for (int k = 0; k < kCols / M; ++k) {
      Word4* q = reinterpret_cast<Word4*>(p + k * M);
      if (STREAM) {
        __builtin_nontemporal_store(r.w[k], q);
      } else {
        *q = r.w[k];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < kCols; ++j)
      if (j < left) p[j] = from_f32<T>(o[j]);
  }
}

// Sum over a wave in a fixed order, the same value in all lanes, without LDS: neighbours within
// rows of 16 lanes, then the rows.
__device__ __forceinline__ float wave_sum_fixed(float v) {
#define SMPK_DPP_ADD(ctrl, rows) \
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, rows, 0xf, false))
  SMPK_DPP_ADD(0xb1, 0xf);   // quad_perm [1, 0, 3, 2]
  SMPK_DPP_ADD(0x4e, 0xf);   // quad_perm [2, 3, 0, 1]
  SMPK_DPP_ADD(0x141, 0xf);  // row_half_mirror
  SMPK_DPP_ADD(0x140, 0xf);  // row_mirror: every lane has its row's sum
  SMPK_DPP_ADD(0x142, 0xa);  // row_bcast15: rows 1 and 3 add the row before
  SMPK_DPP_ADD(0x143, 0xc);  // row_bcast31: rows 2 and 3 add row 1's
#undef SMPK_DPP_ADD
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

}  // namespace smpk
