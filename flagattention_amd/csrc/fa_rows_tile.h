// Tile helpers of the many-row attention kernels (fa_prefill.hip, fa_varlen.hip) and of 4-bit decode
// (fa_mxfp4.hip): vector types, MFMA wrappers, transposing reads, offset copies into LDS and the
// swizzles of K and V rows.
#pragma once

#include "fa_common.h"
#include "fa_wave.h"

namespace fa {

template <typename T>
struct PVec {
  typedef T v8 __attribute__((ext_vector_type(8)));
  typedef T v4 __attribute__((ext_vector_type(4)));
  typedef T v2 __attribute__((ext_vector_type(2)));
};

__device__ inline floatx16 mfma_32x32x16(PVec<__bf16>::v8 a, PVec<__bf16>::v8 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline floatx16 mfma_32x32x16(PVec<_Float16>::v8 a, PVec<_Float16>::v8 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

template <typename T>
__device__ inline typename PVec<T>::v4 lds_tr_read4(const unsigned char* p) {
  typedef short shortx4 __attribute__((ext_vector_type(4)));
  const shortx4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((FA_LDS shortx4*)(p));
  return __builtin_bit_cast(typename PVec<T>::v4, v);
}

// 16 bytes per lane from base + off (32-bit lane offset, uniform base) into LDS.
__device__ inline void lds_dma16_off(const unsigned char* base, unsigned int off, FA_LDS void* lds) {
  const unsigned m0 = __builtin_amdgcn_readfirstlane(
      static_cast<unsigned>(reinterpret_cast<__SIZE_TYPE__>(lds)));
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(off), "s"(base), "s"(m0)
               : "memory", "m0");
}

// Chunk (K) and chunk-pair (V) swizzles of token row r, C chunks per row.
template <int C>
__device__ inline int fk(int r) {
  return C >= 16 ? (r & 15) : ((r >> 1) & 7);  // C = 8: two rows per 256 bytes
}
template <int C>
__device__ inline int fv(int r) {
  return C >= 16 ? (((r & 3) << 1) | ((r >> 2) & 1)) : ((r & 2) | ((r >> 2) & 1));
}

}  // namespace fa
