// Pages of keys and values in 4 bits.
//
// Blocks of 32 neighbouring elements of one head of one token share a power of two 2^(b - 127), b one byte in 2 .. 252 (255: a block with an
// element that is no number or infinite, and all of it reads as no number); an element is a sign, two bits of exponent and one of significand: 0 0.5
// 1 1.5 2 3 4 6.  That is the 4-bit form that gfx950 converts from and to by itself, two elements an instruction, the power applied on the way.
//
// What a page holds of one kv head is one run of bytes (17 lines of 128 bytes at 16 keys of 128 elements), for `page_size` keys, a multiple of 8, of D elements, a multiple of 32:
//   key codes    [page_size][D / 2]               a key is a row: a lane of the matrix cores takes D / 4 neighbouring elements of one key
//   value codes  [page_size / 8][D / 8][8][4]     pieces of eight keys and eight elements: a lane takes eight keys of eight elements, 32 bytes in a row
//   key powers   [page_size][D / 32]
//   value powers [page_size / 8][D / 32][8]       the eight powers that go with a lane's eight keys are 8 bytes in a row
#pragma once
#include "common.h"

typedef __bf16 packed_bf16x2 __attribute__((ext_vector_type(2)));

#define PACKED_BLOCK 32
#define PACKED_NO_NUMBER 255u

struct PackedPage {  // offsets in bytes, from the start of a (page, kv head)
  int dim, page_size;
  __host__ __device__ __forceinline__ int codes() const { return page_size * dim / 2; }
  __host__ __device__ __forceinline__ int powers() const { return page_size * dim / PACKED_BLOCK; }
  __host__ __device__ __forceinline__ int bytes() const { return 2 * (codes() + powers()); }
  // the four bytes of elements 8 granule .. + 8 of the key / value at `offset`
  __device__ __forceinline__ int key_codes(int offset, int granule) const { return (offset * (dim / 8) + granule) * 4; }
  __device__ __forceinline__ int value_codes(int offset, int granule) const { return codes() + (((offset >> 3) * (dim / 8) + granule) * 8 + (offset & 7)) * 4; }
  __device__ __forceinline__ int key_power(int offset, int block) const { return 2 * codes() + offset * (dim / PACKED_BLOCK) + block; }
  __device__ __forceinline__ int value_power(int offset, int block) const { return 2 * codes() + powers() + ((offset >> 3) * (dim / PACKED_BLOCK) + block) * 8 + (offset & 7); }
};

static inline bool packed_fits(int dim, int page_size) { return dim >= 32 && dim <= 256 && dim % 32 == 0 && page_size >= 8 && page_size % 8 == 0; }

// The power as the conversions take it: a float of that exponent (255: no number comes out).
__device__ __forceinline__ float packed_power(unsigned byte) { return __uint_as_float(byte << 23); }

template <int BYTE> __device__ __forceinline__ unsigned unpack_pair(unsigned codes, float power) {  // elements 2 BYTE and 2 BYTE + 1, as bfloat16 (exact)
  union { packed_bf16x2 v; unsigned u; } r;
  r.v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power, BYTE);
  return r.u;
}
