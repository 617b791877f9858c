// Rows of keys and values into the 4-bit pages of packed.h and back.
#include "packed.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// eight elements of a row as floats (`whole`: in 16-byte pieces)
template <typename T> __device__ __forceinline__ void load_eight(const T* from, bool whole, float* x) {
  if (whole) {
    union { u32x4 v[sizeof(T) / 2]; T e[8]; } piece;
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 2; ++i) piece.v[i] = ((const u32x4*)from)[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float(piece.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float(from[i]);
  }
}

// A thread packs eight elements, four neighbours a block.  The exponent of the block's largest magnitude a decides the power: 2^(exponent - 2), one more
// where a's significand is 1.75 or larger (a would be rounded to 8, which the elements do not have), so that a lands on 4 to 6.  Division by the
// power is exact, and what is rounded is rounded once, to the nearest element (ties to the even code), so the bits depend on nothing but the row.
template <typename T>
__global__ void __launch_bounds__(256) packed_store_kernel(const T* x, int stride, int first, int kv_heads, int tokens, unsigned char* pages, int slots_held, const int* slots, PackedPage page, bool whole) {
  const int granules = page.dim / 8, per_token = 2 * kv_heads * granules;
  const long flat = (long)blockIdx.x * blockDim.x + threadIdx.x;
  const int token = (int)(flat / per_token);
  if (token >= tokens) return;  // (whole blocks of 32 leave together: per_token is a multiple of four)
  const int inside = (int)(flat - (long)token * per_token), head_of_both = inside / granules, granule = inside - head_of_both * granules;
  const bool value = head_of_both >= kv_heads;
  const int head = value ? head_of_both - kv_heads : head_of_both, slot = slots[token];
  float v[8];
  load_eight(x + (size_t)token * stride + first + (size_t)inside * 8, whole, v);
  unsigned largest = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) largest = max(largest, __float_as_uint(v[i]) & 0x7fffffffu);
  largest = max(largest, (unsigned)__shfl_xor((int)largest, 1));
  largest = max(largest, (unsigned)__shfl_xor((int)largest, 2));
  if (slot < 0 || slot >= slots_held) return;
  const bool number = largest < 0x7f800000u;
  const unsigned power = number ? (unsigned)min(max((int)((largest + 0x200000u) >> 23) - 2, 2), 252) : PACKED_NO_NUMBER;
  unsigned codes = 0;
  if (number) {
    const float unit = packed_power(power);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0], v[1], unit, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[2], v[3], unit, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[4], v[5], unit, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[6], v[7], unit, 3);
  }
  const int at = slot / page.page_size, offset = slot - at * page.page_size;
  unsigned char* mine = pages + ((size_t)at * kv_heads + head) * page.bytes();
  *(unsigned*)(mine + (value ? page.value_codes(offset, granule) : page.key_codes(offset, granule))) = codes;
  if (granule % 4 == 0) mine[value ? page.value_power(offset, granule / 4) : page.key_power(offset, granule / 4)] = (unsigned char)power;
}

// A thread reads eight elements back: exact in bfloat16 and in float32.
template <typename T>
__global__ void __launch_bounds__(256) packed_rows_kernel(const unsigned char* pages, int kv_heads, int slots_held, const int* slots, int rows, T* keys, T* values, PackedPage page) {
  const int granules = page.dim / 8, per_row = 2 * kv_heads * granules;
  const long flat = (long)blockIdx.x * blockDim.x + threadIdx.x;
  const int row = (int)(flat / per_row);
  if (row >= rows) return;
  const int inside = (int)(flat - (long)row * per_row), head_of_both = inside / granules, granule = inside - head_of_both * granules;
  const bool value = head_of_both >= kv_heads;
  const int head = value ? head_of_both - kv_heads : head_of_both, slot = slots[row];
  unsigned pairs[4] = {0, 0, 0, 0};
  if (slot >= 0 && slot < slots_held) {
    const int at = slot / page.page_size, offset = slot - at * page.page_size;
    const unsigned char* mine = pages + ((size_t)at * kv_heads + head) * page.bytes();
    const unsigned codes = *(const unsigned*)(mine + (value ? page.value_codes(offset, granule) : page.key_codes(offset, granule)));
    const float power = packed_power(mine[value ? page.value_power(offset, granule / 4) : page.key_power(offset, granule / 4)]);
    pairs[0] = unpack_pair<0>(codes, power);
    pairs[1] = unpack_pair<1>(codes, power);
    pairs[2] = unpack_pair<2>(codes, power);
    pairs[3] = unpack_pair<3>(codes, power);
  }
  T* to = (value ? values : keys) + ((size_t)row * kv_heads + head) * page.dim + granule * 8;
  if constexpr (sizeof(T) == 2) {
    *(u32x4*)to = (u32x4){pairs[0], pairs[1], pairs[2], pairs[3]};
  } else {
    u32x4 wide[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      wide[i / 2][i % 2 * 2] = pairs[i] << 16;
      wide[i / 2][i % 2 * 2 + 1] = pairs[i] & 0xffff0000u;
    }
    ((u32x4*)to)[0] = wide[0];
    ((u32x4*)to)[1] = wide[1];
  }
}

// Keys and values of `tokens` rows of x ([token][stride], the keys' heads from column `first`, the values' behind them) into the
// pages [num_pages][kv_heads][bytes] at `slots` (page * page_size + offset; one outside the pages: nowhere).
extern "C" int llmserve_packed_store(const void* x, int is_float, int stride, int first, int tokens, int kv_heads, int dim, void* pages, int num_pages, int page_size, const int* slots, hipStream_t stream) {
  if (tokens == 0) return 0;
  const long held = (long)num_pages * page_size;
  if (!x || !pages || !slots || tokens < 0 || kv_heads <= 0 || num_pages <= 0 || !packed_fits(dim, page_size) || held >= (1L << 31) || first < 0 ||
      (long)first + 2L * kv_heads * dim > stride || (size_t)pages % 16)
    return ERR_BAD_ARGUMENT;
  const long threads = (long)tokens * 2 * kv_heads * (dim / 8), blocks = (threads + 255) / 256;
  if (blocks >= (1L << 31)) return ERR_BAD_ARGUMENT;
  const PackedPage page = {dim, page_size};
  const int piece = is_float ? 4 : 8;
  const bool whole = (size_t)x % 16 == 0 && stride % piece == 0 && first % piece == 0;
  if (is_float)
    packed_store_kernel<float><<<(unsigned)blocks, 256, 0, stream>>>((const float*)x, stride, first, kv_heads, tokens, (unsigned char*)pages, (int)held, slots, page, whole);
  else
    packed_store_kernel<bf16_t><<<(unsigned)blocks, 256, 0, stream>>>((const bf16_t*)x, stride, first, kv_heads, tokens, (unsigned char*)pages, (int)held, slots, page, whole);
  return LAUNCH_STATUS();
}

// keys and values [rows][kv_heads][dim] of the given slots (zeros for one outside the pages)
extern "C" int llmserve_packed_rows(const void* pages, int num_pages, int kv_heads, int dim, int page_size, const int* slots, int rows, void* keys, void* values, int is_float, hipStream_t stream) {
  if (rows == 0) return 0;
  const long held = (long)num_pages * page_size;
  if (!keys || !values || !pages || !slots || rows < 0 || kv_heads <= 0 || num_pages <= 0 || !packed_fits(dim, page_size) || held >= (1L << 31) ||
      ((size_t)keys | (size_t)values | (size_t)pages) % 16)
    return ERR_BAD_ARGUMENT;
  const long threads = (long)rows * 2 * kv_heads * (dim / 8), blocks = (threads + 255) / 256;
  if (blocks >= (1L << 31)) return ERR_BAD_ARGUMENT;
  const PackedPage page = {dim, page_size};
  if (is_float)
    packed_rows_kernel<float><<<(unsigned)blocks, 256, 0, stream>>>((const unsigned char*)pages, kv_heads, (int)held, slots, rows, (float*)keys, (float*)values, page);
  else
    packed_rows_kernel<bf16_t><<<(unsigned)blocks, 256, 0, stream>>>((const unsigned char*)pages, kv_heads, (int)held, slots, rows, (bf16_t*)keys, (bf16_t*)values, page);
  return LAUNCH_STATUS();
}
