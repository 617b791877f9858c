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

// Which rows a thread takes: one, or, of many rows, eight that lie in one piece of a page where their slots follow each other, so that what it writes and reads of values is 32 bytes in a
// row (8,192 rows of 8 heads of 128 in bfloat16, 43 MB: packed in 11.5 us, read back in 9.9; 16 and 14 with one row a thread).  `shift` brings the first row's place in its piece to the groups' beginnings.
template <int ROWS> __device__ __forceinline__ int first_row(long flat, int per_row, const int* slots, int slots_held, int& inside) {
  const int group = (int)(flat / per_row);
  inside = (int)(flat - (long)group * per_row);
  const int shift = ROWS > 1 && slots[0] >= 0 && slots[0] < slots_held ? slots[0] % ROWS : 0;
  return group * ROWS - shift;
}

// Whether the eight slots are a whole piece.
__device__ __forceinline__ bool whole_piece(const int (&slot)[8]) {
  bool whole = slot[0] >= 0 && slot[0] % 8 == 0;
#pragma unroll
  for (int i = 1; i < 8; ++i) whole = whole && slot[i] == slot[0] + i;
  return whole;
}

// Eight elements of a block's granule as codes, four bits each, of the block's power.  The exponent of the block's largest magnitude a decides the power: 2^(exponent - 2), one more
// where a's significand is 1.75 or larger (a would be rounded to 8, which the elements do not have), so that a lands on 4 to 6.  Division by the
// power is exact, and what is rounded is rounded once, to the nearest element (ties to the even code), so the bits depend on nothing but the row.
__device__ __forceinline__ unsigned largest_bits(const float* x) {
  unsigned largest = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) largest = max(largest, __float_as_uint(x[e]) & 0x7fffffffu);
  return largest;
}
__device__ __forceinline__ unsigned pack_eight(const float* x, unsigned largest, unsigned& power) {
  const bool number = largest < 0x7f800000u;
  power = number ? (unsigned)min(max((int)((largest + 0x200000u) >> 23) - 2, 2), 252) : PACKED_NO_NUMBER;
  const float unit = packed_power(power);
  unsigned codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], unit, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], unit, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], unit, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], unit, 3);
  return number ? codes : 0u;
}

// A thread packs eight elements of its rows, four neighbours a block.
template <typename T, int ROWS>
__global__ void __launch_bounds__(256) packed_store_kernel(const T* x, int stride, int first, int kv_heads, int tokens, unsigned char* pages, int slots_held, const int* slots, PackedPage page, bool whole) {
  const int granules = page.dim / 8;
  int inside;
  const int row = first_row<ROWS>((long)blockIdx.x * blockDim.x + threadIdx.x, 2 * kv_heads * granules, slots, slots_held, inside);
  if (row >= tokens) return;  // (whole blocks of 32 leave together: a row has a multiple of four granules)
  const int head_of_both = inside / granules, granule = inside - head_of_both * granules;
  const bool value = head_of_both >= kv_heads;
  const int head = value ? head_of_both - kv_heads : head_of_both;
  int slot[ROWS];
  float v[ROWS][8];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int at = min(max(row + i, 0), tokens - 1);
    slot[i] = row + i >= 0 && row + i < tokens ? slots[at] : -1;
    load_eight(x + (size_t)at * stride + first + (size_t)inside * 8, whole, v[i]);
  }
  unsigned codes[ROWS], power[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    unsigned largest = largest_bits(v[i]);
    largest = max(largest, (unsigned)__shfl_xor((int)largest, 1));
    largest = max(largest, (unsigned)__shfl_xor((int)largest, 2));
    codes[i] = pack_eight(v[i], largest, power[i]);
  }
  if constexpr (ROWS == 8) {
    if (value && whole_piece(slot) && slot[7] < slots_held) {
      const int at = slot[0] / page.page_size, offset = slot[0] - at * page.page_size;
      unsigned char* mine = pages + ((size_t)at * kv_heads + head) * page.bytes();
      u32x4* to = (u32x4*)(mine + page.value_codes(offset, granule));
      to[0] = (u32x4){codes[0], codes[1], codes[2], codes[3]};
      to[1] = (u32x4){codes[4], codes[5], codes[6], codes[7]};
      if (granule % 4 == 0) {
        unsigned* powers = (unsigned*)(mine + page.value_power(offset, granule / 4));
        powers[0] = power[0] | power[1] << 8 | power[2] << 16 | power[3] << 24;
        powers[1] = power[4] | power[5] << 8 | power[6] << 16 | power[7] << 24;
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (slot[i] < 0 || slot[i] >= slots_held) continue;
    const int at = slot[i] / page.page_size, offset = slot[i] - at * page.page_size;
    unsigned char* mine = pages + ((size_t)at * kv_heads + head) * page.bytes();
    *(unsigned*)(mine + (value ? page.value_codes(offset, granule) : page.key_codes(offset, granule))) = codes[i];
    if (granule % 4 == 0) mine[value ? page.value_power(offset, granule / 4) : page.key_power(offset, granule / 4)] = (unsigned char)power[i];
  }
}

// Few rows, rotated as they are packed (one launch of a layer's decode step less): a thread takes 16 elements of a head of a row, which hold eight pairs.  Neighbouring pairs: granules 2 p and 2 p + 1, half a
// block; half pairs: granules p and p + D / 16, of two blocks (heads of a multiple of 64, so that four threads have a block each).  q and k are written back rotated, k is packed as it was
// written back.  (Eight tokens at the 1.5B sizes, in a captured step: 3.1 us, of which little is work: a launch is what it spares.)
template <typename T, bool HALF>
__global__ void __launch_bounds__(256) packed_rotate_store_kernel(T* qkv, int stride, const float2* table, int heads, int kv_heads, int tokens, unsigned char* pages, int slots_held, const int* slots, PackedPage page,
                                                                   bool whole) {
  const int per_head = page.dim / 16, per_row = (heads + 2 * kv_heads) * per_head;
  const int flat = blockIdx.x * blockDim.x + threadIdx.x, token = flat / per_row, inside = flat - token * per_row, head = inside / per_head, p = inside - head * per_head;
  if (token >= tokens) return;                // (whole blocks of 32 leave together: a row has a multiple of four threads with half pairs, of two without)
  const int slot = slots[token];              // (asked for with the rows: behind the stores the compiler would leave it)
  T* row = qkv + (size_t)token * stride + (size_t)head * page.dim;
  const bool value = head >= heads + kv_heads;
  const int granule[2] = {HALF && !value ? p : 2 * p, HALF && !value ? p + per_head : 2 * p + 1};
  float x[2][8];
#pragma unroll
  for (int g = 0; g < 2; ++g) load_eight(row + granule[g] * 8, whole, x[g]);
  if (!value) {
    const float2* angles = table + (size_t)token * (page.dim / 2) + 8 * p;
    float2 turn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) turn[i] = angles[i];
    union { u32x4 v[2 * sizeof(T) / 2]; T e[2][8]; } out;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int g0 = HALF ? 0 : i / 4, e0 = HALF ? i : i % 4 * 2, g1 = HALF ? 1 : i / 4, e1 = HALF ? i : i % 4 * 2 + 1;
      float first, second;
      const float a = x[g0][e0], b = x[g1][e1];
      // (the bits of the kernels that only rotate)
      if (sizeof(T) == 4 || stride % 8 != 0) first = __builtin_fmaf(a, turn[i].x, -(b * turn[i].y)), second = __builtin_fmaf(a, turn[i].y, b * turn[i].x);
      else turn_pair(a, b, turn[i].x, turn[i].y, i == 0, &first, &second);
      out.e[g0][e0] = from_float<T>(first);
      out.e[g1][e1] = from_float<T>(second);
    }
#pragma unroll
    for (int g = 0; g < 2; ++g) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[g][e] = to_float(out.e[g][e]);
      if (whole) {
#pragma unroll
        for (unsigned i = 0; i < sizeof(T) / 2; ++i) ((u32x4*)(row + granule[g] * 8))[i] = out.v[g * (sizeof(T) / 2) + i];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) row[granule[g] * 8 + e] = out.e[g][e];
      }
    }
  }
  unsigned largest[2] = {largest_bits(x[0]), largest_bits(x[1])};
  if (HALF && !value) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      largest[g] = max(largest[g], (unsigned)__shfl_xor((int)largest[g], 1));
      largest[g] = max(largest[g], (unsigned)__shfl_xor((int)largest[g], 2));
    }
  } else {
    largest[0] = max(largest[0], largest[1]);
    largest[0] = largest[1] = max(largest[0], (unsigned)__shfl_xor((int)largest[0], 1));
  }
  if (head < heads || slot < 0 || slot >= slots_held) return;
  const int at = slot / page.page_size, offset = slot - at * page.page_size;
  unsigned char* mine = pages + ((size_t)at * kv_heads + (value ? head - heads - kv_heads : head - heads)) * page.bytes();
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    unsigned power;
    *(unsigned*)(mine + (value ? page.value_codes(offset, granule[g]) : page.key_codes(offset, granule[g]))) = pack_eight(x[g], largest[g], power);
    if (granule[g] % 4 == 0) mine[value ? page.value_power(offset, granule[g] / 4) : page.key_power(offset, granule[g] / 4)] = (unsigned char)power;
  }
}

// A thread reads eight elements of its rows back: exact in bfloat16 and in float32.
template <typename T, int ROWS>
__global__ void __launch_bounds__(256) packed_rows_kernel(const unsigned char* pages, int kv_heads, int slots_held, const int* slots, int rows, T* keys, T* values, PackedPage page) {
  const int granules = page.dim / 8;
  int inside;
  const int row = first_row<ROWS>((long)blockIdx.x * blockDim.x + threadIdx.x, 2 * kv_heads * granules, slots, slots_held, inside);
  if (row >= rows) return;
  const int head_of_both = inside / granules, granule = inside - head_of_both * granules;
  const bool value = head_of_both >= kv_heads;
  const int head = value ? head_of_both - kv_heads : head_of_both;
  int slot[ROWS];
  unsigned codes[ROWS], power[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int given = row + i >= 0 && row + i < rows ? slots[row + i] : -1;
    slot[i] = given >= 0 && given < slots_held ? given : -1;
    codes[i] = power[i] = 0;
  }
  bool together = false;
  if constexpr (ROWS == 8) together = value && whole_piece(slot);
  if (together) {
    const int at = slot[0] / page.page_size, offset = slot[0] - at * page.page_size;
    const unsigned char* mine = pages + ((size_t)at * kv_heads + head) * page.bytes();
    union { u32x4 v[2]; unsigned e[8]; } all;
    all.v[0] = ((const u32x4*)(mine + page.value_codes(offset, granule)))[0];
    all.v[1] = ((const u32x4*)(mine + page.value_codes(offset, granule)))[1];
    const unsigned* powers = (const unsigned*)(mine + page.value_power(offset, granule / 4));
    const unsigned two[2] = {powers[0], powers[1]};
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      codes[i] = all.e[i % 8];
      power[i] = (two[i % 8 / 4] >> (i % 4 * 8)) & 255u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if (slot[i] < 0) continue;
      const int at = slot[i] / page.page_size, offset = slot[i] - at * page.page_size;
      const unsigned char* mine = pages + ((size_t)at * kv_heads + head) * page.bytes();
      codes[i] = *(const unsigned*)(mine + (value ? page.value_codes(offset, granule) : page.key_codes(offset, granule)));
      power[i] = mine[value ? page.value_power(offset, granule / 4) : page.key_power(offset, granule / 4)];
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (row + i < 0 || row + i >= rows) continue;
    const float unit = packed_power(power[i]);
    unsigned pairs[4] = {unpack_pair<0>(codes[i], unit), unpack_pair<1>(codes[i], unit), unpack_pair<2>(codes[i], unit), unpack_pair<3>(codes[i], unit)};
    T* to = (value ? values : keys) + ((size_t)(row + i) * kv_heads + head) * page.dim + granule * 8;
    if constexpr (sizeof(T) == 2) {
      *(u32x4*)to = (u32x4){pairs[0], pairs[1], pairs[2], pairs[3]};
    } else {
      u32x4 wide[2];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        wide[e / 2][e % 2 * 2] = pairs[e] << 16;
        wide[e / 2][e % 2 * 2 + 1] = pairs[e] & 0xffff0000u;
      }
      ((u32x4*)to)[0] = wide[0];
      ((u32x4*)to)[1] = wide[1];
    }
  }
}

// Eight rows a thread from so many rows on that each of the chip's 1,024 SIMDs still has a wave.  us, packed and read back, one row and eight: 8 heads of 128 in bfloat16, 512 rows 6.9 and 10.4,
// 1,024 8.8 and 10.9, 2,048 (the first that take eight) 12.4 and 11.7, 8,192 31.5 and 21.7; 4 heads of 64 in float32, 1,021 rows 6.3 and 11.0.
static inline int rows_a_thread(int rows, int kv_heads, int dim) { return (long)rows * 2 * kv_heads * (dim / 8) >= 8L * 1024 * 64 ? 8 : 1; }
static inline long packed_blocks(int rows, int each, int kv_heads, int dim) {  // (a group more for the shift)
  const long groups = each == 1 ? rows : (long)rows / each + 2;
  return (groups * 2 * kv_heads * (dim / 8) + 255) / 256;
}

// Keys and values of `tokens` rows of x ([token][stride], the keys' heads from column `first`, the values' behind them) into the
// pages [num_pages][kv_heads][bytes] at `slots` (page * page_size + offset; one outside the pages: nowhere).
extern "C" int llmserve_packed_store(const void* x, int is_float, int stride, int first, int tokens, int kv_heads, int dim, void* pages, int num_pages, int page_size, const int* slots, hipStream_t stream) {
  if (tokens == 0) return 0;
  const long held = (long)num_pages * page_size;
  if (!x || !pages || !slots || tokens < 0 || kv_heads <= 0 || num_pages <= 0 || !packed_fits(dim, page_size) || held >= (1L << 31) || first < 0 ||
      (long)first + 2L * kv_heads * dim > stride || (size_t)pages % 16)
    return ERR_BAD_ARGUMENT;
  const int each = rows_a_thread(tokens, kv_heads, dim);
  const long blocks = packed_blocks(tokens, each, kv_heads, dim);
  if (blocks >= (1L << 31)) return ERR_BAD_ARGUMENT;
  const PackedPage page = {dim, page_size};
  const int piece = is_float ? 4 : 8;
  const bool whole = (size_t)x % 16 == 0 && stride % piece == 0 && first % piece == 0;
  const auto launch = [&](auto kernel, auto rows) { kernel<<<(unsigned)blocks, 256, 0, stream>>>(rows, stride, first, kv_heads, tokens, (unsigned char*)pages, (int)held, slots, page, whole); };
  if (is_float && each == 8) launch(packed_store_kernel<float, 8>, (const float*)x);
  else if (is_float) launch(packed_store_kernel<float, 1>, (const float*)x);
  else if (each == 8) launch(packed_store_kernel<bf16_t, 8>, (const bf16_t*)x);
  else launch(packed_store_kernel<bf16_t, 1>, (const bf16_t*)x);
  return LAUNCH_STATUS();
}

// Whether rows are rotated as they are packed: those that a thread takes one of, and with half pairs heads of a multiple of 64.  Of more rows k is read again from what the rotation wrote: 2,048
// tokens at 12/2 heads of 128 rotated in 5.0 us, packed in 4.7, both behind each other 6.1; at 40/8 9.4, 5.7 and 15.1, of 58 MB that are moved 4 are that.
extern "C" int llmserve_packed_rotates(int tokens, int kv_heads, int dim, int pairing) { return rows_a_thread(tokens, kv_heads, dim) == 1 && (pairing == 1 || (pairing == 2 && dim % 64 == 0)); }

// The first heads + kv_heads heads of `tokens` rows rotated in place by the table's angles (pairing 1: neighbours, 2: halves), then as above.
extern "C" int llmserve_packed_rotate_store(void* qkv, int is_float, int stride, const float* table, int pairing, int tokens, int heads, int kv_heads, int dim, void* pages, int num_pages, int page_size,
                                            const int* slots, hipStream_t stream) {
  if (tokens == 0) return 0;
  const long held = (long)num_pages * page_size;
  if (!qkv || !table || !pages || !slots || tokens < 0 || heads <= 0 || kv_heads <= 0 || num_pages <= 0 || !packed_fits(dim, page_size) || held >= (1L << 31) || (heads + 2L * kv_heads) * dim > stride ||
      (size_t)pages % 16 || !llmserve_packed_rotates(tokens, kv_heads, dim, pairing))
    return ERR_BAD_ARGUMENT;
  const long blocks = ((long)tokens * (heads + 2 * kv_heads) * (dim / 16) + 255) / 256;
  if (blocks * 256 >= (1L << 31)) return ERR_BAD_ARGUMENT;
  const PackedPage page = {dim, page_size};
  const bool whole = (size_t)qkv % 16 == 0 && stride % (is_float ? 4 : 8) == 0;
  const auto launch = [&](auto kernel, auto rows) { kernel<<<(unsigned)blocks, 256, 0, stream>>>(rows, stride, (const float2*)table, heads, kv_heads, tokens, (unsigned char*)pages, (int)held, slots, page, whole); };
  if (is_float && pairing == 2) launch(packed_rotate_store_kernel<float, true>, (float*)qkv);
  else if (is_float) launch(packed_rotate_store_kernel<float, false>, (float*)qkv);
  else if (pairing == 2) launch(packed_rotate_store_kernel<bf16_t, true>, (bf16_t*)qkv);
  else launch(packed_rotate_store_kernel<bf16_t, false>, (bf16_t*)qkv);
  return LAUNCH_STATUS();
}

// keys and values [rows][kv_heads][dim] of the given slots (zeros for one outside the pages)
extern "C" int llmserve_packed_rows(const void* pages, int num_pages, int kv_heads, int dim, int page_size, const int* slots, int rows, void* keys, void* values, int is_float, hipStream_t stream) {
  if (rows == 0) return 0;
  const long held = (long)num_pages * page_size;
  if (!keys || !values || !pages || !slots || rows < 0 || kv_heads <= 0 || num_pages <= 0 || !packed_fits(dim, page_size) || held >= (1L << 31) ||
      ((size_t)keys | (size_t)values | (size_t)pages) % 16)
    return ERR_BAD_ARGUMENT;
  const int each = rows_a_thread(rows, kv_heads, dim);
  const long blocks = packed_blocks(rows, each, kv_heads, dim);
  if (blocks >= (1L << 31)) return ERR_BAD_ARGUMENT;
  const PackedPage page = {dim, page_size};
  const auto launch = [&](auto kernel, auto to_keys, auto to_values) { kernel<<<(unsigned)blocks, 256, 0, stream>>>((const unsigned char*)pages, kv_heads, (int)held, slots, rows, to_keys, to_values, page); };
  if (is_float && each == 8) launch(packed_rows_kernel<float, 8>, (float*)keys, (float*)values);
  else if (is_float) launch(packed_rows_kernel<float, 1>, (float*)keys, (float*)values);
  else if (each == 8) launch(packed_rows_kernel<bf16_t, 8>, (bf16_t*)keys, (bf16_t*)values);
  else launch(packed_rows_kernel<bf16_t, 1>, (bf16_t*)keys, (bf16_t*)values);
  return LAUNCH_STATUS();
}
