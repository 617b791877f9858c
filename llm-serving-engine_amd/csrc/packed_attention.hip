// Grouped-query attention over pages in 4 bits (packed.h), softmax in float32.  Compiled once per head size.
//
// A workgroup takes a run of up to 16 CT columns, the (token, query head) pairs of one request that share a kv head, and its four waves take steps
// of 32 keys in turn.  A step of a wave, with v_mfma_f32_16x16x32_bf16:
//   S^T[key][column] = K[key][:] . Q[column][:]           A = rows of keys, two tiles of 16
//   P = exp2(S * scale - the column's reference), masked to the keys that the column's token sees
//   O^T[d][column] += V^T[d][key] P^T[key][column]        A = rows of values, turned
// Codes become bfloat16 in registers (exactly: a code has two bits of significand, its block a power of two), two an instruction; no other
// memory than the codes themselves is touched.  A lane takes D / 4 neighbouring elements of a key, which are the four (at D = 128) slices that it holds of the
// product over D: which elements a slice of the sum is, is free as long as the queries are laid out alike.  The 32 keys are dealt to the rows of the two tiles so that a lane ends with the
// scores of eight neighbouring keys, the slice of keys that the second product wants of it.  Of the values a lane takes eight neighbouring elements of those
// eight keys, 32 bytes in a row; each of the eight is a row of a tile of its own.
//
// A float32 run splits queries and weights into three bfloat16 terms each (24 bits of significand), so all products are exact and sums are float32.
#include "packed.h"

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<multiple of 32>"
#endif
#if HEAD_DIM % 32 != 0 || HEAD_DIM < 32 || HEAD_DIM > 256
#error "HEAD_DIM is a multiple of 32 between 32 and 256"
#endif

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int D = HEAD_DIM;
constexpr int SLICES = D / 32;                // MFMA steps over D, and four-byte pieces of codes that a lane takes of a key
constexpr int TILES = D / 16;                 // tiles of O^T
constexpr int KEYS = 32;                      // keys a step
constexpr int WAVES = 4;
constexpr int SEGMENT = 8192;                 // keys whose pages lie in LDS at a time
constexpr int ENTRIES = SEGMENT / 8 + 2;
constexpr float AHEAD = 8.f;                  // log2 units that a score may run ahead of its column's reference before the sums are rescaled
constexpr float LOG2_E = 1.44269504088896f;
constexpr int CHUNKS = D / 128 + (D % 128) / 64 + (D % 64) / 32;  // runs of 128, 64 or 32 elements of a value
__host__ __device__ constexpr int chunk_width(int c) { return c < D / 128 ? 128 : (D % 128 >= 64 && c == D / 128) ? 64 : 32; }
__host__ __device__ constexpr int chunk_first(int c) { return c <= D / 128 ? c * 128 : D / 128 * 128 + 64; }
constexpr int KEY_POWERS = D % 128 == 0 ? D / 128 : D <= 64 ? 1 : SLICES;  // bytes of powers that a lane takes of a key

union Eight {
  bf16x8 v;
  u32x4 u;
};

struct Step {                                 // what a step takes from memory
  unsigned keys[2][SLICES], key_powers[2][KEY_POWERS];
  u32x4 values[CHUNKS][2];
  u32x2 value_powers[CHUNKS];
};

struct Pages {
  const unsigned char* from;                  // of the kv head
  size_t stride;                              // bytes from one page to the next
  int per_page, shift;                        // pieces of eight keys a page; log2 of it, or -1
  PackedPage page;
};

struct Walk {
  const int* tables;
  int table_width, num_pages;
  const int *query_start, *contexts;
  int requests, heads, kv_heads, window, single;
  int chunk, splits;                          // keys a workgroup walks, and the most workgroups that share a run of columns
  float scale;                                // times log2 e
};

struct Item {                                 // a run of columns
  int request, first_row, group, first, columns, first_position, last_position, from, to;
};

// Item `index`: the requests' columns in runs of `most`, one request's behind the other's.  False: there is no such item.
__device__ __forceinline__ bool find_item(const Walk& w, int index, int most, Item& item) {
  item.group = w.heads / w.kv_heads;
  int request, inside;
  if (w.single) {                             // no request brings more than one token
    const int each = (item.group + most - 1) / most;
    request = index / each;
    inside = index - request * each;
  } else {                                    // each wave for itself: 64 requests at a time
    const int lane = threadIdx.x % WAVE;
    int before = 0;
    request = -1;
    for (int base = 0; base < w.requests; base += WAVE) {
      const int b = base + lane;
      const int items = b < w.requests ? ((w.query_start[b + 1] - w.query_start[b]) * item.group + most - 1) / most : 0;
      int sum = items;
#pragma unroll
      for (int step = 1; step < WAVE; step <<= 1) {
        const int other = __shfl_up(sum, step);
        if (lane >= step) sum += other;
      }
      const unsigned long long found = __ballot(before + sum > index);
      if (found) {
        const int which = __ffsll((unsigned long long)found) - 1;
        request = base + which;
        inside = index - before - __shfl(sum - items, which);
        break;
      }
      before += __shfl(sum, WAVE - 1);
    }
    if (request < 0) return false;
  }
  request = __builtin_amdgcn_readfirstlane(request);
  if (request >= w.requests) return false;
  const int start = w.query_start[request], count = w.query_start[request + 1] - start;
  item.request = request;
  item.first = __builtin_amdgcn_readfirstlane(inside) * most;
  item.columns = min(most, count * item.group - item.first);
  if (item.columns <= 0) return false;
  item.first_row = start;
  const int past = w.contexts[request] - count;
  item.first_position = past + item.first / item.group;
  item.last_position = past + (item.first + item.columns - 1) / item.group;
  item.from = w.window > 0 ? max(0, item.first_position - w.window + 1) / KEYS * KEYS : 0;
  item.to = item.last_position + 1;
  return true;
}

template <int N> __device__ __forceinline__ void load_dwords(unsigned* to, const unsigned char* from) {  // (aligned to the largest power of two up to 16 bytes that divides 4 N)
  constexpr int ALIGN = N % 4 == 0 ? 16 : N % 2 == 0 ? 8 : 4;
  __builtin_memcpy(to, __builtin_assume_aligned(from, ALIGN), N * 4);
}

__device__ __forceinline__ void load_step(Step& s, const Pages& p, const int* entries, int first_entry, int base) {
  const int lane = threadIdx.x % WAVE, r = lane & 15, g = lane >> 4;
  {
    const int piece = base / 8 + (r >> 2), entry = p.shift >= 0 ? piece >> p.shift : piece / p.per_page;
    const unsigned char* mine = p.from + (size_t)entries[entry - first_entry] * p.stride;
    const int offset = (piece - entry * p.per_page) * 8 + (r & 3);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      load_dwords<SLICES>(s.keys[t], mine + p.page.key_codes(offset + 4 * t, g * SLICES));
#pragma unroll
      for (int i = 0; i < KEY_POWERS; ++i)
        s.key_powers[t][i] = mine[p.page.key_power(offset + 4 * t, D % 128 == 0 ? g * KEY_POWERS + i : (g * SLICES + i) / 4)];
    }
  }
  const int piece = base / 8 + g, entry = p.shift >= 0 ? piece >> p.shift : piece / p.per_page;
  const unsigned char* mine = p.from + (size_t)entries[entry - first_entry] * p.stride;
  const int offset = (piece - entry * p.per_page) * 8;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int granule = chunk_first(c) / 8 + r * chunk_width(c) / 128;
    load_dwords<8>((unsigned*)s.values[c], mine + p.page.value_codes(offset, granule));
    load_dwords<2>((unsigned*)&s.value_powers[c], mine + p.page.value_power(offset, granule / 4));
  }
}

template <typename T, int TERMS> __device__ __forceinline__ void split_eight(const float* x, Eight* terms) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float left = x[e];
#pragma unroll
    for (int k = 0; k < TERMS; ++k) {
      terms[k].v[e] = (bf16_t)left;
      if (k + 1 < TERMS) left -= (float)terms[k].v[e];
    }
  }
}

template <typename T, int CT>
__global__ void __launch_bounds__(WAVES * WAVE) packed_attention_kernel(const T* q, int q_stride, T* out, int out_stride, float* partial, const unsigned char* pages, int page_size, Walk w, int items, int whole) {
  constexpr int TERMS = sizeof(T) == 4 ? 3 : 1;
  __shared__ int entries[ENTRIES];
  __shared__ __attribute__((aligned(16))) float results[WAVES][16][D + 4];
  __shared__ float sums[WAVES][16][2];
  const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, r = lane & 15, g = lane >> 4;
  // the longest walks begin first: a request's last columns walk most keys
  const int all = items * w.kv_heads, at = blockIdx.x % all, split = blockIdx.x / all;
  const int kv_head = at % w.kv_heads;
  Item item;
  if (!find_item(w, items - 1 - at / w.kv_heads, 16 * CT, item)) return;
  const int begin = item.from + split * w.chunk, end = min(item.to, begin + w.chunk);
  if (begin >= item.to) return;
  const int parts = (item.to - item.from + w.chunk - 1) / w.chunk;
  Pages p;
  p.page = {D, page_size};
  p.per_page = page_size / 8;
  p.shift = (p.per_page & (p.per_page - 1)) == 0 ? 31 - __clz(p.per_page) : -1;
  p.from = pages + (size_t)kv_head * p.page.bytes();
  p.stride = (size_t)w.kv_heads * p.page.bytes();

  // the queries, and where their tokens stand
  Eight query[CT][TERMS][SLICES];
  int position[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int column = min(ct * 16 + r, item.columns - 1), flat = item.first + column, token = flat / item.group;
    position[ct] = item.first_position - item.first / item.group + token;
    const T* row = q + (size_t)(item.first_row + token) * q_stride + (kv_head * item.group + flat - token * item.group) * D + g * (D / 4);
#pragma unroll
    for (int s = 0; s < SLICES; ++s) {
      float x[8];
      union { u32x4 v[sizeof(T) / 2]; T e[8]; } piece;
      if (whole) {
#pragma unroll
        for (unsigned i = 0; i < sizeof(T) / 2; ++i) piece.v[i] = ((const u32x4*)(row + s * 8))[i];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) piece.e[e] = row[s * 8 + e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = to_float(piece.e[e]);
      Eight terms[TERMS];
      split_eight<T, TERMS>(x, terms);
#pragma unroll
      for (int k = 0; k < TERMS; ++k) query[ct][k][s] = terms[k];
    }
  }
  f32x4 sum[CT][TILES];
  float total[CT], reference[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    total[ct] = 0.f;
    reference[ct] = -INFINITY;
#pragma unroll
    for (int t = 0; t < TILES; ++t) sum[ct][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }

  for (int segment = begin; segment < end; segment += SEGMENT) {
    const int segment_end = min(end, segment + SEGMENT), first_entry = segment / page_size, last_entry = (segment_end + KEYS - 1 - (segment_end + KEYS - 1) % KEYS - 1) / page_size;
    __syncthreads();
    for (int i = first_entry + threadIdx.x; i <= last_entry; i += WAVES * WAVE) {
      const int entry = i < w.table_width ? w.tables[(size_t)item.request * w.table_width + i] : 0;
      entries[i - first_entry] = (unsigned)entry < (unsigned)w.num_pages ? entry : 0;
    }
    __syncthreads();
    int base = segment + wave * KEYS;
    if (base >= segment_end) continue;
    Step now;
    load_step(now, p, entries, first_entry, base);
    for (; base < segment_end; base += WAVES * KEYS) {
      Step next;
      const int following = base + WAVES * KEYS;
      if (following < segment_end) load_step(next, p, entries, first_entry, following);
      // scores: row 4 g + i of tile t is key 8 g + 4 t + i of the step
      f32x4 score[CT][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) score[ct][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < SLICES; ++s) {
          const float power = packed_power(now.key_powers[t][D % 128 == 0 ? s / 4 : D <= 64 ? 0 : s]);
          Eight key;
          key.u = (u32x4){unpack_pair<0>(now.keys[t][s], power), unpack_pair<1>(now.keys[t][s], power), unpack_pair<2>(now.keys[t][s], power), unpack_pair<3>(now.keys[t][s], power)};
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int k = TERMS - 1; k >= 0; --k) score[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(key.v, query[ct][k][s].v, score[ct][t], 0, 0, 0);
        }
      }
      const bool edge = base + KEYS - 1 > item.first_position || (w.window > 0 && base < item.last_position - w.window + 1);
      Eight weight[CT][TERMS];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = score[ct][i / 4][i % 4] * w.scale;
        if (edge) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = base + 8 * g + i;
            if (key > position[ct] || (w.window > 0 && key <= position[ct] - w.window)) x[i] = -INFINITY;
          }
        }
        float largest = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        if (__any(largest > reference[ct] + AHEAD)) {
          largest = fmaxf(largest, __shfl_xor(largest, 16));
          largest = fmaxf(largest, __shfl_xor(largest, 32));
          largest = fmaxf(largest, reference[ct]);
          const float change = reference[ct] == largest ? 1.f : __builtin_amdgcn_exp2f(reference[ct] - largest);
          reference[ct] = largest;
          total[ct] *= change;
#pragma unroll
          for (int t = 0; t < TILES; ++t) sum[ct][t] *= change;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x[i] - reference[ct]);
        split_eight<T, TERMS>(x, weight[ct]);
        if (TERMS == 1) {  // the weights that are multiplied are the weights that are added up
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = (float)weight[ct][0].v[i];
        }
        total[ct] += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
      }
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const int width = chunk_width(c), pairs = width / 32;  // pairs of elements that a lane takes of a key
        u32x2 powers = now.value_powers[c];
        bool poisoned = false;
        Eight marks;
        if (edge) {
          // A value that a column does not see has no part in it, whatever it is: keys beyond the last that any column sees get the smallest power;
          // of the others, those that are no number are taken out, and put back where they are seen.
          marks.u = (u32x4){0u, 0u, 0u, 0u};
          bool mine = false;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int key = base + 8 * g + j;
            const unsigned shift = (j & 3) * 8, byte = (powers[j / 4] >> shift) & 255u;
            const bool unseen = key > item.last_position || (w.window > 0 && key <= item.first_position - w.window), bad = byte == PACKED_NO_NUMBER;
            if (unseen || bad) powers[j / 4] &= ~(255u << shift);
            if (bad && !unseen) {
              marks.u[j / 2] |= 0x3f80u << (j % 2 * 16);
              mine = true;
            }
          }
          poisoned = __any(mine);
        }
        u32x4 turned[8];  // element e of the lane's, eight keys
        {
          unsigned raw[8][4];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float power = __uint_as_float(j % 4 == 3 ? powers[j / 4] >> 1 : powers[j / 4] << (23 - j % 4 * 8));  // (only the exponent of it counts)
            unsigned codes = now.values[c][j / 4][j % 4];
            if (width == 64) codes >>= (r & 1) * 16;
            if (width == 32) codes >>= (r & 3) * 8;
            raw[j][0] = unpack_pair<0>(codes, power);
            if (pairs > 1) raw[j][1] = unpack_pair<1>(codes, power);
            if (pairs > 2) {
              raw[j][2] = unpack_pair<2>(codes, power);
              raw[j][3] = unpack_pair<3>(codes, power);
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (e >= pairs) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              turned[2 * e][j] = __builtin_amdgcn_perm(raw[2 * j + 1][e], raw[2 * j][e], 0x05040100u);
              turned[2 * e + 1][j] = __builtin_amdgcn_perm(raw[2 * j + 1][e], raw[2 * j][e], 0x07060302u);
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (e >= 2 * pairs) continue;
          Eight value;
          value.u = turned[e];
          const int t = chunk_first(c) / 16 + e;
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int k = TERMS - 1; k >= 0; --k) sum[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value.v, weight[ct][k].v, sum[ct][t], 0, 0, 0);
        }
        if (poisoned) {
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            Eight seen;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int key = base + 8 * g + i;
              seen.v[i] = (bf16_t)(key > position[ct] || (w.window > 0 && key <= position[ct] - w.window) ? 0.f : 1.f);
            }
            const f32x4 hit = __builtin_amdgcn_mfma_f32_16x16x32_bf16(marks.v, seen.v, (f32x4){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              if (e >= 2 * pairs) continue;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (hit[i] > 0.f) sum[ct][chunk_first(c) / 16 + e][i] = __uint_as_float(0x7fc00000u);
            }
          }
        }
      }
      now = next;
    }
  }

  // the waves' sums, brought together
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (ct * 16 >= item.columns) break;
    __syncthreads();
    float wave_total = total[ct];
    wave_total += __shfl_xor(wave_total, 16);
    wave_total += __shfl_xor(wave_total, 32);
    if (g == 0) {
      sums[wave][r][0] = reference[ct];
      sums[wave][r][1] = wave_total;
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int each = chunk_width(c) / 16;  // neighbouring elements of a row of the tiles
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < each) results[wave][r][chunk_first(c) + (4 * g + i) * each + e] = sum[ct][chunk_first(c) / 16 + e][i];
    }
    __syncthreads();
    const int columns = min(16, item.columns - ct * 16);
    for (int at = threadIdx.x; at < columns * (D / 4); at += WAVES * WAVE) {
      const int column = at / (D / 4), d = (at - column * (D / 4)) * 4;
      float largest = sums[0][column][0];
#pragma unroll
      for (int v = 1; v < WAVES; ++v) largest = fmaxf(largest, sums[v][column][0]);
      f32x4 result = (f32x4){0.f, 0.f, 0.f, 0.f};
      float weights = 0.f;
#pragma unroll
      for (int v = 0; v < WAVES; ++v) {
        const float share = sums[v][column][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sums[v][column][0] - largest);
        weights += share * sums[v][column][1];
        result += share * *(const f32x4*)&results[v][column][d];
      }
      const int flat = item.first + ct * 16 + column, token = flat / item.group, head = kv_head * item.group + flat - token * item.group;
      const size_t row = item.first_row + token;
      if (parts == 1) {
        const float over = 1.f / weights;
#pragma unroll
        for (int i = 0; i < 4; ++i) out[row * out_stride + head * D + d + i] = from_float<T>(result[i] * over);
      } else {
        float* to = partial + ((row * w.heads + head) * w.splits + split) * (D + 4);
        *(f32x4*)(to + d) = result;
        if (d == 0) {
          to[D] = largest;
          to[D + 1] = weights;
        }
      }
    }
  }
}

// A wave a (token, head) whose keys were split: its parts joined.
template <typename T>
__global__ void __launch_bounds__(WAVE) packed_join_kernel(T* out, int out_stride, const float* partial, Walk w, int most) {
  const int token = blockIdx.x, head = blockIdx.y, lane = threadIdx.x, group = w.heads / w.kv_heads;
  int low = 0, high = w.requests;  // the first request that ends behind the token
  while (low < high) {
    const int middle = (low + high) / 2;
    if (w.query_start[middle + 1] > token) high = middle;
    else low = middle + 1;
  }
  if (low == w.requests || token < w.query_start[low]) return;
  const int start = w.query_start[low], count = w.query_start[low + 1] - start, past = w.contexts[low] - count;
  const int first = ((token - start) * group + head % group) / most * most, columns = min(most, count * group - first);
  const int from = w.window > 0 ? max(0, past + first / group - w.window + 1) / KEYS * KEYS : 0, to = past + (first + columns - 1) / group + 1;
  const int parts = (to - from + w.chunk - 1) / w.chunk;
  if (parts <= 1) return;
  const float* mine = partial + ((size_t)token * w.heads + head) * w.splits * (D + 4);
  float largest = -INFINITY;
  for (int i = 0; i < parts; ++i) largest = fmaxf(largest, mine[(size_t)i * (D + 4) + D]);
  constexpr int EACH = (D + WAVE - 1) / WAVE;
  float result[EACH] = {}, weights = 0.f;
  for (int i = 0; i < parts; ++i) {
    const float* part = mine + (size_t)i * (D + 4);
    const float share = part[D] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(part[D] - largest);
    weights += share * part[D + 1];
#pragma unroll
    for (int e = 0; e < EACH; ++e)
      if (lane + e * WAVE < D) result[e] += share * part[lane + e * WAVE];
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if (lane + e * WAVE < D) out[(size_t)token * out_stride + head * D + lane + e * WAVE] = from_float<T>(result[e] / weights);
}

template <typename T>
static int launch(const void* q, int q_stride, void* out, int out_stride, float* partial, const void* pages, int page_size, const Walk& w, int tokens, int column_tiles, hipStream_t stream) {
  const int group = w.heads / w.kv_heads, most = 16 * column_tiles;
  const long items = w.single ? (long)w.requests * ((group + most - 1) / most) : ((long)tokens * group + most - 1) / most + w.requests;
  const long blocks = items * w.kv_heads * w.splits;
  if (items >= (1L << 31) || blocks >= (1L << 31)) return ERR_BAD_ARGUMENT;
  const int piece = sizeof(T) == 4 ? 4 : 8, whole = (size_t)q % 16 == 0 && q_stride % piece == 0;
  if (column_tiles == 1)
    packed_attention_kernel<T, 1><<<(unsigned)blocks, WAVES * WAVE, 0, stream>>>((const T*)q, q_stride, (T*)out, out_stride, partial, (const unsigned char*)pages, page_size, w, (int)items, whole);
  else
    packed_attention_kernel<T, 2><<<(unsigned)blocks, WAVES * WAVE, 0, stream>>>((const T*)q, q_stride, (T*)out, out_stride, partial, (const unsigned char*)pages, page_size, w, (int)items, whole);
  if (int status = LAUNCH_STATUS()) return status;
  if (w.splits > 1) packed_join_kernel<T><<<dim3(tokens, w.heads), WAVE, 0, stream>>>((T*)out, out_stride, partial, w, most);
  return LAUNCH_STATUS();
}

// q's heads are the first columns of rows of q_stride; tokens, requests: as many rows and requests as the arrays hold; single: no request brings more than one token.  A
// workgroup walks up to `chunk` keys (a multiple of 128), at most `splits` share a run of columns: splits * chunk covers every walk.  partial, where splits > 1:
// float32 [tokens][heads][splits][D + 4].
extern "C" int llmserve_packed_attention(const void* q, int is_float, int q_stride, void* out, int out_stride, void* partial, const void* pages, int num_pages, const int* tables, int table_width,
                                         const int* query_start, const int* contexts, int requests, int tokens, int heads, int kv_heads, int page_size, float scale, int window, int single, int column_tiles,
                                         int chunk, int splits, hipStream_t stream) {
  if (tokens == 0 || requests == 0) return 0;
  if (!q || !out || !pages || !tables || !query_start || !contexts || requests < 0 || tokens < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || num_pages <= 0 || table_width <= 0 ||
      !packed_fits(D, page_size) || (size_t)pages % 16 || q_stride < heads * D || out_stride < heads * D || window < 0 || column_tiles < 1 || column_tiles > 2 || chunk < 128 || chunk % 128 ||
      splits < 1 || splits > 65535 || (splits > 1 && (!partial || (size_t)partial % 16)) || heads > 65535)
    return ERR_BAD_ARGUMENT;
  const Walk w = {tables, table_width, num_pages, query_start, contexts, requests, heads, kv_heads, window, single, chunk, splits, scale * LOG2_E};
  if (is_float) return launch<float>(q, q_stride, out, out_stride, (float*)partial, pages, page_size, w, tokens, column_tiles, stream);
  return launch<bf16_t>(q, q_stride, out, out_stride, (float*)partial, pages, page_size, w, tokens, column_tiles, stream);
}
