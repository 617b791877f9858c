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
constexpr int STAGES = 2;                     // steps that a wave has asked for
constexpr int PIECE = 8 * D + 16;             // bytes in LDS of the codes of eight keys and values (16 spare: the same rows of two pieces lie in other banks)
constexpr int STAGE = 4 * PIECE + 2 * D;      // of a step: four pieces, and their powers
constexpr int ASKS = 4 * ((D + 127) / 128 + 1);  // loads of a step
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

struct Walk {
  const int* tables;
  int table_width, num_pages;
  int page_size, page_shift;                  // log2 of the pieces of eight keys that a page holds, or -1
  unsigned page_reciprocal;                   // 2^32 over them, rounded up
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

typedef const int __attribute__((address_space(4))) Scalar;  // read by scalar loads: what no kernel writes meanwhile

// Where the four pieces of eight keys of a step lie: their pages and their numbers in them.
struct Four {
  unsigned of[4];
};
struct Place {
  Four page, piece;
};

// (wave-uniform: table entries come through the scalar caches.  Entries beyond the table, and those that are no page, are page 0, whose
// keys nobody sees then.)
__device__ __forceinline__ void find_place(Place& to, const Walk& w, Scalar* table, int base) {
  const unsigned per_page = (unsigned)w.page_size / 8;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned piece = (unsigned)base / 8 + i, at = w.page_shift >= 0 ? piece >> w.page_shift : __umulhi(piece, w.page_reciprocal);
    const unsigned entry = at < (unsigned)w.table_width ? (unsigned)table[at] : 0u;
    to.page.of[i] = entry < (unsigned)w.num_pages ? entry : 0u;
    to.piece.of[i] = piece - at * per_page;
  }
}

// Asks for a step: straight into LDS.  A load takes the key codes and the value codes of a piece, 16 bytes a lane (two where heads are wider than
// 128), and one its powers, 4 bytes a lane; where a piece lies is the same for all lanes, what a lane takes of it the same for all pieces.
struct LaneParts {
  unsigned codes[(D + 127) / 128], powers;    // offsets from where the piece's key codes and key powers begin
};
__device__ __forceinline__ LaneParts parts_of_lane(int page_size) {
  LaneParts found;
  const int lane = threadIdx.x % WAVE;
#pragma unroll
  for (int i = 0; i < (D + 127) / 128; ++i) {
    const int unit = i * WAVE + lane;
    found.codes[i] = unit < D / 4 ? unit * 16 : page_size * (D / 2) + (unit - D / 4) * 16;
  }
  found.powers = lane < D / 16 ? lane * 4 : page_size * (D / 32) + (lane - D / 16) * 4;
  return found;
}

template <int SIZE> __device__ __forceinline__ void ask(const unsigned char* from, unsigned offset, unsigned char* to) {
  if constexpr (SIZE == 16) __builtin_amdgcn_global_load_lds((const void __attribute__((address_space(1)))*)(from + offset), (void __attribute__((address_space(3)))*)to, 16, 0, 0);
  else __builtin_amdgcn_global_load_lds((const void __attribute__((address_space(1)))*)(from + offset), (void __attribute__((address_space(3)))*)to, 4, 0, 0);
}

__device__ __forceinline__ void ask_step(unsigned char* stage, const unsigned char* from, const Walk& w, const Place& place, const LaneParts& parts) {
  const int lane = threadIdx.x % WAVE;
  const unsigned stride = (unsigned)w.kv_heads * (unsigned)(w.page_size * (D + D / 16));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned char* codes = from + (size_t)place.page.of[i] * stride + place.piece.of[i] * (4 * D);
#pragma unroll
    for (int j = 0; j < (D + 127) / 128; ++j)
      if ((j + 1) * WAVE <= D / 2 || j * WAVE + lane < D / 2) ask<16>(codes, parts.codes[j], stage + i * PIECE + j * WAVE * 16);
  }
  if (lane < D / 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned char* powers = from + (size_t)place.page.of[i] * stride + ((unsigned)w.page_size * D + place.piece.of[i] * (D / 4));
      ask<4>(powers, parts.powers, stage + 4 * PIECE + i * (D / 2));
    }
  }
}

template <int N> __device__ __forceinline__ void wait_for_asked() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// A step's codes and powers out of LDS.  The reads are written out, with the wait behind them: the compiler would have them wait for all that has been asked for.
__device__ __forceinline__ void read_step(Step& s, const unsigned char* stage) {
  const unsigned lane = threadIdx.x % WAVE, r = lane & 15, g = lane >> 4;
  const unsigned at = (unsigned)(size_t)(const unsigned char __attribute__((address_space(3)))*)stage;
  // key (r >> 2) * 8 + (r & 3) of tile 0, four further of tile 1
  const unsigned keys = at + (r >> 2) * PIECE + (r & 3) * (D / 2) + g * (D / 8), key_powers = at + 4 * PIECE + (r >> 2) * (D / 2) + (r & 3) * (D / 32);
  if constexpr (D == 128) {
    u32x4 k0, k1;
    asm volatile(
        "ds_read_b128 %0, %7\n\tds_read_u8 %2, %9\n\tds_read_b128 %1, %7 offset:256\n\tds_read_u8 %3, %9 offset:16\n\tds_read_b128 %4, %8\n\tds_read_b128 %5, %8 offset:16\n\tds_read_b64 %6, %10\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(k0), "=&v"(k1), "=&v"(s.key_powers[0][0]), "=&v"(s.key_powers[1][0]), "=&v"(s.values[0][0]), "=&v"(s.values[0][1]), "=&v"(s.value_powers[0])
        : "v"(keys), "v"(at + g * PIECE + 4 * D + r * 32), "v"(key_powers + g), "v"(at + 4 * PIECE + g * (D / 2) + D / 4 + (r >> 2) * 8)
        : "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s.keys[0][i] = k0[i];
      s.keys[1][i] = k1[i];
    }
  } else {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < SLICES; ++i) asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(s.keys[t][i]) : "v"(keys), "n"(t * 2 * D + i * 4) : "memory");
#pragma unroll
      for (int i = 0; i < KEY_POWERS; ++i) {
        const unsigned block = D % 128 == 0 ? g * KEY_POWERS + i : (g * SLICES + i) / 4;
        asm volatile("ds_read_u8 %0, %1 offset:%2" : "=v"(s.key_powers[t][i]) : "v"(key_powers + block), "n"(t * (D / 8)) : "memory");
      }
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const unsigned granule = chunk_first(c) / 8 + r * chunk_width(c) / 128, value = at + g * PIECE + 4 * D + granule * 32, power = at + 4 * PIECE + g * (D / 2) + D / 4 + granule / 4 * 8;
      asm volatile("ds_read_b128 %0, %1" : "=v"(s.values[c][0]) : "v"(value) : "memory");
      asm volatile("ds_read_b128 %0, %1 offset:16" : "=v"(s.values[c][1]) : "v"(value) : "memory");
      asm volatile("ds_read_b64 %0, %1" : "=v"(s.value_powers[c]) : "v"(power) : "memory");
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    // used only after the wait
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < SLICES; ++i) asm volatile("" : "+v"(s.keys[t][i]));
#pragma unroll
      for (int i = 0; i < KEY_POWERS; ++i) asm volatile("" : "+v"(s.key_powers[t][i]));
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) asm volatile("" : "+v"(s.values[c][0]), "+v"(s.values[c][1]), "+v"(s.value_powers[c]));
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

// What a wave keeps of its columns.
template <typename T, int CT> struct Columns {
  static constexpr int TERMS = sizeof(T) == 4 ? 3 : 1;
  Eight query[CT][TERMS][SLICES];
  int position[CT];                           // of the lane's column's token
  float reference[CT];                        // log2 of what weights are divided by
  f32x4 total[CT];                            // sums of weights, the same number four times
  f32x4 sum[CT][TILES];
};

__device__ __forceinline__ f32x4 multiply(const Eight& a, const Eight& b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0); }

__device__ __forceinline__ float largest_of(const float* x) { return fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))); }

// One step of 32 keys from `base` on.  EDGE: some column does not see some of them.
template <typename T, int CT, bool EDGE>
__device__ __forceinline__ void take_step(Columns<T, CT>& columns, const Step& now, const Walk& w, const Item& item, int base) {
  constexpr int TERMS = Columns<T, CT>::TERMS;
  const int lane = threadIdx.x % WAVE, r = lane & 15, g = lane >> 4;
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
        for (int k = TERMS - 1; k >= 0; --k) score[ct][t] = multiply(key, columns.query[ct][k][s], score[ct][t]);
    }
  }
  const auto sees = [&](int ct, int i) {
    const int key = base + 8 * g + i;
    return key <= columns.position[ct] && (w.window <= 0 || key > columns.position[ct] - w.window);
  };
  Eight weight[CT][TERMS];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    float x[8];  // log2 of the weights
    const auto relative = [&]() {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = __builtin_fmaf(score[ct][i / 4][i % 4], w.scale, -columns.reference[ct]);
        x[i] = !EDGE || sees(ct, i) ? y : -INFINITY;
      }
    };
    relative();
    if (__any(largest_of(x) > AHEAD)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = !EDGE || sees(ct, i) ? score[ct][i / 4][i % 4] * w.scale : -INFINITY;
      float largest = largest_of(x);
      largest = fmaxf(largest, __shfl_xor(largest, 16));
      largest = fmaxf(largest, __shfl_xor(largest, 32));
      largest = fmaxf(largest, columns.reference[ct]);
      const float change = columns.reference[ct] == largest ? 1.f : __builtin_amdgcn_exp2f(columns.reference[ct] - largest);
      columns.reference[ct] = largest;
      columns.total[ct] *= change;
#pragma unroll
      for (int t = 0; t < TILES; ++t) columns.sum[ct][t] *= change;
      relative();
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float y = __builtin_amdgcn_exp2f(x[i]);
      x[i] = !EDGE || sees(ct, i) ? y : 0.f;
    }
    split_eight<T, TERMS>(x, weight[ct]);
    // the weights that are multiplied are the weights that are added up: by a product with ones, over all 32 keys at once
    Eight ones;
    ones.u = (u32x4){0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
    for (int k = TERMS - 1; k >= 0; --k) columns.total[ct] = multiply(ones, weight[ct][k], columns.total[ct]);
  }
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int width = chunk_width(c), pairs = width / 32;  // pairs of elements that a lane takes of a key
    u32x2 powers = now.value_powers[c];
    bool poisoned = false;
    Eight marks;
    if (EDGE) {
      // A value that a column does not see has no part in it, whatever it is: keys that no column sees get the smallest power; of the
      // others, those that are no number are taken out, and put back where they are seen.
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
    float power[8];
    unsigned codes[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      power[j] = __uint_as_float(j % 4 == 3 ? powers[j / 4] >> 1 : powers[j / 4] << (23 - j % 4 * 8));  // (only the exponent of it counts)
      codes[j] = now.values[c][j / 4][j % 4];
      if (width == 64) codes[j] >>= (r & 1) * 16;
      if (width == 32) codes[j] >>= (r & 3) * 8;
    }
    const auto pair_of = [&](int j, int e) {
      return e == 0 ? unpack_pair<0>(codes[j], power[j]) : e == 1 ? unpack_pair<1>(codes[j], power[j]) : e == 2 ? unpack_pair<2>(codes[j], power[j]) : unpack_pair<3>(codes[j], power[j]);
    };
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e >= pairs) continue;
      Eight even, odd;                          // elements 2 e and 2 e + 1 of the lane's, of its eight keys
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned a = pair_of(2 * j, e), b = pair_of(2 * j + 1, e);
        even.u[j] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        odd.u[j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      }
      const int t = chunk_first(c) / 16 + 2 * e;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int k = TERMS - 1; k >= 0; --k) {
          columns.sum[ct][t] = multiply(even, weight[ct][k], columns.sum[ct][t]);
          columns.sum[ct][t + 1] = multiply(odd, weight[ct][k], columns.sum[ct][t + 1]);
        }
    }
    if (EDGE && poisoned) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        Eight seen;
#pragma unroll
        for (int i = 0; i < 8; ++i) seen.v[i] = (bf16_t)(sees(ct, i) ? 1.f : 0.f);
        const f32x4 hit = multiply(marks, seen, (f32x4){0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (e >= 2 * pairs) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (hit[i] > 0.f) columns.sum[ct][chunk_first(c) / 16 + e][i] = __uint_as_float(0x7fc00000u);
        }
      }
    }
  }
}

template <typename T, int CT>
__global__ void __launch_bounds__(WAVES * WAVE, 2) packed_attention_kernel(const T* q, int q_stride, T* out, int out_stride, float* partial, const unsigned char* pages, Walk w, int items, int whole) {
  constexpr int TERMS = sizeof(T) == 4 ? 3 : 1;
  constexpr int RING = WAVES * STAGES * STAGE, RESULTS = WAVES * 16 * (D + 4) * 4;
  __shared__ __attribute__((aligned(16))) unsigned char memory[RING > RESULTS ? RING : RESULTS];  // the steps' codes, and the waves' sums behind them
  float (*results)[16][D + 4] = (float (*)[16][D + 4])memory;
  __shared__ float sums[WAVES][16][2];
  const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), r = lane & 15, g = lane >> 4;
  // the longest walks begin first: a request's last columns walk most keys
  const int all = items * w.kv_heads, at = blockIdx.x % all, split = blockIdx.x / all;
  const int kv_head = at % w.kv_heads;
  Item item;
  if (!find_item(w, items - 1 - at / w.kv_heads, 16 * CT, item)) return;
  // as many parts as it takes, all of one length
  const int parts = (item.to - item.from + w.chunk - 1) / w.chunk;
  if (split >= parts) return;
  const int each = ((item.to - item.from + parts - 1) / parts + WAVES * KEYS - 1) / (WAVES * KEYS) * (WAVES * KEYS);
  const int begin = item.from + split * each, end = min(item.to, begin + each);
  const unsigned char* from = pages + (size_t)kv_head * (w.page_size * (D + D / 16));
  Scalar* table = (Scalar*)w.tables + (size_t)item.request * w.table_width;

  unsigned char* ring = memory + wave * (STAGES * STAGE);
  const LaneParts lane_parts = parts_of_lane(w.page_size);
  const int own = __builtin_amdgcn_readfirstlane(begin + wave * KEYS);
  Place place;
  int asked = own;
#pragma unroll
  for (int s = 0; s < STAGES; ++s)
    if (asked < end) {
      find_place(place, w, table, asked);
      ask_step(ring + s * STAGE, from, w, place, lane_parts);
      asked += WAVES * KEYS;
    }
  if (asked < end) find_place(place, w, table, asked);
  Columns<T, CT> columns;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int column = min(ct * 16 + r, item.columns - 1), flat = item.first + column, token = flat / item.group;
    columns.position[ct] = item.first_position - item.first / item.group + token;
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
      for (int k = 0; k < TERMS; ++k) columns.query[ct][k][s] = terms[k];
    }
    columns.reference[ct] = -INFINITY;
    columns.total[ct] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < TILES; ++t) columns.sum[ct][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }

  // (the queries have come, and with them what was asked for before: from here on the loads that are counted are those of steps)
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int k = 0; k < TERMS; ++k)
#pragma unroll
      for (int s = 0; s < SLICES; ++s) asm volatile("" : "+v"(columns.query[ct][k][s].u));
  wait_for_asked<0>();
  int stage = 0, base = own;
  const auto next_step = [&](Step& now) {
    if (base + (STAGES - 1) * WAVES * KEYS < end) wait_for_asked<(STAGES - 1) * ASKS>();
    else wait_for_asked<0>();
    read_step(now, ring + stage * STAGE);
    if (asked < end) {
      ask_step(ring + stage * STAGE, from, w, place, lane_parts);
      asked += WAVES * KEYS;
      if (asked < end) find_place(place, w, table, asked);
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  };
  // the steps that all columns see whole lie side by side
  const int whole_from = w.window > 0 ? item.last_position - w.window + 1 : 0, whole_to = min(end, item.first_position - KEYS + 2);
  for (; base < end; base += WAVES * KEYS) {
    for (; base >= whole_from && base < whole_to; base += WAVES * KEYS) {
      Step now;
      next_step(now);
      take_step<T, CT, false>(columns, now, w, item, base);
    }
    if (base >= end) break;
    Step now;
    next_step(now);
    take_step<T, CT, true>(columns, now, w, item, base);
  }

  // the waves' sums, brought together
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (ct * 16 >= item.columns) break;
    __syncthreads();
    if (g == 0) {
      sums[wave][r][0] = columns.reference[ct];
      sums[wave][r][1] = columns.total[ct][0];
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int each = chunk_width(c) / 16;  // neighbouring elements of a row of the tiles
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < each) results[wave][r][chunk_first(c) + (4 * g + i) * each + e] = columns.sum[ct][chunk_first(c) / 16 + e][i];
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
        if (d == 0 && w.splits > 1) partial[(row * w.heads + head) * w.splits * (D + 4) + D + 2] = __int_as_float(1);
      } else {
        float* to = partial + ((row * w.heads + head) * w.splits + split) * (D + 4);
        *(f32x4*)(to + d) = result;
        if (d == 0) *(f32x4*)(to + D) = (f32x4){largest, weights, __int_as_float(parts), 0.f};
      }
    }
  }
}

// A wave a (token, head) whose keys were split: its parts joined.  A part is D sums, the reference that their weights are relative to, the weights' sum, and
// (in the first one) how many parts there are; all of them are asked for at once.
constexpr int JOIN_LANES = D / 4, JOINED = WAVE / JOIN_LANES;  // lanes a part, parts side by side
constexpr int MOST_PARTS = WAVE;

template <typename T>
__global__ void __launch_bounds__(WAVE) packed_join_kernel(T* out, int out_stride, const float* partial, const int* query_start, int requests, int heads, int splits) {
  const int token = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
  const float* mine = partial + ((size_t)token * heads + head) * splits * (D + 4);
  const int tokens = query_start[requests], parts = min(__float_as_int(mine[D + 2]), splits);
  if (token >= tokens || parts <= 1) return;
  const int which = min(lane / JOIN_LANES, JOINED - 1), d = lane % JOIN_LANES * 4;
  float reference = -INFINITY, total = 0.f;
  if (lane < parts) {
    reference = mine[lane * (D + 4) + D];
    total = mine[lane * (D + 4) + D + 1];
  }
  const float largest = wave_max(reference), share = reference == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(reference - largest);
  f32x4 result = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = 0; i < parts; i += JOINED) {
    const float weight = __shfl(share, min(i + which, WAVE - 1));
    if (i + which < parts) result += weight * *(const f32x4*)(mine + (i + which) * (D + 4) + d);
  }
  const float weights = wave_sum(share * total);
#pragma unroll
  for (int other = 1; other < JOINED; ++other)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float far = __shfl(result[i], min(lane + other * JOIN_LANES, WAVE - 1));
      if (lane < JOIN_LANES) result[i] += far;
    }
  if (lane >= JOIN_LANES) return;
  const float over = 1.f / weights;
#pragma unroll
  for (int i = 0; i < 4; ++i) out[(size_t)token * out_stride + head * D + d + i] = from_float<T>(result[i] * over);
}

template <typename T>
static int launch(const void* q, int q_stride, void* out, int out_stride, float* partial, const void* pages, const Walk& w, int tokens, int column_tiles, hipStream_t stream) {
  const int group = w.heads / w.kv_heads, most = 16 * column_tiles;
  const long items = w.single ? (long)w.requests * ((group + most - 1) / most) : ((long)tokens * group + most - 1) / most + w.requests;
  const long blocks = items * w.kv_heads * w.splits;
  if (items >= (1L << 31) || blocks >= (1L << 31)) return ERR_BAD_ARGUMENT;
  const int piece = sizeof(T) == 4 ? 4 : 8, whole = (size_t)q % 16 == 0 && q_stride % piece == 0;
  if (column_tiles == 1)
    packed_attention_kernel<T, 1><<<(unsigned)blocks, WAVES * WAVE, 0, stream>>>((const T*)q, q_stride, (T*)out, out_stride, partial, (const unsigned char*)pages, w, (int)items, whole);
  else
    packed_attention_kernel<T, 2><<<(unsigned)blocks, WAVES * WAVE, 0, stream>>>((const T*)q, q_stride, (T*)out, out_stride, partial, (const unsigned char*)pages, w, (int)items, whole);
  if (int status = LAUNCH_STATUS()) return status;
  if (w.splits > 1) packed_join_kernel<T><<<dim3(tokens, w.heads), WAVE, 0, stream>>>((T*)out, out_stride, partial, w.query_start, w.requests, w.heads, w.splits);
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
      !packed_fits(D, page_size) || (long)page_size * D * kv_heads >= (1L << 30) || !(scale > 0.f) || (size_t)pages % 16 || q_stride < heads * D || out_stride < heads * D || window < 0 || column_tiles < 1 || column_tiles > 2 || chunk < 128 || chunk % 128 ||
      splits < 1 || splits > MOST_PARTS || (splits > 1 && (!partial || (size_t)partial % 16)) || heads > 65535)
    return ERR_BAD_ARGUMENT;
  const unsigned per_page = (unsigned)page_size / 8;
  const bool power_of_two = (per_page & (per_page - 1)) == 0;
  // (a quotient by the reciprocal is exact below 2^32 over the divisor)
  if (!power_of_two && (unsigned long)(table_width + 1) * per_page * per_page >= (1UL << 32)) return ERR_BAD_ARGUMENT;
  const Walk w = {tables, table_width, num_pages, page_size, power_of_two ? 31 - __builtin_clz(per_page) : -1, (unsigned)(((1UL << 32) + per_page - 1) / per_page), query_start, contexts, requests, heads, kv_heads, window, single, chunk, splits, scale * LOG2_E};
  if (is_float) return launch<float>(q, q_stride, out, out_stride, (float*)partial, pages, w, tokens, column_tiles, stream);
  return launch<bf16_t>(q, q_stride, out, out_stride, (float*)partial, pages, w, tokens, column_tiles, stream);
}
