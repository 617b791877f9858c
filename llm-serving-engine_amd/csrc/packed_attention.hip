// Grouped-query attention over pages in 4 bits (packed.h), softmax in float32.  Compiled once per head size.
//
// A workgroup takes a run of columns, the (token, query head) pairs of one request that share a kv head: 16 of them where they are few, and its waves take steps
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
//
// A bfloat16 run takes the weights in one term: they are rounded to bfloat16, to nearest, once, because the second product's matrix instructions take bfloat16 and a second term would be
// the same product again for what is left (over single tokens 2 to 7 % of a call: 64 at 2,048 to 6,144 keys 39.4 -> 42.1 us, 8 at 15,000 to 45,000 63.3 -> 64.8).  The rounded weights are also what is added up, so weights that the division leaves add up to 1, and sums, references and parts that are joined
// stay float32.  Results are off by 0.0018 to 0.0022 of their size against 64 bits (root mean square) where float32 weights leave 0.0015 to 0.0017, which is the rounding of the result alone; what 4 bits
// leave of normally distributed rows is off by 0.11.  The same holds for the framework's attention over pages in bfloat16.
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
constexpr int WAVES = 8;                      // of a workgroup over single tokens
constexpr int UNIT = WAVES * KEYS;            // keys that its waves take side by side: what work is counted in
constexpr int STAGES = 2;                     // steps that a wave has asked for
constexpr int PIECE = 8 * D + 16;             // bytes in LDS of the codes of eight keys and values (16 spare: the same rows of two pieces lie in other banks)
constexpr int STAGE = 4 * PIECE + 2 * D;      // of a step: four pieces, and their powers
constexpr int ASKS = 4 * ((D + 127) / 128 + 1);  // loads of a step
constexpr float AHEAD = 8.f;                  // log2 units that a score may run ahead of its column's reference before the sums are rescaled
constexpr float LOWEST = -3.402823466e38f;    // a column's reference before it has seen a score (finite: one that overflowed to minus infinity has a weight of 0 beside it)
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
  int requests, heads, kv_heads, window;
  float scale;                                // times log2 e
  bool together;                              // those of few columns go with the others
};

struct Item {                                 // a run of columns
  int request, first_row, group, first, columns, first_position, last_position, from, to;
};

// Few columns: those of a single token, or of some that fit one tile of 16.
__device__ __forceinline__ bool few_columns(const Walk& w, int count, int group) { return !w.together && (count == 1 || count * group <= 16); }

struct Request {
  int start, count, context;                  // rows in the step, keys behind it
};
__device__ __forceinline__ Request load_request(const Walk& w, int request) {
  const int start = w.query_start[request];
  return {start, w.query_start[request + 1] - start, w.contexts[request]};
}

// The run of up to `most` columns from `first` on of a request.  False: it has none there.
__device__ __forceinline__ bool make_item(const Walk& w, int index, const Request& request, int first, int most, Item& item) {
  const int group = w.heads / w.kv_heads;
  item.request = index;
  item.group = group;
  item.first = first;
  item.columns = min(most, request.count * group - first);
  item.first_row = request.start;
  const int past = request.context - request.count;
  item.first_position = past + first / group;
  item.last_position = past + (first + item.columns - 1) / group;
  item.from = w.window > 0 ? max(0, item.first_position - w.window + 1) / KEYS * KEYS : 0;
  item.to = item.last_position + 1;
  return item.columns > 0 && item.to > item.from;
}

// Item `index` of the requests of many columns, in runs of `most`, one request's behind the other's.  False: there is no such item.  (each wave for itself, 64 requests at a time)
__device__ __forceinline__ bool find_item(const Walk& w, int index, int most, Item& item) {
  const int lane = threadIdx.x % WAVE, group = w.heads / w.kv_heads;
  int before = 0;
  for (int base = 0; base < w.requests; base += WAVE) {
    const int b = base + lane;
    Request mine = {0, 0, 0};                 // (asked for at once: the walk's first keys wait for every trip to memory before them)
    if (b < w.requests) mine = load_request(w, b);
    const int count = mine.count;
    const int items = few_columns(w, count, group) ? 0 : (count * group + most - 1) / most;
    int sum = items;
#pragma unroll
    for (int step = 1; step < WAVE; step <<= 1) {
      const int other = __shfl_up(sum, step);
      if (lane >= step) sum += other;
    }
    const unsigned long long found = __ballot(before + sum > index);
    if (found) {
      const int which = __ffsll((unsigned long long)found) - 1, inside = index - before - __shfl(sum - items, which);
      const Request request = {__builtin_amdgcn_readfirstlane(__shfl(mine.start, which)), __builtin_amdgcn_readfirstlane(__shfl(count, which)), __builtin_amdgcn_readfirstlane(__shfl(mine.context, which))};
      return make_item(w, __builtin_amdgcn_readfirstlane(base + which), request, __builtin_amdgcn_readfirstlane(inside) * most, most, item);
    }
    before += __shfl(sum, WAVE - 1);
  }
  return false;
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

// Behind a step's last product: the compiler may begin the next block of instructions with moves of the sums (it did, from accumulator registers, at heads wider than 128), and
// keeps the distance that a product's result needs (8 instructions, 12 of the 32 x 32 ones) within a block only.
__device__ __forceinline__ void products_done() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <int N> __device__ __forceinline__ void wait_for_asked() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// A step's codes and powers out of LDS.  The reads are written out, with the wait behind them: the compiler would have them wait for all that has been asked for.  A block of them ends
// with its wait, so that no register is moved, or given to something else, before what is read into it has come.
#define WORDS_1 "ds_read_b32 %[w0], %[keys]\n\t"
#define WORDS_2 WORDS_1 "ds_read_b32 %[w1], %[keys] offset:4\n\t"
#define WORDS_3 WORDS_2 "ds_read_b32 %[w2], %[keys] offset:8\n\t"
#define WORDS_4 WORDS_3 "ds_read_b32 %[w3], %[keys] offset:12\n\t"
#define WORDS_5 WORDS_4 "ds_read_b32 %[w4], %[keys] offset:16\n\t"
#define WORDS_6 WORDS_5 "ds_read_b32 %[w5], %[keys] offset:20\n\t"
#define WORDS_7 WORDS_6 "ds_read_b32 %[w6], %[keys] offset:24\n\t"
#define WORDS_8 WORDS_7 "ds_read_b32 %[w7], %[keys] offset:28\n\t"
#define BYTES_1 "ds_read_u8 %[b0], %[a0]\n\t"
#define BYTES_2 BYTES_1 "ds_read_u8 %[b1], %[a1]\n\t"
#define BYTES_3 BYTES_2 "ds_read_u8 %[b2], %[a2]\n\t"
#define BYTES_5 BYTES_3 "ds_read_u8 %[b3], %[a3]\n\tds_read_u8 %[b4], %[a4]\n\t"
#define BYTES_6 BYTES_5 "ds_read_u8 %[b5], %[a5]\n\t"
#define BYTES_7 BYTES_6 "ds_read_u8 %[b6], %[a6]\n\t"
#define TO_WORDS_1 [w0] "=&v"(words[0])
#define TO_WORDS_2 TO_WORDS_1, [w1] "=&v"(words[1])
#define TO_WORDS_3 TO_WORDS_2, [w2] "=&v"(words[2])
#define TO_WORDS_4 TO_WORDS_3, [w3] "=&v"(words[3])
#define TO_WORDS_5 TO_WORDS_4, [w4] "=&v"(words[4])
#define TO_WORDS_6 TO_WORDS_5, [w5] "=&v"(words[5])
#define TO_WORDS_7 TO_WORDS_6, [w6] "=&v"(words[6])
#define TO_WORDS_8 TO_WORDS_7, [w7] "=&v"(words[7])
#define TO_BYTES_1 [b0] "=&v"(bytes[0])
#define TO_BYTES_2 TO_BYTES_1, [b1] "=&v"(bytes[1])
#define TO_BYTES_3 TO_BYTES_2, [b2] "=&v"(bytes[2])
#define TO_BYTES_5 TO_BYTES_3, [b3] "=&v"(bytes[3]), [b4] "=&v"(bytes[4])
#define TO_BYTES_6 TO_BYTES_5, [b5] "=&v"(bytes[5])
#define TO_BYTES_7 TO_BYTES_6, [b6] "=&v"(bytes[6])
#define AT_1 [a0] "v"(at[0])
#define AT_2 AT_1, [a1] "v"(at[1])
#define AT_3 AT_2, [a2] "v"(at[2])
#define AT_5 AT_3, [a3] "v"(at[3]), [a4] "v"(at[4])
#define AT_6 AT_5, [a5] "v"(at[5])
#define AT_7 AT_6, [a6] "v"(at[6])
#define READ_KEY(w, b) asm volatile(WORDS_##w BYTES_##b "s_waitcnt lgkmcnt(0)" : TO_WORDS_##w, TO_BYTES_##b : [keys] "v"(keys), AT_##b : "memory")
template <int W, int B> __device__ __forceinline__ void read_key(unsigned (&words)[W], unsigned (&bytes)[B], unsigned keys, const unsigned (&at)[B]) {
  if constexpr (W == 1 && B == 1) READ_KEY(1, 1);
  else if constexpr (W == 2 && B == 1) READ_KEY(2, 1);
  else if constexpr (W == 3 && B == 3) READ_KEY(3, 3);
  else if constexpr (W == 5 && B == 5) READ_KEY(5, 5);
  else if constexpr (W == 6 && B == 6) READ_KEY(6, 6);
  else if constexpr (W == 7 && B == 7) READ_KEY(7, 7);
  else {
    static_assert(W == 8 && B == 2, "heads of 32 to 256 in steps of 32, but for 128");
    READ_KEY(8, 2);
  }
}

#define VALUE(i) "ds_read_b128 %[l" #i "], %[v" #i "]\n\tds_read_b128 %[h" #i "], %[v" #i "] offset:16\n\tds_read_b64 %[b" #i "], %[a" #i "]\n\t"
#define TO_VALUE(i) [l##i] "=&v"(low[i]), [h##i] "=&v"(high[i]), [b##i] "=&v"(powers[i])
#define VALUE_AT(i) [v##i] "v"(values[i]), [a##i] "v"(at[i])
// N times eight keys' codes of a granule, and their powers
template <int N> __device__ __forceinline__ void read_values(u32x4 (&low)[N], u32x4 (&high)[N], u32x2 (&powers)[N], const unsigned (&values)[N], const unsigned (&at)[N]) {
  if constexpr (N == 1) asm volatile(VALUE(0) "s_waitcnt lgkmcnt(0)" : TO_VALUE(0) : VALUE_AT(0) : "memory");
  else if constexpr (N == 2) asm volatile(VALUE(0) VALUE(1) "s_waitcnt lgkmcnt(0)" : TO_VALUE(0), TO_VALUE(1) : VALUE_AT(0), VALUE_AT(1) : "memory");
  else if constexpr (N == 3)
    asm volatile(VALUE(0) VALUE(1) VALUE(2) "s_waitcnt lgkmcnt(0)" : TO_VALUE(0), TO_VALUE(1), TO_VALUE(2) : VALUE_AT(0), VALUE_AT(1), VALUE_AT(2) : "memory");
  else {
    static_assert(N == 4, "three chunks, or two of two pieces");
    asm volatile(VALUE(0) VALUE(1) VALUE(2) VALUE(3) "s_waitcnt lgkmcnt(0)"
                 : TO_VALUE(0), TO_VALUE(1), TO_VALUE(2), TO_VALUE(3) : VALUE_AT(0), VALUE_AT(1), VALUE_AT(2), VALUE_AT(3) : "memory");
  }
}

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
    unsigned powers[KEY_POWERS];
#pragma unroll
    for (int i = 0; i < KEY_POWERS; ++i) powers[i] = key_powers + (D % 128 == 0 ? g * KEY_POWERS + i : (g * SLICES + i) / 4);
    read_key(s.keys[0], s.key_powers[0], keys, powers);
#pragma unroll
    for (int i = 0; i < KEY_POWERS; ++i) powers[i] += D / 8;
    read_key(s.keys[1], s.key_powers[1], keys + 2 * D, powers);
    u32x4 low[CHUNKS], high[CHUNKS];
    unsigned values[CHUNKS], value_powers[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const unsigned granule = chunk_first(c) / 8 + r * chunk_width(c) / 128;
      values[c] = at + g * PIECE + 4 * D + granule * 32;
      value_powers[c] = at + 4 * PIECE + g * (D / 2) + D / 4 + granule / 4 * 8;
    }
    read_values(low, high, s.value_powers, values, value_powers);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      s.values[c][0] = low[c];
      s.values[c][1] = high[c];
    }
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
template <typename T> struct Columns {
  static constexpr int TERMS = sizeof(T) == 4 ? 3 : 1;
  Eight query[TERMS][SLICES];
  int position;                               // of the lane's column's token
  float reference;                            // log2 of what weights are divided by
  f32x4 total;                                // sums of weights, the same number four times
  f32x4 sum[TILES];
};

__device__ __forceinline__ f32x4 multiply(const Eight& a, const Eight& b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0); }

__device__ __forceinline__ float largest_of(const float* x) { return fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))); }

// One step of 32 keys from `base` on.  EDGE: some column does not see some of them.
template <bool EDGE, typename T>
__device__ __forceinline__ void take_step(Columns<T>& columns, const Step& now, const Walk& w, const Item& item, int base) {
  constexpr int TERMS = Columns<T>::TERMS;
  const int lane = threadIdx.x % WAVE, r = lane & 15, g = lane >> 4;
  // scores: row 4 g + i of tile t is key 8 g + 4 t + i of the step
  f32x4 score[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    score[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < SLICES; ++s) {
      const float power = packed_power(now.key_powers[t][D % 128 == 0 ? s / 4 : D <= 64 ? 0 : s]);
      Eight key;
      key.u = (u32x4){unpack_pair<0>(now.keys[t][s], power), unpack_pair<1>(now.keys[t][s], power), unpack_pair<2>(now.keys[t][s], power), unpack_pair<3>(now.keys[t][s], power)};
#pragma unroll
      for (int k = TERMS - 1; k >= 0; --k) score[t] = multiply(key, columns.query[k][s], score[t]);
    }
  }
  const auto sees = [&](int i) {
    const int key = base + 8 * g + i;
    return key <= columns.position && (w.window <= 0 || key > columns.position - w.window);
  };
  Eight weight[TERMS];
  float x[8];  // log2 of the weights
  const auto relative = [&]() {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float y = __builtin_fmaf(score[i / 4][i % 4], w.scale, -columns.reference);
      x[i] = !EDGE || sees(i) ? y : -INFINITY;
    }
  };
  relative();
  if (__any(largest_of(x) > AHEAD)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = !EDGE || sees(i) ? score[i / 4][i % 4] * w.scale : -INFINITY;
    float largest = largest_of(x);
    largest = fmaxf(largest, __shfl_xor(largest, 16));
    largest = fmaxf(largest, __shfl_xor(largest, 32));
    largest = fmaxf(largest, columns.reference);
    const float change = columns.reference == largest ? 1.f : __builtin_amdgcn_exp2f(columns.reference - largest);
    columns.reference = largest;
    columns.total *= change;
#pragma unroll
    for (int t = 0; t < TILES; ++t) columns.sum[t] *= change;
    relative();
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = __builtin_amdgcn_exp2f(x[i]);
    x[i] = !EDGE || sees(i) ? y : 0.f;
  }
  split_eight<T, TERMS>(x, weight);           // (bfloat16: rounded here, once, as the matrix instructions take them)
  // the weights that are multiplied are the weights that are added up: by a product with ones, over all 32 keys at once
  Eight ones;
  ones.u = (u32x4){0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
  for (int k = TERMS - 1; k >= 0; --k) columns.total = multiply(ones, weight[k], columns.total);
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
      for (int k = TERMS - 1; k >= 0; --k) {
        columns.sum[t] = multiply(even, weight[k], columns.sum[t]);
        columns.sum[t + 1] = multiply(odd, weight[k], columns.sum[t + 1]);
      }
    }
    if (EDGE && poisoned) {
      Eight seen;
#pragma unroll
      for (int i = 0; i < 8; ++i) seen.v[i] = (bf16_t)(sees(i) ? 1.f : 0.f);
      const f32x4 hit = multiply(marks, seen, (f32x4){0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (e >= 2 * pairs) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (hit[i] > 0.f) columns.sum[chunk_first(c) / 16 + e][i] = __uint_as_float(0x7fc00000u);
      }
    }
  }
}

// Rows in memory as a wave's queries.
template <typename T>
__device__ __forceinline__ void load_queries(Columns<T>& columns, const T* q, int q_stride, const Item& item, int kv_head, bool whole) {
  constexpr int TERMS = Columns<T>::TERMS;
  const int lane = threadIdx.x % WAVE, r = lane & 15, g = lane >> 4;
  const int column = min(r, item.columns - 1), flat = item.first + column, token = flat / item.group;
  columns.position = item.first_position - item.first / item.group + token;
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
    for (int k = 0; k < TERMS; ++k) columns.query[k][s] = terms[k];
  }
  columns.reference = LOWEST;
  columns.total = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int t = 0; t < TILES; ++t) columns.sum[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
}

// What a wave holds of its queries stays in registers from here on.
template <typename T> __device__ __forceinline__ void settle(Columns<T>& columns) {
#pragma unroll
  for (int k = 0; k < Columns<T>::TERMS; ++k)
#pragma unroll
    for (int s = 0; s < SLICES; ++s) asm volatile("" : "+v"(columns.query[k][s].u));
}

// A wave's steps of the keys begin .. end (begin a multiple of 32): every W-th from its own on.  ring: STAGES stages of LDS that are its own.
template <typename T, typename Taken, int W, typename Cols>
__device__ __forceinline__ void walk_keys(Cols& columns, const T* q, int q_stride, const unsigned char* pages, const Walk& w, const Item& item, int kv_head, bool whole, int begin, int end, int wave, unsigned char* ring) {
  const unsigned char* from = pages + (size_t)kv_head * (w.page_size * (D + D / 16));
  Scalar* table = (Scalar*)w.tables + (size_t)item.request * w.table_width;
  const LaneParts lane_parts = parts_of_lane(w.page_size);
  Place place;
  int base = __builtin_amdgcn_readfirstlane(begin + wave * KEYS), asked = base, stage = 0;
#pragma unroll
  for (int s = 0; s < STAGES; ++s)
    if (asked < end) {
      find_place(place, w, table, asked);
      ask_step(ring + s * STAGE, from, w, place, lane_parts);
      asked += W * KEYS;
    }
  if (asked < end) find_place(place, w, table, asked);
  load_queries(columns, q, q_stride, item, kv_head, whole);
  // (the queries have come, and with them what was asked for before: from here on the loads that are counted are those of steps)
  settle(columns);
  wait_for_asked<0>();
  const auto next_step = [&](Taken& now) {
    if (base + (STAGES - 1) * W * KEYS < end) wait_for_asked<(STAGES - 1) * ASKS>();
    else wait_for_asked<0>();
    read_step(now, ring + stage * STAGE);
    if (asked < end) {
      ask_step(ring + stage * STAGE, from, w, place, lane_parts);
      asked += W * KEYS;
      if (asked < end) find_place(place, w, table, asked);
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  };
  // the steps that all columns see whole lie side by side
  const int whole_from = w.window > 0 ? item.last_position - w.window + 1 : 0, whole_to = min(end, item.first_position - KEYS + 2);
  for (; base < end; base += W * KEYS) {
    for (; base >= whole_from && base < whole_to; base += W * KEYS) {
      Taken now;
      next_step(now);
      take_step<false>(columns, now, w, item, base);
      products_done();
    }
    if (base >= end) break;
    Taken now;
    next_step(now);
    take_step<true>(columns, now, w, item, base);
    products_done();
  }
}

// What W waves have of up to 16 columns, joined: take(column, d, four sums from element d on, the weights' reference, their sum).
template <int W, typename Take>
__device__ __forceinline__ void join_waves(const float (*results)[16][D + 4], const float (*sums)[16][2], int count, Take take) {
  for (int at = threadIdx.x; at < count * (D / 4); at += W * WAVE) {
    const int column = at / (D / 4), d = (at - column * (D / 4)) * 4;
    float largest = sums[0][column][0];
#pragma unroll
    for (int v = 1; v < W; ++v) largest = fmaxf(largest, sums[v][column][0]);
    f32x4 result = (f32x4){0.f, 0.f, 0.f, 0.f};
    float weights = 0.f;
#pragma unroll
    for (int v = 0; v < W; ++v) {
      const float share = sums[v][column][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sums[v][column][0] - largest);
      weights += share * sums[v][column][1];
      result += share * *(const f32x4*)&results[v][column][d];
    }
    take(column, d, result, largest, weights);
  }
}

// The sums of W waves, brought together through LDS.  memory: W * 16 * (D + 6) floats, free when all waves have come here.
template <int W, typename T, typename Take>
__device__ __forceinline__ void bring_together(const Columns<T>& columns, int count, int wave, unsigned char* memory, Take take) {
  float (*results)[16][D + 4] = (float (*)[16][D + 4])memory;
  float (*sums)[16][2] = (float (*)[16][2])(memory + W * 16 * (D + 4) * 4);
  const int lane = threadIdx.x % WAVE, r = lane & 15, g = lane >> 4;
  __syncthreads();
  if (g == 0) {
    sums[wave][r][0] = columns.reference;
    sums[wave][r][1] = columns.total[0];
  }
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int each = chunk_width(c) / 16;  // neighbouring elements of a row of the tiles
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < each) results[wave][r][chunk_first(c) + (4 * g + i) * each + e] = columns.sum[chunk_first(c) / 16 + e][i];
  }
  __syncthreads();
  join_waves<W>(results, sums, count, take);
}

template <typename T> __device__ __forceinline__ void write_four(T* to, f32x4 x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) to[i] = from_float<T>(x[i]);
}

template <int W> constexpr int memory_of() {
  constexpr int RING = W * STAGES * STAGE, RESULTS = W * 16 * (D + 6) * 4;
  return RING > RESULTS ? RING : RESULTS;
}

// ---------------------------------------------------------------------------------------------------------------- few columns
//
// Single tokens read all their keys for a handful of columns: the path from memory is what bounds them.  The walks of all (request, tile of 16 columns, kv
// head) lie behind each other, counted in units of 256 keys, and every workgroup takes an equal run of units, wherever in a walk it begins or ends: ragged contexts leave no workgroup
// with more than another.  A walk that one workgroup takes whole is written as it ends.  Of one that is cut every workgroup leaves its part, in a place of its
// own: a workgroup has at most two such, the one that it begins with (place 0) and the one that it breaks off (place 1); who begins a
// walk and breaks it off notes it for the join.  64 tokens over 2,048 to 6,144 keys (4,096 in the mean) at
// 28/4 heads of 128, whole: 37 us, 144 MB at 3.9 TB/s: the longest walk, which one workgroup takes at 4.7 us for 1,000 keys, and its beginning and end.  Cut, all walks together take 27 us, but the joining and what
// goes with it 13.  8 over 15,000 to 45,000 (30,000 in the mean) at 40/8, cut: 49 us, 5.3 TB/s, and 4 for the join.
struct Cut {
  int first_row, group, first, columns, kv_head, parts, place, spare;  // parts 0: none; place: of the first part, the others lie at place 0 of the workgroups behind
};
constexpr int PART = 16 * (D + 4);  // floats of a part: 16 columns of D sums, their reference, the sum of their weights, two spare

struct Streams {
  float* parts;                               // [workgroups][2][PART]
  Cut* cuts;                                  // [workgroups]
  int least;                                  // units a workgroup takes at least; 0: a workgroup takes one walk whole
};

__device__ __forceinline__ int units_of(const Walk& w, const Request& request) {  // of all its columns and kv heads
  const int group = w.heads / w.kv_heads;
  Item item;
  if (!few_columns(w, request.count, group) || !make_item(w, 0, request, 0, 1 << 20, item)) return 0;
  return (item.to - item.from + UNIT - 1) / UNIT * ((request.count * group + 15) / 16) * w.kv_heads;
}

template <typename T>
__global__ void __launch_bounds__(WAVES * WAVE, 2) packed_streams_kernel(const T* q, int q_stride, T* out, int out_stride, const unsigned char* pages, Walk w, Streams streams, int whole) {
  __shared__ __attribute__((aligned(16))) unsigned char memory[memory_of<WAVES>()];
  __shared__ int ends[WAVES * WAVE];          // units of the requests up to a thread's
  __shared__ Request held[WAVES * WAVE];      // the requests, if there are no more than threads
  __shared__ int wave_sums[WAVES];
  const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), group = w.heads / w.kv_heads;
  unsigned char* ring = memory + wave * (STAGES * STAGE);
  const auto take_walk = [&](const Item& item, int kv_head, int begin, int end, float* part) {
    Columns<T> columns;
    walk_keys<T, Step, WAVES>(columns, q, q_stride, pages, w, item, kv_head, whole, begin, end, wave, ring);
    bring_together<WAVES>(columns, item.columns, wave, memory, [&](int column, int d, f32x4 result, float largest, float weights) {
      if (part) {
        *(f32x4*)(part + column * (D + 4) + d) = result;
        if (d == 0) *(f32x4*)(part + column * (D + 4) + D) = (f32x4){largest, weights, 0.f, 0.f};
      } else {
        const int flat = item.first + column, token = flat / item.group, head = kv_head * item.group + flat - token * item.group;
        write_four(out + (size_t)(item.first_row + token) * out_stride + head * D + d, result * (1.f / weights));
      }
    });
  };
  if (streams.least == 0) {
    const int tiles = (group + 15) / 16, request = blockIdx.x / (tiles * w.kv_heads), inside = blockIdx.x - request * (tiles * w.kv_heads);
    const Request mine = load_request(w, request);
    Item item;
    if (!few_columns(w, mine.count, group) || !make_item(w, request, mine, inside / w.kv_heads * 16, 16, item)) return;
    take_walk(item, inside % w.kv_heads, item.from, item.to, nullptr);
    return;
  }
  // where the requests' units end: a run of requests a thread, the threads' sums added up
  const int run = (w.requests + WAVES * WAVE - 1) / (WAVES * WAVE), first_request = threadIdx.x * run;
  int mine = 0;
  for (int b = first_request; b < min(first_request + run, w.requests); ++b) {
    const Request request = load_request(w, b);
    mine += units_of(w, request);
    if (run == 1) held[b] = request;
  }
#pragma unroll
  for (int step = 1; step < WAVE; step <<= 1) {
    const int other = __shfl_up(mine, step);
    if (lane >= step) mine += other;
  }
  if (lane == WAVE - 1) wave_sums[wave] = mine;
  __syncthreads();
  for (int v = 0; v < wave; ++v) mine += wave_sums[v];
  ends[threadIdx.x] = mine;
  __syncthreads();
  const int total = __builtin_amdgcn_readfirstlane(ends[WAVES * WAVE - 1]), share = max(streams.least, (total + (int)gridDim.x - 1) / (int)gridDim.x);
  const int first = min(blockIdx.x * (long)share, (long)total), last = min(first + share, total);
  if (threadIdx.x == 0) streams.cuts[blockIdx.x].parts = 0;
  for (int at = first; at < last;) {
    int low = 0, high = WAVES * WAVE - 1;     // the run of requests that the unit lies in
    while (low < high) {
      const int middle = (low + high) / 2;
      if (ends[middle] > at) high = middle;
      else low = middle + 1;
    }
    int index = __builtin_amdgcn_readfirstlane(low) * run, inside = __builtin_amdgcn_readfirstlane(at - (low > 0 ? ends[low - 1] : 0)), all = 0;
    Request request = {0, 0, 0};
    for (; index < w.requests; ++index) {
      request = run == 1 ? held[index] : load_request(w, index);
      request.start = __builtin_amdgcn_readfirstlane(request.start);
      request.count = __builtin_amdgcn_readfirstlane(request.count);
      request.context = __builtin_amdgcn_readfirstlane(request.context);
      all = units_of(w, request);
      if (inside < all) break;
      inside -= all;
    }
    if (index >= w.requests) break;
    const int each = all / ((request.count * group + 15) / 16 * w.kv_heads);
    const int walk = inside / each, unit = inside - walk * each, units = min(each - unit, last - at);
    Item item;
    // (a request of few columns has several tiles only if it is a single token: all of them walk the same keys)
    if (make_item(w, index, request, walk / w.kv_heads * 16, 16, item)) {
      const int begin = item.from + unit * UNIT, end = min(item.to, begin + units * UNIT), place = at == first ? 0 : 1;
      __syncthreads();                        // (the ring's place has been read)
      take_walk(item, walk % w.kv_heads, begin, end, units == each ? nullptr : streams.parts + ((size_t)blockIdx.x * 2 + place) * PART);
      if (unit == 0 && units < each && threadIdx.x == 0)
        streams.cuts[blockIdx.x] = {item.first_row, item.group, item.first, item.columns, walk % w.kv_heads, (at + each - 1) / share - (int)blockIdx.x + 1, place, 0};
    }
    at += units;
  }
}

// A wave a column of a walk that was cut: its parts joined.  All of them are asked for at once.
constexpr int JOIN_LANES = D / 4, JOINED = WAVE / JOIN_LANES, TOGETHER = 4;  // lanes a part, parts side by side, loads under way

template <typename T>
__global__ void __launch_bounds__(4 * WAVE) packed_join_kernel(T* out, int out_stride, Streams streams, int part_columns) {
  const int workgroup = blockIdx.x, lane = threadIdx.x % WAVE, which = min(lane / JOIN_LANES, JOINED - 1), d = lane % JOIN_LANES * 4;
  const Cut cut = streams.cuts[workgroup];
  if (cut.parts == 0) return;
  const int parts = min(cut.parts, (int)gridDim.x - workgroup);
  const size_t part_size = (size_t)part_columns * (D + 4);
  for (int column = blockIdx.y * 4 + threadIdx.x / WAVE; column < cut.columns; column += gridDim.y * 4) {
    const float* mine = streams.parts + (size_t)workgroup * 2 * part_size + column * (D + 4);
    const auto part_of = [&](int i) { return mine + (size_t)i * 2 * part_size + (i == 0 ? cut.place * part_size : 0); };
    f32x4 result = (f32x4){0.f, 0.f, 0.f, 0.f};
    float weights = 0.f, largest = -INFINITY;
    for (int base = 0; base < parts; base += WAVE) {
      float reference = -INFINITY, total = 0.f;
      if (base + lane < parts) {
        const float* part = part_of(base + lane);
        reference = part[D];
        total = part[D + 1];
      }
      const float larger = fmaxf(largest, wave_max(reference)), change = largest == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(largest - larger);
      const float share = reference == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(reference - larger);
      largest = larger;
      result *= change;
      weights = weights * change + wave_sum(share * total);
      const int end = min(base + WAVE, parts);
      for (int i = base; i < end; i += TOGETHER * JOINED) {
        f32x4 part[TOGETHER];
        float weight[TOGETHER];
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k) {
          const int at = i + k * JOINED + which;
          part[k] = *(const f32x4*)(part_of(min(at, end - 1)) + d);
          weight[k] = __shfl(share, min(at, end - 1) - base);
        }
        // (every part counts, those of a share of 0 too: a value that is no number makes its columns no number wherever their walk was cut)
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k)
          if (i + k * JOINED + which < end) result += weight[k] * part[k];
      }
    }
#pragma unroll
    for (int other = 1; other < JOINED; ++other)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float far = __shfl(result[i], min(lane + other * JOIN_LANES, WAVE - 1));
        if (lane < JOIN_LANES) result[i] += far;
      }
    if (lane >= JOIN_LANES) continue;
    const int flat = cut.first + column, token = flat / cut.group, head = cut.kv_head * cut.group + flat - token * cut.group;
    write_four(out + (size_t)(cut.first_row + token) * out_stride + head * D + d, result * (1.f / weights));
  }
}

// ---------------------------------------------------------------------------------------------------------------- portions
//
// Many columns see the same keys: the matrix cores and the instructions that make codes bfloat16 bound these.  In bfloat16, at heads of a multiple of 64, a wave
// takes 32 columns with v_mfma_f32_32x32x16_bf16, which does 1.8 PFLOP/s here where 16x16x32 does 1.1; a step's codes are made bfloat16 once for them.  Everything else is as
// above: a lane takes D / 2 neighbouring elements of a key, keys are dealt to rows so that a lane ends with the weights of two pieces of eight neighbouring keys, and of the values it takes
// D / 32 neighbouring elements of those keys.  A prompt of 2,047 tokens at 12/2 heads of 128 takes
// 41 us (0.32 PFLOP/s: two rounds of workgroups, each with its beginning and end, the longest walk 17 us), 31 tokens at 640 keys and a portion of 256 at 28/4 18.  Where columns are many, tiles
// are shared: below.
constexpr int PORTION_WAVES = 4, PORTION_THREADS = PORTION_WAVES * WAVE;
constexpr int PORTION_UNIT = PORTION_WAVES * KEYS;  // keys
constexpr int BEGINNING = 4;                  // units that a walk's beginning and end take as long as

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int HALF_BLOCKS = D >= 64 ? D / 64 : 1;

struct WideStep {
  u32x4 keys[HALF_BLOCKS];                    // a block of 32 elements each
  unsigned key_powers[HALF_BLOCKS];
  u32x4 values[2][CHUNKS][2];                 // of pieces h and 2 + h
  u32x2 value_powers[2][CHUNKS];
};

struct WideColumns {                          // a wave's 32
  Eight query[D / 16];
  int position;                               // of the lane's column's token
  float reference, total;                     // total: of the lane's half of the keys
  bool begun;                                 // some key has been seen; before, the reference is 0
  f32x16 sum[D / 32];
};

__device__ __forceinline__ f32x16 multiply(const Eight& a, const Eight& b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0); }

// N blocks of a key, and their powers
#define BLOCK(i, o, p) "ds_read_b128 %[k" #i "], %[keys] offset:" #o "\n\tds_read_u8 %[b" #i "], %[at] offset:" #p "\n\t"
#define TO_BLOCK(i) [k##i] "=&v"(blocks[i]), [b##i] "=&v"(powers[i])
template <int N> __device__ __forceinline__ void read_blocks(u32x4 (&blocks)[N], unsigned (&powers)[N], unsigned keys, unsigned at) {
  if constexpr (N == 1) asm volatile(BLOCK(0, 0, 0) "s_waitcnt lgkmcnt(0)" : TO_BLOCK(0) : [keys] "v"(keys), [at] "v"(at) : "memory");
  else if constexpr (N == 3)
    asm volatile(BLOCK(0, 0, 0) BLOCK(1, 16, 1) BLOCK(2, 32, 2) "s_waitcnt lgkmcnt(0)" : TO_BLOCK(0), TO_BLOCK(1), TO_BLOCK(2) : [keys] "v"(keys), [at] "v"(at) : "memory");
  else {
    static_assert(N == 4, "heads of 64, 192 and 256");
    asm volatile(BLOCK(0, 0, 0) BLOCK(1, 16, 1) BLOCK(2, 32, 2) BLOCK(3, 48, 3) "s_waitcnt lgkmcnt(0)"
                 : TO_BLOCK(0), TO_BLOCK(1), TO_BLOCK(2), TO_BLOCK(3) : [keys] "v"(keys), [at] "v"(at) : "memory");
  }
}

__device__ __forceinline__ void read_step(WideStep& s, const unsigned char* stage) {
  const unsigned lane = threadIdx.x % WAVE, n = lane & 31, h = lane >> 5, at = (unsigned)(size_t)(const unsigned char __attribute__((address_space(3)))*)stage;
  const unsigned row = (n & 0x13) | ((n & 4) << 1) | ((n & 8) >> 1);  // the key that row n of the first product is
  const unsigned keys = at + (row >> 3) * PIECE + (row & 7) * (D / 2) + h * (D / 4), key_powers = at + 4 * PIECE + (row >> 3) * (D / 2) + (row & 7) * (D / 32) + h * (D / 64);
#if HEAD_DIM == 128
  const unsigned values = at + h * PIECE + 4 * D + (n >> 1) * 32, value_powers = at + 4 * PIECE + h * (D / 2) + D / 4 + (n >> 3) * 8;
  asm volatile(
      "ds_read_b128 %0, %10\n\tds_read_b128 %1, %10 offset:16\n\tds_read_u8 %2, %11\n\tds_read_u8 %3, %11 offset:1\n\tds_read_b128 %4, %12\n\tds_read_b128 %5, %12 offset:16\n\t"
      "ds_read_b64 %8, %13\n\tds_read_b128 %6, %12 offset:%14\n\tds_read_b128 %7, %12 offset:%15\n\tds_read_b64 %9, %13 offset:%16\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(s.keys[0]), "=&v"(s.keys[1]), "=&v"(s.key_powers[0]), "=&v"(s.key_powers[1]), "=&v"(s.values[0][0][0]), "=&v"(s.values[0][0][1]), "=&v"(s.values[1][0][0]),
        "=&v"(s.values[1][0][1]), "=&v"(s.value_powers[0][0]), "=&v"(s.value_powers[1][0])
      : "v"(keys), "v"(key_powers), "v"(values), "v"(value_powers), "n"(2 * PIECE), "n"(2 * PIECE + 16), "n"(D)
      : "memory");
#elif HEAD_DIM % 64 == 0
  read_blocks(s.keys, s.key_powers, keys, key_powers);
  u32x4 low[2 * CHUNKS], high[2 * CHUNKS];
  u32x2 powers[2 * CHUNKS];
  unsigned values[2 * CHUNKS], value_powers[2 * CHUNKS];
#pragma unroll
  for (int i = 0; i < 2 * CHUNKS; ++i) {
    const unsigned c = i % CHUNKS, piece = 2 * (i / CHUNKS) + h, granule = chunk_first(c) / 8 + n * chunk_width(c) / 256;
    values[i] = at + piece * PIECE + 4 * D + granule * 32;
    value_powers[i] = at + 4 * PIECE + piece * (D / 2) + D / 4 + granule / 4 * 8;
  }
  read_values(low, high, powers, values, value_powers);
#pragma unroll
  for (int i = 0; i < 2 * CHUNKS; ++i) {
    s.values[i / CHUNKS][i % CHUNKS][0] = low[i];
    s.values[i / CHUNKS][i % CHUNKS][1] = high[i];
    s.value_powers[i / CHUNKS][i % CHUNKS] = powers[i];
  }
#endif
}

template <bool EDGE> __device__ __forceinline__ void take_step(WideColumns& columns, const WideStep& now, const Walk& w, const Item& item, int base) {
  const int lane = threadIdx.x % WAVE, n = lane & 31, h = lane >> 5;
  // scores: value 8 u + j of a lane is key 16 u + 8 h + j of the step
  f32x16 score;
#pragma unroll
  for (int i = 0; i < 16; ++i) score[i] = 0.f;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    const float power = packed_power(now.key_powers[s / 4]);
    const unsigned codes = now.keys[s / 4][s % 4];
    Eight key;
    key.u = (u32x4){unpack_pair<0>(codes, power), unpack_pair<1>(codes, power), unpack_pair<2>(codes, power), unpack_pair<3>(codes, power)};
    score = multiply(key, columns.query[s], score);
  }
  const int highest = columns.position - base - 8 * h, lowest = w.window > 0 ? highest - w.window + 1 : -(1 << 30);
  const auto sees = [&](int i) { return 16 * (i / 8) + i % 8 <= highest && 16 * (i / 8) + i % 8 >= lowest; };
  float x[16];                                // log2 of the weights
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float y = __builtin_fmaf(score[i], w.scale, -columns.reference);
    x[i] = !EDGE || sees(i) ? y : -INFINITY;
  }
  float largest = fmaxf(largest_of(x), largest_of(x + 8));
  if (__any(largest > (columns.begun ? AHEAD : -INFINITY))) {
    largest = fmaxf(largest, __shfl_xor(largest, 32));
    // (a column's first reference is its first largest score, wherever that lies; later ones only rise)
    const float rise = largest > (columns.begun ? 0.f : -INFINITY) ? largest : 0.f, change = columns.begun ? __builtin_amdgcn_exp2f(-rise) : 1.f;
    columns.begun = columns.begun || largest > -INFINITY;
    columns.reference += rise;
    columns.total *= change;
#pragma unroll
    for (int t = 0; t < D / 32; ++t) columns.sum[t] *= change;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] -= rise;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    Eight weight;
#pragma unroll
    for (int j = 0; j < 8; ++j) weight.v[j] = (bf16_t)__builtin_amdgcn_exp2f(x[8 * u + j]);  // (rounded here, once, as the matrix instructions take them)
    // the weights that are multiplied are the weights that are added up
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      union { unsigned u; packed_bf16x2 v; } pair, ones;
      pair.u = weight.u[j];
      ones.u = 0x3f803f80u;
      columns.total = __builtin_amdgcn_fdot2_f32_bf16(pair.v, ones.v, columns.total, false);
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int width = chunk_width(c), first = chunk_first(c) / 32;
      u32x2 powers = now.value_powers[u][c];
      bool poisoned = false;
      Eight marks;
      if (EDGE) {  // (as above: what no column sees is a small number; what is no number is taken out, and put back where it is seen)
        marks.u = (u32x4){0u, 0u, 0u, 0u};
        bool mine = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = base + 16 * u + 8 * h + j;
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
      Eight value[4];                         // the lane's elements (two at a width of 64), of eight keys
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float power0 = __uint_as_float(powers[j / 4] << (23 - j % 4 * 8)), power1 = __uint_as_float(j % 4 == 2 ? powers[j / 4] >> 1 : powers[j / 4] << 15);
        const unsigned a = now.values[u][c][j / 4][j % 4], b = now.values[u][c][j / 4][j % 4 + 1];
        if (width == 128) {                   // two of a granule's four bytes, of two keys
          const unsigned both = __builtin_amdgcn_perm(b, a, n & 1 ? 0x07060302u : 0x05040100u);
          const unsigned a0 = unpack_pair<0>(both, power0), a1 = unpack_pair<1>(both, power0), b0 = unpack_pair<2>(both, power1), b1 = unpack_pair<3>(both, power1);
          value[0].u[j / 2] = __builtin_amdgcn_perm(b0, a0, 0x05040100u);
          value[1].u[j / 2] = __builtin_amdgcn_perm(b0, a0, 0x07060302u);
          value[2].u[j / 2] = __builtin_amdgcn_perm(b1, a1, 0x05040100u);
          value[3].u[j / 2] = __builtin_amdgcn_perm(b1, a1, 0x07060302u);
        } else {                              // one of them
          const unsigned both = __builtin_amdgcn_perm(b, a, (unsigned)((n & 3) | (4 + (n & 3)) << 8));
          const unsigned a0 = unpack_pair<0>(both, power0), b0 = unpack_pair<1>(both, power1);
          value[0].u[j / 2] = __builtin_amdgcn_perm(b0, a0, 0x05040100u);
          value[1].u[j / 2] = __builtin_amdgcn_perm(b0, a0, 0x07060302u);
        }
      }
#pragma unroll
      for (int e = 0; e < width / 32; ++e) columns.sum[first + e] = multiply(value[e], weight, columns.sum[first + e]);
      if (EDGE && poisoned) {
        Eight seen;
#pragma unroll
        for (int j = 0; j < 8; ++j) seen.v[j] = (bf16_t)(sees(8 * u + j) ? 1.f : 0.f);
        f32x16 none;
#pragma unroll
        for (int i = 0; i < 16; ++i) none[i] = 0.f;
        const f32x16 hit = multiply(marks, seen, none);
#pragma unroll
        for (int e = 0; e < width / 32; ++e)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (hit[i] > 0.f) columns.sum[first + e][i] = __uint_as_float(0x7fc00000u);
      }
    }
  }
}

__device__ __forceinline__ void load_queries(WideColumns& columns, const bf16_t* q, int q_stride, const Item& item, int kv_head, bool whole) {
  const int lane = threadIdx.x % WAVE, n = lane & 31, h = lane >> 5, flat = item.first + min(n, item.columns - 1), token = flat / item.group;
  columns.position = item.first_position - item.first / item.group + token;
  const bf16_t* row = q + (size_t)(item.first_row + token) * q_stride + (kv_head * item.group + flat - token * item.group) * D + h * (D / 2);
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    if (whole) {
      columns.query[s].u = *(const u32x4*)(row + s * 8);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) columns.query[s].v[e] = row[s * 8 + e];
    }
  }
  columns.reference = columns.total = 0.f;
  columns.begun = false;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) columns.sum[t][i] = 0.f;
}

__device__ __forceinline__ void settle(WideColumns& columns) {
#pragma unroll
  for (int s = 0; s < D / 16; ++s) asm volatile("" : "+v"(columns.query[s].u));
}

// (memory as above: 16 columns at a time)
template <int W, typename Take>
__device__ __forceinline__ void bring_together(const WideColumns& columns, int count, int wave, unsigned char* memory, Take take) {
  float (*results)[16][D + 4] = (float (*)[16][D + 4])memory;
  float (*sums)[16][2] = (float (*)[16][2])(memory + W * 16 * (D + 4) * 4);
  const int lane = threadIdx.x % WAVE, n = lane & 31, h = lane >> 5, r = n & 15;
  const float total = columns.total + __shfl_xor(columns.total, 32);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (half * 16 >= count) break;
    __syncthreads();
    if (n / 16 == half) {
      if (h == 0) {
        sums[wave][r][0] = columns.begun ? columns.reference : -INFINITY;
        sums[wave][r][1] = total;
      }
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const int each = chunk_width(c) / 32, first = chunk_first(c) / 32;  // neighbouring elements of a row of the tiles
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e < each) results[wave][r][chunk_first(c) + (8 * (i / 4) + 4 * h + i % 4) * each + e] = columns.sum[first + e][i];
      }
    }
    __syncthreads();
    join_waves<W>(results, sums, min(16, count - half * 16), [&](int column, int d, f32x4 result, float largest, float weights) { take(half * 16 + column, d, result, largest, weights); });
  }
}

// Which columns a wave takes: 32 at heads of a multiple of 64 in bfloat16, 16 elsewhere.
template <typename T> constexpr bool WIDE = sizeof(T) == 2 && D % 64 == 0;
template <typename T> constexpr int PORTION_COLUMNS = WIDE<T> ? 32 : 16;
template <typename T> constexpr int PORTION_PART = PORTION_COLUMNS<T> * (D + 4);
template <typename T, bool> struct PortionOf {
  typedef Columns<T> Cols;
  typedef Step Taken;
};
template <typename T> struct PortionOf<T, true> {
  typedef WideColumns Cols;
  typedef WideStep Taken;
};

// The walks of a kernel of portions: whole ones, the workgroup's own, or runs of all walks' units, which lie behind each other (up to 256 requests, one a thread).  A unit is UNIT keys from a multiple
// of ALIGN on, a walk's beginning and end take as long as BEGINS units.  take(item, kv head, the keys from, to, where to leave a part or null).
struct Shares {
  int item_ends[PORTION_THREADS], ends[PORTION_THREADS], wave_sums[2][PORTION_WAVES];
  Request held[PORTION_THREADS];
};

template <int COLUMNS, int UNIT, int ALIGN, int BEGINS, typename Take>
__device__ __forceinline__ void take_walks(const Walk& w, const Streams& streams, int items, Shares& shares, Take take) {
  const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), group = w.heads / w.kv_heads;
  const auto units_of = [&](const Item& item) { return BEGINS + (item.to - item.from / ALIGN * ALIGN + UNIT - 1) / UNIT; };
  // where the requests' items end, then where the items' units end (a run of items a thread)
  const auto added_up = [&](int mine, int* sums) {
#pragma unroll
    for (int step = 1; step < WAVE; step <<= 1) {
      const int other = __shfl_up(mine, step);
      if (lane >= step) mine += other;
    }
    if (lane == WAVE - 1) sums[wave] = mine;
    __syncthreads();
    for (int v = 0; v < wave; ++v) mine += sums[v];
    return mine;
  };
  int all_items = 0, run = 0, share = 1, first = 0, last = 1, total = 0;
  const auto item_at = [&](int index, Item& item) {
    int low = 0, high = PORTION_THREADS - 1;
    while (low < high) {
      const int middle = (low + high) / 2;
      if (shares.item_ends[middle] > index) high = middle;
      else low = middle + 1;
    }
    return make_item(w, low, shares.held[low], (index - (low > 0 ? shares.item_ends[low - 1] : 0)) * COLUMNS, COLUMNS, item);
  };
  // the walk that a unit lies in, and where in it: kv head, unit of it, units
  const auto walk_at = [&](int at, Item& item, int& kv_head, int& unit, int& each) {
    int low = 0, high = PORTION_THREADS - 1;
    while (low < high) {
      const int middle = (low + high) / 2;
      if (shares.ends[middle] > at) high = middle;
      else low = middle + 1;
    }
    int index = __builtin_amdgcn_readfirstlane(low) * run, inside = __builtin_amdgcn_readfirstlane(at - (low > 0 ? shares.ends[low - 1] : 0));
    for (; index < all_items; ++index) {
      each = __builtin_amdgcn_readfirstlane(item_at(index, item) ? units_of(item) : 0);
      if (inside < each * w.kv_heads) break;
      inside -= each * w.kv_heads;
    }
    if (index >= all_items) return false;
    kv_head = inside / each;
    unit = inside - kv_head * each;
    return true;
  };
  if (streams.least > 0) {
    int count = 0;
    if ((int)threadIdx.x < w.requests) {
      shares.held[threadIdx.x] = load_request(w, threadIdx.x);
      const int tokens = shares.held[threadIdx.x].count;
      count = few_columns(w, tokens, group) ? 0 : (max(tokens, 0) * group + COLUMNS - 1) / COLUMNS;
    }
    shares.item_ends[threadIdx.x] = added_up(count, shares.wave_sums[0]);
    __syncthreads();
    all_items = __builtin_amdgcn_readfirstlane(shares.item_ends[PORTION_THREADS - 1]);
    run = (all_items + PORTION_THREADS - 1) / PORTION_THREADS;
    int units = 0;
    for (int i = threadIdx.x * run; i < min((int)(threadIdx.x + 1) * run, all_items); ++i) {
      Item item;
      if (item_at(i, item)) units += units_of(item) * w.kv_heads;
    }
    shares.ends[threadIdx.x] = added_up(units, shares.wave_sums[1]);
    __syncthreads();
    total = __builtin_amdgcn_readfirstlane(shares.ends[PORTION_THREADS - 1]);
    share = max(max(streams.least, BEGINS + 1), (total + (int)gridDim.x - 1) / (int)gridDim.x);
    first = min(blockIdx.x * (long)share, (long)total);
    last = min(first + share, total);
    if (threadIdx.x == 0) streams.cuts[blockIdx.x].parts = 0;
    // a walk is not cut within its beginning: a cut there is one before it (the next workgroup's `first` the same way)
    if (first < last) {
      Item item;
      int kv_head, unit, each;
      if (walk_at(first, item, kv_head, unit, each) && unit <= BEGINS) first -= unit;
      if (last < total && walk_at(last, item, kv_head, unit, each) && unit <= BEGINS) last -= unit;
    }
  }
  for (int at = first; at < last;) {
    Item item;
    int kv_head, begin, taken = 1, each = 1, unit = 0, place = 0;
    if (streams.least == 0) {                 // a walk whole; the longest begin first: a request's last columns walk most keys
      if (!find_item(w, items - 1 - blockIdx.x / w.kv_heads, COLUMNS, item)) return;
      kv_head = blockIdx.x % w.kv_heads;
      begin = item.from / ALIGN * ALIGN;
    } else {
      if (!walk_at(at, item, kv_head, unit, each)) break;
      taken = min(each - unit, last - at);
      place = at == first ? 0 : 1;
      begin = item.from / ALIGN * ALIGN + max(unit - BEGINS, 0) * UNIT;
    }
    item.request = __builtin_amdgcn_readfirstlane(item.request);
    item.first_row = __builtin_amdgcn_readfirstlane(item.first_row);
    item.first = __builtin_amdgcn_readfirstlane(item.first);
    item.columns = __builtin_amdgcn_readfirstlane(item.columns);
    item.first_position = __builtin_amdgcn_readfirstlane(item.first_position);
    item.last_position = __builtin_amdgcn_readfirstlane(item.last_position);
    item.from = __builtin_amdgcn_readfirstlane(item.from);
    item.to = __builtin_amdgcn_readfirstlane(item.to);
    const bool cut = taken < each;
    take(item, kv_head, __builtin_amdgcn_readfirstlane(begin), streams.least == 0 || unit + taken == each ? item.to : item.from / ALIGN * ALIGN + (unit + taken - BEGINS) * UNIT,
         cut ? streams.parts + ((size_t)blockIdx.x * 2 + place) * (COLUMNS * (D + 4)) : nullptr);
    if (cut && unit == 0 && threadIdx.x == 0)
      streams.cuts[blockIdx.x] = {item.first_row, group, item.first, item.columns, kv_head, (at + each - 1) / share - (int)blockIdx.x + 1, place, 0};
    at += taken;
  }
}

template <typename T>
__global__ void __launch_bounds__(PORTION_THREADS, D <= 128 ? 2 : 1) packed_portions_kernel(const T* q, int q_stride, T* out, int out_stride, const unsigned char* pages, Walk w, Streams streams, int items, int whole) {
  constexpr int COLUMNS = PORTION_COLUMNS<T>;
  __shared__ __attribute__((aligned(16))) unsigned char memory[memory_of<PORTION_WAVES>()];
  __shared__ Shares shares;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  take_walks<COLUMNS, PORTION_UNIT, KEYS, BEGINNING>(w, streams, items, shares, [&](const Item& item, int kv_head, int begin, int end, float* part) {
    typename PortionOf<T, WIDE<T>>::Cols columns;
    __syncthreads();                          // (what a walk before this one left in LDS has been read)
    walk_keys<T, typename PortionOf<T, WIDE<T>>::Taken, PORTION_WAVES>(columns, q, q_stride, pages, w, item, kv_head, whole, begin, end, wave, memory + wave * (STAGES * STAGE));
    bring_together<PORTION_WAVES>(columns, item.columns, wave, memory, [&](int column, int d, f32x4 result, float largest, float weights) {
      if (part) {
        *(f32x4*)(part + column * (D + 4) + d) = result;
        if (d == 0) *(f32x4*)(part + column * (D + 4) + D) = (f32x4){largest, weights, 0.f, 0.f};
      } else {
        const int flat = item.first + column, token = flat / item.group, head = kv_head * item.group + flat - token * item.group;
        write_four(out + (size_t)(item.first_row + token) * out_stride + head * D + d, result * (1.f / weights));
      }
    });
  });
}

// ---------------------------------------------------------------------------------------------------------------- bfloat16 portions
//
// The same for portions that have columns enough to fill the chip with 128 a workgroup, 32 a wave: the instructions that make a key bfloat16, which every wave above does for 32 columns, are shared.
// Tiles of 64 keys and values are made bfloat16 in LDS once for the four waves, the next tile's while they multiply with this one's:
//   S^T = K Q^T, O^T += V^T P^T with v_mfma_f32_32x32x16_bf16.
// The keys of 32 are dealt to the rows of the first product so that a lane ends with the weights of two pieces of eight neighbouring keys, the slices that the
// second product takes.  In LDS keys lie in pieces of eight elements, a piece of all 64 keys side by side, values in pieces of eight keys, a piece of all elements side by
// side (eight neighbours exchanged by the number of their 16, so that the writers of one element write to different banks): all reads are whole lines.
// us, as above and so: 2,048 tokens behind 30,000 keys at 12/2 heads 562 and 458, a prompt of 8,192 at 40/8 heads 1,007 and 780, of 2,048 101 and 71, but at 12/2 heads 41 and 59.  The first is 0.80 to 0.85 PFLOP/s (458 to 487 us in different runs): the products alone
// would take 215 us, the weights' exponentials and what else is done a weight fill most of the rest, on the same issue port.
constexpr int TILE = 64, SHARED_COLUMNS = 128;  // keys, columns
constexpr int UNITS_ROUNDS = (2 * D + PORTION_THREADS - 1) / PORTION_THREADS;  // 16-byte units of codes a thread takes of a tile's keys, and of its values
constexpr int SHARED_BEGINNING = 3;           // tiles that a walk's beginning and end take as long as

struct Codes {                                // of a thread, of a tile
  u32x4 keys[UNITS_ROUNDS], values[UNITS_ROUNDS];
  unsigned key_power[UNITS_ROUNDS], value_powers[UNITS_ROUNDS];
};
struct Entries {                              // table entries of a thread's units
  int key[UNITS_ROUNDS], value[UNITS_ROUNDS];
};

struct SharedTiles {
  const unsigned char* from;                  // of the kv head
  const int* table;
  unsigned page_stride;
  PackedPage page;
};

__device__ __forceinline__ unsigned page_of(const Walk& w, unsigned piece) { return w.page_shift >= 0 ? piece >> w.page_shift : __umulhi(piece, w.page_reciprocal); }

// unit u of a tile's keys: key u % 64, block u / 64; of its values: half u % 2 of the eight keys of piece u / (D / 4), granule (u / 2) % (D / 8)
__device__ __forceinline__ void load_entries(Entries& e, const Walk& w, const SharedTiles& tiles, int base) {
#pragma unroll
  for (int i = 0; i < UNITS_ROUNDS; ++i) {
    const unsigned unit = i * PORTION_THREADS + threadIdx.x, key_at = page_of(w, (base + unit % TILE) / 8), value_at = page_of(w, base / 8 + unit / (D / 4));
    e.key[i] = key_at < (unsigned)w.table_width ? tiles.table[key_at] : 0;
    e.value[i] = value_at < (unsigned)w.table_width ? tiles.table[value_at] : 0;
  }
}
__device__ __forceinline__ void load_codes(Codes& c, const Entries& e, const Walk& w, const SharedTiles& tiles, int base) {
  const unsigned per_page = (unsigned)w.page_size / 8;
#pragma unroll
  for (int i = 0; i < UNITS_ROUNDS; ++i) {
    const unsigned unit = i * PORTION_THREADS + threadIdx.x;
    if (2 * D % PORTION_THREADS && unit >= 2 * D) continue;
    {
      const unsigned key = base + unit % TILE, block = unit / TILE, offset = key - page_of(w, key / 8) * per_page * 8;
      const unsigned char* mine = tiles.from + (size_t)((unsigned)e.key[i] < (unsigned)w.num_pages ? (unsigned)e.key[i] : 0u) * tiles.page_stride;
      c.keys[i] = *(const u32x4*)(mine + tiles.page.key_codes(offset, block * 4));
      c.key_power[i] = mine[tiles.page.key_power(offset, block)];
    }
    const unsigned piece = base / 8 + unit / (D / 4), half = unit % 2, granule = unit / 2 % (D / 8), offset = (piece - page_of(w, piece) * per_page) * 8;
    const unsigned char* mine = tiles.from + (size_t)((unsigned)e.value[i] < (unsigned)w.num_pages ? (unsigned)e.value[i] : 0u) * tiles.page_stride;
    c.values[i] = *(const u32x4*)(mine + tiles.page.value_codes(offset + half * 4, granule));
    c.value_powers[i] = *(const unsigned*)(mine + tiles.page.value_power(offset + half * 4, granule / 4));
  }
}

// Values that are no number count as zero, and as what they are where they are seen: `bad` gets, per block of 32 elements, the keys of the tile that have such.
// Keys beyond `last`, which nobody sees, are made small numbers, whatever lies there.
__device__ __forceinline__ void settle_powers(Codes& c, unsigned long long* bad, int base, int last) {
#pragma unroll
  for (int i = 0; i < UNITS_ROUNDS; ++i) {
    const unsigned unit = i * PORTION_THREADS + threadIdx.x;
    if (2 * D % PORTION_THREADS && unit >= 2 * D) continue;
    const unsigned powers = c.value_powers[i], all = powers & (powers >> 4), granule = unit / 2 % (D / 8);
    const int first = unit / (D / 4) * 8 + unit % 2 * 4;  // key of the tile
    if (base + first + 3 > last || ((all & (all >> 2)) & 0x03030303u) != 0u) {  // (bytes of 255, and some others)
      unsigned settled = powers;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool unseen = base + first + j > last, none = ((powers >> (8 * j)) & 255u) == PACKED_NO_NUMBER;
        if (none && !unseen) atomicOr(&bad[granule / 4], 1ull << (first + j));
        if (none || unseen) settled &= ~(255u << (8 * j));
      }
      c.value_powers[i] = settled;
    }
  }
}

// A thread's codes as bfloat16 into LDS, in eight parts: keys [D / 8][64][8] in the first four, values [8][D][8] in the others.
constexpr int UNPACKS = 8;
template <int PART_> __device__ __forceinline__ void unpack_part(const Codes& c, unsigned char* tile) {
#pragma unroll
  for (int i = 0; i < UNITS_ROUNDS; ++i) {
    const unsigned unit = i * PORTION_THREADS + threadIdx.x;
    if (2 * D % PORTION_THREADS && unit >= 2 * D) continue;
    if constexpr (PART_ < 4) {
      const unsigned key = unit % TILE, block = unit / TILE, codes = c.keys[i][PART_];
      const float power = packed_power(c.key_power[i]);
      *(u32x4*)(tile + ((block * 4 + PART_) * TILE + key) * 16) = (u32x4){unpack_pair<0>(codes, power), unpack_pair<1>(codes, power), unpack_pair<2>(codes, power), unpack_pair<3>(codes, power)};
    } else {
      constexpr int E = PART_ - 4;              // elements 2 E and 2 E + 1 of the eight
      const unsigned piece = unit / (D / 4), half = unit % 2, granule = unit / 2 % (D / 8), exchange = (granule >> 1) & 7, powers = c.value_powers[i];
      unsigned raw[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) raw[j] = unpack_pair<E>(c.values[i][j], __uint_as_float(j == 3 ? powers >> 1 : powers << (23 - j * 8)));
      unsigned char* to = tile + TILE * D * 2 + (piece * D + granule * 8) * 16 + half * 8;
      *(u32x2*)(to + ((2 * E) ^ exchange) * 16) = (u32x2){__builtin_amdgcn_perm(raw[1], raw[0], 0x05040100u), __builtin_amdgcn_perm(raw[3], raw[2], 0x05040100u)};
      *(u32x2*)(to + ((2 * E + 1) ^ exchange) * 16) = (u32x2){__builtin_amdgcn_perm(raw[1], raw[0], 0x07060302u), __builtin_amdgcn_perm(raw[3], raw[2], 0x07060302u)};
    }
  }
}
template <int FIRST, int LAST> __device__ __forceinline__ void unpack_parts(const Codes& c, unsigned char* tile) {
  if constexpr (FIRST < LAST) {
    unpack_part<FIRST>(c, tile);
    unpack_parts<FIRST + 1, LAST>(c, tile);
  }
}

struct SharedColumns {                          // a wave's 32
  Eight query[D / 16];
  int position;                               // of the lane's column's token
  int first_position, last_position;          // of the wave's
  float reference, total;                     // total: of the lane's half of the keys
  bool begun;                                 // some key has been seen; before, the reference is 0
  f32x16 sum[D / 32];
};

// A tile of 64 keys from `base` on, with the next tile's codes made bfloat16 on the way (`next`: where to).  In a wave instructions begin in order, and one of these products keeps the
// matrix core busy for eight others: so each is followed by what does not wait for it, a part of the next tile behind those of the scores, weights of later keys
// behind those of the values.  edge: some column does not see some of the keys.
constexpr int KEYS_AHEAD = 3;                 // slices of the keys that have been asked for
template <int S> __device__ __forceinline__ void score_parts(f32x16 (&score)[2], Eight (&key)[KEYS_AHEAD][2], const SharedColumns& columns, const unsigned char* mine, const Codes& codes, unsigned char* next) {
  if constexpr (S < D / 16) {
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      score[sub] = multiply(key[S % KEYS_AHEAD][sub], columns.query[S], score[sub]);
      if constexpr (S + KEYS_AHEAD < D / 16) key[S % KEYS_AHEAD][sub].u = *(const u32x4*)(mine + (2 * (S + KEYS_AHEAD) * TILE + sub * 32) * 16);
    }
    unpack_parts<S * UNPACKS / (D / 16), (S + 1) * UNPACKS / (D / 16)>(codes, next);
    __builtin_amdgcn_sched_barrier(0);
    score_parts<S + 1>(score, key, columns, mine, codes, next);
  }
}

__device__ __forceinline__ void take_tile(SharedColumns& columns, const unsigned char* tile, const Walk& w, int base, bool edge, const Codes& codes, unsigned char* next) {
  const int lane = threadIdx.x % WAVE, n = lane & 31, h = lane >> 5;
  const int row = (n & 0x13) | ((n & 4) << 1) | ((n & 8) >> 1);  // the key that row n of the product is
  f32x16 score[2];
#pragma unroll
  for (int i = 0; i < 16; ++i) score[0][i] = score[1][i] = 0.f;
  const unsigned char* mine = tile + (h * TILE + row) * 16;
  Eight key[KEYS_AHEAD][2];
#pragma unroll
  for (int s = 0; s < KEYS_AHEAD; ++s)
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
      if (s < D / 16) key[s][sub].u = *(const u32x4*)(mine + (2 * s * TILE + sub * 32) * 16);
  score_parts<0>(score, key, columns, mine, codes, next);
  const unsigned char* values = tile + TILE * D * 2 + (h * D + n / 8 * 8) * 16;
  const auto value_of = [&](int f, int t) { return *(const u32x4*)(values + (2 * f * D + t * 32) * 16 + ((n & 7) ^ ((t * 2 + (n >> 4)) & 7)) * 16); };
  Eight value[D / 32];
#pragma unroll
  for (int t = 0; t < D / 32; ++t) value[t].u = value_of(0, t);
  if (edge) {
    const int highest = columns.position - base - 8 * h, lowest = w.window > 0 ? highest - w.window + 1 : -(1 << 30);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int key = 16 * (i / 8) + i % 8;
      if (key > highest || key < lowest) score[i / 16][i % 16] = -INFINITY;
    }
  }
  float x[32];                                // log2 of the weights
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] = __builtin_fmaf(score[i / 16][i % 16], w.scale, -columns.reference);
  float largest = fmaxf(fmaxf(largest_of(x), largest_of(x + 8)), fmaxf(largest_of(x + 16), largest_of(x + 24)));
  if (__any(largest > (columns.begun ? AHEAD : -INFINITY))) {
    largest = fmaxf(largest, __shfl_xor(largest, 32));
    // (a column's first reference is its first tile's largest score, wherever that lies; later ones only rise)
    const float rise = largest > (columns.begun ? 0.f : -INFINITY) ? largest : 0.f, change = columns.begun ? __builtin_amdgcn_exp2f(-rise) : 1.f;
    columns.begun = columns.begun || largest > -INFINITY;
    columns.reference += rise;
    columns.total *= change;
#pragma unroll
    for (int t = 0; t < D / 32; ++t) columns.sum[t] *= change;
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] -= rise;
  }
  Eight weight;                               // (rounded here and below, once, as the matrix instructions take them)
#pragma unroll
  for (int j = 0; j < 8; ++j) weight.v[j] = (bf16_t)__builtin_amdgcn_exp2f(x[j]);
#pragma unroll
  for (int f = 0; f < 4; ++f) {
    Eight later;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < D / 32; ++t) {
      columns.sum[t] = multiply(value[t], weight, columns.sum[t]);
      if (f < 3) value[t].u = value_of(f + 1, t);
    }
    // the weights that are multiplied are the weights that are added up
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      union { unsigned u; packed_bf16x2 v; } pair, ones;
      pair.u = weight.u[j];
      ones.u = 0x3f803f80u;
      columns.total = __builtin_amdgcn_fdot2_f32_bf16(pair.v, ones.v, columns.total, false);
    }
    if (f < 3) {
#pragma unroll
      for (int j = 0; j < 8; ++j) later.v[j] = (bf16_t)__builtin_amdgcn_exp2f(x[8 * (f + 1) + j]);
      weight = later;
    }
#pragma unroll
    for (int t = 0; t < D / 32; ++t) {          // a product, then the next value and a share of the rest
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, (16 + D / 32 - 1) / (D / 32), 0);
    }
  }
}

__global__ void __launch_bounds__(PORTION_THREADS, D <= 128 ? 2 : 1)
packed_shared_kernel(const bf16_t* q, int q_stride, bf16_t* out, int out_stride, const unsigned char* pages, Walk w, Streams streams, int items, int whole, int whole_out) {
  constexpr int TILE_BYTES = TILE * D * 2;
  __shared__ __attribute__((aligned(16))) unsigned char memory[2][2 * TILE_BYTES];  // a tile's keys, then its values
  __shared__ unsigned long long bad[3][D / 32];
  __shared__ Shares shares;
  const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), n = lane & 31, h = lane >> 5, group = w.heads / w.kv_heads;

  take_walks<SHARED_COLUMNS, TILE, TILE, SHARED_BEGINNING>(w, streams, items, shares, [&](const Item& item, int kv_head, int begin, int end, float* part) {
    SharedTiles tiles;
    tiles.page = {D, w.page_size};
    tiles.from = pages + (size_t)kv_head * tiles.page.bytes();
    tiles.table = w.tables + (size_t)item.request * w.table_width;
    tiles.page_stride = (unsigned)w.kv_heads * tiles.page.bytes();
    Entries entries[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) load_entries(entries[i], w, tiles, begin + i * TILE);
    Codes now, next;
    load_codes(now, entries[0], w, tiles, begin);
    load_codes(next, entries[1], w, tiles, begin + TILE);
    SharedColumns columns;
    const int first_column = wave * 32, column = min(first_column + n, item.columns - 1), flat = item.first + column, token = flat / group;
    const int token_zero = item.first_position - item.first / group;  // the position that the request's first token of the step is at
    columns.position = token_zero + token;
    columns.first_position = token_zero + (item.first + min(first_column, item.columns - 1)) / group;
    columns.last_position = token_zero + (item.first + min(first_column + 31, item.columns - 1)) / group;
    const bf16_t* row = q + (size_t)(item.first_row + token) * q_stride + (kv_head * group + flat - token * group) * D + h * 8;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      if (whole) {
        columns.query[s].u = *(const u32x4*)(row + s * 16);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) columns.query[s].v[e] = row[s * 16 + e];
      }
    }
    columns.reference = columns.total = 0.f;
    columns.begun = false;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) columns.sum[t][i] = 0.f;
    __syncthreads();                          // (a walk before this one has been read, and what it marked)
    if (threadIdx.x < 3 * (D / 32)) (&bad[0][0])[threadIdx.x] = 0ull;
    __syncthreads();
    settle_powers(now, bad[0], begin, item.last_position);
    unpack_parts<0, UNPACKS>(now, memory[0]);
    int turn = 0, third = 0;                  // of the tile that is multiplied: its place in LDS, that of its marks
    for (int base = begin; base < end; base += TILE) {
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // (codes under way go on)
      now = next;
      entries[1] = entries[2];
      load_codes(next, entries[1], w, tiles, base + 2 * TILE);
      load_entries(entries[2], w, tiles, base + 3 * TILE);
      if (threadIdx.x < D / 32) bad[third == 0 ? 2 : third - 1][threadIdx.x] = 0ull;  // (those of the tile before, which are those of the next but one)
      const int following = third == 2 ? 0 : third + 1;
      settle_powers(now, bad[following], base + TILE, item.last_position);
      // (a tile behind the last one is made too, of whatever lies there: nobody looks at it)
      take_tile(columns, memory[turn], w, base, base + TILE - 1 > columns.first_position || (w.window > 0 && base < columns.last_position - w.window + 1), now, memory[turn ^ 1]);
      products_done();
      unsigned long long any = 0ull;
#pragma unroll
      for (int t = 0; t < D / 32; ++t) any |= bad[third][t];
      if (any) {                              // hardly ever: values that are no number, for the columns that see them
        const int lowest = w.window > 0 ? max(columns.position - w.window + 1 - base, 0) : 0, highest = min(columns.position - base, TILE - 1);
        const unsigned long long seen = highest < lowest ? 0ull : ((2ull << highest) - 1ull) & ~((1ull << lowest) - 1ull);
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
          if (bad[third][t] & seen) columns.sum[t] += __uint_as_float(0x7fc00000u);
      }
      turn ^= 1;
      third = following;
    }
    const float weights = columns.total + __shfl_xor(columns.total, 32);
    if (first_column + n >= item.columns) return;
    if (part) {
      float* to = part + (first_column + n) * (D + 4);
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(f32x4*)(to + t * 32 + 8 * i + 4 * h) = (f32x4){columns.sum[t][4 * i], columns.sum[t][4 * i + 1], columns.sum[t][4 * i + 2], columns.sum[t][4 * i + 3]};
      if (h == 0) *(f32x4*)(to + D) = (f32x4){columns.begun ? columns.reference : -INFINITY, weights, 0.f, 0.f};
    } else {
      const float over = 1.f / weights;
      bf16_t* to = out + (size_t)(item.first_row + token) * out_stride + (kv_head * group + flat - token * group) * D;
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          union { bf16_t e[4]; u32x2 u; } four;
#pragma unroll
          for (int j = 0; j < 4; ++j) four.e[j] = (bf16_t)(columns.sum[t][4 * i + j] * over);
          if (whole_out) {
            *(u32x2*)(to + t * 32 + 8 * i + 4 * h) = four.u;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) to[t * 32 + 8 * i + 4 * h + j] = four.e[j];
          }
        }
    }
  });
}

// ---------------------------------------------------------------------------------------------------------------- launches

constexpr int WORKGROUPS = 512, PORTION_WORKGROUPS = 512;  // two a CU, as many as its LDS or registers hold (at heads of up to 128)

template <typename T>
static int launch(const void* q, int q_stride, void* out, int out_stride, const void* pages, const Walk& w, const Streams& few, const Streams& many, int tokens, int kinds, bool shared, hipStream_t stream) {
  const int group = w.heads / w.kv_heads, piece = sizeof(T) == 4 ? 4 : 8, whole = (size_t)q % 16 == 0 && q_stride % piece == 0;
  if (kinds & 1) {
    const long blocks = few.least ? WORKGROUPS : (long)w.requests * ((group + 15) / 16) * w.kv_heads;
    if (blocks >= (1L << 31)) return ERR_BAD_ARGUMENT;
    packed_streams_kernel<T><<<(unsigned)blocks, WAVES * WAVE, 0, stream>>>((const T*)q, q_stride, (T*)out, out_stride, (const unsigned char*)pages, w, few, whole);
    if (int status = LAUNCH_STATUS()) return status;
    if (few.least) packed_join_kernel<T><<<dim3(WORKGROUPS, 4), 4 * WAVE, 0, stream>>>((T*)out, out_stride, few, 16);
    if (int status = LAUNCH_STATUS()) return status;
  }
  if (!(kinds & 2)) return 0;
  if constexpr (sizeof(T) == 2) {
    if (shared) {
      const long items = ((long)tokens * group + SHARED_COLUMNS - 1) / SHARED_COLUMNS + w.requests, blocks = many.least ? PORTION_WORKGROUPS : items * w.kv_heads;
      if (blocks >= (1L << 31)) return ERR_BAD_ARGUMENT;
      const int whole_out = (size_t)out % 8 == 0 && out_stride % 4 == 0;
      packed_shared_kernel<<<(unsigned)blocks, PORTION_THREADS, 0, stream>>>((const T*)q, q_stride, (T*)out, out_stride, (const unsigned char*)pages, w, many, (int)items, whole, whole_out);
      if (int status = LAUNCH_STATUS()) return status;
      if (many.least) packed_join_kernel<T><<<dim3(PORTION_WORKGROUPS, SHARED_COLUMNS / 4), 4 * WAVE, 0, stream>>>((T*)out, out_stride, many, SHARED_COLUMNS);
      return LAUNCH_STATUS();
    }
  }
  const long items = ((long)tokens * group + PORTION_COLUMNS<T> - 1) / PORTION_COLUMNS<T> + w.requests, blocks = many.least ? PORTION_WORKGROUPS : items * w.kv_heads;
  if (blocks >= (1L << 31)) return ERR_BAD_ARGUMENT;
  packed_portions_kernel<T><<<(unsigned)blocks, PORTION_THREADS, 0, stream>>>((const T*)q, q_stride, (T*)out, out_stride, (const unsigned char*)pages, w, many, (int)items, whole);
  if (int status = LAUNCH_STATUS()) return status;
  if (many.least) packed_join_kernel<T><<<dim3(PORTION_WORKGROUPS, PORTION_COLUMNS<T> / 4), 4 * WAVE, 0, stream>>>((T*)out, out_stride, many, PORTION_COLUMNS<T>);
  return LAUNCH_STATUS();
}

// Floats of workspace that requests of few columns (kind 0), of many (1), of many that share tiles (2), need where walks may be cut.
extern "C" int llmserve_packed_attention_workspace(int kind) {
  return kind == 0 ? WORKGROUPS * (2 * PART + (int)(sizeof(Cut) / 4)) : PORTION_WORKGROUPS * (2 * (kind == 1 ? 32 : SHARED_COLUMNS) * (D + 4) + (int)(sizeof(Cut) / 4));
}

// q's heads are the first columns of rows of q_stride; tokens, requests: as many rows and requests as the arrays hold.  kinds: 1: some requests may have few columns (a
// single token, or no more than 16 of them in all), 2: some may have more, 4: those share tiles of keys
// (bfloat16), 8 (and not 1): all go as those of many.  few_least, many_least: 0: a walk over the keys of few (many) columns is taken whole by one workgroup; else every
// workgroup takes at least so many units of 256 (128; that share, 64) keys, walks are cut, and there is a workspace.  Those of many columns are cut for up to 256 requests alone.
extern "C" int llmserve_packed_attention(const void* q, int is_float, int q_stride, void* out, int out_stride, void* few_workspace, void* many_workspace, const void* pages, int num_pages, const int* tables,
                                         int table_width, const int* query_start, const int* contexts, int requests, int tokens, int heads, int kv_heads, int page_size, float scale, int window, int kinds,
                                         int few_least, int many_least, hipStream_t stream) {
  if (tokens == 0 || requests == 0) return 0;
  if (!q || !out || !pages || !tables || !query_start || !contexts || requests < 0 || tokens < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || num_pages <= 0 || table_width <= 0 ||
      !packed_fits(D, page_size) || (long)page_size * D * kv_heads >= (1L << 30) || !(scale > 0.f) || (size_t)pages % 16 || q_stride < heads * D || out_stride < heads * D || window < 0 ||
      (kinds & 3) == 0 || kinds < 1 || kinds > 15 || (is_float && (kinds & 4)) || ((kinds & 8) && (kinds & 3) != 2) || few_least < 0 || (few_least > 0 && (!few_workspace || (size_t)few_workspace % 16)) || many_least < 0 ||
      (many_least > 0 && (!many_workspace || (size_t)many_workspace % 16 || requests > PORTION_THREADS)))
    return ERR_BAD_ARGUMENT;
  const unsigned per_page = (unsigned)page_size / 8;
  const bool power_of_two = (per_page & (per_page - 1)) == 0;
  // (a quotient by the reciprocal is exact below 2^32 over the divisor; pieces up to a few tiles beyond the tables are asked for)
  if (!power_of_two && ((unsigned long)table_width * per_page + 64) * per_page >= (1UL << 32)) return ERR_BAD_ARGUMENT;
  const Walk w = {tables, table_width, num_pages, page_size, power_of_two ? 31 - __builtin_clz(per_page) : -1, (unsigned)(((1UL << 32) + per_page - 1) / per_page), query_start, contexts, requests, heads, kv_heads, window, scale * LOG2_E, (kinds & 8) != 0};
  const Streams few = {(float*)few_workspace, (Cut*)((float*)few_workspace + WORKGROUPS * 2 * PART), few_least};
  const bool shared = kinds & 4;
  const Streams many = {(float*)many_workspace, (Cut*)((float*)many_workspace + PORTION_WORKGROUPS * 2 * (shared ? SHARED_COLUMNS : 32) * (D + 4)), many_least};
  if (is_float) return launch<float>(q, q_stride, out, out_stride, pages, w, few, many, tokens, kinds, shared, stream);
  return launch<bf16_t>(q, q_stride, out, out_stride, pages, w, few, many, tokens, kinds, shared, stream);
}
