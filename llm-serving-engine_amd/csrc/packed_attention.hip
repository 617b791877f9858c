// Grouped-query attention over pages in 4 bits (packed.h), softmax in float32.  Compiled once per head size.
#include "packed.h"

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<multiple of 32>"
#endif

// One wave a (token, query head): a lane a key for the scores, a lane some dimensions for the sum of values.
template <typename T>
__global__ void __launch_bounds__(64) packed_attention_kernel(const T* q, int q_stride, T* out, int out_stride, const unsigned char* pages, int num_pages, const int* tables, int table_width,
                                                              const int* query_start, const int* contexts, int requests, int heads, int kv_heads, int page_size, float scale, int window) {
  constexpr int D = HEAD_DIM;
  __shared__ float query[D];
  __shared__ float weights[WAVE];
  const int token = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
  int request = 0;
  while (request < requests && query_start[request + 1] <= token) ++request;
  if (request == requests) return;
  const int context = contexts[request], position = context - query_start[request + 1] + token;
  const int kv_head = head / (heads / kv_heads);
  const PackedPage page = {D, page_size};
  for (int d = lane; d < D; d += WAVE) query[d] = to_float(q[(size_t)token * q_stride + head * D + d]) * scale * 1.44269504088896f;
  __syncthreads();
  constexpr int EACH = (D + WAVE - 1) / WAVE;
  float sum[EACH] = {}, total = 0.f, reference = -INFINITY;
  const int last = min(position, table_width * page_size - 1);
  for (int base = window > 0 ? max(0, position - window + 1) : 0; base <= last; base += WAVE) {
    const int key = base + lane;
    float score = -INFINITY;
    if (key <= last) {
      const int at = tables[(size_t)request * table_width + key / page_size];
      const unsigned char* mine = pages + ((size_t)((unsigned)at < (unsigned)num_pages ? at : 0) * kv_heads + kv_head) * page.bytes();
      score = 0.f;
      for (int g = 0; g < D / 8; ++g) {
        const unsigned codes = *(const unsigned*)(mine + page.key_codes(key % page_size, g));
        const float power = packed_power(mine[page.key_power(key % page_size, g / 4)]);
        const unsigned pairs[4] = {unpack_pair<0>(codes, power), unpack_pair<1>(codes, power), unpack_pair<2>(codes, power), unpack_pair<3>(codes, power)};
        for (int i = 0; i < 4; ++i) score += query[g * 8 + 2 * i] * __uint_as_float(pairs[i] << 16) + query[g * 8 + 2 * i + 1] * __uint_as_float(pairs[i] & 0xffff0000u);
      }
    }
    const float larger = fmaxf(reference, wave_max(score));
    const float change = reference == -INFINITY ? 0.f : exp2f(reference - larger), weight = key > last ? 0.f : exp2f(score - larger);
    reference = larger;
    total = total * change + wave_sum(weight);
    __syncthreads();
    weights[lane] = weight;
    __syncthreads();
    for (int e = 0; e < EACH; ++e) {
      const int d = lane + e * WAVE;
      if (d >= D) continue;
      sum[e] *= change;
      for (int k = 0; k < WAVE && base + k <= last; ++k) {
        const int at = tables[(size_t)request * table_width + (base + k) / page_size], offset = (base + k) % page_size;
        const unsigned char* mine = pages + ((size_t)((unsigned)at < (unsigned)num_pages ? at : 0) * kv_heads + kv_head) * page.bytes();
        const unsigned codes = *(const unsigned*)(mine + page.value_codes(offset, d / 8)) >> (d % 8 / 2 * 8);
        const unsigned pair = unpack_pair<0>(codes, packed_power(mine[page.value_power(offset, d / 32)]));
        sum[e] += weights[k] * __uint_as_float(d % 2 ? pair & 0xffff0000u : pair << 16);
      }
    }
  }
  for (int e = 0; e < EACH; ++e)
    if (lane + e * WAVE < D) out[(size_t)token * out_stride + head * D + lane + e * WAVE] = from_float<T>(sum[e] / total);
}

extern "C" int llmserve_packed_attention(const void* q, int is_float, int q_stride, void* out, int out_stride, void* partial, const void* pages, int num_pages, const int* tables, int table_width,
                                         const int* query_start, const int* contexts, int requests, int tokens, int heads, int kv_heads, int page_size, float scale, int window, int splits, hipStream_t stream) {
  if (tokens == 0 || requests == 0) return 0;
  if (!q || !out || !pages || !tables || !query_start || !contexts || requests < 0 || tokens < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || num_pages <= 0 || table_width <= 0 ||
      !packed_fits(HEAD_DIM, page_size) || (size_t)pages % 16 || q_stride < heads * HEAD_DIM || out_stride < heads * HEAD_DIM || window < 0)
    return ERR_BAD_ARGUMENT;
  const dim3 grid(tokens, heads);
  if (is_float)
    packed_attention_kernel<float><<<grid, 64, 0, stream>>>((const float*)q, q_stride, (float*)out, out_stride, (const unsigned char*)pages, num_pages, tables, table_width, query_start, contexts, requests, heads, kv_heads, page_size, scale, window);
  else
    packed_attention_kernel<bf16_t><<<grid, 64, 0, stream>>>((const bf16_t*)q, q_stride, (bf16_t*)out, out_stride, (const unsigned char*)pages, num_pages, tables, table_width, query_start, contexts, requests, heads, kv_heads, page_size, scale, window);
  return LAUNCH_STATUS();
}
