// A step's index arrays from its requests' lengths.
//
// Request b has its block-table row at slots[b] of the cache's tables ([groups][table_rows][blocks], -1: no page), `starts[b]` tokens cached and counts[b] more in
// this step.  Its tokens follow those of the requests before it; token i of it is at position starts[b] + i, and lies in group g's page
// tables[g][slots[b]][position / page_size] at position % page_size.  A request whose slot is not one of the tables' rows only pads the step: its tokens are at position 0
// and stored nowhere, its context is one token in page 0.  Rows behind the last request's are such tokens of the last one.
//
// A few kilobytes are read and written: what counts is one launch instead of a host's arrays and their copy.  A workgroup of the first
// `token_blocks` takes 256 tokens and needs all requests' ends for that, which it adds up by itself (a few hundred counts, out of the L2); the others take a row of
// a compact table each.  A single token takes 2.5 us, 63 beside a portion of 2,048 with two groups 3.6: the launch, and three trips to memory behind each other.
#include "common.h"

#define PLACE_THREADS 256
#define PLACE_LONGEST (1 << 30)  // positions and counts are taken up to here: no sum of two passes 32 bits
#define PLACE_REQUESTS 4096  // the ends of so many requests lie in LDS

__device__ __forceinline__ int length_of(int given) { return min(max(given, 0), PLACE_LONGEST - 1); }

__global__ void __launch_bounds__(PLACE_THREADS) place_tokens_kernel(const int* tables, int groups, int table_rows, int blocks, const int* slots, const int* starts, const int* counts, int requests,
                                                                      int page_size, int tokens, int width, int token_blocks, int* positions, int* sequence, int* query_start, int* contexts,
                                                                      int* mapping, int mapping_stride, int* compact, int compact_stride) {
  __shared__ int ends[PLACE_REQUESTS];
  __shared__ int sums[PLACE_THREADS / WAVE];
  if ((int)blockIdx.x >= token_blocks) {
    const int row = blockIdx.x - token_blocks, group = row / requests, request = row - group * requests, slot = slots[request];
    const bool real = slot >= 0 && slot < table_rows;
    const int held = real ? (int)(((long)length_of(starts[request]) + length_of(counts[request]) + page_size - 1) / page_size) : 0;
    const int* from = tables + ((size_t)group * table_rows + (real ? slot : 0)) * blocks;
    int* to = compact + (size_t)group * compact_stride + (size_t)request * width;
    for (int i = threadIdx.x; i < width; i += PLACE_THREADS) to[i] = !real ? 0 : i < held && i < blocks ? from[i] : -1;
    return;
  }
  // the requests' ends: a run of counts a thread, the runs' sums added up over the workgroup
  const int run = (requests + PLACE_THREADS - 1) / PLACE_THREADS, first = threadIdx.x * run, lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
  int mine = 0;
  for (int i = first; i < min(first + run, requests); ++i) {
    mine = min(mine + min(max(counts[i], 0), tokens), tokens);
    ends[i] = mine;
  }
  int before = mine;
#pragma unroll
  for (int step = 1; step < WAVE; step <<= 1) {
    const int other = __shfl_up(before, step);
    if (lane >= step) before = min(before + other, tokens);
  }
  if (lane == WAVE - 1) sums[wave] = before;
  __syncthreads();
  int carried = __shfl_up(before, 1);
  if (lane == 0) carried = 0;
  for (int w = 0; w < wave; ++w) carried = min(carried + sums[w], tokens);
  for (int i = first; i < min(first + run, requests); ++i) ends[i] = min(ends[i] + carried, tokens);
  __syncthreads();
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) query_start[0] = 0;
    for (int i = threadIdx.x; i < requests; i += PLACE_THREADS) {
      query_start[i + 1] = ends[i];
      contexts[i] = slots[i] >= 0 && slots[i] < table_rows ? length_of(starts[i]) + length_of(counts[i]) : 1;
    }
  }
  const int token = blockIdx.x * PLACE_THREADS + threadIdx.x;
  if (token >= tokens) return;
  int low = 0, high = requests;  // the first request that ends behind the token
  while (low < high) {
    const int middle = (low + high) / 2;
    if (ends[middle] > token) high = middle;
    else low = middle + 1;
  }
  const int request = min(low, requests - 1), slot = slots[request];
  const bool real = low < requests && slot >= 0 && slot < table_rows;
  const int position = real ? length_of(starts[request]) + token - (request > 0 ? ends[request - 1] : 0) : 0, block = position / page_size;
  positions[token] = position;
  sequence[token] = request;
  for (int g = 0; g < groups; ++g) {
    const int page = real && block < blocks ? tables[((size_t)g * table_rows + slot) * blocks + block] : -1;
    mapping[(size_t)g * mapping_stride + token] = page < 0 ? -1 : page * page_size + (position - block * page_size);
  }
}

extern "C" int llmserve_place_tokens(const int* tables, int groups, int table_rows, int blocks, const int* slots, const int* starts, const int* counts, int requests, int page_size, int tokens,
                                     int width, int* positions, int* sequence, int* query_start, int* contexts, int* mapping, int mapping_stride, int* compact, int compact_stride, hipStream_t stream) {
  if (!tables || !slots || !starts || !counts || !query_start || !contexts || !compact || (tokens > 0 && (!positions || !sequence || !mapping)) || groups < 1 || groups > 64 || table_rows < 1 || blocks < 1 ||
      requests < 1 || requests > PLACE_REQUESTS || page_size < 1 || tokens < 0 || tokens >= PLACE_LONGEST || width < 1)
    return ERR_BAD_ARGUMENT;
  const int token_blocks = tokens > 0 ? (tokens + PLACE_THREADS - 1) / PLACE_THREADS : 1;
  const long all = token_blocks + (long)groups * requests;
  if (all >= (1L << 31)) return ERR_BAD_ARGUMENT;
  place_tokens_kernel<<<(unsigned)all, PLACE_THREADS, 0, stream>>>(tables, groups, table_rows, blocks, slots, starts, counts, requests, page_size, tokens, width, token_blocks, positions, sequence,
                                                                   query_start, contexts, mapping, mapping_stride, compact, compact_stride);
  return LAUNCH_STATUS();
}
