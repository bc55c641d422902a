// Letting tokens go: of every request and kv head the last `recent` tokens and the heaviest of the others, `keep` in
// all, are moved to other pages in their order, with their weights.
//
//   choose   one block per (request, kv head).  The weights are ordered as unsigned words (negative
//            below positive, not-a-number above all); the smallest that is kept is found eight bits at a
//            time by counting how many candidates share the bits found so far, and among equal ones the first are
//            kept.  Integer counts only: the result does not depend on the order in which the threads count.
//   move     the chosen tokens' keys, values, factors and weights, gathered into the new pages.
//
// `weights` lies in pages beside the cache: [pages, kv_heads, page_size] float.  The new pages must not be among the
// requests' old ones: the old are read while the new are written.
#include "fp4.h"

#define CHOOSE_THREADS 1024

__device__ __forceinline__ uint32_t order_word(float w) {     // larger weights, larger words
  const uint32_t bits = __float_as_uint(w);
  if ((bits & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;                      // not a number: kept first
  if ((bits & 0x7fffffffu) == 0) return 0x80000000u;                               // -0 is 0
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__global__ void __launch_bounds__(CHOOSE_THREADS)
choose_tokens_kernel(const float* __restrict__ weights, const int32_t* __restrict__ block_table, int bt_stride,
                     const int32_t* __restrict__ lengths, int longest, int kv_heads, int page_size, int keep, int recent,
                     int32_t* __restrict__ kept) {
  __shared__ int bins[256];
  __shared__ int wave_counts[2][CHOOSE_THREADS / SE_WAVE];
  __shared__ uint32_t found_prefix;
  __shared__ int found_above;
  const int item = blockIdx.y, kvh = blockIdx.x, tid = threadIdx.x;
  const int lane = tid & (SE_WAVE - 1), wave = tid / SE_WAVE;
  const int length = min(lengths[item], longest);      // the block table's rows hold `longest` tokens
  const int32_t* table = block_table + static_cast<int64_t>(item) * bt_stride;
  int32_t* dst = kept + (static_cast<int64_t>(item) * kv_heads + kvh) * keep;
  if (length <= keep) {      // nothing goes
    for (int i = tid; i < keep; i += CHOOSE_THREADS) dst[i] = i < length ? i : -1;
    return;
  }
  const int late = recent < keep ? recent : keep;
  const int candidates = length - late;      // tokens before the recent ones
  const int want = keep - late;              // of which so many stay (fewer than all: length > keep)
  auto word_at = [&](int i) {
    return order_word(weights[(static_cast<int64_t>(table[i / page_size]) * kv_heads + kvh) * page_size + i % page_size]);
  };
  // the want-th largest word: the bits found so far, and how many candidates lie above everything that shares them
  uint32_t prefix = 0;
  int above = 0;
  if (want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += CHOOSE_THREADS) bins[i] = 0;
      __syncthreads();
      const uint32_t high = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
      for (int i = tid; i < candidates; i += CHOOSE_THREADS) {
        const uint32_t w = word_at(i);
        if ((w & high) == prefix) atomicAdd(&bins[w >> shift & 255u], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int sum = above, b = 255;
        while (b > 0 && sum + bins[b] < want) sum += bins[b--];
        found_prefix = prefix | static_cast<uint32_t>(b) << shift;
        found_above = sum;
      }
      __syncthreads();
      prefix = found_prefix;
      above = found_above;
    }
  }
  const int equal_wanted = want - above;     // of the tokens whose word is `prefix`, the first so many
  // in order: which tokens stay, and where they go
  int placed = 0, equal_seen = 0;            // before the current chunk, the same in all threads
  for (int base = 0; base < length; base += CHOOSE_THREADS) {
    const int i = base + tid;
    bool stays = false, equal = false;
    if (i < candidates && want > 0) {
      const uint32_t w = word_at(i);
      stays = w > prefix;
      equal = w == prefix;
    } else if (i >= candidates && i < length) {
      stays = true;
    }
    const uint64_t equal_mask = __ballot(equal);
    const uint64_t before = (1ull << lane) - 1;
    if (lane == 0) wave_counts[0][wave] = __popcll(equal_mask);
    __syncthreads();
    int equal_rank = equal_seen + __popcll(equal_mask & before), equal_total = 0;
    for (int w = 0; w < CHOOSE_THREADS / SE_WAVE; ++w) {
      if (w < wave) equal_rank += wave_counts[0][w];
      equal_total += wave_counts[0][w];
    }
    if (equal && equal_rank < equal_wanted) stays = true;
    const uint64_t stay_mask = __ballot(stays);
    if (lane == 0) wave_counts[1][wave] = __popcll(stay_mask);
    __syncthreads();
    int rank = placed + __popcll(stay_mask & before), total = 0;
    for (int w = 0; w < CHOOSE_THREADS / SE_WAVE; ++w) {
      if (w < wave) rank += wave_counts[1][w];
      total += wave_counts[1][w];
    }
    if (stays && rank < keep) dst[rank] = i;
    placed += total;
    equal_seen += equal_total;
  }
}

// Where a new page's token comes from: the cache offset (in tokens of a kv head's pages) of its old place, or -1.
struct OldPlace {
  int page, off;
};
__device__ __forceinline__ OldPlace old_place(const int32_t* table, const int32_t* kept, int to, int keep, int page_size) {
  const int from = to < keep ? kept[to] : -1;
  if (from < 0) return {-1, 0};
  return {table[from / page_size], from % page_size};
}

// One block per (page of the new table, kv head, request x {keys, values}); E: the size of a stored element.
template <typename E>
__global__ void __launch_bounds__(256)
move_tokens_kernel(E* cache, float* weights, const int32_t* __restrict__ block_table, int bt_stride,
                   const int32_t* __restrict__ new_table, int new_stride, const int32_t* __restrict__ kept,
                   int kv_heads, int page_size, int head_dim, int keep) {
  extern __shared__ int places[];       // [page_size][2]: the old page and offset of every token of the new page
  const int item = blockIdx.z >> 1, which = blockIdx.z & 1, kvh = blockIdx.y;
  const int32_t* table = block_table + static_cast<int64_t>(item) * bt_stride;
  const int32_t* mine = kept + (static_cast<int64_t>(item) * kv_heads + kvh) * keep;
  const int to_page = new_table[static_cast<int64_t>(item) * new_stride + blockIdx.x];
  if (to_page < 0) return;
  const int base = blockIdx.x * page_size;
  for (int t = threadIdx.x; t < page_size; t += blockDim.x) {
    const OldPlace from = old_place(table, mine, base + t, keep, page_size);
    places[2 * t] = from.page;
    places[2 * t + 1] = from.off;
    if (which == 0 && from.page >= 0)
      weights[(static_cast<int64_t>(to_page) * kv_heads + kvh) * page_size + t] =
          weights[(static_cast<int64_t>(from.page) * kv_heads + kvh) * page_size + from.off];
  }
  __syncthreads();
  const int64_t span = static_cast<int64_t>(page_size) * head_dim;
  auto part = [&](int page) { return cache + ((static_cast<int64_t>(page) * 2 + which) * kv_heads + kvh) * span; };
  E* dst = part(to_page);
  if (which == 0) {         // keys: eight neighbouring dims of a token at a time
    struct alignas(16) Eight { E v[8]; };
    for (int i = threadIdx.x; i < page_size * head_dim / 8; i += blockDim.x) {
      const int d8 = i / page_size, t = i % page_size;
      if (places[2 * t] < 0) continue;
      *reinterpret_cast<Eight*>(dst + key_place(page_size, t, d8 * 8)) =
          *reinterpret_cast<const Eight*>(part(places[2 * t]) + key_place(page_size, places[2 * t + 1], d8 * 8));
    }
  } else {
    for (int i = threadIdx.x; i < page_size * head_dim; i += blockDim.x) {
      const int t = i / 8 / head_dim * 8 + i % 8, d = i / 8 % head_dim;      // i: the place in the new page
      if (places[2 * t] < 0) continue;
      dst[i] = part(places[2 * t])[value_place(head_dim, places[2 * t + 1], d)];
    }
  }
}

// The same for the 4-bit cache: codes and factors are moved as they are.
__global__ void __launch_bounds__(256)
move_tokens_fp4_kernel(uint8_t* cache, float* weights, const int32_t* __restrict__ block_table, int bt_stride,
                       const int32_t* __restrict__ new_table, int new_stride, const int32_t* __restrict__ kept,
                       int kv_heads, int page_size, int head_dim, int keep) {
  extern __shared__ int places[];
  const int item = blockIdx.z >> 1, which = blockIdx.z & 1, kvh = blockIdx.y;
  const int32_t* table = block_table + static_cast<int64_t>(item) * bt_stride;
  const int32_t* mine = kept + (static_cast<int64_t>(item) * kv_heads + kvh) * keep;
  const int to_page = new_table[static_cast<int64_t>(item) * new_stride + blockIdx.x];
  if (to_page < 0) return;
  const int base = blockIdx.x * page_size;
  for (int t = threadIdx.x; t < page_size; t += blockDim.x) {
    const OldPlace from = old_place(table, mine, base + t, keep, page_size);
    places[2 * t] = from.page;
    places[2 * t + 1] = from.off;
    if (which == 0 && from.page >= 0)
      weights[(static_cast<int64_t>(to_page) * kv_heads + kvh) * page_size + t] =
          weights[(static_cast<int64_t>(from.page) * kv_heads + kvh) * page_size + from.off];
  }
  __syncthreads();
  const int groups = head_dim / FP4_GROUP;
  const int64_t span = fp4_head_bytes(page_size, head_dim);
  auto part = [&](int page) { return cache + ((static_cast<int64_t>(page) * 2 + which) * kv_heads + kvh) * span; };
  uint8_t* dst = part(to_page);
  for (int i = threadIdx.x; i < page_size * groups; i += blockDim.x) {
    const int group = i / page_size, t = i % page_size;
    if (places[2 * t] < 0) continue;
    const uint8_t* src = part(places[2 * t]);
    const int off = places[2 * t + 1];
    if (which == 0) {
      *reinterpret_cast<uint4*>(dst + fp4_key_code_at(page_size, t, group)) =
          *reinterpret_cast<const uint4*>(src + fp4_key_code_at(page_size, off, group));
      dst[fp4_key_factor_at(page_size, head_dim, t, group)] = src[fp4_key_factor_at(page_size, head_dim, off, group)];
    } else {
      for (int j = 0; j < 16; ++j)
        dst[fp4_value_code_at(head_dim, t, group, j)] = src[fp4_value_code_at(head_dim, off, group, j)];
      dst[fp4_value_factor_at(page_size, head_dim, t, group)] = src[fp4_value_factor_at(page_size, head_dim, off, group)];
    }
  }
}

// kind 0: float, 1: bfloat16, 2: 4 bits.  kept: int32 [items, kv_heads, keep], ascending, -1 behind the last of a
// request that has fewer tokens.
extern "C" int se_evict_tokens(void* cache, int kind, float* weights, const int32_t* block_table, int bt_stride,
                               const int32_t* lengths, int items, int longest, const int32_t* new_table, int new_stride, int keep,
                               int recent, int32_t* kept, int kv_heads, int page_size, int head_dim, hipStream_t stream) {
  if (items <= 0 || keep <= 0) return SE_OK;
  if (recent < 0 || recent > keep || kv_heads <= 0 || kv_heads > 65535 || items > 32767) return SE_ERR_SHAPE;
  if (page_size <= 0 || page_size % 8 || page_size > 4096 || head_dim <= 0 || head_dim % 8) return SE_ERR_SHAPE;
  if (kind == 2 && (head_dim % 32 || page_size % 32)) return SE_ERR_SHAPE;
  choose_tokens_kernel<<<dim3(kv_heads, items), CHOOSE_THREADS, 0, stream>>>(
      weights, block_table, bt_stride, lengths, longest, kv_heads, page_size, keep, recent, kept);
  SE_CHECK_LAUNCH();
  const dim3 grid((keep + page_size - 1) / page_size, kv_heads, items * 2);
  const size_t shared = static_cast<size_t>(page_size) * 2 * sizeof(int);
  if (kind == 0)
    move_tokens_kernel<float><<<grid, 256, shared, stream>>>(static_cast<float*>(cache), weights, block_table, bt_stride,
                                                             new_table, new_stride, kept, kv_heads, page_size, head_dim, keep);
  else if (kind == 1)
    move_tokens_kernel<uint16_t><<<grid, 256, shared, stream>>>(static_cast<uint16_t*>(cache), weights, block_table, bt_stride,
                                                                new_table, new_stride, kept, kv_heads, page_size, head_dim, keep);
  else if (kind == 2)
    move_tokens_fp4_kernel<<<grid, 256, shared, stream>>>(static_cast<uint8_t*>(cache), weights, block_table, bt_stride,
                                                          new_table, new_stride, kept, kv_heads, page_size, head_dim, keep);
  else
    return SE_ERR_SHAPE;
  SE_CHECK_LAUNCH();
  return SE_OK;
}
