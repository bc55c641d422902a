// Letting tokens go: of every request and kv head the last `recent` tokens and the heaviest of the others, `keep` in
// all, are moved to other pages in their order, with their weights.
//
//   choose   one block per (request, kv head).  The weights are ordered as unsigned words (negative below positive,
//            not-a-number above all), read once and kept in registers (up to 32768 tokens; the rest is read again in
//            every pass).  The smallest word that is kept is found eight bits a pass from counts of the candidates
//            that share the bits found so far (integer additions in shared memory, sixteen copies of every count so
//            that the crowd of words with one exponent does not queue up at one address); the search ends early when
//            the words at or above the one found are just those wanted, and among words equal to the smallest the
//            first are kept.  Whole numbers only: the result does not depend on the order in which threads count.
//            One block's chain of passes: 2048 of 2112 tokens 12 us, 8192 of 32768 tokens 40 us, whatever the heads.
//   move     the chosen tokens' keys, values, factors and weights, gathered into the new pages.  Bound by reading: tokens
//            lie in groups of eight in a page, so that a fourth of the tokens, chosen here and there, touches nearly
//            every line of the old pages (4 requests, 8192 of 32768 tokens, bfloat16, 8 heads of 128: 126 us for 537 MB
//            touched and 134 MB written, 5.3 TB/s; 8 requests, 2048 of 2112 tokens in 4 bits: 12.6 us).
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

// the word of a token's weight; a token whose page is gone comes behind every weight
__device__ __forceinline__ uint32_t word_of(int page, float w) {
  return page < 0 ? 1u : order_word(w);
}

#define CHOOSE_WAVES (CHOOSE_THREADS / SE_WAVE)
#define CHOOSE_COPIES 16

// Exclusive prefix sums of `counts` [rounds][CHOOSE_WAVES] in place, and their sum; entries <= CHOOSE_THREADS.
__device__ __forceinline__ int scan_counts(int* counts, int entries, int* wave_sums) {
  const int tid = threadIdx.x, lane = tid & (SE_WAVE - 1), wave = tid / SE_WAVE;
  const int own = tid < entries ? counts[tid] : 0;
  int upto = own;
#pragma unroll
  for (int off = 1; off < SE_WAVE; off <<= 1) {
    const int other = __shfl_up(upto, off, SE_WAVE);
    if (lane >= off) upto += other;
  }
  if (lane == SE_WAVE - 1) wave_sums[wave] = upto;
  __syncthreads();
  int before = 0, total = 0;
  for (int w = 0; w < CHOOSE_WAVES; ++w) {
    if (w < wave) before += wave_sums[w];
    total += wave_sums[w];
  }
  if (tid < entries) counts[tid] = before + upto - own;
  __syncthreads();
  return total;
}

// R: words a thread keeps in registers; tokens beyond R * CHOOSE_THREADS are read again whenever they are looked at.
template <int R>
__global__ void __launch_bounds__(CHOOSE_THREADS)
choose_tokens_kernel(const float* __restrict__ weights, const int32_t* __restrict__ block_table, int bt_stride,
                     const int32_t* __restrict__ lengths, int longest, int kv_heads, int page_size, int keep, int recent,
                     int32_t* __restrict__ kept) {
  __shared__ int round_counts[R * CHOOSE_WAVES];      // per (round of CHOOSE_THREADS tokens, wavefront)
  __shared__ int wave_counts[2][CHOOSE_WAVES];
  __shared__ int bins[256 * CHOOSE_COPIES], own_sum[256], upto_sum[256], found[3];
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
  // The words of tokens base + tid, base + tid + CHOOSE_THREADS, ...: 0, which is no weight's word, for what is no
  // candidate.  The page of the next token is found by adding, not by dividing.
  const int step_pages = CHOOSE_THREADS / page_size, step_off = CHOOSE_THREADS - step_pages * page_size;
  auto read_words = [&](int base, uint32_t (&word)[R]) {
    int page = (base + tid) / page_size, off = (base + tid) - page * page_size;
    int id[R], at[R];       // all page ids on their way at once, then all weights (the first token's for no candidate)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool candidate = base + r * CHOOSE_THREADS + tid < candidates;
      id[r] = candidate ? table[page] : 0;
      at[r] = candidate ? off : 0;
      page += step_pages;
      off += step_off;
      if (off >= page_size) {
        off -= page_size;
        ++page;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float w = weights[(static_cast<int64_t>(max(id[r], 0)) * kv_heads + kvh) * page_size + at[r]];
      word[r] = base + r * CHOOSE_THREADS + tid < candidates ? word_of(id[r], w) : 0u;
    }
  };
  uint32_t word[R];
  read_words(0, word);

  // the want-th largest word, and how many candidates lie at or above it
  uint32_t least = 0;
  int above = 0, at_or_above = 0;      // above: of the candidates that do not share the bits found so far
  for (int shift = 24; want > 0 && shift >= 0 && at_or_above != want; shift -= 8) {
    const uint32_t high = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    for (int i = tid; i < 256 * CHOOSE_COPIES; i += CHOOSE_THREADS) bins[i] = 0;
    __syncthreads();
    auto count = [&](uint32_t w) {
      if (w != 0 && (w & high) == least) atomicAdd(&bins[(w >> shift & 255u) * CHOOSE_COPIES + lane % CHOOSE_COPIES], 1);
    };
#pragma unroll
    for (int r = 0; r < R; ++r) count(word[r]);
    int page = (R * CHOOSE_THREADS + tid) / page_size, off = (R * CHOOSE_THREADS + tid) - page * page_size;
    for (int i = R * CHOOSE_THREADS + tid; i < candidates; i += CHOOSE_THREADS) {
      const int id = table[page];
      count(word_of(id, weights[(static_cast<int64_t>(max(id, 0)) * kv_heads + kvh) * page_size + off]));
      page += step_pages;
      off += step_off;
      if (off >= page_size) {
        off -= page_size;
        ++page;
      }
    }
    __syncthreads();
    if (tid < 256) {      // thread t: bin 255 - t, so that sums run from the largest words down
      int own = 0;
#pragma unroll
      for (int c = 0; c < CHOOSE_COPIES; ++c) own += bins[(255 - tid) * CHOOSE_COPIES + c];
      int upto = own;
#pragma unroll
      for (int off = 1; off < SE_WAVE; off <<= 1) {
        const int other = __shfl_up(upto, off, SE_WAVE);
        if (lane >= off) upto += other;
      }
      own_sum[tid] = own;
      upto_sum[tid] = upto;
    }
    __syncthreads();
    if (tid < 256) {
      int upto = above + upto_sum[tid];
      for (int w = 0; w < tid / SE_WAVE; ++w) upto += upto_sum[w * SE_WAVE + SE_WAVE - 1];
      if (upto >= want && upto - own_sum[tid] < want) {      // one thread
        found[0] = 255 - tid;
        found[1] = upto - own_sum[tid];
        found[2] = upto;
      }
    }
    __syncthreads();
    least |= static_cast<uint32_t>(found[0]) << shift;
    above = found[1];
    at_or_above = found[2];
  }
  // Words above `least` stay; of those equal to it the first so many (all, if the search ended with those wanted).
  const int equal_wanted = at_or_above > want ? want - above : 0x7fffffff;

  const uint64_t before = (1ull << lane) - 1;
  int placed = 0, equal_seen = 0;
  for (int base = 0; base < length; base += R * CHOOSE_THREADS) {      // R rounds at a time; the first from registers
    if (base > 0) read_words(base, word);
    if (equal_wanted != 0x7fffffff) {      // ties: which of the equal ones are among the first
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint64_t mask = __ballot(word[r] == least);
        if (lane == 0) round_counts[r * CHOOSE_WAVES + wave] = __popcll(mask);
      }
      __syncthreads();
      const int total = scan_counts(round_counts, R * CHOOSE_WAVES, wave_counts[0]);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool equal = word[r] == least;
        const uint64_t mask = __ballot(equal);
        // what does not stay becomes 0
        if (equal && equal_seen + round_counts[r * CHOOSE_WAVES + wave] + __popcll(mask & before) >= equal_wanted) word[r] = 0;
      }
      equal_seen += total;
      __syncthreads();
    }
    auto stays = [&](int r) {
      const int i = base + r * CHOOSE_THREADS + tid;
      return (want > 0 && i < candidates && word[r] >= least && word[r] != 0) || (i >= candidates && i < length);
    };
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint64_t mask = __ballot(stays(r));
      if (lane == 0) round_counts[r * CHOOSE_WAVES + wave] = __popcll(mask);
    }
    __syncthreads();
    const int total = scan_counts(round_counts, R * CHOOSE_WAVES, wave_counts[1]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool mine = stays(r);
      const uint64_t mask = __ballot(mine);
      const int rank = placed + round_counts[r * CHOOSE_WAVES + wave] + __popcll(mask & before);
      if (mine && rank < keep) dst[rank] = base + r * CHOOSE_THREADS + tid;
    }
    placed += total;
    __syncthreads();
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

// The same for the 4-bit cache, keys and values in one block: codes and factors are moved as they are.
__global__ void __launch_bounds__(256)
move_tokens_fp4_kernel(uint8_t* cache, float* weights, const int32_t* __restrict__ block_table, int bt_stride,
                       const int32_t* __restrict__ new_table, int new_stride, const int32_t* __restrict__ kept,
                       int kv_heads, int page_size, int head_dim, int keep) {
  extern __shared__ int places[];       // as above; then six numbers for every eight tokens
  const int item = blockIdx.z, kvh = blockIdx.y;
  const int32_t* table = block_table + static_cast<int64_t>(item) * bt_stride;
  const int32_t* mine = kept + (static_cast<int64_t>(item) * kv_heads + kvh) * keep;
  const int to_page = new_table[static_cast<int64_t>(item) * new_stride + blockIdx.x];
  if (to_page < 0) return;
  const int base = blockIdx.x * page_size;
  for (int t = threadIdx.x; t < page_size; t += blockDim.x) {
    const OldPlace from = old_place(table, mine, base + t, keep, page_size);
    places[2 * t] = from.page;
    places[2 * t + 1] = from.off;
    if (from.page >= 0)
      weights[(static_cast<int64_t>(to_page) * kv_heads + kvh) * page_size + t] =
          weights[(static_cast<int64_t>(from.page) * kv_heads + kvh) * page_size + from.off];
  }
  __syncthreads();
  const int groups = head_dim / FP4_GROUP;
  const int64_t span = fp4_head_bytes(page_size, head_dim);
  auto part = [&](int page, int which) { return cache + ((static_cast<int64_t>(page) * 2 + which) * kv_heads + kvh) * span; };
  // Values are moved in pieces of eight neighbouring keys' bytes, of codes (16 * groups of them to eight keys) and then of
  // factors (groups).  Where most tokens stay, the eight come from one or two pieces of the old pages, whose words are
  // read whole; else byte by byte.  (8 x 2048 of 2112 tokens: 15 us with all values byte by byte and keys and values in
  // blocks of their own, 12.6 so.)
  // Of every eight tokens: page and eight of the first and of the last, from which of the two each byte comes (bit 3 of
  // four) and where it lies there (bits 0 to 2), and whether there are eight (1), from those two only (2).
  int* eights = places + 2 * page_size;
  for (int e = threadIdx.x; e < page_size / 8; e += blockDim.x) {
    const int* from = places + 16 * e;
    int flags = 3, select = 0;
    for (int t = 0; t < 8; ++t) {
      const bool first = from[2 * t] == from[0] && from[2 * t + 1] >> 3 == from[1] >> 3;
      const bool last = from[2 * t] == from[14] && from[2 * t + 1] >> 3 == from[15] >> 3;
      if (from[2 * t] < 0) flags = 0;
      if (!first && !last) flags &= 1;
      select |= ((first ? 0 : 8) | (from[2 * t + 1] & 7)) << (4 * t);
    }
    int* to = eights + 6 * e;
    to[0] = from[0], to[1] = from[1] >> 3, to[2] = from[14], to[3] = from[15] >> 3, to[4] = select, to[5] = flags;
  }
  uint8_t* new_keys = part(to_page, 0);
  for (int i = threadIdx.x; i < page_size * groups; i += blockDim.x) {
    const int group = i / page_size, t = i % page_size;
    if (places[2 * t] < 0) continue;
    const uint8_t* src = part(places[2 * t], 0);
    const int off = places[2 * t + 1];
    *reinterpret_cast<uint4*>(new_keys + fp4_key_code_at(page_size, t, group)) =
        *reinterpret_cast<const uint4*>(src + fp4_key_code_at(page_size, off, group));
    new_keys[fp4_key_factor_at(page_size, head_dim, t, group)] = src[fp4_key_factor_at(page_size, head_dim, off, group)];
  }
  __syncthreads();
  const int code_pieces = page_size / 8 * 16 * groups, pieces = code_pieces + page_size / 8 * groups;
  for (int i = threadIdx.x; i < pieces; i += blockDim.x) {
    const bool code = i < code_pieces;
    const int per_eight = code ? 16 * groups : groups, at = code ? i : i - code_pieces;
    const int e = at / per_eight, rest = at - e * per_eight;
    const int64_t start = code ? 0 : fp4_factors_at(page_size, head_dim);
    auto piece = [&](int page, int eight) { return reinterpret_cast<const uint64_t*>(part(page, 1) + start) + eight * per_eight + rest; };
    uint64_t* to = reinterpret_cast<uint64_t*>(part(to_page, 1) + start) + at;
    const int* of = eights + 6 * e;
    const uint32_t select = static_cast<uint32_t>(of[4]);
    if (of[5] == 3) {
      const uint64_t first = *piece(of[0], of[1]), last = *piece(of[2], of[3]);
      uint64_t word = 0;
#pragma unroll
      for (int t = 0; t < 8; ++t)
        word |= ((select >> (4 * t) & 8u ? last : first) >> (8 * (select >> (4 * t) & 7u)) & 255u) << (8 * t);
      *to = word;
      continue;
    }
    const int* from = places + 16 * e;
    auto byte_of = [&](int t) { return reinterpret_cast<const uint8_t*>(piece(from[2 * t], from[2 * t + 1] >> 3))[select >> (4 * t) & 7u]; };
    if (of[5] == 1) {
      uint64_t word = 0;
#pragma unroll
      for (int t = 0; t < 8; ++t) word |= static_cast<uint64_t>(byte_of(t)) << (8 * t);
      *to = word;
    } else {
      for (int t = 0; t < 8; ++t)
        if (from[2 * t] >= 0) reinterpret_cast<uint8_t*>(to)[t] = byte_of(t);
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
#define SE_CHOOSE(R)                                                              \
  choose_tokens_kernel<R><<<dim3(kv_heads, items), CHOOSE_THREADS, 0, stream>>>( \
      weights, block_table, bt_stride, lengths, longest, kv_heads, page_size, keep, recent, kept)
  if (longest <= 4 * CHOOSE_THREADS) SE_CHOOSE(4);
  else if (longest <= 16 * CHOOSE_THREADS) SE_CHOOSE(16);
  else SE_CHOOSE(32);      // more than 32768 tokens: the rest is read again in every pass
#undef SE_CHOOSE
  SE_CHECK_LAUNCH();
  const dim3 grid((keep + page_size - 1) / page_size, kv_heads, kind == 2 ? items : items * 2);
  const size_t shared = static_cast<size_t>(page_size) * 2 * sizeof(int);
  if (kind == 0)
    move_tokens_kernel<float><<<grid, 256, shared, stream>>>(static_cast<float*>(cache), weights, block_table, bt_stride,
                                                             new_table, new_stride, kept, kv_heads, page_size, head_dim, keep);
  else if (kind == 1)
    move_tokens_kernel<uint16_t><<<grid, 256, shared, stream>>>(static_cast<uint16_t*>(cache), weights, block_table, bt_stride,
                                                                new_table, new_stride, kept, kv_heads, page_size, head_dim, keep);
  else if (kind == 2)
    move_tokens_fp4_kernel<<<grid, 256, shared + static_cast<size_t>(page_size / 8) * 6 * sizeof(int), stream>>>(static_cast<uint8_t*>(cache), weights, block_table, bt_stride,
                                                          new_table, new_stride, kept, kv_heads, page_size, head_dim, keep);
  else
    return SE_ERR_SHAPE;
  SE_CHECK_LAUNCH();
  return SE_OK;
}
