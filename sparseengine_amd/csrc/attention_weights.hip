// The softmax weight that every cached key gets from a step's rows:
//
//   out[key] = (key older than the step ? previous[key] : 0) + sum over rows that see it of exp(scale q . k - lse[row])
//
// for every request and kv head; a row is one query token and one of the kv head's query heads, lse its logarithm of
// the sum of exponentials, which the attention kernels give.  Only keys are read, once; the sum over rows stays in
// the registers of the wavefront that owns the keys and is made in one fixed order, so nothing is added atomically
// and the same step gives the same bits.
//
// `previous` and `out` lie in pages beside the cache: [pages, kv_heads, page_size] float.
#include <type_traits>

#include "fp4.h"

// where the keys of a cache kind come from: eight dims of a key at a time
enum SeCacheKind { SE_CACHE_F32 = 0, SE_CACHE_BF16 = 1, SE_CACHE_FP4 = 2 };

// General form, any head size in steps of 8 and any kind of cache (the float path of the engine, and sizes that the
// matrix-core kernel does not take): a lane owns a key, and reads it again for every row.
template <typename T, int KIND>
__global__ void __launch_bounds__(64)
attention_weights_generic_kernel(const T* __restrict__ q, int64_t q_stride, const void* __restrict__ cache,
                                 const int32_t* __restrict__ block_table, int bt_stride,
                                 const int32_t* __restrict__ item_meta, int items, int longest,
                                 const float* __restrict__ lse, const float* previous, float* out, int heads, int kv_heads, int head_dim,
                                 int page_size, float scale, int window) {
  extern __shared__ float q_row[];     // [head_dim]
  const int item = blockIdx.z, kvh = blockIdx.y, group = heads / kv_heads;
  const int q_start = item_meta[item], q_len = item_meta[items + item], ctx_len = min(item_meta[2 * items + item], longest);
  const int pos0 = ctx_len - q_len;
  const int low_key = window > 0 && pos0 - window + 1 > 0 ? pos0 - window + 1 : 0;   // no row sees a key before it
  const int base = blockIdx.x * SE_WAVE;
  if (base >= ctx_len || base + SE_WAVE <= low_key) return;
  const int key = base + threadIdx.x;
  const bool held = key < ctx_len && key >= low_key;
  const int page = held ? block_table[static_cast<int64_t>(item) * bt_stride + key / page_size] : 0;
  const int off = key % page_size;
  float total = 0.f;
  for (int rho = 0; rho < q_len * group; ++rho) {
    const int pos = pos0 + rho / group;
    if (pos < base || (window > 0 && pos - window >= base + SE_WAVE - 1)) continue;     // sees none of the 64 keys
    const int token = q_start + rho / group, head = kvh * group + rho % group;
    __syncthreads();
    for (int d = threadIdx.x; d < head_dim; d += SE_WAVE)
      q_row[d] = to_float(q[token * q_stride + static_cast<int64_t>(head) * head_dim + d]);
    __syncthreads();
    if (!held || key > pos || (window > 0 && key <= pos - window)) continue;
    float dot = 0.f;
    if constexpr (KIND == SE_CACHE_FP4) {
      const uint8_t* part = static_cast<const uint8_t*>(cache) +
                            (static_cast<int64_t>(page) * 2 * kv_heads + kvh) * fp4_head_bytes(page_size, head_dim);
      for (int d = 0; d < head_dim; d += 8) {
        const uint32_t word = *reinterpret_cast<const uint32_t*>(part + fp4_key_code_at(page_size, off, d / 32) + d % 32 / 2);
        const int factor = part[fp4_key_factor_at(page_size, head_dim, off, d / 32)];
#pragma unroll
        for (int j = 0; j < 8; ++j) dot += q_row[d + j] * fp4_value(word >> (4 * j) & 15u, factor);
      }
    } else {
      typedef typename std::conditional<KIND == SE_CACHE_F32, float, bf16_t>::type C;
      const C* part = static_cast<const C*>(cache) + (static_cast<int64_t>(page) * 2 * kv_heads + kvh) * page_size * head_dim;
      for (int d = 0; d < head_dim; d += Vec16<C>::N) {
        Vec16<C> k;
        k.v = *reinterpret_cast<const decltype(k.v)*>(part + key_place(page_size, off, d));
#pragma unroll
        for (int j = 0; j < Vec16<C>::N; ++j) dot += q_row[d + j] * k.get(j);
      }
    }
    total += expf(dot * scale - lse[static_cast<int64_t>(token) * heads + head]);
  }
  if (!held) return;
  const int64_t at = (static_cast<int64_t>(page) * kv_heads + kvh) * page_size + off;
  out[at] = (previous != nullptr && key < pos0 ? previous[at] : 0.f) + total;
}

// The matrix-core form (bfloat16 rows; head size 32 * DS; keys in bfloat16 or 4 bits).  A wavefront owns 32 * KP
// consecutive keys, whose operands it loads once and keeps in registers (4 bits are turned into bfloat16 on the
// way), and goes through the tiles of 16 rows that see any of them:
//   S = Q K^T        v_mfma_f32_16x16x32_bf16, A = 16 rows x 32 dims, B = 32 dims x 16 keys, so that a lane ends up
//                    with four rows of one key and the sum over rows is additions in a lane; the four lanes that
//                    share a key meet once at the end.
// With one tile of rows (decoding) a block is four wavefronts side by side along the keys, and the kernel is bound by
// reading the keys.  With more, the wavefronts of a block take turns at the tiles of the same keys (`row_waves`) and add
// up their sums through shared memory, in order; the kernel is then bound by the exponentials and the products.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

#define WEIGHT_MAX_WAVES 8

template <int DS>
struct WeightKeys {      // groups of 32 keys a wavefront owns: 64 registers of operands at head size 128
  static constexpr int KP = DS <= 2 ? 4 : DS <= 4 ? 2 : 1;
};

template <int DS, int KIND>
__global__ void __launch_bounds__(64 * WEIGHT_MAX_WAVES)
attention_weights_mfma_kernel(const bf16_t* __restrict__ q, int64_t q_stride, const void* __restrict__ cache,
                              const int32_t* __restrict__ block_table, int bt_stride,
                              const int32_t* __restrict__ item_meta, int items, int longest,
                              const float* __restrict__ lse, const float* previous, float* out, int heads, int kv_heads,
                              int page_size, float scale_log2e, int window, int row_waves) {
  constexpr int D = 32 * DS;
  constexpr int KP = WeightKeys<DS>::KP;
  // which eight dims of a lane's operand are those of product step ds: in 4 bits, where a lane's part of a key can be
  // one piece under one factor, neighbouring ones
  constexpr bool WIDE = KIND == SE_CACHE_FP4 && (DS == 2 || DS == 4 || DS == 8);
  __shared__ float sums[WEIGHT_MAX_WAVES][KP * 2][16];
  const int lane = threadIdx.x & (SE_WAVE - 1);
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / SE_WAVE));
  const int n = lane & 15, g = lane >> 4;
  const int item = blockIdx.z, kvh = blockIdx.y, group = heads / kv_heads;
  const int q_start = item_meta[item], q_len = item_meta[items + item], ctx_len = min(item_meta[2 * items + item], longest);
  const int pos0 = ctx_len - q_len, last_key = ctx_len - 1;
  const int low_key = window > 0 && pos0 - window + 1 > 0 ? pos0 - window + 1 : 0;   // no row sees a key before it
  const int waves = blockDim.x / SE_WAVE;
  const int part = wave % row_waves;                                                 // of the rows
  const int k_lo = (blockIdx.x * (waves / row_waves) + wave / row_waves) * (32 * KP), k_hi = k_lo + 32 * KP - 1;
  const bool wanted = k_lo < ctx_len && k_hi >= low_key;      // the same in all wavefronts that share keys
  const int32_t* table = block_table + static_cast<int64_t>(item) * bt_stride;

  auto dims_of = [&](int ds) { return WIDE ? (D / 4) * g + 8 * ds : 32 * ds + 8 * g; };
  // a lane's keys: two neighbours in 4 bits (one piece of memory), else sixteen lanes side by side
  auto key_of = [&](int kp, int b) { return k_lo + 32 * kp + (KIND == SE_CACHE_FP4 ? 2 * n + b : 16 * b + n); };

  float acc[KP][2];
#pragma unroll
  for (int kp = 0; kp < KP; ++kp) acc[kp][0] = acc[kp][1] = 0.f;

  if (wanted) {
    uint4 kf[KP][2][DS];
    if constexpr (KIND == SE_CACHE_FP4) {
      const int64_t head_bytes = fp4_head_bytes(page_size, D), factors = fp4_factors_at(page_size, D);
#pragma unroll
      for (int kp = 0; kp < KP; ++kp) {
        int first = k_lo + 32 * kp;      // of 32 keys in one page; those no one holds take the place of some that are held
        if (first > last_key) first = last_key & ~31;
        if (first + 31 < low_key) first = low_key & ~31;
        const uint8_t* at = static_cast<const uint8_t*>(cache) +
                            (static_cast<int64_t>(table[first / page_size]) * 2 * kv_heads + kvh) * head_bytes;
        const int off = first % page_size + 2 * n;
        if constexpr (WIDE) {
#pragma unroll
          for (int h = 0; h < (DS + 3) / 4; ++h) {      // DS == 2: half a group
            const int grp = DS == 2 ? g >> 1 : g * (DS / 4) + h;
            const uint32_t f = *reinterpret_cast<const uint16_t*>(at + factors + static_cast<int64_t>(grp) * page_size + off);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const uint8_t* codes = at + fp4_key_code_at(page_size, off + b, grp) + (DS == 2 ? (g & 1) * 8 : 0);
              uint32_t w[4];
              if constexpr (DS == 2) {
                const uint2 v = *reinterpret_cast<const uint2*>(codes);
                w[0] = v.x, w[1] = v.y, w[2] = w[3] = 0;
              } else {
                const uint4 v = load16_once(codes);
                w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
              }
#pragma unroll
              for (int i = 0; i < (DS == 2 ? 2 : 4); ++i)
                kf[kp][b][4 * h + i] = fp4_eight(w[i], b == 0 ? fp4_factor_bits<0>(f) : fp4_factor_bits<1>(f));
            }
          }
        } else {
#pragma unroll
          for (int ds = 0; ds < DS; ++ds) {
            const uint32_t f = *reinterpret_cast<const uint16_t*>(at + factors + static_cast<int64_t>(ds) * page_size + off);
#pragma unroll
            for (int b = 0; b < 2; ++b)
              kf[kp][b][ds] = fp4_eight(*reinterpret_cast<const uint32_t*>(at + fp4_key_code_at(page_size, off + b, ds) + 4 * g),
                                        b == 0 ? fp4_factor_bits<0>(f) : fp4_factor_bits<1>(f));
          }
        }
      }
    } else {
#pragma unroll
      for (int kp = 0; kp < KP; ++kp)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int key = max(min(key_of(kp, b), last_key), low_key);
          const bf16_t* row = static_cast<const bf16_t*>(cache) +
                              (static_cast<int64_t>(table[key / page_size]) * 2 * kv_heads + kvh) * page_size * D +
                              (static_cast<int64_t>(g) * page_size + key % page_size) * 8;
#pragma unroll
          for (int ds = 0; ds < DS; ++ds) kf[kp][b][ds] = load16_once(row + static_cast<int64_t>(ds) * 32 * page_size);
        }
    }

    // the tiles with a row that sees one of the keys
    const int rows_total = q_len * group;
    int tile = k_lo > pos0 ? static_cast<int>(static_cast<int64_t>(k_lo - pos0) * group / 16) : 0;
    int until = (rows_total + 15) / 16;
    if (window > 0) {
      const int64_t last_q = static_cast<int64_t>(min(k_hi, last_key)) + window - 1 - pos0;
      if (last_q + 1 < q_len) until = static_cast<int>(((last_q + 1) * group + 15) / 16);
    }
    struct Rows {
      uint4 q[DS];
      float lse2;      // of the lane's row n, in powers of two; +inf: there is no such row
      int pos;
    };
    auto fetch = [&](Rows& r, int t) {
      const int rho = t * 16 + n, rho_c = min(rho, rows_total - 1);
      const int q_idx = rho_c / group, head = kvh * group + rho_c - q_idx * group;
      const bf16_t* row = q + static_cast<int64_t>(q_start + q_idx) * q_stride + static_cast<int64_t>(head) * D;
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) r.q[ds] = *reinterpret_cast<const uint4*>(row + dims_of(ds));
      const float l = lse[static_cast<int64_t>(q_start + q_idx) * heads + head];
      r.lse2 = rho < rows_total ? l * 1.4426950408889634f : INFINITY;
      r.pos = pos0 + q_idx;
    };
    auto weigh = [&](const Rows& r, int t) {
      floatx4 s[KP][2];
#pragma unroll
      for (int kp = 0; kp < KP; ++kp)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          s[kp][b] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ds = 0; ds < DS; ++ds)
            s[kp][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, r.q[ds]),
                                                               __builtin_bit_cast(bf16x8, kf[kp][b][ds]), s[kp][b], 0, 0, 0);
        }
      // lane (g, n): s[kp][b][i] is the score of row 4 g + i for key key_of(kp, b)
      float l[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) l[i] = __shfl(r.lse2, 4 * g + i, SE_WAVE);
      const int pos_min = pos0 + t * 16 / group, pos_max = pos0 + min(t * 16 + 15, rows_total - 1) / group;
      if (k_hi > pos_min || (window > 0 && k_lo <= pos_max - window)) {      // the same in all lanes
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int pos = __shfl(r.pos, 4 * g + i, SE_WAVE);
#pragma unroll
          for (int kp = 0; kp < KP; ++kp)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const int key = key_of(kp, b);
              if (key > pos || (window > 0 && key <= pos - window)) s[kp][b][i] = -INFINITY;
            }
        }
      }
#pragma unroll
      for (int kp = 0; kp < KP; ++kp)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) sum += __builtin_amdgcn_exp2f(fmaf(s[kp][b][i], scale_log2e, -l[i]));
          acc[kp][b] += sum;
        }
    };
    tile += part;
    if (tile < until) {
      Rows a, b;
      fetch(a, tile);
      for (; tile < until; tile += 2 * row_waves) {      // the next tile's rows are on their way meanwhile
        const bool second = tile + row_waves < until;
        if (second) fetch(b, tile + row_waves);
        weigh(a, tile);
        if (!second) break;
        if (tile + 2 * row_waves < until) fetch(a, tile + 2 * row_waves);
        weigh(b, tile + row_waves);
      }
    }
#pragma unroll
    for (int kp = 0; kp < KP; ++kp)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        acc[kp][b] += __shfl_xor(acc[kp][b], 16, SE_WAVE);
        acc[kp][b] += __shfl_xor(acc[kp][b], 32, SE_WAVE);
      }
  }
  if (row_waves > 1) {
    if (g == 0) {
#pragma unroll
      for (int kp = 0; kp < KP; ++kp) sums[wave][2 * kp][n] = acc[kp][0], sums[wave][2 * kp + 1][n] = acc[kp][1];
    }
    __syncthreads();
    if (part != 0 || g != 0) return;
#pragma unroll
    for (int kp = 0; kp < KP; ++kp)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        for (int w = 1; w < row_waves; ++w) acc[kp][b] += sums[wave + w][2 * kp + b][n];
  }
  if (!wanted || g != 0) return;
#pragma unroll
  for (int kp = 0; kp < KP; ++kp)
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int key = key_of(kp, b);
      if (key > last_key || key < low_key) continue;
      const int64_t at = (static_cast<int64_t>(table[key / page_size]) * kv_heads + kvh) * page_size + key % page_size;
      out[at] = (previous != nullptr && key < pos0 ? previous[at] : 0.f) + acc[kp][b];
    }
}

template <int DS, int KIND>
static void launch_weights_mfma(const void* q, int64_t q_stride, const void* cache, const int32_t* block_table, int bt_stride,
                                const int32_t* item_meta, int items, int longest, int most_rows, const float* lse,
                                const float* previous, float* out, int heads, int kv_heads, int page_size, float scale,
                                int window, hipStream_t stream) {
  constexpr int keys = 32 * WeightKeys<DS>::KP;
  // With a single tile there is nothing to share out among the wavefronts of the same keys.
  const int tiles = (most_rows + 15) / 16;
  const int row_waves = tiles <= 1 ? 1 : tiles <= 8 ? 2 : tiles <= 32 ? 4 : 8;
  const int waves = row_waves < 4 ? 4 : row_waves;
  const int per_block = keys * (waves / row_waves);
  const dim3 grid((longest + per_block - 1) / per_block, kv_heads, items);
  attention_weights_mfma_kernel<DS, KIND><<<grid, waves * SE_WAVE, 0, stream>>>(
      static_cast<const bf16_t*>(q), q_stride, cache, block_table, bt_stride, item_meta, items, longest, lse, previous, out,
      heads, kv_heads, page_size, scale * 1.4426950408889634f, window, row_waves);
}

// q [.., heads, head_dim] with token stride q_stride; cache of `kind` (SeCacheKind); item_meta int32 [3, items]:
// first token, new tokens and tokens with them of every request; longest: the largest of the latter; most_new: the
// largest of the new ones.
extern "C" int se_attention_weights(const void* q, int64_t q_stride, const void* cache, int kind,
                                    const int32_t* block_table, int bt_stride, const int32_t* item_meta, int items,
                                    int longest, int most_new, const float* lse, const float* previous, float* out, int heads,
                                    int kv_heads, int head_dim, int page_size, float scale, int window, int dtype,
                                    hipStream_t stream) {
  if (items <= 0 || longest <= 0) return SE_OK;
  if (head_dim <= 0 || head_dim % 8 || head_dim > 512) return SE_ERR_SHAPE;
  if (kv_heads <= 0 || heads % kv_heads || page_size <= 0 || page_size % 8) return SE_ERR_SHAPE;
  if (kind == SE_CACHE_FP4 && (head_dim % 32 || page_size % 32)) return SE_ERR_SHAPE;
  if (kind != SE_CACHE_FP4 && kind != (dtype == SE_F32 ? SE_CACHE_F32 : SE_CACHE_BF16)) return SE_ERR_SHAPE;
  if (kv_heads > 65535 || items > 65535) return SE_ERR_SHAPE;
  const int64_t most_rows = static_cast<int64_t>(most_new) * (heads / kv_heads);
  if (dtype == SE_BF16 && head_dim % 32 == 0 && head_dim <= 256 && most_rows < 0x40000000) {
#define SE_WEIGHTS_MFMA(DS, KIND)                                                                                   \
  launch_weights_mfma<DS, KIND>(q, q_stride, cache, block_table, bt_stride, item_meta, items, longest,              \
                                static_cast<int>(most_rows), lse, previous, out, heads, kv_heads, page_size, scale, window, stream)
#define SE_WEIGHTS_CASE(DS)                                     \
  case DS:                                                      \
    if (kind == SE_CACHE_FP4) SE_WEIGHTS_MFMA(DS, SE_CACHE_FP4); \
    else SE_WEIGHTS_MFMA(DS, SE_CACHE_BF16);                     \
    break;
    switch (head_dim / 32) {
      SE_WEIGHTS_CASE(1) SE_WEIGHTS_CASE(2) SE_WEIGHTS_CASE(3) SE_WEIGHTS_CASE(4)
      SE_WEIGHTS_CASE(5) SE_WEIGHTS_CASE(6) SE_WEIGHTS_CASE(7) SE_WEIGHTS_CASE(8)
    }
#undef SE_WEIGHTS_CASE
#undef SE_WEIGHTS_MFMA
    SE_CHECK_LAUNCH();
    return SE_OK;
  }
  const dim3 grid((longest + SE_WAVE - 1) / SE_WAVE, kv_heads, items);
  const size_t shared = static_cast<size_t>(head_dim) * sizeof(float);
#define SE_WEIGHTS(T, KIND)                                                                                      \
  attention_weights_generic_kernel<T, KIND><<<grid, 64, shared, stream>>>(                                       \
      static_cast<const T*>(q), q_stride, cache, block_table, bt_stride, item_meta, items, longest, lse, previous, out, heads, \
      kv_heads, head_dim, page_size, scale, window)
  if (dtype == SE_F32) {
    if (kind == SE_CACHE_FP4) SE_WEIGHTS(float, SE_CACHE_FP4);
    else SE_WEIGHTS(float, SE_CACHE_F32);
  } else if (dtype == SE_BF16) {
    if (kind == SE_CACHE_FP4) SE_WEIGHTS(bf16_t, SE_CACHE_FP4);
    else SE_WEIGHTS(bf16_t, SE_CACHE_BF16);
  } else {
    return SE_ERR_SHAPE;
  }
#undef SE_WEIGHTS
  SE_CHECK_LAUNCH();
  return SE_OK;
}
