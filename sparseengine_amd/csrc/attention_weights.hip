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

// q [.., heads, head_dim] with token stride q_stride; cache of `kind` (SeCacheKind); item_meta int32 [3, items]:
// first token, new tokens and tokens with them of every request; longest: the largest of the latter.
extern "C" int se_attention_weights(const void* q, int64_t q_stride, const void* cache, int kind,
                                    const int32_t* block_table, int bt_stride, const int32_t* item_meta, int items,
                                    int longest, const float* lse, const float* previous, float* out, int heads,
                                    int kv_heads, int head_dim, int page_size, float scale, int window, int dtype,
                                    hipStream_t stream) {
  if (items <= 0 || longest <= 0) return SE_OK;
  if (head_dim <= 0 || head_dim % 8 || head_dim > 512) return SE_ERR_SHAPE;
  if (kv_heads <= 0 || heads % kv_heads || page_size <= 0 || page_size % 8) return SE_ERR_SHAPE;
  if (kind == SE_CACHE_FP4 && (head_dim % 32 || page_size % 32)) return SE_ERR_SHAPE;
  if (kind != SE_CACHE_FP4 && kind != (dtype == SE_F32 ? SE_CACHE_F32 : SE_CACHE_BF16)) return SE_ERR_SHAPE;
  if (kv_heads > 65535 || items > 65535) return SE_ERR_SHAPE;
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
