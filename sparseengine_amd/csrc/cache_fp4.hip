// Into and out of the 4-bit cache (fp4.h):
//   store:   the keys and values of a step's tokens, as they stand in the q | k | v rows, to their slots (where the
//            norm and rotation kernel has not made the codes itself: no rotation and no norm, a norm per head,
//            neighbouring pairs).  8191 tokens of 8 + 8 heads of 128 take 18.7 us, 2.3 TB/s read and written, half of what a
//            copy reaches: neighbouring lanes take neighbouring tokens, so that values are written side by side, but the
//            16 bytes that the lanes of a load read lie whole rows apart.
//   unpack:  whole pages to the engine's own page layout and type (what attention on many rows, in float32 and at
//            head sizes without a kernel of its own reads).  Bound by writing: the 131 pages of 64 of such a step
//            14 us (2.5 TB/s written), the 256 pages of a context of 16384 tokens 20 us (3.4).
#include "fp4.h"

// One thread per (token, key or value, kv head, group of 32 dims).
template <typename T>
__global__ void __launch_bounds__(256)
fp4_store_kernel(const T* __restrict__ qkv, int64_t row_stride, const int32_t* __restrict__ slots, int tokens,
                 int heads, int kv_heads, int head_dim, uint8_t* __restrict__ cache, int page_size) {
  constexpr int VN = Vec16<T>::N;
  const int groups = head_dim / FP4_GROUP;
  const int per_token = 2 * kv_heads * groups;
  const int64_t index = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (index >= static_cast<int64_t>(tokens) * per_token) return;
  // neighbouring threads take neighbouring tokens: a value's bytes of eight keys lie side by side
  const int token = static_cast<int>(index % tokens), rest = static_cast<int>(index / tokens);
  const int group = rest % groups, head = rest / groups % kv_heads, which = rest / groups / kv_heads;
  const int slot = slots[token];
  if (slot < 0) return;
  const T* src = qkv + token * row_stride + (static_cast<int64_t>(heads) + which * kv_heads + head) * head_dim + group * FP4_GROUP;
  float x[FP4_GROUP];
  float amax = 0.f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < FP4_GROUP / VN; ++i) {
    Vec16<T> v;
    v.v = *reinterpret_cast<const decltype(v.v)*>(src + i * VN);
#pragma unroll
    for (int j = 0; j < VN; ++j) {
      x[i * VN + j] = v.get(j);
      amax = fmaxf(amax, fabsf(x[i * VN + j]));
      finite = finite && (__float_as_uint(x[i * VN + j]) & 0x7f800000u) != 0x7f800000u;
    }
  }
  const int factor = finite ? fp4_factor_of(amax) : FP4_NAN;
  const float inverse = finite ? fp4_inverse(factor) : 0.f;
  const int off = slot % page_size;
  uint8_t* part = cache + ((static_cast<int64_t>(slot / page_size) * 2 + which) * kv_heads + head) * fp4_head_bytes(page_size, head_dim);
  uint32_t words[4] = {0, 0, 0, 0};
#pragma unroll
  for (int d = 0; d < FP4_GROUP; ++d) words[d / 8] |= fp4_code(x[d] * inverse) << (d % 8 * 4);
  if (which == 0) {
    *reinterpret_cast<uint4*>(part + fp4_key_code_at(page_size, off, group)) = uint4{words[0], words[1], words[2], words[3]};
    part[fp4_key_factor_at(page_size, head_dim, off, group)] = static_cast<uint8_t>(factor);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) part[fp4_value_code_at(head_dim, off, group, j)] = static_cast<uint8_t>(words[j / 4] >> (j % 4 * 8));
    part[fp4_value_factor_at(page_size, head_dim, off, group)] = static_cast<uint8_t>(factor);
  }
}

// eight values to eight neighbouring storage elements
template <typename T>
__device__ __forceinline__ void put8(T* dst, const float (&x)[8]) {
  constexpr int VN = Vec16<T>::N;
#pragma unroll
  for (int i = 0; i < 8 / VN; ++i) {
    Vec16<T> v;
#pragma unroll
    for (int j = 0; j < VN; ++j) v.set(j, x[i * VN + j]);
    *reinterpret_cast<decltype(v.v)*>(dst + i * VN) = v.v;
  }
}

// A page of the 4-bit cache to page blockIdx.x of `out` [.., 2, kv_heads, page_size * head_dim] in the order of the
// engine's own cache (key_place, value_place).  Which page: pages[blockIdx.x], or, with a list of (row, column)
// pairs, the block table's entry there; a negative page is left out.  A thread makes eight elements of a key, or
// the eight keys of a group for two neighbouring dims of the values.
// FOR_PRODUCTS: for kernels that multiply the probabilities of many rows with a token's values, those of rows that do not
// see it (0) among them.  A group of values that is not a number is then written as zeros and its token's key as not a number:
// rows that see the token become so as a whole, the others take nothing from it.
template <typename T, bool FOR_PRODUCTS>
__global__ void __launch_bounds__(256)
fp4_unpack_kernel(const uint8_t* __restrict__ cache, const int32_t* __restrict__ pages, int bt_stride,
                  const int2* __restrict__ list, T* __restrict__ out, int kv_heads, int page_size, int head_dim) {
  const int page = list == nullptr ? pages[blockIdx.x]
                                   : pages[static_cast<int64_t>(list[blockIdx.x].x) * bt_stride + list[blockIdx.x].y];
  if (page < 0) return;
  const int which = blockIdx.y / kv_heads, head = blockIdx.y % kv_heads;
  const int64_t part_index = static_cast<int64_t>(which) * kv_heads + head;
  const uint8_t* part = cache + (static_cast<int64_t>(page) * 2 * kv_heads + part_index) * fp4_head_bytes(page_size, head_dim);
  T* dst = out + (static_cast<int64_t>(blockIdx.x) * 2 * kv_heads + part_index) * page_size * head_dim;
  const int groups = head_dim / FP4_GROUP;
  if (which == 0) {
    const int pieces = page_size * head_dim / 8;
    for (int i = threadIdx.x; i < pieces; i += blockDim.x) {
      const int d8 = i / page_size, off = i % page_size;      // dims 8 d8 ..: a quarter of group d8 / 4
      const uint32_t word = *reinterpret_cast<const uint32_t*>(part + fp4_key_code_at(page_size, off, d8 >> 2) + (d8 & 3) * 4);
      const int factor = part[fp4_key_factor_at(page_size, head_dim, off, d8 >> 2)];
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = fp4_value(word >> (4 * j) & 15u, factor);
      if (FOR_PRODUCTS && d8 == 0) {
        const uint8_t* values = part + kv_heads * fp4_head_bytes(page_size, head_dim);
        for (int group = 0; group < groups; ++group)
          if (values[fp4_value_factor_at(page_size, head_dim, off, group)] == FP4_NAN) x[0] = __uint_as_float(0x7fc00000u);
      }
      put8(dst + static_cast<int64_t>(i) * 8, x);             // [head_dim / 8][page_size][8]
    }
  } else {
    const int pairs = page_size / 8 * (head_dim / 2);
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
      const int kg = i / (head_dim / 2), pair = i % (head_dim / 2);     // keys 8 kg .., dims 2 pair, 2 pair + 1
      const int group = pair / 16, j16 = pair % 16;
      const uint2 codes = *reinterpret_cast<const uint2*>(part + fp4_value_code_at(head_dim, kg * 8, group, j16));
      const uint2 factors = *reinterpret_cast<const uint2*>(part + fp4_value_factor_at(page_size, head_dim, kg * 8, group));
      float even[8], odd[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t two = (k < 4 ? codes.x : codes.y) >> (k % 4 * 8);
        const int factor = static_cast<int>((k < 4 ? factors.x : factors.y) >> (k % 4 * 8) & 255u);
        const bool nothing = FOR_PRODUCTS && factor == FP4_NAN;
        even[k] = nothing ? 0.f : fp4_value(two & 15u, factor);
        odd[k] = nothing ? 0.f : fp4_value(two >> 4 & 15u, factor);
      }
      T* at = dst + (static_cast<int64_t>(kg) * head_dim + 2 * pair) * 8;   // [page_size / 8][head_dim][8]
      put8(at, even);
      put8(at + 8, odd);
    }
  }
}

static bool fp4_sizes_taken(int kv_heads, int head_dim, int page_size) {
  return kv_heads > 0 && head_dim > 0 && head_dim % 32 == 0 && head_dim <= 512 && page_size > 0 && page_size % 32 == 0;
}

extern "C" int se_fp4_store(const void* qkv, int64_t row_stride, const int32_t* slots, int tokens, int heads,
                            int kv_heads, int head_dim, void* cache, int page_size, int dtype, hipStream_t stream) {
  if (tokens <= 0) return SE_OK;
  if (!fp4_sizes_taken(kv_heads, head_dim, page_size) || row_stride % 8) return SE_ERR_SHAPE;
  const int64_t threads = static_cast<int64_t>(tokens) * 2 * kv_heads * (head_dim / FP4_GROUP);
  const int64_t blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffff) return SE_ERR_SHAPE;
  if (dtype == SE_F32)
    fp4_store_kernel<float><<<dim3(static_cast<unsigned>(blocks)), 256, 0, stream>>>(
        static_cast<const float*>(qkv), row_stride, slots, tokens, heads, kv_heads, head_dim, static_cast<uint8_t*>(cache), page_size);
  else if (dtype == SE_BF16)
    fp4_store_kernel<bf16_t><<<dim3(static_cast<unsigned>(blocks)), 256, 0, stream>>>(
        static_cast<const bf16_t*>(qkv), row_stride, slots, tokens, heads, kv_heads, head_dim, static_cast<uint8_t*>(cache), page_size);
  else
    return SE_ERR_SHAPE;
  SE_CHECK_LAUNCH();
  return SE_OK;
}

// pages: [count]; or, with `list` (int32 [count, 2]: row, column), a block table with rows of `bt_stride` entries.
extern "C" int se_fp4_unpack(const void* cache, const int32_t* pages, int bt_stride, const int32_t* list, int count,
                             void* out, int kv_heads, int page_size, int head_dim, int dtype, int for_products, hipStream_t stream) {
  if (count <= 0) return SE_OK;
  if (!fp4_sizes_taken(kv_heads, head_dim, page_size) || 2 * kv_heads > 65535) return SE_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(count), static_cast<unsigned>(2 * kv_heads));
#define SE_UNPACK(T, FOR_PRODUCTS)                                                                                      \
  fp4_unpack_kernel<T, FOR_PRODUCTS><<<grid, 256, 0, stream>>>(static_cast<const uint8_t*>(cache), pages, bt_stride,     \
                                                               reinterpret_cast<const int2*>(list), static_cast<T*>(out), \
                                                               kv_heads, page_size, head_dim)
  if (dtype == SE_F32 && !for_products) SE_UNPACK(float, false);
  else if (dtype == SE_BF16 && for_products) SE_UNPACK(bf16_t, true);
  else if (dtype == SE_BF16) SE_UNPACK(bf16_t, false);
  else
    return SE_ERR_SHAPE;
#undef SE_UNPACK
  SE_CHECK_LAUNCH();
  return SE_OK;
}
