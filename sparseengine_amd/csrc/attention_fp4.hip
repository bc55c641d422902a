// Paged causal GQA attention over keys and values in 4 bits (fp4.h) for few rows (decoding), on the matrix cores
// of gfx950.  Units, rows, tiles, partial results and their merge are those of the bfloat16 kernel with one
// wavefront per unit (attention_mfma.hip): a unit is one tile of 16 rows (a row is one query token and one
// head) of one request and kv head, and one range of keys, a multiple of 32 of them but for the last.
//
//   S^T = K Q^T      A = 16 keys x 32 dims, B = 32 dims x 16 rows.  A lane's part of a key are head_dim / 4
//                    neighbouring dims, one contiguous piece of codes under one factor (head size 128: exactly
//                    one group), so the dims of a product step are eight of each of the four lanes' parts; q is
//                    read in the same order.  A-row m of block b is key k0 + 2 m + b: a lane's two keys are
//                    neighbours in memory, and it ends up with the scores of eight consecutive keys of its row.
//   O^T += V^T P^T   A = 16 value dims x 32 keys.  A byte of a value holds two neighbouring dims of one key;
//                    a lane turns the bytes of its eight keys into eight pairs, each under its own key's
//                    factor, and parts them into the operand of the even dims and that of the odd ones.
//
// Every value is exact in bfloat16 after one conversion instruction per pair, so the arithmetic is that of the
// bfloat16 kernel: scores and sums in float, softmax in base 2, probabilities rounded to bfloat16 for the value
// product, the running sum of them unrounded.
//
// head_dim 64, 128 or 256, page_size % 32 == 0 (a step of 32 keys lies in one page).
#include "fp4.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

#define UNIT_FIELDS 8  // item, row_tile, key_begin, key_end, partial_slot (-1: writes out), q_start, q_len, ctx_len

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));

// Maximum / sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48 that share a row.
__device__ __forceinline__ float quad_max(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const uint32_t w = __float_as_uint(v);
  const auto b = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quad_sum(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const uint32_t w = __float_as_uint(v);
  const auto b = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// What a lane holds of a step of 32 keys: head_dim = 32 * DS.
template <int DS>
struct Fp4Step {
  uint32_t k[2][DS];            // codes of its dims of its two keys
  uint32_t kf[(DS + 3) / 4];    // factor bytes of the two keys (low, next), per group of its dims
  uint32_t v[DS][2];            // per 32 dims: the bytes of its pair of dims for its eight keys
  uint32_t vf[DS][2];           // per 32 dims: the factor bytes of its eight keys
};

// Keys and values of the step whose first key is at `off` of the page part pair (keys, values).
template <int DS>
__device__ __forceinline__ void load_step(Fp4Step<DS>& s, const uint8_t* keys, const uint8_t* values, int page_size,
                                          int off, int n, int g) {
  constexpr int D = 32 * DS;
  const int64_t factors = fp4_factors_at(page_size, D);
  const int key = off + 2 * n;
  if constexpr (DS == 2) {
    const uint8_t* at = keys + fp4_key_code_at(page_size, key, g >> 1) + (g & 1) * 8;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint2 w = *reinterpret_cast<const uint2*>(at + 16 * b);
      s.k[b][0] = w.x;
      s.k[b][1] = w.y;
    }
    s.kf[0] = *reinterpret_cast<const uint16_t*>(keys + factors + static_cast<int64_t>(g >> 1) * page_size + key);
  } else {
#pragma unroll
    for (int h = 0; h < DS / 4; ++h) {
      const int group = g * (DS / 4) + h;
      const uint8_t* at = keys + fp4_key_code_at(page_size, key, group);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint4 w = load16_once(at + 16 * b);
        s.k[b][4 * h] = w.x;
        s.k[b][4 * h + 1] = w.y;
        s.k[b][4 * h + 2] = w.z;
        s.k[b][4 * h + 3] = w.w;
      }
      s.kf[h] = *reinterpret_cast<const uint16_t*>(keys + factors + static_cast<int64_t>(group) * page_size + key);
    }
  }
  const int64_t eight = (off >> 3) + g;      // the lane's eight keys
  const uint8_t* code_at = values + (eight * 16 + n) * (DS * 8);
  const uint8_t* factor_at = values + factors + eight * (DS * 8);
#pragma unroll
  for (int h = 0; h < DS / 2; ++h) {
    const uint4 w = load16_once(code_at + 16 * h);
    s.v[2 * h][0] = w.x;
    s.v[2 * h][1] = w.y;
    s.v[2 * h + 1][0] = w.z;
    s.v[2 * h + 1][1] = w.w;
    const uint4 f = *reinterpret_cast<const uint4*>(factor_at + 16 * h);
    s.vf[2 * h][0] = f.x;
    s.vf[2 * h][1] = f.y;
    s.vf[2 * h + 1][0] = f.z;
    s.vf[2 * h + 1][1] = f.w;
  }
}

// The bytes of eight keys (a pair of dims each), each under its own factor: the operand of the even dim, that of
// the odd one.
__device__ __forceinline__ void operands_of(const uint32_t (&codes)[2], const uint32_t (&factors)[2], bf16x8& even, bf16x8& odd) {
  uint32_t p[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    p[4 * h] = SE_FP4_PAIR(codes[h], fp4_factor_bits<0>(factors[h]), 0);
    p[4 * h + 1] = SE_FP4_PAIR(codes[h], fp4_factor_bits<1>(factors[h]), 1);
    p[4 * h + 2] = SE_FP4_PAIR(codes[h], fp4_factor_bits<2>(factors[h]), 2);
    p[4 * h + 3] = SE_FP4_PAIR(codes[h], fp4_factor_bits<3>(factors[h]), 3);
  }
  uint4 e, o;
  e.x = __builtin_amdgcn_perm(p[1], p[0], 0x05040100);
  e.y = __builtin_amdgcn_perm(p[3], p[2], 0x05040100);
  e.z = __builtin_amdgcn_perm(p[5], p[4], 0x05040100);
  e.w = __builtin_amdgcn_perm(p[7], p[6], 0x05040100);
  o.x = __builtin_amdgcn_perm(p[1], p[0], 0x07060302);
  o.y = __builtin_amdgcn_perm(p[3], p[2], 0x07060302);
  o.z = __builtin_amdgcn_perm(p[5], p[4], 0x07060302);
  o.w = __builtin_amdgcn_perm(p[7], p[6], 0x07060302);
  even = __builtin_bit_cast(bf16x8, e);
  odd = __builtin_bit_cast(bf16x8, o);
}

// 0x80 in every byte of `word` that is 255, 0 in the others.
__device__ __forceinline__ uint32_t marks_255(uint32_t word) {
  const uint32_t t = ~word;      // bytes that are 0
  return ~(((t & 0x7f7f7f7fu) + 0x7f7f7f7fu) | t | 0x7f7f7f7fu);
}
__device__ __forceinline__ uint32_t mark_bits(uint32_t marks) {      // bit i: byte i is marked
  return (marks >> 7 & 1u) | (marks >> 14 & 2u) | (marks >> 21 & 4u) | (marks >> 28 & 8u);
}

// The reference maximum of a row is only raised when a step exceeds it by more than this (in powers of two):
// probabilities may then reach 2^SLACK, which float sums and bfloat16 operands hold as well as values below 1,
// and the rescaling of the accumulators becomes rare.
#define SOFTMAX_SLACK 8.f

template <int DS, int NS>   // head_dim = 32 * DS; NS steps of keys in registers at a time
__global__ void __launch_bounds__(256)
paged_attention_fp4_kernel(const bf16_t* __restrict__ q, int64_t q_stride, const uint8_t* __restrict__ cache,
                           const int32_t* __restrict__ block_table, int bt_stride,
                           const int32_t* __restrict__ units, int num_units, bf16_t* __restrict__ out,
                           int64_t out_stride, float* __restrict__ part_o, float* __restrict__ part_ml,
                           float* __restrict__ lse, int heads, int kv_heads, int page_size, float scale_log2e,
                           int window) {
  constexpr int D = 32 * DS;
  const int lane = threadIdx.x & (SE_WAVE - 1);
  const int unit = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x * (blockDim.x / SE_WAVE) + threadIdx.x / SE_WAVE));
  if (unit >= num_units) return;  // whole waves leave together; there is no block barrier below
  const int n = lane & 15;        // row of the tile (B operand column) / A operand row
  const int g = lane >> 4;
  const int kvh = blockIdx.y;
  const int group = heads / kv_heads;

  const int32_t* u = units + static_cast<int64_t>(unit) * UNIT_FIELDS;
  const int item = u[0], row_tile = u[1], key_begin = u[2], slot = u[4];
  int key_end = u[3];
  const int q_start = u[5], q_len = u[6], ctx_len = u[7];
  const int rows_total = q_len * group;

  const int rho = row_tile * 16 + n;
  const bool row_valid = rho < rows_total;
  const int rho_c = row_valid ? rho : rows_total - 1;   // padding rows repeat the last row
  const int q_idx = rho_c / group;
  const int head = kvh * group + rho_c % group;
  const int token = q_start + q_idx;
  const int pos = ctx_len - q_len + q_idx;

  // this tile's largest and smallest position bound the keys that matter
  const int last_row = (row_tile * 16 + 15 < rows_total) ? row_tile * 16 + 15 : rows_total - 1;
  const int pos_max = ctx_len - q_len + last_row / group;
  const int pos_min = ctx_len - q_len + (row_tile * 16) / group;
  if (key_end > pos_max + 1) key_end = pos_max + 1;
  // With a window the request may have given back the pages before the tile's lowest key; the steps begin with
  // the one that holds that key, and a step lies in one page.
  int k_first = key_begin;
  if (window > 0) {
    const int lowest = pos_min - window + 1;
    if (lowest > k_first) k_first = lowest & ~31;
  }

  uint4 qf[DS];
  const bf16_t* q_row = q + static_cast<int64_t>(token) * q_stride + static_cast<int64_t>(head) * D + g * (D / 4);
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) qf[ds] = *reinterpret_cast<const uint4*>(q_row + ds * 8);

  const int32_t* table = block_table + static_cast<int64_t>(item) * bt_stride;
  const int64_t head_bytes = fp4_head_bytes(page_size, D);
  const int64_t plane = kv_heads * head_bytes;
  const uint8_t* cache_head = cache + kvh * head_bytes;

  floatx4 o[DS][2];      // [32 dims][even, odd]
#pragma unroll
  for (int b = 0; b < DS; ++b) o[b][0] = o[b][1] = floatx4{0.f, 0.f, 0.f, 0.f};
  float run_max = -INFINITY, run_sum = 0.f;    // run_sum: this lane's share, added up at the end

  if (k_first < key_end) {
    const int k_last = k_first + (key_end - 1 - k_first) / 32 * 32;    // first key of the last step
    Fp4Step<DS> ring[NS];
    auto fetch = [&](Fp4Step<DS>& s, int k0) {     // beyond the end: the last step once more
      const int k = k0 < k_last ? k0 : k_last;
      const uint8_t* page = cache_head + static_cast<int64_t>(table[k / page_size]) * 2 * plane;
      load_step<DS>(s, page, page + plane, page_size, k % page_size, n, g);
    };
    auto compute = [&](const Fp4Step<DS>& s, int k0) {
      floatx4 sc[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        sc[b] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) {
          const uint32_t f = b == 0 ? fp4_factor_bits<0>(s.kf[ds / 4]) : fp4_factor_bits<1>(s.kf[ds / 4]);
          sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fp4_eight(s.k[b][ds], f)),
                                                          __builtin_bit_cast(bf16x8, qf[ds]), sc[b], 0, 0, 0);
        }
      }
      // lane (g, n): sc[b][i] is the score of key k0 + 8 g + 2 i + b for row n
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = sc[j & 1][j >> 1];
      // the same in all lanes: does any row of the tile not see some key of this step?
      const bool masked = k0 + 31 > pos_min || (window > 0 && k0 <= pos_max - window);
      uint32_t vf[DS][2];
#pragma unroll
      for (int b = 0; b < DS; ++b) vf[b][0] = s.vf[b][0], vf[b][1] = s.vf[b][1];
      uint32_t not_numbers = 0;
      if (masked) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = k0 + 8 * g + j;
          if (key > pos || (window > 0 && key <= pos - window)) p[j] = -INFINITY;
        }
        // Slots past the request's last key hold whatever an earlier owner left: their factors become 0, which
        // is finite.  A row that does not see a key must not take a value that is not a number from it either.
        const int keep = ctx_len - (k0 + 8 * g);      // of the lane's eight keys
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k4 = keep - 4 * h;
          const uint32_t m = k4 >= 4 ? 0xffffffffu : k4 <= 0 ? 0u : (1u << (8 * k4)) - 1u;
#pragma unroll
          for (int b = 0; b < DS; ++b) {
            vf[b][h] &= m;
            not_numbers |= marks_255(vf[b][h]);
          }
        }
      }
      float m = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
      m *= scale_log2e;      // scale > 0: the maximum commutes with it
      if (__builtin_amdgcn_ballot_w64(!(m <= run_max + SOFTMAX_SLACK)) != 0) {
        const float top = quad_max(m);
        if (top > run_max) {
          const float alpha = __builtin_amdgcn_exp2f(run_max - top);     // 0 where there was none
          run_max = top;
          run_sum *= alpha;
#pragma unroll
          for (int b = 0; b < DS; ++b) o[b][0] *= alpha, o[b][1] *= alpha;
        }
      }
      const float ref = run_max == -INFINITY ? 0.f : run_max;      // a row with no key yet: its weights are 0
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f(fmaf(p[j], scale_log2e, -ref));
        sum += p[j];
      }
      run_sum += sum;
      uint4 pf;
      pf.x = floats_to_bf16x2_bits(p[0], p[1]);
      pf.y = floats_to_bf16x2_bits(p[2], p[3]);
      pf.z = floats_to_bf16x2_bits(p[4], p[5]);
      pf.w = floats_to_bf16x2_bits(p[6], p[7]);
      if (__builtin_amdgcn_ballot_w64(not_numbers != 0) != 0) {
        // Rare: a step that some row sees only in part holds values that are not numbers.  They take part as
        // zeros, and the rows that do see their keys are made NaN.
        const int first = window > 0 && pos - window + 1 > k0 ? pos - window + 1 - k0 : 0;   // the row's keys of the step
        const int until = pos + 1 - k0 < 32 ? pos + 1 - k0 : 32;
        const uint32_t seen = until > first ? (0xffffffffu >> (32 - (until - first))) << first : 0u;
#pragma unroll
        for (int b = 0; b < DS; ++b) {
          const uint32_t low = marks_255(vf[b][0]), high = marks_255(vf[b][1]);
          const uint32_t mine = mark_bits(low) | mark_bits(high) << 4;
          uint32_t all = 0;
#pragma unroll
          for (int gg = 0; gg < 4; ++gg) all |= static_cast<uint32_t>(__shfl(static_cast<int>(mine), gg * 16 + n, SE_WAVE)) << (8 * gg);
          const float poison = (all & seen) ? NAN : 0.f;
          o[b][0] += poison;
          o[b][1] += poison;
          vf[b][0] &= ~((low >> 7) * 255u);
          vf[b][1] &= ~((high >> 7) * 255u);
        }
      }
#pragma unroll
      for (int b = 0; b < DS; ++b) {
        bf16x8 even, odd;
        operands_of(s.v[b], vf[b], even, odd);
        o[b][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, __builtin_bit_cast(bf16x8, pf), o[b][0], 0, 0, 0);
        o[b][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, __builtin_bit_cast(bf16x8, pf), o[b][1], 0, 0, 0);
      }
    };
#pragma unroll
    for (int i = 0; i < NS; ++i) fetch(ring[i], k_first + 32 * i);
    for (int k0 = k_first; k0 < key_end; k0 += 32 * NS) {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        if (k0 + 32 * i >= key_end) break;
        compute(ring[i], k0 + 32 * i);
        fetch(ring[i], k0 + 32 * (i + NS));
      }
    }
  }

  // lane (g, n): o[b][e][i] is value dim 32 b + 8 g + 2 i + e of row n
  const float total = quad_sum(run_sum);
  if (slot < 0) {
    if (!row_valid) return;
    const float inv = 1.f / total;
    bf16_t* o_row = out + static_cast<int64_t>(token) * out_stride + static_cast<int64_t>(head) * D + 8 * g;
#pragma unroll
    for (int b = 0; b < DS; ++b) {
      uint4 packed;
      packed.x = floats_to_bf16x2_bits(o[b][0][0] * inv, o[b][1][0] * inv);
      packed.y = floats_to_bf16x2_bits(o[b][0][1] * inv, o[b][1][1] * inv);
      packed.z = floats_to_bf16x2_bits(o[b][0][2] * inv, o[b][1][2] * inv);
      packed.w = floats_to_bf16x2_bits(o[b][0][3] * inv, o[b][1][3] * inv);
      *reinterpret_cast<uint4*>(o_row + b * 32) = packed;
    }
    if (lse != nullptr && g == 0)
      lse[static_cast<int64_t>(token) * heads + head] = (run_max + __log2f(total)) * 0.6931471805599453f;
  } else {
    const int64_t base = (static_cast<int64_t>(slot) * kv_heads + kvh) * 16 + n;
    float* po = part_o + base * D + 8 * g;
#pragma unroll
    for (int b = 0; b < DS; ++b) {
      *reinterpret_cast<float4*>(po + b * 32) = float4{o[b][0][0], o[b][1][0], o[b][0][1], o[b][1][1]};
      *reinterpret_cast<float4*>(po + b * 32 + 4) = float4{o[b][0][2], o[b][1][2], o[b][0][3], o[b][1][3]};
    }
    if (g == 0) {
      part_ml[base * 2] = run_max;
      part_ml[base * 2 + 1] = total;
    }
  }
}

// Units as se_paged_attention_mfma takes them; the merges of split tiles are that entry point's (with no units).
extern "C" int se_paged_attention_fp4(const void* q, int64_t q_stride, const void* cache, const int32_t* block_table,
                                      int bt_stride, const int32_t* units, int num_units, void* out, int64_t out_stride,
                                      float* part_o, float* part_ml, float* lse, int heads, int kv_heads, int head_dim,
                                      int page_size, float scale, int window, hipStream_t stream) {
  if (num_units <= 0) return SE_OK;
  if (kv_heads <= 0 || heads % kv_heads || page_size <= 0 || page_size % 32 || kv_heads > 65535) return SE_ERR_SHAPE;
  if (q_stride % 8 || out_stride % 8 || !(scale > 0.f)) return SE_ERR_SHAPE;
  const float scale_log2e = scale * 1.4426950408889634f;
  const dim3 grid((num_units + 3) / 4, kv_heads);
#define SE_FP4_ATT(DS, NS)                                                                                         \
  case 32 * DS:                                                                                                    \
    paged_attention_fp4_kernel<DS, NS><<<grid, 256, 0, stream>>>(                                                  \
        static_cast<const bf16_t*>(q), q_stride, static_cast<const uint8_t*>(cache), block_table, bt_stride, units, \
        num_units, static_cast<bf16_t*>(out), out_stride, part_o, part_ml, lse, heads, kv_heads, page_size, scale_log2e, window); \
    break;
  switch (head_dim) {
    SE_FP4_ATT(2, 4) SE_FP4_ATT(4, 4) SE_FP4_ATT(8, 2)
    default: return SE_ERR_SHAPE;
  }
#undef SE_FP4_ATT
  SE_CHECK_LAUNCH();
  return SE_OK;
}
