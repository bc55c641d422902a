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
// Every value is exact in bfloat16 after one conversion instruction per pair.  Scores and sums are float, the softmax is
// in base 2; a probability goes into the value product as two bfloat16, the second what the rounding of the first left
// (2^-16 of it is lost), beside an unrounded running sum.  The result is then as near to 64 bits as one computed in float
// and rounded once (a relative error of 0.00167 in the 2-norm, which is that rounding); with one bfloat16, as over the
// engine's own cache, it is 0.00235.  The second product costs 75 instead of 70 us for 4 requests of up to 131071 keys, 48
// instead of 45 for 16 of 16384, 296 instead of 289 for 64 of 30000, 46 instead of 43 for 16 tokens of one on 32768 keys, and
// nothing measurable for 8 of 2100 and at head size 256.
//
// Bound by reading the cache where there are keys enough, and by the latency of a wavefront's first loads else.  48:8
// heads of 128: 4 requests of up to 131071 keys 71 us (5.8 TB/s) and 4.5 us for the merge of their ranges; 8 of up to
// 2100 keys 8.8 + 2.8 us; one of 77 keys 6 us.
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

// What a lane holds of a step of 32 keys: head_dim = 32 * DS.  The values' codes of eight keys are 16 * DS / 2 pieces
// of 16 bytes (the byte of a pair of dims for the eight keys, of two neighbouring groups), read so that the
// sixteen lanes of a load take sixteen pieces side by side: piece 16 h + n of load h.  With P = DS / 2 pieces to a pair
// number j that is j = 16 / P * h + n / P and the groups 2 (n % P) and 2 (n % P) + 1, so that a lane meets two groups
// only and needs the factors of those.
template <int DS>
struct Fp4Step {
  uint32_t k[2][DS];            // codes of its dims of its two keys
  uint32_t kf[(DS + 3) / 4];    // factor bytes of the two keys (low, next), per group of its dims
  uint32_t v[DS / 2][2][2];     // [h][which of the two groups]: the bytes of its pair of dims for its eight keys
  uint32_t vf[2][2];            // [which of the two groups]: the factor bytes of its eight keys
};

// Where a lane's pieces lie from the first key of a step on (keys: of the keys' part of the page; values: of theirs).
template <int DS>
struct Fp4Places {
  uint32_t k, kf, v, vf;
  __device__ __forceinline__ Fp4Places(int page_size, int n, int g) {
    constexpr int D = 32 * DS, P = DS / 2;
    const uint32_t factors = static_cast<uint32_t>(fp4_factors_at(page_size, D));
    const int group = DS == 2 ? g >> 1 : g * (DS / 4);
    k = static_cast<uint32_t>(fp4_key_code_at(page_size, 2 * n, group)) + (DS == 2 ? (g & 1) * 8 : 0);
    kf = factors + static_cast<uint32_t>(group * page_size + 2 * n);
    v = static_cast<uint32_t>(g * 16 * DS * 8 + n * 16);
    vf = factors + static_cast<uint32_t>(g * DS * 8 + n % P * 16);
  }
};

// The step whose first key is at `off` of the page whose keys and values (of the kv head) begin at `keys` and `values`:
// the same in all lanes, so that what depends on them stays in scalar registers.
template <int DS>
__device__ __forceinline__ void load_step(Fp4Step<DS>& s, const uint8_t* keys, const uint8_t* values, int page_size,
                                          int off, const Fp4Places<DS>& at) {
  const uint8_t* codes = keys + static_cast<uint32_t>(off * 16);
  const uint8_t* factors = keys + static_cast<uint32_t>(off);
  if constexpr (DS == 2) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint2 w = *reinterpret_cast<const uint2*>(codes + at.k + 16 * b);
      s.k[b][0] = w.x;
      s.k[b][1] = w.y;
    }
    s.kf[0] = *reinterpret_cast<const uint16_t*>(factors + at.kf);
  } else {
#pragma unroll
    for (int h = 0; h < DS / 4; ++h) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint4 w = load16_once(codes + static_cast<uint32_t>(h * page_size * 16) + at.k + 16 * b);
        s.k[b][4 * h] = w.x;
        s.k[b][4 * h + 1] = w.y;
        s.k[b][4 * h + 2] = w.z;
        s.k[b][4 * h + 3] = w.w;
      }
      s.kf[h] = *reinterpret_cast<const uint16_t*>(factors + static_cast<uint32_t>(h * page_size) + at.kf);
    }
  }
  const uint8_t* pairs = values + static_cast<uint32_t>(off * DS * 16);
#pragma unroll
  for (int h = 0; h < DS / 2; ++h) {
    const uint4 w = load16_once(pairs + at.v + 256 * h);
    s.v[h][0][0] = w.x;
    s.v[h][0][1] = w.y;
    s.v[h][1][0] = w.z;
    s.v[h][1][1] = w.w;
  }
  const uint4 f = *reinterpret_cast<const uint4*>(values + static_cast<uint32_t>(off * DS) + at.vf);
  s.vf[0][0] = f.x;
  s.vf[0][1] = f.y;
  s.vf[1][0] = f.z;
  s.vf[1][1] = f.w;
}

// The factor bytes of eight keys, each as a float's exponent field.
__device__ __forceinline__ void eight_factors(const uint32_t (&bytes)[2], uint32_t (&bits)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    bits[4 * h] = fp4_factor_bits<0>(bytes[h]);
    bits[4 * h + 1] = fp4_factor_bits<1>(bytes[h]);
    bits[4 * h + 2] = fp4_factor_bits<2>(bytes[h]);
    bits[4 * h + 3] = fp4_factor_bits<3>(bytes[h]);
  }
}

// The bytes of eight keys (a pair of dims each), each under its own factor: the operand of the even dim, that of
// the odd one.
__device__ __forceinline__ void operands_of(const uint32_t (&codes)[2], const uint32_t (&factors)[8], bf16x8& even, bf16x8& odd) {
  uint32_t p[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    p[4 * h] = SE_FP4_PAIR(codes[h], factors[4 * h], 0);
    p[4 * h + 1] = SE_FP4_PAIR(codes[h], factors[4 * h + 1], 1);
    p[4 * h + 2] = SE_FP4_PAIR(codes[h], factors[4 * h + 2], 2);
    p[4 * h + 3] = SE_FP4_PAIR(codes[h], factors[4 * h + 3], 3);
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

// What rounding two floats to bfloat16 (`two`) has left of them, rounded to bfloat16.
__device__ __forceinline__ uint32_t rest_of_bf16x2(float lo, float hi, uint32_t two) {
  return floats_to_bf16x2_bits(lo - __uint_as_float(two << 16), hi - __uint_as_float(two & 0xffff0000u));
}

// The reference maximum of a row is only raised when a step exceeds it by more than this (in powers of two):
// probabilities may then reach 2^SLACK, which float sums and bfloat16 operands hold as well as values below 1,
// and the rescaling of the accumulators becomes rare.
#define SOFTMAX_SLACK 8.f

template <int DS, int NS>   // head_dim = 32 * DS; NS steps of keys in registers at a time
__global__ void __launch_bounds__(256, DS == 8 ? 1 : 2)    // head size 256 does not fit half the registers
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

  constexpr int P = DS / 2;
  floatx4 o[P][2][2];      // [load of codes][which of the lane's two groups][even, odd dim]
#pragma unroll
  for (int h = 0; h < P; ++h)
#pragma unroll
    for (int w = 0; w < 2; ++w) o[h][w][0] = o[h][w][1] = floatx4{0.f, 0.f, 0.f, 0.f};
  float run_max = -INFINITY, run_sum = 0.f;    // run_sum: this lane's share, added up at the end

  if (k_first < key_end) {
    const int k_last = k_first + (key_end - 1 - k_first) / 32 * 32;    // first key of the last step
    const Fp4Places<DS> places(page_size, n, g);
    Fp4Step<DS> ring[NS];
    // The page of a step is looked up one fetch ahead: a look-up and the loads behind it are two memory latencies
    // in a row otherwise, in every step.
    int next_page = table[k_first / page_size];
    auto fetch = [&](Fp4Step<DS>& s, int k0) {     // steps in order; beyond the end the last one once more
      const int k = k0 < k_last ? k0 : k_last, after = k0 + 32 < k_last ? k0 + 32 : k_last;
      const uint8_t* page = cache_head + static_cast<int64_t>(next_page) * 2 * plane;
      next_page = table[after / page_size];
      load_step<DS>(s, page, page + plane, page_size, k % page_size, places);
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
      // The values' operands are made here, where the vector unit would otherwise wait for the scores.
      bf16x8 even[P][2], odd[P][2];
      auto make_values = [&](const uint32_t (&vf)[2][2]) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint32_t bits[8];
          eight_factors(vf[w], bits);
#pragma unroll
          for (int h = 0; h < P; ++h) operands_of(s.v[h][w], bits, even[h][w], odd[h][w]);
        }
      };
      make_values(s.vf);
      // lane (g, n): sc[b][i] is the score of key k0 + 8 g + 2 i + b for row n
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = sc[j & 1][j >> 1];
      // the same in all lanes: does any row of the tile not see some key of this step?
      if (__builtin_expect(k0 + 31 > pos_min || (window > 0 && k0 <= pos_max - window), 0)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = k0 + 8 * g + j;
          if (key > pos || (window > 0 && key <= pos - window)) p[j] = -INFINITY;
        }
        // Slots past the request's last key hold whatever an earlier owner left: their factors become 0, which
        // is finite.  A row that does not see a key must not take a value that is not a number from it either: such
        // values take part as zeros here, and the rows that do see their keys are made NaN.
        const int keep = ctx_len - (k0 + 8 * g);      // of the lane's eight keys
        const int first = window > 0 && pos - window + 1 > k0 ? pos - window + 1 - k0 : 0;   // the row's keys of the step
        const int until = pos + 1 - k0 < 32 ? pos + 1 - k0 : 32;
        const uint32_t seen = until > first ? (0xffffffffu >> (32 - (until - first))) << first : 0u;
        uint32_t vf[2][2], mine[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          mine[w] = 0;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int k4 = keep - 4 * half;
            const uint32_t f = s.vf[w][half] & (k4 >= 4 ? 0xffffffffu : k4 <= 0 ? 0u : (1u << (8 * k4)) - 1u);
            const uint32_t marks = marks_255(f);
            mine[w] |= mark_bits(marks) << (4 * half);
            vf[w][half] = f & ~((marks >> 7) * 255u);
          }
        }
        make_values(vf);
        if (__builtin_amdgcn_ballot_w64((mine[0] | mine[1]) != 0) != 0) {
          // a group's marks for the 32 keys lie with lanes of the four quarters; a row's dims of the group with all
          // lanes of its column: row m of the operands, which is dim pair m / P of groups 2 (m % P), is o[..][m % 4]
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              uint32_t all = 0;
#pragma unroll
              for (int gg = 0; gg < 4; ++gg)
                all |= static_cast<uint32_t>(__shfl(static_cast<int>(mine[w]), gg * 16 + i % P, SE_WAVE)) << (8 * gg);
              const float poison = (all & seen) ? NAN : 0.f;
#pragma unroll
              for (int h = 0; h < P; ++h) {
                o[h][w][0][i] += poison;
                o[h][w][1][i] += poison;
              }
            }
        }
      }
      float m = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
      m *= scale_log2e;      // scale > 0: the maximum commutes with it
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(m <= run_max + SOFTMAX_SLACK)) != 0, 0)) {
        const float top = quad_max(m);
        if (top > run_max) {
          const float alpha = __builtin_amdgcn_exp2f(run_max - top);     // 0 where there was none
          run_max = top;
          run_sum *= alpha;
#pragma unroll
          for (int h = 0; h < P; ++h)
#pragma unroll
            for (int w = 0; w < 2; ++w) o[h][w][0] *= alpha, o[h][w][1] *= alpha;
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
      auto add_values = [&](const uint4& weights) {
#pragma unroll
        for (int h = 0; h < P; ++h)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            o[h][w][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even[h][w], __builtin_bit_cast(bf16x8, weights), o[h][w][0], 0, 0, 0);
            o[h][w][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd[h][w], __builtin_bit_cast(bf16x8, weights), o[h][w][1], 0, 0, 0);
          }
      };
      add_values(pf);
      // The rest is made while those products run, and no product waits for the one before it.
      uint4 rest;
      rest.x = rest_of_bf16x2(p[0], p[1], pf.x);
      rest.y = rest_of_bf16x2(p[2], p[3], pf.y);
      rest.z = rest_of_bf16x2(p[4], p[5], pf.z);
      rest.w = rest_of_bf16x2(p[6], p[7], pf.w);
      add_values(rest);
    };
    // (The first loads stay in the order of their steps: mixed, the wait for the first step's in front of the loop, and
    // with it the one at the head of every round, would be a wait for all of them.)
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      fetch(ring[i], k_first + 32 * i);
      __builtin_amdgcn_sched_barrier(0);
    }
    for (int k0 = k_first; k0 < key_end; k0 += 32 * NS) {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        // (No way out from the middle of a round: the wait at its head would be one for the loads just issued.)
        if (k0 + 32 * i < key_end) compute(ring[i], k0 + 32 * i);
        fetch(ring[i], k0 + 32 * (i + NS));
      }
    }
  }

  // lane (g, n): o[h][w][e][i] is, for row n, value dim 32 (2 (m % P) + w) + 2 (16 / P h + m / P) + e with m = 4 g + i
  const float total = quad_sum(run_sum);
  const float inv = 1.f / total;
  const int64_t base = (static_cast<int64_t>(slot) * kv_heads + kvh) * 16 + n;
  if (row_valid) {       // padding rows are nobody's
    bf16_t* o_row = out + static_cast<int64_t>(token) * out_stride + static_cast<int64_t>(head) * D;
    float* po = part_o + base * D;
#pragma unroll
    for (int h = 0; h < P; ++h)
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int m = 4 * g + i;
          const int dim = 32 * (2 * (m % P) + w) + 2 * (16 / P * h + m / P);
          if (slot < 0) *reinterpret_cast<uint32_t*>(o_row + dim) = floats_to_bf16x2_bits(o[h][w][0][i] * inv, o[h][w][1][i] * inv);
          else *reinterpret_cast<float2*>(po + dim) = float2{o[h][w][0][i], o[h][w][1][i]};
        }
    if (g == 0 && slot < 0 && lse != nullptr)
      lse[static_cast<int64_t>(token) * heads + head] = (run_max + __log2f(total)) * 0.6931471805599453f;
    if (g == 0 && slot >= 0) {
      part_ml[base * 2] = run_max;
      part_ml[base * 2 + 1] = total;
    }
  }
}

// Joins a tile's key ranges: one block per (task, kv head, row of the tile), task = {item, row_tile, first_slot,
// num_splits, q_start, q_len}.  256 threads are D / 4 pieces of four dims times as many shares of the ranges; a share's
// ranges are added in their order, then the shares in theirs.  (One block for all rows of a tile leaves the chip to
// eight blocks when one long request is decoded: 256 ranges of one request took 25 us that way, as long as the
// attention itself.)
#define TASK_FIELDS 6
#define MERGE_MAX_SPLITS 256
template <int D>
__global__ void __launch_bounds__(256)
merge_ranges_kernel(const int32_t* __restrict__ tasks, const float* __restrict__ part_o, const float* __restrict__ part_ml,
                    bf16_t* __restrict__ out, int64_t out_stride, float* __restrict__ lse, int heads, int kv_heads) {
  constexpr int PIECES = D / 4, SHARES = 256 / PIECES;
  __shared__ float weight[MERGE_MAX_SPLITS];
  __shared__ float reduced[2][4];
  __shared__ float4 sums[SHARES][PIECES];
  const int32_t* t = tasks + static_cast<int64_t>(blockIdx.x) * TASK_FIELDS;
  const int splits = t[3], q_start = t[4], q_len = t[5];
  const int kvh = blockIdx.y, group = heads / kv_heads;
  const int rho = t[1] * 16 + blockIdx.z;
  if (rho >= q_len * group) return;
  const int tid = threadIdx.x;
  // partial result of range s: base + s * stride
  const int64_t base = (static_cast<int64_t>(t[2]) * kv_heads + kvh) * 16 + blockIdx.z, stride = static_cast<int64_t>(kv_heads) * 16;
  const float m_own = tid < splits ? part_ml[(base + tid * stride) * 2] : -INFINITY;
  const float l_own = tid < splits ? part_ml[(base + tid * stride) * 2 + 1] : 0.f;
  const float m_wave = wave_max(m_own);
  if ((tid & 63) == 0) reduced[0][tid >> 6] = m_wave;
  __syncthreads();
  const float m = fmaxf(fmaxf(reduced[0][0], reduced[0][1]), fmaxf(reduced[0][2], reduced[0][3]));
  const float w_own = tid < splits ? exp2f(m_own - m) : 0.f;
  weight[tid] = w_own;
  const float l_wave = wave_sum(l_own * w_own);
  if ((tid & 63) == 0) reduced[1][tid >> 6] = l_wave;
  __syncthreads();
  const float total = (reduced[1][0] + reduced[1][1]) + (reduced[1][2] + reduced[1][3]);
  const int piece = tid % PIECES, share = tid / PIECES;
  const float* src = part_o + base * D + piece * 4;
  float4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = share; s0 < splits; s0 += 4 * SHARES) {
    float4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (s0 + i * SHARES < splits) v[i] = *reinterpret_cast<const float4*>(src + (s0 + i * SHARES) * stride * D);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (s0 + i * SHARES < splits) {
        const float w = weight[s0 + i * SHARES];
        acc.x += v[i].x * w;
        acc.y += v[i].y * w;
        acc.z += v[i].z * w;
        acc.w += v[i].w * w;
      }
  }
  sums[share][piece] = acc;
  __syncthreads();
  if (share != 0) return;
#pragma unroll
  for (int s = 1; s < SHARES; ++s) {
    const float4 v = sums[s][piece];
    acc.x += v.x;
    acc.y += v.y;
    acc.z += v.z;
    acc.w += v.w;
  }
  const float inv = 1.f / total;
  const int64_t token = q_start + rho / group;
  const int head = kvh * group + rho % group;
  uint2 packed;
  packed.x = floats_to_bf16x2_bits(acc.x * inv, acc.y * inv);
  packed.y = floats_to_bf16x2_bits(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(out + token * out_stride + static_cast<int64_t>(head) * D + piece * 4) = packed;
  if (lse != nullptr && tid == 0) lse[token * heads + head] = (m + __log2f(total)) * 0.6931471805599453f;
}

// The same with a wavefront per row, four rows to a block and no barrier: for so many rows that the chip is full of them.
template <int D>
__global__ void __launch_bounds__(256)
merge_rows_kernel(const int32_t* __restrict__ tasks, const float* __restrict__ part_o, const float* __restrict__ part_ml,
                  bf16_t* __restrict__ out, int64_t out_stride, float* __restrict__ lse, int heads, int kv_heads) {
  constexpr int OWN = D / SE_WAVE, ROUNDS = MERGE_MAX_SPLITS / SE_WAVE, AHEAD = 8;
  const int32_t* t = tasks + static_cast<int64_t>(blockIdx.x) * TASK_FIELDS;
  const int splits = t[3], q_start = t[4], q_len = t[5];
  const int kvh = blockIdx.y, group = heads / kv_heads;
  const int lane = threadIdx.x & (SE_WAVE - 1);
  const int row = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.z * 4 + threadIdx.x / SE_WAVE)), rho = t[1] * 16 + row;
  if (rho >= q_len * group) return;
  const int64_t base = (static_cast<int64_t>(t[2]) * kv_heads + kvh) * 16 + row, stride = static_cast<int64_t>(kv_heads) * 16;
  float m_own[ROUNDS], w[ROUNDS], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int s = r * SE_WAVE + lane;
    m_own[r] = s < splits ? part_ml[(base + s * stride) * 2] : -INFINITY;
    w[r] = s < splits ? part_ml[(base + s * stride) * 2 + 1] : 0.f;
    m = fmaxf(m, m_own[r]);
  }
  m = wave_max(m);
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const float scale = r * SE_WAVE + lane < splits ? exp2f(m_own[r] - m) : 0.f;
    l += w[r] * scale;
    w[r] = scale;
  }
  const float total = wave_sum(l);
  const float* src = part_o + base * D + lane * OWN;
  float acc[OWN];
#pragma unroll
  for (int j = 0; j < OWN; ++j) acc[j] = 0.f;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    for (int s0 = r * SE_WAVE; s0 < min(splits, (r + 1) * SE_WAVE); s0 += AHEAD) {
      float v[AHEAD][OWN];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
#pragma unroll
        for (int j = 0; j < OWN; ++j) v[i][j] = src[(min(s0 + i, splits - 1) * stride) * D + j];      // beyond the last: weight 0
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const float of_range = __shfl(w[r], s0 - r * SE_WAVE + i, SE_WAVE);
#pragma unroll
        for (int j = 0; j < OWN; ++j) acc[j] += s0 + i < splits ? v[i][j] * of_range : 0.f;
      }
    }
  }
  const float inv = 1.f / total;
  const int64_t token = q_start + rho / group;
  const int head = kvh * group + rho % group;
  bf16_t* dst = out + token * out_stride + static_cast<int64_t>(head) * D + lane * OWN;
#pragma unroll
  for (int j = 0; j < OWN; ++j) dst[j] = from_float<bf16_t>(acc[j] * inv);
  if (lse != nullptr && lane == 0) lse[token * heads + head] = (m + __log2f(total)) * 0.6931471805599453f;
}

// From so many rows (padding of tiles among them) on, a row is joined by a wavefront, below by a block.  Attention and merge
// by block / by wavefront, 48:8 heads of 128, one request: a token on 2100 keys 9.2 / 10.9 us, 16 on 32768 keys 46.7 / 47.2,
// 64 on 4096 keys 31.8 / 30.5, 512 on 16384 keys 272 / 264; 64 requests of 2100 keys 37.2 / 36.0.
#define MERGE_MANY_ROWS 2048
// Units and tasks as se_paged_attention_mfma takes them; the tasks also join what the block kernel of the unpacked pages
// has left in the same buffers.
extern "C" int se_paged_attention_fp4(const void* q, int64_t q_stride, const void* cache, const int32_t* block_table,
                                      int bt_stride, const int32_t* units, int num_units, const int32_t* tasks, int num_tasks,
                                      void* out, int64_t out_stride, float* part_o, float* part_ml, float* lse, int heads,
                                      int kv_heads, int head_dim, int page_size, float scale, int window, hipStream_t stream) {
  if (num_units <= 0 && num_tasks <= 0) return SE_OK;
  if (kv_heads <= 0 || heads % kv_heads || page_size <= 0 || page_size % 32 || kv_heads > 65535) return SE_ERR_SHAPE;
  if (fp4_head_bytes(page_size, head_dim) > 0x7fffffff) return SE_ERR_SHAPE;      // places in a page are 32-bit
  if (q_stride % 8 || out_stride % 4 || !(scale > 0.f)) return SE_ERR_SHAPE;
  if (num_tasks > 0 && (!part_o || !part_ml || !tasks)) return SE_ERR_SHAPE;      // splits per task <= 256 (host)
  const float scale_log2e = scale * 1.4426950408889634f;
  const dim3 grid((num_units + 3) / 4, kv_heads);
#define SE_FP4_ATT(DS, NS)                                                                                         \
  case 32 * DS:                                                                                                    \
    if (num_units > 0) {                                                                                           \
      paged_attention_fp4_kernel<DS, NS><<<grid, 256, 0, stream>>>(                                                \
          static_cast<const bf16_t*>(q), q_stride, static_cast<const uint8_t*>(cache), block_table, bt_stride, units, \
          num_units, static_cast<bf16_t*>(out), out_stride, part_o, part_ml, lse, heads, kv_heads, page_size, scale_log2e, \
          window);                                                                                                 \
      SE_CHECK_LAUNCH();                                                                                           \
    }                                                                                                              \
    if (num_tasks > 0) {                                                                                           \
      if (static_cast<int64_t>(num_tasks) * kv_heads * 16 < MERGE_MANY_ROWS)                                       \
        merge_ranges_kernel<32 * DS><<<dim3(num_tasks, kv_heads, 16), 256, 0, stream>>>(                           \
            tasks, part_o, part_ml, static_cast<bf16_t*>(out), out_stride, lse, heads, kv_heads);                  \
      else                                                                                                         \
        merge_rows_kernel<32 * DS><<<dim3(num_tasks, kv_heads, 4), 256, 0, stream>>>(                              \
            tasks, part_o, part_ml, static_cast<bf16_t*>(out), out_stride, lse, heads, kv_heads);                  \
      SE_CHECK_LAUNCH();                                                                                           \
    }                                                                                                              \
    break;
  switch (head_dim) {
    SE_FP4_ATT(2, 4) SE_FP4_ATT(4, 4) SE_FP4_ATT(8, 2)
    default: return SE_ERR_SHAPE;
  }
#undef SE_FP4_ATT
  return SE_OK;
}
