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
// matrix-core kernel does not take): a lane owns a key, four wavefronts share the rows of 64 keys, four rows at a time so
// that a key is read once for four.  Bound by the latency of a few such rounds where rows are few (3 requests of up to
// 300 keys with 5 new tokens each, 12:2 heads of 64 in float32: 9 us; row by row in one wavefront 24 us).
#define GENERIC_WAVES 4
#define GENERIC_ROWS 4
template <typename T, int KIND>
__global__ void __launch_bounds__(GENERIC_WAVES * SE_WAVE)
attention_weights_generic_kernel(const T* __restrict__ q, int64_t q_stride, const void* __restrict__ cache,
                                 const int32_t* __restrict__ block_table, int bt_stride,
                                 const int32_t* __restrict__ item_meta, int items, int longest,
                                 const float* __restrict__ lse, const float* previous, float* out, int heads, int kv_heads, int head_dim,
                                 int page_size, float scale, int window) {
  extern __shared__ float q_rows[];     // [GENERIC_WAVES][GENERIC_ROWS][head_dim]
  __shared__ float sums[GENERIC_WAVES][SE_WAVE];
  const int item = blockIdx.z, kvh = blockIdx.y, group = heads / kv_heads;
  const int lane = threadIdx.x & (SE_WAVE - 1), wave = threadIdx.x / SE_WAVE;
  const int q_start = item_meta[item], q_len = item_meta[items + item], ctx_len = min(item_meta[2 * items + item], longest);
  const int pos0 = ctx_len - q_len, rows = q_len * group;
  const int low_key = window > 0 && pos0 - window + 1 > 0 ? pos0 - window + 1 : 0;   // no row sees a key before it
  const int base = blockIdx.x * SE_WAVE;
  if (base >= ctx_len || base + SE_WAVE <= low_key) return;
  const int key = base + lane;
  const bool held = key < ctx_len && key >= low_key;
  const int page = held ? block_table[static_cast<int64_t>(item) * bt_stride + key / page_size] : 0;
  const int off = key % page_size;
  float* mine = q_rows + wave * GENERIC_ROWS * head_dim;
  float total = 0.f;
  // rows of tokens before the first key see none of the 64
  for (int rho = max(0, base - pos0) * group + wave * GENERIC_ROWS; rho < rows; rho += GENERIC_WAVES * GENERIC_ROWS) {
    if (window > 0 && pos0 + rho / group - window >= base + SE_WAVE - 1) break;     // nor do this one and all after it
    __builtin_amdgcn_wave_barrier();      // (a wavefront's own accesses to shared memory stay in their order)
    for (int i = lane; i < GENERIC_ROWS * head_dim; i += SE_WAVE) {
      const int row = min(rho + i / head_dim, rows - 1);
      mine[i] = to_float(q[(q_start + row / group) * q_stride + static_cast<int64_t>(kvh * group + row % group) * head_dim + i % head_dim]);
    }
    __builtin_amdgcn_wave_barrier();
    if (!held) continue;
    float dot[GENERIC_ROWS] = {0.f, 0.f, 0.f, 0.f};
    if constexpr (KIND == SE_CACHE_FP4) {
      const uint8_t* part = static_cast<const uint8_t*>(cache) +
                            (static_cast<int64_t>(page) * 2 * kv_heads + kvh) * fp4_head_bytes(page_size, head_dim);
      for (int d = 0; d < head_dim; d += 8) {
        const uint32_t word = *reinterpret_cast<const uint32_t*>(part + fp4_key_code_at(page_size, off, d / 32) + d % 32 / 2);
        const int factor = part[fp4_key_factor_at(page_size, head_dim, off, d / 32)];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float k = fp4_value(word >> (4 * j) & 15u, factor);
#pragma unroll
          for (int r = 0; r < GENERIC_ROWS; ++r) dot[r] += mine[r * head_dim + d + j] * k;
        }
      }
    } else {
      typedef typename std::conditional<KIND == SE_CACHE_F32, float, bf16_t>::type C;
      const C* part = static_cast<const C*>(cache) + (static_cast<int64_t>(page) * 2 * kv_heads + kvh) * page_size * head_dim;
      for (int d = 0; d < head_dim; d += Vec16<C>::N) {
        Vec16<C> k;
        k.v = *reinterpret_cast<const decltype(k.v)*>(part + key_place(page_size, off, d));
#pragma unroll
        for (int j = 0; j < Vec16<C>::N; ++j) {
#pragma unroll
          for (int r = 0; r < GENERIC_ROWS; ++r) dot[r] += mine[r * head_dim + d + j] * k.get(j);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < GENERIC_ROWS; ++r) {
      const int row = rho + r, pos = pos0 + row / group;
      if (row >= rows || key > pos || (window > 0 && key <= pos - window)) continue;
      total += expf(dot[r] * scale - lse[static_cast<int64_t>(q_start + row / group) * heads + kvh * group + row % group]);
    }
  }
  sums[wave][lane] = total;
  __syncthreads();
  if (wave != 0 || !held) return;
#pragma unroll
  for (int w = 1; w < GENERIC_WAVES; ++w) total += sums[w][lane];
  const int64_t at = (static_cast<int64_t>(page) * kv_heads + kvh) * page_size + off;
  out[at] = (previous != nullptr && key < pos0 ? previous[at] : 0.f) + total;
}

// The matrix-core form (bfloat16 rows; head size 32 * DS; keys in bfloat16 or 4 bits).  A wavefront owns 32 * KP
// consecutive keys, whose operands it loads once and keeps in registers (4 bits are turned into bfloat16 on the
// way), and goes through the tiles of 16 rows that see any of them:
//   S = Q K^T        v_mfma_f32_16x16x32_bf16, A = 16 rows x 32 dims, B = 32 dims x 16 keys, so that a lane ends up
//                    with four rows of one key and the sum over rows is additions in a lane; the four lanes that
//                    share a key meet once at the end.
// With one tile of rows (decoding; in 4 bits most head sizes have the kernel behind this one for it) a block is four
// wavefronts side by side along the keys, and the kernel is bound by the chain of loads in front of its few products: the
// request's lengths, the page ids, the keys (rows and previous weights are on their way with them).  With more, the wavefronts of a block take turns at the tiles of the same
// keys (`row_waves`), and several blocks do where there are too few of them to fill the chip evenly (`row_blocks`:
// their sums go to a workspace and a second kernel adds them up); everything is added in one order.  The kernel is then bound
// by the vector and the matrix unit in turns: a tile of 16 rows and 128 keys at head size 128 is 32 exponentials, at a quarter
// of the rate, and 64 other instructions of the one (768 clocks), and 32 products of the other (512), whose results the
// exponentials wait for.  2048 rows x 6 heads on 6000 keys would take 85 us of the one, 57 us of the other, and take 168.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

// How a launch goes through the rows.  ONE tile (decoding): no loop, and no rows fetched that are not there.  FEW: rows
// straight into operands.  MANY: vector instructions are dear, and a tile of 16 rows and 128 keys needs
// 96 for its exponentials, their arguments and sums, and as much again went into finding its rows; so the 64 lanes
// find 64 rows (four tiles) at once, and a tile is read row by row (256 contiguous bytes for sixteen lanes) and turned
// into operands through the wavefront's own part of shared memory (rows 16 bytes apart beyond their length: no two
// lanes of a read meet in a bank).  2048 rows x 6 heads on 6000 keys: 241 us with rows found and read tile by tile, 195 us
// so, 0.65 PFLOP/s; the same with 64 keys and three wavefronts per SIMD instead of 128 and two 205 us.
enum WeightRows { ROWS_ONE = 0, ROWS_FEW = 1, ROWS_MANY = 2 };

// Groups of 32 keys a wavefront owns: as many as the registers hold where the work that a tile of rows costs whatever the
// keys is to be shared (MANY at head size 128: 128 registers of operands).
template <int DS, int MODE>
struct WeightShape {
  static constexpr int KP = MODE == ROWS_MANY ? (DS == 1 ? 8 : DS <= 4 ? 4 : DS <= 6 ? 2 : 1)
                            : MODE == ROWS_ONE ? (DS == 1 ? 8 : DS == 2 ? 6 : DS <= 4 ? 4 : 2)
                                               : (DS <= 2 ? 4 : DS <= 4 ? 2 : 1);
  static constexpr int WAVES = 4;      // of a block
  static constexpr int PER_SIMD = MODE == ROWS_MANY ? 2 : 1;
};

template <int DS, int KIND, int MODE>
__global__ void __launch_bounds__((64 * WeightShape<DS, MODE>::WAVES), (WeightShape<DS, MODE>::PER_SIMD))
attention_weights_mfma_kernel(const bf16_t* __restrict__ q, int64_t q_stride, const void* __restrict__ cache,
                              const int32_t* __restrict__ block_table, int bt_stride,
                              const int32_t* __restrict__ item_meta, int items, int longest,
                              const float* __restrict__ lse, const float* previous, float* out, int heads, int kv_heads,
                              int page_size, float scale_log2e, int window, int row_waves, int row_blocks,
                              float* __restrict__ partial) {
  constexpr int D = 32 * DS;
  constexpr int KP = WeightShape<DS, MODE>::KP, waves = WeightShape<DS, MODE>::WAVES;
  constexpr int ROW_BYTES = 64 * DS + 16;      // of a row in shared memory
  // which eight dims of a lane's operand are those of product step ds: in 4 bits, where a lane's part of a key can be
  // one piece under one factor, neighbouring ones
  constexpr bool WIDE = KIND == SE_CACHE_FP4 && (DS == 2 || DS == 4 || DS == 8);
  __shared__ float sums[waves][KP * 2][16];
  constexpr int INFO = MODE == ROWS_MANY ? waves : 1;
  __shared__ __align__(16) int64_t row_places[INFO][2][64];
  __shared__ __align__(16) float row_lse2[INFO][2][64];
  __shared__ __align__(16) int row_pos[INFO][2][64];
  __shared__ __align__(16) unsigned char staged[MODE == ROWS_MANY ? waves * 16 * ROW_BYTES : 16];
  const int lane = threadIdx.x & (SE_WAVE - 1);
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / SE_WAVE));
  const int n = lane & 15, g = lane >> 4;
  const int item = blockIdx.z, kvh = blockIdx.y, group = heads / kv_heads;
  const int q_start = item_meta[item], q_len = item_meta[items + item], ctx_len = min(item_meta[2 * items + item], longest);
  const int pos0 = ctx_len - q_len, last_key = ctx_len - 1;
  const int low_key = window > 0 && pos0 - window + 1 > 0 ? pos0 - window + 1 : 0;   // no row sees a key before it
  const int row_block = blockIdx.x % row_blocks, key_block = blockIdx.x / row_blocks;
  const int part = wave % row_waves;                                                 // of the block's share of the rows
  const int k_lo = (key_block * (waves / row_waves) + wave / row_waves) * (32 * KP), k_hi = k_lo + 32 * KP - 1;
  const bool wanted = k_lo < ctx_len && k_hi >= low_key;      // the same in all wavefronts that share keys
  const int32_t* table = block_table + static_cast<int64_t>(item) * bt_stride;

  auto dims_of = [&](int ds) { return WIDE ? (D / 4) * g + 8 * ds : 32 * ds + 8 * g; };
  // a lane's keys: two neighbours in 4 bits (one piece of memory), else sixteen lanes side by side
  auto key_of = [&](int kp, int b) { return k_lo + 32 * kp + (KIND == SE_CACHE_FP4 ? 2 * n + b : 16 * b + n); };

  // where a lane's key has its weight (some held key's for one that is not held)
  auto place_of = [&](int kp, int b) {
    if constexpr (KIND == SE_CACHE_FP4) {      // 32 keys lie in one page: scalar work
      const int first = max(min(k_lo + 32 * kp, last_key & ~31), low_key & ~31);
      return (static_cast<int64_t>(table[first / page_size]) * kv_heads + kvh) * page_size + first % page_size + 2 * n + b;
    } else {
      const int key = max(min(key_of(kp, b), last_key), low_key);
      return (static_cast<int64_t>(table[key / page_size]) * kv_heads + kvh) * page_size + key % page_size;
    }
  };

  float acc[KP][2], before[KP][2];
  int64_t place[KP][2];
#pragma unroll
  for (int kp = 0; kp < KP; ++kp) acc[kp][0] = acc[kp][1] = before[kp][0] = before[kp][1] = 0.f;

  if (wanted) {
    // the tiles with a row that sees one of the keys
    const int rows_total = q_len * group;
    int tile = k_lo > pos0 ? static_cast<int>(static_cast<int64_t>(k_lo - pos0) * group / 16) : 0;
    int until = (rows_total + 15) / 16;
    if (window > 0) {
      const int64_t last_q = static_cast<int64_t>(min(k_hi, last_key)) + window - 1 - pos0;
      if (last_q + 1 < q_len) until = static_cast<int>(((last_q + 1) * group + 15) / 16);
    }
    struct Rows {
      uint4 q[DS];     // the lane's operands (MANY: not used)
      int64_t at;      // where its row begins (MANY only)
      float lse;       // of that row
      int pos, rho;    // rho >= rows_total: there is no such row
    };
    // a lane's row of the next tile to be fetched: row `rho` of the request is head `row_head` of token `row_token`
    if constexpr (MODE != ROWS_MANY) tile += row_block * row_waves + part;
    const int tile_step = row_waves * row_blocks;
    int rho = tile * 16 + n;
    int row_token = rho / group, row_head = rho - row_token * group;
    const int step = tile_step * 16, step_tokens = step / group, step_heads = step - step_tokens * group;
    auto fetch = [&](Rows& r) {      // the wavefront's tiles, one after the other
      const bool valid = rho < rows_total;
      const int q_idx = valid ? row_token : q_len - 1, head = kvh * group + (valid ? row_head : group - 1);
      const int64_t row_at = static_cast<int64_t>(q_start + q_idx) * q_stride + static_cast<int64_t>(head) * D;
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) r.q[ds] = *reinterpret_cast<const uint4*>(q + row_at + dims_of(ds));
      r.lse = lse[static_cast<int64_t>(q_start + q_idx) * heads + head];   // not looked at here: that would be a wait
      r.pos = pos0 + q_idx;
      r.rho = rho;
      rho += step;
      row_token += step_tokens;
      row_head += step_heads;
      if (row_head >= group) {
        row_head -= group;
        ++row_token;
      }
    };
    Rows a, b;      // the next tile's rows are on their way while one is worked on; beyond the last tile the last row once more
    if constexpr (MODE != ROWS_MANY) fetch(a);
    if constexpr (MODE == ROWS_FEW) fetch(b);
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

    if (MODE == ROWS_ONE && g == 0) {      // on their way with the keys
#pragma unroll
      for (int kp = 0; kp < KP; ++kp)
#pragma unroll
        for (int b2 = 0; b2 < 2; ++b2) {
          place[kp][b2] = place_of(kp, b2);
          const int key = key_of(kp, b2);
          if (previous != nullptr && key < pos0 && key >= low_key) before[kp][b2] = previous[place[kp][b2]];
        }
    }
    // rows: a lane's operand of row n; l, pos: lse (in powers of two) and position of rows 4 g + i
    auto weigh = [&](const uint4 (&rows)[DS], const float (&l)[4], const int (&pos)[4], bool some_hidden) {
      floatx4 s[KP][2];
#pragma unroll
      for (int kp = 0; kp < KP; ++kp)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          s[kp][b] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ds = 0; ds < DS; ++ds)
            s[kp][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, rows[ds]),
                                                               __builtin_bit_cast(bf16x8, kf[kp][b][ds]), s[kp][b], 0, 0, 0);
        }
      // lane (g, n): s[kp][b][i] is the score of row 4 g + i for key key_of(kp, b)
      if (__builtin_expect(some_hidden, 0)) {      // the same in all lanes
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int hidden = window > 0 ? pos[i] - window : -1;      // the last key too old
#pragma unroll
          for (int kp = 0; kp < KP; ++kp)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const int key = key_of(kp, b);
              s[kp][b][i] = ((key > pos[i]) | (key <= hidden)) ? -INFINITY : s[kp][b][i];
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
    // (No way out from the middle of a round: the wait at its head would be one for the loads just issued.)
    auto weigh_tile = [&](const Rows& r) {
      const float lse2 = r.rho < rows_total ? r.lse * 1.4426950408889634f : INFINITY;     // in powers of two
      float l[4];
      int pos[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) l[i] = __shfl(lse2, 4 * g + i, SE_WAVE), pos[i] = __shfl(r.pos, 4 * g + i, SE_WAVE);
      const int pos_min = __builtin_amdgcn_readlane(r.pos, 0), pos_max = __builtin_amdgcn_readlane(r.pos, 15);
      weigh(r.q, l, pos, k_hi > pos_min || (window > 0 && k_lo <= pos_max - window));
    };
    if constexpr (MODE == ROWS_ONE) {
      if (tile < until) weigh_tile(a);
    } else if constexpr (MODE == ROWS_FEW) {
      for (; tile < until; tile += 2 * tile_step) {
        weigh_tile(a);
        fetch(a);
        if (tile + tile_step < until) weigh_tile(b);
        fetch(b);
      }
    } else {
      // Four tiles at a time: lane l works out where row l of the 64 lies, its lse and its position, for the four tiles
      // after those at hand, and leaves them in the wavefront's own shared memory (a wavefront's own accesses to it stay
      // in their order).  The tile after the one at hand is on its way: its vectors lane, 64 + lane, ... in the order of
      // its rows.  (A macro and plain vectors of this scope: an array of them that a lambda fills through a reference, or of
      // the runtime's vector type, ends up in scratch memory.)
      const int groups_until = (until + 3) / 4, group_step = tile_step;
      int row_group = tile / 4 + row_block * row_waves + part;      // of 64 rows
      unsigned char* mine = staged + wave * 16 * ROW_BYTES;
      int64_t(*places)[64] = row_places[wave];
      float(*lse2)[64] = row_lse2[wave];
      int(*positions)[64] = row_pos[wave];
      Rows info;
      info.rho = 0;
      rho = row_group * 64 + lane;
      row_token = rho / group, row_head = rho - row_token * group;
      const int info_step = group_step * 64, info_tokens = info_step / group, info_heads = info_step - info_tokens * group;
      auto ask = [&]() {
        const bool valid = rho < rows_total;
        const int q_idx = valid ? row_token : q_len - 1, head = kvh * group + (valid ? row_head : group - 1);
        info.at = static_cast<int64_t>(q_start + q_idx) * q_stride + static_cast<int64_t>(head) * D;
        info.lse = lse[static_cast<int64_t>(q_start + q_idx) * heads + head];
        info.pos = pos0 + q_idx;
        info.rho = rho;
        rho += info_step;
        row_token += info_tokens;
        row_head += info_heads;
        if (row_head >= group) row_head -= group, ++row_token;
      };
      auto keep_info = [&](int buffer) {
        places[buffer][lane] = info.at;
        lse2[buffer][lane] = info.rho < rows_total ? info.lse * 1.4426950408889634f : INFINITY;    // +inf: there is no such row
        positions[buffer][lane] = info.pos;
      };
      se_u32x4 next[DS];
#define WEIGHT_READ_ROWS(BUFFER, TILE)                                                                                    \
  _Pragma("unroll") for (int i = 0; i < DS; ++i)                                                                          \
      next[i] = *reinterpret_cast<const se_u32x4*>(q + places[BUFFER][16 * (TILE) + (64 * i + lane) / (4 * DS)] +         \
                                                   (64 * i + lane) % (4 * DS) * 8);
      int buffer = 0;
      if (row_group < groups_until) {
        ask();
        keep_info(0);
        __builtin_amdgcn_wave_barrier();
        WEIGHT_READ_ROWS(0, 0)
      }
      for (; row_group < groups_until; row_group += group_step, buffer ^= 1) {
        const int pos_min = __builtin_amdgcn_readfirstlane(positions[buffer][0]);
        const int pos_max = __builtin_amdgcn_readfirstlane(positions[buffer][63]);
        const bool some_hidden = k_hi > pos_min || (window > 0 && k_lo <= pos_max - window);      // from some of the 64 rows
        ask();      // beyond the last rows: the last one
#pragma unroll 1      // four copies of the body would hoist each other's work into more registers than there are
        for (int t = 0; t < 4; ++t) {
#pragma unroll
          for (int i = 0; i < DS; ++i)
            *reinterpret_cast<se_u32x4*>(mine + (64 * i + lane) / (4 * DS) * ROW_BYTES + (64 * i + lane) % (4 * DS) * 16) = next[i];
          if (t == 2) keep_info(buffer ^ 1);
          __builtin_amdgcn_wave_barrier();
          WEIGHT_READ_ROWS((t < 3 ? buffer : buffer ^ 1), (t + 1 & 3))
          uint4 rows[DS];
#pragma unroll
          for (int ds = 0; ds < DS; ++ds) rows[ds] = *reinterpret_cast<const uint4*>(mine + n * ROW_BYTES + dims_of(ds) * 2);
          const float4 l4 = *reinterpret_cast<const float4*>(&lse2[buffer][16 * t + 4 * g]);
          const int4 p4 = *reinterpret_cast<const int4*>(&positions[buffer][16 * t + 4 * g]);
          __builtin_amdgcn_wave_barrier();
          const float l[4] = {l4.x, l4.y, l4.z, l4.w};
          const int p[4] = {p4.x, p4.y, p4.z, p4.w};
          weigh(rows, l, p, some_hidden);
        }
      }
#undef WEIGHT_READ_ROWS
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
      if (row_blocks > 1) {
        partial[((static_cast<int64_t>(row_block) * items + item) * kv_heads + kvh) * longest + key] = acc[kp][b];
        continue;
      }
      if constexpr (MODE == ROWS_ONE) {
        out[place[kp][b]] = before[kp][b] + acc[kp][b];
      } else {
        const int64_t at = place_of(kp, b);
        out[at] = (previous != nullptr && key < pos0 ? previous[at] : 0.f) + acc[kp][b];
      }
    }
}

// The same for one tile of rows (decoding) over a cache in 4 bits at head sizes whose part of a key is one piece to a
// lane: a wavefront goes through `per_wave` groups of 32 keys with the codes, factors and previous weights of
// ONE_TILE_DEPTH groups on their way, and turns a group into operands when its turn comes.  Owning 128 keys and ending,
// as the kernel above does, spends more instructions on finding rows, pages and places than on the keys (16 requests of
// up to 8200 keys, 48:8 heads of 128: 19 us, now 15.6; 64 of up to 30000 keys 281 us, now 215, 4.1 TB/s of codes, factors
// and weights, where attention over the same pages reads at 4.6).  The sums of a group's two keys to a lane meet in one
// pass over the four lanes that share them.  HIDDEN: some request has several tokens, whose rows do not all see the last keys; with a single
// token a key that it cannot see is one whose weight is not written.
#define ONE_TILE_DEPTH 4
template <int DS, bool HIDDEN>
__global__ void __launch_bounds__(256, 2)
attention_weights_one_tile_fp4_kernel(const bf16_t* __restrict__ q, int64_t q_stride, const uint8_t* __restrict__ cache,
                                      const int32_t* __restrict__ block_table, int bt_stride,
                                      const int32_t* __restrict__ item_meta, int items, int longest,
                                      const float* __restrict__ lse, const float* previous, float* out, int heads,
                                      int kv_heads, int page_size, float scale_log2e, int window, int per_wave) {
  static_assert(DS == 2 || DS == 4 || DS == 8, "a lane's part of a key lies in one piece of memory per group");
  constexpr int D = 32 * DS, DEPTH = ONE_TILE_DEPTH;
  constexpr int PIECES = (DS + 3) / 4, WORDS = DS == 2 ? 2 : 4;      // of a lane's part of a key: groups of dims, words of codes
  const int lane = threadIdx.x & (SE_WAVE - 1);
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / SE_WAVE));
  const int n = lane & 15, g = lane >> 4;
  const int item = blockIdx.z, kvh = blockIdx.x, group = heads / kv_heads;
  const int q_start = item_meta[item], q_len = item_meta[items + item], ctx_len = min(item_meta[2 * items + item], longest);
  const int pos0 = ctx_len - q_len;
  const int low_key = window > 0 && pos0 - window + 1 > 0 ? pos0 - window + 1 : 0;
  const int first = low_key / 32 + (static_cast<int>(blockIdx.y) * 4 + wave) * per_wave;      // of the wavefront's groups
  const int last = min(first + per_wave, (ctx_len + 31) / 32) - 1;
  if (first > last) return;
  const int32_t* table = block_table + static_cast<int64_t>(item) * bt_stride;

  // a page's bytes of a group of dims that this lane reads, relative to the group of keys
  const int64_t head_bytes = fp4_head_bytes(page_size, D), factors = fp4_factors_at(page_size, D);
  const int dims = DS == 2 ? g >> 1 : g * PIECES;      // its first group of dims
  const int lane_codes = (dims * page_size + 2 * n) * 16 + (DS == 2 ? (g & 1) * 8 : 0);
  const int lane_factors = static_cast<int>(factors) + dims * page_size + (2 * n & ~3), half_shift = (n & 1) * 16;
  const int lane_key = 2 * n + (g >> 1);               // whose weight it reads, and writes if g is even
  const float* old = previous != nullptr ? previous : out;      // out: read, but not taken

  // the rows: lane (g, n) has dims of row n as an operand, and what belongs to rows 4 g + i
  const int rows = q_len * group, row = min(n, rows - 1);
  uint4 rows_q[DS];
  {
    const bf16_t* at = q + static_cast<int64_t>(q_start + row / group) * q_stride + static_cast<int64_t>(kvh * group + row % group) * D + (D / 4) * g;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) rows_q[ds] = *reinterpret_cast<const uint4*>(at + 8 * ds);
  }
  float l[4];      // turned into powers of two below; +inf: there is no such row
  int pos[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = min(4 * g + i, rows - 1), token = r / group;
    const float of_row = lse[static_cast<int64_t>(q_start + token) * heads + kvh * group + r - token * group];
    l[i] = of_row;
    pos[i] = pos0 + token;
  }
  // asked for before the keys: a wait for what comes later would be one for them too
  __builtin_amdgcn_sched_barrier(0);

  se_u32x4 codes[DEPTH][2][PIECES];
  uint32_t factor[DEPTH][PIECES];      // of two lanes' keys (16 bits would be widened, or packed, where they are waited for)
  float before[DEPTH];
  int64_t place[DEPTH];
  int page = first * 32 / page_size, off = first * 32 - page * page_size, asked = first;
  const int last_page = last * 32 / page_size;
  int id = table[page], next_id = table[min(page + 1, last_page)];
#define ONE_TILE_ASK(S)                                                                                                  \
  {                                                                                                                      \
    const uint8_t* at = cache + (static_cast<int64_t>(id) * 2 * kv_heads + kvh) * head_bytes;                            \
    _Pragma("unroll") for (int h = 0; h < PIECES; ++h) {                                                                 \
      factor[S][h] = *reinterpret_cast<const uint32_t*>(at + off + lane_factors + h * page_size);                        \
      _Pragma("unroll") for (int b = 0; b < 2; ++b) {                                                                    \
        const uint8_t* piece = at + off * 16 + lane_codes + h * page_size * 16 + b * 16;                                 \
        if constexpr (DS == 2) {                                                                                         \
          const uint2 v = *reinterpret_cast<const uint2*>(piece);                                                        \
          codes[S][b][h] = se_u32x4{v.x, v.y, 0, 0};                                                                     \
        } else {                                                                                                         \
          codes[S][b][h] = __builtin_nontemporal_load(reinterpret_cast<const se_u32x4*>(piece));                         \
        }                                                                                                                \
      }                                                                                                                  \
    }                                                                                                                    \
    place[S] = (static_cast<int64_t>(id) * kv_heads + kvh) * page_size + off;                                            \
    before[S] = old[place[S] + lane_key];                                                                                \
    if (asked < last) { /* beyond the last group: that one once more */                                                  \
      ++asked;                                                                                                           \
      off += 32;                                                                                                         \
      if (off == page_size) {                                                                                            \
        off = 0;                                                                                                         \
        id = next_id;                                                                                                    \
        ++page;                                                                                                          \
        next_id = table[min(page + 1, last_page)];                                                                       \
      }                                                                                                                  \
    }                                                                                                                    \
  }
#pragma unroll
  for (int s = 0; s < DEPTH; ++s) {
    ONE_TILE_ASK(s)
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < 4; ++i) l[i] = 4 * g + i < rows ? l[i] * 1.4426950408889634f : INFINITY;

#define ONE_TILE_WEIGH(S, AT)                                                                                            \
  {                                                                                                                      \
    floatx4 sc[2];                                                                                                       \
    _Pragma("unroll") for (int b = 0; b < 2; ++b) {                                                                      \
      sc[b] = floatx4{0.f, 0.f, 0.f, 0.f};                                                                               \
      _Pragma("unroll") for (int h = 0; h < PIECES; ++h) {                                                               \
        const uint32_t two = factor[S][h] >> half_shift, f = b == 0 ? fp4_factor_bits<0>(two) : fp4_factor_bits<1>(two); \
        _Pragma("unroll") for (int w = 0; w < WORDS; ++w)                                                                \
          sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, rows_q[WORDS * h + w]),             \
                                                          __builtin_bit_cast(bf16x8, fp4_eight(codes[S][b][h][w], f)),   \
                                                          sc[b], 0, 0, 0);                                               \
      }                                                                                                                  \
    }                                                                                                                    \
    float sum[2];                                                                                                        \
    _Pragma("unroll") for (int b = 0; b < 2; ++b) {                                                                      \
      const int key = 32 * (AT) + 2 * n + b;                                                                             \
      sum[b] = 0.f;                                                                                                      \
      _Pragma("unroll") for (int i = 0; i < 4; ++i) {                                                                    \
        float v = fmaf(sc[b][i], scale_log2e, -l[i]);                                                                    \
        if (HIDDEN) v = ((key > pos[i]) | (window > 0 & key <= pos[i] - window)) ? -INFINITY : v;                        \
        sum[b] += __builtin_amdgcn_exp2f(v);                                                                             \
      }                                                                                                                  \
    }                                                                                                                    \
    /* lanes of g = 0, 1 end up with the first key's sum over the four lanes, those of g = 2, 3 with the second's */    \
    const auto half = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum[0]), __float_as_uint(sum[1]), false, false);  \
    const float two = __uint_as_float(half[0]) + __uint_as_float(half[1]);                                               \
    const auto rest = __builtin_amdgcn_permlane16_swap(__float_as_uint(two), __float_as_uint(two), false, false);        \
    const float total = __uint_as_float(rest[0]) + __uint_as_float(rest[1]);                                             \
    const int key = 32 * (AT) + lane_key;                                                                                \
    const float was = previous != nullptr && key < pos0 ? before[S] : 0.f;                                               \
    if ((AT) <= last && (g & 1) == 0 && key < ctx_len && key >= low_key) out[place[S] + lane_key] = was + total;         \
  }
  int at = first;
  for (; at + DEPTH <= last; at += DEPTH) {      // while groups are left that are not yet on their way
#pragma unroll
    for (int s = 0; s < DEPTH; ++s) {
      ONE_TILE_WEIGH(s, at + s)
      ONE_TILE_ASK(s)
    }
  }
#pragma unroll
  for (int s = 0; s < DEPTH; ++s) {
    ONE_TILE_WEIGH(s, at + s)
  }
#undef ONE_TILE_ASK
#undef ONE_TILE_WEIGH
}

// Adds up the sums of `row_blocks` blocks of every key.
__global__ void __launch_bounds__(256)
join_weights_kernel(const float* __restrict__ partial, int row_blocks, const int32_t* __restrict__ block_table, int bt_stride,
                    const int32_t* __restrict__ item_meta, int items, int longest, const float* previous, float* out,
                    int kv_heads, int page_size, int window) {
  const int item = blockIdx.z, kvh = blockIdx.y, key = blockIdx.x * blockDim.x + threadIdx.x;
  const int q_len = item_meta[items + item], ctx_len = min(item_meta[2 * items + item], longest), pos0 = ctx_len - q_len;
  const int low_key = window > 0 && pos0 - window + 1 > 0 ? pos0 - window + 1 : 0;
  if (key >= ctx_len || key < low_key) return;
  float sum = 0.f;
  for (int s = 0; s < row_blocks; ++s) sum += partial[((static_cast<int64_t>(s) * items + item) * kv_heads + kvh) * longest + key];
  const int page = block_table[static_cast<int64_t>(item) * bt_stride + key / page_size];
  const int64_t at = (static_cast<int64_t>(page) * kv_heads + kvh) * page_size + key % page_size;
  out[at] = (previous != nullptr && key < pos0 ? previous[at] : 0.f) + sum;
}

// Blocks that share the rows of the same keys: enough for six rounds of one block of eight wavefronts per CU, as long
// as a wavefront has at least four tiles (2048 rows x 6 heads on 6000 keys, 8 kv heads: 376 blocks alone run in one
// round and a half, 241 us).
#define WEIGHT_BLOCKS 1536
// Wavefronts of the one-tile kernel: more than run at once (five per SIMD), since requests differ in length (16 x 8200
// keys: 19 us with 2048, 17.6 with 4096, 15.6 with 16384; 64 x 30000 keys 217 us with any).
#define ONE_TILE_WAVES 16384
static int many_rows_keys(int head_dim) {      // of a wavefront, as WeightShape has it
  const int ds = head_dim / 32;
  return 32 * (ds == 1 ? 8 : ds <= 4 ? 4 : ds <= 6 ? 2 : 1);
}
static bool weights_on_matrix_cores(int head_dim, int64_t most_rows, int dtype) {
  return dtype == SE_BF16 && head_dim % 32 == 0 && head_dim <= 256 && most_rows < 0x40000000;
}
// How many sums of every key a call leaves in its workspace: float [that, items, kv_heads, longest] (1: none is used).
// Up to 32 tiles of rows it is 1 (the callers rely on it).
extern "C" int se_attention_weights_splits(int items, int longest, int most_new, int heads, int kv_heads, int head_dim, int dtype) {
  if (items <= 0 || longest <= 0 || kv_heads <= 0 || heads % kv_heads || head_dim <= 0) return 1;
  const int64_t most_rows = static_cast<int64_t>(most_new) * (heads / kv_heads);
  const int64_t tiles = (most_rows + 15) / 16;
  if (!weights_on_matrix_cores(head_dim, most_rows, dtype) || tiles <= 32) return 1;
  const int64_t keys = many_rows_keys(head_dim);
  const int64_t blocks = (longest + keys - 1) / keys * kv_heads * items;
  int64_t splits = (WEIGHT_BLOCKS + blocks - 1) / blocks;
  if (splits > tiles / 32) splits = tiles / 32;
  return splits < 1 ? 1 : splits > 16 ? 16 : static_cast<int>(splits);
}

template <int DS, int KIND>
static void launch_weights_mfma(const void* q, int64_t q_stride, const void* cache, const int32_t* block_table, int bt_stride,
                                const int32_t* item_meta, int items, int longest, int most_new, const float* lse,
                                const float* previous, float* out, int heads, int kv_heads, int page_size, float scale,
                                int window, int splits, float* partial, hipStream_t stream) {
  // With a single tile there is nothing to share out among the wavefronts of the same keys.
  const int tiles = static_cast<int>((static_cast<int64_t>(most_new) * (heads / kv_heads) + 15) / 16);
  constexpr bool ONE_TILE_FP4 = KIND == SE_CACHE_FP4 && (DS == 2 || DS == 4 || DS == 8);
  if constexpr (ONE_TILE_FP4) {
    if (tiles <= 1) {
      // groups of a wavefront, in whole rounds of those on their way
      const int64_t reach = static_cast<int64_t>(window) + most_new + 62;      // a window may be as long as an int holds
      const int64_t span = window > 0 && reach < longest ? reach : longest;
      const int64_t groups = (span + 31) / 32, all = groups * kv_heads * items;
      int per_wave = static_cast<int>((all + ONE_TILE_WAVES - 1) / ONE_TILE_WAVES);
      per_wave = (per_wave + ONE_TILE_DEPTH - 1) / ONE_TILE_DEPTH * ONE_TILE_DEPTH;
      const dim3 grid(kv_heads, static_cast<unsigned>((groups + 4 * per_wave - 1) / (4 * per_wave)), items);
#define SE_WEIGHTS_ONE_TILE(HIDDEN)                                                                                        \
  attention_weights_one_tile_fp4_kernel<DS, HIDDEN><<<grid, 256, 0, stream>>>(                                             \
      static_cast<const bf16_t*>(q), q_stride, static_cast<const uint8_t*>(cache), block_table, bt_stride, item_meta, items, longest, \
      lse, previous, out, heads, kv_heads, page_size, scale * 1.4426950408889634f, window, per_wave)
      if (most_new > 1) SE_WEIGHTS_ONE_TILE(true);
      else SE_WEIGHTS_ONE_TILE(false);
#undef SE_WEIGHTS_ONE_TILE
      return;
    }
  }
#define SE_WEIGHTS_LAUNCH(MODE, ROW_WAVES, ROW_BLOCKS)                                                                     \
  {                                                                                                                        \
    constexpr int waves = WeightShape<DS, MODE>::WAVES;                                                                    \
    const int per_block = 32 * WeightShape<DS, MODE>::KP * (waves / (ROW_WAVES));                                          \
    const dim3 grid((longest + per_block - 1) / per_block * (ROW_BLOCKS), kv_heads, items);                                \
    attention_weights_mfma_kernel<DS, KIND, MODE><<<grid, waves * SE_WAVE, 0, stream>>>(                                   \
        static_cast<const bf16_t*>(q), q_stride, cache, block_table, bt_stride, item_meta, items, longest, lse, previous, out, \
        heads, kv_heads, page_size, scale * 1.4426950408889634f, window, ROW_WAVES, ROW_BLOCKS, partial);                  \
  }
  if (tiles <= 1) {
    if constexpr (!ONE_TILE_FP4) SE_WEIGHTS_LAUNCH(ROWS_ONE, 1, 1)
  } else if (tiles <= 8) SE_WEIGHTS_LAUNCH(ROWS_FEW, 2, 1)
  else if (tiles <= 32) SE_WEIGHTS_LAUNCH(ROWS_FEW, 4, 1)
  else SE_WEIGHTS_LAUNCH(ROWS_MANY, waves, splits)
#undef SE_WEIGHTS_LAUNCH
  if (splits > 1)
    join_weights_kernel<<<dim3((longest + 255) / 256, kv_heads, items), 256, 0, stream>>>(
        partial, splits, block_table, bt_stride, item_meta, items, longest, previous, out, kv_heads, page_size, window);
}

// q [.., heads, head_dim] with token stride q_stride; cache of `kind` (SeCacheKind); item_meta int32 [3, items]:
// first token, new tokens and tokens with them of every request; longest: the largest of the latter; most_new: the
// largest of the new ones; workspace: what se_attention_weights_splits says.
extern "C" int se_attention_weights(const void* q, int64_t q_stride, const void* cache, int kind,
                                    const int32_t* block_table, int bt_stride, const int32_t* item_meta, int items,
                                    int longest, int most_new, const float* lse, const float* previous, float* out, int heads,
                                    int kv_heads, int head_dim, int page_size, float scale, int window, int dtype,
                                    float* workspace, hipStream_t stream) {
  if (items <= 0 || longest <= 0) return SE_OK;
  if (head_dim <= 0 || head_dim % 8 || head_dim > 512) return SE_ERR_SHAPE;
  if (kv_heads <= 0 || heads % kv_heads || page_size <= 0 || page_size % 8) return SE_ERR_SHAPE;
  if (kind == SE_CACHE_FP4 && (head_dim % 32 || page_size % 32)) return SE_ERR_SHAPE;
  if (kind != SE_CACHE_FP4 && kind != (dtype == SE_F32 ? SE_CACHE_F32 : SE_CACHE_BF16)) return SE_ERR_SHAPE;
  if (kv_heads > 65535 || items > 65535) return SE_ERR_SHAPE;
  if (!(scale > 0.f)) return SE_ERR_SHAPE;      // masked scores are -inf before it is applied
  const int64_t most_rows = static_cast<int64_t>(most_new) * (heads / kv_heads);
  if (weights_on_matrix_cores(head_dim, most_rows, dtype)) {
    const int splits = se_attention_weights_splits(items, longest, most_new, heads, kv_heads, head_dim, dtype);
    if (splits > 1 && workspace == nullptr) return SE_ERR_SHAPE;
#define SE_WEIGHTS_MFMA(DS, KIND)                                                                                   \
  launch_weights_mfma<DS, KIND>(q, q_stride, cache, block_table, bt_stride, item_meta, items, longest,              \
                                most_new, lse, previous, out, heads, kv_heads, page_size, scale, window, splits, workspace, stream)
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
  const size_t shared = static_cast<size_t>(GENERIC_WAVES * GENERIC_ROWS) * head_dim * sizeof(float);      // 32 KB at most
#define SE_WEIGHTS(T, KIND)                                                                                      \
  attention_weights_generic_kernel<T, KIND><<<grid, GENERIC_WAVES * SE_WAVE, shared, stream>>>(                  \
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
