// Decode attention of rows that share prefixes, over the paged cache in the model's type.
//
// Row b attends over positions 0..p_b of its cache layer. Rows of a group begin with the same tokens; these are read
// once for all of them, each row's own tokens by the row:
//   prefix_attend_kernel  a workgroup takes 16 queries (row, head) of a group and one KV head and a part of the
//                         prefix's tokens, and leaves the unnormalised sum, the maximum and the sum of weights;
//   prefix_decode_kernel  a workgroup takes one row and KV head and 1024 of the row's own tokens, rotates and appends
//                         the new one, and joins what it has with the prefix's parts (a row with several chunks: the
//                         workgroup that ends last does).
// Both walk tokens 32 (fp32: 16) at a time, a wave each, with a running maximum and sum:
//   S^T = K Q^T, bf16: v_mfma_f32_16x16x32_bf16 on keys as they lie in memory, with the rotated query, already scaled,
//   as two bf16 parts (2^-17 of an element together);
//   O^T = V^T P^T with P as two bf16 parts; values are turned to the operand's order by one byte permutation for two
//   of them.
// fp32 takes v_mfma_f32_16x16x4_f32, which rounds nothing but the sums. Both products are 16 queries wide; columns
// without a query repeat the last one. A lane's scores are those of the tokens whose values it holds, so P never moves.
#include <atomic>
#include <chrono>

#include "cdb_amd.h"
#include "kv8_common.h"
#include "kv8_host.h"

namespace cdb {

constexpr int kWaves = 4;
constexpr int kChunk = 1024;     // own tokens of a workgroup
constexpr int kMaxChunks = 64;   // of a row; longer contexts take longer chunks
constexpr int kMaxParts = CDB_PREFIX_MAX_PARTS;  // of a prefix
constexpr int kColumns = 16;     // queries of a product
static_assert(kMaxParts <= 64, "a lane weighs a part");

struct PrefixParams {
  const void *q, *k_new, *v_new;
  void *k_pool, *v_pool;
  int64_t layer_stride, pool_blocks;
  const int32_t *cache_layer, *block_table, *table_row, *seqlens;
  int32_t cache_layer0, num_layers, table_rows, table_width, max_positions, bs_log2;
  const float *cos, *sin;
  const void *q_bias, *k_bias;
  const int32_t *listed, *groups, *items, *row_info;
  int32_t num_listed, num_groups, num_items;
  void* out;
  float* shared;   // [items][KV heads][kColumns][D + 2]: O, the maximum and the sum of a prefix's part
  float* partials; // [rows][heads][max_chunks][D + 2]: the same of a chunk of own tokens
  uint64_t* tags;  // [rows][KV heads][slices][max_chunks]: equal to `tag` where this call's partials are whole
  uint64_t tag;
  int32_t max_chunks, num_rows, num_heads, num_kv_heads, group, slices;
  float scale_log2;
  int64_t q_stride, kv_stride;
  bool vec;
};

// Where one KV head's tokens of a table row lie, 16 at a time.
struct Tokens {
  const char *k, *v;  // of the cache layer and head
  const int32_t* table;
  int64_t pool_blocks, row_bytes;
  int bs_log2;

  // Byte offset of the 16 tokens from `t` on (a multiple of 16).
  CDB_DEVICE int64_t at(int t, bool& lost) const {
    const int block = table[t >> bs_log2];
    lost = block < 0 || block >= pool_blocks;
    return (((int64_t)(lost ? 0 : block) << bs_log2) + (t & ((1 << bs_log2) - 1))) * row_bytes;
  }
};

// The operands of a step: 2 tiles of 16 tokens in bf16, one in fp32. Lane (r, g) holds token r of the keys, elements
// 32j + 8g.. (fp32: 16j + 4g..), and of the values tokens 4g..4g+3 of each tile, elements r * D / 16 and up.
template <typename T, int D> struct StepRegs;

template <int D> struct StepRegs<bf16_t, D> {
  static constexpr int kTiles = 2, kRuns = D / 32, kWords = D / 32;
  static constexpr int kQueryWords = 2 * kRuns * 64 * 4;  // of LDS: two parts
  u32x4_t k[kTiles][kRuns];
  uint32_t v[4 * kTiles][kWords];

  CDB_DEVICE void load_key(int a, const char* tile, uint32_t token, int g) {
#pragma unroll
    for (int j = 0; j < kRuns; ++j) k[a][j] = *reinterpret_cast<const u32x4_t*>(tile + (token + (32 * j + 8 * g) * 2u));
  }
  CDB_DEVICE void load_value(int i, const char* tile, uint32_t token, int r) {
    const char* p = tile + (token + (uint32_t)r * (D / 8));
    if constexpr (kWords == 3) {  // aligned to 4 bytes
      typedef uint32_t u32x3_t __attribute__((ext_vector_type(3), aligned(4)));
      const u32x3_t x = *reinterpret_cast<const u32x3_t*>(p);
#pragma unroll
      for (int w = 0; w < 3; ++w) v[i][w] = x[w];
    } else {
      Vec<bf16_t, D / 16> x;
      x.load(reinterpret_cast<const bf16_t*>(p));
#pragma unroll
      for (int w = 0; w < kWords; ++w) v[i][w] = x.w[w];
    }
  }
  // Elements d and d + 1 (d even) of column c, scaled already, to LDS.
  static CDB_DEVICE void store_query(uint32_t* to, int c, int d, float x0, float x1) {
    to += ((d >> 5) * 64 + ((d & 31) >> 3) * 16 + c) * 4 + ((d & 7) >> 1);
    const uint32_t y = pack_bf16x2(x0, x1);
    to[0] = y;
    to[kRuns * 64 * 4] = pack_bf16x2(x0 - __uint_as_float(y << 16), x1 - __uint_as_float(y & 0xffff0000u));
  }
  CDB_DEVICE void scores(const uint32_t* query, int lane, f32x4_t* s) const {
#pragma unroll
    for (int a = 0; a < kTiles; ++a) s[a] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 1; p >= 0; --p)
#pragma unroll
      for (int j = 0; j < kRuns; ++j) {
        const bf16x8_t q = *reinterpret_cast<const bf16x8_t*>(query + ((p * kRuns + j) * 64 + lane) * 4);
#pragma unroll
        for (int a = 0; a < kTiles; ++a)
          s[a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, k[a][j]), q, s[a], 0, 0, 0);
      }
  }
  CDB_DEVICE void accumulate(const f32x4_t* p, f32x4_t* acc) const {
    union { uint32_t w[4]; bf16x8_t v; } hi, lo;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float x = p[i >> 2][i & 3], y = p[i >> 2][(i & 3) + 1];
      hi.w[i >> 1] = pack_bf16x2(x, y);
      lo.w[i >> 1] = pack_bf16x2(x - __uint_as_float(hi.w[i >> 1] << 16),
                                 y - __uint_as_float(hi.w[i >> 1] & 0xffff0000u));
    }
#pragma unroll
    for (int m = 0; m < D / 16; ++m) {
      union { uint32_t w[4]; bf16x8_t v; } x;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x.w[i] = __builtin_amdgcn_perm(v[2 * i + 1][m >> 1], v[2 * i][m >> 1], m & 1 ? 0x07060302u : 0x05040100u);
      acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.v, lo.v, acc[m], 0, 0, 0);
      acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.v, hi.v, acc[m], 0, 0, 0);
    }
  }
};

template <int D> struct StepRegs<float, D> {
  static constexpr int kTiles = 1, kRuns = D / 16, kWords = D / 16;
  static constexpr int kQueryWords = kRuns * 64 * 4;
  f32x4_t k[kTiles][kRuns];
  float v[4][kWords];

  CDB_DEVICE void load_key(int a, const char* tile, uint32_t token, int g) {
#pragma unroll
    for (int j = 0; j < kRuns; ++j) k[a][j] = *reinterpret_cast<const f32x4_t*>(tile + (token + (16 * j + 4 * g) * 4u));
  }
  CDB_DEVICE void load_value(int i, const char* tile, uint32_t token, int r) {
    Vec<float, kWords> x;
    x.load(reinterpret_cast<const float*>(tile + (token + (uint32_t)r * (D / 4))));
#pragma unroll
    for (int w = 0; w < kWords; ++w) v[i][w] = x.get(w);
  }
  static CDB_DEVICE void store_query(uint32_t* to, int c, int d, float x0, float x1) {
    to += ((d >> 4) * 64 + ((d & 15) >> 2) * 16 + c) * 4 + (d & 3);
    to[0] = __float_as_uint(x0);
    to[1] = __float_as_uint(x1);
  }
  CDB_DEVICE void scores(const uint32_t* query, int lane, f32x4_t* s) const {
    s[0] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kRuns; ++j) {
      const f32x4_t q = *reinterpret_cast<const f32x4_t*>(query + (j * 64 + lane) * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[0][j][i], q[i], s[0], 0, 0, 0);
    }
  }
  CDB_DEVICE void accumulate(const f32x4_t* p, f32x4_t* acc) const {
#pragma unroll
    for (int m = 0; m < D / 16; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][m], p[0][i], acc[m], 0, 0, 0);
  }
};

// A wave's running maximum and sum (of query r, over the lane's own tokens) and O^T: rows are elements, row x of
// product m element x * D / 16 + m.
template <typename T, int D> struct Walk {
  static constexpr int kTiles = StepRegs<T, D>::kTiles;
  float top, sum;
  bool missing;
  f32x4_t acc[D / 16];

  CDB_DEVICE void start() {
    top = -INFINITY;
    sum = 0.f;
    missing = false;
#pragma unroll
    for (int m = 0; m < D / 16; ++m) acc[m] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  }
  // Scores, in units of log2, to weights. Tokens outside [lo, hi) of a tile have none.
  CDB_DEVICE void weigh(f32x4_t* s, const int* lo, const int* hi, int g) {
    float most = top;
#pragma unroll
    for (int a = 0; a < kTiles; ++a) {
      if (lo[a] > 0 || hi[a] < 16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[a][i] = 4 * g + i >= lo[a] && 4 * g + i < hi[a] ? s[a][i] : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) most = fmaxf(most, s[a][i]);
    }
    most = column_max(most);
    if (__any(most > top)) {
      const float keep = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top - most);  // the first finds zeros
      sum *= keep;
#pragma unroll
      for (int m = 0; m < D / 16; ++m) acc[m] *= keep;
      top = most;
    }
    const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int a = 0; a < kTiles; ++a)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[a][i] = __builtin_amdgcn_exp2f(s[a][i] - from);
        sum += s[a][i];
      }
  }
  // Tokens [lo, hi), step `first` of every `stride`.
  CDB_DEVICE void tokens(const Tokens& at, const uint32_t* query, int lo, int hi, int first, int stride) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    if (lo >= hi) return;
    const int t0 = lo >> 4, tiles = ((hi + 15) >> 4) - t0;
    const uint32_t row_bytes = (uint32_t)at.row_bytes;
    for (int window = 0; window < tiles; window += 64) {
      const int count = min(64, tiles - window);
      int64_t where = 0;
      bool lost = false;
      if (lane < count) where = at.at((t0 + window + lane) * 16, lost);
      missing = missing || __ballot(lost) != 0;
      auto offset = [&](int j) __attribute__((always_inline)) -> int64_t {
        const uint32_t a = __builtin_amdgcn_readlane((int)(uint32_t)where, j);
        const uint32_t b = __builtin_amdgcn_readlane((int)(uint32_t)(where >> 32), j);
        return (int64_t)(((uint64_t)b << 32) | a);
      };
      StepRegs<T, D> x;
      int from[kTiles], to[kTiles];
      // Of a tile that sticks out of the range the nearest token inside stands for those outside; the last step's
      // second tile may be missing: the first stands in for it.
      auto bounds = [&](int step, int a, int& b0, int& b1) __attribute__((always_inline)) -> int {
        const int j = min(kTiles * step + a, count - 1), t = (t0 + window + j) * 16;
        b0 = max(lo - t, 0);
        b1 = min(hi - t, 16);
        return j;
      };
      auto load_keys = [&](int step) __attribute__((always_inline)) {
#pragma unroll
        for (int a = 0; a < kTiles; ++a) {
          int b0, b1;
          const int64_t tile = offset(bounds(step, a, b0, b1));
          x.load_key(a, at.k + tile, (uint32_t)min(max(r, b0), b1 - 1) * row_bytes, g);
        }
      };
      auto load_values = [&](int step) __attribute__((always_inline)) {
#pragma unroll
        for (int a = 0; a < kTiles; ++a) {
          int b0, b1;
          const int64_t tile = offset(bounds(step, a, b0, b1));
#pragma unroll
          for (int i = 0; i < 4; ++i)
            x.load_value(4 * a + i, at.v + tile, (uint32_t)min(max(4 * g + i, b0), b1 - 1) * row_bytes, r);
        }
      };
      const int steps = (count + kTiles - 1) / kTiles;
      if (first < steps) {
        load_keys(first);
        __builtin_amdgcn_sched_barrier(0);  // keys before values, as in the steps: the waits count on it
        load_values(first);
      }
      for (int step = first; step < steps; step += stride) {
        // The loads ahead repeat the step at the end: a branch around them would make the wait for this step's
        // values one for the next keys too.
        const int ahead = step + stride < steps ? step + stride : step;
        f32x4_t s[kTiles];
        x.scores(query, lane, s);
        load_keys(ahead);
#pragma unroll
        for (int a = 0; a < kTiles; ++a) {
          bounds(step, a, from[a], to[a]);
          if (kTiles * step + a >= count) to[a] = 0;
        }
        weigh(s, from, to, g);
        x.accumulate(s, acc);
        __builtin_amdgcn_sched_barrier(0);
        load_values(ahead);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  // O, the maximum and the sum of each column to LDS: [column][D + 4].
  CDB_DEVICE void leave(float* to, int cols) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    float total = column_sum(sum);
    if (missing) total = NAN;
    if (r >= cols) return;
    float* mine = to + r * (D + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int m = 0; m < D / 16; m += 2)
        *reinterpret_cast<f32x2_t*>(mine + (4 * g + i) * (D / 16) + m) = (f32x2_t){acc[m][i], acc[m + 1][i]};
    if (g == 0) {
      mine[D] = total == 0.f ? -INFINITY : top;  // no token yet, or none above -infinity
      mine[D + 1] = total;
    }
  }
};

// Query head `head` of row b, rotated and scaled, as column c of the query operand: a wave's work.
template <typename T, int D, int STYLE>
CDB_DEVICE void turn_query(const PrefixParams& P, uint32_t* query, int c, int b, int head, int p) {
  const int lane = threadIdx.x & 63, d = min(2 * lane, D - 2);
  const int64_t angle = STYLE == 0 ? 0 : (int64_t)p * (D / 2);
  const T* bias = static_cast<const T*>(P.q_bias);
  float x[2];
  load_rotated<T, D, STYLE, 2>(static_cast<const T*>(P.q) + b * P.q_stride + (int64_t)head * D,
                               bias == nullptr ? nullptr : bias + (int64_t)head * D, P.cos + angle, P.sin + angle, d,
                               P.vec, x);
  if (2 * lane < D) StepRegs<T, D>::store_query(query, c, d, mul_rn(x[0], P.scale_log2), mul_rn(x[1], P.scale_log2));
}

// What a row's launch arguments come to: whether it is padding, or has none of its own that can be served.
struct RowPlace {
  int p, layer, trow, own;  // own: the first of its own tokens
  bool bad;
};
template <int STYLE> CDB_DEVICE RowPlace place_of_row(const PrefixParams& P, int b) {
  RowPlace x;
  x.p = P.seqlens[b];
  x.layer = P.cache_layer0 + (P.cache_layer == nullptr ? 0 : P.cache_layer[b]);
  x.trow = P.table_row == nullptr ? b : P.table_row[b];
  x.own = P.row_info[4 * b + 1];
  x.bad = (int64_t)x.p >= ((int64_t)P.table_width << P.bs_log2) || (STYLE != 0 && x.p >= P.max_positions) ||
          x.layer < 0 || x.layer >= P.num_layers || x.trow < 0 || x.trow >= P.table_rows || x.own < 0 || x.own > x.p;
  return x;
}
template <typename T, int D> CDB_DEVICE Tokens tokens_of(const PrefixParams& P, int layer, int trow, int kvh) {
  Tokens x;
  const int64_t base = ((int64_t)layer * P.layer_stride + (int64_t)kvh * D) * (int64_t)sizeof(T);
  x.k = static_cast<const char*>(P.k_pool) + base;
  x.v = static_cast<const char*>(P.v_pool) + base;
  x.table = P.block_table + (int64_t)trow * P.table_width;
  x.pool_blocks = P.pool_blocks;
  x.row_bytes = (int64_t)P.num_kv_heads * D * (int64_t)sizeof(T);
  x.bs_log2 = P.bs_log2;
  return x;
}

template <typename T, int D, int STYLE>
__global__ void __launch_bounds__(64 * kWaves) prefix_attend_kernel(PrefixParams P) {
  __shared__ __align__(16) uint32_t query[StepRegs<T, D>::kQueryWords];
  __shared__ __align__(16) float join[kWaves * kColumns * (D + 4)];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int item = blockIdx.x / P.num_kv_heads, kvh = blockIdx.x - item * P.num_kv_heads;
  const int n = P.items[4 * item], q0 = P.items[4 * item + 1];
  if (n < 0 || n >= P.num_groups) return;  // no item
  const int first = P.groups[4 * n], count = P.groups[4 * n + 1], length = P.groups[4 * n + 2];
  if (count <= 0 || count > P.num_listed || first < 0 || first > P.num_listed - count) return;
  const int64_t queries = (int64_t)count * P.group;
  if (q0 < 0 || q0 >= queries) return;
  const int cols = (int)min((int64_t)kColumns, queries - q0);
  int lo = P.items[4 * item + 2], hi = P.items[4 * item + 3];
  const int leader = P.listed[first];
  int layer = -1, trow = -1;
  if (leader >= 0 && leader < P.num_rows) {
    layer = P.cache_layer0 + (P.cache_layer == nullptr ? 0 : P.cache_layer[leader]);
    trow = P.table_row == nullptr ? leader : P.table_row[leader];
  }
  const bool bad = layer < 0 || layer >= P.num_layers || trow < 0 || trow >= P.table_rows || lo < 0 || hi > length ||
                   (int64_t)length > ((int64_t)P.table_width << P.bs_log2);
  for (int c = wave; c < kColumns; c += kWaves) {
    const int at = q0 + min(c, cols - 1);
    const int b = P.listed[first + at / P.group];
    const int p = b >= 0 && b < P.num_rows ? P.seqlens[b] : -1;
    if (p >= 0 && (STYLE == 0 || p < P.max_positions))
      turn_query<T, D, STYLE>(P, query, c, b, kvh * P.group + at % P.group, p);
    else if (2 * (threadIdx.x & 63) < D)  // a padding row, or one that gets NaN
      StepRegs<T, D>::store_query(query, c, 2 * (threadIdx.x & 63), 0.f, 0.f);
  }
  __syncthreads();
  Walk<T, D> walk;
  walk.start();
  if (bad) walk.missing = true;
  else walk.tokens(tokens_of<T, D>(P, layer, trow, kvh), query, lo, hi, wave, kWaves);
  walk.leave(join + wave * cols * (D + 4), cols);
  __syncthreads();
  float* to = P.shared + ((int64_t)item * P.num_kv_heads + kvh) * kColumns * (D + 2);
  for (int i = threadIdx.x; i < cols * D; i += 64 * kWaves) {
    const int c = i / D, d = i - c * D;
    float m[kWaves], most = -INFINITY, o = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      m[w] = join[(w * cols + c) * (D + 4) + D];
      most = fmaxf(most, m[w]);
    }
    const float from = most == -INFINITY ? 0.f : most;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float* x = join + (w * cols + c) * (D + 4);
      const float f = __builtin_amdgcn_exp2f(m[w] - from);
      o = fmaf(f, x[d], o);
      l = fmaf(f, x[D + 1], l);
    }
    to[c * (D + 2) + d] = o;
    if (d == 0) {
      to[c * (D + 2) + D] = most;
      to[c * (D + 2) + D + 1] = l;
    }
  }
}

template <typename T, int D, int STYLE>
__global__ void __launch_bounds__(64 * kWaves) prefix_decode_kernel(PrefixParams P) {
  __shared__ __align__(16) uint32_t query[StepRegs<T, D>::kQueryWords];
  __shared__ __align__(16) T fresh[2][D];
  __shared__ float weights[kColumns][kMaxChunks + kMaxParts];
  __shared__ bool all_marked;
  extern __shared__ __align__(16) float join[];
  constexpr int kPlace = D + 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.x / P.num_kv_heads, kvh = blockIdx.x - b * P.num_kv_heads;
  const int chunk = blockIdx.y;
  RowPlace row = place_of_row<STYLE>(P, b);
  const int p = row.p;
  T* out = static_cast<T*>(P.out) + ((int64_t)b * P.num_heads + (int64_t)kvh * P.group) * D;
  // The row's queries within its group, and the prefix's parts.
  const int n0 = P.row_info[4 * b], item0 = P.row_info[4 * b + 2], parts = P.row_info[4 * b + 3];
  if (parts == 0) {
    row.bad = row.bad || row.own != 0;
  } else if (!row.bad) {
    const int64_t last = item0 + (((int64_t)n0 + P.group - 1) / kColumns + 1) * parts;  // behind the row's last item
    if (parts < 0 || parts > kMaxParts || n0 < 0 || item0 < 0 || last > P.num_items) {
      row.bad = true;
    } else {
      const int n = P.items[4 * item0], first = n >= 0 && n < P.num_groups ? P.groups[4 * n] : -1;
      const int leader = first >= 0 && first < P.num_listed ? P.listed[first] : -1;
      row.bad = leader < 0 || leader >= P.num_rows ||
                (P.cache_layer != nullptr && P.cache_layer[leader] != P.cache_layer[b]);
    }
  }
  if (p < 0 || row.bad) {
    if (chunk == 0)
      for (int i = threadIdx.x; i < P.group * D; i += 64 * kWaves) Elem<T>::store(out + i, p < 0 ? 0.f : NAN);
    return;
  }
  // A row with more chunks than the workspace has partials for takes longer ones.
  const int own = p - row.own;  // cached tokens of its own, the new one besides
  const int pieces = max(1, (own + kChunk - 1) / kChunk);
  const int most_chunks = min(P.max_chunks, kMaxChunks);
  const int length = kChunk * ((pieces + most_chunks - 1) / most_chunks);
  const int chunks = max(1, (own + length - 1) / length);
  if (chunk >= chunks) return;
  const int lo = row.own + chunk * length, hi = min(p, lo + length);
  const bool ends = chunk == chunks - 1;  // the new token is in this chunk
  const Tokens at = tokens_of<T, D>(P, row.layer, row.trow, kvh);

  for (int slice = 0; slice < P.group; slice += kColumns) {
    const int cols = min(kColumns, P.group - slice);
    for (int c = wave; c < kColumns; c += kWaves)
      turn_query<T, D, STYLE>(P, query, c, b, kvh * P.group + slice + min(c, cols - 1), p);
    Walk<T, D> walk;
    walk.start();
    if (ends && wave == kWaves - 1) {
      const int lane = threadIdx.x & 63, d = min(2 * lane, D - 2);
      const int64_t angle = STYLE == 0 ? 0 : (int64_t)p * (D / 2), from = b * P.kv_stride + (int64_t)kvh * D;
      const T* bias = static_cast<const T*>(P.k_bias);
      float x[2], y[2];
      load_f32<T, 2>(static_cast<const T*>(P.v_new) + from + d, y, P.vec);
      load_rotated<T, D, STYLE, 2>(static_cast<const T*>(P.k_new) + from, bias == nullptr ? nullptr : bias + kvh * D,
                                   P.cos + angle, P.sin + angle, d, P.vec, x);
      bool lost = false;
      const int64_t tile = at.at(p & ~15, lost) + (int64_t)(p & 15) * at.row_bytes;
      walk.missing = lost;
      Vec<T, 2> k, v;
      k.set_pair(0, x[0], x[1]);
      v.set_pair(0, y[0], y[1]);
      if (2 * lane < D) {
        k.store(&fresh[0][d]);
        v.store(&fresh[1][d]);
        if (!lost && slice == 0) {
          k.store(reinterpret_cast<T*>(const_cast<char*>(at.k) + tile) + d);
          v.store(reinterpret_cast<T*>(const_cast<char*>(at.v) + tile) + d);
        }
      }
    }
    __syncthreads();
    if (ends && wave == kWaves - 1) {
      // The new token as the first of a tile.
      const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
      StepRegs<T, D> x;
#pragma unroll
      for (int a = 0; a < StepRegs<T, D>::kTiles; ++a) x.load_key(a, reinterpret_cast<const char*>(fresh[0]), 0, g);
#pragma unroll
      for (int i = 0; i < 4 * StepRegs<T, D>::kTiles; ++i)
        x.load_value(i, reinterpret_cast<const char*>(fresh[1]), 0, r);
      f32x4_t s[StepRegs<T, D>::kTiles];
      x.scores(query, lane, s);
      const int from[2] = {0, 0}, to[2] = {1, 0};
      walk.weigh(s, from, to, g);
      x.accumulate(s, walk.acc);
    }
    walk.tokens(at, query, lo, hi, wave, kWaves);
    walk.leave(join + wave * cols * kPlace, cols);
    __syncthreads();

    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t shared_stride = (int64_t)P.num_kv_heads * kColumns * (D + 2);
    auto shared_of = [&](int c) __attribute__((always_inline)) -> const float* {
      const int n = n0 + slice + c;
      return P.shared + (((int64_t)item0 + n / kColumns * parts) * P.num_kv_heads + kvh) * kColumns * (D + 2) +
             n % kColumns * (D + 2);
    };
    if (chunks > 1) {
      for (int i = tid; i < cols * D; i += 64 * kWaves) {
        const int c = i / D, d = i - c * D;
        float m[kWaves], most = -INFINITY, o = 0.f, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          m[w] = join[(w * cols + c) * kPlace + D];
          most = fmaxf(most, m[w]);
        }
        const float from = most == -INFINITY ? 0.f : most;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float* x = join + (w * cols + c) * kPlace;
          const float f = __builtin_amdgcn_exp2f(m[w] - from);
          o = fmaf(f, x[d], o);
          l = fmaf(f, x[D + 1], l);
        }
        const int h = kvh * P.group + slice + c;
        float* to = P.partials + (((int64_t)b * P.num_heads + h) * P.max_chunks + chunk) * (D + 2);
        __hip_atomic_store(to + d, o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (d == 0) {
          __hip_atomic_store(to + D, most, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          __hip_atomic_store(to + D + 1, l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
      }
      // The workgroup that finds every chunk of the row marked whole joins them, in order. Partials and marks
      // are stored past the XCD's cache and each store is waited for, and a workgroup marks its own chunk
      // before it looks: whichever marks last sees all. (Several may; they store the same values.) The marks
      // are taken back for the next launch of a captured graph, which has the same tag.
      uint64_t* tags = P.tags + (((int64_t)b * P.num_kv_heads + kvh) * P.slices + slice / kColumns) * P.max_chunks;
      __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (wave == 0) {
        if (lane == 0) __hip_atomic_store(tags + chunk, P.tag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const bool whole =
            lane >= chunks || __hip_atomic_load(tags + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == P.tag;
        const bool all = __ballot(whole) == ~0ull;
        if (lane == 0) all_marked = all;
      }
      __syncthreads();
      if (!all_marked) {
        if (slice + kColumns < P.group) __syncthreads();
        continue;
      }
    }
    // Weights of the waves, or of the chunks, and of the prefix's parts, a wave a column.
    const int mine = chunks > 1 ? chunks : kWaves;
    const float* rows = P.partials + ((int64_t)b * P.num_heads + kvh * P.group + slice) * P.max_chunks * (D + 2);
    for (int c = wave; c < cols; c += kWaves) {
      float m0 = -INFINITY, l0 = 0.f, m1 = -INFINITY, l1 = 0.f;
      if (lane < mine) {
        if (chunks > 1) {
          const float* x = rows + ((int64_t)c * P.max_chunks + lane) * (D + 2) + D;
          m0 = __hip_atomic_load(x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          l0 = __hip_atomic_load(x + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        } else {
          m0 = join[(lane * cols + c) * kPlace + D];
          l0 = join[(lane * cols + c) * kPlace + D + 1];
        }
      }
      if (lane < parts) {
        const float* x = shared_of(c) + lane * shared_stride + D;
        m1 = x[0];
        l1 = x[1];
      }
      const float most = wave_max(fmaxf(m0, m1)), from = most == -INFINITY ? 0.f : most;
      const float f0 = __builtin_amdgcn_exp2f(m0 - from), f1 = __builtin_amdgcn_exp2f(m1 - from);
      const float total = wave_sum(fmaf(f0, l0, f1 * l1));
      if (lane < mine) weights[c][lane] = f0 / total;
      if (lane < parts) weights[c][kMaxChunks + lane] = f1 / total;
    }
    __syncthreads();
    for (int i = tid; i < cols * (D / 2); i += 64 * kWaves) {
      const int c = i / (D / 2), d = 2 * (i - c * (D / 2));
      float o0 = 0.f, o1 = 0.f;
      const float* x = shared_of(c) + d;
      for (int n = 0; n < parts; ++n) {
        const f32x2_t y = *reinterpret_cast<const f32x2_t*>(x + n * shared_stride);
        o0 = fmaf(weights[c][kMaxChunks + n], y[0], o0);
        o1 = fmaf(weights[c][kMaxChunks + n], y[1], o1);
      }
      for (int n = 0; n < mine; ++n) {
        float y0, y1;
        if (chunks > 1) {
          const uint64_t y = __hip_atomic_load(
              reinterpret_cast<const uint64_t*>(rows + ((int64_t)c * P.max_chunks + n) * (D + 2) + d), __ATOMIC_RELAXED,
              __HIP_MEMORY_SCOPE_AGENT);
          y0 = __uint_as_float((uint32_t)y);
          y1 = __uint_as_float((uint32_t)(y >> 32));
        } else {
          y0 = join[(n * cols + c) * kPlace + d];
          y1 = join[(n * cols + c) * kPlace + d + 1];
        }
        o0 = fmaf(weights[c][n], y0, o0);
        o1 = fmaf(weights[c][n], y1, o1);
      }
      T* to = out + (int64_t)(slice + c) * D + d;
      Elem<T>::store(to, o0);
      Elem<T>::store(to + 1, o1);
    }
    if (chunks > 1 && tid < chunks) {
      uint64_t* tags = P.tags + (((int64_t)b * P.num_kv_heads + kvh) * P.slices + slice / kColumns) * P.max_chunks;
      __hip_atomic_store(tags + tid, (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (slice + kColumns < P.group) __syncthreads();
  }
}

template <typename T, int D, int STYLE> static int prefix_style(const PrefixParams& P, hipStream_t stream) {
  const dim3 wg(64 * kWaves);
  if (P.num_items > 0) {
    prefix_attend_kernel<T, D, STYLE><<<dim3((unsigned)(P.num_items * P.num_kv_heads)), wg, 0, stream>>>(P);
    if (hipGetLastError() != hipSuccess) return CDB_ERR_HIP;
  }
  const int64_t most = ((int64_t)P.table_width << P.bs_log2) / kChunk + 1;
  const dim3 grid((unsigned)(P.num_rows * P.num_kv_heads), (unsigned)min((int64_t)P.max_chunks, most));
  const size_t lds = sizeof(float) * kWaves * min(P.group, kColumns) * (D + 4);
  prefix_decode_kernel<T, D, STYLE><<<grid, wg, lds, stream>>>(P);
  return hipGetLastError() == hipSuccess ? CDB_OK : CDB_ERR_HIP;
}
template <typename T, int D> static int prefix_dim(const PrefixParams& P, int style, hipStream_t stream) {
  if (style == 0) return prefix_style<T, D, 0>(P, stream);
  return style == 1 ? prefix_style<T, D, 1>(P, stream) : prefix_style<T, D, 2>(P, stream);
}
template <typename T> static int prefix_type(const PrefixParams& P, int dim, int style, hipStream_t stream) {
  switch (dim) {
    case 64: return prefix_dim<T, 64>(P, style, stream);
    case 96: return prefix_dim<T, 96>(P, style, stream);
    case 128: return prefix_dim<T, 128>(P, style, stream);
    default: return CDB_ERR_UNSUPPORTED;
  }
}

// Bytes of one row's partials and marks for one chunk.
static int64_t chunk_bytes(int32_t num_heads, int32_t num_kv_heads, int32_t head_dim) {
  const int64_t slices = ((int64_t)num_heads / num_kv_heads + kColumns - 1) / kColumns;
  return (int64_t)num_heads * (head_dim + 2) * 4 + num_kv_heads * slices * 8;
}
// Bytes of the partials of prefixes, a multiple of 16.
static int64_t shared_bytes(int64_t num_items, int32_t num_kv_heads, int32_t head_dim) {
  return num_items * num_kv_heads * kColumns * (head_dim + 2) * 4;
}

// A tag that no other call of this process has, and that memory does not hold by chance.
static uint64_t next_tag() {
  static std::atomic<uint64_t> calls{(uint64_t)std::chrono::steady_clock::now().time_since_epoch().count() << 20};
  uint64_t z = calls.fetch_add(1, std::memory_order_relaxed) * 0x9e3779b97f4a7c15ull;
  z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
  z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
  return (z ^ (z >> 31)) | 1;
}

}  // namespace cdb

extern "C" int64_t cdb_prefix_decode_workspace_bytes(int32_t num_rows, int32_t num_items, int32_t num_heads,
                                                     int32_t num_kv_heads, int32_t head_dim, int32_t max_own) {
  if (num_rows < 0 || num_items < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      head_dim <= 0 || max_own <= 0)
    return -1;
  const int64_t chunks = min(((int64_t)max_own + cdb::kChunk - 1) / cdb::kChunk, (int64_t)cdb::kMaxChunks);
  return cdb::shared_bytes(num_items, num_kv_heads, head_dim) +
         max((int64_t)num_rows, (int64_t)1) * chunks * cdb::chunk_bytes(num_heads, num_kv_heads, head_dim);
}

extern "C" int cdb_prefix_decode_attention(
    const void* q, const void* k_new, const void* v_new, void* k_pool, void* v_pool, int64_t layer_stride,
    int32_t num_cache_layers, int64_t pool_blocks, const int32_t* cache_layer, int32_t cache_layer0,
    const int32_t* block_table, const int32_t* table_row, int32_t table_rows, int32_t table_width,
    const int32_t* seqlens, const float* rope_cos, const float* rope_sin, int32_t rope_style, int32_t max_positions,
    const void* q_bias, const void* k_bias, const int32_t* listed, int32_t num_listed, const int32_t* groups,
    int32_t num_groups, const int32_t* items, int32_t num_items, const int32_t* row_info, void* out, void* workspace,
    int64_t workspace_bytes, int32_t num_rows, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t block_size, float scale, int64_t q_stride, int64_t kv_stride, int32_t dtype, hipStream_t stream) {
  using namespace cdb;
  if (rope_style < 0 || rope_style > 2) return CDB_ERR_UNSUPPORTED;
  if (dtype != CDB_DTYPE_F32 && dtype != CDB_DTYPE_BF16) return CDB_ERR_UNSUPPORTED;
  if (head_dim != 64 && head_dim != 96 && head_dim != 128) return CDB_ERR_UNSUPPORTED;
  if (num_rows < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || table_rows <= 0 ||
      table_width <= 0 || num_cache_layers <= 0 || pool_blocks <= 0 || pool_blocks > 0x7fffffffll || num_listed < 0 ||
      num_groups < 0 || num_items < 0)
    return CDB_ERR_SHAPE;
  if (block_size < 16 || (block_size & (block_size - 1)) != 0) return CDB_ERR_SHAPE;
  if (num_rows == 0) return CDB_OK;
  if (q == nullptr || k_new == nullptr || v_new == nullptr || k_pool == nullptr || v_pool == nullptr ||
      block_table == nullptr || seqlens == nullptr || row_info == nullptr || out == nullptr || workspace == nullptr)
    return CDB_ERR_NULL;
  if (rope_style != 0 && (rope_cos == nullptr || rope_sin == nullptr)) return CDB_ERR_NULL;
  if (num_items != 0 && (listed == nullptr || groups == nullptr || items == nullptr)) return CDB_ERR_NULL;
  if (rope_style != 0 && max_positions <= 0) return CDB_ERR_SHAPE;
  const int size = dtype == CDB_DTYPE_F32 ? 4 : 2;
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  if (row * size * 16 > 0x7fffffffll || (int64_t)table_width * block_size > (1ll << 30)) return CDB_ERR_SHAPE;
  if (layer_stride < 0 || (num_cache_layers > 1 && layer_stride < pool_blocks * block_size * row)) return CDB_ERR_SHAPE;
  if (table_row == nullptr && table_rows < num_rows) return CDB_ERR_SHAPE;
  if ((int64_t)num_rows * num_kv_heads > 0x7fffffffll || (int64_t)num_items * num_kv_heads > 0x7fffffffll)
    return CDB_ERR_SHAPE;
  if (!(scale > 0.f) || !(scale < INFINITY)) return CDB_ERR_SHAPE;
  if (q_stride == 0) q_stride = (int64_t)num_heads * head_dim;
  if (kv_stride == 0) kv_stride = row;
  if (q_stride < (int64_t)num_heads * head_dim || kv_stride < row) return CDB_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || reinterpret_cast<uintptr_t>(k_pool) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(v_pool) % 16 != 0 || layer_stride * size % 16 != 0)
    return CDB_ERR_SHAPE;
  const int64_t left = workspace_bytes - shared_bytes(num_items, num_kv_heads, head_dim);
  const int64_t chunks = left < 0 ? 0 : min(left / (num_rows * chunk_bytes(num_heads, num_kv_heads, head_dim)),
                                            (int64_t)kMaxChunks);
  if (chunks < 1) return CDB_ERR_CAPACITY;
  PrefixParams P{};
  P.q = q; P.k_new = k_new; P.v_new = v_new; P.k_pool = k_pool; P.v_pool = v_pool;
  P.layer_stride = layer_stride; P.num_layers = num_cache_layers; P.pool_blocks = pool_blocks;
  P.cache_layer = cache_layer; P.cache_layer0 = cache_layer0;
  P.block_table = block_table; P.table_row = table_row; P.table_rows = table_rows; P.table_width = table_width;
  P.seqlens = seqlens; P.cos = rope_cos; P.sin = rope_sin;
  P.max_positions = rope_style != 0 ? max_positions : 0;
  P.bs_log2 = __builtin_ctz(block_size);
  P.q_bias = q_bias; P.k_bias = k_bias;
  P.listed = listed; P.groups = groups; P.items = items; P.row_info = row_info;
  P.num_listed = num_listed; P.num_groups = num_groups; P.num_items = num_items;
  P.out = out; P.shared = static_cast<float*>(workspace);
  P.partials = P.shared + shared_bytes(num_items, num_kv_heads, head_dim) / 4;
  P.max_chunks = (int32_t)chunks;
  P.slices = (num_heads / num_kv_heads + kColumns - 1) / kColumns;
  P.tags = reinterpret_cast<uint64_t*>(P.partials + (int64_t)num_rows * num_heads * chunks * (head_dim + 2));
  P.tag = next_tag();
  P.num_rows = num_rows; P.num_heads = num_heads; P.num_kv_heads = num_kv_heads; P.group = num_heads / num_kv_heads;
  P.scale_log2 = scale * 1.4426950408889634f;
  P.q_stride = q_stride; P.kv_stride = kv_stride;
  P.vec = kv8_aligned(size, {q, k_new, v_new, q_bias, k_bias, rope_cos, rope_sin}, {q_stride, kv_stride});
  return dtype == CDB_DTYPE_F32 ? prefix_type<float>(P, head_dim, rope_style, stream)
                                : prefix_type<bf16_t>(P, head_dim, rope_style, stream);
}
