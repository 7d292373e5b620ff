// Decode attention of rows that share prefixes, over the paged cache in the model's type.
//
// Row b attends over positions 0..p_b of its cache layer. Rows of a group begin with the same tokens; these are read
// once for 16 or 128 of the group's queries of a KV head, each row's own tokens by the row, and what the two leave is
// joined: with m, l and O a part's
// largest score, sum of weights and weighted sum of values, M = max m, out = sum 2^(m - M) O / sum 2^(m - M) l.
//   prefix_attend_kernel  a workgroup takes 16 or 128 queries (row, head) of a group, one KV head and a part of the
//                         prefix's tokens, and leaves m, l and O of each query;
//   prefix_decode_kernel  a workgroup of two waves takes one row and KV head and 1024 of the row's own tokens, rotates
//                         and appends the new one, and joins what it has with the prefix's parts (a row with several
//                         chunks: the workgroup that ends last does).
// Both walk tokens 32 (fp32: 16) at a time, a wave each, with a running maximum and sum:
//   S^T = K Q^T, bf16: v_mfma_f32_16x16x32_bf16 on keys as they lie in memory, with the rotated query, already scaled,
//   as two bf16 parts (2^-16 of an element together);
//   O^T = V^T P^T with P as two bf16 parts; values are turned to the operand's order by one byte permutation for two
//   of them. One part of Q and P each would halve the products and leave 2^-9 of an element, which is what the kernel
//   for rows without prefixes has (paged_decode_attention.hip: queries rounded to bf16 when rotated, weights for their
//   product). Here the result is the formula's on the cached numbers to one rounding, the output's, in any cut.
// fp32 takes v_mfma_f32_16x16x4_f32, which rounds nothing but the sums. Both products are 16 queries wide; columns
// without a query repeat the last one. A lane's scores are those of the tokens whose values it holds, so P never moves.
//
// Bounds, bf16, heads of 128: own tokens, by the bytes: 256 rows x 16 KV heads of 32 to 512 own tokens take 93 us,
// 3.9 TB/s, of the 125 us with 2 x 2048 shared ones, whose part is bound by the products' chain (30 us). 32000 tokens
// shared by 64 rows of 32 heads on 8 KV heads: 84 us, in which a SIMD has matrix work for 27 and vector work (weights
// and their parts) for as much, at two waves that wait for the same steps; the rows' own tokens take 20 more. In fp32,
// 64 rows of 16 heads after 2048 tokens take 31, 47 and 49 us with heads of 64, 96 and 128 (floors 7, 10 and 14); heads
// of 96 keep 144 bytes a lane in scratch there, though nothing spills.

#include "call_tag.h"
#include "cdb_amd.h"
#include "kv8_common.h"
#include "kv8_host.h"

namespace cdb {

constexpr int kRowWaves = 2;     // of a row's
constexpr int kChunk = 1024;     // own tokens of a workgroup
constexpr int kMaxChunks = 64;   // of a row; longer contexts take longer chunks
constexpr int kMaxParts = CDB_PREFIX_MAX_PARTS;  // of a prefix
constexpr int kColumns = 16;     // queries of a product
constexpr int kQueries = CDB_PREFIX_QUERIES;  // of an item
constexpr int kItem = CDB_PREFIX_ITEM;        // words of an item
static_assert(CDB_PREFIX_FEW == kColumns && kQueries == 128, "queries of an item's waves");
// A prefix's workgroup: four waves of the same 16 queries, each with every fourth step, loaded by itself; or four of 32
// queries each on two parts of the tokens, which share a step's loads in LDS. The plan takes the first kind for groups
// of up to 32 queries: 8 groups of 8 (32, 33, 64) queries on 2048 tokens, 16 KV heads, take 41 (64, 74, 121) us with
// their own tokens on the first kind and 50 (74, 76, 106) on the second; one group of 16 (24, 33) on 16000 tokens 43
// (54, 72) and 50 (52, 54); 2 of 8 (24, 64) on 8000, 32 heads on 8, 40 (39, 46) and 38 (40, 43). So the rule, which
// sees neither the tokens nor the KV heads, loses up to 7% for few queries on long prefixes of few KV heads.
template <bool kFew> constexpr int kWaves = kFew ? 4 : 8;
static_assert(kMaxParts <= 64, "a lane weighs a part");

struct PrefixParams {
  const void *q, *k_new, *v_new;
  void *k_pool, *v_pool;
  int64_t layer_stride, pool_blocks;
  const int32_t *cache_layer, *block_table, *table_row, *seqlens;
  int32_t cache_layer0, num_layers, table_rows, table_width, max_positions, bs_log2;
  const float *cos, *sin;
  const void *q_bias, *k_bias;
  const int32_t *listed, *items, *row_info;
  int32_t num_listed, num_items, num_few;
  void* out;
  float* shared;   // [items][KV heads][queries of the item's kind][D + 2]: O, the maximum and the sum of a prefix's part
  float* partials; // [rows][heads][max_chunks][D + 2]: the same of a chunk of own tokens
  uint64_t* tags;  // [rows][KV heads][slices][max_chunks]: equal to `tag` where this call's partials are whole
  uint64_t tag;
  int32_t max_chunks, num_rows, num_heads, num_kv_heads, group, slices;
  float scale_log2;
  int64_t q_stride, kv_stride;
  bool vec;
};

// Queries that an item has room for, and where the first of them lies: queries of all items before it.
template <bool kFew> constexpr int kRoom = kFew ? kColumns : kQueries;
CDB_DEVICE int64_t room_of(const PrefixParams& P, int64_t item, bool few) {
  return few ? item * kColumns : item * kQueries - (int64_t)P.num_few * (kQueries - kColumns);
}

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

// Two numbers, each as two bf16 ones of its sign that it is the sum of, to 2^-16: the next one toward zero, which is never
// the number itself, and the rest, which is never zero. So an infinite key or value meets two factors of one sign, and
// their products' sum is the infinity that the whole factor gives; a part rounded to the nearest leaves a rest that may be
// zero or of the other sign, and NaN. Zero is zero twice. This and the zeros for values outside a range (Walk::weigh) cost
// 0.3 us of 16.4 for 8 rows after 900 tokens, 1.4 of 77 for 99 rows of 55 heads, 1-2 of 100 for 32000 shared tokens.
template <bool kPositive> CDB_DEVICE void split_bf16x2(float x, float y, uint32_t& hi, uint32_t& lo) {
  auto first = [](float v) __attribute__((always_inline)) -> uint32_t {
    const uint32_t b = __float_as_uint(v);
    if constexpr (kPositive) return __builtin_elementwise_sub_sat(b, 1u) & 0xffff0000u;
    return (__builtin_elementwise_sub_sat(b & 0x7fffffffu, 1u) & 0x7fff0000u) | (b & 0x80000000u);
  };
  const uint32_t a = first(x), b = first(y);
  hi = __builtin_amdgcn_perm(b, a, 0x07060302u);
  lo = pack_bf16x2(x - __uint_as_float(a), y - __uint_as_float(b));
}

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
    for (int j = 0; j < kRuns; ++j)
      k[a][j] = *reinterpret_cast<const u32x4_t*>(tile + (token + (32 * j + 8 * g) * 2u));
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
  // Elements d..d + 7 of column c, scaled already, to LDS.
  static CDB_DEVICE void store_query(uint32_t* to, int c, int d, const float* x) {
    to += ((d >> 5) * 64 + ((d & 31) >> 3) * 16 + c) * 4;
    u32x4_t hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t a, b;
      split_bf16x2<false>(x[2 * i], x[2 * i + 1], a, b);
      hi[i] = a;
      lo[i] = b;
    }
    *reinterpret_cast<u32x4_t*>(to) = lo;
    *reinterpret_cast<u32x4_t*>(to + kRuns * 64 * 4) = hi;
  }
  typedef bf16x8_t Operand;
  static constexpr int kOperands = 2 * kRuns;  // of a query: the second parts, then the first ones
  // query(n, i): operand i of column tile n.
  template <int NC, typename F> CDB_DEVICE void scores(F query, f32x4_t (*s)[kTiles]) const {
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int a = 0; a < kTiles; ++a) s[n][a] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kOperands; ++i)
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const Operand q = query(n, i);
#pragma unroll
        for (int a = 0; a < kTiles; ++a)
          s[n][a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, k[a][i % kRuns]), q, s[n][a],
                                                            0, 0, 0);
      }
  }
  template <int NC> CDB_DEVICE void accumulate(const f32x4_t (*p)[kTiles], f32x4_t (*acc)[D / 16]) const {
    union { uint32_t w[4]; bf16x8_t v; } hi[NC], lo[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int i = 0; i < 8; i += 2)
        split_bf16x2<true>(p[n][i >> 2][i & 3], p[n][i >> 2][(i & 3) + 1], hi[n].w[i >> 1], lo[n].w[i >> 1]);
#pragma unroll
    for (int m = 0; m < D / 16; ++m) {
      union { uint32_t w[4]; bf16x8_t v; } x;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x.w[i] = __builtin_amdgcn_perm(v[2 * i + 1][m >> 1], v[2 * i][m >> 1], m & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        acc[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.v, lo[n].v, acc[n][m], 0, 0, 0);
      }
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        acc[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.v, hi[n].v, acc[n][m], 0, 0, 0);
      }
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
  static CDB_DEVICE void store_query(uint32_t* to, int c, int d, const float* x) {
    to += ((d >> 4) * 64 + ((d & 15) >> 2) * 16 + c) * 4;
    *reinterpret_cast<f32x4_t*>(to) = (f32x4_t){x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4_t*>(to + 16 * 4) = (f32x4_t){x[4], x[5], x[6], x[7]};
  }
  typedef f32x4_t Operand;
  static constexpr int kOperands = kRuns;
  template <int NC, typename F> CDB_DEVICE void scores(F query, f32x4_t (*s)[kTiles]) const {
#pragma unroll
    for (int n = 0; n < NC; ++n) s[n][0] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kRuns; ++j)
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const Operand q = query(n, j);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[0][j][i], q[i], s[n][0], 0, 0, 0);
      }
  }
  template <int NC> CDB_DEVICE void accumulate(const f32x4_t (*p)[kTiles], f32x4_t (*acc)[D / 16]) const {
#pragma unroll
    for (int m = 0; m < D / 16; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < NC; ++n)
          acc[n][m] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][m], p[n][0][i], acc[n][m], 0, 0, 0);
  }
};

// The staged walk: a workgroup's waves that take the same tokens share them in LDS. Two parts of the tokens are walked
// side by side, by four waves each; a part's step lies as [keys, values][token][D], rows 16 bytes apart, which spreads
// the operands' reads over all banks. While a step is multiplied the next one's loads are on the way. Computing the
// next step's scores while this one is weighed, with a third step in LDS, takes 252 registers and turns the 105 us of
// the 32000 tokens above into 113.
template <typename T, int D> struct Stage {
  static constexpr int kTiles = StepRegs<T, D>::kTiles, kStep = 16 * kTiles;
  static constexpr int kPieces = D * (int)sizeof(T) / 16;  // of 16 bytes, of a row
  static constexpr int kUnits = (kPieces + 15) / 16;       // of a thread
  static constexpr int kRow = D * (int)sizeof(T) + 16, kPlane = kStep * kRow, kPart = 2 * kPlane, kBytes = 2 * kPart;
  u32x4_t w[2][kTiles][kUnits];

  // `i` of the part's 256 threads: piece i % 16 (and every 16th from there) of row i / 16 of each tile.
  CDB_DEVICE void load(const Tokens& at, const int64_t* tile, const int* b0, const int* b1, int i) {
#pragma unroll
    for (int a = 0; a < kTiles; ++a) {
      const uint32_t row = (uint32_t)min(max(i >> 4, b0[a]), b1[a] - 1) * (uint32_t)at.row_bytes;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const uint32_t piece = min((i & 15) + 16 * u, kPieces - 1) * 16;
        w[0][a][u] = *reinterpret_cast<const u32x4_t*>(at.k + tile[a] + (row + piece));
        w[1][a][u] = *reinterpret_cast<const u32x4_t*>(at.v + tile[a] + (row + piece));
      }
    }
  }
  CDB_DEVICE void store(char* part, int i) const {
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int a = 0; a < kTiles; ++a)
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          const int piece = (i & 15) + 16 * u;
          if (kPieces % 16 == 0 || piece < kPieces)
            *reinterpret_cast<u32x4_t*>(part + p * kPlane + (16 * a + (i >> 4)) * kRow + piece * 16) = w[p][a][u];
        }
  }
};

// A wave's running maxima and sums for NC times 16 queries (of query r, over the lane's own tokens) and O^T: rows are
// elements, row x of product m element x * D / 16 + m.
template <typename T, int D, int NC> struct Walk {
  static constexpr int kTiles = StepRegs<T, D>::kTiles;
  float top[NC], sum[NC];
  bool missing;
  f32x4_t acc[NC][D / 16];
  int lane;

  CDB_DEVICE void start(int l) {
    lane = l;
    missing = false;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      top[n] = -INFINITY;
      sum[n] = 0.f;
#pragma unroll
      for (int m = 0; m < D / 16; ++m) acc[n][m] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
  }
  // Scores, in units of log2, to weights. Tokens outside [lo, hi) of a tile have none, and values of zero (kZeros: they
  // are already): another token stands for them, whose value may be infinite.
  template <bool kZeros = false> CDB_DEVICE void weigh(f32x4_t (*s)[kTiles], const int* lo, const int* hi, int g) {
    bool edge = false;
#pragma unroll
    for (int a = 0; a < kTiles; ++a) edge = edge || lo[a] > 0 || hi[a] < 16;
    if (edge) {
#pragma unroll
      for (int a = 0; a < kTiles; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = 4 * g + i >= lo[a] && 4 * g + i < hi[a];
#pragma unroll
          for (int n = 0; n < NC; ++n) s[n][a][i] = in ? s[n][a][i] : -INFINITY;
          if constexpr (!kZeros) {
#pragma unroll
            for (int w = 0; w < StepRegs<T, D>::kWords; ++w) x.v[4 * a + i][w] = in ? x.v[4 * a + i][w] : 0;
          }
        }
    }
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      float most = top[n];
#pragma unroll
      for (int a = 0; a < kTiles; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) most = fmaxf(most, s[n][a][i]);
      if (__any(most > top[n])) {
        most = column_max(most);
        const float keep = top[n] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top[n] - most);  // the first finds zeros
        sum[n] *= keep;
#pragma unroll
        for (int m = 0; m < D / 16; ++m) acc[n][m] *= keep;
        top[n] = most;
      }
      const float from = top[n] == -INFINITY ? 0.f : top[n];
#pragma unroll
      for (int a = 0; a < kTiles; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[n][a][i] = __builtin_amdgcn_exp2f(s[n][a][i] - from);
          sum[n] += s[n][a][i];
        }
    }
  }
  // Tokens [lo, hi), step `first` of every `stride`: `open` puts the first step on its way, `tokens` walks.
  StepRegs<T, D> x;
  int64_t where;  // lane j: byte offset of tile window + j
  int lo, hi, first, stride, count, window;

  CDB_DEVICE int64_t offset(int j) const {
    const uint32_t a = __builtin_amdgcn_readlane((int)(uint32_t)where, j);
    const uint32_t b = __builtin_amdgcn_readlane((int)(uint32_t)(where >> 32), j);
    return (int64_t)(((uint64_t)b << 32) | a);
  }
  // Of a tile that sticks out of the range the nearest token inside stands for those outside; the last step's second
  // tile may be missing: the first stands in for it.
  CDB_DEVICE int bounds(int step, int a, int& b0, int& b1) const {
    const int j = min(kTiles * step + a, count - 1), t = ((lo >> 4) + window + j) * 16;
    b0 = max(lo - t, 0);
    b1 = min(hi - t, 16);
    return j;
  }
  CDB_DEVICE void load_keys(const Tokens& at, int step, int r, int g) {
#pragma unroll
    for (int a = 0; a < kTiles; ++a) {
      int b0, b1;
      const int64_t tile = offset(bounds(step, a, b0, b1));
      x.load_key(a, at.k + tile, (uint32_t)min(max(r, b0), b1 - 1) * (uint32_t)at.row_bytes, g);
    }
  }
  CDB_DEVICE void load_values(const Tokens& at, int step, int r, int g) {
#pragma unroll
    for (int a = 0; a < kTiles; ++a) {
      int b0, b1;
      const int64_t tile = offset(bounds(step, a, b0, b1));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x.load_value(4 * a + i, at.v + tile, (uint32_t)min(max(4 * g + i, b0), b1 - 1) * (uint32_t)at.row_bytes, r);
    }
  }
  CDB_DEVICE void look_up(const Tokens& at, int w) {
    const int r = lane & 15, g = lane >> 4;
    window = w;
    count = min(64, ((hi + 15) >> 4) - (lo >> 4) - w);
    where = 0;
    bool lost = false;
    if (lane < count) where = at.at(((lo >> 4) + w + lane) * 16, lost);
    missing = missing || __ballot(lost) != 0;
    if (kTiles * first < count) {
      load_keys(at, first, r, g);
      __builtin_amdgcn_sched_barrier(0);  // keys before values, as in the steps: the waits count on it
      load_values(at, first, r, g);
    }
  }
  CDB_DEVICE void open(const Tokens& at, int from, int to, int which, int of) {
    lo = from;
    hi = to;
    first = which;
    stride = of;
    count = 0;
    if (lo < hi) look_up(at, 0);
  }
  // The lane's place in the query operands: columns without a query read the last one's.
  CDB_DEVICE void slots(int cols, int* slot) const {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int c = min(16 * n + (lane & 15), cols - 1);
      slot[n] = (c >> 4) * (StepRegs<T, D>::kQueryWords / 4) + (lane & 48) + (c & 15);
    }
  }
  // Operand i of column tile n as it lies in LDS.
  CDB_DEVICE static typename StepRegs<T, D>::Operand operand(const uint32_t* query, const int* slot, int n, int i) {
    return *reinterpret_cast<const typename StepRegs<T, D>::Operand*>(query + slot[n] * 4 + i * 64 * 4);
  }
  CDB_DEVICE void tokens(const Tokens& at, const uint32_t* query, int cols) {
    int slot[NC];
    slots(cols, slot);
    const int r = lane & 15, g = lane >> 4;
    const int tiles = lo < hi ? ((hi + 15) >> 4) - (lo >> 4) : 0;
    for (int w = 0; w < tiles; w += 64) {
      if (w != 0) look_up(at, w);
      const int steps = (count + kTiles - 1) / kTiles;
      for (int step = first; step < steps; step += stride) {
        // The loads ahead repeat the step at the end: a branch around them would make the wait for this step's
        // values one for the next keys too.
        const int ahead = step + stride < steps ? step + stride : step;
        f32x4_t s[NC][kTiles];
        x.template scores<NC>(
            [&](int n, int i) __attribute__((always_inline)) { return operand(query, slot, n, i); }, s);
        load_keys(at, ahead, r, g);
        int from[kTiles], to[kTiles];
#pragma unroll
        for (int a = 0; a < kTiles; ++a) {
          bounds(step, a, from[a], to[a]);
          if (kTiles * step + a >= count) to[a] = 0;
        }
        weigh(s, from, to, g);
        x.template accumulate<NC>(s, acc);
        __builtin_amdgcn_sched_barrier(0);
        load_values(at, ahead, r, g);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  // The staged walk over [lo, hi) for all of a workgroup's threads; `lds` holds the queries, which every wave takes
  // from there first. A wave without queries only loads.
  CDB_DEVICE void shared_tokens(const Tokens& at, uint32_t* lds, int run, int part, int cols, int from, int to) {
    typedef Stage<T, D> S;
    typedef typename StepRegs<T, D>::Operand Operand;
    constexpr int kOps = StepRegs<T, D>::kOperands;
    const int r = lane & 15, g = lane >> 4, i = threadIdx.x & 255;
    lo = from;
    hi = to;
    const int tiles = ((hi + 15) >> 4) - (lo >> 4), steps = (tiles + kTiles - 1) / kTiles, turns = (steps + 1) / 2;
    window = -64;
    // Two turns' loads are on the way while one is multiplied. The loads at the end repeat the last step: a branch
    // around them would make the waits for the turn before ones for them too.
    S stage[2];
    auto load = [&](S& to_stage, int turn) __attribute__((always_inline)) {
      const int step = min(2 * turn + part, steps - 1), first_tile = kTiles * step;
      if (first_tile >= window + 64) {
        window = first_tile & ~63;
        count = min(64, tiles - window);
        bool lost = false;
        where = 0;
        if (lane < count) where = at.at(((lo >> 4) + window + lane) * 16, lost);
        missing = missing || __ballot(lost) != 0;
      }
      int64_t tile[kTiles];
      int b0[kTiles], b1[kTiles];
#pragma unroll
      for (int a = 0; a < kTiles; ++a) tile[a] = offset(bounds(step - window / kTiles, a, b0[a], b1[a]));
      to_stage.load(at, tile, b0, b1, i);
    };
    load(stage[0], 0);
    load(stage[1], 1);
    Operand q[NC][kOps];
    int slot[NC];
    slots(max(cols, 1), slot);
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int o = 0; o < kOps; ++o) q[n][o] = operand(lds + NC * run * StepRegs<T, D>::kQueryWords, slot, n, o);
    __syncthreads();  // the tokens take the queries' place
    char* ring = reinterpret_cast<char*>(lds) + part * S::kPart;
    stage[0].store(ring, i);
    lds_barrier();
    auto turn_of = [&](int turn, S& free_stage, const S& next_stage, const char* now, char* next)
                       __attribute__((always_inline)) {
      const int step = 2 * turn + part;
      load(free_stage, turn + 2);
      if (cols > 0 && step < steps) {
#pragma unroll
        for (int a = 0; a < kTiles; ++a) x.load_key(a, now + a * 16 * S::kRow, r * S::kRow, g);
        f32x4_t s[NC][kTiles];
        x.template scores<NC>([&](int n, int o) __attribute__((always_inline)) { return q[n][o]; }, s);
#pragma unroll
        for (int a = 0; a < kTiles; ++a)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x.load_value(4 * a + e, now + S::kPlane + a * 16 * S::kRow, (4 * g + e) * S::kRow, r);
        int first_in[kTiles], end_in[kTiles];
#pragma unroll
        for (int a = 0; a < kTiles; ++a) {
          const int t = ((lo >> 4) + kTiles * step + a) * 16;
          first_in[a] = max(lo - t, 0);
          end_in[a] = min(hi - t, 16);
        }
        weigh(s, first_in, end_in, g);
        x.template accumulate<NC>(s, acc);
      }
      next_stage.store(next, i);
      lds_barrier();
    };
    for (int turn = 0; turn < turns; turn += 2) {
      turn_of(turn, stage[0], stage[1], ring, ring + S::kBytes);
      if (turn + 1 < turns) turn_of(turn + 1, stage[1], stage[0], ring + S::kBytes, ring);
    }
  }
  // O, the maximum and the sum of each column: [column][stride].
  CDB_DEVICE void leave(float* to, int cols, int stride) {
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      float total = column_sum(sum[n]);
      if (missing) total = NAN;
      if (16 * n + r >= cols) continue;
      float* mine = to + (16 * n + r) * stride;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int m = 0; m < D / 16; m += 2)
          *reinterpret_cast<f32x2_t*>(mine + (4 * g + i) * (D / 16) + m) = (f32x2_t){acc[n][m][i], acc[n][m + 1][i]};
      if (g == 0) {
        mine[D] = total == 0.f ? -INFINITY : top[n];  // no token yet, or none above -infinity
        mine[D + 1] = total;
      }
    }
  }
  // Takes in what another wave has left for the same columns.
  CDB_DEVICE void join(const float* from, int cols, int stride) {
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const float* other = from + min(16 * n + r, cols - 1) * stride;
      const float most = fmaxf(top[n], other[D]), base = most == -INFINITY ? 0.f : most;
      const float f0 = __builtin_amdgcn_exp2f(top[n] - base), f1 = __builtin_amdgcn_exp2f(other[D] - base);
      sum[n] = fmaf(sum[n], f0, g == 0 ? f1 * other[D + 1] : 0.f);  // a column's sum is that of its four lanes
      top[n] = most;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int m = 0; m < D / 16; m += 2) {
          const f32x2_t y = *reinterpret_cast<const f32x2_t*>(other + (4 * g + i) * (D / 16) + m);
          acc[n][m][i] = fmaf(acc[n][m][i], f0, f1 * y[0]);
          acc[n][m + 1][i] = fmaf(acc[n][m + 1][i], f0, f1 * y[1]);
        }
    }
  }
};

// 16 elements of a column of the query operands: of query head `head` of row b at position p, rotated and scaled; NaN,
// or zeros, where there is no such query.
template <typename T, int D, int STYLE>
CDB_DEVICE void turn_query(const PrefixParams& P, uint32_t* query, int c, int piece, int b, int head, int p,
                           float none) {
  const int d = STYLE == 1 ? 8 * piece : 16 * piece;
  float x[8], y[8];
  if (p >= 0) {
    const int64_t angle = STYLE == 0 ? 0 : (int64_t)p * (D / 2);
    const T* bias = static_cast<const T*>(P.q_bias);
    load_rotated_pair<T, D, STYLE, 8>(static_cast<const T*>(P.q) + b * P.q_stride + (int64_t)head * D,
                                      bias == nullptr ? nullptr : bias + (int64_t)head * D, P.cos + angle,
                                      P.sin + angle, d, P.vec, x, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = mul_rn(x[i], P.scale_log2);
      y[i] = mul_rn(y[i], P.scale_log2);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i] = none;
  }
  query += (c >> 4) * StepRegs<T, D>::kQueryWords;
  StepRegs<T, D>::store_query(query, c & 15, d, x);
  StepRegs<T, D>::store_query(query, c & 15, STYLE == 1 ? d + D / 2 : d + 8, y);
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

// Words of LDS: the queries, and in their place later the staged tokens, and what half of the waves leave to the other.
template <typename T, int D, bool kFew> struct AttendLds {
  static constexpr int kQ = StepRegs<T, D>::kQueryWords * (kRoom<kFew> / 16);
  static constexpr int kJoin = kWaves<kFew> / 2 * (kFew ? 16 : 32) * (D + 4);
  static constexpr int kStages = kFew ? 0 : Stage<T, D>::kBytes / 2;
  static constexpr int kMost = kQ > kJoin ? kQ : kJoin, kWords = kMost > kStages ? kMost : kStages;
};

template <typename T, int D, int STYLE, bool kFew>
__global__ void __launch_bounds__(64 * kWaves<kFew>, (kFew ? 3 : 2)) prefix_attend_kernel(PrefixParams P) {
  constexpr int kThreads = 64 * kWaves<kFew>, NC = kFew ? 1 : 2;
  __shared__ __align__(16) uint32_t lds[AttendLds<T, D, kFew>::kWords];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int at_item = blockIdx.x / P.num_kv_heads, kvh = blockIdx.x - at_item * P.num_kv_heads;
  const int item = at_item + (kFew ? 0 : P.num_few);
  const int4 head = reinterpret_cast<const int4*>(P.items + (int64_t)kItem * item)[0];
  const int4 tail = reinterpret_cast<const int4*>(P.items + (int64_t)kItem * item)[1];
  const int first = head.x, count = head.y, length = head.w, q0 = tail.x, lo = tail.y, hi = tail.z;
  if (count <= 0 || count > P.num_listed || first < 0 || first > P.num_listed - count) return;  // no item
  const int64_t queries = (int64_t)count * P.group;
  if (q0 < 0 || q0 >= queries) return;
  const int cols = (int)min((int64_t)kRoom<kFew>, queries - q0);
  // The row through which the tokens are read: the group's first, or the first behind it that is no padding.
  int leader = head.z, layer = -1, trow = -1;
  if (leader >= 0 && leader < P.num_rows && P.seqlens[leader] < 0) {
    leader = -1;
    for (int i = 0; i < count && leader < 0; i += kWave) {
      const int b = i + lane < count ? P.listed[first + i + lane] : -1;
      const uint64_t live = __ballot(b >= 0 && b < P.num_rows && P.seqlens[b] >= 0);
      if (live != 0) leader = __builtin_amdgcn_readlane(b, __ffsll((unsigned long long)live) - 1);
    }
    if (leader < 0) return;  // no row that asks for the tokens
  }
  if (leader >= 0 && leader < P.num_rows) {
    layer = P.cache_layer0 + (P.cache_layer == nullptr ? 0 : P.cache_layer[leader]);
    trow = P.table_row == nullptr ? leader : P.table_row[leader];
  }
  const bool bad = layer < 0 || layer >= P.num_layers || trow < 0 || trow >= P.table_rows || lo < 0 || hi > length ||
                   (int64_t)length > ((int64_t)P.table_width << P.bs_log2);
  const int runs = kFew ? 1 : 4, run = wave & (runs - 1), part = wave / runs, parts = kWaves<kFew> / runs;
  const int mine = min(16 * NC, cols - 16 * NC * run);  // may be none
  const Tokens at_prefix = tokens_of<T, D>(P, bad ? 0 : layer, bad ? 0 : trow, kvh);
  Walk<T, D, NC> walk;
  walk.start(lane);
  if (bad) walk.missing = true;
  if constexpr (kFew) walk.open(at_prefix, bad ? 0 : lo, bad ? 0 : hi, part, parts);
  constexpr int kPieces = D / 16;
#pragma unroll 2
  for (int i = threadIdx.x; i < cols * kPieces; i += kThreads) {
    const int c = i / kPieces, at = q0 + c;
    const int b = P.listed[first + at / P.group];
    int p = b >= 0 && b < P.num_rows ? P.seqlens[b] : -1;
    // A padding row, or one that gets NaN: for not being at its group's cache layer, from here.
    const bool stranger = p >= 0 && P.cache_layer != nullptr && P.cache_layer0 + P.cache_layer[b] != layer;
    if (stranger || (STYLE != 0 && p >= P.max_positions)) p = -1;
    turn_query<T, D, STYLE>(P, lds, c, i - c * kPieces, b, kvh * P.group + at % P.group, p, stranger ? NAN : 0.f);
  }
  __syncthreads();
  if constexpr (kFew) {
    walk.tokens(at_prefix, lds, mine);
  } else if (!bad && lo < hi) {
    walk.shared_tokens(at_prefix, lds, run, part, mine, lo, hi);
  }
  float* to = P.shared + (room_of(P, item, kFew) * P.num_kv_heads + kvh * kRoom<kFew>) * (D + 2);
  // Waves with the same queries are joined in halves.
  float* join = reinterpret_cast<float*>(lds) + run * 16 * NC * (D + 4);
  constexpr int kSlot = 16 * NC * (D + 4);
  for (int half = parts >> 1; half > 0; half >>= 1) {
    __syncthreads();
    if (mine > 0 && part >= half && part < 2 * half) walk.leave(join + (part - half) * runs * kSlot, mine, D + 4);
    __syncthreads();
    if (mine > 0 && part < half) walk.join(join + part * runs * kSlot, mine, D + 4);
  }
  if (mine > 0 && part == 0) walk.leave(to + 16 * NC * run * (D + 2), mine, D + 2);
}

template <typename T, int D, int STYLE>
__global__ void __launch_bounds__(64 * kRowWaves, 3) prefix_decode_kernel(PrefixParams P) {
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
  const int n0 = P.row_info[4 * b], item0 = P.row_info[4 * b + 2], given = P.row_info[4 * b + 3];
  row.bad = row.bad || given < -kMaxParts || given > kMaxParts;
  const int parts = row.bad ? 0 : given < 0 ? -given : given;
  const bool few = given < 0;
  const int each_log2 = few ? 4 : 7, each = 1 << each_log2;  // queries of an item
  if (parts == 0) {
    row.bad = row.bad || row.own != 0;
  } else {
    const int64_t last = item0 + ((((int64_t)n0 + P.group - 1) >> each_log2) + 1) * parts;  // behind the row's last item
    row.bad = row.bad || n0 < 0 || item0 < (few ? 0 : P.num_few) || last > (few ? P.num_few : P.num_items);
  }
  if (p < 0 || row.bad) {
    if (chunk == 0)
      for (int i = threadIdx.x; i < P.group * D; i += 64 * kRowWaves) Elem<T>::store(out + i, p < 0 ? 0.f : NAN);
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
    // Opaque, so that nothing derived from the lane is kept over the loop (it takes one turn but for groups of more
    // than 16, and the registers are needed inside).
    int tid = threadIdx.x;
    __asm__ volatile("" : "+v"(tid));
    const int lane = tid & 63;
    Walk<T, D, 1> walk;
    walk.start(lane);
    walk.open(at, lo, hi, wave, kRowWaves);  // on its way before the queries are turned
    for (int i = tid; i < cols * (D / 16); i += 64 * kRowWaves)
      turn_query<T, D, STYLE>(P, query, i / (D / 16), i % (D / 16), b, kvh * P.group + slice + i / (D / 16), p, 0.f);
    if (ends && wave == kRowWaves - 1) {
      const int d = min(2 * lane, D - 2);
      const int64_t angle = STYLE == 0 ? 0 : (int64_t)p * (D / 2), from = b * P.kv_stride + (int64_t)kvh * D;
      const T* bias = static_cast<const T*>(P.k_bias);
      float x[2], y[2];
      load_f32<T, 2>(static_cast<const T*>(P.v_new) + from + d, y, P.vec);
      load_rotated<T, D, STYLE, 2>(static_cast<const T*>(P.k_new) + from, bias == nullptr ? nullptr : bias + kvh * D,
                                   P.cos + angle, P.sin + angle, d, P.vec, x);
      bool lost = false;
      const int64_t tile = at.at(p & ~15, lost) + (int64_t)(p & 15) * at.row_bytes;
      walk.missing = walk.missing || lost;
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
    walk.tokens(at, query, cols);
    if (ends && wave == kRowWaves - 1) {
      // The new token as the first of a tile, with zeros for the values of the others.
      const int r = lane & 15, g = lane >> 4;
#pragma unroll
      for (int a = 0; a < StepRegs<T, D>::kTiles; ++a)
        walk.x.load_key(a, reinterpret_cast<const char*>(fresh[0]), 0, g);
      walk.x.load_value(0, reinterpret_cast<const char*>(fresh[1]), 0, r);
#pragma unroll
      for (int i = 0; i < 4 * StepRegs<T, D>::kTiles; ++i)
#pragma unroll
        for (int w = 0; w < StepRegs<T, D>::kWords; ++w) walk.x.v[i][w] = i == 0 && g == 0 ? walk.x.v[i][w] : 0;
      f32x4_t s[1][StepRegs<T, D>::kTiles];
      int slot[1];
      walk.slots(cols, slot);
      walk.x.template scores<1>(
          [&](int n, int i) __attribute__((always_inline)) { return walk.operand(query, slot, n, i); }, s);
      const int from[2] = {0, 0}, to[2] = {1, 0};
      walk.template weigh<true>(s, from, to, g);
      walk.x.template accumulate<1>(s, walk.acc);
    }
    walk.leave(join + wave * cols * kPlace, cols, kPlace);
    __syncthreads();

    const int64_t shared_stride = (int64_t)P.num_kv_heads * each * (D + 2);
    const float* shared0 = P.shared + (room_of(P, item0, few) * P.num_kv_heads + kvh * each) * (D + 2);
    auto shared_of = [&](int c) __attribute__((always_inline)) -> const float* {
      const int n = n0 + slice + c;
      return shared0 + (n >> each_log2) * parts * shared_stride + (n & (each - 1)) * (D + 2);
    };
    if (chunks > 1) {
      for (int i = tid; i < cols * D; i += 64 * kRowWaves) {
        const int c = i / D, d = i - c * D;
        float m[kRowWaves], most = -INFINITY, o = 0.f, l = 0.f;
#pragma unroll
        for (int w = 0; w < kRowWaves; ++w) {
          m[w] = join[(w * cols + c) * kPlace + D];
          most = fmaxf(most, m[w]);
        }
        const float from = most == -INFINITY ? 0.f : most;
#pragma unroll
        for (int w = 0; w < kRowWaves; ++w) {
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
    const int mine = chunks > 1 ? chunks : kRowWaves;
    const float* rows = P.partials + ((int64_t)b * P.num_heads + kvh * P.group + slice) * P.max_chunks * (D + 2);
    for (int c = wave; c < cols; c += kRowWaves) {
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
    for (int i = tid; i < cols * (D / 2); i += 64 * kRowWaves) {
      const int c = i / (D / 2), d = 2 * (i - c * (D / 2));
      float o0 = 0.f, o1 = 0.f;
      const float* x = shared_of(c) + d;
      for (int n = 0; n < parts; n += 8) {
        f32x2_t y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          y[j] = *reinterpret_cast<const f32x2_t*>(x + (int64_t)min(n + j, parts - 1) * shared_stride);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float f = n + j < parts ? weights[c][kMaxChunks + min(n + j, kMaxParts - 1)] : 0.f;
          if (n + j < parts) {
            o0 = fmaf(f, y[j][0], o0);
            o1 = fmaf(f, y[j][1], o1);
          }
        }
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
  if (P.num_few > 0) {
    prefix_attend_kernel<T, D, STYLE, true>
        <<<dim3((unsigned)(P.num_few * P.num_kv_heads)), dim3(64 * kWaves<true>), 0, stream>>>(P);
    if (hipGetLastError() != hipSuccess) return CDB_ERR_HIP;
  }
  if (P.num_items > P.num_few) {
    prefix_attend_kernel<T, D, STYLE, false>
        <<<dim3((unsigned)((P.num_items - P.num_few) * P.num_kv_heads)), dim3(64 * kWaves<false>), 0, stream>>>(P);
    if (hipGetLastError() != hipSuccess) return CDB_ERR_HIP;
  }
  const int64_t most = ((int64_t)P.table_width << P.bs_log2) / kChunk + 1;
  const dim3 grid((unsigned)(P.num_rows * P.num_kv_heads), (unsigned)min((int64_t)P.max_chunks, most));
  const size_t lds = sizeof(float) * kRowWaves * min(P.group, kColumns) * (D + 4);
  prefix_decode_kernel<T, D, STYLE><<<grid, dim3(64 * kRowWaves), lds, stream>>>(P);
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
static int64_t shared_bytes(int64_t num_few, int64_t num_items, int32_t num_kv_heads, int32_t head_dim) {
  return (num_few * kColumns + (num_items - num_few) * kQueries) * num_kv_heads * (head_dim + 2) * 4;
}

}  // namespace cdb

extern "C" int64_t cdb_prefix_decode_plan_workspace_bytes(int32_t num_rows, int32_t num_few, int32_t num_items,
                                                          int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                                          int32_t max_own) {
  if (num_rows < 0 || num_few < 0 || num_items < num_few || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      head_dim <= 0 || max_own <= 0)
    return -1;
  const int64_t chunks = min(((int64_t)max_own + cdb::kChunk - 1) / cdb::kChunk, (int64_t)cdb::kMaxChunks);
  return cdb::shared_bytes(num_few, num_items, num_kv_heads, head_dim) +
         max((int64_t)num_rows, (int64_t)1) * chunks * cdb::chunk_bytes(num_heads, num_kv_heads, head_dim);
}

extern "C" int64_t cdb_prefix_decode_workspace_bytes(int32_t num_rows, int32_t num_items, int32_t num_heads,
                                                     int32_t num_kv_heads, int32_t head_dim, int32_t max_own) {
  return cdb_prefix_decode_plan_workspace_bytes(num_rows, 0, num_items, num_heads, num_kv_heads, head_dim, max_own);
}

extern "C" int cdb_prefix_decode_attention(
    const void* q, const void* k_new, const void* v_new, void* k_pool, void* v_pool, int64_t layer_stride,
    int32_t num_cache_layers, int64_t pool_blocks, const int32_t* cache_layer, int32_t cache_layer0,
    const int32_t* block_table, const int32_t* table_row, int32_t table_rows, int32_t table_width,
    const int32_t* seqlens, const float* rope_cos, const float* rope_sin, int32_t rope_style, int32_t max_positions,
    const void* q_bias, const void* k_bias, const int32_t* listed, int32_t num_listed, const int32_t* items,
    int32_t num_items, int32_t num_few, const int32_t* row_info, void* out, void* workspace,
    int64_t workspace_bytes, int32_t num_rows, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t block_size, float scale, int64_t q_stride, int64_t kv_stride, int32_t dtype, hipStream_t stream) {
  using namespace cdb;
  if (rope_style < 0 || rope_style > 2) return CDB_ERR_UNSUPPORTED;
  if (dtype != CDB_DTYPE_F32 && dtype != CDB_DTYPE_BF16) return CDB_ERR_UNSUPPORTED;
  if (head_dim != 64 && head_dim != 96 && head_dim != 128) return CDB_ERR_UNSUPPORTED;
  if (num_rows < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || table_rows <= 0 ||
      table_width <= 0 || num_cache_layers <= 0 || pool_blocks <= 0 || pool_blocks > 0x7fffffffll || num_listed < 0 ||
      num_items < 0 || num_few < 0 || num_few > num_items)
    return CDB_ERR_SHAPE;
  if (block_size < 16 || (block_size & (block_size - 1)) != 0) return CDB_ERR_SHAPE;
  if (num_rows == 0) return CDB_OK;
  if (q == nullptr || k_new == nullptr || v_new == nullptr || k_pool == nullptr || v_pool == nullptr ||
      block_table == nullptr || seqlens == nullptr || row_info == nullptr || out == nullptr || workspace == nullptr)
    return CDB_ERR_NULL;
  if (rope_style != 0 && (rope_cos == nullptr || rope_sin == nullptr)) return CDB_ERR_NULL;
  if (num_items != 0 && (listed == nullptr || items == nullptr)) return CDB_ERR_NULL;
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
      reinterpret_cast<uintptr_t>(v_pool) % 16 != 0 || reinterpret_cast<uintptr_t>(items) % 16 != 0 ||
      layer_stride * size % 16 != 0)
    return CDB_ERR_SHAPE;
  const int64_t left = workspace_bytes - shared_bytes(num_few, num_items, num_kv_heads, head_dim);
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
  P.listed = listed; P.items = items; P.row_info = row_info;
  P.num_listed = num_listed; P.num_items = num_items; P.num_few = num_few;
  P.out = out; P.shared = static_cast<float*>(workspace);
  P.partials = P.shared + shared_bytes(num_few, num_items, num_kv_heads, head_dim) / 4;
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
