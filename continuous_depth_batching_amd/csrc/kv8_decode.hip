// Decode attention over the 8-bit paged KV cache, with fused rotation and append.
//
// One workgroup of 4 waves takes 1024 tokens of one row and KV head, with all query heads that share it; a
// wave takes every fourth pair of 16-token tiles and keeps a running maximum and sum of its own. The waves
// are joined through LDS, and a row's chunks through fp32 partials by the workgroup that ends last. Bytes
// from HBM bound it, so the arithmetic goes where it costs least:
//   S^T = K Q^T runs on the codes themselves, v_mfma_scale_f32_16x16x128_f8f6f4 with the tile's scale
//   as the operand's: a key costs no vector instruction. The query is taken as 3 e4m3 parts, each 16
//   times finer than the one before; what they leave of it is 2^-13.8 of the head's largest element.
//   fp32 models take 3 bf16 parts, 2^-24, and widen the codes to bf16, which is exact.
//   O^T = V^T P^T runs in fp16, which holds a code exactly and P to 2^-11: it is raised by 2^15, so that
//   keys down to 2^-29 of the row's largest keep that, and none is off by more than 2^-40 of it. fp32 models
//   take P as 2 fp16 parts (2^-23, and 2^-51 of the largest). Codes widen with their scale, in a unit that follows
//   the tiles' scales, one instruction a pair.
//   Both products are 16 query heads wide (columns without a head repeat the last). A lane's four scores
//   are those of the four tokens it holds of V, so P never moves.
//
// Measured (a launch from a graph): 256 rows of 32..2048 tokens, 16 heads x 128, 107-110 us (4.8 TB/s of cached
// codes; 118 with chunks of 512 tokens, 128 with a merge launch of its own); 21 rows of 4k..32k tokens, 32 heads
// on 8 x 128, 113 us (5.2 TB/s); one row of 900 tokens 9.6-10.5 us, a chain of latencies: position, block ids,
// tiles and query, 7 pairs a wave, the join. The same loads without arithmetic take 85 and 104 us.
#include <atomic>
#include <chrono>
#include <type_traits>

#include "cdb_amd.h"
#include "kv8_common.h"
#include "kv8_host.h"

namespace cdb {

// Waves and tokens of a workgroup. Each wave has its own look-ups and its share of the join, so fewer and
// longer ones cost less where many rows fill the device (256 rows: 8 waves 132 us, 4 waves 108, 2 waves 108),
// and more are faster alone (one row: 8.4, 9.3 and 13.7 us).
constexpr int kWaves = 4;
constexpr int kChunk = 1024;
constexpr int kMaxChunks = 64;           // of a row; longer contexts take longer chunks
constexpr int kSkew = 2 * (kWaves - 1);  // pairs that the wave that appends leaves to the others first
// Waves a SIMD, as many as the registers allow.
template <typename T, int D> constexpr int kDecodeWaves = sizeof(T) == 4 ? (D == 64 ? 4 : 3) : (D == 64 ? 5 : 4);

struct Kv8DecodeParams {
  const void *q, *k_new, *v_new;
  Kv8Cache cache;
  const int32_t *cache_layer, *block_table, *table_row, *seqlens;
  int32_t cache_layer0, table_rows, table_width, max_positions, bs_log2;
  const float *cos, *sin;
  const void *q_bias, *k_bias;
  void* out;
  float* partials;  // [rows][heads][max_chunks][D + 2]: O, the maximum and the sum of a chunk
  uint64_t* tags;   // [rows][KV heads][slices][max_chunks]: equal to `tag` where this call's partials are whole
  uint64_t tag;
  int32_t max_chunks, num_rows, num_heads, group, slices;
  float scale_log2;
  int64_t q_stride, kv_stride;
  bool vec;
};

// What a lane holds of a 16-token tile: token r of the keys (16-byte units g, g + 4) and group g of the
// values (elements 4r..4r+3 of each 64), 16 bytes for every 64 elements; 8 for the last 32 of a head of 96.
template <int D> struct KeyRegs {
  static constexpr int kFull = D / 64;
  static constexpr bool kTail = D % 64 != 0;
  u32x4_t w[kFull];
  u32x2_t t;

  static CDB_DEVICE int64_t at(int j, int r, int g) { return j * 1024 + (g * 16 + r) * 16; }
  static CDB_DEVICE int tail_lane(int r, int g) { return (g >> 1) * 256 + r * 16 + (g & 1) * 8; }
  // `on` all ones, or zero: then every lane reads the first lane's, one line of the tile.
  CDB_DEVICE void load(const uint8_t* p, int r, int g, int on = -1) {
#pragma unroll
    for (int j = 0; j < kFull; ++j)
      w[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p + j * 1024 + (((g * 16 + r) * 16) & on)));
    if constexpr (kTail)
      t = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t*>(p + kFull * 1024 + (tail_lane(r, g) & on)));
  }
  CDB_DEVICE void store(uint8_t* p, int r, int g) const {
#pragma unroll
    for (int j = 0; j < kFull; ++j) *reinterpret_cast<u32x4_t*>(p + at(j, r, g)) = w[j];
    if constexpr (kTail) *reinterpret_cast<u32x2_t*>(p + kFull * 1024 + tail_lane(r, g)) = t;
  }
  // Operand of the 128-deep product: the lane's D / 4 codes, and zeros up to 32.
  CDB_DEVICE i32x8_t operand() const {
    i32x8_t x = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < kFull; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * j + i] = (int)w[j][i];
    if constexpr (kTail) {
      x[4 * kFull] = (int)t[0];
      x[4 * kFull + 1] = (int)t[1];
    }
    return x;
  }
  // Where element d of head c lies among the operands of the 64 lanes, 32 bytes each; elements D..127 are the
  // padding.
  static CDB_DEVICE int place(int d, int c) {
    const bool tail = kTail && d >= 64 * kFull;
    const int g = tail ? (d & 31) >> 3 : (d & 63) >> 4;
    const int byte = tail ? 16 * kFull + ((d >> 5) & 1) * 8 + (d & 7) : (d >> 6) * 16 + (d & 15);
    return (g * 16 + c) * 32 + byte;
  }
};

template <int D> struct ValueRegs {
  static constexpr int kFull = D / 64, kWords = D / 16;
  static constexpr bool kTail = D % 64 != 0;
  uint32_t w[kWords];

  CDB_DEVICE void load(const uint8_t* p, int r, int g, int on = -1) {
#pragma unroll
    for (int j = 0; j < kFull; ++j) {
      const u32x4_t x = __builtin_nontemporal_load(
          reinterpret_cast<const u32x4_t*>(p + j * 256 + ((g * (4 * D) + r * 16) & on)));
#pragma unroll
      for (int i = 0; i < 4; ++i) w[4 * j + i] = x[i];
    }
    if constexpr (kTail) {
      const u32x2_t x = __builtin_nontemporal_load(
          reinterpret_cast<const u32x2_t*>(p + kFull * 256 + ((g * (4 * D) + r * 8) & on)));
      w[4 * kFull] = x[0];
      w[4 * kFull + 1] = x[1];
    }
  }
  CDB_DEVICE void store(uint8_t* p, int r, int g) const {
    p += g * (4 * D);
#pragma unroll
    for (int j = 0; j < kFull; ++j)
      *reinterpret_cast<u32x4_t*>(p + j * 256 + r * 16) = (u32x4_t){w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]};
    if constexpr (kTail)
      *reinterpret_cast<u32x2_t*>(p + kFull * 256 + r * 8) = (u32x2_t){w[4 * kFull], w[4 * kFull + 1]};
  }
  CDB_DEVICE void clear() {
#pragma unroll
    for (int m = 0; m < kWords; ++m) w[m] = 0;
  }
  // The head element of word m, and of row `row` of value product m.
  static CDB_DEVICE int element(int m, int row) {
    return m < 4 * kFull ? 64 * (m >> 2) + 4 * row + (m & 3) : 64 * kFull + 2 * row + (m - 4 * kFull);
  }
};

// A lane's share of 16 query heads, as the operand of the products with the keys: e4m3 parts with a scale
// each, or for fp32 models bf16 parts. The first takes a tile in one product a part and no vector instruction,
// but its sums keep only some 16 bits of the largest term (measured: results 2.6e-5 off in fp32, where the
// second, with the codes widened to bf16, is 2e-7 off).
template <int D, bool kWide> struct QueryRegs {
  static constexpr int kParts = 3;
  const uint32_t* at;  // they stay in LDS: 24 registers fewer let a fourth wave run on each SIMD
  int byte;

  // Columns past the last head repeat it; what they give is not used.
  CDB_DEVICE void load(const uint32_t* codes, const int* bytes, int cols, int r, int g) {
    const int c = min(r, cols - 1);
    byte = bytes[c];
    at = codes + (g * 16 + c) * 8;
  }
  // Elements d and d + 1 (d even; zeros from D on) of head c, already scaled by scale * log2(e); top: the
  // largest finite size in the head.
  static CDB_DEVICE void store(uint32_t* codes, int* bytes, int c, int d, float x0, float x1, float top) {
    const int b = max(scale_byte(top), 4 * kParts);
    bytes[c] = b;
    const float inv = inverse_scale_of(b);
    x0 = mul_rn(x0, inv);
    x1 = mul_rn(x1, inv);
    uint8_t* to = reinterpret_cast<uint8_t*>(codes) + KeyRegs<D>::place(d, c);
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      const uint32_t y = codes_of(x0, x1, 0.f, 0.f);
      const f32x2_t back = __builtin_amdgcn_cvt_pk_f32_fp8((int)y, false);
      x0 = 16.f * (x0 - back.x);
      x1 = 16.f * (x1 - back.y);
      *reinterpret_cast<uint16_t*>(to + p * 64 * 32) = (uint16_t)y;
    }
  }
  CDB_DEVICE f32x4_t scores(const KeyRegs<D>& k, uint32_t k_byte) const {
    const i32x8_t a = k.operand();
    f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = kParts - 1; p >= 0; --p) {
      const i32x8_t w = *reinterpret_cast<const i32x8_t*>(at + p * 64 * 8);
      s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, w, s, 0, 0, 0, (int)k_byte, 0, byte - 4 * p);
    }
    return s;
  }
  static constexpr int kWords = kParts * 64 * 8;  // of LDS
};

template <int D> struct QueryRegs<D, true> {
  static constexpr int kParts = 3, kRuns = D / 32;
  bf16x8_t w[kParts][kRuns];

  CDB_DEVICE void load(const uint32_t* codes, const int*, int cols, int r, int g) {
    const int c = min(r, cols - 1);
#pragma unroll
    for (int p = 0; p < kParts; ++p)
#pragma unroll
      for (int m = 0; m < kRuns; ++m) {
        w[p][m] = *reinterpret_cast<const bf16x8_t*>(codes + ((p * kRuns + m) * 64 + g * 16 + c) * 4);
      }
  }
  static CDB_DEVICE void store(uint32_t* codes, int*, int c, int d, float x0, float x1, float) {
    if (d >= D) return;
    const int at = KeyRegs<D>::place(d, c), m = (at & 31) >> 3;  // run m of 8 elements of lane slot at / 32
    uint32_t* to = codes + (m * 64 + (at >> 5)) * 4 + ((at & 7) >> 1);
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      const uint32_t y = pack_bf16x2(x0, x1);
      x0 -= __uint_as_float(y << 16);
      x1 -= __uint_as_float(y & 0xffff0000u);
      to[p * kRuns * 64 * 4] = y;
    }
  }
  CDB_DEVICE f32x4_t scores(const KeyRegs<D>& k, uint32_t k_byte) const {
    using K = KeyRegs<D>;
    const float f = scale_of(k_byte);
    f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < kRuns; ++m) {
      uint32_t y[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (K::kTail) y[i] = m < 2 * K::kFull ? k.w[m >> 1 < K::kFull ? m >> 1 : 0][2 * (m & 1) + i] : k.t[i];
        else y[i] = k.w[m >> 1][2 * (m & 1) + i];
      }
      const bf16x8_t a = widen_bf16(y[0], f, y[1], f);
#pragma unroll
      for (int p = kParts - 1; p >= 0; --p) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, w[p][m], s, 0, 0, 0);
    }
    return s;
  }
  static constexpr int kWords = kParts * kRuns * 64 * 4;
};

// One wave's share of a chunk: a running maximum and sum (of the lane's query head r, over its own
// tokens), and O^T with element rows and head columns, in the values' unit.
template <int D, bool kWide> struct Attention {
  static constexpr int kTiles = D / 16, kPParts = kWide ? 2 : 1;
  // Probabilities are counted in units of 2^-15, the largest then being 2^15, within fp16: its smallest step, 2^-24,
  // stands for 2^-39. That is, scores are counted from `low`, 15 below the maximum (0 below a very large one, where
  // 15 would round to 16 or nothing, and keys that far below are gone in fp32 all the same). fp32 models count from
  // the maximum and raise by a product, which is exact: the 15 would cost an exponent near 0 three of its bits.
  static constexpr int kRaise = 15;
  static constexpr float kFrom = kWide ? 0.f : (float)kRaise, kTimes = kWide ? 0x1p15f : 1.f;
  using Unit = ValueUnit<std::conditional_t<kWide, float, bf16_t>>;
  float top, low, sum;
  Unit unit;
  f32x4_t acc[kTiles];

  CDB_DEVICE void start() {
    top = -INFINITY;
    low = sum = 0.f;
    unit = Unit();
#pragma unroll
    for (int m = 0; m < kTiles; ++m) acc[m] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  }
  // Scores of one tile (in units of log2), tokens `seen` and up of it left out.
  CDB_DEVICE f32x4_t scores(const KeyRegs<D>& k, uint32_t k_byte, const QueryRegs<D, kWide>& q, int seen, int g) const {
    f32x4_t s = q.scores(k, k_byte);
    if (seen < kTile) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = 4 * g + i < seen ? s[i] : -INFINITY;
    }
    return s;
  }
  CDB_DEVICE void scale_acc(float f) {
#pragma unroll
    for (int m = 0; m < kTiles; ++m) acc[m] *= f;
  }
  CDB_DEVICE void move_acc(int by) {
#pragma unroll
    for (int m = 0; m < kTiles; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][i] = ldexpf(acc[m][i], by);
  }
  // Probabilities of two tiles' scores, in the order of the value products' tokens.
  CDB_DEVICE void softmax(const f32x4_t* s, f16x8_t* parts) {
    float most = top;
#pragma unroll
    for (int i = 0; i < 4; ++i) most = fmaxf(fmaxf(most, s[0][i]), s[1][i]);
    most = column_max(most);
    if (__any(most > top)) {
      const float now = most - (fabsf(most) < kWideScore ? kFrom : 0.f);
      const float keep = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(low - now);  // the first count finds zeros
      sum *= keep;
      scale_acc(keep);
      top = most;
      low = most == -INFINITY ? 0.f : now;
    }
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = __builtin_amdgcn_exp2f(s[i >> 2][i & 3] - low);
      if constexpr (kWide) p[i] *= kTimes;
      sum += p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const f16x2_t y = __builtin_convertvector((f32x2_t){p[i], p[i + 1]}, f16x2_t);
      parts[0][i] = y[0];
      parts[0][i + 1] = y[1];
      if constexpr (kWide) {
        const f16x2_t z = __builtin_convertvector(
            (f32x2_t){(p[i] - (float)y[0]) * kSecondRaise, (p[i + 1] - (float)y[1]) * kSecondRaise}, f16x2_t);
        parts[kPParts - 1][i] = z[0];
        parts[kPParts - 1][i + 1] = z[1];
      }
    }
  }
  CDB_DEVICE void values(const ValueRegs<D>& v0, const ValueRegs<D>& v1, int e0, int e1, const f16x8_t* parts) {
    if (abs(e0 - e1) > Unit::kExact) {
      // No unit holds both tiles: the smaller one by itself first, the other one's values flushed.
      const int low = min(e0, e1);
      if (unit.moves(low)) move_acc(unit.move(low));
      products(v0, v1, unit.scale(e0 == low ? e0 : kNothing), unit.scale(e1 == low ? e1 : kNothing), parts);
      e0 = e0 == low ? kNothing : e0;
      e1 = e1 == low ? kNothing : e1;
    }
    if (unit.moves(e0) || unit.moves(e1)) move_acc(unit.move(max(e0, e1)));
    products(v0, v1, unit.scale(e0), unit.scale(e1), parts);
  }
  // Values that widen to nothing (NaN to NaN all the same: the row has it anyhow).
  static constexpr int kNothing = -1000;
  CDB_DEVICE void products(const ValueRegs<D>& v0, const ValueRegs<D>& v1, float s0, float s1, const f16x8_t* parts) {
#pragma unroll
    for (int m = 0; m < kTiles; ++m) {
      if constexpr (kWide) {
        const f16x8_t v = widen_f16(v0.w[m], s0 / kSecondRaise, v1.w[m], s1 / kSecondRaise);
        acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, parts[kPParts - 1], acc[m], 0, 0, 0);
      }
      acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen_f16(v0.w[m], s0, v1.w[m], s1), parts[0], acc[m], 0, 0, 0);
    }
  }
};

// A row's new key and value as codes.
template <int D> struct Fresh {
  uint32_t key[4][8];     // as the operand of lane group g
  uint32_t value[D / 4];  // by element
};

// Put the new token at offset `off` of its tile, held in registers, and the tile back.
template <int D>
CDB_DEVICE void append_token(const Kv8Cache& cache, const Fresh<D>& fresh, int64_t tile, int off, int r, int g,
                             int k_old, int k_now, int v_old, int v_now, KeyRegs<D>& k, ValueRegs<D>& v) {
  using K = KeyRegs<D>;
  using V = ValueRegs<D>;
  const bool k_grown = __builtin_amdgcn_readfirstlane(off != 0 && k_now != k_old);
  const bool v_grown = __builtin_amdgcn_readfirstlane(off != 0 && v_now != v_old);
  if (k_grown && r < off) {
    const float f = growth_of(k_old, k_now);
#pragma unroll
    for (int j = 0; j < K::kFull; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) k.w[j][i] = recode(k.w[j][i], f);
    if constexpr (K::kTail) {
      k.t[0] = recode(k.t[0], f);
      k.t[1] = recode(k.t[1], f);
    }
  }
#pragma unroll
  for (int j = 0; j < K::kFull; ++j) {
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(&fresh.key[g][4 * j]);
#pragma unroll
    for (int i = 0; i < 4; ++i) k.w[j][i] = r == off ? x[i] : k.w[j][i];
  }
  if constexpr (K::kTail) {
    k.t[0] = r == off ? fresh.key[g][4 * K::kFull] : k.t[0];
    k.t[1] = r == off ? fresh.key[g][4 * K::kFull + 1] : k.t[1];
  }
  const uint32_t before = tokens_below(off - 4 * g), here = tokens_below(off + 1 - 4 * g) & ~before;
  if (v_grown) {
    const float f = growth_of(v_old, v_now);
#pragma unroll
    for (int m = 0; m < V::kWords; ++m) v.w[m] = (v.w[m] & ~before) | (recode(v.w[m], f) & before);
  }
#pragma unroll
  for (int m = 0; m < V::kWords; ++m) {
    const int d = V::element(m, r);
    const uint32_t c = (fresh.value[d >> 2] >> (8 * (d & 3))) & 255u;
    v.w[m] = (v.w[m] & ~here) | (c * 0x01010101u & here);
  }
  const int64_t v_tile = tile + cache.plane_tiles;
  if (r == off || (k_grown && r < off)) k.store(cache.codes + tile * (kTile * D), r, g);
  if (here != 0 || (v_grown && before != 0)) v.store(cache.codes + v_tile * (kTile * D), r, g);
  if (r == 0 && g == 0) {
    cache.scales[tile] = (uint8_t)k_now;
    cache.scales[v_tile] = (uint8_t)v_now;
  }
}

template <typename T, int D, int STYLE>
__global__ void __launch_bounds__(64 * kWaves, (kDecodeWaves<T, D>)) kv8_decode_kernel(Kv8DecodeParams P) {
  constexpr bool kWide = sizeof(T) == 4;
  using Query = QueryRegs<D, kWide>;
  __shared__ __align__(32) uint32_t q_codes[Query::kWords];
  __shared__ int q_bytes[16];
  __shared__ __align__(16) Fresh<D> fresh;
  __shared__ float weights[16][kMaxChunks];
  __shared__ bool all_marked;
  extern __shared__ __align__(16) float join[];
  constexpr int kJoin = D + 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = P.cache.num_kv_heads;
  const int b = blockIdx.x / heads, kvh = blockIdx.x - b * heads;
  const int chunk = blockIdx.y;
  const int p = P.seqlens[b];
  T* out = static_cast<T*>(P.out) + ((int64_t)b * P.num_heads + (int64_t)kvh * P.group) * D;
  const int layer = P.cache_layer0 + (P.cache_layer == nullptr ? 0 : P.cache_layer[b]);
  const int trow = P.table_row == nullptr ? b : P.table_row[b];
  const bool bad = (int64_t)p >= ((int64_t)P.table_width << P.bs_log2) || (STYLE != 0 && p >= P.max_positions) ||
                   layer < 0 || layer >= P.cache.num_layers || trow < 0 || trow >= P.table_rows;
  if (p < 0 || bad) {
    if (chunk == 0)
      for (int i = threadIdx.x; i < P.group * D; i += 64 * kWaves) Elem<T>::store(out + i, p < 0 ? 0.f : NAN);
    return;
  }
  // A row with more chunks than the workspace has partials for takes longer ones.
  const int pieces = (p + kChunk) / kChunk;
  const int most_chunks = min(P.max_chunks, kMaxChunks);
  const int length = kChunk * ((pieces + most_chunks - 1) / most_chunks);
  const int first = chunk * length;
  if (first > p) return;
  const int chunks = (p + length) / length;
  const bool ends = chunk == chunks - 1;                       // the row's last tile is in this chunk
  const int whole = ends ? (p - first) >> 4 : length >> 4;     // tiles before it
  const int off = p & 15;
  const int32_t* table = P.block_table + (int64_t)trow * P.table_width;
  const int bs_mask = (1 << P.bs_log2) - 1;
  const int64_t angle = STYLE == 0 ? 0 : (int64_t)p * (D / 2);
  const int64_t plane = P.cache.plane_tiles * (kTile * D);
  auto tile_of = [&](int t, bool& lost) -> int64_t {
    const int block = table[t >> P.bs_log2];
    lost = block < 0 || block >= P.cache.pool_blocks;
    return P.cache.tile(layer, 0, lost ? 0 : block, kvh, (t & bs_mask) >> 4);
  };

  for (int slice = 0; slice < P.group; slice += 16) {
    const int cols = min(16, P.group - slice);
    // Opaque, so that nothing derived from the lane is kept over the loop (it takes one turn but for
    // groups of more than 16, and the registers are needed inside).
    int tid = threadIdx.x;
    __asm__ volatile("" : "+v"(tid));
    const int lane = tid & 63, r = lane & 15, g = lane >> 4;
    KeyRegs<D> k[2];
    ValueRegs<D> v[2];
    // Lane j looks up tile window + j of the chunk: where it lies, and its scales.
    int64_t where = 0;
    uint32_t bytes = 0;
    int count = 0;
    bool missing = false;
    auto look_up = [&](int window) __attribute__((always_inline)) {
      count = min(64, whole - window);
      bool lost = false;
      if (lane < count) {
        const int64_t tile = tile_of(first + (window + lane) * kTile, lost);
        bytes = P.cache.scales[tile] | (uint32_t)P.cache.scales[tile + P.cache.plane_tiles] << 8;
        where = tile * (kTile * D);
      }
      missing = missing || __ballot(lost) != 0;
    };
    auto codes_at = [&](int j) __attribute__((always_inline)) -> const uint8_t* {
      const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)where, j);
      const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(where >> 32), j);
      return P.cache.codes + (((uint64_t)hi << 32) | lo);
    };
    // The second tile of the last pair may be missing: the first stands in for it, with no probability.
    auto load_keys = [&](int pair, int on) __attribute__((always_inline)) {
      k[0].load(codes_at(2 * pair), r, g, on);
      k[1].load(codes_at(min(2 * pair + 1, count - 1)), r, g, on);
    };
    auto load_values = [&](int pair, int on) __attribute__((always_inline)) {
      v[0].load(codes_at(2 * pair) + plane, r, g, on);
      v[1].load(codes_at(min(2 * pair + 1, count - 1)) + plane, r, g, on);
    };
    const bool owner = ends && wave == kWaves - 1;
    // The wave that appends has its hands full: the others take the first kSkew pairs among themselves.
    const int start = owner ? kSkew + kWaves - 1 : wave;
    auto load_first = [&]() __attribute__((always_inline)) {
      if (2 * start < count) {
        load_keys(start, -1);
        __builtin_amdgcn_sched_barrier(0);  // keys before values, as in the steps: the waits count on it
        load_values(start, -1);
      }
    };
    look_up(0);
    // The row's last tile goes to the last wave, which has the fewest others. What a wave takes first is on
    // its way before the queries are turned.
    int64_t end_tile = 0;
    uint32_t end_k = 0, end_v = 0;
    bool lost_end = false;
    if (owner) {
      end_tile = tile_of(p & ~15, lost_end);
      k[0].load(P.cache.codes + end_tile * (kTile * D), r, g);
      v[0].load(P.cache.codes + end_tile * (kTile * D) + plane, r, g);
      end_k = P.cache.scales[end_tile];
      end_v = P.cache.scales[end_tile + P.cache.plane_tiles];
      missing = missing || lost_end;
    } else {
      load_first();
    }

    // A wave turns a head, two elements a lane. A query stays in LDS as e4m3 parts in the order of the key
    // operand, part i holding what the parts before it left, times 16^i.
    const int d = min(2 * lane, D - 2);
    const bool real = 2 * lane < D;
    const int turners = ends ? kWaves - 1 : kWaves;
    if (!owner) {
      for (int c = wave; c < cols; c += turners) {
        const int64_t h = kvh * P.group + slice + c;
        const T* bias = static_cast<const T*>(P.q_bias);
        float x[2];
        if (bias != nullptr) bias += h * D;
        load_rotated<T, D, STYLE, 2>(static_cast<const T*>(P.q) + (int64_t)b * P.q_stride + h * D, bias, P.cos + angle,
                                     P.sin + angle, d, P.vec, x);
        x[0] *= P.scale_log2;
        x[1] *= P.scale_log2;
        const float most = all_max(fmaxf(finite_abs(x[0]), finite_abs(x[1])));
        Query::store(q_codes, q_bytes, c, 2 * lane, real ? x[0] : 0.f, real ? x[1] : 0.f, most);
      }
    }
    lds_barrier();
    if (owner) {  // they have arrived by now
      end_k = scale_byte_read(end_k);
      end_v = scale_byte_read(end_v);
    }
    if (owner && slice == 0) {
      // The row's new key and value, as codes at the scale that their tile will have: this wave's alone.
      const T* bias = static_cast<const T*>(P.k_bias);
      const int64_t row = (int64_t)b * P.kv_stride + (int64_t)kvh * D;
      float x[2], y[2];
      load_f32<T, 2>(static_cast<const T*>(P.v_new) + row + d, y, P.vec);
      load_rotated<T, D, STYLE, 2>(static_cast<const T*>(P.k_new) + row, bias == nullptr ? nullptr : bias + kvh * D,
                                   P.cos + angle, P.sin + angle, d, P.vec, x);
      const int k_new = scale_byte(all_max(fmaxf(finite_abs(x[0]), finite_abs(x[1]))));
      const int v_new = scale_byte(all_max(fmaxf(finite_abs(y[0]), finite_abs(y[1]))));
      const int k_old = (int)end_k, v_old = (int)end_v;
      end_k = off != 0 ? max(k_new, k_old) : k_new;
      end_v = off != 0 ? max(v_new, v_old) : v_new;
      const float k_scale = scale_of(end_k), v_scale = scale_of(end_v);
      if (real) {
        const int at = KeyRegs<D>::place(d, 0);
        *reinterpret_cast<uint16_t*>(reinterpret_cast<uint8_t*>(fresh.key) + (at >> 9) * 32 + (at & 31)) =
            (uint16_t)codes_of(x[0], x[1], 0.f, 0.f, k_scale);
        *reinterpret_cast<uint16_t*>(reinterpret_cast<uint8_t*>(fresh.value) + d) =
            (uint16_t)codes_of(y[0], y[1], 0.f, 0.f, v_scale);
      }
      __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (!lost_end) append_token<D>(P.cache, fresh, end_tile, off, r, g, k_old, end_k, v_old, end_v, k[0], v[0]);
    }
    Query q;
    q.load(q_codes, q_bytes, cols, r, g);

    Attention<D, kWide> state;
    state.start();
    f16x8_t parts[Attention<D, kWide>::kPParts];
    f32x4_t s[2];
    if (owner) {
      end_v = __builtin_amdgcn_readfirstlane(end_v);  // the unit stays in scalar registers
      const uint32_t seen = tokens_below(off + 1 - 4 * g);  // what lies behind counts for nothing, NaN among it
#pragma unroll
      for (int m = 0; m < ValueRegs<D>::kWords; ++m) v[0].w[m] &= seen;
      v[1].clear();
      s[0] = state.scores(k[0], end_k, q, off + 1, g);
      s[1] = (f32x4_t){-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      state.softmax(s, parts);
      state.values(v[0], v[1], (int)end_v, (int)end_v, parts);
      load_first();
    }
    // The loads ahead are not left out at the end but read a line each: a branch around them would make the
    // wait for this pair's values one for the next pair's keys too.
    for (int window = 0; window < whole; window += 64) {
      if (window != 0) {
        look_up(window);
        load_first();
      }
      for (int pair = start; 2 * pair < count;) {
        const int next = pair + (ends && pair < kSkew ? kWaves - 1 : kWaves);
        const int on = 2 * next < count ? -1 : 0, ahead = on ? next : pair;
        const uint32_t b0 = __builtin_amdgcn_readlane((int)bytes, 2 * pair);
        const uint32_t b1 = __builtin_amdgcn_readlane((int)bytes, min(2 * pair + 1, count - 1));
        s[0] = state.scores(k[0], scale_byte_read(b0 & 255), q, kTile, g);
        s[1] = state.scores(k[1], scale_byte_read(b1 & 255), q, 2 * pair + 1 < count ? kTile : 0, g);
        load_keys(ahead, on);
        state.softmax(s, parts);
        state.values(v[0], v[1], (int)scale_byte_read(b0 >> 8), (int)scale_byte_read(b1 >> 8), parts);
        __builtin_amdgcn_sched_barrier(0);
        load_values(ahead, on);
        __builtin_amdgcn_sched_barrier(0);
        pair = next;
      }
    }

    // Join the waves: [wave][column][D + 2] holds O, the maximum and the sum.
    float sum = ldexpf(column_sum(state.sum), -state.kRaise);
    if (missing) sum = NAN;
    if (r < cols) {
      float* mine = join + (wave * cols + r) * kJoin;
      const int back = state.unit.back() - state.kRaise;
#pragma unroll
      for (int m = 0; m < D / 16; m += 2)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x2_t*>(mine + ValueRegs<D>::element(m, 4 * g + i)) =
              (f32x2_t){ldexpf(state.acc[m][i], back), ldexpf(state.acc[m + 1][i], back)};
      if (g == 0) {
        mine[D] = sum == 0.f ? -INFINITY : state.low;  // no key yet, or none above -infinity
        mine[D + 1] = sum;
      }
    }
    __syncthreads();
    for (int i = tid; i < cols * D; i += 64 * kWaves) {
      const int c = i / D, d = i - c * D;
      const float* part = join + c * kJoin;
      const int stride = cols * kJoin;
      float m4[kWaves], most = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        m4[w] = part[w * stride + D];
        most = fmaxf(most, m4[w]);
      }
      float o = 0.f, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(m4[w] - most);
        o = fmaf(f, part[w * stride + d], o);
        l = fmaf(f, part[w * stride + D + 1], l);
      }
      if (chunks == 1) {
        Elem<T>::store(out + (int64_t)slice * D + i, o / l);
      } else {
        const int h = kvh * P.group + slice + c;
        float* to = P.partials + (((int64_t)b * P.num_heads + h) * P.max_chunks + chunk) * (D + 2);
        __hip_atomic_store(to + d, o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (d == 0) {
          __hip_atomic_store(to + D, most, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          __hip_atomic_store(to + D + 1, l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
      }
    }
    if (chunks > 1) {
      // The workgroup that finds every chunk of the row marked whole joins them, in order. Partials and marks
      // are stored past the XCD's cache and each store is waited for, and a workgroup marks its own chunk
      // before it looks: whichever marks last sees all. (Several may; they store the same values.) The marks
      // are taken back for the next launch of a captured graph, which has the same tag.
      uint64_t* tags = P.tags + (((int64_t)b * heads + kvh) * P.slices + (slice >> 4)) * P.max_chunks;
      __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (wave == 0) {
        if (lane == 0) __hip_atomic_store(tags + chunk, P.tag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const bool whole_chunk =
            lane >= chunks || __hip_atomic_load(tags + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == P.tag;
        const bool all = __ballot(whole_chunk) == ~0ull;
        if (lane == 0) all_marked = all;
      }
      __syncthreads();
      if (all_marked) {
        const int h0 = kvh * P.group + slice;
        const float* rows = P.partials + ((int64_t)b * P.num_heads + h0) * P.max_chunks * (D + 2);
        // Weights of the chunks, a wave a head.
        for (int c = wave; c < cols; c += kWaves) {
          const float* x = rows + ((int64_t)c * P.max_chunks + min(lane, chunks - 1)) * (D + 2);
          const float m = lane < chunks ? __hip_atomic_load(x + D, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                                        : -INFINITY;
          const float l = __hip_atomic_load(x + D + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          const float f = __builtin_amdgcn_exp2f(m - wave_max(m));
          const float total = wave_sum(lane < chunks ? f * l : 0.f);
          weights[c][lane] = lane < chunks ? f / total : 0.f;
        }
        __syncthreads();
        for (int i = tid; i < cols * (D / 2); i += 64 * kWaves) {
          const int c = i / (D / 2), d = 2 * (i - c * (D / 2));
          const uint64_t* x = reinterpret_cast<const uint64_t*>(rows + (int64_t)c * P.max_chunks * (D + 2) + d);
          float o0 = 0.f, o1 = 0.f;
          for (int n = 0; n < chunks; n += 8) {
            uint64_t y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
              y[j] = __hip_atomic_load(x + (int64_t)min(n + j, chunks - 1) * ((D + 2) / 2), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float f = weights[c][min(n + j, 63)];
              if (n + j < chunks) {
                o0 = fmaf(f, __uint_as_float((uint32_t)y[j]), o0);
                o1 = fmaf(f, __uint_as_float((uint32_t)(y[j] >> 32)), o1);
              }
            }
          }
          T* to = out + (int64_t)(slice + c) * D + d;
          Elem<T>::store(to, o0);
          Elem<T>::store(to + 1, o1);
        }
        if (tid < chunks) __hip_atomic_store(tags + tid, (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    if (slice + 16 < P.group) __syncthreads();
  }
}

template <typename T, int D>
static int decode_dim(const Kv8DecodeParams& P, int style, hipStream_t stream) {
  const int64_t most = ((int64_t)P.table_width << P.bs_log2) / kChunk + 1;
  const dim3 grid((unsigned)(P.num_rows * P.cache.num_kv_heads), (unsigned)min((int64_t)P.max_chunks, most));
  const dim3 wg(64 * kWaves);
  const size_t lds = sizeof(float) * kWaves * min(P.group, 16) * (D + 4);
  if (style == 0) kv8_decode_kernel<T, D, 0><<<grid, wg, lds, stream>>>(P);
  else if (style == 1) kv8_decode_kernel<T, D, 1><<<grid, wg, lds, stream>>>(P);
  else kv8_decode_kernel<T, D, 2><<<grid, wg, lds, stream>>>(P);
  return hipGetLastError() == hipSuccess ? CDB_OK : CDB_ERR_HIP;
}

template <typename T> static int decode_type(const Kv8DecodeParams& P, int dim, int style, hipStream_t stream) {
  switch (dim) {
    case 64: return decode_dim<T, 64>(P, style, stream);
    case 96: return decode_dim<T, 96>(P, style, stream);
    case 128: return decode_dim<T, 128>(P, style, stream);
    default: return CDB_ERR_UNSUPPORTED;
  }
}

}  // namespace cdb

namespace cdb {

// Bytes of one row's partials and marks for one chunk.
static int64_t chunk_bytes(int32_t num_heads, int32_t num_kv_heads, int32_t head_dim) {
  const int64_t slices = ((int64_t)num_heads / num_kv_heads + 15) / 16;
  return (int64_t)num_heads * (head_dim + 2) * 4 + num_kv_heads * slices * 8;
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

extern "C" int64_t cdb_kv8_decode_workspace_bytes(int32_t num_rows, int32_t num_heads, int32_t num_kv_heads,
                                                  int32_t head_dim, int32_t max_seqlen) {
  if (num_rows < 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || max_seqlen <= 0) return -1;
  const int64_t chunks = min(((int64_t)max_seqlen + cdb::kChunk - 1) / cdb::kChunk, (int64_t)cdb::kMaxChunks);
  return max((int64_t)num_rows, (int64_t)1) * chunks * cdb::chunk_bytes(num_heads, num_kv_heads, head_dim);
}

extern "C" int cdb_kv8_decode_attention(const void* q, const void* k_new, const void* v_new, void* codes, void* scales,
                                        int32_t num_cache_layers, int64_t pool_blocks, const int32_t* cache_layer,
                                        int32_t cache_layer0, const int32_t* block_table, const int32_t* table_row,
                                        int32_t table_rows, int32_t table_width, const int32_t* seqlens,
                                        const float* rope_cos, const float* rope_sin, int32_t rope_style,
                                        int32_t max_positions, const void* q_bias, const void* k_bias, void* out,
                                        void* workspace, int64_t workspace_bytes, int32_t num_rows, int32_t num_heads,
                                        int32_t num_kv_heads, int32_t head_dim, int32_t block_size, float scale,
                                        int64_t q_stride, int64_t kv_stride, int32_t dtype, hipStream_t stream) {
  using namespace cdb;
  if (rope_style < 0 || rope_style > 2) return CDB_ERR_UNSUPPORTED;
  if (dtype != CDB_DTYPE_F32 && dtype != CDB_DTYPE_BF16) return CDB_ERR_UNSUPPORTED;
  if (num_rows < 0 || num_heads <= 0 || table_rows <= 0 || table_width <= 0) return CDB_ERR_SHAPE;
  if (num_rows == 0) return CDB_OK;
  if (q == nullptr || k_new == nullptr || v_new == nullptr || block_table == nullptr || seqlens == nullptr ||
      out == nullptr || workspace == nullptr)
    return CDB_ERR_NULL;
  if (rope_style != 0 && (rope_cos == nullptr || rope_sin == nullptr)) return CDB_ERR_NULL;
  if (rope_style != 0 && max_positions <= 0) return CDB_ERR_SHAPE;
  Kv8DecodeParams P{};
  const int code =
      kv8_cache_of(&P.cache, codes, scales, num_cache_layers, pool_blocks, num_kv_heads, head_dim, block_size);
  if (code != CDB_OK) return code;
  if (num_heads % num_kv_heads != 0 || (int64_t)num_rows * num_kv_heads > 0x7fffffffll) return CDB_ERR_SHAPE;
  if (table_row == nullptr && table_rows < num_rows) return CDB_ERR_SHAPE;
  if ((int64_t)table_width * block_size > (1ll << 30)) return CDB_ERR_SHAPE;
  if (!(scale > 0.f) || !(scale < INFINITY)) return CDB_ERR_SHAPE;
  if (q_stride == 0) q_stride = (int64_t)num_heads * head_dim;
  if (kv_stride == 0) kv_stride = (int64_t)num_kv_heads * head_dim;
  if (q_stride < (int64_t)num_heads * head_dim || kv_stride < (int64_t)num_kv_heads * head_dim) return CDB_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return CDB_ERR_SHAPE;
  const int64_t chunks = min(workspace_bytes / (num_rows * chunk_bytes(num_heads, num_kv_heads, head_dim)),
                             (int64_t)kMaxChunks);
  if (workspace_bytes < 0 || chunks < 1) return CDB_ERR_CAPACITY;
  const int size = dtype == CDB_DTYPE_F32 ? 4 : 2;
  P.q = q; P.k_new = k_new; P.v_new = v_new;
  P.cache_layer = cache_layer; P.cache_layer0 = cache_layer0;
  P.block_table = block_table; P.table_row = table_row; P.table_rows = table_rows; P.table_width = table_width;
  P.seqlens = seqlens; P.cos = rope_cos; P.sin = rope_sin;
  P.max_positions = rope_style != 0 ? max_positions : 0;
  P.bs_log2 = __builtin_ctz(block_size);
  P.q_bias = q_bias; P.k_bias = k_bias; P.out = out; P.partials = static_cast<float*>(workspace);
  P.max_chunks = (int32_t)chunks;
  P.slices = (num_heads / num_kv_heads + 15) / 16;
  P.tags = reinterpret_cast<uint64_t*>(P.partials + (int64_t)num_rows * num_heads * chunks * (head_dim + 2));
  P.tag = next_tag();
  P.num_rows = num_rows; P.num_heads = num_heads; P.group = num_heads / num_kv_heads;
  P.scale_log2 = scale * 1.4426950408889634f;
  P.q_stride = q_stride; P.kv_stride = kv_stride;
  P.vec = kv8_aligned(size, {q, k_new, v_new, q_bias, k_bias, rope_cos, rope_sin}, {q_stride, kv_stride});
  return dtype == CDB_DTYPE_F32 ? decode_type<float>(P, head_dim, rope_style, stream)
                                : decode_type<bf16_t>(P, head_dim, rope_style, stream);
}
