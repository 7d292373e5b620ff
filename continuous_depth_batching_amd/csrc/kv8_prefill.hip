// Varlen causal prefill attention over the 8-bit paged KV cache.
//
// One workgroup of 4 waves takes 128 query tokens of a sequence and one query head, a wave 32 of them, and walks
// the keys in blocks of 32, two tiles, with a running maximum and sum (the maximum moves only when a score outgrows
// it by 2^6). Codes go from memory to registers; each wave loads the next block's keys and values as soon as this
// block's are used up, so nothing waits on LDS or on another wave.
//   S^T = K Q^T in bf16: a code times a power of two is exact there, so scores are the products' fp32 sums.
//   O^T = V^T P^T in fp16, which holds a code exactly and P to 2^-11: it is raised by 2^9, so that keys down to 2^-23
//   of the query's largest keep that, and none is off by more than 2^-34 of it. Values widen with their scale, in a
//   unit that follows the tiles' scales. fp32 models: queries as 3 bf16 parts (2^-24), P as 2 fp16 parts (2^-23, and
//   2^-45 of the largest).
// A lane's 16 scores are those of the 16 tokens whose values it holds, so P never moves; queries are the columns of
// both products, so maximum and sum are a lane's own and its neighbour's, 32 lanes away.
//
// Bound: instruction issue. A wave's block takes 16 matrix instructions of 32 cycles and some 180 vector ones of 4
// (64 widen codes, 32 are fma and exponential): 512 cycles of a SIMD's matrix core and 770 of its issue, which the two
// waves of a SIMD hardly overlap (1270 a block). Measured (a launch from a graph, on cards whose clocks differ; the
// first launches after idling take up to 1060): two sequences of 6000..8190 tokens, 32 heads on 8 x 128, 870-950 us
// (860-940 TFLOP/s; a large bf16 product reaches 1199); 24 fresh prompts of 24..1300 tokens, 16 heads, 43-48 us, where
// the longest tile's chain of blocks is most of it; four chunks of some 110 tokens after 16000, cut in 8 parts,
// 107-117 us; one of 8000 in fp32, 1070-1205. Tried on one card, where these took 873, 47 and 113, and were slower or
// no faster: the scores on the codes themselves with queries of 3 e4m3 parts (876, 52 and 116 us); blocks staged in
// LDS, 5 ahead, at 3 waves a SIMD (845, 52 and 124); waves of one workgroup parting the keys of the same queries (927,
// 57 and 118); 64 queries a wave, which widens each code once for twice the queries but leaves one wave a SIMD (1024,
// 80 and 131); products and vector instructions interleaved by hand (957, 76 and 135); the tile list, longest first,
// from its end (957, 61 and 119); long tiles of fresh prompts in two parts (64).
#include "cdb_amd.h"
#include "kv8_common.h"
#include "kv8_host.h"

namespace cdb {

constexpr int kQueries = 128;  // query tokens of a tile: 32 a wave
constexpr int kMaxSplits = 64;  // parts of a tile's keys: a lane each in the merge

struct Kv8PrefillParams {
  const void* q;
  Kv8Cache cache;
  int64_t layer;
  const int32_t *block_table, *table_row, *cu_q, *past, *tile_seq, *tile_q0;
  int32_t table_rows, table_width, num_seqs, num_tiles, num_heads, group, bs_log2, splits;
  int64_t tokens;
  void* out;
  float* partials;
  float scale_log2;
};

// What a lane (c, h) = (lane % 32, lane / 32) holds of a block of 32 keys, two tiles: of the keys, 16-byte
// units 2j + h of token c; of the values, the words of groups h and h + 2 of each tile for its elements.
template <int D> struct BlockRegs {
  static constexpr int kUnits = D / 32, kWords = D / 32;
  u32x4_t k[kUnits];
  uint32_t v[2][2][kWords];  // [tile][group half][element]

  CDB_DEVICE void load_keys(const uint8_t* p) {
#pragma unroll
    for (int j = 0; j < kUnits; ++j) k[j] = *reinterpret_cast<const u32x4_t*>(p + j * 512);
  }
  CDB_DEVICE void load_values(int a, const uint8_t* tile, int c, int h) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if constexpr (D == 128) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(tile + 2 * s * (4 * D) + (h * (4 * D) + c * 16));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[a][s][i] = w[i];
      } else {
        const u32x2_t w = *reinterpret_cast<const u32x2_t*>(tile + 2 * s * (4 * D) + (h * (4 * D) + c * 8));
        v[a][s][0] = w[0];
        v[a][s][1] = w[1];
        if constexpr (D == 96)
          v[a][s][2] = *reinterpret_cast<const uint32_t*>(tile + 2 * s * (4 * D) + 256 + (h * (4 * D) + c * 4));
      }
    }
  }
  // Head element of row `row` of value product i.
  static CDB_DEVICE int value_element(int i, int row) {
    if constexpr (D == 128) return 4 * row + i;
    return i < 2 ? 2 * row + i : 64 + row;
  }
};

CDB_DEVICE float half_max(float v) {
  const f32x2_t x = pair32(v);
  return fmaxf(x[0], x[1]);
}

// A lane's share of 32 queries as the operand of the products with the keys: bf16 as it is, fp32 as 3 bf16 parts.
template <typename T, int D> struct BlockQuery {
  static constexpr int kParts = sizeof(T) == 4 ? 3 : 1, kSteps = D / 16;
  bf16x8_t w[kSteps][kParts];

  CDB_DEVICE void load(const T* q, int h) {
#pragma unroll
    for (int m = 0; m < kSteps; ++m) {
      const T* at = q + 32 * (m >> 1) + 16 * h + 8 * (m & 1);
      if constexpr (kParts == 1) {
        w[m][0] = *reinterpret_cast<const bf16x8_t*>(at);
      } else {
        float x[8];
        load_f32<T, 8>(at, x, true);
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const __bf16 y = (__bf16)x[i];
            w[m][p][i] = y;
            x[i] -= (float)y;
          }
      }
    }
  }
  CDB_DEVICE f32x16_t scores(const BlockRegs<D>& x, int k_byte) const {
    const float f = scale_of(k_byte);
    f32x16_t s;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
    for (int m = 0; m < kSteps; ++m) {
      const bf16x8_t k = widen_bf16(x.k[m >> 1][2 * (m & 1)], f, x.k[m >> 1][2 * (m & 1) + 1], f);
#pragma unroll
      for (int p = kParts - 1; p >= 0; --p) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, w[m][p], s, 0, 0, 0);
    }
    return s;
  }
};

// 0x80 in each byte of w that holds the NaN code.
CDB_DEVICE uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// How far scores may outgrow the maximum that the sums are counted from before they are counted anew, and what
// probabilities are raised by: 2^15 is then the largest, within fp16, and its smallest step, 2^-24, stands for 2^-33.
// Less slack moves more blocks (two sequences of 6000..8190 tokens: 908 us with 4, 900 with 6, 898 with 8).
// fp32 models raise by a product, which is exact: in the exponent it would cost one near 0 some of its bits.
constexpr float kSlack = 6.f, kRaise = 9.f;

// Waves a SIMD: three where the registers allow it (bf16 heads of 96 spill 2; 5000 tokens of 55 such heads took 360 us
// against 380); bf16 heads of 128 would spill 27, and take 904 and 125 us for 900 and 113.
template <typename T, int D> constexpr int kPrefillWaves = D == 64 || (sizeof(T) == 2 && D == 96) ? 3 : 2;

template <typename T, int D>
__global__ void __launch_bounds__(256, (kPrefillWaves<T, D>)) kv8_prefill_kernel(Kv8PrefillParams P) {
  using Regs = BlockRegs<D>;
  constexpr bool kWide = sizeof(T) == 4;
  constexpr int kPParts = kWide ? 2 : 1;
  constexpr int kTiles = D / 32;
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = P.cache.num_kv_heads;
  // KV heads vary fastest over the workgroups, so the query heads that share one meet on one XCD.
  const int kvh = blockIdx.x % heads;
  const int rest = blockIdx.x / heads;
  const int n = rest / P.group, head = kvh * P.group + rest % P.group;
  const int s = P.tile_seq[n];
  if (s < 0 || s >= P.num_seqs) return;
  const int64_t token0 = P.cu_q[s];
  const int num = P.cu_q[s + 1] - (int)token0, past = P.past[s];
  const int q0 = P.tile_q0[n], w0 = q0 + 32 * wave;
  if (token0 < 0 || num < 0 || token0 + num > P.tokens || past < 0 || q0 < 0 || q0 >= num || w0 >= num) return;
  const int query = w0 + c, pos = past + query;
  const int64_t total = (int64_t)past + num;
  const int trow = P.table_row[s];
  const bool bad = total > ((int64_t)P.table_width << P.bs_log2) || trow < 0 || trow >= P.table_rows;

  // Blocks of 32 keys: the tile's, this part's of them, and of those the ones that the wave's queries see.
  const int blocks = (past + min(q0 + kQueries, num) + 31) / 32;
  const int part = blockIdx.y, parts = P.splits;
  const int from = parts == 1 ? 0 : (uint32_t)blocks * part / parts;
  const int end = parts == 1 ? blocks : (int)((uint32_t)blocks * (part + 1) / parts);
  const int to = bad ? 0 : min(end, (past + min(w0 + 32, num) + 31) / 32);

  BlockQuery<T, D> q;
  q.load(static_cast<const T*>(P.q) + ((token0 + min(query, num - 1)) * P.num_heads + head) * D, h);
  f32x16_t acc[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
  // Scores are counted, in units of log2, from -`shift`, anew once they pass `limit`.
  float shift = 0.f, limit = -INFINITY, sum = 0.f;
  ValueUnit<T> unit;  // that the accumulators are counted in
  bool missing = bad;
  const int32_t* table = P.block_table + (int64_t)(bad ? 0 : trow) * P.table_width;
  const int bs_mask = (1 << P.bs_log2) - 1;
  const int64_t plane = P.cache.plane_tiles * (kTile * D);

  for (int window = from; window < to; window += 32) {
    const int count = min(32, to - window);
    // Lane j looks up tile j of the window; for one past the sequence its last, masked.
    int64_t where = 0;
    uint32_t bytes = 0x0101u;
    bool lost = false;
    if (lane < 2 * count) {
      const int t = min(window * 32 + lane * kTile, (int)total - 1);
      const int block = table[t >> P.bs_log2];
      lost = block < 0 || block >= P.cache.pool_blocks;
      const int64_t tile = P.cache.tile(P.layer, 0, lost ? 0 : block, kvh, (t & bs_mask) >> 4);
      bytes = scale_byte_read(P.cache.scales[tile]) | scale_byte_read(P.cache.scales[tile + P.cache.plane_tiles]) << 8;
      where = tile * (kTile * D);
    }
    missing = missing || __ballot(lost) != 0;
    auto codes_at = [&](int j) __attribute__((always_inline)) -> const uint8_t* {
      const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)where, j);
      const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(where >> 32), j);
      return P.cache.codes + (((uint64_t)hi << 32) | lo);
    };
    Regs x;
    auto load_keys = [&](int i) __attribute__((always_inline)) {
      const uint8_t *t0 = codes_at(2 * i), *t1 = codes_at(2 * i + 1);
      x.load_keys((c & 16 ? t1 : t0) + ((c & 15) * 16 + h * 256));
    };
    auto load_values = [&](int i) __attribute__((always_inline)) {
      x.load_values(0, codes_at(2 * i) + plane, c, h);
      x.load_values(1, codes_at(2 * i + 1) + plane, c, h);
    };
    load_keys(0);
    __builtin_amdgcn_sched_barrier(0);
    load_values(0);
    for (int i = 0; i < count; ++i) {
      // The loads ahead repeat the last block at the end: a branch around them would make the wait for this
      // block's values one for the next block's keys too.
      const int ahead = min(i + 1, count - 1);
      const int key0 = (window + i) * 32;
      const uint32_t b0 = __builtin_amdgcn_readlane((int)bytes, 2 * i);
      const uint32_t b1 = __builtin_amdgcn_readlane((int)bytes, 2 * i + 1);
      f32x16_t sc = q.scores(x, (int)((c & 16 ? b1 : b0) & 255));
      load_keys(ahead);
      const bool diagonal = key0 + 31 > past + w0;  // some query of the wave does not see some key of the block
      if (diagonal) {
        __asm__ volatile("");  // keeps this a branch: most blocks have nothing to mask
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (key0 + (e >> 2) * 8 + 4 * h + (e & 3) > pos) sc[e] = -INFINITY;
      }
      float most = sc[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) most = fmaxf(most, sc[e]);
      if (__any(most * P.scale_log2 > limit)) {
        most = half_max(most) * P.scale_log2;
        const bool more = most > limit;
        const float moved = (!kWide && fabsf(most) < kWideScore ? kRaise : 0.f) - most;
        const float keep = more && limit != -INFINITY ? __builtin_amdgcn_exp2f(moved - shift) : 1.f;
        sum *= keep;  // the first count finds zeros
#pragma unroll
        for (int m = 0; m < kTiles; ++m) acc[m] *= keep;
        shift = more ? moved : shift;
        limit = more ? most + kSlack : limit;
      }
      if (__any(fabsf(shift) >= kWideScore)) {
        // Rounded as the maximum was, so that the difference is exact: a fused product keeps what here is many units.
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = __builtin_amdgcn_exp2f(add_rn(mul_rn(sc[e], P.scale_log2), shift));
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], P.scale_log2, shift));
      }
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const int t = key0 + kTile * a;
        const int v_exp = (int)((a ? b1 : b0) >> 8);
        if (unit.moves(v_exp)) {
          const int by = unit.move(v_exp);
#pragma unroll
          for (int m = 0; m < kTiles; ++m)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[m][e] = ldexpf(acc[m][e], by);
        }
        const float v_scale = unit.scale(v_exp);
        f16x8_t pp[kPParts];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          constexpr float kTimes = kWide ? 0x1p9f : 1.f;
          const f32x2_t x2 = {sc[8 * a + e] * kTimes, sc[8 * a + e + 1] * kTimes};
          const f16x2_t y = __builtin_convertvector(x2, f16x2_t);
          pp[0][e] = y[0];
          pp[0][e + 1] = y[1];
          if constexpr (kWide) {
            sum += x2[0];
            sum += x2[1];
            const f16x2_t z = __builtin_convertvector(
                (f32x2_t){(x2[0] - (float)y[0]) * kSecondRaise, (x2[1] - (float)y[1]) * kSecondRaise}, f16x2_t);
            pp[kPParts - 1][e] = z[0];
            pp[kPParts - 1][e + 1] = z[1];
          } else {
            sum = __builtin_amdgcn_fdot2(y, (f16x2_t){(_Float16)1.f, (_Float16)1.f}, sum, false);
          }
        }
        if (diagonal) {
          // A value counts only for the queries that see its token: codes behind the sequence are taken out,
          // and so are NaN codes, which a probability of zero would not keep from the other queries; those that
          // do see one get it by a product of where NaN is with what is seen.
          uint32_t any_nan = 0;
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int m = 0; m < Regs::kWords; ++m) {
              uint32_t& w = x.v[a][g][m];
              w &= tokens_below((int)(total - t) - 4 * (h + 2 * g));
              any_nan |= nan_bytes(w);
            }
          if (__any(any_nan != 0)) {
            f16x8_t seen;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              seen[e] = t + (e >> 2) * 8 + 4 * h + (e & 3) <= pos ? (_Float16)1.f : (_Float16)0.f;
#pragma unroll
            for (int m = 0; m < kTiles; ++m) {
              uint32_t where_nan[2];
#pragma unroll
              for (int g = 0; g < 2; ++g) {
                const uint32_t hit = nan_bytes(x.v[a][g][m]) >> 7;  // 1 in each such byte
                where_nan[g] = hit * 0x38u;                         // the code of 1
                x.v[a][g][m] &= ~(hit * 0xffu);
              }
              f32x16_t met;
#pragma unroll
              for (int e = 0; e < 16; ++e) met[e] = 0.f;
              const f16x8_t ones = widen_f16(where_nan[0], 1.f, where_nan[1], 1.f);
              met = __builtin_amdgcn_mfma_f32_32x32x16_f16(ones, seen, met, 0, 0, 0);
#pragma unroll
              for (int e = 0; e < 16; ++e) acc[m][e] = met[e] != 0.f ? NAN : acc[m][e];
            }
          }
        }
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
          if constexpr (kWide) {
            const float s2 = v_scale / kSecondRaise;
            const f16x8_t v2 = widen_f16(x.v[a][0][m], s2, x.v[a][1][m], s2);
            acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v2, pp[kPParts - 1], acc[m], 0, 0, 0);
          }
          const f16x8_t v = widen_f16(x.v[a][0][m], v_scale, x.v[a][1][m], v_scale);
          acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pp[0], acc[m], 0, 0, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      load_values(ahead);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  sum += shfl_xor_f32(sum, 32);
  const float top = sum == 0.f ? -INFINITY : -shift;  // a query that has seen no key
  if (missing) sum = NAN;
  if (query >= num) return;
  if (P.splits == 1) {
    T* out = static_cast<T*>(P.out) + ((token0 + query) * P.num_heads + head) * D;
    const float inv = 1.f / sum;
#pragma unroll
    for (int m = 0; m < kTiles; ++m)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        Elem<T>::store(out + Regs::value_element(m, (e >> 2) * 8 + 4 * h + (e & 3)),
                       ldexpf(acc[m][e] * inv, unit.back()));
    return;
  }
  float* to_part = P.partials +
                   ((((int64_t)n * P.splits + part) * P.num_heads + head) * kQueries + (query - q0)) * (D + 2);
#pragma unroll
  for (int m = 0; m < kTiles; ++m)
#pragma unroll
    for (int e = 0; e < 16; ++e) to_part[Regs::value_element(m, (e >> 2) * 8 + 4 * h + (e & 3))] =
        ldexpf(acc[m][e], unit.back() - (int)kRaise);
  if (h == 0) {
    to_part[D] = top;
    to_part[D + 1] = ldexpf(sum, -(int)kRaise);
  }
}

// One wave joins the parts of a query and head, in order.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv8_prefill_merge_kernel(Kv8PrefillParams P) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int head = (int)(item % P.num_heads);
  const int64_t rest = item / P.num_heads;
  const int n = (int)(rest / kQueries), i = (int)(rest % kQueries);
  if (n >= P.num_tiles) return;
  const int s = P.tile_seq[n];
  if (s < 0 || s >= P.num_seqs) return;
  const int64_t token0 = P.cu_q[s];
  const int num = P.cu_q[s + 1] - (int)token0, query = P.tile_q0[n] + i;
  if (token0 < 0 || num < 0 || token0 + num > P.tokens || P.past[s] < 0 || P.tile_q0[n] < 0 || P.tile_q0[n] >= num ||
      query >= num)
    return;
  const int64_t stride = (int64_t)P.num_heads * kQueries * (D + 2);
  const float* x = P.partials + (((int64_t)n * P.splits * P.num_heads + head) * kQueries + i) * (D + 2);
  // Lane p weighs part p; every lane then joins two elements.
  float top = -INFINITY, l = 0.f;
  if (lane < P.splits) {
    const f32x2_t y = *reinterpret_cast<const f32x2_t*>(x + lane * stride + D);
    top = y[0];
    l = y[1];
  }
  const float f = __builtin_amdgcn_exp2f(top - wave_max(top));
  l = wave_sum(f * l);
  if (2 * lane >= D) return;
  f32x2_t o = {0.f, 0.f};
#pragma unroll 4
  for (int p = 0; p < P.splits; ++p) {
    const f32x2_t y = *reinterpret_cast<const f32x2_t*>(x + p * stride + 2 * lane);
    const float g = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), p));
    o[0] = fmaf(g, y[0], o[0]);
    o[1] = fmaf(g, y[1], o[1]);
  }
  T* out = static_cast<T*>(P.out) + ((token0 + query) * P.num_heads + head) * D + 2 * lane;
  Elem<T>::store(out, o[0] / l);
  Elem<T>::store(out + 1, o[1] / l);
}

template <typename T, int D> static int prefill_dim(const Kv8PrefillParams& P, hipStream_t stream) {
  const int64_t items = (int64_t)P.num_tiles * P.num_heads;
  kv8_prefill_kernel<T, D><<<dim3((unsigned)items, (unsigned)P.splits), dim3(256), 0, stream>>>(P);
  if (hipGetLastError() != hipSuccess) return CDB_ERR_HIP;
  if (P.splits == 1) return CDB_OK;
  kv8_prefill_merge_kernel<T, D><<<dim3((unsigned)(items * (kQueries / 4))), dim3(256), 0, stream>>>(P);
  return hipGetLastError() == hipSuccess ? CDB_OK : CDB_ERR_HIP;
}

template <typename T> static int prefill_type(const Kv8PrefillParams& P, int dim, hipStream_t stream) {
  switch (dim) {
    case 64: return prefill_dim<T, 64>(P, stream);
    case 96: return prefill_dim<T, 96>(P, stream);
    case 128: return prefill_dim<T, 128>(P, stream);
    default: return CDB_ERR_UNSUPPORTED;
  }
}

}  // namespace cdb

extern "C" int64_t cdb_kv8_prefill_workspace_bytes(int32_t num_tiles, int32_t splits, int32_t num_heads,
                                                   int32_t head_dim) {
  if (num_tiles < 0 || splits <= 0 || splits > cdb::kMaxSplits || num_heads <= 0 || head_dim <= 0) return -1;
  return splits == 1 ? 0 : (int64_t)num_tiles * splits * num_heads * cdb::kQueries * (head_dim + 2) * 4;
}

extern "C" int cdb_kv8_prefill_attention(const void* q, const void* codes, const void* scales,
                                         int32_t num_cache_layers, int64_t pool_blocks, int32_t layer,
                                         const int32_t* block_table, const int32_t* table_row, int32_t table_rows,
                                         int32_t table_width, const int32_t* cu_q, const int32_t* past,
                                         int32_t num_seqs, const int32_t* tile_seq, const int32_t* tile_q0,
                                         int32_t num_tiles, void* out, int64_t tokens, int32_t splits, void* workspace,
                                         int64_t workspace_bytes, int32_t num_heads, int32_t num_kv_heads,
                                         int32_t head_dim, int32_t block_size, float scale, int32_t dtype,
                                         hipStream_t stream) {
  using namespace cdb;
  if (dtype != CDB_DTYPE_F32 && dtype != CDB_DTYPE_BF16) return CDB_ERR_UNSUPPORTED;
  if (num_seqs < 0 || num_tiles < 0 || tokens < 0 || num_heads <= 0 || table_rows <= 0 || table_width <= 0 ||
      layer < 0 || layer >= num_cache_layers || splits <= 0 || splits > kMaxSplits || tokens > 0x7fffff00ll)
    return CDB_ERR_SHAPE;
  if (num_seqs == 0 || num_tiles == 0 || tokens == 0) return CDB_OK;
  if (q == nullptr || out == nullptr || block_table == nullptr || table_row == nullptr || cu_q == nullptr ||
      past == nullptr || tile_seq == nullptr || tile_q0 == nullptr || (splits > 1 && workspace == nullptr))
    return CDB_ERR_NULL;
  Kv8PrefillParams P{};
  const int code = kv8_cache_of(&P.cache, const_cast<void*>(codes), const_cast<void*>(scales), num_cache_layers,
                                pool_blocks, num_kv_heads, head_dim, block_size);
  if (code != CDB_OK) return code;
  if (num_heads % num_kv_heads != 0 || (int64_t)num_tiles * num_heads * (kQueries / 4) > 0x7fffffffll)
    return CDB_ERR_SHAPE;
  if ((int64_t)table_width * block_size > (1ll << 30)) return CDB_ERR_SHAPE;
  if (!(scale > 0.f) || !(scale < INFINITY)) return CDB_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(q) % 16 != 0 || reinterpret_cast<uintptr_t>(out) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return CDB_ERR_SHAPE;
  if (workspace_bytes < cdb_kv8_prefill_workspace_bytes(num_tiles, splits, num_heads, head_dim))
    return CDB_ERR_CAPACITY;
  P.q = q; P.layer = layer;
  P.block_table = block_table; P.table_row = table_row; P.cu_q = cu_q; P.past = past;
  P.tile_seq = tile_seq; P.tile_q0 = tile_q0;
  P.table_rows = table_rows; P.table_width = table_width; P.num_seqs = num_seqs; P.num_tiles = num_tiles;
  P.num_heads = num_heads; P.group = num_heads / num_kv_heads; P.bs_log2 = __builtin_ctz(block_size);
  P.splits = splits; P.tokens = tokens; P.out = out; P.partials = static_cast<float*>(workspace);
  P.scale_log2 = scale * 1.4426950408889634f;
  return dtype == CDB_DTYPE_F32 ? prefill_type<float>(P, head_dim, stream) : prefill_type<bf16_t>(P, head_dim, stream);
}
