// Decode attention over the 8-bit paged KV cache, with fused rotation and append.
//
// One workgroup of 4 waves takes one chunk of one row and KV head, with all query heads that share
// it; a wave takes every fourth pair of 16-token tiles, keeps a running maximum and sum of its own,
// and the waves are joined through LDS, the chunks through fp32 partials. Bytes from HBM bound it, so
// the arithmetic goes where it costs least:
//   S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16, 16 query heads a product (unused
//   columns are zero): the codes widen to bf16 with their tile's scale in one instruction a pair
//   and exactly, and a lane's four scores are the four tokens it holds of V, so P never moves.
//   The query and P, which bf16 does not hold exactly, are taken as sums of 2 bf16 parts (3 for
//   fp32 models): what is rounded is then 2^-17 (2^-25) of a value, below the output's rounding.
#include "cdb_amd.h"
#include "kv8_common.h"
#include "kv8_host.h"

namespace cdb {

constexpr int kChunk = 256;  // tokens of a workgroup's chunk

struct Kv8DecodeParams {
  const void *q, *k_new, *v_new;
  Kv8Cache cache;
  const int32_t *cache_layer, *block_table, *table_row, *seqlens;
  int32_t cache_layer0, table_rows, table_width, max_positions, bs_log2;
  const float *cos, *sin;
  const void *q_bias, *k_bias;
  void* out;
  float* partials;
  int32_t max_chunks, num_rows, num_heads, group;
  float scale_log2;
  int64_t q_stride, kv_stride;
  bool vec;
};

// Elements of a lane's share of a 16-token tile: kUnits16 16-byte pieces, then 8 bytes for the last
// 32 elements of a head of 96.
template <int D> struct TileRegs {
  static constexpr int kFull = D / 64;
  static constexpr bool kTail = D % 64 != 0;
  u32x4_t k[kFull], v[kFull];
  u32x2_t kt, vt;

  CDB_DEVICE void load(const uint8_t* kp, const uint8_t* vp, int r, int g) {
#pragma unroll
    for (int j = 0; j < kFull; ++j) {
      k[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(kp + j * 1024 + (g * 16 + r) * 16));
      v[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(vp + g * (4 * D) + j * 256 + r * 16));
    }
    if constexpr (kTail) {
      kt = *reinterpret_cast<const u32x2_t*>(kp + kFull * 1024 + (g >> 1) * 256 + r * 16 + (g & 1) * 8);
      vt = *reinterpret_cast<const u32x2_t*>(vp + g * (4 * D) + kFull * 256 + r * 8);
    }
  }
  CDB_DEVICE void store_keys(uint8_t* kp, int r, int g) const {
#pragma unroll
    for (int j = 0; j < kFull; ++j) *reinterpret_cast<u32x4_t*>(kp + j * 1024 + (g * 16 + r) * 16) = k[j];
    if constexpr (kTail)
      *reinterpret_cast<u32x2_t*>(kp + kFull * 1024 + (g >> 1) * 256 + r * 16 + (g & 1) * 8) = kt;
  }
  CDB_DEVICE void store_values(uint8_t* vp, int r, int g) const {
#pragma unroll
    for (int j = 0; j < kFull; ++j) *reinterpret_cast<u32x4_t*>(vp + g * (4 * D) + j * 256 + r * 16) = v[j];
    if constexpr (kTail) *reinterpret_cast<u32x2_t*>(vp + g * (4 * D) + kFull * 256 + r * 8) = vt;
  }
  CDB_DEVICE void clear() {
#pragma unroll
    for (int j = 0; j < kFull; ++j) k[j] = v[j] = (u32x4_t){0, 0, 0, 0};
    if constexpr (kTail) kt = vt = (u32x2_t){0, 0};
  }
  // Words 2h, 2h + 1 of the keys of product m = 2j + h; the tail is the last product.
  CDB_DEVICE uint32_t key_word(int m, int i) const {
    if constexpr (kTail)
      if (m == 2 * kFull) return kt[i];
    return k[m >> 1][2 * (m & 1) + i];
  }
  // First element of a lane group's run of 8 in product m.
  static CDB_DEVICE int key_element(int m, int g) {
    return m < 2 * kFull ? 64 * (m >> 1) + 16 * g + 8 * (m & 1) : 64 * kFull + 8 * g;
  }
  CDB_DEVICE uint32_t value_word(int m) const {
    if constexpr (kTail)
      if (m >= 4 * kFull) return vt[m - 4 * kFull];
    return v[m >> 2][m & 3];
  }
  // Output element of accumulator register i of value product m.
  static CDB_DEVICE int value_element(int m, int g, int i) {
    return m < 4 * kFull ? 64 * (m >> 2) + 4 * (4 * g + i) + (m & 3) : 64 * kFull + 2 * (4 * g + i) + (m - 4 * kFull);
  }
};

// x as a sum of kParts bf16 values, 8 at a time.
template <int kParts> CDB_DEVICE void split_bf16(const float* x, bf16x8_t* out) {
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __bf16 b = (__bf16)rest[i];
      out[p][i] = b;
      rest[i] -= (float)b;
    }
  }
}

template <typename T, int D, int STYLE>
__global__ void __launch_bounds__(256) kv8_decode_kernel(Kv8DecodeParams P) {
  using Regs = TileRegs<D>;
  constexpr int kQParts = sizeof(T) == 4 ? 3 : 2, kPParts = kQParts;
  constexpr int kKeySteps = D / 32, kValueTiles = D / 16;
  extern __shared__ float lds[];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
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
      for (int i = tid; i < P.group * D; i += 256) Elem<T>::store(out + i, p < 0 ? 0.f : NAN);
    return;
  }
  // A row with more chunks than the workspace has partials for takes longer ones.
  const int pieces = (p + kChunk) / kChunk;
  const int length = kChunk * ((pieces + P.max_chunks - 1) / P.max_chunks);
  const int first = chunk * length;
  if (first > p) return;
  const int chunks = (p + length) / length;
  const int tiles = (min(length, p + 1 - first) + kTile - 1) / kTile;
  const int last = (p - first) >> 4;  // the tile the row appends to, counted in this chunk
  const int off = p & 15;
  const int32_t* table = P.block_table + (int64_t)trow * P.table_width;
  const int bs_mask = (1 << P.bs_log2) - 1;
  const int64_t angle = STYLE == 0 ? 0 : (int64_t)p * (D / 2);

  for (int slice = 0; slice < P.group; slice += 16) {
    const int cols = min(16, P.group - slice);
    if (slice != 0) {
      __threadfence_block();
      __syncthreads();
    }
    bf16x8_t q[kKeySteps][kQParts];
    {
      const int h = kvh * P.group + slice + min(r, cols - 1);
      const T* src = static_cast<const T*>(P.q) + (int64_t)b * P.q_stride + (int64_t)h * D;
      const T* bias = P.q_bias == nullptr ? nullptr : static_cast<const T*>(P.q_bias) + (int64_t)h * D;
#pragma unroll
      for (int m = 0; m < kKeySteps; ++m) {
        float x[8];
        load_rotated<T, D, STYLE, 8>(src, bias, P.cos + angle, P.sin + angle, Regs::key_element(m, g), P.vec, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = r < cols ? x[i] * P.scale_log2 : 0.f;
        split_bf16<kQParts>(x, q[m]);
      }
    }
    float top = -INFINITY, sum = 0.f;
    f32x4_t acc[kValueTiles];
#pragma unroll
    for (int m = 0; m < kValueTiles; ++m) acc[m] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    bool missing = false;

    for (int window = 0; window < tiles; window += 64) {
      // Lane j looks up tile window + j: where it lies, and its scales.
      const int count = min(64, tiles - window);
      int64_t where = 0;
      uint32_t k_byte = 0, v_byte = 0;
      bool lost = false;
      if (lane < count) {
        const int t = first + (window + lane) * kTile;
        const int block = table[t >> P.bs_log2];
        lost = block < 0 || block >= P.cache.pool_blocks;
        where = P.cache.tile(layer, 0, lost ? 0 : block, kvh, (t & bs_mask) >> 4);
        k_byte = P.cache.scales[where];
        v_byte = P.cache.scales[where + P.cache.plane_tiles];
      }
      const uint64_t lost_mask = __ballot(lost);
      missing = missing || lost_mask != 0;
      auto tile_at = [&](int j) -> int64_t {
        const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)where, j);
        const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(where >> 32), j);
        return (int64_t)(((uint64_t)hi << 32) | lo);
      };
      auto load = [&](Regs* regs, int pair) {
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const int j = 2 * pair + a;
          if (j < count) {
            const int64_t tile = tile_at(j);
            regs[a].load(P.cache.codes + tile * (kTile * D), P.cache.codes + (tile + P.cache.plane_tiles) * (kTile * D),
                         r, g);
          } else {
            regs[a].clear();
          }
        }
      };
      Regs cur[2], next[2];
      if (2 * wave < count) load(cur, wave);
      for (int pair = wave; 2 * pair < count; pair += 4) {
        if (2 * (pair + 4) < count) load(next, pair + 4);
        float k_scale[2], v_scale[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const int j = min(2 * pair + a, 63);
          k_scale[a] = scale_of(__builtin_amdgcn_readlane((int)k_byte, j));
          v_scale[a] = scale_of(__builtin_amdgcn_readlane((int)v_byte, j));
        }
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const int j = 2 * pair + a;
          if (window + j != last) continue;
          if (slice == 0 && !((lost_mask >> j) & 1)) {
            // Append: the tile is in this wave's registers, and no other wave reads it.
            const int64_t tile = tile_at(j);
            const T* k_src = static_cast<const T*>(P.k_new) + (int64_t)b * P.kv_stride + (int64_t)kvh * D;
            const T* v_src = static_cast<const T*>(P.v_new) + (int64_t)b * P.kv_stride + (int64_t)kvh * D;
            const T* bias = P.k_bias == nullptr ? nullptr : static_cast<const T*>(P.k_bias) + (int64_t)kvh * D;
            float x[kKeySteps][8], y[kValueTiles];
            float k_top = 0.f, v_top = 0.f;
#pragma unroll
            for (int m = 0; m < kKeySteps; ++m) {
              load_rotated<T, D, STYLE, 8>(k_src, bias, P.cos + angle, P.sin + angle, Regs::key_element(m, g), P.vec,
                                           x[m]);
#pragma unroll
              for (int i = 0; i < 8; ++i) k_top = fmaxf(k_top, finite_abs(x[m][i]));
            }
#pragma unroll
            for (int m = 0; m < kValueTiles; ++m) {
              const int d = m < 4 * Regs::kFull ? 64 * (m >> 2) + 4 * r + (m & 3)
                                                : 64 * Regs::kFull + 2 * r + (m - 4 * Regs::kFull);
              y[m] = Elem<T>::load(v_src + d);
              v_top = fmaxf(v_top, finite_abs(y[m]));
            }
            const int k_old = min((int)__builtin_amdgcn_readlane((int)k_byte, j), 254);
            const int v_old = min((int)__builtin_amdgcn_readlane((int)v_byte, j), 254);
            int k_now = __builtin_amdgcn_readfirstlane(scale_byte(wave_max(k_top)));
            int v_now = __builtin_amdgcn_readfirstlane(scale_byte(wave_max(v_top)));
            if (off != 0) {
              k_now = max(k_now, k_old);
              v_now = max(v_now, v_old);
            }
            const float k_inv = inverse_scale_of(k_now), v_inv = inverse_scale_of(v_now);
            const bool k_grown = off != 0 && k_now != k_old, v_grown = off != 0 && v_now != v_old;
            const float k_f = recode_factor(k_old, k_now), v_f = recode_factor(v_old, v_now);
            const uint32_t before = tokens_below(off - 4 * g), here = tokens_below(off + 1 - 4 * g) & ~before;
            if (k_grown && r < off) {
#pragma unroll
              for (int w = 0; w < Regs::kFull; ++w)
#pragma unroll
                for (int i = 0; i < 4; ++i) cur[a].k[w][i] = recode(cur[a].k[w][i], k_f);
              if constexpr (Regs::kTail)
#pragma unroll
                for (int i = 0; i < 2; ++i) cur[a].kt[i] = recode(cur[a].kt[i], k_f);
            }
            if (r == off) {
#pragma unroll
              for (int m = 0; m < kKeySteps; ++m)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  const uint32_t w = codes_of(mul_rn(x[m][4 * i], k_inv), mul_rn(x[m][4 * i + 1], k_inv),
                                              mul_rn(x[m][4 * i + 2], k_inv), mul_rn(x[m][4 * i + 3], k_inv));
                  if (m < 2 * Regs::kFull) cur[a].k[m >> 1][2 * (m & 1) + i] = w;
                  else cur[a].kt[i] = w;
                }
            }
            auto put = [&](uint32_t w, float v) {
              const float s = mul_rn(v, v_inv);
              if (v_grown) w = (w & ~before) | (recode(w, v_f) & before);
              return (w & ~here) | (codes_of(s, s, s, s) & here);
            };
#pragma unroll
            for (int m = 0; m < kValueTiles; ++m) {
              if (m < 4 * Regs::kFull) cur[a].v[m >> 2][m & 3] = put(cur[a].v[m >> 2][m & 3], y[m]);
              else cur[a].vt[m - 4 * Regs::kFull] = put(cur[a].vt[m - 4 * Regs::kFull], y[m]);
            }
            uint8_t* k_at = P.cache.codes + tile * (kTile * D);
            uint8_t* v_at = P.cache.codes + (tile + P.cache.plane_tiles) * (kTile * D);
            if (r == off || (k_grown && r < off)) cur[a].store_keys(k_at, r, g);
            if (here != 0 || (v_grown && before != 0)) cur[a].store_values(v_at, r, g);
            if (lane == 0) {
              P.cache.scales[tile] = (uint8_t)k_now;
              P.cache.scales[tile + P.cache.plane_tiles] = (uint8_t)v_now;
            }
            k_scale[a] = scale_of(k_now);
            v_scale[a] = scale_of(v_now);
          }
          // Codes behind the new token count for nothing, NaN among them.
          const uint32_t seen = tokens_below(off + 1 - 4 * g);
#pragma unroll
          for (int w = 0; w < Regs::kFull; ++w)
#pragma unroll
            for (int i = 0; i < 4; ++i) cur[a].v[w][i] &= seen;
          if constexpr (Regs::kTail) {
            cur[a].vt[0] &= seen;
            cur[a].vt[1] &= seen;
          }
        }

        f32x4_t s[2];
        float most = top;
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          s[a] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int m = 0; m < kKeySteps; ++m) {
            const bf16x8_t k = widen_bf16(cur[a].key_word(m, 0), k_scale[a], cur[a].key_word(m, 1), k_scale[a]);
#pragma unroll
            for (int part = kQParts - 1; part >= 0; --part)
              s[a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[m][part], s[a], 0, 0, 0);
          }
          if (window + 2 * pair + a >= last) {
            const int keep = window + 2 * pair + a == last ? off - 4 * g : -1;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[a][i] = i <= keep ? s[a][i] : -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) most = fmaxf(most, s[a][i]);
        }
        most = column_max(most);
        const float keep = __builtin_amdgcn_exp2f(top - most);
        top = most;
        float prob[8];
        float add = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          prob[i] = __builtin_amdgcn_exp2f(s[i >> 2][i & 3] - most);
          add += prob[i];
        }
        sum = sum * keep + add;
        bf16x8_t pp[kPParts];
        split_bf16<kPParts>(prob, pp);
#pragma unroll
        for (int m = 0; m < kValueTiles; ++m) {
          acc[m] *= keep;
          const bf16x8_t v = widen_bf16(cur[0].value_word(m), v_scale[0], cur[1].value_word(m), v_scale[1]);
#pragma unroll
          for (int part = kPParts - 1; part >= 0; --part)
            acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pp[part], acc[m], 0, 0, 0);
        }
        cur[0] = next[0];
        cur[1] = next[1];
      }
    }

    // Join the waves: [wave][column][D + 2] holds O, the maximum and the sum.
    sum = column_sum(sum);
    if (missing) sum = NAN;
    if (r < cols) {
      float* mine = lds + (wave * cols + r) * (D + 2);
#pragma unroll
      for (int m = 0; m < kValueTiles; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) mine[Regs::value_element(m, g, i)] = acc[m][i];
      if (g == 0) {
        mine[D] = top;
        mine[D + 1] = sum;
      }
    }
    __syncthreads();
    for (int i = tid; i < cols * D; i += 256) {
      const int c = i / D, d = i - c * D;
      const float* part = lds + c * (D + 2);
      const int stride = cols * (D + 2);
      float m4[4], most = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        m4[w] = part[w * stride + D];
        most = fmaxf(most, m4[w]);
      }
      float o = 0.f, l = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(m4[w] - most);
        o = fmaf(f, part[w * stride + d], o);
        l = fmaf(f, part[w * stride + D + 1], l);
      }
      if (chunks == 1) {
        Elem<T>::store(out + (int64_t)slice * D + i, o / l);
      } else {
        const int h = kvh * P.group + slice + c;
        float* to = P.partials + (((int64_t)b * P.num_heads + h) * P.max_chunks + chunk) * (D + 2);
        to[d] = o;
        if (d == 0) {
          to[D] = most;
          to[D + 1] = l;
        }
      }
    }
  }
}

// One wave joins the chunks of a row and query head, in order.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv8_decode_merge_kernel(Kv8DecodeParams P) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= (int64_t)P.num_rows * P.num_heads) return;
  const int b = (int)(item / P.num_heads);
  const int p = P.seqlens[b];
  const int layer = P.cache_layer0 + (P.cache_layer == nullptr ? 0 : P.cache_layer[b]);
  const int trow = P.table_row == nullptr ? b : P.table_row[b];
  if (p < kChunk || (int64_t)p >= ((int64_t)P.table_width << P.bs_log2) || layer < 0 || layer >= P.cache.num_layers ||
      trow < 0 || trow >= P.table_rows || (P.max_positions > 0 && p >= P.max_positions))
    return;
  const int pieces = (p + kChunk) / kChunk;
  const int length = kChunk * ((pieces + P.max_chunks - 1) / P.max_chunks);
  const int chunks = (p + length) / length;
  if (chunks == 1) return;
  const float* part = P.partials + item * P.max_chunks * (D + 2);
  float most = -INFINITY;
  for (int c = 0; c < chunks; ++c) most = fmaxf(most, part[c * (D + 2) + D]);
  float o[2] = {0.f, 0.f}, l = 0.f;
  for (int c = 0; c < chunks; ++c) {
    const float* x = part + c * (D + 2);
    const float f = __builtin_amdgcn_exp2f(x[D] - most);
    l = fmaf(f, x[D + 1], l);
    o[0] = fmaf(f, x[lane], o[0]);
    if (lane + 64 < D) o[1] = fmaf(f, x[lane + 64], o[1]);
  }
  T* out = static_cast<T*>(P.out) + item * D;
  Elem<T>::store(out + lane, o[0] / l);
  if (lane + 64 < D) Elem<T>::store(out + lane + 64, o[1] / l);
}

template <typename T, int D>
static int decode_dim(const Kv8DecodeParams& P, int style, hipStream_t stream) {
  const int64_t most = ((int64_t)P.table_width << P.bs_log2) / kChunk + 1;
  const dim3 grid((unsigned)(P.num_rows * P.cache.num_kv_heads), (unsigned)min((int64_t)P.max_chunks, most)), wg(256);
  const size_t lds = sizeof(float) * 4 * min(P.group, 16) * (D + 2);
  if (style == 0) kv8_decode_kernel<T, D, 0><<<grid, wg, lds, stream>>>(P);
  else if (style == 1) kv8_decode_kernel<T, D, 1><<<grid, wg, lds, stream>>>(P);
  else kv8_decode_kernel<T, D, 2><<<grid, wg, lds, stream>>>(P);
  if (hipGetLastError() != hipSuccess) return CDB_ERR_HIP;
  if (grid.y == 1) return CDB_OK;
  const int64_t items = (int64_t)P.num_rows * P.num_heads;
  kv8_decode_merge_kernel<T, D><<<dim3((unsigned)((items + 3) / 4)), wg, 0, stream>>>(P);
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

extern "C" int64_t cdb_kv8_decode_workspace_bytes(int32_t num_rows, int32_t num_heads, int32_t num_kv_heads,
                                                  int32_t head_dim, int32_t max_seqlen) {
  if (num_rows < 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || max_seqlen <= 0) return -1;
  const int64_t chunks = ((int64_t)max_seqlen + cdb::kChunk - 1) / cdb::kChunk;
  return max((int64_t)num_rows, (int64_t)1) * num_heads * chunks * (head_dim + 2) * 4;
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
  const int code = kv8_cache_of(&P.cache, codes, scales, num_cache_layers, pool_blocks, num_kv_heads, head_dim, block_size);
  if (code != CDB_OK) return code;
  if (num_heads % num_kv_heads != 0 || (int64_t)num_rows * num_kv_heads > 0x7fffffffll) return CDB_ERR_SHAPE;
  if (table_row == nullptr && table_rows < num_rows) return CDB_ERR_SHAPE;
  if ((int64_t)table_width * block_size > (1ll << 30)) return CDB_ERR_SHAPE;
  if (!(scale > 0.f) || !(scale < INFINITY)) return CDB_ERR_SHAPE;
  if (q_stride == 0) q_stride = (int64_t)num_heads * head_dim;
  if (kv_stride == 0) kv_stride = (int64_t)num_kv_heads * head_dim;
  if (q_stride < (int64_t)num_heads * head_dim || kv_stride < (int64_t)num_kv_heads * head_dim) return CDB_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return CDB_ERR_SHAPE;
  const int64_t row_bytes = (int64_t)num_rows * num_heads * (head_dim + 2) * 4;
  const int64_t chunks = min(workspace_bytes / row_bytes, (int64_t)65535);
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
  P.num_rows = num_rows; P.num_heads = num_heads; P.group = num_heads / num_kv_heads;
  P.scale_log2 = scale * 1.4426950408889634f;
  P.q_stride = q_stride; P.kv_stride = kv_stride;
  P.vec = kv8_aligned(size, {q, k_new, v_new, q_bias, k_bias, rope_cos, rope_sin}, {q_stride, kv_stride});
  return dtype == CDB_DTYPE_F32 ? decode_type<float>(P, head_dim, rope_style, stream)
                                : decode_type<bf16_t>(P, head_dim, rope_style, stream);
}
