// Varlen causal prefill attention over the 8-bit paged KV cache.
#include "cdb_amd.h"
#include "kv8_common.h"
#include "kv8_host.h"

namespace cdb {

constexpr int kQueries = 128;  // query tokens of a tile: 32 a wave

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

// What one lane holds of a block of 32 keys (two tiles): of the keys, 16-byte units 2j + h of token
// lane % 32; of the values, the words of groups h and h + 2 of each tile for the lane's elements.
template <int D> struct BlockRegs {
  static constexpr int kUnits = D / 32, kWords = D / 32;
  u32x4_t k[kUnits];
  uint32_t v[2][2][kWords];  // [tile][group half][element]

  CDB_DEVICE void load_keys(const uint8_t* k0, const uint8_t* k1, int c, int h) {
    const uint8_t* p = (c & 16 ? k1 : k0) + (c & 15) * 16 + h * 256;
#pragma unroll
    for (int j = 0; j < kUnits; ++j) k[j] = *reinterpret_cast<const u32x4_t*>(p + j * 512);
  }
  CDB_DEVICE void load_values(int a, const uint8_t* vp, int c, int h) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint8_t* p = vp + (h + 2 * s) * (4 * D);
      if constexpr (D == 128) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(p + c * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[a][s][i] = w[i];
      } else {
        const u32x2_t w = *reinterpret_cast<const u32x2_t*>(p + c * 8);
        v[a][s][0] = w[0];
        v[a][s][1] = w[1];
        if constexpr (D == 96) v[a][s][2] = *reinterpret_cast<const uint32_t*>(p + 256 + c * 4);
      }
    }
  }
  // Head element of accumulator row `row` of value product i.
  static CDB_DEVICE int value_element(int i, int row) {
    if constexpr (D == 128) return 4 * row + i;
    return i < 2 ? 2 * row + i : 64 + row;
  }
};

// Eight codes (two words) as fp16, scaled by a power of two.
CDB_DEVICE f16x8_t widen_f16(uint32_t w0, uint32_t w1, float s) {
  union { f16x2_t p[4]; f16x8_t v; } u;
  u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, s, false);
  u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, s, true);
  u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, s, false);
  u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, s, true);
  return u.v;
}

CDB_DEVICE float half_max(float v) {
  const f32x2_t x = pair32(v);
  return fmaxf(x[0], x[1]);
}

template <typename T, int D>
__global__ void __launch_bounds__(256, 2) kv8_prefill_kernel(Kv8PrefillParams P) {
  using Regs = BlockRegs<D>;
  constexpr bool kWide = sizeof(T) == 4;
  constexpr int kQParts = kWide ? 3 : 1, kPParts = kWide ? 2 : 1;
  constexpr int kSteps = D / 16, kTiles = D / 32;
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
  const int w0 = P.tile_q0[n] + 32 * wave;
  if (token0 < 0 || num < 0 || token0 + num > P.tokens || past < 0 || w0 < 0 || w0 >= num) return;
  const int query = w0 + c, pos = past + query;
  const int64_t total = (int64_t)past + num;
  const int trow = P.table_row[s];
  const bool bad = total > ((int64_t)P.table_width << P.bs_log2) || trow < 0 || trow >= P.table_rows;

  const int tile_end = past + min(P.tile_q0[n] + kQueries, num), wave_end = past + min(w0 + 32, num);
  const int blocks = (tile_end + 31) / 32;
  const int part = blockIdx.y;
  const int from = (int)((int64_t)blocks * part / P.splits);
  const int to = bad ? 0 : min((int)((int64_t)blocks * (part + 1) / P.splits), (wave_end + 31) / 32);

  bf16x8_t q[kSteps][kQParts];
  {
    const T* src = static_cast<const T*>(P.q) + ((token0 + min(query, num - 1)) * P.num_heads + head) * D;
#pragma unroll
    for (int m = 0; m < kSteps; ++m) {
      const T* at = src + 32 * (m >> 1) + 16 * h + 8 * (m & 1);
      if constexpr (kWide) {
        float x[8];
        load_f32<T, 8>(at, x, true);
#pragma unroll
        for (int p = 0; p < kQParts; ++p)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const __bf16 y = (__bf16)x[i];
            q[m][p][i] = y;
            x[i] -= (float)y;
          }
      } else {
        q[m][0] = *reinterpret_cast<const bf16x8_t*>(at);
      }
    }
  }
  f32x16_t acc[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
  float top = -INFINITY, sum = 0.f;
  int ref = 1;  // biased exponent that the accumulators are counted in
  bool missing = bad;
  const int32_t* table = P.block_table + (int64_t)(bad ? 0 : trow) * P.table_width;
  const int bs_mask = (1 << P.bs_log2) - 1;

  for (int window = from; window < to; window += 32) {
    const int count = min(32, to - window);
    int64_t where = 0;
    uint32_t k_byte = 0, v_byte = 0;
    bool lost = false;
    if (lane < 2 * count) {
      const int t = window * 32 + lane * kTile;
      if (t < total) {
        const int block = table[t >> P.bs_log2];
        lost = block < 0 || block >= P.cache.pool_blocks;
        where = P.cache.tile(P.layer, 0, lost ? 0 : block, kvh, (t & bs_mask) >> 4);
        k_byte = P.cache.scales[where];
        v_byte = P.cache.scales[where + P.cache.plane_tiles];
      }
    }
    missing = missing || __ballot(lost) != 0;
    auto codes_at = [&](int j) -> const uint8_t* {
      const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)where, j);
      const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(where >> 32), j);
      return P.cache.codes + (int64_t)(((uint64_t)hi << 32) | lo) * (kTile * D);
    };
    const int64_t plane = P.cache.plane_tiles * (kTile * D);
    auto load = [&](Regs& x, int i) {
      const uint8_t *t0 = codes_at(2 * i), *t1 = codes_at(2 * i + 1);
      x.load_keys(t0, t1, c, h);
      x.load_values(0, t0 + plane, c, h);
      x.load_values(1, t1 + plane, c, h);
    };
    Regs cur, next;
    load(cur, 0);
    for (int i = 0; i < count; ++i) {
      if (i + 1 < count) load(next, i + 1);
      const int key0 = (window + i) * 32;
      const float k_scale = scale_of(c & 16 ? __builtin_amdgcn_readlane((int)k_byte, 2 * i + 1)
                                            : __builtin_amdgcn_readlane((int)k_byte, 2 * i));
      f32x16_t sc;
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] = 0.f;
#pragma unroll
      for (int m = 0; m < kSteps; ++m) {
        const bf16x8_t k = widen_bf16(cur.k[m >> 1][2 * (m & 1)], k_scale, cur.k[m >> 1][2 * (m & 1) + 1], k_scale);
#pragma unroll
        for (int p = kQParts - 1; p >= 0; --p) sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q[m][p], sc, 0, 0, 0);
      }
      if (key0 + 31 > past + w0) {  // some query of the wave does not see some key of the block
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (key0 + (e >> 2) * 8 + 4 * h + (e & 3) > pos) sc[e] = -INFINITY;
      }
      float most = sc[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) most = fmaxf(most, sc[e]);
      most = fmaxf(top, half_max(most) * P.scale_log2);
      const float base = most == -INFINITY ? 0.f : most;  // a query that has seen no key yet
      if (__any(most > top)) {
        const float keep = __builtin_amdgcn_exp2f(top - base);
        sum *= keep;
#pragma unroll
        for (int m = 0; m < kTiles; ++m) acc[m] *= keep;
        top = most;
      }
      float prob[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        prob[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], P.scale_log2, -base));
        sum += prob[e];
      }
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const int t = key0 + kTile * a;
        if (t >= total) continue;
        const int v_exp = max((int)__builtin_amdgcn_readlane((int)v_byte, 2 * i + a), 1);
        if (v_exp > ref) {
          const float f = shrink_of(ref, v_exp);
#pragma unroll
          for (int m = 0; m < kTiles; ++m) acc[m] *= f;
          ref = v_exp;
        }
        const float v_scale = shrink_of(v_exp, ref);
        if (t + kTile > total) {  // codes behind the sequence count for nothing, NaN among them
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int m = 0; m < Regs::kWords; ++m) cur.v[a][g][m] &= tokens_below((int)(total - t) - 4 * (h + 2 * g));
        }
        f16x8_t pp[kPParts];
        {
          float left[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) left[e] = prob[8 * a + e];
#pragma unroll
          for (int p = 0; p < kPParts; ++p)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const f16x2_t y = __builtin_convertvector((f32x2_t){left[e], left[e + 1]}, f16x2_t);
              pp[p][e] = y[0];
              pp[p][e + 1] = y[1];
              left[e] -= (float)y[0];
              left[e + 1] -= (float)y[1];
            }
        }
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
          const f16x8_t v = widen_f16(cur.v[a][0][m], cur.v[a][1][m], v_scale);
#pragma unroll
          for (int p = kPParts - 1; p >= 0; --p)
            acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pp[p], acc[m], 0, 0, 0);
        }
      }
      cur = next;
    }
  }

  sum += shfl_xor_f32(sum, 32);
  if (missing) sum = NAN;
  const float back = scale_of(ref);
  if (query >= num) return;
  if (P.splits == 1) {
    T* out = static_cast<T*>(P.out) + ((token0 + query) * P.num_heads + head) * D;
    const float inv = back / sum;
#pragma unroll
    for (int m = 0; m < kTiles; ++m)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        Elem<T>::store(out + Regs::value_element(m, (e >> 2) * 8 + 4 * h + (e & 3)), acc[m][e] * inv);
    return;
  }
  float* to_part = P.partials +
                   ((((int64_t)n * P.splits + part) * P.num_heads + head) * kQueries + (32 * wave + c)) * (D + 2);
#pragma unroll
  for (int m = 0; m < kTiles; ++m)
#pragma unroll
    for (int e = 0; e < 16; ++e) to_part[Regs::value_element(m, (e >> 2) * 8 + 4 * h + (e & 3))] = acc[m][e] * back;
  if (h == 0) {
    to_part[D] = top;
    to_part[D + 1] = sum;
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
  if (token0 < 0 || num < 0 || token0 + num > P.tokens || P.past[s] < 0 || P.tile_q0[n] < 0 || query >= num) return;
  const int64_t stride = (int64_t)P.num_heads * kQueries * (D + 2);
  const float* x = P.partials + (((int64_t)n * P.splits * P.num_heads + head) * kQueries + i) * (D + 2);
  float most = -INFINITY;
  for (int p = 0; p < P.splits; ++p) most = fmaxf(most, x[p * stride + D]);
  float o[2] = {0.f, 0.f}, l = 0.f;
  for (int p = 0; p < P.splits; ++p) {
    const float* y = x + p * stride;
    const float f = __builtin_amdgcn_exp2f(y[D] - most);
    l = fmaf(f, y[D + 1], l);
    o[0] = fmaf(f, y[lane], o[0]);
    if (lane + 64 < D) o[1] = fmaf(f, y[lane + 64], o[1]);
  }
  T* out = static_cast<T*>(P.out) + ((token0 + query) * P.num_heads + head) * D;
  Elem<T>::store(out + lane, o[0] / l);
  if (lane + 64 < D) Elem<T>::store(out + lane + 64, o[1] / l);
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
  if (num_tiles < 0 || splits <= 0 || num_heads <= 0 || head_dim <= 0) return -1;
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
      layer < 0 || layer >= num_cache_layers || splits <= 0 || splits > 65535)
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
  if (workspace_bytes < cdb_kv8_prefill_workspace_bytes(num_tiles, splits, num_heads, head_dim)) return CDB_ERR_CAPACITY;
  P.q = q; P.layer = layer;
  P.block_table = block_table; P.table_row = table_row; P.cu_q = cu_q; P.past = past;
  P.tile_seq = tile_seq; P.tile_q0 = tile_q0;
  P.table_rows = table_rows; P.table_width = table_width; P.num_seqs = num_seqs; P.num_tiles = num_tiles;
  P.num_heads = num_heads; P.group = num_heads / num_kv_heads; P.bs_log2 = __builtin_ctz(block_size);
  P.splits = splits; P.tokens = tokens; P.out = out; P.partials = static_cast<float*>(workspace);
  P.scale_log2 = scale * 1.4426950408889634f;
  return dtype == CDB_DTYPE_F32 ? prefill_type<float>(P, head_dim, stream) : prefill_type<bf16_t>(P, head_dim, stream);
}
