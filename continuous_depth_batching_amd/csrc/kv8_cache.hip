// Filling the 8-bit KV cache: the rotating, quantising write of a batch of tokens, and the block
// tables, slot maps and attention tiles of a batch from its requests' lengths.
#include <type_traits>

#include "cdb_amd.h"
#include "kv8_common.h"
#include "kv8_host.h"

namespace cdb {

struct Kv8WriteParams {
  const void *q, *k, *v;
  void* q_out;
  Kv8Cache cache;
  int64_t layer;
  const int64_t* rows;
  int64_t pool_rows;
  const int32_t* positions;
  const float *cos, *sin;
  const void *q_bias, *k_bias;
  int64_t tokens, q_stride, kv_stride;
  int32_t num_heads, max_positions, chunk, heads_each;
  int64_t chunks, kv_blocks;  // chunks of tokens; workgroups of the cache write, before those that rotate queries
  bool vec;
};

// The elements of a head whose values a lane r (of 16) holds: 16-byte loads of bf16 for heads of 128, and the
// pieces of a tile that such a lane stores, 16 bytes a group and 4 elements.
template <int D> struct ValuePieces {
  static constexpr int kMost = D == 128 ? 8 : 4;
  static constexpr int kPieces = D == 96 ? 2 : 1;
  static CDB_DEVICE int element(int j, int r) { return j == 0 ? kMost * r : 64 + 2 * r; }
};

// Whether a whole tile's keys and values are read past the caches. For bf16 heads of 128 that pays where q, k and v are
// not in a cache (7700 tokens of 16 heads: 38.5 us against 41.7) and is as good where they have just been written (33.2
// both); it costs elsewhere (bf16 heads of 96: 117 against 111; fp32 heads of 128: 70 against 62, of 64: 41 against
// 36). Shorter runs never are: 1500 single tokens take 97 us with it and 87 so (82 in a kernel without the choice).
template <typename T, int D> constexpr bool kHeadOnce = sizeof(T) == 2 && D == 128;

// The angles of a lane's units of a key: kept while the wave goes through its heads.
template <int D, int STYLE> struct KeyAngles {
  static constexpr int kUnits = D / 16, kParts = (kUnits + 3) / 4;
  static constexpr bool kPaired = STYLE == 1 && D == 128;  // units g and g + 4 are each other's partners
  static constexpr int kSets = STYLE == 0 ? 0 : kPaired ? 1 : kParts, kLen = STYLE == 1 ? 16 : 8;
  float cos[kSets + 1][kLen], sin[kSets + 1][kLen];

  CDB_DEVICE void load(const float* c, const float* s, int g, bool vec) {
#pragma unroll
    for (int j = 0; j < kSets; ++j) {
      const int u = min(g + 4 * j, kUnits - 1);
      const int at = STYLE == 1 ? 16 * (u < kUnits / 2 ? u : u - kUnits / 2) : 8 * u;
      load_f32<float, kLen>(c + at, cos[j], vec);
      load_f32<float, kLen>(s + at, sin[j], vec);
    }
  }
  // Units g + 4j of a head, x + bias, rotated, in fp32 with every product and sum rounded once.
  template <typename T>
  CDB_DEVICE void key(const T* head, const T* bias, int g, bool vec, bool once, float x[kParts][16]) const {
    auto unit = [&](int u, float* to) __attribute__((always_inline)) {
      if (kHeadOnce<T, D> && once) load_f32<T, 16, true>(head + 16 * u, to, vec);
      else load_f32<T, 16>(head + 16 * u, to, vec);
      if (bias != nullptr) {
        float b[16];
        load_f32<T, 16>(bias + 16 * u, b, vec);
#pragma unroll
        for (int i = 0; i < 16; ++i) to[i] = add_rn(to[i], b[i]);
      }
    };
#pragma unroll
    for (int j = 0; j < kParts; ++j)
      if (g + 4 * j < kUnits) unit(g + 4 * j, x[j]);
    if constexpr (kPaired) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float a = x[0][i], b = x[kParts - 1][i];
        x[0][i] = sub_rn(mul_rn(a, cos[0][i]), mul_rn(b, sin[0][i]));
        x[kParts - 1][i] = add_rn(mul_rn(b, cos[0][i]), mul_rn(a, sin[0][i]));
      }
    } else if constexpr (STYLE == 1) {
#pragma unroll
      for (int j = 0; j < kParts; ++j) {
        const int u = g + 4 * j;
        if (u >= kUnits) continue;
        const bool low = u < kUnits / 2;
        float p[16];
        unit(low ? u + kUnits / 2 : u - kUnits / 2, p);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float ps = mul_rn(p[i], sin[j][i]);
          x[j][i] = add_rn(mul_rn(x[j][i], cos[j][i]), low ? -ps : ps);
        }
      }
    } else if constexpr (STYLE == 2) {
#pragma unroll
      for (int j = 0; j < kParts; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float a = x[j][2 * i], b = x[j][2 * i + 1];
          x[j][2 * i] = sub_rn(mul_rn(a, cos[j][i]), mul_rn(b, sin[j][i]));
          x[j][2 * i + 1] = add_rn(mul_rn(b, cos[j][i]), mul_rn(a, sin[j][i]));
        }
    }
  }
};

// One wave writes the tokens of one KV head that start a run inside its chunk. A run is the tokens that a batch
// brings for one tile, 16 at most, each as far from the first in the batch as in the tile, so a tile's scale is known
// to the wave that writes it: the maximum over the run, and for a tile that held earlier tokens their scale too.
// Tokens in between that are left out (padding, a slot or position out of range) do not end a run: two waves would
// meet in the tile.
// Lane (r, g) = (lane % 16, lane / 16) holds units g, g + 4 of token r of the key tile, and group g of
// some elements of the value tile, which are the tile's own pieces of 16 bytes.
// first: the run's first token; run: a bit for each token of the tile that it writes, the first token's the lowest.
template <typename T, int D, int STYLE>
CDB_DEVICE void write_run(const Kv8WriteParams& P, int64_t first, uint32_t run, int64_t tile, int head,
                          const KeyAngles<D, STYLE>& angles) {
  using V = ValuePieces<D>;
  constexpr int kUnits = D / 16;
  constexpr int kParts = (kUnits + 3) / 4;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int off = __builtin_ctz(run);
  const bool once = run == 0xffffu;
  const int64_t block = tile >> P.cache.tile_log2;
  const int sub = (int)(tile & ((1 << P.cache.tile_log2) - 1));
  const T* k = static_cast<const T*>(P.k) + head * D;
  const T* v = static_cast<const T*>(P.v) + head * D;
  const T* k_bias = P.k_bias == nullptr ? nullptr : static_cast<const T*>(P.k_bias) + head * D;
  const int64_t k_tile = P.cache.tile(P.layer, 0, block, head, sub);
  const int64_t v_tile = P.cache.tile(P.layer, 1, block, head, sub);
  uint8_t* k_codes = P.cache.codes + k_tile * (kTile * D);
  uint8_t* v_codes = P.cache.codes + v_tile * (kTile * D);
  int k_old = 0, v_old = 0;
  if (off > 0) {
    k_old = (int)scale_byte_read(P.cache.scales[k_tile]);
    v_old = (int)scale_byte_read(P.cache.scales[v_tile]);
  }

  // Values: tokens 4g..4g+3 of the lane's elements, on their way while the keys are worked on.
  Vec<T, V::kMost> y0[4];
  Vec<T, 2> y1[4];  // of heads of 96
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int slot = 4 * g + i;
    const T* src = v + (first + (run >> slot & 1 ? slot - off : 0)) * P.kv_stride;
    if (kHeadOnce<T, D> && once) y0[i] = load_raw<T, V::kMost, true>(src + V::element(0, r), P.vec);
    else y0[i] = load_raw<T, V::kMost>(src + V::element(0, r), P.vec);
    if constexpr (V::kPieces == 2) y1[i] = load_raw<T, 2>(src + V::element(1, r), P.vec);
  }

  // Keys: token r of the tile is the (r - off)th from the run's first.
  const bool live = (run >> r & 1) != 0;
  float x[kParts][16];
  angles.template key<T>(k + (first + (live ? r - off : 0)) * P.kv_stride, k_bias, g, P.vec, once, x);
  // The largest size among them, infinities and NaN left out: those are looked for, and almost never found.
  auto size = [](float z, bool finite) {
    const uint32_t bits = size_bits(z);
    return finite && bits >= kNotFinite ? 0u : bits;
  };
  auto k_size = [&](bool finite) __attribute__((always_inline)) {
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < kParts; ++j)
      if (g + 4 * j < kUnits) {
#pragma unroll
        for (int i = 0; i < 16; ++i) most = max(most, size(x[j][i], finite));
      }
    return live ? most : 0u;
  };
  uint32_t k_top = k_size(false);
  if (__any(k_top >= kNotFinite)) k_top = k_size(true);
  int k_now = scale_byte(all_max(__uint_as_float(k_top)));
  if (off > 0) k_now = max(k_now, k_old);
  const float k_scale = scale_of(k_now);
  const bool k_grown = off > 0 && k_now != k_old;

#pragma unroll
  for (int j = 0; j < kParts; ++j) {
    const int u = g + 4 * j;
    if (u >= kUnits) continue;
    u32x4_t* at = reinterpret_cast<u32x4_t*>(k_codes + u * 256 + r * 16);
    if (live) {
      u32x4_t w;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = codes_of(x[j][4 * i], x[j][4 * i + 1], x[j][4 * i + 2], x[j][4 * i + 3], k_scale);
      *at = w;
    } else if (k_grown && r < off) {
      const float f = growth_of(k_old, k_now);
      u32x4_t w = *at;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = recode(w[i], f);
      *at = w;
    }
  }

  const uint32_t before = tokens_below(off - 4 * g);  // earlier tokens of the group
  const uint32_t fresh = tokens_in(run >> (4 * g));   // the run's
  auto v_size = [&](bool finite) __attribute__((always_inline)) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t most = 0;
#pragma unroll
      for (int e = 0; e < V::kMost; ++e) most = max(most, size(y0[i].get(e), finite));
      if constexpr (V::kPieces == 2) most = max(most, max(size(y1[i].get(0), finite), size(y1[i].get(1), finite)));
      if (fresh & (255u << (8 * i))) top = max(top, most);
    }
    return top;
  };
  uint32_t v_top = v_size(false);
  if (__any(v_top >= kNotFinite)) v_top = v_size(true);
  int v_now = scale_byte(all_max(__uint_as_float(v_top)));
  if (off > 0) v_now = max(v_now, v_old);
  const float v_scale = scale_of(v_now);
  const bool v_grown = off > 0 && v_now != v_old;
  if (fresh != 0u || (v_grown && before != 0u)) {
    const float f = growth_of(v_old, v_now);
    auto store = [&](const auto* y, int element, auto size) __attribute__((always_inline)) {
      constexpr int kSize = decltype(size)::value, kStep = kSize < 4 ? 2 : 4;
      uint32_t* at = reinterpret_cast<uint32_t*>(v_codes + g * (4 * D)) + element;
#pragma unroll
      for (int e = 0; e < kSize; e += kStep) {
        uint32_t out[4] = {0u, 0u, 0u, 0u};
        if (fresh != ~0u) {
#pragma unroll
          for (int i = 0; i < kStep; i += 2) {
            const u32x2_t kept = *reinterpret_cast<const u32x2_t*>(at + e + i);
            out[i] = kept[0];
            out[i + 1] = kept[1];
          }
        }
#pragma unroll
        for (int i = 0; i < kStep; ++i) {
          const uint32_t c =
              codes_of(y[0].get(e + i), y[1].get(e + i), y[2].get(e + i), y[3].get(e + i), v_scale);
          uint32_t w = out[i];
          if (v_grown) w = (w & ~before) | (recode(w, f) & before);
          out[i] = (c & fresh) | (w & ~fresh);
        }
        if constexpr (kStep == 4) *reinterpret_cast<u32x4_t*>(at + e) = (u32x4_t){out[0], out[1], out[2], out[3]};
        else *reinterpret_cast<u32x2_t*>(at + e) = (u32x2_t){out[0], out[1]};
      }
    };
    store(y0, V::element(0, r), std::integral_constant<int, V::kMost>());
    if constexpr (V::kPieces == 2) store(y1, V::element(1, r), std::integral_constant<int, 2>());
  }
  if (lane == 0) {
    P.cache.scales[k_tile] = (uint8_t)k_now;
    P.cache.scales[v_tile] = (uint8_t)v_now;
  }
}

// The rotated queries, and the keys and values as codes, bound by HBM bytes: 7700 tokens of 16 heads x 128 in
// 38.5 us (158 MB, 4.1 TB/s), the queries alone 15 us. 61 single tokens take 5.4 us, two dependent loads and a store;
// past 1024 tokens a wave takes 16, and 1500 single ones, each a run of its own, 87 us.
template <typename T, int D, int STYLE>
__global__ void __launch_bounds__(256) kv8_write_kernel(Kv8WriteParams P) {
  const int lane = threadIdx.x & 63;
  if (blockIdx.x < P.kv_blocks) {
    const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int heads = P.cache.num_kv_heads;
    const int groups = (heads + P.heads_each - 1) / P.heads_each;
    const int64_t chunk = item / groups;
    const int head = (int)(item - chunk * groups) * P.heads_each;
    if (chunk >= P.chunks) return;
    // Lane t holds the slots of token base + t and of the one before it; a run reaches at most 15
    // tokens past the chunk.
    const int64_t base = chunk * P.chunk, idx = base + lane;
    const bool near = lane < P.chunk + 16;
    auto slot = [&](int64_t i, int& position) -> int64_t {
      position = 0;
      if (!near || i < 0 || i >= P.tokens) return -1;
      const int64_t row = P.rows[i];
      if (STYLE != 0) position = P.positions[i];
      const bool out = row < 0 || row >= P.pool_rows || (STYLE != 0 && (position < 0 || position >= P.max_positions));
      return out ? -1 : row;
    };
    int position, unused;
    const int64_t row = slot(idx, position);
    const int64_t prev = slot(idx - 1, unused);
    bool follows = row >= 0 && prev >= 0 && row == prev + 1 && (row & 15) != 0;
    // Behind a token left out, the last one before it that is not decides.
    const int64_t reach = min(idx, row & 15);
    bool open = row >= 0 && prev < 0 && reach > 1;
    for (int d = 2; __any(open); ++d) {
      const int64_t before = open ? slot(idx - d, unused) : -1;
      if (open && before >= 0) follows = row == before + d;
      open = open && before < 0 && d < reach;
    }
    uint64_t starts = __ballot(row >= 0 && !follows && lane < P.chunk);
    while (starts != 0) {
      const int s = __builtin_ctzll(starts);
      starts &= starts - 1;
      const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)row, s);
      const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(row >> 32), s);
      const int64_t row0 = (int64_t)(((uint64_t)hi << 32) | lo);
      // The tokens from s on that go with it, up to the first that does not.
      const bool same = row >= 0 && row - row0 == lane - s && (row >> 4) == (row0 >> 4);
      const uint64_t others = __ballot(row >= 0 && !same) >> s;
      const uint64_t with = (__ballot(same) >> s) & (others == 0 ? ~0ull : (others & -others) - 1);
      const int slot0 = (int)(lo & 15), r = lane & 15;
      const uint32_t run = (uint32_t)with << slot0;
      KeyAngles<D, STYLE> angles;
      if constexpr (STYLE != 0) {
        const int p = __shfl(position, s + (run >> r & 1 ? r - slot0 : 0));
        angles.load(P.cos + (int64_t)p * (D / 2), P.sin + (int64_t)p * (D / 2), lane >> 4, P.vec);
      }
      for (int h = head; h < min(head + P.heads_each, heads); ++h)
        write_run<T, D, STYLE>(P, base + s, run, row0 >> 4, h, angles);
    }
    return;
  }
  // Queries: 16 elements a thread, two pieces of 8 (STYLE 1: one of each half).
  const int64_t item = (int64_t)(blockIdx.x - P.kv_blocks) * 256 + threadIdx.x;
  constexpr int kUnits = D / 16;
  const int u = (int)(item % kUnits);
  const int64_t th = item / kUnits;
  const int64_t t = th / P.num_heads;
  const int h = (int)(th - t * P.num_heads);
  if (t >= P.tokens) return;
  const int64_t row = P.rows[t];
  if (row < 0) return;
  int64_t angle = 0;
  bool bad = false;
  if constexpr (STYLE != 0) {
    const int p = P.positions[t];
    bad = p < 0 || p >= P.max_positions;
    angle = bad ? 0 : (int64_t)p * (D / 2);
  }
  const T* q = static_cast<const T*>(P.q) + t * P.q_stride + h * D;
  const T* bias = P.q_bias == nullptr ? nullptr : static_cast<const T*>(P.q_bias) + h * D;
  T* out = static_cast<T*>(P.q_out) + (t * P.num_heads + h) * D;
  constexpr int kApart = STYLE == 1 ? D / 2 : 8;
  const int d = STYLE == 1 ? 8 * u : 16 * u;
  float x[2][8];
  load_rotated_pair<T, D, STYLE, 8>(q, bias, P.cos + angle, P.sin + angle, d, P.vec, x[0], x[1]);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    Vec<T, 8> w;
#pragma unroll
    for (int i = 0; i < 8; i += 2) w.set_pair(i, bad ? NAN : x[half][i], bad ? NAN : x[half][i + 1]);
    w.store(out + d + half * kApart);
  }
}

template <typename T, int D>
static int write_style(const Kv8WriteParams& P, int style, int64_t blocks, hipStream_t stream) {
  const dim3 grid((unsigned)blocks), wg(256);
  if (style == 0) kv8_write_kernel<T, D, 0><<<grid, wg, 0, stream>>>(P);
  else if (style == 1) kv8_write_kernel<T, D, 1><<<grid, wg, 0, stream>>>(P);
  else kv8_write_kernel<T, D, 2><<<grid, wg, 0, stream>>>(P);
  return hipGetLastError() == hipSuccess ? CDB_OK : CDB_ERR_HIP;
}

template <typename T>
static int write_dim(const Kv8WriteParams& P, int dim, int style, int64_t blocks, hipStream_t stream) {
  switch (dim) {
    case 64: return write_style<T, 64>(P, style, blocks, stream);
    case 96: return write_style<T, 96>(P, style, blocks, stream);
    case 128: return write_style<T, 128>(P, style, blocks, stream);
    default: return CDB_ERR_UNSUPPORTED;
  }
}

// -- batch layout -------------------------------------------------------------------------------------------------

struct LayoutParams {
  const int32_t *past, *lens, *table_row, *free_blocks;
  int32_t* table;
  int32_t num_seqs, table_rows, table_width, num_free, bs_log2;
  int32_t *cu_q, *positions, *tile_seq, *tile_q0, *counts;
  int64_t* rows;
  int32_t token_capacity, tile_capacity;
};

constexpr int kTileQueries = 128;

// The sums of a layout stay below 2^31 by saturating there: such a batch is refused as a whole.
constexpr uint32_t kLayoutMost = 0x7fffffffu;
CDB_DEVICE uint32_t add_up(uint32_t a, uint32_t b) { return min(a + b, kLayoutMost); }

// Inclusive scan over the lanes of a wave.
CDB_DEVICE uint32_t wave_scan(uint32_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t up = __shfl_up(v, d);
    if (lane >= d) v = add_up(v, up);
  }
  return v;
}

// The last i with first[i] <= x, for ascending first[0..n] with first[0] <= x < first[n].
CDB_DEVICE int last_at_most(const int32_t* first, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Tiles of a sequence whose key range ends past x (tile j's ends at past + min(128 (j + 1), len)).
CDB_DEVICE int tiles_past(int x, int past, int len) {
  const int y = x - past;
  if (y >= len) return 0;
  const int tiles = (len + kTileQueries - 1) / kTileQueries;
  return y < 0 ? tiles : tiles - y / kTileQueries;
}

// Every workgroup scans the requests' lengths into LDS (a few microseconds' work that saves a second launch and any
// order between workgroups), then takes its share of tokens, new blocks and tiles. A tile's place in the
// longest-first list is the number of tiles before it in that order: counted per request in closed form, a wave's
// lanes splitting the requests. kEach: requests a thread scans.
//
// Bound by its chain of latencies (launch, lengths, scan, search, block id, store) and not by bytes: 24 prompts,
// 7700 tokens, 5.3 us; 1000 requests, 150000 tokens, 9.5 us (four tokens a thread after one search: 7.0 and 11.2).
template <int kThreads, int kEach> __global__ void __launch_bounds__(kThreads) batch_layout_kernel(LayoutParams P) {
  constexpr int kWaves = kThreads / 64;
  extern __shared__ int32_t lds[];
  const int S = P.num_seqs;
  int32_t* cu = lds;                 // [S + 1] first token
  int32_t* taken = cu + S + 1;       // [S + 1] first new block
  int32_t* tiles = taken + S + 1;    // [S + 1] first tile
  int32_t* begin = tiles + S + 1;    // [S] cached tokens
  __shared__ uint32_t part[kWaves][3];
  __shared__ int32_t status;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) status = 0;
  const int64_t most = (int64_t)P.table_width << P.bs_log2;
  const int bs_mask = (1 << P.bs_log2) - 1;
  int past[kEach], len[kEach], row[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int s = min(tid * kEach + i, S - 1);
    past[i] = S > 0 ? P.past[s] : 0;
    len[i] = S > 0 ? P.lens[s] : 0;
    row[i] = S == 0 || P.table_row == nullptr ? s : P.table_row[s];
  }
  __syncthreads();
  uint32_t sum[3] = {0, 0, 0};
  auto add = [&](int i) __attribute__((always_inline)) {
    sum[0] = add_up(sum[0], len[i]);
    sum[1] = add_up(sum[1], ((past[i] + len[i] + bs_mask) >> P.bs_log2) - ((past[i] + bs_mask) >> P.bs_log2));
    sum[2] = add_up(sum[2], (len[i] + kTileQueries - 1) / kTileQueries);
  };
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const bool real = tid * kEach + i < S;
    const bool bad = past[i] < 0 || len[i] < 0 || (int64_t)past[i] + len[i] > most || row[i] < 0 ||
                     row[i] >= P.table_rows;
    if (real && bad) atomicOr(&status, CDB_LAYOUT_BAD_REQUEST);
    if (!real || bad) past[i] = len[i] = 0;
    add(i);
  }
  uint32_t upto[3];
#pragma unroll
  for (int c = 0; c < 3; ++c) {
    const uint32_t all = wave_scan(sum[c]);
    if (lane == 63) part[wave][c] = all;
    const uint32_t up = __shfl_up(all, 1);
    upto[c] = lane == 0 ? 0u : up;
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < 3; ++c) {
    sum[c] = upto[c];
    for (int w = 0; w < wave; ++w) sum[c] = add_up(sum[c], part[w][c]);
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int s = tid * kEach + i;
    if (s < S) {
      cu[s] = (int)sum[0];
      taken[s] = (int)sum[1];
      tiles[s] = (int)sum[2];
      begin[s] = past[i];
    }
    add(i);
  }
  if (tid == kThreads - 1) {
    cu[S] = (int)sum[0];
    taken[S] = (int)sum[1];
    tiles[S] = (int)sum[2];
  }
  __syncthreads();
  // Of a batch too large to count nothing is laid out.
  const bool over = (uint32_t)cu[S] == kLayoutMost;
  const int num_tokens = over ? 0 : cu[S], num_taken = over ? 0 : taken[S], num_tiles = over ? 0 : tiles[S];
  if (blockIdx.x == 0) {
    for (int s = tid; s <= S; s += kThreads) P.cu_q[s] = cu[s];
    if (tid == 0) {
      P.counts[0] = cu[S];
      P.counts[1] = tiles[S];
      P.counts[2] = taken[S];
      P.counts[3] = status | (over || cu[S] > P.token_capacity ? CDB_LAYOUT_TOKENS_FULL : 0) |
                    (tiles[S] > P.tile_capacity ? CDB_LAYOUT_TILES_FULL : 0) |
                    (taken[S] > P.num_free ? CDB_LAYOUT_NO_BLOCKS : 0);
    }
  }
  const int64_t stride = (int64_t)gridDim.x * kThreads;
  const int64_t id = (int64_t)blockIdx.x * kThreads + tid;
  auto table_at = [&](int s) {
    return P.table + (int64_t)(P.table_row == nullptr ? s : P.table_row[s]) * P.table_width;
  };

  for (int64_t t = id; t < P.token_capacity; t += stride) {
    int pos = -1;
    int64_t row = -1;
    if (t < num_tokens) {
      const int s = last_at_most(cu, S, (int)t);
      pos = begin[s] + (int)t - cu[s];
      const int held = (begin[s] + bs_mask) >> P.bs_log2, column = pos >> P.bs_log2;
      int block;
      if (column < held) {
        block = table_at(s)[column];
      } else {
        const int n = taken[s] + column - held;
        block = n < P.num_free ? P.free_blocks[n] : -1;
      }
      if (block >= 0) row = ((int64_t)block << P.bs_log2) + (pos & bs_mask);
    }
    P.positions[t] = pos;
    P.rows[t] = row;
  }
  for (int64_t n = id; n < num_taken; n += stride) {
    const int s = last_at_most(taken, S, (int)n);
    const int column = ((begin[s] + bs_mask) >> P.bs_log2) + (int)n - taken[s];
    table_at(s)[column] = n < P.num_free ? P.free_blocks[n] : -1;
  }
  for (int64_t n = num_tiles + id; n < P.tile_capacity; n += stride) {
    P.tile_seq[n] = -1;
    P.tile_q0[n] = 0;
  }
  for (int64_t n = (int64_t)blockIdx.x * kWaves + wave; n < num_tiles; n += (int64_t)gridDim.x * kWaves) {
    const int s = last_at_most(tiles, S, (int)n);
    const int q0 = ((int)n - tiles[s]) * kTileQueries;
    const int end = begin[s] + min(q0 + kTileQueries, cu[s + 1] - cu[s]);
    int before = 0;
    for (int o = lane; o < S; o += 64) before += tiles_past(o < s ? end - 1 : end, begin[o], cu[o + 1] - cu[o]);
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) before += __shfl_xor(before, m);
    if (lane == 0 && before < P.tile_capacity) {
      P.tile_seq[before] = s;
      P.tile_q0[before] = q0;
    }
  }
}

// A token a thread and a tile a wave, up to what the device holds at once.
template <int kThreads, int kEach> static void layout_launch(const LayoutParams& P, size_t lds, hipStream_t stream) {
  const int64_t want = max((int64_t)P.token_capacity / kThreads, (int64_t)P.tile_capacity / (kThreads / 64)) + 1;
  const int64_t most = 256 * (1024 / kThreads);
  batch_layout_kernel<kThreads, kEach><<<dim3((unsigned)min(want, most)), dim3(kThreads), lds, stream>>>(P);
}

}  // namespace cdb

extern "C" int cdb_kv8_write(const void* q, const void* k, const void* v, void* q_out, void* codes, void* scales,
                             int32_t num_cache_layers, int64_t pool_blocks, int32_t layer, const int64_t* rows,
                             const int32_t* positions, const float* rope_cos, const float* rope_sin,
                             int32_t rope_style, int32_t max_positions, const void* q_bias, const void* k_bias,
                             int64_t tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                             int32_t block_size, int64_t q_stride, int64_t kv_stride, int32_t dtype,
                             hipStream_t stream) {
  using namespace cdb;
  if (tokens < 0 || num_heads < 0 || layer < 0 || layer >= num_cache_layers) return CDB_ERR_SHAPE;
  if (rope_style < 0 || rope_style > 2) return CDB_ERR_UNSUPPORTED;
  if (tokens == 0) return CDB_OK;
  if (k == nullptr || v == nullptr || rows == nullptr) return CDB_ERR_NULL;
  if (num_heads > 0 && (q == nullptr || q_out == nullptr)) return CDB_ERR_NULL;
  if (rope_style != 0 && (rope_cos == nullptr || rope_sin == nullptr || positions == nullptr)) return CDB_ERR_NULL;
  if (rope_style != 0 && max_positions <= 0) return CDB_ERR_SHAPE;
  Kv8WriteParams P{};
  const int code =
      kv8_cache_of(&P.cache, codes, scales, num_cache_layers, pool_blocks, num_kv_heads, head_dim, block_size);
  if (code != CDB_OK) return code;
  if (dtype != CDB_DTYPE_F32 && dtype != CDB_DTYPE_BF16) return CDB_ERR_UNSUPPORTED;
  if (q_stride == 0) q_stride = (int64_t)num_heads * head_dim;
  if (kv_stride == 0) kv_stride = (int64_t)num_kv_heads * head_dim;
  if ((num_heads > 0 && q_stride < (int64_t)num_heads * head_dim) || kv_stride < (int64_t)num_kv_heads * head_dim)
    return CDB_ERR_SHAPE;
  if (q_out != nullptr && reinterpret_cast<uintptr_t>(q_out) % 16 != 0) return CDB_ERR_SHAPE;
  const int size = dtype == CDB_DTYPE_F32 ? 4 : 2;
  P.q = q; P.k = k; P.v = v; P.q_out = q_out;
  P.layer = layer; P.rows = rows; P.pool_rows = pool_blocks * block_size; P.positions = positions;
  P.cos = rope_cos; P.sin = rope_sin; P.q_bias = q_bias; P.k_bias = k_bias;
  P.tokens = tokens; P.q_stride = q_stride; P.kv_stride = kv_stride;
  P.num_heads = num_heads; P.max_positions = max_positions;
  P.vec = kv8_aligned(size, {q, k, v, q_bias, k_bias, rope_cos, rope_sin}, {q_stride, kv_stride});
  // A chunk of 16 tokens is one tile's worth of a prompt. Few tokens take one a wave, so that a decode
  // batch, whose every token is a run of its own, is not written 16 runs one after the other.
  P.chunk = tokens <= 1024 ? 1 : 16;
  P.chunks = (tokens + P.chunk - 1) / P.chunk;
  // Two heads a wave share the angles, which are twice a bf16 head's bytes: 7700 tokens of 16 x 128 take 41.8 us
  // against 44.1 with one (both before keys and values were read past the caches). In fp32 they are not, and the
  // larger waves cost more: 2300 of 55 x 96 37.6 against 35.1.
  P.heads_each = tokens <= 1024 || size == 4 ? 1 : 2;
  P.kv_blocks = (P.chunks * ((num_kv_heads + P.heads_each - 1) / P.heads_each) + 3) / 4;
  const int64_t q_blocks = (tokens * num_heads * (head_dim / 16) + 255) / 256;
  if (P.kv_blocks + q_blocks > 0x7fffffffll) return CDB_ERR_SHAPE;
  return dtype == CDB_DTYPE_F32 ? write_dim<float>(P, head_dim, rope_style, P.kv_blocks + q_blocks, stream)
                                : write_dim<bf16_t>(P, head_dim, rope_style, P.kv_blocks + q_blocks, stream);
}

extern "C" int cdb_batch_layout(const int32_t* past, const int32_t* lens, int32_t num_seqs, int32_t* block_table,
                                const int32_t* table_row, int32_t table_rows, int32_t table_width,
                                const int32_t* free_blocks, int32_t num_free, int32_t block_size, int32_t* cu_q,
                                int32_t* positions, int64_t* rows, int32_t token_capacity, int32_t* tile_seq,
                                int32_t* tile_q0, int32_t tile_capacity, int32_t* counts, hipStream_t stream) {
  using namespace cdb;
  if (num_seqs < 0 || num_seqs > CDB_LAYOUT_MAX_SEQS || table_rows < 0 || table_width <= 0 || num_free < 0 ||
      token_capacity < 0 || tile_capacity < 0)
    return CDB_ERR_SHAPE;
  if (block_size <= 0 || (block_size & (block_size - 1)) != 0) return CDB_ERR_SHAPE;
  if ((int64_t)table_width * block_size > (1ll << 30)) return CDB_ERR_SHAPE;
  if (table_row == nullptr && table_rows < num_seqs) return CDB_ERR_SHAPE;
  if (cu_q == nullptr || counts == nullptr) return CDB_ERR_NULL;
  if (num_seqs > 0 && (past == nullptr || lens == nullptr || block_table == nullptr)) return CDB_ERR_NULL;
  if ((token_capacity > 0 && (positions == nullptr || rows == nullptr)) ||
      (tile_capacity > 0 && (tile_seq == nullptr || tile_q0 == nullptr)) || (num_free > 0 && free_blocks == nullptr))
    return CDB_ERR_NULL;
  LayoutParams P{};
  P.past = past; P.lens = lens; P.table_row = table_row; P.free_blocks = free_blocks; P.table = block_table;
  P.num_seqs = num_seqs; P.table_rows = table_rows; P.table_width = table_width; P.num_free = num_free;
  P.bs_log2 = __builtin_ctz(block_size);
  P.cu_q = cu_q; P.positions = positions; P.rows = rows; P.tile_seq = tile_seq; P.tile_q0 = tile_q0; P.counts = counts;
  P.token_capacity = token_capacity; P.tile_capacity = tile_capacity;
  const size_t lds = sizeof(int32_t) * (4 * (size_t)num_seqs + 3);
  // Small workgroups start and scan sooner, large ones scan more requests at once: 24 prompts take 5.3 us in
  // workgroups of 256 and 6.6 in those of 1024, 1000 requests 9.7 us in 256, 9.5 in 512, 10.6 in 1024.
  if (num_seqs <= 256) layout_launch<256, 1>(P, lds, stream);
  else if (num_seqs <= 1024) layout_launch<512, 2>(P, lds, stream);
  else layout_launch<1024, (CDB_LAYOUT_MAX_SEQS + 1023) / 1024>(P, lds, stream);
  return hipGetLastError() == hipSuccess ? CDB_OK : CDB_ERR_HIP;
}
