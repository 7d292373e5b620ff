// Device helpers of the 8-bit KV cache kernels.
//
// The cache holds tiles of 16 tokens of one KV head, keys and values apart: e4m3 codes and one
// power-of-two scale a tile, kept as its biased exponent (byte b stands for 2^(b - 127)). A scale
// that is a power of two makes every step but the rounding to e4m3 itself exact: scaling a value
// down, widening a code to bf16 or fp16, and rescaling a code when a tile's scale grows.
//
// Tile t (counted over [layer, plane, block, head, block_size / 16]) has its codes at t * 16 * D and
// its scale at t. Inside a tile the codes lie as the MFMA kernels read them, 16 bytes a lane:
//   keys   [D / 16][16 tokens][16]: unit u of token r holds elements 16u..16u+15;
//   values [4][D][4 tokens]: group g of element d holds tokens 4g..4g+3.
#pragma once

#include "cdb_common.h"

namespace cdb {

constexpr int kTile = 16;  // tokens of a tile

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// A tile's scale byte as every reader takes it, 1 to 254: 0, of a tile that was never written, is read as 1, and 255,
// which no write leaves, as 254.
CDB_DEVICE uint32_t scale_byte_read(uint32_t b) { return min(max(b, 1u), 254u); }
// 2^(b - 127) of a scale byte, as the conversion instructions take it.
CDB_DEVICE float scale_of(uint32_t b) { return __uint_as_float(b << 23); }
// 2^(127 - b): the factor that brings a value to a code. Bytes above 253 give 0.
CDB_DEVICE float inverse_scale_of(uint32_t b) { return b >= 254u ? 0.f : __uint_as_float((254u - b) << 23); }

// The byte of the smallest power of two s with amax / s <= 448 = 1.75 * 2^8, for a finite amax >= 0:
// its exponent less 8, one more where the mantissa is above 1.75.
CDB_DEVICE int scale_byte(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int b = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(b, 1), 254);
}

// |x| where x is finite, else 0: infinities and NaN take no part in a tile's scale.
CDB_DEVICE float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// |x| as bits, which order as the sizes do; from kNotFinite on, x is an infinity or NaN.
constexpr uint32_t kNotFinite = 0x7f800000u;
CDB_DEVICE uint32_t size_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Four values as e4m3 codes in one word: divided by a scale, rounded to nearest even. The conversion makes an
// infinity or NaN the NaN code by itself (both forms checked over every code, every midpoint and its neighbours).
typedef short s16x2_t __attribute__((ext_vector_type(2)));
CDB_DEVICE uint32_t codes_of(float a, float b, float c, float d, float scale) {
  s16x2_t w = {0, 0};
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, a, b, scale, false);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, c, d, scale, true);
  return __builtin_bit_cast(uint32_t, w);
}
CDB_DEVICE uint32_t codes_of(float a, float b, float c, float d) {
  const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Codes of one word rounded again for a scale `growth` times larger.
CDB_DEVICE uint32_t recode(uint32_t w, float growth) {
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return codes_of(lo.x, lo.y, hi.x, hi.y, growth);
}
// 2^(now - old) for old <= now; where it leaves the normal range every code rounds to 0 all the same.
CDB_DEVICE float growth_of(int old, int now) { return scale_of((uint32_t)min(127 + now - old, 254)); }

// Byte mask of a word's tokens below n (n <= 0: none, n >= 4: all).
CDB_DEVICE uint32_t tokens_below(int n) { return n <= 0 ? 0u : n >= 4 ? ~0u : (1u << (8 * n)) - 1u; }

// Byte mask of the low four bits of m.
CDB_DEVICE uint32_t tokens_in(uint32_t m) { return (((m & 15u) * 0x00204081u) & 0x01010101u) * 255u; }

// N storage elements as they lie; vec as for load_f32, kOnce: they are read once and need no place in the caches.
template <typename T, int N, bool kOnce = false> CDB_DEVICE Vec<T, N> load_raw(const T* p, bool vec) {
  Vec<T, N> x;
  if (vec) {
    if constexpr (kOnce) x.load_nt(p);
    else x.load(p);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) x.set_pair(i, Elem<T>::load(p + i), Elem<T>::load(p + i + 1));
  }
  return x;
}

// N storage elements as fp32; vec: p is aligned for 16-byte loads (8-byte ones where N elements are 8 bytes).
template <typename T, int N, bool kOnce = false> CDB_DEVICE void load_f32(const T* p, float* out, bool vec) {
  if (vec) {
    Vec<T, N> x;
    if constexpr (kOnce) x.load_nt(p);
    else x.load(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = x.get(i);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = Elem<T>::load(p + i);
  }
}

// N consecutive elements of a head, from element d on: x + bias, rotated, in fp32 with every product
// and sum rounded once. STYLE 1 pairs element d with d + D/2, STYLE 2 pairs even and odd elements.
// Runs of N must not cross D/2 (STYLE 1); cos/sin point at the position's row of D/2 angles.
template <typename T, int D, int STYLE, int N>
CDB_DEVICE void load_rotated(const T* head, const T* bias, const float* cos, const float* sin, int d, bool vec,
                             float* out) {
  load_f32<T, N>(head + d, out, vec);
  if (bias != nullptr) {
    float b[N];
    load_f32<T, N>(bias + d, b, vec);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = add_rn(out[i], b[i]);
  }
  if constexpr (STYLE == 1) {
    const bool low = d < D / 2;
    const int pd = low ? d + D / 2 : d - D / 2;
    const int a = low ? d : pd;
    float p[N], c[N], s[N];
    load_f32<T, N>(head + pd, p, vec);
    if (bias != nullptr) {
      float b[N];
      load_f32<T, N>(bias + pd, b, vec);
#pragma unroll
      for (int i = 0; i < N; ++i) p[i] = add_rn(p[i], b[i]);
    }
    load_f32<float, N>(cos + a, c, vec);
    load_f32<float, N>(sin + a, s, vec);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float ps = mul_rn(p[i], s[i]);
      out[i] = add_rn(mul_rn(out[i], c[i]), low ? -ps : ps);
    }
  } else if constexpr (STYLE == 2) {
    float c[N / 2], s[N / 2];
    load_f32<float, N / 2>(cos + d / 2, c, vec);
    load_f32<float, N / 2>(sin + d / 2, s, vec);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float e = out[2 * i], o = out[2 * i + 1];
      out[2 * i] = sub_rn(mul_rn(e, c[i]), mul_rn(o, s[i]));
      out[2 * i + 1] = add_rn(mul_rn(o, c[i]), mul_rn(e, s[i]));
    }
  }
}

// Two runs of N elements of a head, x + bias, rotated: STYLE 1 the elements from d on, in its first half, and
// those from d + D/2 on, which share their angles; otherwise the elements from d on and from d + N on.
template <typename T, int D, int STYLE, int N>
CDB_DEVICE void load_rotated_pair(const T* head, const T* bias, const float* cos, const float* sin, int d, bool vec,
                                  float* a, float* b) {
  if constexpr (STYLE == 1) {
    float c[N], s[N];
    load_f32<T, N>(head + d, a, vec);
    load_f32<T, N>(head + d + D / 2, b, vec);
    load_f32<float, N>(cos + d, c, vec);
    load_f32<float, N>(sin + d, s, vec);
    if (bias != nullptr) {
      float e[N];
      load_f32<T, N>(bias + d, e, vec);
#pragma unroll
      for (int i = 0; i < N; ++i) a[i] = add_rn(a[i], e[i]);
      load_f32<T, N>(bias + d + D / 2, e, vec);
#pragma unroll
      for (int i = 0; i < N; ++i) b[i] = add_rn(b[i], e[i]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float x = a[i], y = b[i];
      a[i] = sub_rn(mul_rn(x, c[i]), mul_rn(y, s[i]));
      b[i] = add_rn(mul_rn(y, c[i]), mul_rn(x, s[i]));
    }
  } else {
    load_rotated<T, D, STYLE, N>(head, bias, cos, sin, d, vec, a);
    load_rotated<T, D, STYLE, N>(head, bias, cos, sin, d + N, vec, b);
  }
}

// A value and the one of the lane that differs in bit 4 (or 5), in either order: two vector
// instructions, against the LDS round trip of a permute.
CDB_DEVICE f32x2_t pair16(float v) {
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return (f32x2_t){__uint_as_float(x[0]), __uint_as_float(x[1])};
}
CDB_DEVICE f32x2_t pair32(float v) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return (f32x2_t){__uint_as_float(x[0]), __uint_as_float(x[1])};
}

// Max, and sum, over the four lanes that differ in bits 4 and 5.
CDB_DEVICE float column_max(float v) {
  f32x2_t x = pair16(v);
  x = pair32(fmaxf(x[0], x[1]));
  return fmaxf(x[0], x[1]);
}
CDB_DEVICE float all_max(float v) { return column_max(row16_max(v)); }  // over the wave
CDB_DEVICE float column_sum(float v) {
  f32x2_t x = pair16(v);
  x = pair32(x[0] + x[1]);
  return x[0] + x[1];
}

// 8 codes (two words) widened to bf16 with their scale: exact, e4m3 has 4 significant bits.
CDB_DEVICE bf16x8_t widen_bf16(uint32_t w0, float s0, uint32_t w1, float s1) {
  union { bf16x2_t p[4]; bf16x8_t v; } u;
  u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s0, false);
  u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s0, true);
  u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s1, false);
  u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s1, true);
  return u.v;
}

// 8 codes (two words) widened to fp16 by powers of two.
CDB_DEVICE f16x8_t widen_f16(uint32_t w0, float s0, uint32_t w1, float s1) {
  union { f16x2_t p[4]; f16x8_t v; } u;
  u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, s0, false);
  u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, s0, true);
  u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, s1, false);
  u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, s1, true);
  return u.v;
}

// Scores of this size and more are spaced too widely for a raise: a sum with it would round by more than fp16 has room.
constexpr float kWideScore = 0x1p22f;

// fp32 models take probabilities as two fp16 parts. The second, what the first leaves, is raised by 2^11 and meets
// values lowered by as much: it is then as large as the first, as far above fp16's smallest step. Values are raised by
// 2^7 (448 * 2^7 is within fp16), which keeps the lowered ones exact down to scales 2^11 below the unit.
constexpr float kSecondRaise = 2048.f;
template <typename T> constexpr int kValueRaise = sizeof(T) == 4 ? 7 : 0;

// The unit that values are widened in and products with them counted in: 2^(ref - 127). fp16 holds the values of a
// tile exactly if its scale is at most the unit and no more than 2^kExact below it, so the unit moves where a tile's
// is not, and the accumulators, fp32, move with it: up with a larger scale, and down for a smaller one, but never
// more than 2^60 below the largest scale met, so that 2^30 products of 2^31 at most stay within fp32. Values of
// tiles 2^(60 + kExact) and more below the largest scale met lose bits, the last of them 2^94 below it (fp32 models:
// 2^101).
template <typename T> struct ValueUnit {
  static constexpr int kExact = sizeof(T) == 4 ? 11 : 15, kDeep = 60;
  int ref = 1, met = 1;

  // Whether a tile of this scale needs another unit.
  CDB_DEVICE bool moves(int b) const { return (uint32_t)(ref - b) > (uint32_t)kExact; }
  // Takes it; returns the power of two that the accumulators move by.
  CDB_DEVICE int move(int b) {
    met = max(met, b);
    const int to = max(b, met - kDeep), by = ref - to;
    ref = to;
    return by;
  }
  // A scale in the unit, as the conversions take it.
  CDB_DEVICE float scale(int b) const { return scale_of((uint32_t)max(127 + b + kValueRaise<T> - ref, 1)); }
  // The exponent that brings an accumulator back.
  CDB_DEVICE int back() const { return ref - 127 - kValueRaise<T>; }
};

// The cache as a kernel sees it: all strides in tiles.
struct Kv8Cache {
  uint8_t* codes;
  uint8_t* scales;
  int64_t plane_tiles;  // pool_blocks * num_kv_heads * tiles of a block
  int64_t pool_blocks;
  int32_t num_layers;
  int32_t num_kv_heads;
  int32_t tile_log2;    // log2 of the tiles of a block

  CDB_DEVICE int64_t tile(int64_t layer, int plane, int64_t block, int head, int sub) const {
    return (layer * 2 + plane) * plane_tiles + ((block * num_kv_heads + head) << tile_log2) + sub;
  }
};

}  // namespace cdb
