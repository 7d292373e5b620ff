// Host-side argument checks shared by the 8-bit KV cache entry points.
#pragma once

#include <initializer_list>

#include "cdb_amd.h"
#include "kv8_common.h"

namespace cdb {

inline int kv8_cache_of(Kv8Cache* c, void* codes, void* scales, int32_t num_layers, int64_t pool_blocks,
                        int32_t num_kv_heads, int32_t head_dim, int32_t block_size) {
  if (codes == nullptr || scales == nullptr) return CDB_ERR_NULL;
  if (num_layers <= 0 || pool_blocks <= 0 || num_kv_heads <= 0) return CDB_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 96 && head_dim != 128) return CDB_ERR_UNSUPPORTED;
  if (block_size < kTile || (block_size & (block_size - 1)) != 0) return CDB_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(codes) % 16 != 0) return CDB_ERR_SHAPE;
  // Block ids are int32 and slots block * block_size are int64; the tile count must fit 63 bits.
  if (pool_blocks > 0x7fffffffll) return CDB_ERR_SHAPE;
  c->codes = static_cast<uint8_t*>(codes);
  c->scales = static_cast<uint8_t*>(scales);
  c->num_layers = num_layers;
  c->pool_blocks = pool_blocks;
  c->num_kv_heads = num_kv_heads;
  c->tile_log2 = __builtin_ctz(block_size / kTile);
  c->plane_tiles = (pool_blocks * num_kv_heads) << c->tile_log2;
  return CDB_OK;
}

// Whether 16-byte loads may be used: every base address and row stride is a multiple of 16 bytes.
inline bool kv8_aligned(int size, std::initializer_list<const void*> bases, std::initializer_list<int64_t> strides) {
  for (const void* p : bases)
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  for (int64_t s : strides)
    if (s * size % 16 != 0) return false;
  return true;
}

}  // namespace cdb
