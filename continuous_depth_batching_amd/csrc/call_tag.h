// Tags of calls, by which workgroups tell that a workspace's partial results are this call's.
#pragma once

#include <atomic>
#include <chrono>
#include <cstdint>

namespace cdb {

// A tag that no other call of this process has, and that memory does not hold by chance.
inline uint64_t next_tag() {
  static std::atomic<uint64_t> calls{(uint64_t)std::chrono::steady_clock::now().time_since_epoch().count() << 20};
  uint64_t z = calls.fetch_add(1, std::memory_order_relaxed) * 0x9e3779b97f4a7c15ull;
  z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
  z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
  return (z ^ (z >> 31)) | 1;
}

}  // namespace cdb
