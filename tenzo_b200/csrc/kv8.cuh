// The INT8 caches as the calls on drafted trees and bounded caches see them (kv8_rows.cu, attention_tree.cu): blocks of `slots` tokens behind a table, so that the
// block pools (16 slots) and the contiguous cache (one block a sequence) are one thing. Sixteen tokens that start at a multiple of sixteen never
// straddle a block: 2 KB of codes and 64 bytes of scales that one copy each brings in.
#pragma once
#include "kv4.cuh"

namespace tz {

constexpr int kK8Hd = 128, kK8Chunk = 16;
constexpr int kK8ErrWait = kK4ErrWait, kK8ErrIndex = kK4ErrIndex;     // bits of the error flags

// Row of a token in the pools: codes at 128 times this, scales, weight and position at this.
__device__ __forceinline__ size_t kv8_row(const tenzo_kv8_cache& c, int layer, int kvh, int block, int slot) {
    return (((size_t)block * c.n_layers + layer) * c.n_kv + kvh) * c.slots + slot;
}
// Block of a place; -1 for a table entry out of range. The caller has checked the table row and the place.
__device__ __forceinline__ int kv8_block(const tenzo_kv8_cache& c, int seq, int place) {
    const int id = ld_l2(c.block_table + (size_t)seq * c.table_stride + place / c.slots);
    return id >= 0 && id < c.n_blocks ? id : -1;
}

inline bool kv8_aligned(const void* p, uintptr_t to) { return !(reinterpret_cast<uintptr_t>(p) & (to - 1)); }
inline bool kv8_cache_ok(const tenzo_kv8_cache& c) {
    if (!c.k || !c.v || !c.scale_k || !c.scale_v || !c.block_table) return false;
    if (!kv8_aligned(c.k, 16) || !kv8_aligned(c.v, 16) || !kv8_aligned(c.scale_k, 16) || !kv8_aligned(c.scale_v, 16)) return false;
    if (c.n_blocks <= 0 || c.n_layers <= 0 || c.n_kv <= 0 || c.slots <= 0 || c.slots % kK8Chunk || c.table_rows <= 0 || c.table_stride <= 0) return false;
    // (a row's number is an int in the copies' coordinates; the quotients never pass 64 bits)
    return (long long)c.n_blocks * c.n_layers <= 0x7fffffffLL && (long long)c.n_kv * c.slots <= 0x7fffffffLL / ((long long)c.n_blocks * c.n_layers);
}
// Whether two ranges of memory have bytes in common (a null range has none).
inline bool kv8_overlap(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + b_bytes && y < x + a_bytes;
}
inline size_t kv8_table_bytes(const tenzo_kv8_cache& c) { return (size_t)c.table_rows * c.table_stride * sizeof(int); }
inline size_t kv8_rows(const tenzo_kv8_cache& c) { return (size_t)c.n_blocks * c.n_layers * c.n_kv * c.slots; }
inline long long kv8_places(const tenzo_kv8_cache& c) { return (long long)c.table_stride * c.slots; }

}  // namespace tz
