// How attention over pages is laid out over the units (plain C++: host code only).
#pragma once
#include <stdint.h>

namespace pq {

constexpr int kPagedFewRows = 16;             // rows a sequence that the kernel for few rows takes
constexpr int kPagedMostRows = 256;           // rows of the largest tile

// Rows of a workgroup of the kernel that a call of `rows` rows a sequence runs.  A tile of 256 rows makes its keys for twice as many rows as one of 128, but half as
// many workgroups share the work.  With 32 heads over 8, 256 and 128 rows (before a tile's codes were asked for earlier): 1273 and 1393 us for 2 K tokens behind 32 K, 121
// and 131 for 512 behind 8 K, 707 and 751 for eight such sequences, 279 and 295 for eight of up to that length; but 23 and 21 for 100 behind 1000, and 152 and 144 for 2 K
// behind 2 K.
inline int paged_tile_rows(int64_t rows, int64_t max_kv) { return rows <= kPagedFewRows ? 16 : rows <= 128 || max_kv <= 4096 ? 128 : kPagedMostRows; }

inline int64_t paged_tiles(int B, int N, int Nk, int max_q, int max_kv) {
    const int64_t rows = static_cast<int64_t>(max_q) * (N / Nk), tile = paged_tile_rows(rows, max_kv);
    return B * ((rows + tile - 1) / tile);
}

// Workgroups a KV head that the pages of all sequences are dealt out to: as many as stand on the device at once (two on every unit, one of 256 rows), no more than
// there can be pages.  0: the row tiles alone fill the device, or nothing can be cut.
inline int paged_units(int B, int N, int Nk, int max_q, int max_kv, int n_cus) {
    const int64_t tiles = paged_tiles(B, N, Nk, max_q, max_kv), slots = n_cus > 0 ? n_cus : 256;
    const int64_t units = (paged_tile_rows(static_cast<int64_t>(max_q) * (N / Nk), max_kv) == kPagedMostRows ? 1 : 2) * slots / Nk;
    const int64_t most = tiles * ((static_cast<int64_t>(max_kv) + 127) / 128), n = units < most ? units : most;
    return n > tiles ? static_cast<int>(n) : 0;
}

}  // namespace pq
