// How attention over pages is laid out over the units (plain C++: host code only).
#pragma once
#include <stdint.h>

namespace pq {

constexpr int kPagedFewRows = 16;             // rows a sequence that the kernel for few rows takes

// rows of a workgroup of the kernel that a call of `rows` rows a sequence runs
inline int paged_tile_rows(int64_t rows) { return rows <= kPagedFewRows ? 16 : 128; }

inline int64_t paged_tiles(int B, int N, int Nk, int max_q) {
    const int64_t rows = static_cast<int64_t>(max_q) * (N / Nk), tile = paged_tile_rows(rows);
    return B * ((rows + tile - 1) / tile);
}

// Workgroups a KV head that the pages of all sequences are dealt out to: two on every unit, no more than there can be pages.  0: the row tiles alone
// fill the device, or nothing can be cut.
inline int paged_units(int B, int N, int Nk, int max_q, int max_kv, int n_cus) {
    const int64_t tiles = paged_tiles(B, N, Nk, max_q), units = 2 * static_cast<int64_t>(n_cus > 0 ? n_cus : 256) / Nk;
    const int64_t most = tiles * ((static_cast<int64_t>(max_kv) + 127) / 128), n = units < most ? units : most;
    return n > tiles ? static_cast<int>(n) : 0;
}

}  // namespace pq
