// How attention over pages is laid out over the units (plain C++: host code only).
#pragma once
#include <stdint.h>

namespace pq {

constexpr int kPagedFewRows = 16;             // rows a sequence that the kernel for few rows takes

// rows of a workgroup of the kernel that a call of `rows` rows a sequence runs
inline int paged_tile_rows(int64_t rows) { return rows <= kPagedFewRows ? 16 : 128; }

// Slices a sequence may be cut into: enough that two workgroups stand on every unit, twice as many where sequences can differ (the device deals
// the slices out by the lengths it finds; a workgroup without one ends at once), no more than there are pages.
inline int paged_splits(int B, int N, int Nk, int max_q, int max_kv, int n_cus) {
    const int64_t rows = static_cast<int64_t>(max_q) * (N / Nk), tile = paged_tile_rows(rows);
    const int64_t planes = static_cast<int64_t>(B) * Nk * ((rows + tile - 1) / tile), slots = 2 * static_cast<int64_t>(n_cus > 0 ? n_cus : 256);
    if (planes >= slots) return 1;
    int64_t n = (slots + planes - 1) / planes;
    if (B > 1) n *= 2;
    const int64_t pages = (static_cast<int64_t>(max_kv) + 127) / 128;
    n = n < pages ? n : pages;
    return static_cast<int>(n < 1 ? 1 : n);
}

}  // namespace pq
