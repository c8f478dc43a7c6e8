// What the paged cache's kernels share: a sequence's extent, its pages, which of its keys exist, and keys from polar codes.
#pragma once
#include "pq_mfma.h"
#include "pq_paged_internal.h"

namespace pq {

typedef __attribute__((address_space(3))) uint32_t lds_u32;
typedef __attribute__((address_space(3))) floatx2_a lds_f2;

// Everything the device is told is brought within what the host has checked, so that no table entry or count leads out of a buffer: a page
// outside of the pool does not exist (its tokens are not seen, nothing is written to it).
struct PagedSequence {
    int first, rows, kv, past, sealed;        // its packed rows from `first` on; tokens in all, those before the call (may be negative), sealed pages
};

__device__ __forceinline__ int within(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

__device__ __forceinline__ PagedSequence paged_sequence(const PagedCache& c, int b) {
    PagedSequence s;
    s.first = within(c.q_start[b], 0, c.T);
    s.rows = within(c.q_start[b + 1], s.first, c.T) - s.first;
    s.kv = within(c.kv_len[b], 0, c.max_kv);
    s.past = s.kv - s.rows;
    s.sealed = c.n_sealed ? within(c.n_sealed[b], 0, s.kv / kPageTokens) : 0;
    return s;
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// of a workgroup's own sequence: in scalar registers
__device__ __forceinline__ PagedSequence own_sequence(const PagedCache& c, int b) {
    const PagedSequence s = paged_sequence(c, b);
    return PagedSequence{uniform(s.first), uniform(s.rows), uniform(s.kv), uniform(s.past), uniform(s.sealed)};
}

// Physical pages of logical page p < W (the same in all lanes), -1 where there is none.
__device__ __forceinline__ int page_of(const int32_t* table, int n, int64_t at) {
    const int p = uniform(table[at]);
    return static_cast<unsigned>(p) < static_cast<unsigned>(n) ? p : -1;
}
__device__ __forceinline__ int key_page(const PagedCache& c, const PagedSequence& s, int b, int p) {
    if (p < s.sealed) return page_of(c.pages, c.codes.n, static_cast<int64_t>(b) * c.W + p);
    return p - s.sealed < c.Wo ? page_of(c.open_pages, c.keys.n, static_cast<int64_t>(b) * c.Wo + (p - s.sealed)) : -1;
}
__device__ __forceinline__ int value_page(const PagedCache& c, int b, int p) { return page_of(c.value_pages, c.values.n, static_cast<int64_t>(b) * c.W + p); }

// How many pages a slice of the sequence holds.  `slots` workgroups' worth of slices are dealt out over all sequences by their pages and
// row tiles, so that a batch of unequal sequences keeps the device as busy as an even one; from the device's own lengths, which the host need not know.
__device__ __forceinline__ int pages_per_slice(const PagedCache& c, int pages, int n_splits, int slots, int tile_rows) {
    if (n_splits == 1 || pages <= 1) return pages > 0 ? pages : 1;
    const int rep = c.N / c.Nk;
    int64_t total = 0;
    for (int i = threadIdx.x & 63; i < c.B; i += kWave) {
        const PagedSequence s = paged_sequence(c, i);
        total += static_cast<int64_t>((s.kv + kPageTokens - 1) / kPageTokens) * ((s.rows * rep + tile_rows - 1) / tile_rows);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
    int64_t per = (total * c.Nk + slots - 1) / slots;
    per = per < 1 ? 1 : per > pages ? pages : per;
    int n = (pages + static_cast<int>(per) - 1) / static_cast<int>(per);
    n = n < n_splits ? n : n_splits;
    return uniform((pages + n - 1) / n);
}

__device__ __forceinline__ float both_rows_max(float v) {        // of lanes l and l ^ 16
    typedef unsigned int uint2_x __attribute__((ext_vector_type(2)));
    const uint2_x r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}

// ---- rows to LDS ------------------------------------------------------------------------------------------------------
// 16 bytes per lane from `offset` bytes behind a (uniform) address into 1 KiB of LDS at `lds` (uniform), lane after lane.  Not known to the
// compiler's count of loads in flight, which would make every read of LDS wait for them: rows_arrived() before the data is read, by the wavefront
// that asked for it, and a barrier behind that before others read it.  The load reads M0 one wait state after a scalar write at the earliest; inside
// an asm statement that is ours to see to.
__device__ __forceinline__ u32x4_a rows_at(const void* p) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return u32x4_a{static_cast<uint32_t>(uniform(static_cast<int>(a))), static_cast<uint32_t>(uniform(static_cast<int>(a >> 32))) & 0xffffu, 0xffffffffu, 0x00020000u};
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void rows_to_lds(u32x4_a rows, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(offset), "s"(rows), "s"(uniform(static_cast<int>(lds))) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void rows_arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// ---- keys from codes --------------------------------------------------------------------------------------------------
// A sealed key enters the score product as float16 whatever the model's type: r cos a and r sin a come out of one multiply-add each that
// rounds to float16 (bfloat16 would take a conversion more and round eight times as coarsely).  So that nothing leaves float16's range, a
// page's radii are scaled by a power of two, and so are a bfloat16 query's elements; both are taken back with the score's scale.
constexpr int kHalfTop = 13;                  // scaled magnitudes lie below 2^13

// the e with v < 2^e, for a finite v > 0 (0 for anything else)
__device__ __forceinline__ int exponent_above(float v) {
    return v > 0.0f && v < INFINITY ? __builtin_amdgcn_frexp_expf(v) : 0;
}

__device__ __forceinline__ uint32_t cos_sin_half(float turns) {
    return pack_pair<F16>(__builtin_amdgcn_cosf(turns), __builtin_amdgcn_sinf(turns));
}
constexpr float kTurn = 0.15915494309189535f;

// r * (low half, high half of cs), rounded to float16, into the low (LO) or high half of a word
template <bool SIN, bool LO>
__device__ __forceinline__ void times_half(uint32_t& w, float r, uint32_t cs) {
    if constexpr (LO && !SIN) asm("v_fma_mixlo_f16 %0, %1, %2, 0 op_sel_hi:[0,1,0]" : "=v"(w) : "v"(r), "v"(cs));
    else if constexpr (LO) asm("v_fma_mixlo_f16 %0, %1, %2, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]" : "=v"(w) : "v"(r), "v"(cs));
    else if constexpr (!SIN) asm("v_fma_mixhi_f16 %0, %1, %2, 0 op_sel_hi:[0,1,0]" : "+v"(w) : "v"(r), "v"(cs));
    else asm("v_fma_mixhi_f16 %0, %1, %2, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]" : "+v"(w) : "v"(r), "v"(cs));
}

// 16 bytes of a key: pairs 4 c .. 4 c + 3 as (x x x x y y y y), from their radii and angles' cos and sin
__device__ __forceinline__ u32x4_a quad_of_pairs(const float (&r)[4], const uint32_t (&cs)[4]) {
    u32x4_a k;
    uint32_t w[4];
    times_half<false, true>(w[0], r[0], cs[0]);
    times_half<false, false>(w[0], r[1], cs[1]);
    times_half<false, true>(w[1], r[2], cs[2]);
    times_half<false, false>(w[1], r[3], cs[3]);
    times_half<true, true>(w[2], r[0], cs[0]);
    times_half<true, false>(w[2], r[1], cs[1]);
    times_half<true, true>(w[3], r[2], cs[2]);
    times_half<true, false>(w[3], r[3], cs[3]);
    k.x = w[0]; k.y = w[1]; k.z = w[2]; k.w = w[3];
    return k;
}

// four 6-bit codes in the low 24 bits -> one a byte
__device__ __forceinline__ uint32_t unpack_codes6(uint32_t x) {
    return (x & 0x3Fu) | ((x & 0xFC0u) << 2) | ((x & 0x3F000u) << 4) | ((x & 0xFC0000u) << 6);
}

// float16 or bfloat16 words of a query, times 2^e, as float16 words (exact within float16's range: bfloat16 has fewer digits)
template <typename T>
__device__ __forceinline__ uint32_t scaled_half(uint32_t w, float factor) {
    return pack_pair<F16>(lo2f<T>(static_cast<uint16_t>(w & 0xffffu)) * factor, lo2f<T>(static_cast<uint16_t>(w >> 16)) * factor);
}

}  // namespace pq
