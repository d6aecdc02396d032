// Sequences whose keys and values lie in pages, as the append (paged_append.hip) and the attention (paged_attention.hip) see them.
//
// A cache holds `pages` pages of `page` tokens (a power of two from 16 to 256) for each of KV heads:
//   keys    [pages, KV, page, D]              a token's row as the matrix instruction wants it
//   values  [pages, KV, page / 16, D, 16]     blocks of sixteen tokens, d by d: the operand of V^T P^T holds neighbouring keys of one d, so that a lane
//                                             reads them in one go and nothing is transposed in the attention
// in 16 bits, or in 8 as e4m3 with a scale 2^(byte - 127) for each page and head ([pages, KV]).  A power of two moves the exponent alone: a value keeps
// its four significant bits under any scale, and only what falls below the format's range (2^-9 of the scale; the page's largest value is 2^7.8 of it or more) is lost.
//
// Every index that comes from device memory is bounded before it is used: a sequence's rows to the tokens of the call, its keys to what the table reaches, a page's
// number to the cache (one outside of it holds no keys and takes none, and so does what lies behind the table).
#pragma once
#include <type_traits>

#include "common.h"

namespace mhip {

constexpr int kBlock = 16;                 // tokens of a block of values

struct Sequences {
    const int32_t* table;                  // [B, width]: page numbers
    const int32_t* lengths;                // [B]: keys, the call's tokens among them
    const int32_t* starts;                 // [B + 1]: first row of each sequence's tokens
    int B, width, T, page_shift;

    __device__ __forceinline__ int start(int b) const { return min(max(starts[b], 0), T); }
    __device__ __forceinline__ int tokens(int b) const { return max(min(starts[b + 1], T) - start(b), 0); }
    // the keys that have a place; the position behind the last token, which may lie behind the table
    __device__ __forceinline__ int reach() const { return width << page_shift; }
    __device__ __forceinline__ int keys(int b) const { return min(max(lengths[b], 0), reach()); }
    __device__ __forceinline__ int end(int b) const { return min(max(lengths[b], 0), 1 << 30); }
    // the same where it only matters which keys a token sees: no further behind the table than its tokens are many (below 2^25)
    __device__ __forceinline__ int bounded_end(int b) const { return min(max(lengths[b], 0), reach() + tokens(b)); }
};

// Between what lanes of a wave write to LDS and what others of the same wave read of it, either way round.  The hardware serves a wave's accesses to LDS in order, so that nothing waits: this keeps
// the compiler from another order, which may not know that the addresses meet.
__device__ __forceinline__ void wave_in_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// sum over the lanes up to this one
__device__ __forceinline__ int wave_scan(int v) {
    auto step = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
        v += __builtin_amdgcn_update_dpp(0, v, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
    };
    step(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xF>{});      // row_shr 1, 2, 4, 8 inside sixteen lanes
    step(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xF>{});
    step(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xF>{});
    step(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xF>{});
    step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});      // row_bcast 15, 31
    step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});
    return v;
}

// The sequence that unit `u` belongs to where sequence b has units(b) of them, -1 behind the last; `first`: units in front of the sequence.  By a whole wave, 64
// sequences a step; u is the same in all lanes.
template <typename F>
__device__ __forceinline__ int sequence_of(int B, int u, F units, int& first) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int n = b0 + lane < B ? units(b0 + lane) : 0, sum = wave_scan(n);
        const uint64_t m = __ballot(before + sum > u);
        if (m) {
            const int l = __builtin_ctzll(m);
            first = before + __builtin_amdgcn_readlane(sum - n, l);
            return b0 + l;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return -1;
}

// 2^(byte - 127); the byte 0, which no append writes, as 1
__device__ __forceinline__ float scale_of(uint32_t byte) { return __builtin_bit_cast(float, max(byte, 1u) << 23); }

// What the two entry points ask of a cache and of sequences before anything is planned or launched: their sizes, and then what they point to.
int check_sizes(const char* what, const mhip_paged_cache* c, const mhip_sequences* s);
int check_paged(const char* what, const mhip_paged_cache* c, const mhip_sequences* s, int dtype, bool* empty);

inline Sequences sequences(const mhip_paged_cache* c, const mhip_sequences* s) {
    return {s->table, s->lengths, s->starts, (int)s->sequences, (int)s->width, (int)s->tokens, __builtin_ctzll((uint64_t)c->page_size)};
}

}  // namespace mhip
