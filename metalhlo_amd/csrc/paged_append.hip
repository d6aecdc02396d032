// Keys and values of new tokens into a paged cache (paged.h), the position rotation applied on the way; in 8 bits with the page's scale.
//
//   position  p = lengths[b] - tokens(b) + i of token i of sequence b, its page table[b, p / page], its slot p % page
//   rotation  of the first R elements of a head, as mhip_rope turns them: with x = [x1 | x2] (halves) y = [x1 cos - x2 sin | x1 sin + x2 cos], row p of `freqs`
//             holding the cosines and then the sines.  fp32, and one rounding, to the type that is stored.
//   8 bits    the page's scale is the least power of two under which its largest value is at most 448.  Where the page holds tokens already it never shrinks, and
//             where it grows by 2^n the held values are multiplied by 2^-n and rounded, which changes none that stays above 2^-6 of the new scale.
//
// Bound by memory: every new value is read once and written once.  9450 tokens of 32 query and 8 key heads of 128 in 8 bits (218 MB) 46 us, 4.7 TB/s, 32000 (737 MB)
// 140 us, 5.3 TB/s; 6300 of 16 heads of 96 in 16 bits (92 MB) 20 us, 4.5 TB/s; a decode step of 48 sequences 5.6 us and of one 4.7, which is latency.
// Where scales grow in a decode step, which of 48 sequences' 768 some nearly always do, the few lanes of a row move the page's held values: 25 to 84 us, and 67 where all grow.  Two kernels:
//
//   paged_append_kernel   A wave a block of sixteen tokens, a workgroup a page (a scale needs all of its tokens), with a few heads of keys, values or queries one behind the other: the cosines and sines stay in
//                         registers from head to head, and the next head is on its way while this one's scale is found and its values are stored.  Values pass through LDS, which turns a block's rows into its columns.
//   append_few_kernel     No more tokens than sequences (a decode step): a row of a token is a few lanes' work, and a workgroup takes many heads of one page.
#include "paged.h"

namespace mhip {
namespace {

struct AppendArgs {
    const void *k, *v, *q;
    void* q_out;
    const float* freqs;
    char *keys, *values;
    uint8_t *key_scales, *value_scales;
    Sequences s;
    int pages, KV, H, R, positions, heads_a_part, parts;
    int64_t ks[2], vs[2], qs[2], os[2];       // token and head strides in elements
};

// 8 floats of 16 bytes of T
template <typename T>
__device__ __forceinline__ void to_floats(u32x4 w, float* x) {
    const Vec16<T> t = __builtin_bit_cast(Vec16<T>, w);
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = Elem<T>::to_f32(t.v[e]);
}
template <typename T>
__device__ __forceinline__ u32x4 to_vector(const float* x) {
    Vec16<T> t;
#pragma unroll
    for (int e = 0; e < 8; e++) t.v[e] = Elem<T>::from_f32(x[e]);
    return __builtin_bit_cast(u32x4, t);
}
// four e4m3 of x * inv, of `most` at most where that is finite; e4m3 has no infinities, so what is not finite becomes NaN
__device__ __forceinline__ uint32_t pack8(const float* x, float inv, float most) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        y[e] = x[e] * inv;
        y[e] = fabsf(y[e]) <= 448.f ? __builtin_amdgcn_fmed3f(y[e], -most, most) : __builtin_nanf("");
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}
// the held values of four tokens or d under the grown scale
__device__ __forceinline__ uint32_t moved8(uint32_t w, float factor) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    const float x[4] = {lo[0], lo[1], hi[0], hi[1]};
    return pack8(x, factor, 448.f);
}
__device__ __forceinline__ float finite_max(float m, float x) { return fmaxf(m, fabsf(x) < INFINITY ? fabsf(x) : 0.f); }

// The exponent byte of the least scale of at least 2^-126 with amax <= 448 * scale (448 = 1.75 * 2^8).
__device__ __forceinline__ int scale_byte(float amax) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, amax);
    return max((int)(bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000 ? 1 : 0), 1);
}

// Rows of keys and queries are whole lines and are stored past the caches (us, plain | so: 9450 tokens of 32 and 8 heads of 128 into pages of 64 49.3 | 39.2, of 16 48.6 | 37.2, of 256 52.2 | 46.5;
// where only a part of a row is turned, so that a store has parts of lines, 64 of 128 elements 48.6 | 43.0, 48 of 96 in 12600 tokens of 16 heads 44.8 | 36.7, in 6300 17.9 | 19.0;
// loads so: 47.6, and 23.7 | 32.3 where two heads share a line).
template <typename V, typename T>
__device__ __forceinline__ void put_stream(T* p, V v) { __builtin_nontemporal_store(v, reinterpret_cast<V*>(p)); }

// The page that unit u of a launch fills: `slot0` .. `slot1` of page `page_no` (which may be none of the cache's) take the tokens from row `row` on, whose positions begin at `pos`.
struct Fill {
    int page_no, slot0, slot1, pos;
    int64_t row;
    __device__ __forceinline__ bool find(const AppendArgs& a, int u) {
        const int shift = a.s.page_shift, page = 1 << shift;
        int first;
        auto touched = [&](int b) __attribute__((always_inline)) {
            const int n = a.s.tokens(b), end = a.s.end(b), begin = max(end - n, 0);
            return n ? ((end + page - 1) >> shift) - (begin >> shift) : 0;
        };
        const int b = sequence_of(a.s.B, u, touched, first);
        if (b < 0) return false;
        const int n = a.s.tokens(b), end = a.s.end(b), begin = max(end - n, 0);       // (more tokens than keys: the first ones have no place)
        const int at = (begin >> shift) + u - first;
        if (at < begin >> shift || at << shift >= end) return false;                  // (starts that are no starts: their sums may have wrapped)
        pos = max(begin, at << shift);
        const int stop = min(min(end, (at + 1) << shift), a.R ? a.positions : end);
        if (pos >= stop) return false;
        page_no = at < a.s.width ? a.s.table[(int64_t)b * a.s.width + at] : -1;
        slot0 = pos & (page - 1);
        slot1 = slot0 + stop - pos;
        row = a.s.start(b) + (n - (end - pos));
        return true;
    }
};

// the scale's byte for a page whose new tokens reach `top`, and whether the old ones have to follow it
// most: under the scale 2^120 what would be rounded to 256, which is 2^128, ends at the number below it (247 becomes 240, not quite half a step from 256)
struct Scale {
    float inv, factor, most;
    int byte;
    bool moves;
    __device__ __forceinline__ Scale(float top, int was, bool begun) {
        was = begun ? max(was, 1) : 0;
        byte = max(scale_byte(top), was);
        inv = scale_of(254 - byte);
        most = byte == 247 ? 247.f : 448.f;
        moves = begun && byte > was;
        factor = scale_of(127 + was - byte > 0 ? 127 + was - byte : 1);
    }
};
// the values that a page holds under a grown scale, by `lanes` lanes of which this one is `lane`
__device__ __forceinline__ void move_keys(char* page, int slot0, int D, float factor, int lane, int lanes) {
    u32x4* held = reinterpret_cast<u32x4*>(page);
    for (int i = lane; i < slot0 * D / 16; i += lanes) {
        u32x4 w = held[i];
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = moved8(w[e], factor);
        held[i] = w;
    }
}
__device__ __forceinline__ void move_values(char* page, int slot0, int D, float factor, int lane, int lanes) {
    const int whole = slot0 / kBlock * D, rest = slot0 % kBlock;                       // sixteen bytes of a d each
    move_keys(page, slot0 / kBlock * kBlock, D, factor, lane, lanes);
    for (int i = lane; i < D * rest; i += lanes) {                                   // (byte by byte: the bytes behind them are being written)
        char* p = page + (whole + i / rest) * 16 + i % rest;
        *p = (char)(moved8((uint8_t)*p, factor) & 255);
    }
}

// x, y: eight elements each of the two halves of a rotated pair of pieces
__device__ __forceinline__ void turn(float* x, float* y, const f32x4 (&co)[2], const f32x4 (&si)[2]) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float u = x[e], w = y[e], c = co[e >> 2][e & 3], s = si[e >> 2][e & 3];
        x[e] = u * c - w * s;
        y[e] = u * s + w * c;
    }
}

template <typename T, int D, bool EIGHT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void paged_append_kernel(AppendArgs a) {
    constexpr int kLanes = D / 16;                                        // lanes of a row: each has two pieces of eight elements
    constexpr int kRows = kLanes <= 4 ? 16 : 8;                           // rows that a wave reads at once
    constexpr int kTurns = kBlock / kRows;
    constexpr int kPairs = D / 2, kGroups = kPairs <= 16 ? 4 : kPairs <= 32 ? 2 : 1, kMine = kBlock / kGroups;
    constexpr int kPieces = D / 8, kRead = kPieces <= 4 ? 16 : kPieces <= 8 ? 8 : 4, kReads = kBlock / kRead;     // of a row of values; rows a read, reads a block
    __shared__ float tops[2][WAVES];
    __shared__ __attribute__((aligned(16))) T turned_values[WAVES][kBlock][D];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Fill f;
    const int unit = (int)blockIdx.x / a.parts, part = (int)blockIdx.x - unit * a.parts;
    if (!f.find(a, unit)) return;
    const int page = 1 << a.s.page_shift, s0 = f.slot0, s1 = f.slot1;
    const bool on_page = (uint32_t)f.page_no < (uint32_t)a.pages;

    // heads [head0, head1) of keys, values or queries
    const int kv_parts = (a.KV + a.heads_a_part - 1) / a.heads_a_part;
    const bool is_v = part >= kv_parts && part < 2 * kv_parts, is_q = part >= 2 * kv_parts;
    const int head0 = (part - (is_q ? 2 * kv_parts : is_v ? kv_parts : 0)) * a.heads_a_part, head1 = min(head0 + a.heads_a_part, is_q ? a.H : a.KV);
    if (!is_q && !on_page) return;
    const int64_t page_head0 = (int64_t)f.page_no * a.KV;
    const uint8_t* scales = is_v ? a.value_scales : a.key_scales;
    uint8_t* scales_out = is_v ? a.value_scales : a.key_scales;
    // the largest value of the page's new tokens: one barrier a head, on places that alternate
    auto of_page = [&](float top, int head) __attribute__((always_inline)) {
        top = wave_max(top);
        if (WAVES > 1) {
            if (lane == 0) tops[head & 1][wave] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WAVES; w++) top = fmaxf(top, tops[head & 1][w]);
        }
        return top;
    };

    if (!is_v) {
        const T* x = is_q ? static_cast<const T*>(a.q) : static_cast<const T*>(a.k);
        const int64_t xs = is_q ? a.qs[0] : a.ks[0], xh = is_q ? a.qs[1] : a.ks[1];
        // lane l of a row: pieces l and l + R / 16 of the rotated elements, which belong together, or one of each half of those behind them, so that neighbours' pieces are neighbours
        const int l = lane % kLanes, r = lane / kLanes;
        const bool turned = l < a.R / 16;
        const int d1 = turned ? 8 * l : a.R / 2 + 8 * l, d2 = d1 + (turned ? a.R : D - a.R) / 2;
        bool in[kTurns];
        f32x4 co[kTurns][2], si[kTurns][2];
        const T* rows[kTurns];
#pragma unroll
        for (int t = 0; t < kTurns; t++) {
            const int slot = wave * kBlock + t * kRows + r;
            in[t] = slot >= s0 && slot < s1 && r < kRows;
            rows[t] = x + (f.row + slot - s0) * xs;
            if (in[t] && turned) {
                const f32x4* cs = reinterpret_cast<const f32x4*>(a.freqs + (int64_t)(f.pos + slot - s0) * a.R + 8 * l);
                const f32x4* sn = reinterpret_cast<const f32x4*>(a.freqs + (int64_t)(f.pos + slot - s0) * a.R + 8 * l + a.R / 2);
                co[t][0] = cs[0]; co[t][1] = cs[1];
                si[t][0] = sn[0]; si[t][1] = sn[1];
            }
        }
        u32x4 raw[kTurns][2];
        auto ask = [&](int head) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < kTurns; t++) {
                raw[t][0] = raw[t][1] = u32x4{0, 0, 0, 0};
                if (!in[t]) continue;
                raw[t][0] = *reinterpret_cast<const u32x4*>(rows[t] + head * xh + d1);
                raw[t][1] = *reinterpret_cast<const u32x4*>(rows[t] + head * xh + d2);
            }
        };
        ask(head0);
        for (int head = head0; head < head1; head++) {
            float y[kTurns][16], top = 0.f;
            const int64_t page_head = page_head0 + head;
            const int was = EIGHT && !is_q && s0 ? scales[page_head] : 0;
#pragma unroll
            for (int t = 0; t < kTurns; t++) {
                to_floats<T>(raw[t][0], y[t]);
                to_floats<T>(raw[t][1], y[t] + 8);
            }
            if (head + 1 < head1) ask(head + 1);
#pragma unroll
            for (int t = 0; t < kTurns; t++) {
                if (turned) turn(y[t], y[t] + 8, co[t], si[t]);
                if (!in[t]) continue;
                if (EIGHT) {
#pragma unroll
                    for (int e = 0; e < 16; e++) top = finite_max(top, y[t][e]);
                }
            }
            float inv = 1.f, most = 448.f;
            if (EIGHT && !is_q) {
                const Scale sc(of_page(top, head), was, s0 > 0);
                inv = sc.inv;
                most = sc.most;
                if (sc.moves) move_keys(a.keys + page_head * page * D, s0, D, sc.factor, threadIdx.x, 64 * WAVES);
                if (threadIdx.x == 0) scales_out[page_head] = (uint8_t)sc.byte;
            }
#pragma unroll
            for (int t = 0; t < kTurns; t++) {
                if (!in[t]) continue;
                const int slot = wave * kBlock + t * kRows + r;
                if (is_q || !EIGHT) {
                    T* out = is_q ? static_cast<T*>(a.q_out) + (f.row + slot - s0) * a.os[0] + head * a.os[1] : reinterpret_cast<T*>(a.keys) + (page_head * page + slot) * D;
                    put_stream<u32x4>(out + d1, to_vector<T>(y[t]));
                    put_stream<u32x4>(out + d2, to_vector<T>(y[t] + 8));
                } else {
                    char* out = a.keys + (page_head * page + slot) * D;
                    put_stream<u32x2>(out + d1, u32x2{pack8(y[t], inv, most), pack8(y[t] + 4, inv, most)});
                    put_stream<u32x2>(out + d2, u32x2{pack8(y[t] + 8, inv, most), pack8(y[t] + 12, inv, most)});
                }
            }
        }
        return;
    }

    // ---- values: a lane reads a piece of a row, and writes (in 8 bits) two neighbouring d of kMine tokens, which lie side by side in the block
    const int pr = lane / kPieces, pc = lane % kPieces, pair = lane % kPairs, group = lane / kPairs;
    u32x4 raw[kReads];
    auto ask = [&](int head) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kReads; i++) {
            const int slot = wave * kBlock + i * kRead + pr;
            raw[i] = u32x4{0, 0, 0, 0};
            if (pr < kRead && slot >= s0 && slot < s1) raw[i] = *reinterpret_cast<const u32x4*>(static_cast<const T*>(a.v) + (f.row + slot - s0) * a.vs[0] + head * a.vs[1] + 8 * pc);
        }
    };
    ask(head0);
    const int slot = wave * kBlock + group * kMine;
    const bool mine = group < kGroups && slot + kMine > s0 && slot < s1, all = slot >= s0 && slot + kMine <= s1;
    for (int head = head0; head < head1; head++) {
        const int64_t page_head = page_head0 + head;
        const int was = EIGHT && s0 ? scales[page_head] : 0;
        wave_in_order();                                                  // (the head before has been read)
#pragma unroll
        for (int i = 0; i < kReads; i++)
            if (pr < kRead) *reinterpret_cast<u32x4*>(&turned_values[wave][i * kRead + pr][8 * pc]) = raw[i];
        wave_in_order();
        if (head + 1 < head1) ask(head + 1);
        if constexpr (!EIGHT) {
            // in 16 bits a lane writes eight tokens of one d, its neighbour the other eight: a store of the wave is a kilobyte in one piece
            // (us, two d of sixteen tokens a lane | so: 6300 tokens of 16 heads of 96 24.2 | 19.0, of 128 27.4 | 21.2, 8192 of 12 heads of 64 15.9 | 11.2, past the caches level)
            typedef T eight __attribute__((ext_vector_type(8)));
#pragma unroll
            for (int i = 0; i < (D + 31) / 32; i++) {
                const int d = 32 * i + lane / 2, t0 = 8 * (lane & 1), at = wave * kBlock + t0;
                eight w;
#pragma unroll
                for (int t = 0; t < 8; t++) w[t] = turned_values[wave][t0 + t][d];
                if (at + 8 <= s0 || at >= s1) continue;
                T* out = reinterpret_cast<T*>(a.values) + ((page_head * (page / kBlock) + wave) * D + d) * kBlock + t0;
                if (at >= s0 && at + 8 <= s1) {
                    *reinterpret_cast<eight*>(out) = w;
                } else {
#pragma unroll
                    for (int t = 0; t < 8; t++)
                        if (at + t >= s0 && at + t < s1) out[t] = w[t];
                }
            }
            continue;
        }
        float y[2][kMine], top = 0.f;
#pragma unroll
        for (int t = 0; t < kMine; t++) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(&turned_values[wave][(group % kGroups) * kMine + t][2 * pair]);
            y[0][t] = Elem<T>::to_f32(__builtin_bit_cast(T, (uint16_t)w));
            y[1][t] = Elem<T>::to_f32(__builtin_bit_cast(T, (uint16_t)(w >> 16)));
            top = finite_max(finite_max(top, y[0][t]), y[1][t]);
        }
        const Scale sc(of_page(top, head), was, s0 > 0);
        const float inv = sc.inv, most = sc.most;
        if (sc.moves) move_values(a.values + page_head * page * D, s0, D, sc.factor, threadIdx.x, 64 * WAVES);
        if (threadIdx.x == 0) scales_out[page_head] = (uint8_t)sc.byte;
        if (!mine) continue;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int64_t at16 = ((page_head * (page / kBlock) + wave) * D + 2 * pair + j) * kBlock + group * kMine;
            if (all) {
                uint32_t w[kMine / 4];
#pragma unroll
                for (int e = 0; e < kMine / 4; e++) w[e] = pack8(y[j] + 4 * e, inv, most);
                __builtin_memcpy(__builtin_assume_aligned(a.values + at16, kMine), w, kMine);
            } else {
#pragma unroll
                for (int t = 0; t < kMine; t++) {
                    if (slot + t < s0 || slot + t >= s1) continue;
                    const float four[4] = {y[j][t], 0.f, 0.f, 0.f};
                    a.values[at16 + t] = (char)(pack8(four, inv, most) & 255);
                }
            }
        }
    }
}

// A row of a token for D / 16 lanes: all new tokens of one page and one head of keys, values or queries, one after the other.  The first token's row stays in registers between the
// search for the page's largest value and the store; further ones are read again.
template <typename T, int D, bool EIGHT>
__global__ __launch_bounds__(256) void append_few_kernel(AppendArgs a) {
    constexpr int kLanes = D / 16, kItems = 64 / kLanes;                  // lanes of an item, items of a wave
    const int lane = threadIdx.x & 63, l = lane % kLanes;
    Fill f;
    if (!f.find(a, blockIdx.x)) return;
    const int item = ((int)blockIdx.y * 4 + (threadIdx.x >> 6)) * kItems + lane / kLanes;
    const bool is_q = item >= 2 * a.KV, is_v = !is_q && item >= a.KV;
    const int head = is_q ? item - 2 * a.KV : is_v ? item - a.KV : item;
    if (lane >= kItems * kLanes || (is_q ? head >= a.H : (uint32_t)f.page_no >= (uint32_t)a.pages)) return;
    const int page = 1 << a.s.page_shift;
    const int64_t page_head = (int64_t)f.page_no * a.KV + head;
    uint8_t* scales = is_v ? a.value_scales : a.key_scales;
    const int was = EIGHT && !is_q && f.slot0 ? scales[page_head] : 0;

    const bool turned = !is_v && l < a.R / 16;
    const int d1 = is_v ? 16 * l : turned ? 8 * l : a.R / 2 + 8 * l, d2 = d1 + (is_v ? 8 : (turned ? a.R : D - a.R) / 2);
    const T* x = is_q ? static_cast<const T*>(a.q) + head * a.qs[1] : is_v ? static_cast<const T*>(a.v) + head * a.vs[1] : static_cast<const T*>(a.k) + head * a.ks[1];
    const int64_t xs = is_q ? a.qs[0] : is_v ? a.vs[0] : a.ks[0];
    auto row_of = [&](int i, float (&y)[16]) __attribute__((always_inline)) {
        const T* row = x + (f.row + i) * xs;
        const u32x4 w1 = *reinterpret_cast<const u32x4*>(row + d1), w2 = *reinterpret_cast<const u32x4*>(row + d2);
        f32x4 co[2], si[2];
        if (turned) {
            const f32x4* cs = reinterpret_cast<const f32x4*>(a.freqs + (int64_t)(f.pos + i) * a.R + 8 * l);
            const f32x4* sn = reinterpret_cast<const f32x4*>(a.freqs + (int64_t)(f.pos + i) * a.R + 8 * l + a.R / 2);
            co[0] = cs[0]; co[1] = cs[1];
            si[0] = sn[0]; si[1] = sn[1];
        }
        to_floats<T>(w1, y);
        to_floats<T>(w2, y + 8);
        if (turned) turn(y, y + 8, co, si);
    };
    const int n = f.slot1 - f.slot0;
    float y0[16], inv = 1.f, most = 448.f;
    row_of(0, y0);
    if (EIGHT && !is_q) {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 16; e++) top = finite_max(top, y0[e]);
        for (int i = 1; i < n; i++) {
            float y[16];
            row_of(i, y);
#pragma unroll
            for (int e = 0; e < 16; e++) top = finite_max(top, y[e]);
        }
        if constexpr (kLanes == 6) {
            const int base = lane - l;
            float most = 0.f;
#pragma unroll
            for (int j = 0; j < kLanes; j++) most = fmaxf(most, __shfl(top, base + j, 64));
            top = most;
        } else {
#pragma unroll
            for (int j = 1; j < kLanes; j *= 2) top = fmaxf(top, __shfl_xor(top, j, 64));
        }
        const Scale sc(top, was, f.slot0 > 0);
        inv = sc.inv;
        most = sc.most;
        if (sc.moves) {
            if (is_v) move_values(a.values + page_head * page * D, f.slot0, D, sc.factor, l, kLanes);
            else move_keys(a.keys + page_head * page * D, f.slot0, D, sc.factor, l, kLanes);
        }
        if (l == 0) scales[page_head] = (uint8_t)sc.byte;
    }
    for (int i = 0; i < n; i++) {
        float y[16];
        if (i == 0) {
#pragma unroll
            for (int e = 0; e < 16; e++) y[e] = y0[e];
        } else {
            row_of(i, y);
        }
        const int slot = f.slot0 + i;
        if (is_v) {
            const int64_t at16 = ((page_head * (page / kBlock) + slot / kBlock) * D + d1) * kBlock + slot % kBlock;
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                if constexpr (EIGHT) {
                    const uint32_t w = pack8(y + e, inv, most);
#pragma unroll
                    for (int j = 0; j < 4; j++) a.values[at16 + (e + j) * kBlock] = (char)(w >> 8 * j);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) reinterpret_cast<T*>(a.values)[at16 + (e + j) * kBlock] = Elem<T>::from_f32(y[e + j]);
                }
            }
        } else if (is_q || !EIGHT) {
            T* out = is_q ? static_cast<T*>(a.q_out) + (f.row + i) * a.os[0] + head * a.os[1] : reinterpret_cast<T*>(a.keys) + (page_head * page + slot) * D;
            *reinterpret_cast<u32x4*>(out + d1) = to_vector<T>(y);
            *reinterpret_cast<u32x4*>(out + d2) = to_vector<T>(y + 8);
        } else {
            char* out = a.keys + (page_head * page + slot) * D;
            *reinterpret_cast<u32x2*>(out + d1) = u32x2{pack8(y, inv, most), pack8(y + 4, inv, most)};
            *reinterpret_cast<u32x2*>(out + d2) = u32x2{pack8(y + 8, inv, most), pack8(y + 12, inv, most)};
        }
    }
}

template <typename T, int D, bool EIGHT>
int launch(hipStream_t st, AppendArgs a, int64_t units) {
    if (a.s.T <= a.s.B) {
        const int items = 4 * (64 / (D / 16));
        hipLaunchKernelGGL((append_few_kernel<T, D, EIGHT>), dim3((unsigned)units, (unsigned)((2 * a.KV + a.H + items - 1) / items)), dim3(256), 0, st, a);
        return check_launch("paged_append");
    }
    auto parts = [&](int heads) { return 2 * ((a.KV + heads - 1) / heads) + (a.H + heads - 1) / heads; };
    // Heads of a workgroup: what they share (the page's place, cosines and sines) against waves to fill the device with.  us, one | two | four | eight heads, buffers larger than the caches: 9450 tokens of
    // 32 and 8 heads of 128 51.7 | 46.6 | 48.7 | 55.7 (14700, 7300 waves with two, four), 32000 162 | 140 | 140 | 142, of 32 and 32 heads 320 | 257 | 248 | 255, 6300 of 16 and 16 of 96
    // 21.2 | 20.5 | 21.6 | 22.4 (9800, 4900 waves), 300 tokens 6.0 | 6.2 | 9.1 | 15.0
    a.heads_a_part = 4;
    while (a.heads_a_part > 1 && units * (1 << (a.s.page_shift - 4)) * parts(a.heads_a_part) < 8000) a.heads_a_part /= 2;
    // All heads of a page run side by side, and a token's row is read and written in one go: page after page of one part of the heads first was 52.4 and 159 us where 9450 and 32000 take 48.7 and 142
    a.parts = parts(a.heads_a_part);
    if (units * a.parts >= (int64_t)1 << (26 - (a.s.page_shift - 4))) return fail(MHIP_ERR_UNSUPPORTED, "paged_append: more threads than a launch has");       // (2^32 of them)
    const dim3 grid((unsigned)(units * a.parts));
    switch (a.s.page_shift) {
        case 4: hipLaunchKernelGGL((paged_append_kernel<T, D, EIGHT, 1>), grid, dim3(64), 0, st, a); break;
        case 5: hipLaunchKernelGGL((paged_append_kernel<T, D, EIGHT, 2>), grid, dim3(128), 0, st, a); break;
        case 6: hipLaunchKernelGGL((paged_append_kernel<T, D, EIGHT, 4>), grid, dim3(256), 0, st, a); break;
        case 7: hipLaunchKernelGGL((paged_append_kernel<T, D, EIGHT, 8>), grid, dim3(512), 0, st, a); break;
        default: hipLaunchKernelGGL((paged_append_kernel<T, D, EIGHT, 16>), grid, dim3(1024), 0, st, a); break;
    }
    return check_launch("paged_append");
}

template <typename T, bool EIGHT>
int launch_d(hipStream_t st, const AppendArgs& a, int64_t D, int64_t units) {
    switch (D) {
        case 32: return launch<T, 32, EIGHT>(st, a, units);
        case 64: return launch<T, 64, EIGHT>(st, a, units);
        case 96: return launch<T, 96, EIGHT>(st, a, units);
        default: return launch<T, 128, EIGHT>(st, a, units);
    }
}

}  // namespace

int check_sizes(const char* what, const mhip_paged_cache* c, const mhip_sequences* s) {
    if (!c || !s) return fail(MHIP_ERR_INVALID_ARGUMENT, "%s: NULL cache or sequences", what);
    if (c->pages <= 0 || c->heads <= 0 || s->sequences < 0 || s->width < 0 || s->tokens < 0) return fail(MHIP_ERR_INVALID_ARGUMENT, "%s: a size is negative, or the cache has no pages or heads", what);
    if (c->head_size < 32 || c->head_size > 128 || c->head_size % 32) return fail(MHIP_ERR_UNSUPPORTED, "%s: head size %lld (need 32, 64, 96 or 128)", what, (long long)c->head_size);
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
        return fail(MHIP_ERR_UNSUPPORTED, "%s: page size %lld (need a power of two from 16 to 256)", what, (long long)c->page_size);
    // (every size by itself in front of a product with it)
    if (c->pages > INT32_MAX || c->heads > 1024 || c->pages * c->heads > INT32_MAX || s->sequences > 65536 || s->tokens > (1 << 24) || s->width > (1 << 20) || s->width * c->page_size > (1 << 24))
        return fail(MHIP_ERR_UNSUPPORTED, "%s: more than 65536 sequences, 2^24 tokens, 2^24 keys a sequence, 1024 heads or 2^31 pages times heads", what);
    return MHIP_OK;
}

int check_paged(const char* what, const mhip_paged_cache* c, const mhip_sequences* s, int dtype, bool* empty) {
    *empty = false;
    if (const int rc = check_sizes(what, c, s)) return rc;
    if (dtype != MHIP_BF16 && dtype != MHIP_F16) return fail(MHIP_ERR_UNSUPPORTED, "%s: dtype %d (need bf16 or f16)", what, dtype);
    if (!c->key_scales != !c->value_scales) return fail(MHIP_ERR_INVALID_ARGUMENT, "%s: scales of keys without scales of values", what);
    if (s->sequences == 0 || s->tokens == 0) { *empty = true; return MHIP_OK; }
    if (!s->starts || !s->lengths || (s->width && !s->table)) return fail(MHIP_ERR_INVALID_ARGUMENT, "%s: NULL table, lengths or starts", what);
    if (!c->keys || !c->values) return fail(MHIP_ERR_INVALID_ARGUMENT, "%s: NULL cache", what);
    if (((uintptr_t)c->keys | (uintptr_t)c->values) & 15) return fail(MHIP_ERR_UNSUPPORTED, "%s: the cache must be 16-byte aligned", what);
    return MHIP_OK;
}

}  // namespace mhip

using namespace mhip;

extern "C" int mhip_paged_append(void* stream, const mhip_paged_cache* cache, const mhip_sequences* seqs, const void* k, const void* v, const void* q, void* q_out,
                                 int64_t q_heads, const float* freqs, int64_t positions, int64_t rotated, const int64_t* strides, int dtype) {
    bool empty;
    if (const int rc = check_paged("paged_append", cache, seqs, dtype, &empty)) return rc;
    const int64_t D = cache->head_size;
    if (rotated < 0 || rotated > D || rotated % 16) return fail(MHIP_ERR_UNSUPPORTED, "paged_append: %lld rotated elements of %lld (need a multiple of 16)", (long long)rotated, (long long)D);
    if (positions < 0 || positions > INT32_MAX) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_append: %lld positions", (long long)positions);
    if (rotated && !freqs) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_append: NULL freqs");
    if (q && (!q_out || q_heads <= 0)) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_append: queries without a result or heads");
    if (q && q_heads > 32768) return fail(MHIP_ERR_UNSUPPORTED, "paged_append: %lld query heads", (long long)q_heads);
    if (empty) return MHIP_OK;
    if (!k || !v || !strides) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_append: NULL tensor");
    if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (uintptr_t)(q ? q_out : nullptr) | (uintptr_t)(rotated ? freqs : nullptr)) & 15)
        return fail(MHIP_ERR_UNSUPPORTED, "paged_append: tensors must be 16-byte aligned");
    for (int i = 0; i < (q ? 8 : 4); i++)
        if (strides[i] % 8) return fail(MHIP_ERR_UNSUPPORTED, "paged_append: strides must be multiples of 8 elements");
    AppendArgs a{k, v, q, q_out, freqs, (char*)cache->keys, (char*)cache->values, cache->key_scales, cache->value_scales, sequences(cache, seqs),
                 (int)cache->pages, (int)cache->heads, (int)(q ? q_heads : 0), (int)rotated, (int)positions, 1, {}, {}, {}, {}};
    for (int i = 0; i < 2; i++) {
        a.ks[i] = strides[i];
        a.vs[i] = strides[2 + i];
        if (q) { a.qs[i] = strides[4 + i]; a.os[i] = strides[6 + i]; }
    }
    // pages that n tokens can reach: n / page and one more, and one more for where they begin
    const int64_t units = seqs->tokens / cache->page_size + 2 * (seqs->sequences < seqs->tokens ? seqs->sequences : seqs->tokens);
    const bool eight = cache->key_scales != nullptr;
    hipStream_t st = as_stream(stream);
    if (dtype == MHIP_BF16) return eight ? launch_d<bf16_t, true>(st, a, D, units) : launch_d<bf16_t, false>(st, a, D, units);
    return eight ? launch_d<f16_t, true>(st, a, D, units) : launch_d<f16_t, false>(st, a, D, units);
}
