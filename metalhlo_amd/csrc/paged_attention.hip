// Attention over a paged cache (paged.h): O = softmax(scale Q K^T) V, rows of queries from one token of a sequence to a whole prompt behind a long context.
//
//   rows   of a sequence and a key/value head: its tokens times the G = H / KV query heads that share the head, row = token * G + query head, so that K and V are read
//          once for all of them.  A token's position is lengths[b] - tokens(b) + i; with the causal rule it sees the keys up to its own.
//   line   All the work of a launch in one line, sequence by sequence, head by head and tile by tile, each as long as its keys: workgroup w takes the w-th of equal shares.  The lengths are not known
//          on the host, and a batch may hold one long sequence among short ones: the line is measured on the device, by every workgroup for itself.  (Parts of one length for the whole launch
//          instead: 48 sequences of 1600 to 8000 keys 117 us | 96.)  A part of a tile leaves its reference maximum, its sum and its unnormalised rows in the workspace, and the last one
//          to arrive puts them together in order (arrive.h): results do not depend on who that is.  Without a workspace a workgroup takes whole tiles.
//
// Two kernels.  Up to 32 rows a sequence on average (decode steps): paged_rows_kernel, whose waves have keys of their own and load them straight into matrix operands;
// its time is that of reading K and V: 64 sequences of 4096 keys, 8 heads of 128 in 8 bits (537 MB), 88 us, 6.1 TB/s; 48 of 1600 to 8000 keys (477 MB) 90 us; one token over some hundred keys 8 us, which is latency.
// More rows: paged_tile_kernel, 128 rows whose four waves share K and V in LDS, in the queries' type; its time is the matrix products' and the exponentials' between them:
// 32 over 8 heads of 128, four pieces of 1024 tokens behind 7168 600 us, 860 TFLOP/s (16-bit pages 613).
//
// fp32 sums, softmax state and scores (a key's scale is applied to its score in the first kernel, while it is converted in the second where the type holds that); probabilities are rounded to the queries' type in front of the second product,
// whose error of half a step each (2^-9 for bf16) is, averaged over keys whose values are independent, nine tenths of the result's own rounding (both together 2.3e-3 of the result's norm, that alone 1.7e-3).  Values in 8 bits become the queries' type exactly,
// scale and all, except that f16 ends at 65504 and at 2^-24.
#include <algorithm>
#include <cmath>

#include "arrive.h"
#include "attention_common.h"
#include "paged.h"

namespace mhip {
namespace {

// Division of numbers below 2^30 by one that the host knows: n / d = umulhi(n, m) >> s with m = ceil(2^(32 + s) / d), 2^(s + 2) > d.
struct Divider {
    uint32_t m;
    int s;
    explicit Divider(uint32_t d) : s(0) {
        while ((4u << s) <= d) s++;
        m = (uint32_t)((((uint64_t)1 << (32 + s)) + d - 1) / d);
        if (d == 1) m = 0;                                                 // (2^32)
    }
    __device__ __forceinline__ int operator()(int n) const { return m ? (int)(__umulhi((uint32_t)n, m) >> s) : n; }
};

struct PagedArgs {
    const void* q;
    void* o;
    const char *keys, *values;
    const uint8_t *key_scales, *value_scales;
    Sequences s;
    int pages, KV, G, is_causal, shares, units;
    float c;                                  // |scale| * log2(e), a tiny number instead of 0 (which times -inf is none)
    uint32_t sign;                            // 0x80008000 where the scale is negative: of the queries
    int64_t qs[2], os[2];                     // token and head strides in elements
    float* part;                              // workspace, NULL: keys are not dealt
    uint64_t* words;
    uint64_t tag;
    Divider by_group, by_heads, by_shares;    // G, KV, shares
    int unit_shift;                           // log2 of the keys that one unit of the line stands for
};

constexpr int kMostParts = 64;

// The work of a launch is one line: sequence by sequence, each head's and tile's own stretch as long as the work it stands for, and workgroup w takes the w-th share, which may be a part of one
// tile's keys, or the end of one, several whole ones and the beginning of another.  Every workgroup has the same to do whatever the lengths, and leaves two parts at most.
// The first `more` shares are per + 1 long, the others per.
struct Line {
    int per, more;
    // `all`: the line's length; `longest`: a tile's stretch (one that were dealt over more than kMostParts workgroups would keep the last of them too long)
    __device__ __forceinline__ Line(const Divider& by_shares, int shares, int all, int longest) {
        per = by_shares(all);
        more = all - per * shares;
        if (per < 1 || longest > (kMostParts - 1) * per) {
            per = (longest + kMostParts - 2) / (kMostParts - 1);
            more = 0;
        }
    }
    __device__ __forceinline__ int begin(int w) const { return w * per + min(w, more); }
    __device__ __forceinline__ int owner(int g) const { return g < more * (per + 1) ? g / (per + 1) : more + (g - more * (per + 1)) / per; }
};

// The first 64 sequences, in a wave's own LDS.  `keys`: the position behind its last token, which is more than it has keys where it has outgrown its table; `line`: the keys that its tiles' stretches of the
// line are made for.
struct Known { int start[64], tokens[64], keys[64], line[64]; };
struct Found { int b, before, start, tokens, keys, line; };
__device__ __forceinline__ void known_of(const Sequences& s, Known& known, int lane) {
    known.start[lane] = lane < s.B ? s.start(lane) : 0;
    known.tokens[lane] = lane < s.B ? s.tokens(lane) : 0;
    known.keys[lane] = lane < s.B ? s.bounded_end(lane) : 0;
    known.line[lane] = lane < s.B ? s.keys(lane) : 0;
}
// The sequence that place g of the line lies in, when one has stretch(tokens, keys) of it; `before`: where it begins.  False behind the last.
template <typename F>
__device__ __forceinline__ bool found_at(const Sequences& s, const Known& known, int lane, int g, F stretch, Found& at) {
    const int mine = stretch(known.tokens[lane], known.line[lane]), sum = wave_scan(mine);
    int length;
    if (const uint64_t m = __ballot(sum > g)) {
        at.b = __builtin_ctzll(m);
        at.before = __builtin_amdgcn_readlane(sum - mine, at.b);
        length = __builtin_amdgcn_readlane(mine, at.b);
        at.start = __builtin_amdgcn_readfirstlane(known.start[at.b]);
        at.tokens = __builtin_amdgcn_readfirstlane(known.tokens[at.b]);
        at.keys = __builtin_amdgcn_readfirstlane(known.keys[at.b]);
        at.line = __builtin_amdgcn_readfirstlane(known.line[at.b]);
    } else {
        at.before = __builtin_amdgcn_readlane(sum, 63);
        int further;
        at.b = 64 + sequence_of(s.B - 64, g - at.before, [&](int i) { return stretch(s.tokens(64 + i), s.keys(64 + i)); }, further);
        if (at.b < 64) return false;
        at.before += further;
        at.start = __builtin_amdgcn_readfirstlane(s.start(at.b));
        at.tokens = __builtin_amdgcn_readfirstlane(s.tokens(at.b));
        at.keys = __builtin_amdgcn_readfirstlane(s.bounded_end(at.b));
        at.line = __builtin_amdgcn_readfirstlane(s.keys(at.b));
        length = stretch(at.tokens, at.line);
    }
    return g >= at.before && g - at.before < length;                       // (starts that are no starts: their sums may have wrapped)
}

// The parts of a tile that is split: in workgroups `first` to first + parts - 1, the first one's at slot 2 first + 1 (the end of its share), the others' at 2 w (the beginning).
struct Split { int first, parts; };
__device__ __forceinline__ Split split_of(const Line& line, int shares, int share, int origin, int length) {
    const int first = min(max(line.owner(origin), 0), share);
    return {first, min(line.owner(origin + length - 1) - first + 1, min(kMostParts, shares - first))};
}

// Words at an address that is the same in all lanes, and that no launch writes while another reads them: read by scalar loads.
typedef const __attribute__((address_space(4))) int32_t* uniform_words;

// The page that holds key 16 `block` of sequence b, clamped to one that exists; `ok`: whether the table names it.
__device__ __forceinline__ int page_of(const PagedArgs& a, const int32_t* table, int block, bool& ok) {
    const int at = block >> (a.s.page_shift - 4);
    ok = at < a.s.width;
    const int page = ok ? table[at] : 0;
    ok = ok && (uint32_t)page < (uint32_t)a.pages;
    return ok ? page : 0;
}

// sixteen bits of eight e4m3, times 2^e of `scale`
template <typename T>
__device__ __forceinline__ u32x4 widen(u32x2 w, float scale) {
    u32x4 r;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if constexpr (std::is_same<T, bf16_t>::value) {
            const auto two = (e & 1) ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[e >> 1], scale, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[e >> 1], scale, false);
            r[e] = __builtin_bit_cast(uint32_t, two);
        } else {
            const auto two = (e & 1) ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[e >> 1], scale, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[e >> 1], scale, false);
            r[e] = __builtin_bit_cast(uint32_t, two);
        }
    }
    return r;
}

// A finite value under its scale may be more than f16 holds, which ends at 65504 then: an infinity times the weight zero of a key that a row does not see were a NaN of that row's.  (A NaN stays one.)
// The greatest e4m3 is 448, so that no scale up to 2^7 needs it: the tile kernel, which is short of vector instructions, asks (us, four f16 pieces of 1024 tokens behind 7168 over 8-bit pages, not at all |
// always 600 | 614, not at all | asked 615 | 622); the rows kernel, whose registers have no room for another way through its loop, does it always (64 sequences of 4096 keys 88.1 | 88.8).
__device__ __forceinline__ u32x4 ended(u32x4 w) {
    typedef _Float16 two __attribute__((ext_vector_type(2)));
    const two most = {(_Float16)65504.f, (_Float16)65504.f};
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = __builtin_bit_cast(uint32_t, __builtin_elementwise_maximum(__builtin_elementwise_minimum(__builtin_bit_cast(two, (uint32_t)w[e]), most), -most));
    return w;
}

// A key's value that is not finite makes the results of the rows that see it so, and of no others, but zero times it is no zero: where a result is not finite, the keys are
// gone through once more with such values left out of the second product where some rows see them and others do not, and they are added to the rows behind it, one by one.
template <typename T, bool EIGHT>
__device__ __forceinline__ uint32_t tamed(uint32_t w, bool& any) {
    uint32_t wild;                                                         // the top bit of each that is not finite
    if constexpr (EIGHT) wild = ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
    else if constexpr (std::is_same<T, bf16_t>::value) wild = ((w & 0x7FFF7FFFu) + 0x00800080u) & 0x80008000u;
    else wild = ((w & 0x7FFF7FFFu) + 0x04000400u) & 0x80008000u;
    any |= wild != 0;
    return w & ~(EIGHT ? (wild >> 7) * 0xFFu : (wild >> 15) * 0xFFFFu);
}
// what a value adds to a result besides
template <typename T, bool EIGHT>
__device__ __forceinline__ float wild_of(const char* p) {
    if constexpr (EIGHT) return (*reinterpret_cast<const uint8_t*>(p) & 0x7F) == 0x7F ? __builtin_nanf("") : 0.f;
    const float x = Elem<T>::to_f32(*reinterpret_cast<const T*>(p));
    return fabsf(x) < INFINITY ? 0.f : x;
}
// where key `key` of head `head` has its d = 0 in the values, NULL where the table names no page; from one d to the next it is sixteen values
template <int D, int SIZE>
__device__ __forceinline__ const char* value_at(const PagedArgs& a, const int32_t* table, int head, int key) {
    bool ok;
    const int page = page_of(a, table, key >> 4, ok), blocks = a.s.page_shift - 4;
    return ok ? a.values + (((((int64_t)page * a.KV + head) << blocks) + ((key >> 4) & ((1 << blocks) - 1))) * (16 * D) + (key & 15)) * SIZE : nullptr;
}

// x and the two numbers of w: a row's sum is that of the rounded weights, which are the ones that its values are multiplied with.  (With the weights' own sum a mean of values that are all f16's greatest number
// is an infinity where the rounding went up.)
template <typename T>
__device__ __forceinline__ float plus_two(uint32_t w, float x) {
    typedef T two __attribute__((ext_vector_type(2)));
    const two one = {(T)1.f, (T)1.f};
    if constexpr (std::is_same<T, bf16_t>::value) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(two, w), one, x, false);
    else return __builtin_amdgcn_fdot2(__builtin_bit_cast(two, w), one, x, false);
}

template <typename T> struct Mfma16P;
template <> struct Mfma16P<bf16_t> {
    __device__ static f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mfma16P<f16_t> {
    __device__ static f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// Parts of a tile of ROWS rows: [slot][ROWS][D] sums, then [slot][ROWS] pairs of reference maximum and sum; two slots a workgroup.
template <int ROWS, int D>
struct Parts {
    float *sums, *state;
    __device__ __forceinline__ Parts(const PagedArgs& a, int slot) : sums(a.part + (int64_t)slot * ROWS * D), state(a.part + 2 * (int64_t)a.shares * ROWS * D + (int64_t)slot * ROWS * 2) {}
};

__device__ __forceinline__ void store_two(float* p, float x, float y) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), (uint64_t)__builtin_bit_cast(uint32_t, x) | (uint64_t)__builtin_bit_cast(uint32_t, y) << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ u32x2 load_two(const float* p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return u32x2{(uint32_t)v, (uint32_t)(v >> 32)};
}

// By the last workgroup of a tile: its parts put together in order.  `rows`: of the tile, from row `row0` of the sequence that starts at token `start`.
// The sums of a tile of few rows lie row by row, those of many as the lanes of their waves hold them (the stores pass the L2: sixteen bytes of each of 64 rows at a time went to memory as such).
template <typename T, int ROWS, int D, int THREADS>
__device__ __forceinline__ void join(const PagedArgs& a, const Split& split, int start, int head, int row0, int rows) {
    constexpr int kFours = D / 4, kAll = (ROWS * kFours + THREADS - 1) / THREADS;             // fours of numbers of a row; a thread's of a full tile
    constexpr bool kByLanes = ROWS > 32;
    const int all = kByLanes ? (rows + 31) / 32 * 32 * kFours : rows * kFours;
    auto row_of = [](int idx) { return kByLanes ? idx / (64 * (D / 8)) * 32 + (idx & 31) : idx / kFours; };
    auto four_of = [](int idx) { return kByLanes ? (idx >> 6) % (D / 8) * 2 + (idx >> 5 & 1) : idx % kFours; };
    // AHEAD parts of ITEMS fours are asked for at once, sixteen loads that arrive after one latency: with one four at a time the sixteen of a tile of 128 rows took 40 us
    auto put = [&](auto ahead, auto items) __attribute__((always_inline)) {
        constexpr int AHEAD = decltype(ahead)::value, ITEMS = decltype(items)::value < kAll ? decltype(items)::value : kAll;
        for (int idx0 = threadIdx.x; idx0 < all; idx0 += ITEMS * THREADS) {
            float m[ITEMS], l[ITEMS];
            f32x4 o[ITEMS];
#pragma unroll
            for (int i = 0; i < ITEMS; i++) {
                m[i] = -INFINITY;
                l[i] = 0.f;
                o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            for (int p0 = 0; p0 < split.parts; p0 += AHEAD) {
                u32x2 st[ITEMS][AHEAD];
                f32x4 v[ITEMS][AHEAD];
#pragma unroll
                for (int p = 0; p < AHEAD; p++) {
                    const int q = min(p0 + p, split.parts - 1);
                    const Parts<ROWS, D> at(a, 2 * (split.first + q) + (q ? 0 : 1));
#pragma unroll
                    for (int i = 0; i < ITEMS; i++) {
                        const int idx = min(idx0 + i * THREADS, all - 1);
                        st[i][p] = load_two(at.state + 2 * row_of(idx));
                        v[i][p] = load_part(parts_rsrc(at.sums), (uint32_t)(idx * 16));
                    }
                }
#pragma unroll
                for (int i = 0; i < ITEMS; i++) {
                    float top = m[i];
#pragma unroll
                    for (int p = 0; p < AHEAD; p++) top = fmaxf(top, p0 + p < split.parts ? __builtin_bit_cast(float, (uint32_t)st[i][p].x) : -INFINITY);
                    const float use = top == -INFINITY ? 0.f : top, old = weight(m[i], use);
                    m[i] = top;
                    l[i] *= old;
                    o[i] *= old;
#pragma unroll
                    for (int p = 0; p < AHEAD; p++) {
                        const float al = p0 + p < split.parts ? weight(__builtin_bit_cast(float, (uint32_t)st[i][p].x), use) : 0.f;
                        l[i] = fmaf(__builtin_bit_cast(float, (uint32_t)st[i][p].y), al, l[i]);
#pragma unroll
                        for (int e = 0; e < 4; e++) o[i][e] = fmaf(v[i][p][e], al, o[i][e]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < ITEMS; i++) {
                const int idx = idx0 + i * THREADS;
                if (idx >= all || row_of(idx) >= rows) continue;
                const float inv = l[i] != 0.f ? 1.f / l[i] : 0.f;
                const int r = row0 + row_of(idx), token = a.by_group(r);
                T* out = static_cast<T*>(a.o) + (int64_t)(start + token) * a.os[0] + (int64_t)(head * a.G + r - token * a.G) * a.os[1] + 4 * four_of(idx);
                *reinterpret_cast<u32x2*>(out) = u32x2{Mfma32A<T>::pack2(o[i][0] * inv, o[i][1] * inv), Mfma32A<T>::pack2(o[i][2] * inv, o[i][3] * inv)};
            }
        }
    };
    using std::integral_constant;
    if (ROWS > 32 && split.parts <= 2) put(integral_constant<int, 2>{}, integral_constant<int, 8>{});
    else if (split.parts <= 4) put(integral_constant<int, 4>{}, integral_constant<int, 4>{});
    else if (split.parts <= 8 || ROWS > 32) put(integral_constant<int, 8>{}, integral_constant<int, 2>{});
    else put(integral_constant<int, 16>{}, integral_constant<int, 1>{});
}

// ---------------------------------------------------------------- few rows
// A wave takes blocks of 4 kLane keys of its own, kLane = 16 neighbouring ones (8 of a 16-bit cache) to each quarter of its lanes:
//   S^T = K Q^T    v_mfma_f32_16x16x32, kLane / 4 tiles j of sixteen keys: operand row i is key kLane (i / 4) + 4 j + i % 4, so that a lane of the result holds keys 4 j + r of its
//                  quarter's kLane, r = 0 .. 3.  Which of the elements of D a step takes from a lane does not matter as long as it takes the same from K and Q: a
//                  lane loads sixteen bytes of a key at a time, two steps' worth in 8 bits.
//   O^T += V^T P^T operand row = d; the eight keys that a lane holds of it in a step are neighbours in the cache's block, so that one load of sixteen bytes feeds two steps (one of a 16-bit cache), and
//                  they are those whose probabilities the lane has just computed.
// Two blocks are in registers or on their way; K of the next but one is asked for behind this one's scores, V behind its second product.  The loads of K and V pass the caches, which no one else
// would find them in (us, plain | so: 64 sequences of 4096 keys 97.8 | 88.2), and the page numbers and scales come by scalar loads, which the vector loads do not queue behind.  The kernel holds what the registers
// do: a spill of a few words costs a launch 10 us whatever its size, since scratch memory is set up for it.
//
// SINGLE: no sequence has more tokens than its place among as many others suggests, one, and a tile is one token's G rows, which see the same keys; else the rows of a tile may see
// different numbers of them.
//
// The line is in steps of 256 keys (more where there were over 2^29 of them), tile by tile and head by head.
constexpr int kStepShift = 8;

// Workgroups of a unit: what the registers allow, and what the launch counts on.
constexpr int rows_kernel_workgroups(int tiles, int64_t D, bool single) { return tiles == 1 ? (D <= 64 && single ? 3 : 2) : (D <= 64 ? 2 : 1); }

template <typename T, int D, bool EIGHT, int TILES, int WAVES, bool SINGLE>
__global__ __launch_bounds__(64 * WAVES, rows_kernel_workgroups(TILES, D, SINGLE)) void paged_rows_kernel(PagedArgs a) {
    constexpr int ROWS = 16 * TILES, kLane = EIGHT ? 16 : 8, NT = kLane / 4, kKeys = 4 * kLane, kBlocks = kKeys / kBlock;
    constexpr int NS = D / 32, NF = D / 16, SIZE = EIGHT ? 1 : 2;
    constexpr int KD = D * SIZE / 16;                       // dwords of a key that a lane holds
    static_assert((1 << kStepShift) % (WAVES * kKeys) == 0, "a step is the same number of blocks for every wave");
    __shared__ __attribute__((aligned(16))) float sums[WAVES][TILES][NF][64][4];
    __shared__ float ml[2][WAVES][ROWS];
    constexpr bool kQueriesInLds = TILES == 1 && (EIGHT || !SINGLE);      // (what else does not fit the registers)
    __shared__ __attribute__((aligned(16))) u32x4 queries[kQueriesInLds ? WAVES : 1][NS][64];
    __shared__ int last;
    auto scale_word = [](const uint8_t* scales, int at) __attribute__((always_inline)) { return (uint32_t)*(uniform_words)((uintptr_t)(scales + at) & ~(uintptr_t)3); };
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, lg = lane >> 4;

    // ---- this workgroup's share of the line
    __shared__ Known known[WAVES];
    known_of(a.s, known[wave], lane);
    const int tile_rows = SINGLE ? a.G : ROWS;
    auto tiles_of = [&](int tokens) __attribute__((always_inline)) { return SINGLE ? tokens : (tokens * a.G + ROWS - 1) / ROWS; };
    auto steps_of = [&](int keys) __attribute__((always_inline)) { return max((keys + (1 << a.unit_shift) - 1) >> a.unit_shift, 1); };
    int longest = 1, steps = 0;
    auto count = [&](int tokens, int keys) __attribute__((always_inline)) {
        const int n = steps_of(keys);
        if (tokens) longest = max(longest, n);
        steps += tiles_of(tokens) * n;
    };
    count(known[wave].tokens[lane], known[wave].line[lane]);
    for (int b = 64 + lane; b < a.s.B; b += 64) count(a.s.tokens(b), a.s.keys(b));
    longest = __builtin_amdgcn_readfirstlane((int)wave_max((float)longest));      // of one sequence (exact: at most 2^16)
    steps = __builtin_amdgcn_readlane(wave_scan(steps), 63) * a.KV;           // of all heads
    Line line(a.by_shares, a.shares, steps, longest);
    // Shares of a few steps: a share that is the end of one tile and the beginning of another costs two rounds of first loads and of joining.  Where stretches that are rounded up to l steps fit as many
    // shares of l, every workgroup has one part of one tile.  us, plain | rounded: 16 sequences of 2800 to 4000 keys (8 heads of 128, 8 bits) 32.4 | 27.9, 64 of them 85.4 | 79.0, with four tokens each 97 | 81,
    // 24 of 600 to 6000 42.3 | 37.0, 64 of 300 to 600 25.6 | 19.2, one of 30000 22.0 | 19.8; but 30 of 450 to 900, 12 heads of 64, 18.5 | 19.4.  More than 16 steps a share: level
    // Where there is a share for every step, shares of two make half as many parts to join, and of two steps none; three to sixteen steps that a unit each takes are quicker in as many parts.
    // us, one | two, 8 heads of 128 in 8 bits where nothing else is said:
    //   no more steps than units   1000 keys 9.9 | 10.8, 2000 10.0 | 10.9, 4000 10.3 | 11.1; 12 heads of 64 1000 keys 8.3 | 8.9, 3000 8.4 | 9.1; 8 sequences of 1000 11.1 | 11.9, with four tokens each 12.8 | 13.5
    //   longer ones                6000 keys 12.1 | 11.7, 8000 12.3 | 12.0; 2 heads of 96, 15000 12.3 | 11.0
    //   more steps                 8 sequences of 1500 15.7 | 12.3, 16 of 1000 16.4 | 12.7, 4 of 4000 16.0 | 12.4; 10 of 1000, 12 heads of 64, 10.0 | 9.2; 8 of 1500 in 16 bits 16.1 | 14.7
    //   two steps                  8 sequences of 250 to 500, 2 heads of 96, 8.0 | 7.1
    const bool ample = line.per == 1 && !line.more;
    const bool apart = ample && longest > 2 && longest <= 16 && steps <= a.units;
    if (line.per <= 16 && !apart && a.s.B <= 64) {
        const int n = steps_of(known[wave].line[lane]), tiles = tiles_of(known[wave].tokens[lane]);
        for (int l = line.per + (ample || line.more ? 1 : 0), l1 = line.per + line.per / 4 + 1; l <= l1; l++) {
            const int of = (int)(((float)n + (float)l - 0.5f) / (float)l);       // n / l, rounded up (n and l below 2^16, l of a few)
            const int shares = __builtin_amdgcn_readlane(wave_scan(tiles * of), 63) * a.KV;
            if (shares > a.shares) continue;
            known[wave].line[lane] = of * l << a.unit_shift;
            line.per = l;
            line.more = 0;
            steps = shares * l;
            break;
        }
    }
    wave_in_order();                                                         // (`known`)
    int g = line.begin(blockIdx.x);
    const int stop = min(line.begin(blockIdx.x + 1), steps);
    const int page_bytes = (D * SIZE) << a.s.page_shift;

    for (int segment = 0; g < stop; segment++) {
        // ---- the head that step g belongs to
        Found at;
        if (!found_at(a.s, known[wave], lane, g, [&](int tokens, int keys) { return tiles_of(tokens) * a.KV * steps_of(keys); }, at)) return;
        const int b = at.b, tokens = at.tokens, keys = at.keys, first = at.start;
        const int mine = steps_of(at.line), pair = (g - at.before) / mine, s0 = g - at.before - pair * mine;
        if (!a.part && s0) {                                                  // without a workspace a head is its beginning's, whole
            g += mine - s0;
            continue;
        }
        const int s1 = a.part ? min(mine, s0 + stop - g) : mine;
        const int tile = a.by_heads(pair), head = pair - tile * a.KV, origin = g - s0;             // of the head on the line
        g += s1 - s0;
        const int rows = tokens * a.G;
        int end = keys;                                                       // of the keys that the tile's last row sees
        if (a.is_causal) end = max(keys - tokens + a.by_group(min((tile + 1) * tile_rows, rows) - 1) + 1, 0);
        end = min(end, a.s.reach());
        const int k0 = s0 << a.unit_shift, k1 = min(end, s1 << a.unit_shift);
        const bool parted = s1 - s0 < mine;
        const Split split = parted ? split_of(line, a.shares, blockIdx.x, origin, mine) : Split{0, 1};
        uint64_t seen = 0;
        if (parted && threadIdx.x == 0) seen = arrive_look(a.words + split.first);

        // ---- queries: row li of each tile.  d of step s: see d_of
        auto d_of = [&](int s) __attribute__((always_inline)) {
            if (!EIGHT || (s | 1) >= NS) return 32 * s + 8 * lg;                // (an odd last step is loaded by itself)
            return 64 * (s >> 1) + 16 * lg + 8 * (s & 1);
        };
        u32x4 qf[TILES][NS];
        int limit[TILES];                                                    // keys that the row sees
        int open = k1;                                                       // the least of them: blocks in front of it need no mask
#pragma unroll
        for (int x = 0; x < TILES; x++) {
            const int row = tile * tile_rows + 16 * x + li, token = a.by_group(row);
            const bool mine = row < rows && (!SINGLE || 16 * x + li < a.G);
            const T* qp = static_cast<const T*>(a.q) + (int64_t)(first + token) * a.qs[0] + (int64_t)(head * a.G + row - token * a.G) * a.qs[1];
#pragma unroll
            for (int s = 0; s < NS; s++) qf[x][s] = (mine ? *reinterpret_cast<const u32x4*>(qp + d_of(s)) : u32x4{0, 0, 0, 0}) ^ a.sign;
            limit[x] = SINGLE ? k1 : min(a.is_causal ? keys - tokens + token + 1 : keys, k1);
            open = min(open, mine ? limit[x] : k1);
        }
        if (!SINGLE) open = -(int)wave_max((float)-open);
        if constexpr (kQueriesInLds) {
#pragma unroll
            for (int s = 0; s < NS; s++) queries[wave][s][lane] = qf[0][s];
        }
        auto query = [&](int x, int s) __attribute__((always_inline)) {
            if constexpr (kQueriesInLds) return queries[wave][s][lane];
            else return qf[x][s];
        };

        uniform_words table = (uniform_words)(uintptr_t)(a.s.table + (int64_t)b * a.s.width);
        // where the sixteen-token blocks of a block of keys lie, in keys and in values alike; bit i of `absent`: the table names no page for block i
        struct Place { int64_t at[kBlocks]; int32_t page[kBlocks]; uint32_t absent, ks[kBlocks], vs[kBlocks]; };
        auto ask = [&](Place& p, int key) __attribute__((always_inline)) {
            p.absent = 0;
#pragma unroll
            for (int i = 0; i < kBlocks; i++) {
                const int block = (key >> 4) + i, at = min(block >> (a.s.page_shift - 4), a.s.width - 1);
                p.page[i] = table[at];
                const bool ok = (uint32_t)p.page[i] < (uint32_t)a.pages;
                p.absent |= ok ? 0u : 1u << i;
                p.page[i] = (ok ? p.page[i] : 0) * a.KV + head;
                if (EIGHT) {                                                    // the aligned words that hold the two bytes; nothing waits for them here
                    p.ks[i] = scale_word(a.key_scales, p.page[i]);
                    p.vs[i] = scale_word(a.value_scales, p.page[i]);
                }
                p.at[i] = (int64_t)p.page[i] * page_bytes + (block & ((1 << (a.s.page_shift - 4)) - 1)) * (16 * D * SIZE);
            }
        };
        auto chosen = [&](const auto& list, int which) __attribute__((always_inline)) {
            const auto a0 = list[0], a1 = list[1], a2 = list[kBlocks > 2 ? 2 : 0], a3 = list[kBlocks > 2 ? 3 : 1];
            const auto low = (which & 1) ? a1 : a0, high = (which & 1) ? a3 : a2;
            return kBlocks > 2 && (which & 2) ? high : low;
        };
        const int key_block = kLane * (li >> 2) / kBlock, value_block = kLane * lg / kBlock;
        const int key_off = ((kLane * (li >> 2) % kBlock) + (li & 3)) * (D * SIZE) + 16 * lg, value_off = li * (16 * SIZE) + kLane * lg % kBlock * SIZE;
        struct Block { uint32_t k[NT][KD], v[NF][4], ks, vs, absent; };           // (scales: a byte for each of its kBlocks)
        auto load_k = [&](Block& blk, const Place& p) __attribute__((always_inline)) {
            const char* kp = a.keys + chosen(p.at, key_block) + key_off;
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int s = 0; s < KD / 4; s++) {
                    const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kp + 4 * j * (D * SIZE) + 64 * s));
#pragma unroll
                    for (int e = 0; e < 4; e++) blk.k[j][4 * s + e] = w[e];
                }
            if constexpr (KD % 4) {
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const u32x2 w = *reinterpret_cast<const u32x2*>(kp + 4 * j * (D * SIZE) + KD / 4 * 64 - 8 * lg);
                    blk.k[j][KD - 2] = w.x;
                    blk.k[j][KD - 1] = w.y;
                }
            }
            blk.ks = blk.vs = 0;
            if (EIGHT) {
#pragma unroll
                for (int i = 0; i < kBlocks; i++) {
                    blk.ks |= (p.ks[i] >> 8 * ((uint32_t)(uintptr_t)(a.key_scales + p.page[i]) & 3) & 255) << 8 * i;
                    blk.vs |= (p.vs[i] >> 8 * ((uint32_t)(uintptr_t)(a.value_scales + p.page[i]) & 3) & 255) << 8 * i;
                }
            }
            blk.absent = p.absent;
        };
        auto load_v = [&](Block& blk, const Place& p) __attribute__((always_inline)) {
            const char* vp = a.values + chosen(p.at, value_block) + value_off;
#pragma unroll
            for (int f = 0; f < NF; f++) {
                const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vp + 16 * f * (16 * SIZE)));
#pragma unroll
                for (int e = 0; e < 4; e++) blk.v[f][e] = w[e];
            }
        };

        f32x4 oacc[TILES][NF];
        float m_run[TILES], l_run[TILES];
        auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int x = 0; x < TILES; x++) {
                m_run[x] = -INFINITY;
                l_run[x] = 0.f;
#pragma unroll
                for (int f = 0; f < NF; f++) oacc[x][f] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        };
        clear();
        bool tame = false;
        // the scale of this quarter's keys or values
        auto scale_at = [&](uint32_t bytes) __attribute__((always_inline)) { return scale_of(bytes >> 8 * value_block & 255); };
        // scores and probabilities of a block
        auto scored = [&](const Block& blk, int key, u32x4 (&pb)[TILES][NT / 2]) __attribute__((always_inline)) {
            const int at = key + kLane * lg;                                // first key of this quarter
            const bool masked = key + kKeys > open || blk.absent;
            const bool ok = !(blk.absent >> value_block & 1);
            const float c = EIGHT ? a.c * scale_at(blk.ks) : a.c;
            float sv[TILES][4 * NT];
#pragma unroll
            for (int j = 0; j < NT; j++) {
                u32x4 kf[NS];
#pragma unroll
                for (int s = 0; s < NS; s++) {
                    if constexpr (EIGHT) kf[s] = widen<T>(u32x2{blk.k[j][2 * s], blk.k[j][2 * s + 1]}, 1.f);
                    else kf[s] = u32x4{blk.k[j][4 * s], blk.k[j][4 * s + 1], blk.k[j][4 * s + 2], blk.k[j][4 * s + 3]};
                }
#pragma unroll
                for (int x = 0; x < TILES; x++) {
                    f32x4 s4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int s = 0; s < NS; s++) s4 = Mfma16P<T>::run(kf[s], query(x, s), s4);
#pragma unroll
                    for (int r = 0; r < 4; r++) sv[x][4 * j + r] = s4[r] * c;
                }
            }
#pragma unroll
            for (int x = 0; x < TILES; x++) {
                if (masked) {
                    const int n = ok ? limit[x] - at : 0;
#pragma unroll
                    for (int e = 0; e < 4 * NT; e++) sv[x][e] = e < n ? sv[x][e] : -INFINITY;
                }
                float top = sv[x][0];
#pragma unroll
                for (int e = 1; e < 4 * NT; e++) top = fmaxf(top, sv[x][e]);
                const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, top), __builtin_bit_cast(uint32_t, top), false, false);
                top = fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
                top = half_max(top);
                const float m_new = moved_reference(m_run[x], top), use = m_new == -INFINITY ? 0.f : m_new;
                const float alpha = weight(m_run[x], use);
                m_run[x] = m_new;
                float lsum[2] = {0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 2 * NT; e++) {
                    const uint32_t two = Mfma32A<T>::pack2(weight(sv[x][2 * e], use), weight(sv[x][2 * e + 1], use));
                    pb[x][e >> 2][e & 3] = two;
                    lsum[e & 1] = plus_two<T>(two, lsum[e & 1]);
                }
                l_run[x] = l_run[x] * alpha + (lsum[0] + lsum[1]);
                if (__any(alpha != 1.f)) {
#pragma unroll
                    for (int f = 0; f < NF; f++) oacc[x][f] *= alpha;
                }
            }
        };
        auto added = [&](Block& blk, int key, const u32x4 (&pb)[TILES][NT / 2], uint32_t vs8, uint32_t absent) __attribute__((always_inline)) {
            if (key + kKeys > k1 || absent) {
                // values that no key of this part stands for may hold anything, a NaN among it
                const int n = absent >> value_block & 1 ? 0 : k1 - key - kLane * lg;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    constexpr int kPer = 4 / SIZE;
                    const int left = min(max(n - kPer * e, 0), kPer) * SIZE;
                    const uint32_t keep = left == 4 ? ~0u : (1u << (8 * left)) - 1;
#pragma unroll
                    for (int f = 0; f < NF; f++) blk.v[f][e] &= keep;
                }
            }
            if (!SINGLE && tame && key + kKeys > open) {
                bool wild = false;
#pragma unroll
                for (int f = 0; f < NF; f++)
#pragma unroll
                    for (int e = 0; e < 4; e++) blk.v[f][e] = tamed<T, EIGHT>(blk.v[f][e], wild);
            }
            const float vs = EIGHT ? scale_at(vs8) : 1.f;
#pragma unroll
            for (int f = 0; f < NF; f++)
#pragma unroll
                for (int h = 0; h < NT / 2; h++) {
                    u32x4 vf;
                    if constexpr (EIGHT) vf = widen<T>(u32x2{blk.v[f][2 * h], blk.v[f][2 * h + 1]}, vs);
                    if constexpr (EIGHT && std::is_same<T, f16_t>::value) vf = ended(vf);
                    if constexpr (!EIGHT) vf = u32x4{blk.v[f][0], blk.v[f][1], blk.v[f][2], blk.v[f][3]};
#pragma unroll
                    for (int x = 0; x < TILES; x++) oacc[x][f] = Mfma16P<T>::run(vf, pb[x][h], oacc[x][f]);
                }
        };
        constexpr int kStride = WAVES * kKeys;
        const int start = k0 + wave * kKeys, blocks = start < k1 ? (k1 - start + kStride - 1) / kStride : 0;
        if (blocks) {
            Place p;
            Block one, two;
            auto key_of = [&](int i) __attribute__((always_inline)) { return start + i * kStride; };
            auto attend = [&](Block& blk, int i, int next) __attribute__((always_inline)) {
                u32x4 pb[TILES][NT / 2];
                if (next) ask(p, key_of(min(i + 2, blocks - 1)));             // (a block behind the last is the last again)
                scored(blk, key_of(i), pb);
                __builtin_amdgcn_sched_barrier(0);
                const uint32_t vs8 = blk.vs, absent = blk.absent;
                if (next) load_k(blk, p);
                added(blk, key_of(i), pb, vs8, absent);
                __builtin_amdgcn_sched_barrier(0);
                if (next) load_v(blk, p);
            };
            for (;;) {
                ask(p, start);
                load_k(one, p);
                load_v(one, p);
                ask(p, key_of(min(1, blocks - 1)));
                load_k(two, p);
                load_v(two, p);
                int i = 0;
                for (; i + 2 < blocks; i += 2) {
                    attend(one, i, 1);
                    attend(two, i + 1, 1);
                }
                attend(one, i, 0);
                if (i + 1 < blocks) attend(two, i + 1, 0);
                if (SINGLE || open >= k1 || tame) break;
                bool odd = false;
#pragma unroll
                for (int x = 0; x < TILES; x++)
#pragma unroll
                    for (int f = 0; f < NF; f++)
#pragma unroll
                        for (int r = 0; r < 4; r++) odd |= !(fabsf(oacc[x][f][r]) < INFINITY);
                if (!__any(odd)) break;
                tame = true;                                                  // (see `tamed`)
                clear();
            }
            if (!SINGLE && tame) {
#pragma unroll 1
                for (int i = 0; i < blocks; i++) {
                    if (key_of(i) + kKeys <= open) continue;
#pragma unroll 1
                    for (int kk = key_of(i); kk < min(key_of(i) + kKeys, k1); kk++) {
                        const char* vp = value_at<D, SIZE>(a, a.s.table + (int64_t)b * a.s.width, head, kk);
                        if (!vp) continue;
#pragma unroll
                        for (int f = 0; f < NF; f++)
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                const float w = wild_of<T, EIGHT>(vp + (16 * f + 4 * lg + r) * (16 * SIZE));
#pragma unroll
                                for (int x = 0; x < TILES; x++) oacc[x][f][r] += kk < limit[x] ? w : 0.f;
                            }
                    }
                }
            }
        }

        if (parted && threadIdx.x == 0) arrive_claim(a.words + split.first, seen, a.tag);
        // ---- the waves' states, four sums a thread: O^T tile f holds d = 16 f + 4 g + e of group g
        if (segment) __syncthreads();                                        // (the segment before has been read)
#pragma unroll
        for (int x = 0; x < TILES; x++) {
            float l = l_run[x];
            l += __shfl_xor(l, 16, 64);
            l = half_sum(l);
            if (lg == 0) { ml[0][wave][16 * x + li] = m_run[x]; ml[1][wave][16 * x + li] = l; }
#pragma unroll
            for (int f = 0; f < NF; f++) *reinterpret_cast<f32x4*>(sums[wave][x][f][lane]) = oacc[x][f];
        }
        __syncthreads();
        constexpr int kFours = D / 4;
        const int here = min(tile_rows, rows - tile * tile_rows);
        const Parts<ROWS, D> own(a, 2 * (int)blockIdx.x + (s0 ? 0 : 1));
        for (int idx = threadIdx.x; idx < here * kFours; idx += 64 * WAVES) {
            const int row = idx / kFours, four = idx % kFours;
            float m = -INFINITY, l = 0.f;
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < WAVES; w++) m = fmaxf(m, ml[0][w][row]);
            const float use = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                const float al = weight(ml[0][w][row], use);
                l = fmaf(ml[1][w][row], al, l);
                const f32x4 v = *reinterpret_cast<const f32x4*>(sums[w][row >> 4][four >> 2][(four & 3) * 16 + (row & 15)]);
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = fmaf(v[e], al, o[e]);
            }
            if (!parted) {
                const float inv = l != 0.f ? 1.f / l : 0.f;
                const int r = tile * tile_rows + row, token = a.by_group(r);
                T* out = static_cast<T*>(a.o) + (int64_t)(first + token) * a.os[0] + (int64_t)(head * a.G + r - token * a.G) * a.os[1] + 4 * four;
                *reinterpret_cast<u32x2*>(out) = u32x2{Mfma32A<T>::pack2(o[0] * inv, o[1] * inv), Mfma32A<T>::pack2(o[2] * inv, o[3] * inv)};
            } else {
                store_part(parts_rsrc(own.sums), (uint32_t)(idx * 16), o);
                if (four == 0) store_two(own.state + 2 * row, m, l);
            }
        }
        if (parted && arrive_last(a.words + split.first, split.parts, &last)) join<T, ROWS, D, 64 * WAVES>(a, split, first, head, tile * tile_rows, here);
    }
}

// ---------------------------------------------------------------- many rows
// 128 rows, 32 a wave, over stages of 64 keys that lie in LDS in the queries' type, two of them: the next one is on its way in registers and is converted and put down behind this one's products.
// Two workgroups a unit, so that one is at its products while the other is at its weights; a wave at its products goes first (s_setprio: 647 us | 639).  A stage of all eight waves of a unit takes
// some 3000 cycles, of which the matrix units are busy 2048 (1024 a wave, two waves each), LDS 2560 (32 KB of operands a wave, and two stages that are put down) and the vector units some 2600 (the
// exponentials 1024 of them): three pipes that are full to 70 and 85 in a hundred, none of which leaves room for much.
//
// WAVES = 8, where keys of 128 numbers lie in 16 bits and sequences have 256 rows: a thread has half the pieces to stage, so that keys and values are asked for together.  us, 128 rows | 256: four
// pieces of 1024 tokens behind 7168 702 | 641, one of 512 behind 32000 361 | 345, prompts of 2048 tokens 212 | 207, 512 rows over 2000 keys 76 | 69; but heads of 96 566 | 615, and 8-bit pages
// 297 | 299 and 195 | 198.  (64 rows a wave, so that a row of K from LDS feeds two products: 609 | 848, for one workgroup a unit has nothing to do meanwhile.)
//
//   S^T = K Q^T     v_mfma_f32_32x32x16: operand row i of tile j is key 32 j + 16 (r / 8) + 8 h + r % 8 where register r of half h of the result is row i, so that
//   O^T += V^T P^T  a half's eight registers of a step are the probabilities of eight neighbouring keys: sixteen bytes of a row of V^T.
constexpr int kStage = 64;

template <int D>
__device__ __forceinline__ uint32_t tk_off(int key, int chunk) {          // K [64][D]: chunks of eight elements, rotated by the key
    constexpr int kMask = D >= 128 ? 15 : D >= 64 ? 7 : 3;
    if constexpr (D == 96) return (uint32_t)(key * 208 + chunk * 16);     // (twelve chunks: a row of thirteen instead)
    else return (uint32_t)(key * (D * 2) + ((chunk ^ ((D == 128 ? key : D == 64 ? key >> 1 : key >> 2) & kMask)) << 4));
}
__device__ __forceinline__ uint32_t tv_off(int d, int chunk) {            // V^T [D][64]
    return (uint32_t)(d * 128 + ((chunk ^ ((d >> 1) & 7)) << 4));
}

// The line's stretches: a tile's is its keys and what a tile costs besides (kTileCost keys' worth: 16 times 64 tokens behind 2000 take 84 us where it is 128, 74 with 400, 76 with 600), which grows from tile to tile by the tokens of one where the causal rule holds; head by head.
constexpr int kTileCost = 384;
template <int ROWS>
struct Stretch {
    int tiles, first, grows;
    __device__ __forceinline__ Stretch(const PagedArgs& a, int tokens, int keys) {
        const int wide = a.by_group(ROWS + a.G - 1);
        tiles = (tokens * a.G + ROWS - 1) / ROWS;
        first = (((a.is_causal ? max(keys - tokens, 0) + wide : keys) + kTileCost) >> a.unit_shift) + 1;
        grows = a.is_causal ? wide >> a.unit_shift : 0;
    }
    __device__ __forceinline__ int before(int t) const { return t * first + grows * (t * (t - 1) / 2); }
    __device__ __forceinline__ int length(int t) const { return first + grows * t; }
    // the tile that place x lies in
    __device__ __forceinline__ int tile(int x) const {
        const float f = (float)first - 0.5f * (float)grows;
        int t = grows ? (int)((__builtin_sqrtf(f * f + 2.f * (float)grows * (float)x) - f) / (float)grows) : x / first;
        t = min(max(t, 0), tiles - 1);
        while (t > 0 && before(t) > x) t--;
        while (t < tiles - 1 && before(t + 1) <= x) t++;
        return __builtin_amdgcn_readfirstlane(t);
    }
};

template <typename T, int D, bool EIGHT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void paged_tile_kernel(PagedArgs a) {
    constexpr int ROWS = 32 * WAVES, kThreads = 64 * WAVES;
    constexpr int NS = D / 16, NF = D / 32, SIZE = EIGHT ? 1 : 2;
    constexpr int kKBytes = D == 96 ? 64 * 208 : 64 * D * 2, kVBytes = D * 128;
    constexpr int kPieces = 64 * D * SIZE / 16, kMine = (kPieces + kThreads - 1) / kThreads;      // pieces of sixteen bytes of K, and of V, of a stage; a thread's
    __shared__ __attribute__((aligned(16))) char lds[2][kKBytes + kVBytes];
    __shared__ Known known[WAVES];
    __shared__ int last;
    // Where f16 does not hold 8-bit keys times their page's scale (it holds what scales from 2^-15 to 2^7 make) they are widened without, and the scores of the block of sixteen take the scale:
    // a stage's four bytes, 0 for a block whose keys have it.  (us, four f16 pieces of 1024 tokens behind 7168 over 8-bit pages 607 without this, 620 with it; every block's scale with the scores 632 to 648.)
    constexpr bool kLeft = EIGHT && std::is_same<T, f16_t>::value;
    __shared__ uint32_t scales_left[2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 31, lh = lane >> 5;

    // ---- this workgroup's share of the line.  Eight neighbours of the launch, which are on eight XCDs, take shares an eighth of the line apart: what an XCD's workgroups read at a time belongs to few heads
    known_of(a.s, known[wave], lane);
    wave_in_order();
    int longest = 1, shortest = 1 << 30, all = 0, count = 0;
    auto add = [&](int tokens, int keys) __attribute__((always_inline)) {
        const Stretch<ROWS> st(a, tokens, keys);
        if (!st.tiles) return;
        longest = max(longest, st.length(st.tiles - 1));
        shortest = min(shortest, st.first);
        all += st.before(st.tiles);
        count += st.tiles;
    };
    add(known[wave].tokens[lane], known[wave].line[lane]);
    for (int b = 64 + lane; b < a.s.B; b += 64) add(a.s.tokens(b), a.s.keys(b));
    longest = (int)(wave_max((float)longest) * 1.00001f) + 1;
    shortest = -(int)wave_max((float)-shortest);
    all = __builtin_amdgcn_readlane(wave_scan(all), 63) * a.KV;
    count = __builtin_amdgcn_readlane(wave_scan(count), 63) * a.KV;
    // Where no tile has many keys, or there is a tile for every share and short ones that come last and fill the gaps (a prompt from its beginning), a workgroup takes one whole tile instead, and
    // none is joined; so it does without a workspace.  us, shares | tiles: 16 times 64 tokens behind 500 45 | 29, two of 512 50 | 42, one of 300 behind 2000 46 | 81; four prompts of 2048 tokens
    // 270 | 196, one of 4000 199 | 180; three pieces of 550 to 930 tokens behind 5000 to 7000 304 | 480
    const bool tiles = !a.part || longest <= (1024 + kTileCost) >> a.unit_shift || (count >= a.shares && shortest <= (512 + kTileCost) >> a.unit_shift);
    const Line line(a.by_shares, a.shares, all, longest);
    if ((int)blockIdx.x >= (tiles ? count : a.shares)) return;
    const int share = a.shares & 7 ? blockIdx.x : (blockIdx.x & 7) * (a.shares >> 3) + (blockIdx.x >> 3);
    int g = tiles ? 0 : line.begin(share);
    const int stop = tiles ? 1 : min(line.begin(share + 1), all);

    for (int segment = 0; g < stop; segment++) {
    Found found;
    int tile, head, off0 = 0, off1, length, origin = 0;
    if (tiles) {
        const int unit = a.by_heads(blockIdx.x);
        head = blockIdx.x - unit * a.KV;
        int level;
        if (a.s.B <= 64) {
            // the last tiles of all sequences, then those in front of them, ...: `level` of them lie in front of this one's
            const int own = (known[wave].tokens[lane] * a.G + ROWS - 1) / ROWS;
            auto before = [&](int n) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(wave_scan(min(own, n)), 63); };
            int low = 0;
            for (int step = 1 << (31 - __builtin_clz(a.s.T * a.G / ROWS + 1)); step; step >>= 1)
                if (before(low + step) <= unit) low += step;
            level = low;
            const int has = own > level ? 1 : 0, place = wave_scan(has) - has, wanted = unit - before(level);
            const uint64_t m = __ballot(has && place == wanted);
            if (!m) return;
            found.b = __builtin_ctzll(m);
            found.start = __builtin_amdgcn_readfirstlane(known[wave].start[found.b]);
            found.tokens = __builtin_amdgcn_readfirstlane(known[wave].tokens[found.b]);
            found.keys = __builtin_amdgcn_readfirstlane(known[wave].keys[found.b]);
            found.line = __builtin_amdgcn_readfirstlane(known[wave].line[found.b]);
        } else {
            if (!found_at(a.s, known[wave], lane, unit, [&](int tokens, int keys) { return Stretch<ROWS>(a, tokens, keys).tiles; }, found)) return;
            level = unit - found.before;
        }
        const Stretch<ROWS> st(a, found.tokens, found.line);
        tile = st.tiles - 1 - level;
        off1 = length = st.length(tile);
        g = stop;
    } else {
        if (!found_at(a.s, known[wave], lane, g, [&](int tokens, int keys) { const Stretch<ROWS> st(a, tokens, keys); return a.KV * st.before(st.tiles); }, found)) return;
        const Stretch<ROWS> st(a, found.tokens, found.line);
        const int of_head = st.before(st.tiles), x = g - found.before;
        head = x / of_head;
        tile = st.tile(x - head * of_head);
        off0 = x - head * of_head - st.before(tile);
        length = st.length(tile);
        origin = g - off0;
        off1 = min(length, off0 + stop - g);
        g += off1 - off0;
    }
    const int tokens = found.tokens, keys = found.keys, first = found.start;
    const int rows = tokens * a.G, row = tile * ROWS + 32 * wave + li, token = a.by_group(row);
    int end = keys;                                                          // of the keys that the tile's last row sees
    if (a.is_causal) end = max(keys - tokens + a.by_group(min((tile + 1) * ROWS, rows) - 1) + 1, 0);
    end = min(end, a.s.reach());
    auto cut = [&](int off) __attribute__((always_inline)) { return off == 0 ? 0 : off >= length ? end : min(max((off << a.unit_shift) - 96, 0) & ~(kStage - 1), end); };
    const int k0 = cut(off0), k1 = cut(off1);
    const bool parted = off0 > 0 || off1 < length;
    const Split split = parted ? split_of(line, a.shares, share, origin, length) : Split{0, 1};
    uint64_t seen = 0;
    if (parted && threadIdx.x == 0) seen = arrive_look(a.words + split.first);

    u32x4 qf[NS];
    {
        const T* qp = static_cast<const T*>(a.q) + (int64_t)(first + token) * a.qs[0] + (int64_t)(head * a.G + row - token * a.G) * a.qs[1];
#pragma unroll
        for (int s = 0; s < NS; s++) qf[s] = (row < rows ? *reinterpret_cast<const u32x4*>(qp + 16 * s + 8 * lh) : u32x4{0, 0, 0, 0}) ^ a.sign;
    }
    const int limit = row < rows ? min(a.is_causal ? keys - tokens + token + 1 : keys, k1) : 0;
    const int open = -(int)wave_max((float)-(row < rows ? limit : k1));              // blocks in front of it need no mask
    const int seen_keys = (int)wave_max((float)limit);                               // blocks behind it concern no row of the wave
    const int mixed = a.is_causal ? keys - tokens + a.by_group(tile * ROWS) + 1 : k1;       // keys from here on are seen by some rows of the tile only

    const int32_t* table = a.s.table + (int64_t)found.b * a.s.width;
    uniform_words scalar_table = (uniform_words)(uintptr_t)table;
    // Sixteen tokens' keys are as many bytes in a row as their values are, kPer pieces of sixteen bytes: piece `idx` of a stage lies at the same place of both
    constexpr int kPer = D * SIZE;
    const int page_blocks = a.s.page_shift - 4;
    // In 16 bits a thread's pieces of both do not fit the registers: values are asked for when the next keys lie in LDS
    constexpr bool kApart = !EIGHT && D > 64 && WAVES == 4;
    struct Stage { u32x4 k[kMine], v[kApart ? 1 : kMine]; uint32_t ks[kMine], vs[kMine]; };
    struct Pages { int at[kMine]; uint32_t absent; };       // bit i of `absent`: the table names no page for block i
    auto ask = [&](Pages& p, int key) __attribute__((always_inline)) {
        p.absent = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int at = min(((key >> 4) + i) >> page_blocks, a.s.width - 1);
            p.absent |= (uint32_t)scalar_table[at] < (uint32_t)a.pages ? 0u : 1u << i;
        }
#pragma unroll
        for (int i = 0; i < kMine; i++) {
            const int block = ((int)threadIdx.x + kThreads * i) / kPer;
            const int at = min(((key >> 4) + (kPer % 64 ? block : __builtin_amdgcn_readfirstlane(block))) >> page_blocks, a.s.width - 1);
            const int page = kPer % 64 ? table[at] : scalar_table[at];
            p.at[i] = ((uint32_t)page < (uint32_t)a.pages ? page : 0) * a.KV + head;
        }
    };
    auto load = [&](u32x4 (&w)[kMine], uint32_t (&scale)[kMine], const char* from, const uint8_t* scales, const Pages& p, int key) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kMine; i++) {
            const int idx = threadIdx.x + kThreads * i;
            if (kPieces % kThreads && idx >= kPieces) continue;
            const int block = ((key >> 4) + (kPer % 64 ? idx / kPer : __builtin_amdgcn_readfirstlane(idx / kPer))) & ((1 << page_blocks) - 1);
            w[i] = *reinterpret_cast<const u32x4*>(from + (((int64_t)p.at[i] << page_blocks) + block) * (16 * kPer) + idx % kPer * 16);
            if (EIGHT) scale[i] = scales[p.at[i]];
        }
    };
    auto values_of = [](Stage& st) __attribute__((always_inline)) -> u32x4 (&)[kMine] {
        if constexpr (kApart) return st.k;
        else return st.v;
    };
    auto load_k = [&](Stage& st, const Pages& p, int key) __attribute__((always_inline)) { load(st.k, st.ks, a.keys, a.key_scales, p, key); };
    auto load_v = [&](Stage& st, const Pages& p, int key) __attribute__((always_inline)) { load(values_of(st), st.vs, a.values, a.value_scales, p, key); };
    auto put_k = [&](Stage& st, char* to, uint32_t* left) __attribute__((always_inline)) {
        constexpr int kKeyPieces = D * SIZE / 16;
#pragma unroll
        for (int i = 0; i < kMine; i++) {
            const int idx = threadIdx.x + kThreads * i, k = idx / kKeyPieces, kc = idx % kKeyPieces;
            if (kPieces % kThreads && idx >= kPieces) continue;
            if constexpr (EIGHT) {
                float scale = scale_of(st.ks[i]);
                if constexpr (kLeft) {
                    const bool held = scale >= 0x1p-15f && scale <= 0x1p7f;
                    if (idx % kPer == 0) reinterpret_cast<uint8_t*>(left)[idx / kPer] = held ? 0 : (uint8_t)max(st.ks[i], 1u);
                    scale = held ? scale : 1.f;
                }
                *reinterpret_cast<u32x4*>(to + tk_off<D>(k, 2 * kc)) = widen<T>(u32x2{st.k[i].x, st.k[i].y}, scale);
                *reinterpret_cast<u32x4*>(to + tk_off<D>(k, 2 * kc + 1)) = widen<T>(u32x2{st.k[i].z, st.k[i].w}, scale);
            } else {
                *reinterpret_cast<u32x4*>(to + tk_off<D>(k, kc)) = st.k[i];
            }
        }
    };
    auto put_v = [&](Stage& st, uint32_t absent, int key, char* to, bool tame) __attribute__((always_inline)) {
        const bool leave = tame && key + kStage > mixed, last_ones = key + kStage > k1 || absent;
#pragma unroll
        for (int i = 0; i < kMine; i++) {
            const int idx = threadIdx.x + kThreads * i;
            if (kPieces % kThreads && idx >= kPieces) continue;
            u32x4 w = values_of(st)[i];
            const int block = idx / kPer, d = idx % kPer / SIZE, half = EIGHT ? 0 : idx & 1;
            // values that no key of this part stands for may hold anything, a NaN among it
            if (last_ones) {
                const int n = absent >> block & 1 ? 0 : k1 - key - 16 * block - 8 * half;
                constexpr int kOf = 4 / SIZE;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int left = min(max(n - kOf * e, 0), kOf) * SIZE;
                    w[e] &= left == 4 ? ~0u : (1u << (8 * left)) - 1;
                }
            }
            if (leave) {
                bool wild = false;
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = tamed<T, EIGHT>(w[e], wild);
            }
            char* tv = to + kKBytes;
            if constexpr (EIGHT) {
                const float scale = scale_of(st.vs[i]);
                u32x4 low = widen<T>(u32x2{w.x, w.y}, scale), high = widen<T>(u32x2{w.z, w.w}, scale);
                if (std::is_same<T, f16_t>::value && __any(scale > 128.f)) {
                    low = ended(low);
                    high = ended(high);
                }
                *reinterpret_cast<u32x4*>(tv + tv_off(d, 2 * block)) = low;
                *reinterpret_cast<u32x4*>(tv + tv_off(d, 2 * block + 1)) = high;
            } else {
                *reinterpret_cast<u32x4*>(tv + tv_off(d, 2 * block + half)) = w;
            }
        }
    };

    f32x16 oacc[NF];
#pragma unroll
    for (int f = 0; f < NF; f++) oacc[f] = f32x16{};
    float m_run = -INFINITY, l_run = 0.f;
    // row li of a tile of S^T is key `of` of its 32
    const int of = 16 * (li >> 4) + 8 * ((li >> 2) & 1) + 4 * ((li >> 3) & 1) + (li & 3);

    auto scores = [&](u32x4 (&pb)[4], const char* from, const uint32_t* left_at, int key, uint32_t absent) __attribute__((always_inline)) {
        f32x16 sv[2];
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            sv[j] = f32x16{};
#pragma unroll
            for (int s = 0; s < NS; s++)
                sv[j] = Mfma32A<T>::run(*reinterpret_cast<const u32x4*>(from + tk_off<D>(32 * j + of, 2 * s + lh)), qf[s], sv[j]);
        }
        __builtin_amdgcn_s_setprio(0);
        if constexpr (kLeft) {
            const uint32_t left = __builtin_amdgcn_readfirstlane(*left_at);
            if (__builtin_expect(left != 0, 0)) {
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const uint32_t byte = left >> 8 * (2 * j + (r >> 3)) & 255;
                        sv[j][r] *= byte ? scale_of(byte) : 1.f;
                    }
            }
        }
        float top = -INFINITY;
        if (key + kStage > open || absent) {
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int at = 32 * j + 16 * (r >> 3) + 8 * lh + (r & 7);
                    const bool in = key + at < limit && !(absent >> (2 * j + (r >> 3)) & 1);
                    sv[j][r] = in ? sv[j][r] : -INFINITY;
                }
        }
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int r = 0; r < 16; r += 2) top = fmaxf(fmaxf(top, sv[j][r]), sv[j][r + 1]);
        // (the products are scaled in one step with the subtraction; a.c > 0)
        top = half_max(top) * a.c;
        const float m_new = moved_reference(m_run, top), use = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = weight(m_run, use);
        m_run = m_new;
        float lsum[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const uint32_t two = Mfma32A<T>::pack2(__builtin_amdgcn_exp2f(fmaf(sv[j][r], a.c, -use)), __builtin_amdgcn_exp2f(fmaf(sv[j][r + 1], a.c, -use)));
                pb[2 * j + (r >> 3)][(r >> 1) & 3] = two;
                lsum[j] = plus_two<T>(two, lsum[j]);
            }
        l_run = l_run * alpha + (lsum[0] + lsum[1]);
        if (__any(alpha != 1.f)) {
#pragma unroll
            for (int f = 0; f < NF; f++) oacc[f] *= alpha;
        }
    };
    auto product = [&](const u32x4 (&pb)[4], const char* from) __attribute__((always_inline)) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int ks = 0; ks < 4; ks++)
#pragma unroll
            for (int f = 0; f < NF; f++)
                oacc[f] = Mfma32A<T>::run(*reinterpret_cast<const u32x4*>(from + kKBytes + tv_off(32 * f + li, 2 * ks + lh)), pb[ks], oacc[f]);
        __builtin_amdgcn_s_setprio(0);
    };

    auto go = [&](bool tame) __attribute__((always_inline)) {
        Pages pg;
        Stage st;
        ask(pg, k0);
        uint32_t absent = pg.absent;
        load_k(st, pg, k0);
        if constexpr (kApart) put_k(st, lds[0], &scales_left[0]);
        load_v(st, pg, k0);
        if constexpr (!kApart) put_k(st, lds[0], &scales_left[0]);
        put_v(st, absent, k0, lds[0], tame);
        ask(pg, k0 + kStage);
        __syncthreads();
        // (which of the two stages is known at compile time, so that an address in LDS is a lane's own and a constant.  us: four pieces of 1024 tokens behind 7168 611 | 602, three of 550 to 930 285 | 281)
        auto stage = [&](auto which, int key) __attribute__((always_inline)) {
            char *now = lds[decltype(which)::value], *next = lds[decltype(which)::value ^ 1];
            const bool more = key + kStage < k1;
            const uint32_t then = pg.absent;
            if (more) {
                load_k(st, pg, key + kStage);
                if constexpr (!kApart) {
                    load_v(st, pg, key + kStage);
                    ask(pg, key + 2 * kStage);
                }
            }
            u32x4 pb[4];
            if (key < seen_keys) scores(pb, now, &scales_left[decltype(which)::value], key, absent);
            if (kApart && more) {
                put_k(st, next, &scales_left[0]);
                load_v(st, pg, key + kStage);
                ask(pg, key + 2 * kStage);
            }
            if (key < seen_keys) product(pb, now);
            if (more) {
                if constexpr (!kApart) put_k(st, next, &scales_left[decltype(which)::value ^ 1]);
                put_v(st, then, key + kStage, next, tame);
            }
            __syncthreads();
            absent = then;
            return more;
        };
        for (int key = k0; key < k1; key += 2 * kStage)
            if (!stage(std::integral_constant<int, 0>{}, key) || !stage(std::integral_constant<int, 1>{}, key + kStage)) break;
    };
    if (segment) __syncthreads();                                            // (the segment before has been read)
    bool tame = false;
    while (k0 < k1) {
        go(tame);
        if (mixed >= k1 || tame) break;
        bool odd = false;
#pragma unroll
        for (int f = 0; f < NF; f++)
#pragma unroll
            for (int r = 0; r < 16; r++) odd |= !(fabsf(oacc[f][r]) < INFINITY);
        if (!__syncthreads_or(odd)) break;
        tame = true;                                                         // (see `tamed`)
#pragma unroll
        for (int f = 0; f < NF; f++) oacc[f] = f32x16{};
        m_run = -INFINITY;
        l_run = 0.f;
    }
    if (tame) {
#pragma unroll 1
        for (int kk = max(k0, mixed) & ~(kStage - 1); kk < k1; kk++) {
            const char* vp = kk < k0 ? nullptr : value_at<D, SIZE>(a, table, head, kk);
            if (!vp) continue;
#pragma unroll
            for (int f = 0; f < NF; f++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const float x = wild_of<T, EIGHT>(vp + (32 * f + 8 * (r >> 2) + 4 * lh + (r & 3)) * (16 * SIZE));
                    oacc[f][r] += kk < limit ? x : 0.f;
                }
        }
    }

    l_run = half_sum(l_run);
    if (!parted) {
        if (row < rows) {
            const float inv = l_run != 0.f ? 1.f / l_run : 0.f;
            T* out = static_cast<T*>(a.o) + (int64_t)(first + token) * a.os[0] + (int64_t)(head * a.G + row - token * a.G) * a.os[1] + 4 * lh;
#pragma unroll
            for (int f = 0; f < NF; f++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    *reinterpret_cast<u32x2*>(out + 32 * f + 8 * g) =
                        u32x2{Mfma32A<T>::pack2(oacc[f][4 * g] * inv, oacc[f][4 * g + 1] * inv), Mfma32A<T>::pack2(oacc[f][4 * g + 2] * inv, oacc[f][4 * g + 3] * inv)};
        }
        continue;
    }
    if (threadIdx.x == 0) arrive_claim(a.words + split.first, seen, a.tag);
    const Parts<ROWS, D> own(a, 2 * share + (off0 ? 0 : 1));
    if (row < rows) {
        const __amdgpu_buffer_rsrc_t rs = parts_rsrc(own.sums);
        const int r = 32 * wave + li;
#pragma unroll
        for (int f = 0; f < NF; f++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                store_part(rs, (uint32_t)((((wave * NF + f) * 4 + g) * 64 + lane) * 16), f32x4{oacc[f][4 * g], oacc[f][4 * g + 1], oacc[f][4 * g + 2], oacc[f][4 * g + 3]});
        if (lh == 0) store_two(own.state + 2 * r, m_run, l_run);
    }
    if (arrive_last(a.words + split.first, split.parts, &last)) join<T, ROWS, D, kThreads>(a, split, first, head, tile * ROWS, min(ROWS, rows - tile * ROWS));
    }
}

// The launch that serves these sizes: rows of a workgroup's tile, the workgroups that share the work, and log2 of the keys that a unit of their line stands for.
struct Plan { int rows, shares, unit_shift; bool single; int64_t tiles; };

// Of sizes that check_sizes lets pass; refused is what has more rows than the kernels' integers hold, or more tiles than a launch of a workgroup each has threads for (2^32).
int plan_of(const mhip_paged_cache* c, const mhip_sequences* s, int64_t q_heads, Plan& p) {
    if (q_heads <= 0 || q_heads % c->heads) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_attention: %lld query heads over %lld key heads", (long long)q_heads, (long long)c->heads);
    if (s->sequences == 0 || s->tokens == 0) return MHIP_OK;
    if (q_heads / c->heads >= ((1 << 30) + s->tokens - 1) / s->tokens) return fail(MHIP_ERR_UNSUPPORTED, "paged_attention: more than 2^30 rows");
    const int64_t G = q_heads / c->heads, average = (s->tokens + s->sequences - 1) / s->sequences * G;
    const int rows = average <= 16 ? 16 : average <= 32 ? 32 : average >= 256 && c->head_size == 128 && !c->key_scales ? 256 : 128;
    const double tiles = (double)(s->tokens * G / rows + (s->sequences < s->tokens ? s->sequences : s->tokens)) * c->heads;      // that there can be
    if (rows >= 128 && tiles * (2 * rows) >= 4294967296.0) return fail(MHIP_ERR_UNSUPPORTED, "paged_attention: more tiles than a launch has workgroups");      // (two threads a row)
    const int64_t keys = s->width * c->page_size;
    auto most = [&](int shift) { return rows >= 128 ? tiles * (double)((2 * (keys + 2 * kTileCost) >> shift) + 1) : tiles * (double)((keys >> shift) + 1); };
    const bool single = s->tokens <= s->sequences && G <= rows && rows < 128;
    int shift = rows >= 128 ? 0 : kStepShift;
    while (most(shift) > (double)(1 << 29)) shift++;
    int shares = (rows >= 128 ? 256 / rows : rows_kernel_workgroups(rows / 16, c->head_size, single)) * compute_units();
    if (rows < 128 && most(shift) < shares) shares = (int)most(shift);                                                     // (a step is the least share)
    p = {rows, shares, shift, single, (int64_t)tiles};
    return MHIP_OK;
}

int64_t workspace_of(const mhip_paged_cache* c, const Plan& p) { return (int64_t)p.shares * (2 * p.rows * (c->head_size + 2) * 4 + 8); }

template <typename T, int D, bool EIGHT>
int launch(hipStream_t st, const PagedArgs& a, const Plan& p) {
    const dim3 grid((unsigned)(p.rows >= 128 && (!a.part || p.tiles >= p.shares) ? std::max<int64_t>(p.tiles, p.shares) : p.shares));
    if (p.rows == 16 && p.single) hipLaunchKernelGGL((paged_rows_kernel<T, D, EIGHT, 1, 4, true>), grid, dim3(256), 0, st, a);
    else if (p.rows == 16) hipLaunchKernelGGL((paged_rows_kernel<T, D, EIGHT, 1, 4, false>), grid, dim3(256), 0, st, a);
    else if (p.rows == 32 && p.single) hipLaunchKernelGGL((paged_rows_kernel<T, D, EIGHT, 2, 4, true>), grid, dim3(256), 0, st, a);
    else if (p.rows == 32) hipLaunchKernelGGL((paged_rows_kernel<T, D, EIGHT, 2, 4, false>), grid, dim3(256), 0, st, a);
    else if (p.rows == 128) hipLaunchKernelGGL((paged_tile_kernel<T, D, EIGHT, 4>), grid, dim3(256), 0, st, a);
    else if constexpr (D == 128 && !EIGHT) hipLaunchKernelGGL((paged_tile_kernel<T, D, EIGHT, 8>), grid, dim3(512), 0, st, a);
    return check_launch("paged_attention");
}

template <typename T, bool EIGHT>
int launch_d(hipStream_t st, const PagedArgs& a, const Plan& p, int64_t D) {
    switch (D) {
        case 32: return launch<T, 32, EIGHT>(st, a, p);
        case 64: return launch<T, 64, EIGHT>(st, a, p);
        case 96: return launch<T, 96, EIGHT>(st, a, p);
        default: return launch<T, 128, EIGHT>(st, a, p);
    }
}

}  // namespace
}  // namespace mhip

using namespace mhip;

extern "C" int64_t mhip_paged_attention_workspace(const mhip_paged_cache* cache, const mhip_sequences* seqs, int64_t q_heads) {
    Plan p{};
    return check_sizes("paged_attention_workspace", cache, seqs) || plan_of(cache, seqs, q_heads, p) ? 0 : workspace_of(cache, p);
}

extern "C" int mhip_paged_attention(void* stream, const mhip_paged_cache* cache, const mhip_sequences* seqs, const void* q, void* o, int64_t q_heads, float scale,
                                    int is_causal, const int64_t* strides, int dtype, void* workspace, int64_t workspace_bytes) {
    bool empty;
    if (const int rc = check_paged("paged_attention", cache, seqs, dtype, &empty)) return rc;
    Plan p{};
    if (const int rc = plan_of(cache, seqs, q_heads, p)) return rc;
    if (empty) return MHIP_OK;
    if (!q || !o || !strides) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_attention: NULL tensor");
    if (((uintptr_t)q | (uintptr_t)o | (uintptr_t)workspace) & 15) return fail(MHIP_ERR_UNSUPPORTED, "paged_attention: tensors must be 16-byte aligned");
    for (int i = 0; i < 4; i++)
        if (strides[i] % 8) return fail(MHIP_ERR_UNSUPPORTED, "paged_attention: strides must be multiples of 8 elements");
    PagedArgs a{q, o, (const char*)cache->keys, (const char*)cache->values, cache->key_scales, cache->value_scales, sequences(cache, seqs),
                (int)cache->pages, (int)cache->heads, (int)(q_heads / cache->heads), is_causal ? 1 : 0, p.shares, compute_units(), scale == 0.f ? 1e-30f : std::fabs(scale) * kLog2e, std::signbit(scale) ? 0x80008000u : 0u, {strides[0], strides[1]}, {strides[2], strides[3]},
                nullptr, nullptr, 0, Divider((uint32_t)(q_heads / cache->heads)), Divider((uint32_t)cache->heads), Divider((uint32_t)p.shares), p.unit_shift};
    if (workspace && workspace_bytes >= workspace_of(cache, p)) {
        a.part = static_cast<float*>(workspace);
        a.words = reinterpret_cast<uint64_t*>(a.part + 2 * (int64_t)p.shares * p.rows * (cache->head_size + 2));
        a.tag = launch_tag();
    }
    hipStream_t st = as_stream(stream);
    const bool eight = cache->key_scales != nullptr;
    const int64_t D = cache->head_size;
    if (dtype == MHIP_BF16) return eight ? launch_d<bf16_t, true>(st, a, p, D) : launch_d<bf16_t, false>(st, a, p, D);
    return eight ? launch_d<f16_t, true>(st, a, p, D) : launch_d<f16_t, false>(st, a, p, D);
}
