// Attention over a paged cache (paged.h): O = softmax(scale Q K^T) V, rows of queries from one token of a sequence to a whole prompt behind a long context.
//
//   rows   of a sequence and a key/value head: its tokens times the G = H / KV query heads that share the head, row = token * G + query head, so that K and V are read
//          once for all of them.  A token's position is keys(b) - tokens(b) + i; with the causal rule it sees the keys up to its own.
//   parts  The keys of a tile of rows are dealt over parts of one length for the whole launch, chosen on the device from all sequences' lengths such that the
//          parts fill it: the lengths are not known on the host, and a batch may hold one long sequence among short ones.  A part leaves its
//          reference maximum, its sum and its unnormalised rows in the workspace, and the last one to arrive puts them together (arrive.h).
//
// Two kernels.  Up to 32 rows a sequence on average (decode steps): paged_rows_kernel, whose waves have keys of their own and load them straight into matrix operands;
// its time is that of reading K and V.  More rows: paged_tile_kernel, 128 rows whose four waves share K and V in LDS, in the queries' type; its time is the matrix products'.
//
// fp32 sums, softmax state and scores (a key's scale is applied to its score in the first kernel, while it is converted in the second); probabilities are rounded to the queries' type in front of the second product,
// whose error of half a step each (2^-9 for bf16) is below the result's own rounding once it is averaged over keys.  Values in 8 bits become the queries' type exactly,
// scale and all, except that f16 ends at 65504 and at 2^-24.
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
    int pages, KV, G, is_causal, target;
    float c;                                  // scale * log2(e)
    int64_t qs[2], os[2];                     // token and head strides in elements
    float* part;                              // workspace, NULL: keys are not dealt
    uint64_t* words;
    uint64_t tag;
    Divider by_group, by_heads, by_shares;    // G, KV, target
    int step_shift;                           // log2 of the keys of a step (few rows)
};

// What a workgroup computes.
struct Task { int b, tile, part, parts, k0, k1, first, tokens, keys; };

constexpr int kMostParts = 64;

// Unit u of the launch: tiles of ROWS rows of every sequence, times the parts of its keys.  Parts are a multiple of STEP keys.
template <int ROWS, int STEP>
__device__ __forceinline__ bool task_of(const PagedArgs& a, int u, Task& t) {
    const int lane = threadIdx.x & 63;
    int per = 1 << 28;                                                  // keys a part
    auto tiles = [&](int b) __attribute__((always_inline)) { return (a.s.tokens(b) * a.G + ROWS - 1) / ROWS; };
    if (a.part) {
        float all = 0.f;
        int most = 0;
        for (int b = lane; b < a.s.B; b += 64) {
            const int keys = a.s.keys(b);
            all += (float)tiles(b) * (float)keys;
            most = max(most, keys);
        }
        all = wave_sum(all);
        const int longest = (int)wave_max((float)most);
        const float share = fminf(all * (float)a.KV / (float)a.target, (float)(1 << 27));
        per = max((int)share, longest / kMostParts);
        per = max((per + STEP) / STEP * STEP, 4 * STEP);
    }
    auto parts_of = [&](int keys) __attribute__((always_inline)) { return max((keys + per - 1) / per, 1); };
    auto units = [&](int b) __attribute__((always_inline)) { return tiles(b) * parts_of(a.s.keys(b)); };
    int before;
    t.b = sequence_of(a.s.B, u, units, before);
    if (t.b < 0) return false;
    t.tokens = __builtin_amdgcn_readfirstlane(a.s.tokens(t.b));
    t.keys = __builtin_amdgcn_readfirstlane(a.s.keys(t.b));
    t.first = __builtin_amdgcn_readfirstlane(a.s.start(t.b));
    const int dealt = parts_of(t.keys), count = tiles(t.b), r = u - before;
    if (r < 0 || r >= dealt * count) return false;                      // (starts that are no starts: their sums may have wrapped)
    t.tile = count - 1 - r / dealt;                                     // (the longest first where the causal rule shortens them)
    t.part = r % dealt;
    int end = t.keys;                                                   // of the keys that the tile's last row sees
    if (a.is_causal) {
        const int last = a.by_group(min((t.tile + 1) * ROWS - 1, t.tokens * a.G - 1));
        end = max(t.keys - t.tokens + last + 1, 0);
    }
    t.parts = parts_of(end);
    if (t.part >= t.parts) return false;
    t.k0 = t.part * per;
    t.k1 = min(end, t.k0 + per);
    return true;
}

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

// Parts of a tile of ROWS rows: [unit * KV + head][ROWS][D] sums, then [..][ROWS] pairs of reference maximum and sum.
template <int ROWS, int D>
struct Parts {
    float *sums, *state;
    __device__ Parts(const PagedArgs& a, int slot, int64_t slots) : sums(a.part + (int64_t)slot * ROWS * D), state(a.part + slots * ROWS * D + (int64_t)slot * ROWS * 2) {}
};

__device__ __forceinline__ void store_two(float* p, float x, float y) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), (uint64_t)__builtin_bit_cast(uint32_t, x) | (uint64_t)__builtin_bit_cast(uint32_t, y) << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ u32x2 load_two(const float* p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return u32x2{(uint32_t)v, (uint32_t)(v >> 32)};
}

// By the last workgroup of a tile: its parts put together in order; part i is at slot `slot0` + `apart` i, from the second on `shift` further.
template <typename T, int ROWS, int D, int THREADS>
__device__ __forceinline__ void join(const PagedArgs& a, const Task& t, int head, int slot0, int apart, int shift, int64_t slots) {
    constexpr int kFours = D / 4;
    const int rows = min(ROWS, t.tokens * a.G - t.tile * ROWS);
    // AHEAD parts are asked for at once: up to 16 of them arrive after one latency
    auto put = [&](auto ahead) __attribute__((always_inline)) {
        constexpr int AHEAD = decltype(ahead)::value;
        for (int idx = threadIdx.x; idx < rows * kFours; idx += THREADS) {
            const int row = idx / kFours, four = idx % kFours;
            float m = -INFINITY, l = 0.f;
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
            for (int p0 = 0; p0 < t.parts; p0 += AHEAD) {
                u32x2 st[AHEAD];
                f32x4 v[AHEAD];
#pragma unroll
                for (int p = 0; p < AHEAD; p++) {
                    const int q = min(p0 + p, t.parts - 1);
                    const Parts<ROWS, D> at(a, slot0 + q * apart + (q ? shift : 0), slots);
                    st[p] = load_two(at.state + 2 * row);
                    v[p] = load_part(parts_rsrc(at.sums), (uint32_t)((row * kFours + four) * 16));
                }
                float top = m;
#pragma unroll
                for (int p = 0; p < AHEAD; p++) top = fmaxf(top, p0 + p < t.parts ? __builtin_bit_cast(float, (uint32_t)st[p].x) : -INFINITY);
                const float use = top == -INFINITY ? 0.f : top, old = weight(m, use);
                m = top;
                l *= old;
                o *= old;
#pragma unroll
                for (int p = 0; p < AHEAD; p++) {
                    const float al = p0 + p < t.parts ? weight(__builtin_bit_cast(float, (uint32_t)st[p].x), use) : 0.f;
                    l = fmaf(__builtin_bit_cast(float, (uint32_t)st[p].y), al, l);
#pragma unroll
                    for (int e = 0; e < 4; e++) o[e] = fmaf(v[p][e], al, o[e]);
                }
            }
            const float inv = l != 0.f ? 1.f / l : 0.f;
            const int r = t.tile * ROWS + row;
            const int token = a.by_group(r);
            T* out = static_cast<T*>(a.o) + (int64_t)(t.first + token) * a.os[0] + (int64_t)(head * a.G + r - token * a.G) * a.os[1] + 4 * four;
            *reinterpret_cast<u32x2*>(out) = u32x2{Mfma32A<T>::pack2(o[0] * inv, o[1] * inv), Mfma32A<T>::pack2(o[2] * inv, o[3] * inv)};
        }
    };
    if (t.parts <= 4) put(std::integral_constant<int, 4>{});
    else if (t.parts <= 8 || ROWS > 32) put(std::integral_constant<int, 8>{});
    else put(std::integral_constant<int, 16>{});
}

// ---------------------------------------------------------------- few rows
// A wave takes blocks of 4 kLane keys of its own, kLane = 16 neighbouring ones (8 of a 16-bit cache) to each quarter of its lanes:
//   S^T = K Q^T    v_mfma_f32_16x16x32, kLane / 4 tiles j of sixteen keys: operand row i is key kLane (i / 4) + 4 j + i % 4, so that a lane of the result holds keys 4 j + r of its
//                  quarter's kLane, r = 0 .. 3.  Which of the elements of D a step takes from a lane does not matter as long as it takes the same from K and Q: a
//                  lane loads sixteen bytes of a key at a time, two steps' worth in 8 bits.
//   O^T += V^T P^T operand row = d; the eight keys that a lane holds of it in a step are neighbours in the cache's block, so that one load of sixteen bytes feeds two steps (one of a 16-bit cache), and
//                  they are those whose probabilities the lane has just computed.
// Two blocks are in registers or on their way; K of the next but one is asked for behind this one's scores, V behind its second product.
//
// The keys of the launch are one line of steps of 256 keys (more where there were over 2^29 of them): sequence by sequence, tile by tile, head by head.  Workgroup w takes the w-th share of the line, which may be a part of one
// head's keys, or the end of one, several whole ones and the beginning of another: every workgroup has the same to read, whatever the lengths.
constexpr int kStepShift = 8;

// Workgroups of a unit: what the registers allow, and what the launch counts on.
constexpr int rows_kernel_workgroups(int tiles, int64_t D) { return tiles == 1 ? 2 : (D <= 64 ? 2 : 1); }

// The line and its shares: the first `more` workgroups have per + 1 steps, the others per.
struct Line {
    int per, more;
    __device__ __forceinline__ int begin(int w) const { return w * per + min(w, more); }
    __device__ __forceinline__ int owner(int g) const { return g < more * (per + 1) ? g / (per + 1) : more + (g - more * (per + 1)) / per; }
};

template <typename T, int D, bool EIGHT, int TILES, int WAVES>
__global__ __launch_bounds__(64 * WAVES, rows_kernel_workgroups(TILES, D)) void paged_rows_kernel(PagedArgs a) {
    constexpr int ROWS = 16 * TILES, kLane = EIGHT ? 16 : 8, NT = kLane / 4, kKeys = 4 * kLane, kBlocks = kKeys / kBlock;
    constexpr int NS = D / 32, NF = D / 16, SIZE = EIGHT ? 1 : 2;
    constexpr int KD = D * SIZE / 16;                       // dwords of a key that a lane holds
    static_assert((1 << kStepShift) % (WAVES * kKeys) == 0, "a step is the same number of blocks for every wave");
    __shared__ __attribute__((aligned(16))) float sums[WAVES][TILES][NF][64][4];
    __shared__ float ml[2][WAVES][ROWS];
    __shared__ int last;
    // (read by scalar loads)
    typedef const __attribute__((address_space(4))) int32_t* uniform_words;
    auto scale_word = [](const uint8_t* scales, int at) __attribute__((always_inline)) { return (uint32_t)*(uniform_words)((uintptr_t)(scales + at) & ~(uintptr_t)3); };
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, lg = lane >> 4;

    // ---- this workgroup's share of the line.  A wave keeps the first 64 sequences in LDS
    __shared__ int known[WAVES][3][64];                                       // (a wave's own copy: nobody waits)
    auto tiles_of = [&](int tokens) __attribute__((always_inline)) { return (tokens * a.G + ROWS - 1) / ROWS; };
    auto steps_of = [&](int keys) __attribute__((always_inline)) { return max((keys + (1 << a.step_shift) - 1) >> a.step_shift, 1); };
    const int own_start = lane < a.s.B ? a.s.start(lane) : 0, own_tokens = lane < a.s.B ? a.s.tokens(lane) : 0, own_keys = lane < a.s.B ? a.s.keys(lane) : 0;
    known[wave][0][lane] = own_start;
    known[wave][1][lane] = own_tokens;
    known[wave][2][lane] = own_keys;
    int longest = own_tokens ? steps_of(own_keys) : 1, steps = own_tokens ? tiles_of(own_tokens) * steps_of(own_keys) : 0;
    for (int b = 64 + lane; b < a.s.B; b += 64)
        if (const int tokens = a.s.tokens(b)) {
            const int n = steps_of(a.s.keys(b));
            longest = max(longest, n);
            steps += tiles_of(tokens) * n;
        }
    longest = (int)wave_max((float)longest);                                  // of one sequence (exact: at most 2^16)
    steps = __builtin_amdgcn_readlane(wave_scan(steps), 63) * a.KV;           // of all heads
    Line line;
    line.per = a.by_shares(steps);
    line.more = steps - line.per * a.target;
    if (line.per < 1 || longest > (kMostParts - 1) * line.per) {
        line.per = (longest + kMostParts - 2) / (kMostParts - 1);
        line.more = 0;
    }
    int g = line.begin(blockIdx.x);
    const int stop = min(line.begin(blockIdx.x + 1), steps);
    const int page_bytes = (D * SIZE) << a.s.page_shift;

    for (int segment = 0; g < stop; segment++) {
        // ---- the head that step g belongs to
        int before, b, tokens, keys, first;
        {
            const int n = known[wave][1][lane], units = n ? tiles_of(n) * a.KV * steps_of(known[wave][2][lane]) : 0, sum = wave_scan(units);
            if (const uint64_t m = __ballot(sum > g)) {
                b = __builtin_ctzll(m);
                before = __builtin_amdgcn_readlane(sum - units, b);
                first = __builtin_amdgcn_readfirstlane(known[wave][0][b]);
                tokens = __builtin_amdgcn_readfirstlane(known[wave][1][b]);
                keys = __builtin_amdgcn_readfirstlane(known[wave][2][b]);
            } else {
                before = __builtin_amdgcn_readlane(sum, 63);
                int further;
                b = 64 + sequence_of(a.s.B - 64, g - before, [&](int i) { return a.s.tokens(64 + i) ? tiles_of(a.s.tokens(64 + i)) * a.KV * steps_of(a.s.keys(64 + i)) : 0; }, further);
                if (b < 64) return;
                before += further;
                first = __builtin_amdgcn_readfirstlane(a.s.start(b));
                tokens = __builtin_amdgcn_readfirstlane(a.s.tokens(b));
                keys = __builtin_amdgcn_readfirstlane(a.s.keys(b));
            }
        }
        if (g < before || g - before >= tiles_of(tokens) * a.KV * steps_of(keys)) return;     // (starts that are no starts: their sums may have wrapped)
        const int mine = steps_of(keys), pair = (g - before) / mine, s0 = g - before - pair * mine;
        if (!a.part && s0) {                                                  // without a workspace a head is its beginning's, whole
            g += mine - s0;
            continue;
        }
        const int s1 = a.part ? min(mine, s0 + stop - g) : mine;
        const int tile = a.by_heads(pair), head = pair - tile * a.KV, origin = g - s0;             // of the head on the line
        g += s1 - s0;
        const int rows = tokens * a.G;
        int end = keys;                                                       // of the keys that the tile's last row sees
        if (a.is_causal) end = max(keys - tokens + a.by_group(min((tile + 1) * ROWS, rows) - 1) + 1, 0);
        const int k0 = s0 << a.step_shift, k1 = min(end, s1 << a.step_shift);
        const bool split = s1 - s0 < mine;
        const int owner0 = split ? min(max(line.owner(origin), 0), (int)blockIdx.x) : 0;
        const int parts = split ? min(line.owner(origin + mine - 1) - owner0 + 1, min(kMostParts, (int)gridDim.x - owner0)) : 1;
        uint64_t* word = nullptr;
        uint64_t seen = 0;
        if (split) {
            // a split head begins in workgroup owner0 and is the only one to do so without ending there
            word = a.words + owner0;
            if (threadIdx.x == 0) seen = arrive_look(word);
        }

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
            const int row = tile * ROWS + 16 * x + li, token = a.by_group(row);
            const T* qp = static_cast<const T*>(a.q) + (int64_t)(first + token) * a.qs[0] + (int64_t)(head * a.G + row - token * a.G) * a.qs[1];
#pragma unroll
            for (int s = 0; s < NS; s++) qf[x][s] = row < rows ? *reinterpret_cast<const u32x4*>(qp + d_of(s)) : u32x4{0, 0, 0, 0};
            limit[x] = min(a.is_causal ? keys - tokens + token + 1 : keys, k1);
            open = min(open, row < rows ? limit[x] : k1);
        }
        open = -(int)wave_max((float)-open);

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
                if (EIGHT) {                                                    // the aligned words that hold the two bytes; taken apart where they are used, so that nothing waits for them here
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
        struct Block { uint32_t k[NT][KD], v[NF][4]; Place p; };
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
            blk.p = p;
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
#pragma unroll
        for (int x = 0; x < TILES; x++) {
            m_run[x] = -INFINITY;
            l_run[x] = 0.f;
#pragma unroll
            for (int f = 0; f < NF; f++) oacc[x][f] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        // the scale of this quarter's keys or values
        auto scale_at = [&](const Place& p, const uint32_t (&words)[kBlocks], const uint8_t* scales) __attribute__((always_inline)) {
            uint32_t bytes[kBlocks];
#pragma unroll
            for (int i = 0; i < kBlocks; i++) bytes[i] = max(words[i] >> 8 * ((uint32_t)(uintptr_t)(scales + p.page[i]) & 3) & 255, 1u) << 23;
            return __builtin_bit_cast(float, chosen(bytes, value_block));
        };
        // scores and probabilities of a block
        auto scored = [&](const Block& blk, int key, u32x4 (&pb)[TILES][NT / 2]) __attribute__((always_inline)) {
            const int at = key + kLane * lg;                                // first key of this quarter
            const bool masked = key + kKeys > open || blk.p.absent;
            const bool ok = !(blk.p.absent >> value_block & 1);
            const float c = EIGHT ? a.c * scale_at(blk.p, blk.p.ks, a.key_scales) : a.c;
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
                    for (int s = 0; s < NS; s++) s4 = Mfma16P<T>::run(kf[s], qf[x][s], s4);
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
                float lsum = 0.f;
#pragma unroll
                for (int e = 0; e < 4 * NT; e++) {
                    sv[x][e] = weight(sv[x][e], use);
                    lsum += sv[x][e];
                }
                l_run[x] = l_run[x] * alpha + lsum;
                if (__any(alpha != 1.f)) {
#pragma unroll
                    for (int f = 0; f < NF; f++) oacc[x][f] *= alpha;
                }
#pragma unroll
                for (int e = 0; e < 2 * NT; e++) pb[x][e >> 2][e & 3] = Mfma32A<T>::pack2(sv[x][2 * e], sv[x][2 * e + 1]);
            }
        };
        auto added = [&](Block& blk, int key, const u32x4 (&pb)[TILES][NT / 2], const Place& p) __attribute__((always_inline)) {
            if (key + kKeys > k1 || p.absent) {
                // values that no key of this part stands for may hold anything, a NaN among it
                const int n = p.absent >> value_block & 1 ? 0 : k1 - key - kLane * lg;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    constexpr int kPer = 4 / SIZE;
                    const int left = min(max(n - kPer * e, 0), kPer) * SIZE;
                    const uint32_t keep = left == 4 ? ~0u : (1u << (8 * left)) - 1;
#pragma unroll
                    for (int f = 0; f < NF; f++) blk.v[f][e] &= keep;
                }
            }
            const float vs = EIGHT ? scale_at(p, p.vs, a.value_scales) : 1.f;
#pragma unroll
            for (int f = 0; f < NF; f++)
#pragma unroll
                for (int h = 0; h < NT / 2; h++) {
                    u32x4 vf;
                    if constexpr (EIGHT) vf = widen<T>(u32x2{blk.v[f][2 * h], blk.v[f][2 * h + 1]}, vs);
                    else vf = u32x4{blk.v[f][0], blk.v[f][1], blk.v[f][2], blk.v[f][3]};
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
                const Place was = blk.p;
                if (next) load_k(blk, p);
                added(blk, key_of(i), pb, was);
                __builtin_amdgcn_sched_barrier(0);
                if (next) load_v(blk, p);
            };
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
        }

        if (split && threadIdx.x == 0) arrive_claim(word, seen, a.tag);
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
        const int here = min(ROWS, rows - tile * ROWS);
        // a workgroup leaves at most two parts: the end of a head that began in front of its share, and the beginning of one that ends behind it
        const Parts<ROWS, D> own(a, 2 * (int)blockIdx.x + (s0 ? 0 : 1), 2 * (int64_t)gridDim.x);
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
            if (!split) {
                const float inv = l != 0.f ? 1.f / l : 0.f;
                const int r = tile * ROWS + row, token = a.by_group(r);
                T* out = static_cast<T*>(a.o) + (int64_t)(first + token) * a.os[0] + (int64_t)(head * a.G + r - token * a.G) * a.os[1] + 4 * four;
                *reinterpret_cast<u32x2*>(out) = u32x2{Mfma32A<T>::pack2(o[0] * inv, o[1] * inv), Mfma32A<T>::pack2(o[2] * inv, o[3] * inv)};
            } else {
                store_part(parts_rsrc(own.sums), (uint32_t)(idx * 16), o);
                if (four == 0) store_two(own.state + 2 * row, m, l);
            }
        }
        if (!split || !arrive_last(word, parts, &last)) continue;
        const Task t{b, tile, 0, parts, 0, 0, first, tokens, keys};
        join<T, ROWS, D, 64 * WAVES>(a, t, head, 2 * owner0 + 1, 2, -1, 2 * (int64_t)gridDim.x);
    }
}

// ---------------------------------------------------------------- many rows
// 128 rows, 32 a wave, over stages of 64 keys that lie in LDS in the queries' type, two of them: the next one is on its way in registers and is converted and put down
// behind this one's products.
//   S^T = K Q^T     v_mfma_f32_32x32x16: operand row i of tile j is key 32 j + 16 (r / 8) + 8 h + r % 8 where register r of half h of the result is row i, so that
//   O^T += V^T P^T  a half's eight registers of a step are the probabilities of eight neighbouring keys: sixteen bytes of a row of V^T.
constexpr int kTileRows = 128, kStage = 64;

template <int D>
__device__ __forceinline__ uint32_t tk_off(int key, int chunk) {          // K [64][D]: chunks of eight elements, rotated by the key
    constexpr int kMask = D >= 128 ? 15 : D >= 64 ? 7 : 3;
    if constexpr (D == 96) return (uint32_t)(key * 208 + chunk * 16);     // (twelve chunks: a row of thirteen instead)
    else return (uint32_t)(key * (D * 2) + ((chunk ^ ((D == 128 ? key : D == 64 ? key >> 1 : key >> 2) & kMask)) << 4));
}
__device__ __forceinline__ uint32_t tv_off(int d, int chunk) {            // V^T [D][64]
    return (uint32_t)(d * 128 + ((chunk ^ ((d >> 1) & 7)) << 4));
}

template <typename T, int D, bool EIGHT>
__global__ __launch_bounds__(256, 2) void paged_tile_kernel(PagedArgs a) {
    constexpr int NS = D / 16, NF = D / 32, SIZE = EIGHT ? 1 : 2;
    constexpr int kKBytes = D == 96 ? 64 * 208 : 64 * D * 2, kVBytes = D * 128;
    constexpr int kPieces = 64 * D * SIZE / 16, kMine = (kPieces + 255) / 256;      // pieces of sixteen bytes of K, and of V, of a stage; a thread's
    __shared__ __attribute__((aligned(16))) char lds[2][kKBytes + kVBytes];
    __shared__ int last;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 31, lh = lane >> 5;
    const int unit = a.by_heads(blockIdx.x), head = blockIdx.x - unit * a.KV;
    Task t;
    if (!task_of<kTileRows, kStage>(a, unit, t)) return;
    const int slot0 = (unit - t.part) * a.KV + head;
    uint64_t seen = 0;
    if (t.parts > 1 && threadIdx.x == 0) seen = arrive_look(a.words + slot0);

    const int rows = t.tokens * a.G, row = t.tile * kTileRows + 32 * wave + li, token = a.by_group(row);
    u32x4 qf[NS];
    {
        const T* qp = static_cast<const T*>(a.q) + (int64_t)(t.first + token) * a.qs[0] + (int64_t)(head * a.G + row - token * a.G) * a.qs[1];
#pragma unroll
        for (int s = 0; s < NS; s++) qf[s] = row < rows ? *reinterpret_cast<const u32x4*>(qp + 16 * s + 8 * lh) : u32x4{0, 0, 0, 0};
    }
    const int limit = row < rows ? min(a.is_causal ? t.keys - t.tokens + token + 1 : t.keys, t.k1) : 0;
    const int open = -(int)wave_max((float)-(row < rows ? limit : t.k1));            // blocks in front of it need no mask
    const int seen_keys = (int)wave_max((float)limit);                               // blocks behind it concern no row of the wave

    const int32_t* table = a.s.table + (int64_t)t.b * a.s.width;
    const int page = 1 << a.s.page_shift;
    // piece i of a thread: K: key and piece of its row; V: a d's keys of a block (EIGHT), or half of them
    constexpr int kKeyPieces = D * SIZE / 16;
    struct Stage { u32x4 k[kMine], v[kMine]; float ks[kMine], vs[kMine]; bool ok[kMine]; };
    struct Pages { int k[kMine], v[kMine]; bool v_ok[kMine]; };
    auto ask = [&](Pages& p, int key) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kMine; i++) {
            const int idx = threadIdx.x + 256 * i;
            bool ok;
            p.k[i] = page_of(a, table, (key + idx / kKeyPieces) >> 4, ok);
            p.v[i] = page_of(a, table, (key >> 4) + idx / (D * SIZE), p.v_ok[i]);
        }
    };
    auto load = [&](Stage& st, const Pages& p, int key) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kMine; i++) {
            const int idx = threadIdx.x + 256 * i;
            if (kPieces % 256 && idx >= kPieces) continue;
            const int kk = (key + idx / kKeyPieces) & (page - 1);
            const int64_t kh = (int64_t)p.k[i] * a.KV + head, vh = (int64_t)p.v[i] * a.KV + head;
            st.k[i] = *reinterpret_cast<const u32x4*>(a.keys + (kh * page + kk) * (D * SIZE) + idx % kKeyPieces * 16);
            const int vb = ((key >> 4) + idx / (D * SIZE)) & ((page >> 4) - 1);
            st.v[i] = *reinterpret_cast<const u32x4*>(a.values + ((vh << (a.s.page_shift - 4)) + vb) * (D * 16 * SIZE) + idx % (D * SIZE) * 16);
            st.ok[i] = p.v_ok[i];
            if (EIGHT) {
                st.ks[i] = scale_of(a.key_scales[kh]);
                st.vs[i] = scale_of(a.value_scales[vh]);
            }
        }
    };
    auto put = [&](Stage& st, int key, char* to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kMine; i++) {
            const int idx = threadIdx.x + 256 * i;
            if (kPieces % 256 && idx >= kPieces) continue;
            const int k = idx / kKeyPieces, kc = idx % kKeyPieces;
            const int block = idx / (D * SIZE), d = idx % (D * SIZE) / SIZE, half = EIGHT ? 0 : idx & 1;
            // values that no key of this part stands for may hold anything, a NaN among it
            const int n = st.ok[i] ? t.k1 - key - 16 * block - 8 * half : 0;
            if (n < 16 / SIZE) {
                constexpr int kPer = 4 / SIZE;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int left = min(max(n - kPer * e, 0), kPer) * SIZE;
                    st.v[i][e] &= left == 4 ? ~0u : (1u << (8 * left)) - 1;
                }
            }
            char* tk = to;
            char* tv = to + kKBytes;
            if constexpr (EIGHT) {
                *reinterpret_cast<u32x4*>(tk + tk_off<D>(k, 2 * kc)) = widen<T>(u32x2{st.k[i].x, st.k[i].y}, st.ks[i]);
                *reinterpret_cast<u32x4*>(tk + tk_off<D>(k, 2 * kc + 1)) = widen<T>(u32x2{st.k[i].z, st.k[i].w}, st.ks[i]);
                *reinterpret_cast<u32x4*>(tv + tv_off(d, 2 * block)) = widen<T>(u32x2{st.v[i].x, st.v[i].y}, st.vs[i]);
                *reinterpret_cast<u32x4*>(tv + tv_off(d, 2 * block + 1)) = widen<T>(u32x2{st.v[i].z, st.v[i].w}, st.vs[i]);
            } else {
                *reinterpret_cast<u32x4*>(tk + tk_off<D>(k, kc)) = st.k[i];
                *reinterpret_cast<u32x4*>(tv + tv_off(d, 2 * block + half)) = st.v[i];
            }
        }
    };

    f32x16 oacc[NF];
#pragma unroll
    for (int f = 0; f < NF; f++) oacc[f] = f32x16{};
    float m_run = -INFINITY, l_run = 0.f;
    // row li of a tile of S^T is key `of` of its 32
    const int of = 16 * (li >> 4) + 8 * ((li >> 2) & 1) + 4 * ((li >> 3) & 1) + (li & 3);

    auto attend = [&](const char* from, int key, uint32_t absent) __attribute__((always_inline)) {
        f32x16 sv[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            sv[j] = f32x16{};
#pragma unroll
            for (int s = 0; s < NS; s++)
                sv[j] = Mfma32A<T>::run(*reinterpret_cast<const u32x4*>(from + tk_off<D>(32 * j + of, 2 * s + lh)), qf[s], sv[j]);
        }
        float top = -INFINITY;
        if (key + kStage > open || absent) {
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int at = 32 * j + 16 * (r >> 3) + 8 * lh + (r & 7);
                    const bool in = key + at < limit && !(absent >> (2 * j + (r >> 3)) & 1);
                    sv[j][r] = in ? sv[j][r] * a.c : -INFINITY;
                    top = fmaxf(top, sv[j][r]);
                }
        } else {
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    sv[j][r] *= a.c;
                    top = fmaxf(top, sv[j][r]);
                }
        }
        top = half_max(top);
        const float m_new = moved_reference(m_run, top), use = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = weight(m_run, use);
        m_run = m_new;
        float lsum = 0.f;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                sv[j][r] = weight(sv[j][r], use);
                lsum += sv[j][r];
            }
        l_run = l_run * alpha + lsum;
        if (__any(alpha != 1.f)) {
#pragma unroll
            for (int f = 0; f < NF; f++) oacc[f] *= alpha;
        }
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            u32x4 pb;
#pragma unroll
            for (int e = 0; e < 4; e++) pb[e] = Mfma32A<T>::pack2(sv[ks >> 1][8 * (ks & 1) + 2 * e], sv[ks >> 1][8 * (ks & 1) + 2 * e + 1]);
#pragma unroll
            for (int f = 0; f < NF; f++)
                oacc[f] = Mfma32A<T>::run(*reinterpret_cast<const u32x4*>(from + kKBytes + tv_off(32 * f + li, 2 * ks + lh)), pb, oacc[f]);
        }
    };

    if (t.k0 < t.k1) {
        Pages pg;
        Stage st;
        ask(pg, t.k0);
        load(st, pg, t.k0);
        ask(pg, t.k0 + kStage);
        put(st, t.k0, lds[0]);
        __syncthreads();
        int at = 0;
        for (int key = t.k0; key < t.k1; key += kStage) {
            const bool more = key + kStage < t.k1;
            if (more) {
                load(st, pg, key + kStage);
                ask(pg, key + 2 * kStage);
            }
            if (key < seen_keys) {
                // blocks of sixteen keys whose page the table does not name
                uint32_t absent = 0;
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    bool ok;
                    page_of(a, table, (key >> 4) + n, ok);
                    absent |= (ok ? 0u : 1u) << n;
                }
                attend(lds[at], key, absent);
            }
            if (more) put(st, key + kStage, lds[at ^ 1]);
            __syncthreads();
            at ^= 1;
        }
    }

    l_run = half_sum(l_run);
    const int64_t slots = gridDim.x;
    if (t.parts == 1) {
        if (row < rows) {
            const float inv = l_run != 0.f ? 1.f / l_run : 0.f;
            T* out = static_cast<T*>(a.o) + (int64_t)(t.first + token) * a.os[0] + (int64_t)(head * a.G + row - token * a.G) * a.os[1] + 4 * lh;
#pragma unroll
            for (int f = 0; f < NF; f++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    *reinterpret_cast<u32x2*>(out + 32 * f + 8 * g) =
                        u32x2{Mfma32A<T>::pack2(oacc[f][4 * g] * inv, oacc[f][4 * g + 1] * inv), Mfma32A<T>::pack2(oacc[f][4 * g + 2] * inv, oacc[f][4 * g + 3] * inv)};
        }
        return;
    }
    if (threadIdx.x == 0) arrive_claim(a.words + slot0, seen, a.tag);
    const Parts<kTileRows, D> own(a, slot0 + t.part * a.KV, slots);
    if (row < rows) {
        const __amdgpu_buffer_rsrc_t rs = parts_rsrc(own.sums);
        const int r = 32 * wave + li;
#pragma unroll
        for (int f = 0; f < NF; f++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                store_part(rs, (uint32_t)((r * D + 32 * f + 8 * g + 4 * lh) * 4), f32x4{oacc[f][4 * g], oacc[f][4 * g + 1], oacc[f][4 * g + 2], oacc[f][4 * g + 3]});
        if (lh == 0) store_two(own.state + 2 * r, m_run, l_run);
    }
    if (!arrive_last(a.words + slot0, t.parts, &last)) return;
    join<T, kTileRows, D, 256>(a, t, head, slot0, a.KV, 0, slots);
}

// The launch that serves these sizes: rows of a workgroup's tile, workgroups that share the work (few rows) or that parts are meant to fill, the grid, and the places for parts and counts.
struct Plan { int rows, target; int64_t grid, slots, words; int step_shift; };

Plan plan_of(const mhip_paged_cache* c, const mhip_sequences* s, int64_t q_heads) {
    const int64_t G = q_heads / c->heads, average = (s->tokens + s->sequences - 1) / s->sequences * G;
    const int rows = average <= 16 ? 16 : average <= 32 ? 32 : kTileRows;
    if (rows != kTileRows) {
        const int target = rows_kernel_workgroups(rows / 16, c->head_size) * compute_units();
        // (more keys a step where the line could have more than 2^29 steps)
        const double tiles = (double)(s->tokens * G / rows + s->sequences) * c->heads;
        int shift = kStepShift;
        while (tiles * (double)((s->width * c->page_size >> shift) + 1) > (double)(1 << 29)) shift++;
        return {rows, target, target, 2 * target, target, shift};
    }
    const int target = 2 * compute_units();
    const int64_t units = s->tokens * G / rows + (s->sequences < s->tokens ? s->sequences : s->tokens) + target / c->heads + 1;
    return {rows, target, units * c->heads, units * c->heads, units * c->heads, 0};
}

int64_t workspace_of(const mhip_paged_cache* c, const Plan& p) { return p.slots * p.rows * (c->head_size + 2) * 4 + p.words * 8; }

template <typename T, int D, bool EIGHT>
int launch(hipStream_t st, const PagedArgs& a, const Plan& p) {
    const dim3 grid((unsigned)p.grid);
    if (p.rows == 16) hipLaunchKernelGGL((paged_rows_kernel<T, D, EIGHT, 1, 4>), grid, dim3(256), 0, st, a);
    else if (p.rows == 32) hipLaunchKernelGGL((paged_rows_kernel<T, D, EIGHT, 2, 4>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_tile_kernel<T, D, EIGHT>), grid, dim3(256), 0, st, a);
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
    if (!cache || !seqs || cache->heads <= 0 || q_heads <= 0 || q_heads % cache->heads || seqs->sequences <= 0 || seqs->tokens <= 0) return 0;
    return workspace_of(cache, plan_of(cache, seqs, q_heads));
}

extern "C" int mhip_paged_attention(void* stream, const mhip_paged_cache* cache, const mhip_sequences* seqs, const void* q, void* o, int64_t q_heads, float scale,
                                    int is_causal, const int64_t* strides, int dtype, void* workspace, int64_t workspace_bytes) {
    bool empty;
    if (const int rc = check_paged("paged_attention", cache, seqs, dtype, &empty)) return rc;
    if (q_heads <= 0 || q_heads % cache->heads) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_attention: %lld query heads over %lld key heads", (long long)q_heads, (long long)cache->heads);
    if (empty) return MHIP_OK;
    if (!q || !o || !strides) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_attention: NULL tensor");
    if (((uintptr_t)q | (uintptr_t)o | (uintptr_t)workspace) & 15) return fail(MHIP_ERR_UNSUPPORTED, "paged_attention: tensors must be 16-byte aligned");
    for (int i = 0; i < 4; i++)
        if (strides[i] % 8) return fail(MHIP_ERR_UNSUPPORTED, "paged_attention: strides must be multiples of 8 elements");
    if (seqs->tokens * (q_heads / cache->heads) >= 1 << 30) return fail(MHIP_ERR_UNSUPPORTED, "paged_attention: more than 2^30 rows");
    const Plan p = plan_of(cache, seqs, q_heads);
    if (p.grid >= 1 << 30) return fail(MHIP_ERR_UNSUPPORTED, "paged_attention: more workgroups than a launch has");
    PagedArgs a{q, o, (const char*)cache->keys, (const char*)cache->values, cache->key_scales, cache->value_scales, sequences(cache, seqs),
                (int)cache->pages, (int)cache->heads, (int)(q_heads / cache->heads), is_causal ? 1 : 0, p.target, scale * kLog2e, {strides[0], strides[1]}, {strides[2], strides[3]},
                nullptr, nullptr, 0, Divider((uint32_t)(q_heads / cache->heads)), Divider((uint32_t)cache->heads), Divider((uint32_t)p.target), p.step_shift};
    if (workspace && workspace_bytes >= workspace_of(cache, p)) {
        a.part = static_cast<float*>(workspace);
        a.words = reinterpret_cast<uint64_t*>(a.part + p.slots * p.rows * (cache->head_size + 2));
        a.tag = launch_tag();
    }
    hipStream_t st = as_stream(stream);
    const bool eight = cache->key_scales != nullptr;
    const int64_t D = cache->head_size;
    if (dtype == MHIP_BF16) return eight ? launch_d<bf16_t, true>(st, a, p, D) : launch_d<bf16_t, false>(st, a, p, D);
    return eight ? launch_d<f16_t, true>(st, a, p, D) : launch_d<f16_t, false>(st, a, p, D);
}
