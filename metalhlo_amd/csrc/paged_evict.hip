// Eviction from a paged cache (paged.h): of each sequence and head the last `recent` keys stay, and of those in front of them the `keep` whose weight (paged_weighed.hip adds it up) is greatest; they
// move to the front in their order, keys, values and weights, and the pages behind are free.
//
//   select   evict_select_kernel, a workgroup a sequence and head: the keep-th greatest weight by its bits, eleven at a time (a histogram of those that agree with it so far), then the positions of what
//            stays in order, of equal weights the first ones.  Weights compare as numbers, NaN above all.
//   move     evict_move_kernel, 256 places of a sequence and head at a time.  Keys are rows of bytes; a block holds sixteen tokens of a d, so that values change places in registers.  In 8 bits a page takes
//            the greatest scale of those its keys come from, under which the others are rounded anew.
//
// us: 32 sequences of 2800 to 4000 keys, 8 heads of 128 in 8 bits, cut to 1750 (235 MB) 80: move 67, select 14; two of up to 50000 keys, 8 heads of 96 in 16 bits, cut to 8500 in place (107 MB) 119: select 65, which is
// 16 workgroups' whole work, gather 53, copy 23.  The move is one round of workgroups, each of which waits for place -> page -> block four times over.
//
// A key never moves backwards, so that where it lies and where it goes are the same pages a workgroup moves a sequence and head from the front on, each step read before it is written (IN_PLACE).
// That is one compute unit's bandwidth a head: few heads are gathered into the workspace instead, by the whole device, and copied back.
#include <algorithm>

#include "paged.h"

namespace mhip {
namespace {

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64, kBins = 2048;
constexpr int kWindow = 256;              // places that a workgroup moves at a time: whole pages

struct SelectArgs {
    const float* weights;
    const int32_t *table, *lengths;
    int32_t *list, *left;                 // [B, KV, cap] positions, [B] kept
    int width, pages, KV, page_shift, keep, recent;
    int64_t cap;
};

// numbers in the order of these, -0 and 0 alike, NaN above all; 0 is none of them
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);
    return x != x ? 0xFFFFFFFFu : u >> 31 ? ~u : u | 0x80000000u;
}

// PER: sixty-fours of positions of a wave, whose weights it keeps in registers (no more than the table reaches, a sixteenth of it a wave); LDS: as many more that lie there; PER 0: they are read again for each pass.
// us, two sequences of 50000 positions and 8 heads, read again | kept: 114 | 65; 32 sequences of 2800 to 4000 19 | 14.
template <int PER, int LDS>
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(SelectArgs a) {
    __shared__ uint32_t more[LDS ? LDS * kSelectThreads : 1];
    __shared__ int bins[kBins];
    __shared__ int found[2];                                                // the bin that the keep-th lies in; how many lie above it
    __shared__ int sure[kSelectWaves], ties[kSelectWaves];
    const int b = blockIdx.x / a.KV, h = blockIdx.x - b * a.KV;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = min(max(a.lengths[b], 0), a.width << a.page_shift), first = max(n - a.recent, 0);
    const int32_t* table = a.table + (int64_t)b * a.width;
    const int mask = (1 << a.page_shift) - 1;
    // a wave a stretch of positions, sixty-four at a time
    const int per = (n + 64 * kSelectWaves - 1) / (64 * kSelectWaves), p0 = wave * per * 64;
    // 0 where the table names no page
    auto key_at = [&](int pos) __attribute__((always_inline)) {
        const int page = table[pos >> a.page_shift];
        return (uint32_t)page < (uint32_t)a.pages ? ordered(a.weights[(((int64_t)page * a.KV + h) << a.page_shift) + (pos & mask)]) : 0u;
    };
    uint32_t kept[PER ? PER : 1];
    if constexpr (PER > 0) {
        // (all pages are asked for, and then all weights)
        auto fill = [&](int base) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int pos = p0 + 64 * (base + i) + lane;
                kept[i] = base + i < per && pos < n ? (uint32_t)table[pos >> a.page_shift] : 0xFFFFFFFFu;
            }
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int pos = p0 + 64 * (base + i) + lane;
                const bool there = kept[i] < (uint32_t)a.pages;
                float w = 0.f;
                if (there) w = a.weights[(((int64_t)kept[i] * a.KV + h) << a.page_shift) + (pos & mask)];
                kept[i] = there ? ordered(w) : 0u;
            }
        };
        if constexpr (LDS > 0) {
            fill(PER);
#pragma unroll
            for (int i = 0; i < LDS; i++) more[i * kSelectThreads + threadIdx.x] = kept[i];
        }
        fill(0);
    }
    // f(position, key) for a wave's positions, in order, all lanes at a time (key 0 behind the last)
    auto each = [&](auto f) __attribute__((always_inline)) {
        if constexpr (PER > 0) {
#pragma unroll
            for (int i = 0; i < PER; i++)
                if (i < per) f(p0 + 64 * i + lane, kept[i]);
            if constexpr (LDS > 0)
                for (int i = PER; i < per; i++) f(p0 + 64 * i + lane, more[(i - PER) * kSelectThreads + threadIdx.x]);
        } else {
            for (int i = 0; i < per; i++) {
                const int pos = p0 + 64 * i + lane;
                f(pos, pos < n ? key_at(pos) : 0u);
            }
        }
    };

    // ---- the keep-th greatest: `known` are its upper bits, `wanted` its place among those that have them
    uint32_t known = 0;
    int wanted = a.keep;
    bool all = first <= a.keep;                                             // all in front stay
    for (int pass = 0; pass < 3 && !all && a.keep > 0; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, count = pass == 2 ? 1024 : 2048, above = pass == 1 ? 21 : 10;
        for (int i = threadIdx.x; i < kBins; i += kSelectThreads) bins[i] = 0;
        __syncthreads();
        each([&](int pos, uint32_t key) __attribute__((always_inline)) {
            if (key && pos < first && (pass == 0 || key >> above == known >> above)) atomicAdd(&bins[(key >> shift) & (count - 1)], 1);
        });
        __syncthreads();
        if (wave == 0) {
            // lane l has the l-th of 64 stretches from the top
            const int stretch = count / 64;
            int mine = 0;
            for (int i = 0; i < stretch; i++) mine += bins[count - 1 - (lane * stretch + i)];
            const int upto = wave_scan(mine);
            const uint64_t m = __ballot(upto >= wanted);
            if (!m) {
                if (lane == 0) found[0] = -1;                               // (fewer than `keep` have a page)
            } else if (lane == __builtin_ctzll(m)) {
                int over = upto - mine, i = 0;
                while (over + bins[count - 1 - (lane * stretch + i)] < wanted) over += bins[count - 1 - (lane * stretch + i++)];
                found[0] = count - 1 - (lane * stretch + i);
                found[1] = over;
            }
        }
        __syncthreads();
        if (found[0] < 0) all = true;
        else {
            known |= (uint32_t)found[0] << shift;
            wanted -= found[1];
        }
        __syncthreads();
    }
    // what stays: keys above `border`, the first `wanted` that equal it, and the last ones
    const uint32_t border = all ? 0u : a.keep > 0 ? known : 0xFFFFFFFFu;
    if (all || a.keep == 0) wanted = 0;

    // ---- counted, then written
    auto is_sure = [&](int pos, uint32_t key) __attribute__((always_inline)) { return key && (pos >= first || key > border); };
    auto is_tie = [&](int pos, uint32_t key) __attribute__((always_inline)) { return key && pos < first && key == border && wanted > 0; };
    int n_sure = 0, n_ties = 0;
    each([&](int pos, uint32_t key) __attribute__((always_inline)) {
        n_sure += __builtin_popcountll(__ballot(is_sure(pos, key)));
        n_ties += __builtin_popcountll(__ballot(is_tie(pos, key)));
    });
    if (lane == 0) { sure[wave] = n_sure; ties[wave] = n_ties; }
    __syncthreads();
    int at = 0, tied = 0, total = 0, total_ties = 0;
    for (int w = 0; w < kSelectWaves; w++) {
        if (w == wave) { at = total; tied = total_ties; }
        total += sure[w];
        total_ties += ties[w];
    }
    at += min(tied, wanted);
    total += min(total_ties, wanted);
    if (h == 0 && threadIdx.x == 0) a.left[b] = total;
    int32_t* list = a.list + (int64_t)blockIdx.x * a.cap;
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    each([&](int pos, uint32_t key) __attribute__((always_inline)) {
        const bool tie = is_tie(pos, key);
        const uint64_t tie_mask = __ballot(tie);
        const bool stays = is_sure(pos, key) || (tie && tied + __builtin_popcountll(tie_mask & below) < wanted);
        const uint64_t m = __ballot(stays);
        if (stays) list[at + __builtin_popcountll(m & below)] = pos;
        at += __builtin_popcountll(m);
        tied += __builtin_popcountll(tie_mask);
    });
}

// A cache and the pages that sequences have in it; without a table sequence b has pages b * width + 0 .. width - 1.
struct Pool {
    char *keys, *values;
    uint8_t *key_scales, *value_scales;
    float* weights;
    const int32_t* table;
    int width, pages;
    // page `j` of sequence b, -1 for none
    __device__ __forceinline__ int page(int b, int j) const {
        if (j >= width) return -1;
        const int p = table ? table[(int64_t)b * width + j] : b * width + j;
        return (uint32_t)p < (uint32_t)pages ? p : -1;
    }
};

struct MoveArgs {
    Pool from, to;
    const int32_t *list, *left;           // positions [B, KV, cap], NULL: as they lie; keys of each sequence
    int KV, page_shift, windows;
    int64_t cap;
};

template <int D, int SIZE, bool LISTED, bool IN_PLACE>
__global__ __launch_bounds__(kWindow) void evict_move_kernel(MoveArgs a) {
    constexpr int kPer = D * SIZE / 16;                                     // pieces of sixteen bytes of a key
    constexpr bool EIGHT = SIZE == 1;
    __shared__ int from_row[kWindow], to_row[kWindow / kBlock];             // page * KV + head, -1 for none
    __shared__ int from_slot[kWindow];
    __shared__ int scale[2][kWindow], top[2][kWindow / kBlock];              // of keys and of values
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int unit = IN_PLACE ? blockIdx.x : blockIdx.x / a.windows, b = unit / a.KV, h = unit - b * a.KV;
    const int count = (int)min((int64_t)a.left[b], a.cap), mask = (1 << a.page_shift) - 1;
    for (int w = IN_PLACE ? 0 : blockIdx.x - unit * a.windows; w * kWindow < count; w++) {
        const int i = w * kWindow + t;
        // ---- where the places' keys come from
        if (IN_PLACE) __syncthreads();                                      // (the window before is done)
        if (t < 2 * (kWindow / kBlock)) top[t & 1][t >> 1] = 0;
        int row = -1, slot = 0, to = -1;
        if (i < count) {
            const int src = LISTED ? a.list[(int64_t)unit * a.cap + i] : i, page = a.from.page(b, src >> a.page_shift), into = a.to.page(b, i >> a.page_shift);
            slot = src & mask;
            row = page < 0 ? -1 : page * a.KV + h;
            to = into < 0 ? -1 : into * a.KV + h;
        }
        from_row[t] = row;
        from_slot[t] = slot;
        if ((t & (kBlock - 1)) == 0) to_row[t / kBlock] = to;
        float weight = 0.f;
        if (row >= 0) weight = a.from.weights[((int64_t)row << a.page_shift) + slot];
        if (EIGHT) {
            scale[0][t] = row >= 0 ? a.from.key_scales[row] : 0;
            scale[1][t] = row >= 0 ? a.from.value_scales[row] : 0;
            __syncthreads();
            atomicMax(&top[0][t >> a.page_shift], scale[0][t]);
            atomicMax(&top[1][t >> a.page_shift], scale[1][t]);
        }
        __syncthreads();
        auto settled = [&]() __attribute__((always_inline)) {
            if constexpr (IN_PLACE) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
            }
        };
        // 2^n that token `at`'s keys or values take
        auto factor = [&](int which, int at) __attribute__((always_inline)) {
            const int e = 127 + max(scale[which][at], 1) - max(top[which][at >> a.page_shift], 1);
            return e > 0 ? __builtin_bit_cast(float, (uint32_t)e << 23) : 0.f;
        };
        const int here = min(count - w * kWindow, kWindow);
        if (IN_PLACE) settled();
        if (row >= 0 && to >= 0) a.to.weights[((int64_t)to << a.page_shift) + (i & mask)] = weight;

        // ---- keys, a piece of sixteen bytes a thread, so many turns at once
        constexpr int kTurn = 4;                                            // (us, 32 sequences, two | four | eight: 82.5 | 81 | 119)
        for (int p0 = 0; p0 < here * kPer; p0 += kTurn * kWindow) {
            // (where a piece goes, -1 for none, is formed once and decides about the load and about the store)
            u32x4 v[kTurn];
            int token[kTurn], into[kTurn];
#pragma unroll
            for (int j = 0; j < kTurn; j++) {
                const int p = p0 + j * kWindow + t;
                token[j] = min(p / kPer, kWindow - 1);
                const int source = from_row[token[j]];
                into[j] = p < here * kPer && source >= 0 ? to_row[token[j] / kBlock] : -1;
                v[j] = u32x4{0, 0, 0, 0};
                if (into[j] >= 0) v[j] = *reinterpret_cast<const u32x4*>(a.from.keys + ((((int64_t)source << a.page_shift) + from_slot[token[j]]) * kPer + p % kPer) * 16);
            }
            settled();
#pragma unroll
            for (int j = 0; j < kTurn; j++) {
                if (into[j] < 0) continue;
                const int p = p0 + j * kWindow + t, at = (w * kWindow + token[j]) & mask;
                if constexpr (EIGHT) {
                    const float f = factor(0, token[j]);
                    if (f != 1.f)
#pragma unroll
                        for (int e = 0; e < 4; e++) v[j][e] = moved8(v[j][e], f);
                }
                *reinterpret_cast<u32x4*>(a.to.keys + ((((int64_t)into[j] << a.page_shift) + at) * kPer + p % kPer) * 16) = v[j];
            }
        }
        // ---- values: a wave sixteen places, a lane a d of them or two.  Their tokens come from a few blocks, whose sixteen tokens of a d are sixteen neighbouring numbers: four blocks are asked for at a
        // time, and numbers change places in registers.  (32 sequences of 3400 keys cut to 1750: a load for each number 120 us, a block's numbers in one go but block after block 105, four blocks 81; numbers that are rounded anew four in a word and not one by one, 73; bytes put in their place by one instruction, 67.)
        constexpr int kHalves = (D + 63) / 64, kFrom = 4, kWords = 4 * SIZE, kPerWord = 4 / SIZE;
        typedef uint32_t Words __attribute__((ext_vector_type(kFrom * kWords)));
        for (int block0 = 0; block0 * kBlock < here; block0 += kWindow / 64) {
            const int block = block0 + wave, into = block * kBlock < here ? to_row[block] : -1;       // (sixteen blocks a window, four a turn)
            uint32_t v[kHalves][kWords] = {};
            uint32_t held = 0;                                              // bit e: token e has a value
            if (into >= 0) {
                const int r = from_row[block * kBlock + (lane & 15)], s = from_slot[block * kBlock + (lane & 15)];
                const int r1 = __shfl_up(r, 1, 64), s1 = __shfl_up(s, 1, 64);
                held = (uint32_t)__ballot(r >= 0) & 0xFFFFu;
                const uint32_t begins = (uint32_t)__ballot(r >= 0 && ((lane & 15) == 0 || r != r1 || s >> 4 != s1 >> 4)) & 0xFFFFu;      // tokens that are the first of their block
                // of token e in lane e: the word of its block's that it lies in, counted over all blocks (behind them for none), and which bytes of that and of the word it goes to make the latter
                const int order = __builtin_popcount(begins & ((2u << (lane & 15)) - 1)) - 1;
                const uint32_t one = (uint32_t)(s % kPerWord * SIZE) + 4, place = (uint32_t)(lane % kPerWord) * (8 * SIZE);
                const int words = r >= 0 ? order * kWords + (s & 15) / kPerWord : kBlock * kWords;
                const uint32_t bytes = EIGHT ? (0x03020100u & ~(0xFFu << place)) | one << place : (0x03020100u & ~(0xFFFFu << place)) | (one | (one + 1) << 8) << place;
                uint32_t left = begins;
                for (int base = 0; left; base += kFrom) {
                    Words from[kHalves];
#pragma unroll
                    for (int j = 0; j < kFrom; j++) {
                        const int e = left ? __builtin_ctz(left) : __builtin_ctz(begins);            // (none left: the first again)
                        left &= left - 1;
                        const int row = __builtin_amdgcn_readlane(r, e), slot = __builtin_amdgcn_readlane(s, e);
                        const char* at = a.from.values + (((int64_t)row << (a.page_shift - 4)) + (slot >> 4)) * (D * 16 * SIZE);
#pragma unroll
                        for (int x = 0; x < kHalves; x++)
#pragma unroll
                            for (int q = 0; q < SIZE; q++) {
                                const u32x4 w = *reinterpret_cast<const u32x4*>(at + min(64 * x + lane, D - 1) * (16 * SIZE) + 16 * q);
#pragma unroll
                                for (int k = 0; k < 4; k++) from[x][j * kWords + 4 * q + k] = w[k];
                            }
                    }
                    auto put = [&](auto whole) __attribute__((always_inline)) {
#pragma unroll
                        for (int e = 0; e < kBlock; e++) {
                            const int word = __builtin_amdgcn_readlane(words, e) - base * kWords;
                            if (!decltype(whole)::value && (uint32_t)word >= (uint32_t)(kFrom * kWords)) continue;
                            const uint32_t which = __builtin_amdgcn_readlane(bytes, e);
#pragma unroll
                            for (int x = 0; x < kHalves; x++) v[x][e / kPerWord] = __builtin_amdgcn_perm(from[x][word], v[x][e / kPerWord], which);
                        }
                    };
                    if (held == 0xFFFF && base == 0 && !left) put(std::true_type{});      // (all sixteen are of these blocks)
                    else put(std::false_type{});
                }
            }
            settled();
            if (into < 0) continue;
            float f[EIGHT ? kBlock : 1];
            bool even = true;                                               // no number is rounded anew
            if constexpr (EIGHT) {
                const float own = factor(1, block * kBlock + (lane & 15));
                even = !__any(own != 1.f);
#pragma unroll
                for (int e = 0; e < kBlock; e++) f[e] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, own), e));
            }
            const int at = (w * kWindow + block * kBlock) & mask;
            char* out = a.to.values + (((int64_t)into << (a.page_shift - 4)) + (at >> 4)) * (D * 16 * SIZE);
#pragma unroll
            for (int x = 0; x < kHalves; x++) {
                const int d = 64 * x + lane;
                if (D % 64 && d >= D) continue;
                if constexpr (EIGHT) {
                    if (!even)
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(v[x][q], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(v[x][q], true);
                            const float y[4] = {lo[0] * f[4 * q], lo[1] * f[4 * q + 1], hi[0] * f[4 * q + 2], hi[1] * f[4 * q + 3]};       // (under its own scale a number is itself again)
                            v[x][q] = pack8(y, 1.f, 448.f);
                        }
                }
                char* to = out + d * (16 * SIZE);
                if (held == 0xFFFF) {
#pragma unroll
                    for (int q = 0; q < SIZE; q++) reinterpret_cast<u32x4*>(to)[q] = u32x4{v[x][4 * q], v[x][4 * q + 1], v[x][4 * q + 2], v[x][4 * q + 3]};
                } else {
                    // (what lies behind the last key stays as it is)
#pragma unroll
                    for (int e = 0; e < kBlock; e++) {
                        if (!(held >> e & 1)) continue;
                        if constexpr (EIGHT) reinterpret_cast<uint8_t*>(to)[e] = (uint8_t)(v[x][e >> 2] >> 8 * (e & 3));
                        else reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)(v[x][e >> 1] >> 16 * (e & 1));
                    }
                }
            }
        }
        if constexpr (EIGHT) {
            const int pg = t << a.page_shift;                               // the window's page t
            if (pg < here && to_row[pg / kBlock] >= 0) {
                a.to.key_scales[to_row[pg / kBlock]] = (uint8_t)top[0][t];
                a.to.value_scales[to_row[pg / kBlock]] = (uint8_t)top[1][t];
            }
        }
        if (!IN_PLACE) break;
    }
}

// Workspace: the list, and the pages that few heads are gathered into.
struct Room { int64_t cap, list, pages, keys, scales, weights, all; int width; };
Room room_of(const mhip_paged_cache* c, const mhip_sequences* s, int64_t keep, int64_t recent, bool staged) {
    Room r{};
    auto up = [](int64_t n) { return (n + 255) & ~(int64_t)255; };
    r.cap = std::max<int64_t>(std::min(keep + recent, s->width * c->page_size), 1);
    r.list = up(s->sequences * c->heads * r.cap * 4);
    r.all = r.list;
    if (staged) {
        r.width = (int)((r.cap + c->page_size - 1) / c->page_size);
        r.pages = s->sequences * r.width;
        const int64_t rows = r.pages * c->heads, tokens = rows * c->page_size;
        r.keys = up(tokens * c->head_size * (c->key_scales ? 1 : 2));
        r.scales = c->key_scales ? up(rows) : 0;
        r.weights = up(tokens * 4);
        r.all += 2 * r.keys + 2 * r.scales + r.weights;
    }
    return r;
}

// Heads from which on each of them is one workgroup's where it lies.
constexpr int64_t kManyHeads = 256;
bool gathers(const mhip_paged_cache* c, const mhip_sequences* s, bool in_place) { return in_place && s->sequences * c->heads < kManyHeads; }

int check_evict(const char* what, const mhip_paged_cache* c, const mhip_sequences* s, int64_t keep, int64_t recent) {
    if (const int rc = check_sizes(what, c, s)) return rc;
    if (keep < 0 || recent < 0) return fail(MHIP_ERR_INVALID_ARGUMENT, "%s: keys to keep are negative", what);
    if (keep > INT32_MAX / 2 || recent > INT32_MAX / 2) return fail(MHIP_ERR_UNSUPPORTED, "%s: more than 2^30 keys to keep", what);
    if (s->sequences * c->heads * 1024 >= (int64_t)1 << 32) return fail(MHIP_ERR_UNSUPPORTED, "%s: more than 2^22 sequences times heads", what);
    const int64_t windows = (std::min(keep + recent, s->width * c->page_size) + kWindow - 1) / kWindow;
    if (s->sequences * c->heads * windows >= (int64_t)1 << 24) return fail(MHIP_ERR_UNSUPPORTED, "%s: more than 2^32 keys to keep in all", what);
    return MHIP_OK;
}

template <int D, int SIZE>
int move(hipStream_t st, MoveArgs a, const Pool* between, int64_t units, bool in_place) {
    const dim3 all((unsigned)(units * a.windows));
    if (between) {
        const Pool last = a.to;
        a.to = *between;
        hipLaunchKernelGGL((evict_move_kernel<D, SIZE, true, false>), all, dim3(kWindow), 0, st, a);
        a.from = *between;
        a.to = last;
        a.list = nullptr;
        hipLaunchKernelGGL((evict_move_kernel<D, SIZE, false, false>), all, dim3(kWindow), 0, st, a);
    } else if (in_place) {
        hipLaunchKernelGGL((evict_move_kernel<D, SIZE, true, true>), dim3((unsigned)units), dim3(kWindow), 0, st, a);
    } else {
        hipLaunchKernelGGL((evict_move_kernel<D, SIZE, true, false>), all, dim3(kWindow), 0, st, a);
    }
    return check_launch("paged_evict");
}

template <int SIZE>
int move_d(hipStream_t st, const MoveArgs& a, const Pool* between, int64_t units, bool in_place, int64_t D) {
    switch (D) {
        case 32: return move<32, SIZE>(st, a, between, units, in_place);
        case 64: return move<64, SIZE>(st, a, between, units, in_place);
        case 96: return move<96, SIZE>(st, a, between, units, in_place);
        default: return move<128, SIZE>(st, a, between, units, in_place);
    }
}

}  // namespace
}  // namespace mhip

using namespace mhip;

extern "C" int64_t mhip_paged_evict_workspace(const mhip_paged_cache* cache, const mhip_sequences* seqs, int64_t keep, int64_t recent, int in_place, int64_t* least) {
    if (least) *least = 0;
    if (check_evict("paged_evict_workspace", cache, seqs, keep, recent)) return 0;
    if (least) *least = room_of(cache, seqs, keep, recent, false).all;
    return room_of(cache, seqs, keep, recent, gathers(cache, seqs, in_place != 0)).all;
}

extern "C" int mhip_paged_evict(void* stream, const mhip_paged_cache* cache, const mhip_sequences* seqs, float* weights, int64_t keep, int64_t recent, const int32_t* into, int64_t into_width,
                                int32_t* left, void* workspace, int64_t workspace_bytes) {
    if (const int rc = check_evict("paged_evict", cache, seqs, keep, recent)) return rc;
    if (!cache->key_scales != !cache->value_scales) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_evict: scales of keys without scales of values");
    const int64_t B = seqs->sequences, reach = seqs->width * cache->page_size;
    if (into && (into_width < 0 || into_width > (1 << 20) || into_width * cache->page_size < std::min(keep + recent, reach)))
        return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_evict: %lld pages for what stays are too few, or too many", (long long)into_width);
    if (B == 0) return MHIP_OK;
    if (!seqs->lengths || (seqs->width && !seqs->table) || !weights || !left || !cache->keys || !cache->values) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_evict: NULL tensor");
    if (((uintptr_t)cache->keys | (uintptr_t)cache->values | (uintptr_t)workspace) & 15) return fail(MHIP_ERR_UNSUPPORTED, "paged_evict: cache and workspace must be 16-byte aligned");
    const Room least = room_of(cache, seqs, keep, recent, false);
    if (!workspace || workspace_bytes < least.all) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_evict: a workspace of %lld bytes is needed", (long long)least.all);
    const int page_shift = __builtin_ctzll((uint64_t)cache->page_size);
    char* room = static_cast<char*>(workspace);
    hipStream_t st = as_stream(stream);
    const SelectArgs sel{weights, seqs->table, seqs->lengths, reinterpret_cast<int32_t*>(room), left, (int)seqs->width, (int)cache->pages, (int)cache->heads, page_shift, (int)keep, (int)recent, least.cap};
    auto select = [&](auto per, auto lds) {
        hipLaunchKernelGGL((evict_select_kernel<decltype(per)::value, decltype(lds)::value>), dim3((unsigned)(B * cache->heads)), dim3(kSelectThreads), 0, st, sel);
        return check_launch("paged_evict");
    };
    constexpr std::integral_constant<int, 0> kNone{};
    constexpr std::integral_constant<int, 4> kFour{};
    constexpr std::integral_constant<int, 16> kSixteen{};
    constexpr std::integral_constant<int, 32> kAll{};
    const int rc_select = reach <= 4 * kSelectThreads ? select(kFour, kNone) : reach <= 16 * kSelectThreads ? select(kSixteen, kNone) : reach <= 32 * kSelectThreads ? select(kAll, kNone)
                        : reach <= 64 * kSelectThreads ? select(kAll, kAll) : select(kNone, kNone);
    if (rc_select) return rc_select;
    const Pool here{(char*)cache->keys, (char*)cache->values, cache->key_scales, cache->value_scales, weights, seqs->table, (int)seqs->width, (int)cache->pages};
    Pool there = here, between{};
    if (into) {
        there.table = into;
        there.width = (int)into_width;
    }
    const Room staged = room_of(cache, seqs, keep, recent, true);
    const bool gather = gathers(cache, seqs, !into) && workspace_bytes >= staged.all && staged.pages * cache->heads <= INT32_MAX;
    if (gather) {
        char* p = room + staged.list;
        between = {p, p + staged.keys, reinterpret_cast<uint8_t*>(p + 2 * staged.keys), reinterpret_cast<uint8_t*>(p + 2 * staged.keys + staged.scales),
                   reinterpret_cast<float*>(p + 2 * staged.keys + 2 * staged.scales), nullptr, staged.width, (int)staged.pages};
    }
    const int windows = (int)((least.cap + kWindow - 1) / kWindow);
    const MoveArgs mv{here, there, sel.list, left, (int)cache->heads, page_shift, windows, least.cap};
    return cache->key_scales ? move_d<1>(st, mv, gather ? &between : nullptr, B * cache->heads, !into, cache->head_size)
                             : move_d<2>(st, mv, gather ? &between : nullptr, B * cache->heads, !into, cache->head_size);
}
