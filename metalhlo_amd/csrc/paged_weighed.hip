// Attention over a paged cache that adds up the weights it gives: beside O = softmax(scale Q K^T) V, for every key and key head the sum over the call's tokens and the query heads of the head
// of the softmax weight, what an eviction (paged_evict.hip) goes by.
//
// The attention (paged_attention.h, kTells) leaves of each row the reference maximum and one over the sum of its weights, taken before they are rounded: 8 bytes a row.
//   few rows    it leaves the scores too, and paged_add_kernel adds w = exp2(s - m) / l up over a key's rows: time is that of the scores' bytes, behind the attention's.
//   many rows   paged_weigh_kernel forms
//     S = K Q^T       v_mfma_f32_16x16x32, keys as the rows of the result, so that a lane has four keys of a query and the keys of a tile stay in the operand registers while the queries go by
//     w = exp2(c S - m) / l
//   and adds w up over its rows, which are a lane's own and, behind the last, sixteen lanes'.  It is bound by the exponentials and the latency between them; half the products' work is done twice, which
//   costs less than sending 4 bytes of every weight through memory.
// Each key's sum is one thread's, one wave's or eight waves', added in order: nothing is atomic and results do not depend on what runs when.  Sums are fp32.
// us: 40 sequences of up to 6000 keys, 32 over 8 heads of 128 in 8 bits (352 MB), 95 (attention 88, adding 8); three prompts of up to 1408 tokens, the same heads in 16 bits (38 GFLOP), 125 (86 and 54 by
// themselves, each with its launch).
#include "paged_attention.h"

namespace mhip {
namespace {

constexpr int kTile = 64;                 // keys of a wave

// ALL: eight waves take the rows of the same 64 keys in turn, the next ones' queries on their way; else each of four has 64 keys of its own.  `span`: keys of a unit of work, a multiple of what a workgroup
// takes at a time.  Units go key block by key block, the longest first: a causal prompt's first keys are seen by all of its tokens.
constexpr int weigh_waves(bool all) { return all ? 8 : 4; }
template <typename T, int D, bool EIGHT, bool ALL>
__global__ __launch_bounds__(64 * weigh_waves(ALL), ALL ? (D <= 32 ? 4 : 2) : 1) void paged_weigh_kernel(PagedArgs a, float* weights, int span) {
    constexpr int NS = D / 32, SIZE = EIGHT ? 1 : 2, WAVES = weigh_waves(ALL), kStep = ALL ? kTile : WAVES * kTile, kTurn = ALL ? 16 * WAVES : 16;
    constexpr int kPieces = D / 8, kRow = 2 * D + 16;       // pieces of sixteen bytes of a query; bytes from one to the next in LDS, where sixteen of the same piece are all 64 banks
    __shared__ float sums[ALL ? WAVES : 1][kTile];
    __shared__ __attribute__((aligned(16))) char queries[WAVES][16 * kRow];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, lg = lane >> 4, H = a.G * a.KV, mask = (1 << a.s.page_shift) - 1;
    auto d_of = [&](int s) __attribute__((always_inline)) {                   // of a lane's eight numbers of step s: in 8 bits two steps come in one load
        if (!EIGHT || (s | 1) >= NS) return 32 * s + 8 * lg;
        return 64 * (s >> 1) + 16 * lg + 8 * (s & 1);
    };
    const bool even = kTurn % a.G == 0;
    const int64_t q_turn = even ? kTurn / a.G * a.qs[0] : 0, t_turn = even ? (int64_t)2 * (kTurn / a.G) * H : 0;
    for (int unit = blockIdx.x;; unit += gridDim.x) {
        // ---- the unit's sequence, head and stretch of keys
        auto parts_of = [&](int b) __attribute__((always_inline)) { return a.s.tokens(b) ? (a.s.keys(b) + span - 1) / span : 0; };
        int b, head, part;
        if (ALL && a.s.B <= 64) {
            // the first stretches of all sequences, then the second ones: `part` is the greatest with no more than `at` in front of it
            const int mine = lane < a.s.B ? parts_of(lane) : 0, at = a.by_heads(unit);
            auto before = [&](int p) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(wave_scan(min(mine, p)), 63); };
            int lo = 0, hi = __builtin_amdgcn_readfirstlane((int)wave_max((float)mine));       // (exact: below 2^23)
            if (at >= before(hi)) return;
            while (lo + 1 < hi) {
                const int mid = (lo + hi) >> 1;
                (before(mid) <= at ? lo : hi) = mid;
            }
            part = lo;
            head = unit - at * a.KV;
            const int ahead = wave_scan(mine > part ? 1 : 0), wanted = at - before(part) + 1;
            b = __builtin_ctzll(__ballot(mine > part && ahead == wanted));
        } else {
            int before;
            b = sequence_of(a.s.B, unit, [&](int b) __attribute__((always_inline)) { return a.KV * parts_of(b); }, before);
            if (b < 0) return;
            part = a.by_heads(unit - before);
            head = unit - before - part * a.KV;
            if (part >= parts_of(b)) return;                                // (starts that are no starts: their sums may have wrapped)
        }
        const int first = a.s.start(b), tokens = a.s.tokens(b), keys = a.s.keys(b), end = a.s.bounded_end(b), rows = tokens * a.G;
        uniform_words table = (uniform_words)(uintptr_t)(a.s.table + (int64_t)b * a.s.width);
        for (int k0 = part * span; k0 < min(keys, (part + 1) * span); k0 += kStep) {
            const int key0 = k0 + (ALL ? 0 : kTile * wave);
            // ---- keys: row li of tile j is key key0 + 16 j + li
            u32x4 kf[4][NS];
            float c[4];
            bool held[4];
            int row_of[4];                                                  // page * KV + head
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int at = min((key0 + 16 * j) >> a.s.page_shift, a.s.width - 1), page = table[at];
                held[j] = key0 + 16 * j < keys && (uint32_t)page < (uint32_t)a.pages;
                row_of[j] = (held[j] ? page : 0) * a.KV + head;
                c[j] = EIGHT ? a.c * scale_of(a.key_scales[row_of[j]]) : a.c;
                const char* kp = a.keys + (((int64_t)row_of[j] << a.s.page_shift) + ((key0 + 16 * j) & mask) + li) * (D * SIZE);
                if constexpr (EIGHT) {
#pragma unroll
                    for (int s = 0; s < NS; s++) kf[j][s] = widen<T>(*reinterpret_cast<const u32x2*>(kp + d_of(s)), 1.f) ^ a.sign;
                } else {
#pragma unroll
                    for (int s = 0; s < NS; s++) kf[j][s] = *reinterpret_cast<const u32x4*>(kp + 2 * d_of(s)) ^ a.sign;
                }
            }
            // the key that this lane stores, and what it had
            const int mine = key0 + 16 * (li >> 2) + 4 * lg + (li & 3), own = li >> 2;
            const bool stores = mine < keys && (own == 0 ? held[0] : own == 1 ? held[1] : own == 2 ? held[2] : held[3]) && (!ALL || wave == 0);
            const int own_row = own == 0 ? row_of[0] : own == 1 ? row_of[1] : own == 2 ? row_of[2] : row_of[3];
            float* const to = weights + (((int64_t)own_row << a.s.page_shift) + (mine & mask));
            const float had = stores && mine < end - tokens ? *to : 0.f;      // (the call's own tokens begin with it)

            float sum[4][4];
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int r = 0; r < 4; r++) sum[j][r] = 0.f;
            // token i sees the keys up to end - tokens + i
            const int row0 = a.is_causal ? (max(key0 - (end - tokens), 0) * a.G) & ~15 : 0;
            // Queries come a piece of sixteen bytes a lane, neighbouring lanes neighbouring pieces, and turn into operands in the wave's own LDS: a row a lane, as the operand has it, is 64 lines
            // for the L1 to look up in place of 16 a load (three prompts of up to 1500 tokens, 32 over 8 heads of 128: 62 us | 54).
            u32x4 pieces[NS];
            u32x2 told;
            const T* qp[NS];
            const float* tp;
            // (by turns; rows r0 .. r0 + 15 are mostly those of the turn before, so many tokens on)
            auto ask = [&](int r0, bool begins) __attribute__((always_inline)) {
                if (r0 >= rows) return;
                if (!begins && even && r0 + 16 <= rows) {
#pragma unroll
                    for (int s = 0; s < NS; s++) qp[s] += q_turn;
                    tp += t_turn;
                } else {
                    auto query_of = [&](int row, int& token) __attribute__((always_inline)) {
                        row = min(row, rows - 1);
                        token = a.by_group(row);
                        return row - token * a.G + head * a.G;
                    };
                    int token, query;
#pragma unroll
                    for (int s = 0; s < NS; s++) {
                        query = query_of(r0 + (64 * s + lane) / kPieces, token);
                        qp[s] = static_cast<const T*>(a.q) + (int64_t)(first + token) * a.qs[0] + (int64_t)query * a.qs[1] + (64 * s + lane) % kPieces * 8;
                    }
                    query = query_of(r0 + li, token);
                    tp = a.more + 2 * ((int64_t)(first + token) * H + query);
                }
#pragma unroll
                for (int s = 0; s < NS; s++) pieces[s] = *reinterpret_cast<const u32x4*>(qp[s]);
                told = *reinterpret_cast<const u32x2*>(tp);
            };
            int r0 = row0 + (ALL ? 16 * wave : 0);
            if (key0 < keys) ask(r0, true);
            for (; key0 < keys && r0 < rows; r0 += kTurn) {
#pragma unroll
                for (int s = 0; s < NS; s++) *reinterpret_cast<u32x4*>(queries[wave] + (64 * s + lane) / kPieces * kRow + (64 * s + lane) % kPieces * 16) = pieces[s];
                const float from = -__builtin_bit_cast(float, (uint32_t)told.x), over = __builtin_bit_cast(float, (uint32_t)told.y);
                wave_in_order();
                ask(r0 + kTurn, false);
                u32x4 q[NS];
#pragma unroll
                for (int s = 0; s < NS; s++) q[s] = *reinterpret_cast<const u32x4*>(queries[wave] + li * kRow + 2 * d_of(s));
                wave_in_order();
                f32x4 s4[4];
#pragma unroll
                for (int s = 0; s < NS; s++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s4[j] = Mfma16P<T>::run(kf[j][s], q[s], s ? s4[j] : f32x4{0.f, 0.f, 0.f, 0.f});
                // (the first of the rows sees the whole tile: so do all)
                const bool whole = r0 + 16 <= rows && key0 + kTile <= min(a.is_causal ? end - tokens + (int)a.by_group(r0) + 1 : keys, keys);
                int limit = 0;                                              // keys that are seen, of key 4 lg of the tile on
                if (!whole && r0 + li < rows) limit = min(a.is_causal ? end - tokens + (int)a.by_group(r0 + li) + 1 : keys, keys) - key0 - 4 * lg;
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++) s4[j][r] = __builtin_amdgcn_exp2f(fmaf(s4[j][r], c[j], from));
                if (whole) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int r = 0; r < 4; r++) sum[j][r] = fmaf(s4[j][r], over, sum[j][r]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int r = 0; r < 4; r++) sum[j][r] += 16 * j + r < limit ? s4[j][r] * over : 0.f;
                }
            }
            // ---- over the sixteen lanes; lane li keeps tile li / 4, key 4 lg + li % 4 of it
            float kept = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float v = sum[j][r];
                    v += __shfl_xor(v, 1, 64);
                    v += __shfl_xor(v, 2, 64);
                    v += __shfl_xor(v, 4, 64);
                    v += __shfl_xor(v, 8, 64);
                    if (li == 4 * j + r) kept = v;
                }
            if constexpr (ALL) {
                __syncthreads();                                            // (the keys before have been added up)
                sums[wave][lane] = kept;
                __syncthreads();
                if (wave == 0) {
                    kept = 0.f;
#pragma unroll
                    for (int x = 0; x < WAVES; x++) kept += sums[x][lane];
                }
            }
            if (stores) *to = had + kept;
        }
    }
}

// Where the attention has left its scores: a thread four keys, 1024 a workgroup.  `blocks`: workgroups of a sequence and head.
__global__ __launch_bounds__(256) void paged_add_kernel(PagedArgs a, float* weights, int blocks) {
    const int H = a.G * a.KV, mask = (1 << a.s.page_shift) - 1, all = a.s.B * a.KV * blocks;
    for (int unit = blockIdx.x; unit < all; unit += gridDim.x) {
        const int pair = unit / blocks, b = a.by_heads(pair), head = pair - b * a.KV;
        const int first = a.s.start(b), tokens = a.s.tokens(b), keys = a.s.keys(b), end = a.s.bounded_end(b);
        const int key = ((unit - pair * blocks) * 256 + (int)threadIdx.x) * 4;
        if (!tokens || key >= keys) continue;
        const int page = a.s.table[(int64_t)b * a.s.width + (key >> a.s.page_shift)];
        if ((uint32_t)page >= (uint32_t)a.pages) continue;
        float* const to = weights + (((int64_t)page * a.KV + head) << a.s.page_shift) + (key & mask);
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int token = 0; token < tokens; token++) {
            const int seen = a.is_causal ? end - tokens + token + 1 - key : 4;  // of the four
            if (seen <= 0) continue;                                          // (these were not written)
            const int64_t row = (int64_t)(first + token) * H + head * a.G;
            const f32x4 before = sum;
#pragma unroll 4
            for (int g = 0; g < a.G; g++) {
                const f32x4 s = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(a.scores + (row + g) * a.score_stride + key));
                const float m = a.more[2 * (row + g)], inv = a.more[2 * (row + g) + 1];
#pragma unroll
                for (int e = 0; e < 4; e++) sum[e] = fmaf(__builtin_amdgcn_exp2f(s[e] - m), inv, sum[e]);
            }
            // (what a row does not see is -inf there, but zero times its `inv` may be NaN.  us, 40 sequences of up to 6000 keys, asked at each addition | here: 8.6 | 7.8)
#pragma unroll
            for (int e = 1; e < 4; e++) sum[e] = e < seen ? sum[e] : before[e];
        }
        const f32x4 had = *reinterpret_cast<const f32x4*>(to);                // (the call's own tokens begin with it)
#pragma unroll
        for (int e = 0; e < 4; e++) sum[e] += key + e < end - tokens ? had[e] : 0.f;
        if (key + 4 <= keys) *reinterpret_cast<f32x4*>(to) = sum;
        else
            for (int e = 0; key + e < keys; e++) to[e] = e == 0 ? sum[0] : e == 1 ? sum[1] : sum[2];
    }
}

// Scores that few rows leave are read in place of the keys where they are fewer bytes, written and read; us, keys read again | scores: 40 sequences of up to 6000 keys, 32 over 8 heads of 128 in 8 bits, 134 | 95.
constexpr int64_t kMostScores = (int64_t)1 << 30;

struct Weighed {
    Plan p;
    int64_t told, parts, scores;          // bytes
    int span, grid, stride, blocks;
    bool all;
};
int weighed_plan(const char* what, const mhip_paged_cache* c, const mhip_sequences* s, int64_t q_heads, Weighed& r) {
    if (const int rc = check_sizes(what, c, s)) return rc;
    if (const int rc = plan_of(c, s, q_heads, r.p)) return rc;
    if (s->sequences == 0 || s->tokens == 0) return MHIP_OK;
    r.told = (s->tokens * q_heads * 8 + 255) & ~(int64_t)255;
    r.parts = (workspace_of(c, r.p, 3) + 255) & ~(int64_t)255;
    r.all = r.p.rows >= 128;
    r.stride = (int)((s->width * c->page_size + 63) & ~(int64_t)63);
    r.blocks = (r.stride + 1023) / 1024;
    const double scores = 4.0 * (double)(s->tokens * q_heads) * r.stride;
    const bool fewer = 8 * (q_heads / c->heads) <= c->head_size * (c->key_scales ? 1 : 2);
    if (!r.all && fewer && scores <= (double)kMostScores && (double)(s->sequences * c->heads) * r.blocks < (double)(1 << 30)) r.scores = (int64_t)scores;
    const int step = r.all ? kTile : 4 * kTile;
    const double sequences = (double)std::min(s->sequences, s->tokens), keys = (double)(s->width * c->page_size);
    r.span = step;
    while (sequences * c->heads * (keys / r.span + 1) > (double)(1 << 29)) r.span *= 2;
    r.grid = (int)std::min<double>(4.0 * compute_units(), sequences * c->heads * (keys / r.span + 1));
    return MHIP_OK;
}

template <typename T, int D, bool EIGHT>
int weigh(hipStream_t st, const PagedArgs& a, float* weights, const Weighed& r) {
    if (r.all) hipLaunchKernelGGL((paged_weigh_kernel<T, D, EIGHT, true>), dim3((unsigned)r.grid), dim3(64 * weigh_waves(true)), 0, st, a, weights, r.span);
    else hipLaunchKernelGGL((paged_weigh_kernel<T, D, EIGHT, false>), dim3((unsigned)r.grid), dim3(256), 0, st, a, weights, r.span);
    return check_launch("paged_attention_weighed");
}
template <typename T, bool EIGHT>
int weigh_d(hipStream_t st, const PagedArgs& a, float* weights, const Weighed& r, int64_t D) {
    switch (D) {
        case 32: return weigh<T, 32, EIGHT>(st, a, weights, r);
        case 64: return weigh<T, 64, EIGHT>(st, a, weights, r);
        case 96: return weigh<T, 96, EIGHT>(st, a, weights, r);
        default: return weigh<T, 128, EIGHT>(st, a, weights, r);
    }
}

}  // namespace
}  // namespace mhip

using namespace mhip;

extern "C" int64_t mhip_paged_attention_weighed_workspace(const mhip_paged_cache* cache, const mhip_sequences* seqs, int64_t q_heads, int64_t* least) {
    Weighed r{};
    if (least) *least = 0;
    if (weighed_plan("paged_attention_weighed_workspace", cache, seqs, q_heads, r)) return 0;
    if (least) *least = r.told;
    return r.told + r.parts + r.scores;
}

extern "C" int mhip_paged_attention_weighed(void* stream, const mhip_paged_cache* cache, const mhip_sequences* seqs, const void* q, void* o, float* weights, int64_t q_heads, float scale, int is_causal,
                                            const int64_t* strides, int dtype, void* workspace, int64_t workspace_bytes) {
    bool empty;
    if (const int rc = check_paged("paged_attention_weighed", cache, seqs, dtype, &empty)) return rc;
    Weighed r{};
    if (const int rc = weighed_plan("paged_attention_weighed", cache, seqs, q_heads, r)) return rc;
    if (empty) return MHIP_OK;
    if (!weights) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_attention_weighed: NULL weights");
    if (const int rc = check_tensors("paged_attention_weighed", q, o, strides, workspace)) return rc;
    if (!workspace || workspace_bytes < r.told) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_attention_weighed: a workspace of %lld bytes is needed", (long long)r.told);
    const bool eight = cache->key_scales != nullptr;
    const int64_t D = cache->head_size;
    hipStream_t st = as_stream(stream);
    PagedArgs a = args_of(cache, sequences(cache, seqs), r.p, q, o, q_heads, scale, is_causal, strides);
    a.more = static_cast<float*>(workspace);
    if (workspace_bytes >= r.told + r.parts) give_room(a, cache, r.p, static_cast<char*>(workspace) + r.told, 3);
    if (r.scores && !((uintptr_t)weights & 15) && workspace_bytes >= r.told + r.parts + r.scores) {
        a.scores = reinterpret_cast<float*>(static_cast<char*>(workspace) + r.told + r.parts);
        a.score_stride = r.stride;
        a.score_bytes = (uint32_t)r.scores;
    }
    if (const int rc = launch_form<kTells>("paged_attention_weighed", st, a, r.p, D, eight, dtype)) return rc;
    if (seqs->width == 0) return MHIP_OK;                                    // (no key has a place)
    if (a.scores) {
        hipLaunchKernelGGL(paged_add_kernel, dim3((unsigned)std::min<int64_t>(seqs->sequences * cache->heads * r.blocks, 1 << 20)), dim3(256), 0, st, a, weights, r.blocks);
        return check_launch("paged_attention_weighed");
    }
    if (dtype == MHIP_BF16) return eight ? weigh_d<bf16_t, true>(st, a, weights, r, D) : weigh_d<bf16_t, false>(st, a, weights, r, D);
    return eight ? weigh_d<f16_t, true>(st, a, weights, r, D) : weigh_d<f16_t, false>(st, a, weights, r, D);
}
