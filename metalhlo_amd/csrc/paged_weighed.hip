// Attention over a paged cache that adds up the weights it gives: beside O = softmax(scale Q K^T) V, for every key and key head the sum over the call's tokens and the query heads of the head
// of the softmax weight, what an eviction (paged_evict.hip) goes by.
//
// The attention (paged_attention.h, kTells) leaves of each row the reference maximum and one over the sum of its weights, taken before they are rounded: 8 bytes a row.  A second launch forms
//   S = K Q^T       v_mfma_f32_16x16x32, keys as the rows of the result, so that a lane has four keys of a query and the keys of a tile stay in the operand registers while the queries go by
//   w = exp2(c S - m) / l
// and adds w up over its rows, which are a lane's own and, behind the last, sixteen lanes': each key's sum is one wave's (or four's, added in order), so that nothing is atomic and results do not depend on
// what runs when.  Sums are fp32.
#include "paged_attention.h"

namespace mhip {
namespace {

constexpr int kTile = 64;                 // keys of a wave

// ALL: four waves take the rows of the same 64 keys in turn; else each has 64 keys of its own.  `span`: keys of a unit of work, a multiple of what a workgroup takes at a time.
template <typename T, int D, bool EIGHT, bool ALL>
__global__ __launch_bounds__(256) void paged_weigh_kernel(PagedArgs a, float* weights, int span) {
    constexpr int NS = D / 32, SIZE = EIGHT ? 1 : 2, kStep = ALL ? kTile : 4 * kTile;
    __shared__ float sums[ALL ? 4 : 1][kTile];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, lg = lane >> 4, H = a.G * a.KV, mask = (1 << a.s.page_shift) - 1;
    auto d_of = [&](int s) __attribute__((always_inline)) {                   // of a lane's eight numbers of step s: in 8 bits two steps come in one load
        if (!EIGHT || (s | 1) >= NS) return 32 * s + 8 * lg;
        return 64 * (s >> 1) + 16 * lg + 8 * (s & 1);
    };
    auto units = [&](int b) __attribute__((always_inline)) { return a.s.tokens(b) ? a.KV * ((a.s.keys(b) + span - 1) / span) : 0; };
    for (int unit = blockIdx.x;; unit += gridDim.x) {
        int before;
        const int b = sequence_of(a.s.B, unit, units, before);
        if (b < 0) return;
        const int first = a.s.start(b), tokens = a.s.tokens(b), keys = a.s.keys(b), end = a.s.bounded_end(b), rows = tokens * a.G;
        const int a_head = (keys + span - 1) / span, head = (unit - before) / a_head, part = unit - before - head * a_head;
        if (head >= a.KV) return;                                           // (starts that are no starts: their sums may have wrapped)
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
                    for (int s = 0; s < NS; s++) kf[j][s] = widen<T>(*reinterpret_cast<const u32x2*>(kp + d_of(s)), 1.f);
                } else {
#pragma unroll
                    for (int s = 0; s < NS; s++) kf[j][s] = *reinterpret_cast<const u32x4*>(kp + 2 * d_of(s));
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
            if (key0 < keys)
                for (int r0 = row0 + (ALL ? 16 * wave : 0); r0 < rows; r0 += ALL ? 64 : 16) {
                    const int row = min(r0 + li, rows - 1), token = a.by_group(row), query = head * a.G + row - token * a.G;
                    const T* qp = static_cast<const T*>(a.q) + (int64_t)(first + token) * a.qs[0] + (int64_t)query * a.qs[1];
                    u32x4 qf[NS];
#pragma unroll
                    for (int s = 0; s < NS; s++) qf[s] = *reinterpret_cast<const u32x4*>(qp + d_of(s)) ^ a.sign;
                    const float* told = a.more + 2 * ((int64_t)(first + token) * H + query);
                    const float m = told[0], inv = told[1];
                    const int limit = r0 + li < rows ? min(a.is_causal ? end - tokens + token + 1 : keys, keys) - key0 - 4 * lg : 0;      // of key 4 lg of the tile on
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        f32x4 s4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int s = 0; s < NS; s++) s4 = Mfma16P<T>::run(kf[j][s], qf[s], s4);
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const float w = __builtin_amdgcn_exp2f(fmaf(s4[r], c[j], -m)) * inv;
                            sum[j][r] += 16 * j + r < limit ? w : 0.f;
                        }
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
                if (wave == 0) kept = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
            }
            if (stores) *to = had + kept;
        }
    }
}

struct Weighed {
    Plan p;
    int64_t told, parts;                  // bytes
    int span, grid;
    bool all;
};
int weighed_plan(const char* what, const mhip_paged_cache* c, const mhip_sequences* s, int64_t q_heads, Weighed& r) {
    if (const int rc = check_sizes(what, c, s)) return rc;
    if (const int rc = plan_of(c, s, q_heads, r.p)) return rc;
    if (s->sequences == 0 || s->tokens == 0) return MHIP_OK;
    r.told = (s->tokens * q_heads * 8 + 255) & ~(int64_t)255;
    r.parts = workspace_of(c, r.p, 3);
    r.all = r.p.rows >= 128;
    const int step = r.all ? kTile : 4 * kTile;
    const double sequences = (double)std::min(s->sequences, s->tokens), keys = (double)(s->width * c->page_size);
    r.span = step;
    while (sequences * c->heads * (keys / r.span + 1) > (double)(1 << 29)) r.span *= 2;
    r.grid = (int)std::min<double>(4.0 * compute_units(), sequences * c->heads * (keys / r.span + 1));
    return MHIP_OK;
}

template <typename T, int D, bool EIGHT>
int weigh(hipStream_t st, const PagedArgs& a, float* weights, const Weighed& r) {
    if (r.all) hipLaunchKernelGGL((paged_weigh_kernel<T, D, EIGHT, true>), dim3((unsigned)r.grid), dim3(256), 0, st, a, weights, r.span);
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
    return r.told + r.parts;
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
    if (const int rc = launch_form<kTells>("paged_attention_weighed", st, a, r.p, D, eight, dtype)) return rc;
    if (seqs->width == 0) return MHIP_OK;                                    // (no key has a place)
    if (dtype == MHIP_BF16) return eight ? weigh_d<bf16_t, true>(st, a, weights, r, D) : weigh_d<bf16_t, false>(st, a, weights, r, D);
    return eight ? weigh_d<f16_t, true>(st, a, weights, r, D) : weigh_d<f16_t, false>(st, a, weights, r, D);
}
