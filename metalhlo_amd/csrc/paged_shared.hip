// Attention of sequences that have a prefix in common, whose keys and values lie in pages of their own: O = softmax(scale Q [K_prefix; K_own]^T) V.
//
// The prefix is read once for all rows of the call.  Launches of the kernels of paged_attention.h:
//   first   the rows of all sequences as one sequence's over the prefix, without a mask; each leaves its sums, unnormalised and in fp32, with their reference maximum and sum (kLeaves), and
//           paged_join_kernel puts together what a tile's workgroups have left of it
//   then    each sequence over its own keys; where a row's result is formed, what has been left for it is one more part (kGoesOn)
// What is left is 4 (D + 2) bytes a row and query head, written and read once.
#include "paged_attention.h"

namespace mhip {
namespace {

// The parts of the prefix put together, for all tiles by the whole device: by the last of a tile's workgroups to arrive, as elsewhere, 32 parts of 128 rows are two megabytes for one unit (64 tokens
// behind 12000 keys 110 us with it, 29 without).  64 items of four numbers a workgroup, whose waves take every fourth part, eight at a time: one turn for up to 32 parts, two for the 64 that there are at
// most (one thread an item 13.6 us for 33 MB).
template <int ROWS, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
    constexpr int kBlocks = ROWS * D / 4 / 64, kAhead = 8, kWaves = 4;
    __shared__ f32x4 sums[kWaves][64];
    __shared__ float state[kWaves][64][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int unit = blockIdx.x / kBlocks, head = unit / a.tiles, tile = unit - head * a.tiles, idx = (blockIdx.x - unit * kBlocks) * 64 + lane;
    const int row = row_of_item<ROWS, D>(idx), four = four_of_item<ROWS, D>(idx), rows = rows_of_all(a, lane) * a.G, r = tile * ROWS + row;
    if (tile * ROWS >= rows) return;
    const int first = a.dealt[2 * unit], parts = a.dealt[2 * unit + 1];
    if (parts == 0) return;
    float m = -INFINITY, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = wave; p0 < parts && r < rows; p0 += kWaves * kAhead) {
        float st[kAhead][2];
        f32x4 v[kAhead];
#pragma unroll
        for (int p = 0; p < kAhead; p++) {
            const int q = min(p0 + kWaves * p, parts - 1);
            const Parts<ROWS, D> at(a, 2 * (first + q) + (q ? 0 : 1));
            st[p][0] = at.state[2 * row];
            st[p][1] = at.state[2 * row + 1];
            v[p] = reinterpret_cast<const f32x4*>(at.sums)[idx];
        }
        float top = m;
#pragma unroll
        for (int p = 0; p < kAhead; p++) top = fmaxf(top, p0 + kWaves * p < parts ? st[p][0] : -INFINITY);
        const float use = top == -INFINITY ? 0.f : top, old = weight(m, use);
        m = top;
        l *= old;
        o *= old;
#pragma unroll
        for (int p = 0; p < kAhead; p++) {
            if (p0 + kWaves * p >= parts) break;
            const float al = weight(st[p][0], use);
            l = fmaf(st[p][1], al, l);
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = fmaf(v[p][e], al, o[e]);
        }
    }
    sums[wave][lane] = o;
    state[wave][lane][0] = m;
    state[wave][lane][1] = l;
    __syncthreads();
    if (wave || r >= rows) return;
#pragma unroll
    for (int w = 1; w < kWaves; w++) m = fmaxf(m, state[w][lane][0]);
    const float use = m == -INFINITY ? 0.f : m;
    o = f32x4{0.f, 0.f, 0.f, 0.f};
    l = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        const float al = weight(state[w][lane][0], use);
        const f32x4 v = sums[w][lane];
        l = fmaf(state[w][lane][1], al, l);
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = fmaf(v[e], al, o[e]);
    }
    const int token = a.by_group(r);
    put_four<bf16_t, D, kLeaves>(a, token, head * a.G + r - token * a.G, four, m, l, o);
}

template <int ROWS>
int join_all(hipStream_t st, const PagedArgs& a, int64_t D) {
    auto go = [&](auto kern, int d) {
        hipLaunchKernelGGL(kern, dim3((unsigned)(a.KV * a.tiles * (ROWS * d / 256))), dim3(256), 0, st, a);
        return check_launch("paged_attention_shared");
    };
    switch (D) {
        case 32: return go(paged_join_kernel<ROWS, 32>, 32);
        case 64: return go(paged_join_kernel<ROWS, 64>, 64);
        case 96: return go(paged_join_kernel<ROWS, 96>, 96);
        default: return go(paged_join_kernel<ROWS, 128>, 128);
    }
}


struct Shared {
    mhip_sequences all;                   // the prefix's pages, and the rows of all sequences
    Plan first, then;
    int tiles;                            // of the prefix, a head
    int64_t left, dealt, parts;           // bytes: what is left for rows, where tiles' parts are, parts of either launch
};

int shared_plan(const char* what, const mhip_paged_cache* c, const int32_t* prefix, int64_t prefix_width, const int32_t* prefix_length, const mhip_sequences* s, int64_t q_heads, Shared& r) {
    if (const int rc = check_sizes(what, c, s)) return rc;
    r.all = {prefix, prefix_length, s->starts, 1, prefix_width, s->tokens};
    if (const int rc = check_sizes(what, c, &r.all)) return rc;
    if (const int rc = plan_of(c, s, q_heads, r.then)) return rc;
    if (s->sequences == 0 || s->tokens == 0) return MHIP_OK;
    if (const int rc = plan_of(c, &r.all, q_heads, r.first, false)) return rc;
    r.left = (s->tokens * q_heads * (c->head_size + 2) * 4 + 255) & ~(int64_t)255;
    r.tiles = (int)((s->tokens * (q_heads / c->heads) + r.first.rows - 1) / r.first.rows);
    if (c->heads * (int64_t)r.tiles * (r.first.rows * c->head_size / 256) >= 1 << 24) return fail(MHIP_ERR_UNSUPPORTED, "%s: more rows than a launch has threads for", what);
    r.dealt = ((int64_t)c->heads * r.tiles * 8 + 255) & ~(int64_t)255;
    r.parts = std::max(workspace_of(c, r.first), workspace_of(c, r.then));
    return MHIP_OK;
}

}  // namespace
}  // namespace mhip

using namespace mhip;

extern "C" int64_t mhip_paged_attention_shared_workspace(const mhip_paged_cache* cache, int64_t prefix_width, const mhip_sequences* seqs, int64_t q_heads, int64_t* least) {
    Shared r{};
    if (least) *least = 0;
    if (shared_plan("paged_attention_shared_workspace", cache, nullptr, prefix_width, nullptr, seqs, q_heads, r)) return 0;
    if (least) *least = r.left + r.dealt;
    return r.left + r.dealt + r.parts;
}

extern "C" int mhip_paged_attention_shared(void* stream, const mhip_paged_cache* cache, const int32_t* prefix, int64_t prefix_width, const int32_t* prefix_length, const mhip_sequences* seqs, const void* q,
                                           void* o, int64_t q_heads, float scale, int is_causal, const int64_t* strides, int dtype, void* workspace, int64_t workspace_bytes) {
    bool empty;
    if (const int rc = check_paged("paged_attention_shared", cache, seqs, dtype, &empty)) return rc;
    Shared r{};
    if (const int rc = shared_plan("paged_attention_shared", cache, prefix, prefix_width, prefix_length, seqs, q_heads, r)) return rc;
    if (empty) return MHIP_OK;
    if (!prefix_length || (prefix_width && !prefix)) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_attention_shared: NULL prefix");
    if (const int rc = check_tensors("paged_attention_shared", q, o, strides, workspace)) return rc;
    if (!workspace || workspace_bytes < r.left + r.dealt) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_attention_shared: a workspace of %lld bytes is needed", (long long)(r.left + r.dealt));
    const bool room = workspace_bytes >= r.left + r.dealt + r.parts, eight = cache->key_scales != nullptr;
    char* parts = static_cast<char*>(workspace) + r.left + r.dealt;
    hipStream_t st = as_stream(stream);
    PagedArgs a = args_of(cache, sequences(cache, &r.all), r.first, q, o, q_heads, scale, 0, strides);
    a.more = static_cast<float*>(workspace);
    a.last = (int)seqs->sequences;
    a.dealt = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + r.left);
    a.tiles = r.tiles;
    if (room) give_room(a, cache, r.first, parts);
    if (const int rc = launch_form<kLeaves>("paged_attention_shared", st, a, r.first, cache->head_size, eight, dtype)) return rc;
    if (room) {
        const int64_t D = cache->head_size;
        const int rc = r.first.rows == 16 ? join_all<16>(st, a, D) : r.first.rows == 32 ? join_all<32>(st, a, D) : r.first.rows == 128 ? join_all<128>(st, a, D) : join_all<256>(st, a, D);
        if (rc) return rc;
    }
    a = args_of(cache, sequences(cache, seqs), r.then, q, o, q_heads, scale, is_causal, strides);
    a.more = static_cast<float*>(workspace);
    if (room) give_room(a, cache, r.then, parts);
    return launch_form<kGoesOn>("paged_attention_shared", st, a, r.then, cache->head_size, eight, dtype);
}
