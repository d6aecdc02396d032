// Attention of sequences that have a prefix in common, whose keys and values lie in pages of their own: O = softmax(scale Q [K_prefix; K_own]^T) V.
//
// The prefix is read once for all rows of the call.  Two launches of the kernels of paged_attention.h:
//   first   the rows of all sequences as one sequence's over the prefix, without a mask; each leaves its sums, unnormalised and in fp32, with their reference maximum and sum (kLeaves)
//   then    each sequence over its own keys; where a row's result is formed, what has been left for it is one more part (kGoesOn)
// What is left is 4 (D + 2) bytes a row and query head, written and read once.
#include "paged_attention.h"

using namespace mhip;

namespace {

struct Shared {
    mhip_sequences all;                   // the prefix's pages, and the rows of all sequences
    Plan first, then;
    int64_t left, parts;                  // bytes
};

int shared_plan(const char* what, const mhip_paged_cache* c, const int32_t* prefix, int64_t prefix_width, const int32_t* prefix_length, const mhip_sequences* s, int64_t q_heads, Shared& r) {
    if (const int rc = check_sizes(what, c, s)) return rc;
    r.all = {prefix, prefix_length, s->starts, 1, prefix_width, s->tokens};
    if (const int rc = check_sizes(what, c, &r.all)) return rc;
    if (const int rc = plan_of(c, s, q_heads, r.then)) return rc;
    if (s->sequences == 0 || s->tokens == 0) return MHIP_OK;
    if (const int rc = plan_of(c, &r.all, q_heads, r.first, false)) return rc;
    r.left = (s->tokens * q_heads * (c->head_size + 2) * 4 + 255) & ~(int64_t)255;
    r.parts = std::max(workspace_of(c, r.first), workspace_of(c, r.then));
    return MHIP_OK;
}

}  // namespace

extern "C" int64_t mhip_paged_attention_shared_workspace(const mhip_paged_cache* cache, int64_t prefix_width, const mhip_sequences* seqs, int64_t q_heads, int64_t* least) {
    Shared r{};
    if (least) *least = 0;
    if (shared_plan("paged_attention_shared_workspace", cache, nullptr, prefix_width, nullptr, seqs, q_heads, r)) return 0;
    if (least) *least = r.left;
    return r.left + r.parts;
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
    if (!workspace || workspace_bytes < r.left) return fail(MHIP_ERR_INVALID_ARGUMENT, "paged_attention_shared: a workspace of %lld bytes is needed", (long long)r.left);
    const bool room = workspace_bytes >= r.left + r.parts, eight = cache->key_scales != nullptr;
    char* parts = static_cast<char*>(workspace) + r.left;
    hipStream_t st = as_stream(stream);
    PagedArgs a = args_of(cache, sequences(cache, &r.all), r.first, q, o, q_heads, scale, 0, strides);
    a.more = static_cast<float*>(workspace);
    a.last = (int)seqs->sequences;
    if (room) give_room(a, cache, r.first, parts);
    if (const int rc = launch_form<kLeaves>("paged_attention_shared", st, a, r.first, cache->head_size, eight, dtype)) return rc;
    a = args_of(cache, sequences(cache, seqs), r.then, q, o, q_heads, scale, is_causal, strides);
    a.more = static_cast<float*>(workspace);
    if (room) give_room(a, cache, r.then, parts);
    return launch_form<kGoesOn>("paged_attention_shared", st, a, r.then, cache->head_size, eight, dtype);
}
