// mhip_paged_attention: the kernels are in paged_attention.h.
#include "paged_attention.h"

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
    if (const int rc = check_tensors("paged_attention", q, o, strides, workspace)) return rc;
    PagedArgs a = args_of(cache, sequences(cache, seqs), p, q, o, q_heads, scale, is_causal, strides);
    if (workspace && workspace_bytes >= workspace_of(cache, p)) give_room(a, cache, p, workspace);
    return launch_form<kPlain>("paged_attention", as_stream(stream), a, p, cache->head_size, cache->key_scales != nullptr, dtype);
}
