// Keys and values of new tokens into a paged cache (paged.h), the position rotation applied on the way; in 8 bits with the page's scale.
//
//   position  p = keys(b) - tokens(b) + i of token i of sequence b, its page table[b, p / page], its slot p % page
//   rotation  of the first R elements of a head, as mhip_rope turns them: with x = [x1 | x2] (halves) y = [x1 cos - x2 sin | x1 sin + x2 cos], row p of `freqs`
//             holding the cosines and then the sines.  fp32, and one rounding, to the type that is stored.
//   8 bits    the page's scale is the least power of two under which its largest value is at most 448.  Where the page holds tokens already it never shrinks, and
//             where it grows by 2^n the held values are multiplied by 2^-n and rounded, which changes none that stays above 2^-6 of the new scale.
//
// Bound by memory: every new value is read once and written once.  A workgroup takes one page's new tokens of one head, of keys or values (a page's scale needs all of
// them), or of one query head, whose rotation is the keys' own; a wave takes blocks of sixteen tokens and keeps them in registers in fp32 until the page's largest value is known.
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
    int pages, KV, H, R, positions;
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
// four e4m3 of x * inv; e4m3 has no infinities, so what is not finite becomes NaN
__device__ __forceinline__ uint32_t pack8(const float* x, float inv) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        y[e] = x[e] * inv;
        y[e] = fabsf(y[e]) <= 448.f ? y[e] : __builtin_nanf("");
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}
// the held values of four tokens or d under the grown scale
__device__ __forceinline__ uint32_t moved8(uint32_t w, float factor) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    const float x[4] = {lo[0], lo[1], hi[0], hi[1]};
    return pack8(x, factor);
}
__device__ __forceinline__ float finite_max(float m, float x) { return fmaxf(m, fabsf(x) < INFINITY ? fabsf(x) : 0.f); }

// The exponent byte of the least scale of at least 2^-126 with amax <= 448 * scale (448 = 1.75 * 2^8).
__device__ __forceinline__ int scale_byte(float amax) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, amax);
    return max((int)(bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000 ? 1 : 0), 1);
}

template <typename T, int D, bool EIGHT, int WAVES, int BLOCKS>
__global__ __launch_bounds__(64 * WAVES) void paged_append_kernel(AppendArgs a) {
    constexpr int kLanes = D / 16;                                        // lanes of a row: each has two pieces of eight elements
    constexpr int kRows = kLanes <= 2 ? 16 : kLanes == 4 ? 16 : 8;        // rows that a wave reads at once
    constexpr int kTurns = kBlock / kRows;
    __shared__ float tops[WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int shift = a.s.page_shift, page = 1 << shift;

    // ---- the page that this workgroup fills
    int first;
    auto touched = [&](int b) __attribute__((always_inline)) {
        const int n = a.s.tokens(b), end = a.s.keys(b), begin = max(end - n, 0);
        return n ? ((end + page - 1) >> shift) - (begin >> shift) : 0;
    };
    const int b = sequence_of(a.s.B, (int)blockIdx.x, touched, first);
    if (b < 0) return;
    const int n = a.s.tokens(b), end = a.s.keys(b), begin = max(end - n, 0);          // (more tokens than keys: the first ones have no place)
    const int at = (begin >> shift) + (int)blockIdx.x - first;
    if (at < begin >> shift || at << shift >= end) return;                            // (starts that are no starts: their sums may have wrapped)
    const int p0 = max(begin, at << shift), p1 = min(min(end, (at + 1) << shift), a.R ? a.positions : end);
    const int page_no = a.s.table[(int64_t)b * a.s.width + at];
    if (p0 >= p1) return;
    const int s0 = p0 & (page - 1), s1 = s0 + p1 - p0;
    const int64_t row0 = a.s.start(b) + (n - (end - p0));                               // of slot s0

    const int part = blockIdx.y;                                                       // keys, values, queries
    const bool is_v = part >= a.KV && part < 2 * a.KV, is_q = part >= 2 * a.KV;
    const int head = is_q ? part - 2 * a.KV : is_v ? part - a.KV : part;
    if (!is_q && (uint32_t)page_no >= (uint32_t)a.pages) return;
    const int64_t page_head = (int64_t)page_no * a.KV + head;

    if (!is_v) {
        const T* x = is_q ? static_cast<const T*>(a.q) + head * a.qs[1] : static_cast<const T*>(a.k) + head * a.ks[1];
        const int64_t xs = is_q ? a.qs[0] : a.ks[0];
        // lane l of a row: pieces l and l + R / 16 of the rotated elements, which belong together, or two of those behind them
        const int l = lane % kLanes, r = lane / kLanes;
        const bool turned = l < a.R / 16;
        const int d1 = turned ? 8 * l : a.R + 16 * (l - a.R / 16), d2 = turned ? d1 + a.R / 2 : d1 + 8;
        float y[BLOCKS][kTurns][16];
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < BLOCKS; c++) {
            const int block = c * WAVES + wave;
#pragma unroll
            for (int t = 0; t < kTurns; t++) {
                const int slot = block * kBlock + t * kRows + r;
                const bool in = slot >= s0 && slot < s1 && r < kRows;
                if (!in) {
#pragma unroll
                    for (int e = 0; e < 16; e++) y[c][t][e] = 0.f;
                    continue;
                }
                const T* row = x + (row0 + slot - s0) * xs;
                float f[16];
                to_floats<T>(*reinterpret_cast<const u32x4*>(row + d1), f);
                to_floats<T>(*reinterpret_cast<const u32x4*>(row + d2), f + 8);
                if (turned) {
                    const f32x4* cs = reinterpret_cast<const f32x4*>(a.freqs + (int64_t)(p0 + slot - s0) * a.R + 8 * l);
                    const f32x4* sn = reinterpret_cast<const f32x4*>(a.freqs + (int64_t)(p0 + slot - s0) * a.R + 8 * l + a.R / 2);
                    const f32x4 co[2] = {cs[0], cs[1]}, si[2] = {sn[0], sn[1]};
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float u = f[e], w = f[e + 8], cc = co[e >> 2][e & 3], ss = si[e >> 2][e & 3];
                        f[e] = u * cc - w * ss;
                        f[e + 8] = u * ss + w * cc;
                    }
                }
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    y[c][t][e] = f[e];
                    if (EIGHT) top = finite_max(top, f[e]);
                }
            }
        }
        float inv = 1.f, factor = 1.f;
        if (EIGHT && !is_q) {
            const int was = s0 ? max((int)a.key_scales[page_head], 1) : 0;
            top = wave_max(top);
            if (WAVES > 1) {
                if (lane == 0) tops[wave] = top;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < WAVES; w++) top = fmaxf(top, tops[w]);
            }
            const int byte = max(scale_byte(top), was);
            inv = scale_of(254 - byte);
            if (s0 && byte > was) {
                factor = scale_of(127 + was - byte > 0 ? 127 + was - byte : 1);
                u32x4* held = reinterpret_cast<u32x4*>(a.keys + page_head * page * D);
                for (int i = threadIdx.x; i < s0 * D / 16; i += 64 * WAVES) {
                    u32x4 w = held[i];
#pragma unroll
                    for (int e = 0; e < 4; e++) w[e] = moved8(w[e], factor);
                    held[i] = w;
                }
            }
            if (byte != was && threadIdx.x == 0) a.key_scales[page_head] = (uint8_t)byte;
        }
#pragma unroll
        for (int c = 0; c < BLOCKS; c++) {
            const int block = c * WAVES + wave;
#pragma unroll
            for (int t = 0; t < kTurns; t++) {
                const int slot = block * kBlock + t * kRows + r;
                if (slot < s0 || slot >= s1 || r >= kRows) continue;
                if (is_q || !EIGHT) {
                    T* out = is_q ? static_cast<T*>(a.q_out) + (row0 + slot - s0) * a.os[0] + head * a.os[1] : reinterpret_cast<T*>(a.keys) + (page_head * page + slot) * D;
                    *reinterpret_cast<u32x4*>(out + d1) = to_vector<T>(y[c][t]);
                    *reinterpret_cast<u32x4*>(out + d2) = to_vector<T>(y[c][t] + 8);
                } else {
                    char* out = a.keys + (page_head * page + slot) * D;
                    *reinterpret_cast<u32x2*>(out + d1) = u32x2{pack8(y[c][t], inv), pack8(y[c][t] + 4, inv)};
                    *reinterpret_cast<u32x2*>(out + d2) = u32x2{pack8(y[c][t] + 8, inv), pack8(y[c][t] + 12, inv)};
                }
            }
        }
        return;
    }

    // ---- values: a lane has two neighbouring d of kMine tokens, which lie side by side in the block
    constexpr int kPairs = D / 2, kGroups = kPairs <= 16 ? 4 : kPairs <= 32 ? 2 : 1, kMine = kBlock / kGroups;
    const int pair = lane % kPairs, group = lane / kPairs;
    const bool mine = group < kGroups;
    const T* x = static_cast<const T*>(a.v) + head * a.vs[1] + 2 * pair;
    float y[BLOCKS][2][kMine];
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < BLOCKS; c++)
#pragma unroll
        for (int t = 0; t < kMine; t++) {
            const int slot = (c * WAVES + wave) * kBlock + group * kMine + t;
            uint32_t w = 0;
            if (mine && slot >= s0 && slot < s1) w = *reinterpret_cast<const uint32_t*>(x + (row0 + slot - s0) * a.vs[0]);
            y[c][0][t] = Elem<T>::to_f32(__builtin_bit_cast(T, (uint16_t)w));
            y[c][1][t] = Elem<T>::to_f32(__builtin_bit_cast(T, (uint16_t)(w >> 16)));
            if (EIGHT) top = finite_max(finite_max(top, y[c][0][t]), y[c][1][t]);
        }
    float inv = 1.f;
    if (EIGHT) {
        const int was = s0 ? max((int)a.value_scales[page_head], 1) : 0;
        top = wave_max(top);
        if (WAVES > 1) {
            if (lane == 0) tops[wave] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WAVES; w++) top = fmaxf(top, tops[w]);
        }
        const int byte = max(scale_byte(top), was);
        inv = scale_of(254 - byte);
        if (s0 && byte > was) {
            const float factor = scale_of(127 + was - byte > 0 ? 127 + was - byte : 1);
            char* held = a.values + page_head * page * D;
            const int whole = s0 / kBlock * D, rest = s0 % kBlock;               // sixteen bytes of a d each
            for (int i = threadIdx.x; i < whole; i += 64 * WAVES) {
                u32x4 w = reinterpret_cast<u32x4*>(held)[i];
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = moved8(w[e], factor);
                reinterpret_cast<u32x4*>(held)[i] = w;
            }
            for (int i = threadIdx.x; i < D * rest; i += 64 * WAVES) {           // (byte by byte: the bytes behind them are being written)
                char* p = held + (whole + i / rest) * 16 + i % rest;
                *p = (char)(moved8((uint8_t)*p, factor) & 255);
            }
        }
        if (byte != was && threadIdx.x == 0) a.value_scales[page_head] = (uint8_t)byte;
    }
    if (!mine) return;
#pragma unroll
    for (int c = 0; c < BLOCKS; c++) {
        const int block = c * WAVES + wave, slot = block * kBlock + group * kMine;
        if (slot + kMine <= s0 || slot >= s1) continue;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int64_t at16 = ((page_head * (page / kBlock) + block) * D + 2 * pair + j) * kBlock + group * kMine;
            if (slot >= s0 && slot + kMine <= s1) {
                if constexpr (EIGHT) {
                    uint32_t w[kMine / 4];
#pragma unroll
                    for (int e = 0; e < kMine / 4; e++) w[e] = pack8(y[c][j] + 4 * e, inv);
                    __builtin_memcpy(__builtin_assume_aligned(a.values + at16, kMine), w, kMine);
                } else {
                    T w[kMine];
#pragma unroll
                    for (int e = 0; e < kMine; e++) w[e] = Elem<T>::from_f32(y[c][j][e]);
                    __builtin_memcpy(__builtin_assume_aligned(reinterpret_cast<T*>(a.values) + at16, kMine >= 8 ? 16 : 8), w, 2 * kMine);
                }
            } else {
#pragma unroll
                for (int t = 0; t < kMine; t++) {
                    if (slot + t < s0 || slot + t >= s1) continue;
                    if constexpr (EIGHT) {
                        const float four[4] = {y[c][j][t], 0.f, 0.f, 0.f};
                        a.values[at16 + t] = (char)(pack8(four, inv) & 255);
                    } else {
                        reinterpret_cast<T*>(a.values)[at16 + t] = Elem<T>::from_f32(y[c][j][t]);
                    }
                }
            }
        }
    }
}

template <typename T, int D, bool EIGHT>
int launch(hipStream_t st, const AppendArgs& a, int64_t units) {
    const dim3 grid((unsigned)units, (unsigned)(2 * a.KV + (a.q ? a.H : 0)));
    switch (a.s.page_shift) {
        case 4: hipLaunchKernelGGL((paged_append_kernel<T, D, EIGHT, 1, 1>), grid, dim3(64), 0, st, a); break;
        case 5: hipLaunchKernelGGL((paged_append_kernel<T, D, EIGHT, 2, 1>), grid, dim3(128), 0, st, a); break;
        case 6: hipLaunchKernelGGL((paged_append_kernel<T, D, EIGHT, 4, 1>), grid, dim3(256), 0, st, a); break;
        case 7: hipLaunchKernelGGL((paged_append_kernel<T, D, EIGHT, 4, 2>), grid, dim3(256), 0, st, a); break;
        default: hipLaunchKernelGGL((paged_append_kernel<T, D, EIGHT, 4, 4>), grid, dim3(256), 0, st, a); break;
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

int check_paged(const char* what, const mhip_paged_cache* c, const mhip_sequences* s, int dtype, bool* empty) {
    *empty = false;
    if (!c || !s) return fail(MHIP_ERR_INVALID_ARGUMENT, "%s: NULL cache or sequences", what);
    if (dtype != MHIP_BF16 && dtype != MHIP_F16) return fail(MHIP_ERR_UNSUPPORTED, "%s: dtype %d (need bf16 or f16)", what, dtype);
    if (c->pages <= 0 || c->heads <= 0 || s->sequences < 0 || s->width < 0 || s->tokens < 0) return fail(MHIP_ERR_INVALID_ARGUMENT, "%s: a size is negative, or the cache has no pages or heads", what);
    if (c->head_size < 32 || c->head_size > 128 || c->head_size % 32) return fail(MHIP_ERR_UNSUPPORTED, "%s: head size %lld (need 32, 64, 96 or 128)", what, (long long)c->head_size);
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
        return fail(MHIP_ERR_UNSUPPORTED, "%s: page size %lld (need a power of two from 16 to 256)", what, (long long)c->page_size);
    if (c->pages * c->heads > INT32_MAX || c->pages > INT32_MAX || c->heads > 1024 || s->sequences > 65536 || s->tokens > (1 << 24) || s->width > (1 << 20) || s->width * c->page_size > (1 << 24))
        return fail(MHIP_ERR_UNSUPPORTED, "%s: more than 65536 sequences, 2^24 tokens, 2^24 keys a sequence or 1024 heads", what);
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
                 (int)cache->pages, (int)cache->heads, (int)(q ? q_heads : 0), (int)rotated, (int)positions, {}, {}, {}, {}};
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
