// What a model answered, as log probabilities: of given tokens, with the entropy of each row's distribution and its most likely alternatives.
//
//   m = max x, l = sum exp(x - m):  log p = (x - m) - log l,  entropy = log l - sum exp(x - m) (x - m) / l
//
// One pass over the logits.  A lane keeps a reference instead of the maximum, which moves when a piece of sixteen bytes exceeds it by more than 8 (powers of two up to 2^8 are as exact
// as those below one), its sum, the sum of the products, and its own greatest value with the piece that holds it.  Bound by memory and, in 16 bits, as much by the exponentials: six instructions and
// a quarter-rate one a value.
//
// The alternatives need no second pass over the row: the `top`-th greatest of the maxima of 64 groups of eight lanes is a bound that `top` values reach, so only lanes whose own maximum reaches it look
// at their pieces again; of 50257 random values some thirty to fifty are found for 20 and sorted in one wave.  Values are ordered by (value, lower index first) all
// the way, a piece's index standing for its values', so that the bound is one among equals too.  Where a row is built so that more than kMost values reach the bound, the row is read once for each alternative.
//
// Few rows are dealt over several workgroups each, and the last one to arrive puts the parts together (arrive.h).
#include "arrive.h"
#include "common.h"

namespace mhip {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64, kGroup = kThreads / 64, kMost = 4096, kMaxTop = 64, kMaxParts = 64;
constexpr float kLn2 = 0.69314718055994531f, kLog2eT = 1.4426950408889634f;

struct LogProbArgs {
    const void* x;
    const void* tokens;
    float *log_p, *entropy, *top_p;
    int32_t* top_id;
    int64_t vocab;
    int top, wide_tokens, parts;
    int64_t pieces;                     // of a part
    float4* state;                      // [row][part]: reference, l, t
    uint64_t* lists;                    // [row][part][64]
    uint64_t* words;
    uint64_t tag;
};

// A key grows with the value, a NaN above all, and falls with the index.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.f);            // (-0 and 0 are equal)
    return v != v ? ~0u : (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return __builtin_bit_cast(float, o == ~0u ? 0x7FC00000u : (o >> 31) ? o & 0x7FFFFFFFu : ~o); }
__device__ __forceinline__ uint64_t key_of(float v, uint32_t index) { return (uint64_t)ordered(v) << 32 | (uint32_t)~index; }

__device__ __forceinline__ uint64_t lane_key(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__shfl((int)(v >> 32), lane, 64) << 32 | (uint32_t)__shfl((int)v, lane, 64);
}
__device__ __forceinline__ uint64_t exchange(uint64_t v, int lane, int j, bool greater) {
    const uint64_t w = lane_key(v, lane ^ j);
    return (w > v) == greater ? w : v;
}
// a wave's keys, the greatest in lane 0
__device__ inline uint64_t sorted(uint64_t v, int lane) {
#pragma unroll
    for (int k = 2; k <= 64; k *= 2)
#pragma unroll
        for (int j = k / 2; j; j /= 2) v = exchange(v, lane, j, ((lane & k) == 0) == ((lane & j) == 0));
    return v;
}
// the 64 greatest of two sorted lists, sorted
__device__ inline uint64_t merged(uint64_t a, uint64_t b, int lane) {
    const uint64_t r = lane_key(b, 63 - lane);
    uint64_t v = a > r ? a : r;
#pragma unroll
    for (int j = 32; j; j /= 2) v = exchange(v, lane, j, (lane & j) == 0);
    return v;
}

// sums under a reference: l = sum 2^d, t = sum 2^d d, d = log2(e) (x - ref)
struct Sums { float ref, l, t; };
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.ref, b.ref), use = m == -INFINITY ? 0.f : m;
    const float da = fmaxf((a.ref - use) * kLog2eT, -300.f), db = fmaxf((b.ref - use) * kLog2eT, -300.f);
    const float ea = __builtin_amdgcn_exp2f(da), eb = __builtin_amdgcn_exp2f(db);
    return {m, a.l * ea + b.l * eb, ea * (a.t + a.l * da) + eb * (b.t + b.l * db)};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void token_log_probs_kernel(LogProbArgs a) {
    constexpr int EPV = 16 / sizeof(T);
    __shared__ uint64_t found[kMost];
    __shared__ Sums wave_sums[kWaves];
    __shared__ uint64_t groups[64], bound, best[kWaves];
    __shared__ int count, last;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = blockIdx.x % a.parts;
    const int64_t row = blockIdx.x / a.parts;
    uint64_t seen = 0;
    if (a.parts > 1 && threadIdx.x == 0) seen = arrive_look(a.words + row);
    const T* x = static_cast<const T*>(a.x) + row * a.vocab;
    // pieces of sixteen aligned bytes; the row begins `off` values into the first one
    const int off = (int)((uintptr_t)x & 15) / (int)sizeof(T);
    const int pieces = (int)((a.vocab + off + EPV - 1) / EPV);
    const int p0 = (int)min((int64_t)part * a.pieces, (int64_t)pieces), p1 = (int)min((int64_t)p0 + a.pieces, (int64_t)pieces);
    const u32x4* base = reinterpret_cast<const u32x4*>(x - off);
    auto read = [&](int p, float (&v)[EPV]) __attribute__((always_inline)) {
        const int64_t i0 = (int64_t)p * EPV - off;
        if (i0 >= 0 && i0 + EPV <= a.vocab) {
            const Vec16<T> w = __builtin_bit_cast(Vec16<T>, base[p]);
#pragma unroll
            for (int e = 0; e < EPV; e++) v[e] = Elem<T>::to_f32(w.v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < EPV; e++) v[e] = i0 + e >= 0 && i0 + e < a.vocab ? Elem<T>::to_f32(x[i0 + e]) : -INFINITY;
        }
    };

    // ---- the sums, and each lane's greatest value
    Sums s{-INFINITY, 0.f, 0.f};
    float most = -INFINITY;
    int where = p0 + (int)threadIdx.x;
    auto take = [&](const float (&v)[EPV], int p) __attribute__((always_inline)) {
        float m = v[0];
#pragma unroll
        for (int e = 1; e < EPV; e++) m = fmaxf(m, v[e]);
        if (m > most) { most = m; where = p; }
        if (m > s.ref + 8.f) {                                            // (from -inf on: any number)
            const float d = fmaxf((s.ref - m) * kLog2eT, -300.f), f = __builtin_amdgcn_exp2f(d);
            s.t = f * (s.t + s.l * d);
            s.l *= f;
            s.ref = m;
        }
        const float ref = s.ref == -INFINITY ? 0.f : s.ref;
#pragma unroll
        for (int e = 0; e < EPV; e++) {
            // (2^-300 is zero, and so is its product: a masked value adds nothing)
            const float raw = (v[e] - ref) * kLog2eT, d = raw < -300.f ? -300.f : raw, f = __builtin_amdgcn_exp2f(d);
            s.l += f;
            s.t = fmaf(f, d, s.t);
        }
    };
    int p = p0 + threadIdx.x;
    for (; p + 3 * kThreads < p1; p += 4 * kThreads) {
        float v[4][EPV];
#pragma unroll
        for (int i = 0; i < 4; i++) read(p + i * kThreads, v[i]);
#pragma unroll
        for (int i = 0; i < 4; i++) take(v[i], p + i * kThreads);
    }
    for (; p < p1; p += kThreads) {
        float v[EPV];
        read(p, v);
        take(v, p);
    }
    if (a.parts > 1 && threadIdx.x == 0) arrive_claim(a.words + row, seen, a.tag);
    const bool not_a_number = s.l != s.l;
#pragma unroll
    for (int j = 1; j < 64; j *= 2) s = joined(s, Sums{__shfl_xor(s.ref, j, 64), __shfl_xor(s.l, j, 64), __shfl_xor(s.t, j, 64)});
    if (lane == 0) wave_sums[wave] = s;

    // ---- the alternatives of this part
    uint64_t list = 0;
    if (a.top) {
        uint64_t key = 0;
        if (p0 + (int)threadIdx.x < p1) {
            if (not_a_number) {                                           // (or an infinity: its sums are no numbers either)
                for (int q = p0 + threadIdx.x; q < p1 && most == most; q += kThreads) {
                    float v[EPV];
                    read(q, v);
#pragma unroll
                    for (int e = 0; e < EPV; e++)
                        if (v[e] != v[e]) { most = v[e]; where = q; }
                }
            }
            key = key_of(most, (uint32_t)where);
        }
        uint64_t group = key;
#pragma unroll
        for (int j = 1; j < kGroup; j *= 2) {
            const uint64_t w = lane_key(group, lane ^ j);
            group = w > group ? w : group;
        }
        if (lane % kGroup == 0) groups[threadIdx.x / kGroup] = group;
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
        if (wave == 0) {
            const uint64_t v = sorted(groups[lane], lane), b = lane_key(v, a.top - 1);
            if (lane == 0) bound = b;
        }
        __syncthreads();
        const uint64_t limit = bound;
        auto look = [&](auto each) __attribute__((always_inline)) {
            for (int q = p0 + threadIdx.x; q < p1; q += kThreads) {
                float v[EPV];
                read(q, v);
#pragma unroll
                for (int e = 0; e < EPV; e++) {
                    const int64_t i = (int64_t)q * EPV - off + e;
                    if (i >= 0 && i < a.vocab) each(v[e], q, (uint32_t)i);
                }
            }
        };
        if (key >= limit)
            look([&](float v, int q, uint32_t i) __attribute__((always_inline)) {
                if (key_of(v, (uint32_t)q) < limit) return;
                const int n = atomicAdd(&count, 1);
                if (n < kMost) found[n] = key_of(v, i);
            });
        __syncthreads();
        const int n = count;
        if (n <= kMost) {
            // wave w sorts 64 of every 64 kWaves
            for (int f = wave * 64; f < n; f += kThreads) {
                const uint64_t v = sorted(f + lane < n ? found[f + lane] : 0, lane);
                list = f == wave * 64 ? v : merged(list, v, lane);
            }
            if (n > 64) {
                __syncthreads();
                if (wave) found[wave * 64 + lane] = list;
                __syncthreads();
                if (wave == 0)
                    for (int w = 1; w < kWaves && w * 64 < n; w++) list = merged(list, found[w * 64 + lane], lane);
            }
        } else {
            uint64_t before = ~(uint64_t)0;
            for (int r = 0; r < a.top; r++) {
                uint64_t mine = 0;
                look([&](float v, int, uint32_t i) __attribute__((always_inline)) {
                    const uint64_t k = key_of(v, i);
                    if (k < before && k > mine) mine = k;
                });
#pragma unroll
                for (int j = 1; j < 64; j *= 2) {
                    const uint64_t w = lane_key(mine, lane ^ j);
                    mine = w > mine ? w : mine;
                }
                if (lane == 0) best[wave] = mine;
                __syncthreads();
                before = 0;
#pragma unroll
                for (int w = 0; w < kWaves; w++) before = best[w] > before ? best[w] : before;
                if (lane == r) list = before;
                __syncthreads();
            }
        }
    }
    __syncthreads();
    s = wave_sums[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) s = joined(s, wave_sums[w]);

    if (a.parts > 1) {
        float* to = reinterpret_cast<float*>(a.state + row * a.parts);
        uint64_t* lists = a.lists + row * a.parts * 64;
        if (threadIdx.x == 0) {
            store_part(to + 4 * part, s.ref);
            store_part(to + 4 * part + 1, s.l);
            store_part(to + 4 * part + 2, s.t);
        }
        if (a.top && wave == 0) __hip_atomic_store(lists + part * 64 + lane, list, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (!arrive_last(a.words + row, a.parts, &last)) return;
        s = Sums{-INFINITY, 0.f, 0.f};
        for (int q = 0; q < a.parts; q++) s = joined(s, Sums{load_part(to + 4 * q), load_part(to + 4 * q + 1), load_part(to + 4 * q + 2)});
        if (a.top) {
            list = 0;
            for (int q = wave; q < a.parts; q += kWaves) {
                const uint64_t v = __hip_atomic_load(lists + q * 64 + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                list = q == wave ? v : merged(list, v, lane);
            }
            found[threadIdx.x] = list;
            __syncthreads();
            if (wave == 0)
                for (int w = 1; w < kWaves && w < a.parts; w++) list = merged(list, found[w * 64 + lane], lane);
        }
    }
    if (wave) return;
    const float log_l = __builtin_amdgcn_logf(s.l) * kLn2;
    if (lane == 0) {
        const int64_t token = a.wide_tokens ? static_cast<const int64_t*>(a.tokens)[row] : static_cast<const int32_t*>(a.tokens)[row];
        a.log_p[row] = token >= 0 && token < a.vocab ? Elem<T>::to_f32(x[token]) - s.ref - log_l : __builtin_nanf("");
        if (a.entropy) a.entropy[row] = log_l - s.t / s.l * kLn2;
    }
    if (lane < a.top) {
        a.top_p[row * a.top + lane] = value_of((uint32_t)(list >> 32)) - s.ref - log_l;
        a.top_id[row * a.top + lane] = (int32_t)~(uint32_t)list;
    }
}

// How a row is dealt: parts of at least 4096 values (a piece for every thread), as many as fill the device twice.
int parts_of(int64_t rows, int64_t vocab) {
    const int64_t want = 2 * (int64_t)compute_units() / (rows ? rows : 1), most = vocab / 4096;
    const int64_t n = want < most ? want : most;
    return n < 2 ? 1 : n > kMaxParts ? kMaxParts : (int)n;
}

int size_of(int dtype) { return dtype == MHIP_F32 ? 4 : 2; }

}  // namespace
}  // namespace mhip

using namespace mhip;

extern "C" int64_t mhip_token_log_probs_workspace(int64_t rows, int64_t vocab, int top) {
    if (rows <= 0 || vocab <= 0) return 0;
    const int64_t parts = parts_of(rows, vocab);
    return parts == 1 ? 0 : rows * parts * (16 + (top ? 512 : 0)) + rows * 8;
}

extern "C" int mhip_token_log_probs(void* stream, const void* logits, const void* tokens, float* log_probs, float* entropy, float* top_log_probs, int32_t* top_ids,
                                    int64_t rows, int64_t vocab, int top, int dtype, int token_dtype, void* workspace, int64_t workspace_bytes) {
    if (rows < 0 || vocab <= 0 || vocab > (1 << 30)) return fail(MHIP_ERR_INVALID_ARGUMENT, "token_log_probs: %lld rows of %lld", (long long)rows, (long long)vocab);
    if (top < 0 || top > kMaxTop || top > vocab) return fail(MHIP_ERR_INVALID_ARGUMENT, "token_log_probs: %d alternatives of %lld (up to 64)", top, (long long)vocab);
    if (dtype != MHIP_BF16 && dtype != MHIP_F16 && dtype != MHIP_F32) return fail(MHIP_ERR_UNSUPPORTED, "token_log_probs: dtype %d (need bf16, f16 or f32)", dtype);
    if (token_dtype != MHIP_I32 && token_dtype != MHIP_I64) return fail(MHIP_ERR_UNSUPPORTED, "token_log_probs: token dtype %d (need i32 or i64)", token_dtype);
    if (rows == 0) return MHIP_OK;
    if (!logits || !tokens || !log_probs || (top && (!top_log_probs || !top_ids))) return fail(MHIP_ERR_INVALID_ARGUMENT, "token_log_probs: NULL tensor");
    if ((uintptr_t)logits % size_of(dtype) || (uintptr_t)workspace % 16) return fail(MHIP_ERR_INVALID_ARGUMENT, "token_log_probs: misaligned buffer");
    LogProbArgs a{logits, tokens, log_probs, entropy, top_log_probs, top_ids, vocab, top, token_dtype == MHIP_I64, 1, 0, nullptr, nullptr, nullptr, 0};
    const int parts = parts_of(rows, vocab);
    if (parts > 1 && workspace && workspace_bytes >= mhip_token_log_probs_workspace(rows, vocab, top)) {
        a.parts = parts;
        a.state = static_cast<float4*>(workspace);
        a.lists = reinterpret_cast<uint64_t*>(a.state + rows * parts);
        a.words = a.lists + (top ? rows * parts * 64 : 0);
        a.tag = launch_tag();
    }
    const int64_t per = 16 / size_of(dtype), pieces = (vocab + per - 1) / per + 1;
    a.pieces = (pieces + a.parts - 1) / a.parts;
    if (rows * a.parts > INT32_MAX) return fail(MHIP_ERR_UNSUPPORTED, "token_log_probs: more rows than a launch has workgroups");
    const dim3 grid((unsigned)(rows * a.parts));
    hipStream_t st = as_stream(stream);
    if (dtype == MHIP_BF16) hipLaunchKernelGGL(token_log_probs_kernel<bf16_t>, grid, dim3(kThreads), 0, st, a);
    else if (dtype == MHIP_F16) hipLaunchKernelGGL(token_log_probs_kernel<f16_t>, grid, dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL(token_log_probs_kernel<float>, grid, dim3(kThreads), 0, st, a);
    return check_launch("token_log_probs");
}
