// What a model answered, as log probabilities: of given tokens, with the entropy of each row's distribution and its most likely alternatives.
//
//   m = max x, l = sum exp(x - m):  log p = (x - m) - log l,  entropy = log l - sum exp(x - m) (x - m) / l
//
// One pass over the logits.  A lane keeps a reference instead of the maximum, which moves when a piece of sixteen bytes exceeds it by more than 8 (weights up to e^8 = 2^11.5 are as
// exact as those below one, and their sums far from fp32's end), its sum, the sum of the products, and its own greatest value with the piece that holds it.  Bound by memory in 32 bits; in 16 bits as much by the instructions, seven and a
// quarter-rate exponential a value: 4096 rows of 50257 bf16 (412 MB) take 75 us, 5.5 TB/s, without alternatives and 90 us with 20.  Few rows are bound by latency: three take 11 us, 300 of 32003
// f32 (38 MB) 10 us without and 13 us with five alternatives.
//
// The alternatives need no second pass over the row: the `top`-th greatest of the maxima of 64 groups of four lanes (eight of a larger workgroup) is a bound that `top` values reach, so only the pieces of lanes (or classes of
// a lane's pieces) whose own maximum reaches it are looked at again; of 50257 random values some thirty to fifty are found for 20 and sorted in one wave.  Values are ordered by (value, lower index first) all
// the way, a piece's index standing for its values', so that the bound is one among equals too.  Where a row is built so that more than kMost values reach the bound, the row is read once for each alternative.
//
// Few rows are dealt over several workgroups each, and the last one to arrive puts the parts together (arrive.h).
#include <type_traits>

#include "arrive.h"
#include "common.h"

namespace mhip {
namespace {

constexpr int kMost = 1536, kMaxTop = 64, kMaxParts = 64;
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

template <int CTRL>
__device__ __forceinline__ uint32_t moved(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xF, 0xF, false); }
// the word of lane ^ J, in the register file
template <int J>
__device__ __forceinline__ uint32_t word_of(uint32_t v) {
    if constexpr (J == 1) return moved<0xB1>(v);                          // quad_perm
    else if constexpr (J == 2) return moved<0x4E>(v);
    else if constexpr (J == 3) return moved<0x1B>(v);
    else if constexpr (J == 7) return moved<0x141>(v);                    // row_half_mirror
    else if constexpr (J == 4) return moved<0x1B>(moved<0x141>(v));
    else if constexpr (J == 8) return moved<0x128>(v);                    // row_ror
    else if constexpr (J == 15) return moved<0x140>(v);                   // row_mirror
    else if constexpr (J == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (threadIdx.x & 16) ? r[0] : r[1];
    } else if constexpr (J == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (threadIdx.x & 32) ? r[0] : r[1];
    } else if constexpr (J == 31) return word_of<16>(word_of<15>(v));
    else return word_of<32>(word_of<31>(v));                              // 63
}
template <int J>
__device__ __forceinline__ uint64_t key_at(uint64_t v) { return (uint64_t)word_of<J>((uint32_t)(v >> 32)) << 32 | word_of<J>((uint32_t)v); }
template <int J>
__device__ __forceinline__ uint64_t greater(uint64_t v) {
    const uint64_t w = key_at<J>(v);
    return w > v ? w : v;
}
// lanes i and i ^ J: the one whose `bit` is clear has the greater key afterwards
template <int J>
__device__ __forceinline__ void order(uint64_t& v, int lane, int bit) {
    const uint64_t w = key_at<J>(v);
    v = (w > v) == ((lane & bit) == 0) ? w : v;
}
// groups of 2 J lanes whose keys rise and fall once, each sorted
template <int J>
__device__ __forceinline__ void settle(uint64_t& v, int lane) {
    order<J>(v, lane, J);
    if constexpr (J > 1) settle<J / 2>(v, lane);
}
// a wave's keys, the greatest in lane 0: sorted groups of K lanes are mirrored against one another, which leaves both halves such groups
template <int K = 2>
__device__ __forceinline__ uint64_t sorted(uint64_t v, int lane) {
    order<K - 1>(v, lane, K / 2);
    if constexpr (K > 2) settle<K / 4>(v, lane);
    if constexpr (K < 64) return sorted<2 * K>(v, lane);
    else return v;
}
// the 64 greatest of two sorted lists, sorted
__device__ __forceinline__ uint64_t merged(uint64_t a, uint64_t b, int lane) {
    const uint64_t r = key_at<63>(b);
    uint64_t v = a > r ? a : r;
    settle<32>(v, lane);
    return v;
}

// sums under a reference: l = sum 2^d, t = sum 2^d d, d = log2(e) (x - ref)
struct Sums { float ref, l, t; };
// of the wave's lanes, under the greatest of their references
__device__ __forceinline__ Sums joined(Sums s) {
    const float m = wave_max(s.ref);
    const float d = fmaxf((s.ref - (m == -INFINITY ? 0.f : m)) * kLog2eT, -300.f), f = __builtin_amdgcn_exp2f(d);
    return {m, wave_sum(s.l * f), wave_sum(f * (s.t + s.l * d))};
}

// kClasses: a lane's pieces fall into so many classes, in turn, each with a greatest value of its own.
template <typename T, int kThreads, int kClasses>
__global__ __launch_bounds__(kThreads) void token_log_probs_kernel(LogProbArgs a) {
    constexpr int EPV = 16 / sizeof(T), kWaves = kThreads / 64, kGroup = kThreads / 64;
    constexpr int kAhead = 4;                                             // pieces that are asked for together
    static_assert(kAhead % kClasses == 0, "a piece's class is its place among those");
    __shared__ uint64_t found[kMost];
    __shared__ Sums wave_sums[kWaves];
    __shared__ uint64_t groups[64], bound, best[kWaves];
    __shared__ uint16_t holders[kClasses * kThreads];
    __shared__ int count, holding, last;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = blockIdx.x % a.parts;
    const int64_t row = blockIdx.x / a.parts;
    uint64_t seen = 0;
    if (a.parts > 1 && threadIdx.x == 0) seen = arrive_look(a.words + row);
    const T* x = static_cast<const T*>(a.x) + row * a.vocab;
    // pieces of sixteen aligned bytes; the row begins `off` values into piece 0.  Pieces [whole0, whole1) lie inside the row; one in front of them and one behind are read value by value
    const int off = (int)((uintptr_t)x & 15) / (int)sizeof(T);
    const int pieces = (int)((a.vocab + off + EPV - 1) / EPV);
    const int p0 = (int)min((int64_t)part * a.pieces, (int64_t)pieces), p1 = (int)min((int64_t)p0 + a.pieces, (int64_t)pieces);
    const int whole0 = max(p0, off ? 1 : 0), whole1 = min(p1, (int)((a.vocab + off) / EPV));
    const bool head = p0 == 0 && p1 > 0 && (off || whole1 == 0), tail = p1 == pieces && p1 - 1 >= whole1 && !(head && p1 == 1);
    const u32x4* base = reinterpret_cast<const u32x4*>(x - off);
    auto whole = [&](int p, float (&v)[EPV]) __attribute__((always_inline)) {
        const Vec16<T> w = __builtin_bit_cast(Vec16<T>, base[p]);
#pragma unroll
        for (int e = 0; e < EPV; e++) v[e] = Elem<T>::to_f32(w.v[e]);
    };
    auto broken = [&](int p, float (&v)[EPV]) __attribute__((always_inline)) {
        const int i0 = p * EPV - off, n = (int)a.vocab;
        T t[EPV];
#pragma unroll
        for (int e = 0; e < EPV; e++) t[e] = x[min(max(i0 + e, 0), n - 1)];       // (all on their way before the first is used)
#pragma unroll
        for (int e = 0; e < EPV; e++) v[e] = i0 + e >= 0 && i0 + e < n ? Elem<T>::to_f32(t[e]) : -INFINITY;
    };

    // ---- the sums, and each lane's greatest value.  Weights are 2^(x log2(e) - c) with c = ref log2(e) rounded: 2^slip times what they are to be, `slip` being what the
    // rounding took (2^-8 at most).  Where a lane of the wave has a reference beyond 2^16 it is subtracted before the multiplication
    Sums s{-INFINITY, 0.f, 0.f};
    float c = 0.f, slip = 0.f, most[kClasses];
    int where[kClasses];
#pragma unroll
    for (int i = 0; i < kClasses; i++) {
        most[i] = -INFINITY;
        where[i] = -1;
    }
    bool far = false;
    auto take = [&](const float (&v)[EPV], int p, float& most, int& where) __attribute__((always_inline)) {
        float m = fmaxf(v[0], v[1]);
#pragma unroll
        for (int e = 2; e < EPV; e += 2) m = fmaxf(fmaxf(m, v[e]), v[e + 1]);
        where = m > most ? p : where;
        most = fmaxf(m, most);
        if (__builtin_expect(__any(m > s.ref + 8.f), 0)) {                // (from -inf on: any number)
            const float to = m > s.ref + 8.f ? m : s.ref;
            const bool none = to == -INFINITY;
            c = none ? 0.f : to * kLog2eT;
            const float slips = !none && fabsf(to) <= 65536.f ? fmaf(to, kLog2eT, -c) : 0.f;
            const float d = none ? 0.f : fmaxf((s.ref - to) * kLog2eT - slip + slips, -300.f), f = __builtin_amdgcn_exp2f(d);
            s.t = f * (s.t + s.l * d);
            s.l *= f;
            s.ref = to;
            slip = slips;
            far = __any(fabsf(to) > 65536.f && !none);
        }
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(far), 0)) {
            const float ref = s.ref == -INFINITY ? 0.f : s.ref;
#pragma unroll
            for (int e = 0; e < EPV; e++) {
                const float d = fmaf(v[e] - ref, kLog2eT, slip), f = __builtin_amdgcn_exp2f(d);
                s.l += f;
                s.t = fmaf(f, fmaxf(d, -300.f), s.t);
            }
        } else {
#pragma unroll
            for (int e = 0; e < EPV; e++) {
                // (the weight of a masked value is zero, and so is its product with -300; a NaN stays one)
                const float d = fmaf(v[e], kLog2eT, -c), f = __builtin_amdgcn_exp2f(d);
                s.l += f;
                s.t = fmaf(f, fmaxf(d, -300.f), s.t);
            }
        }
    };
    if (head && threadIdx.x == kThreads - 1) {
        float v[EPV];
        broken(0, v);
        where[0] = 0;
        take(v, 0, most[0], where[0]);
    }
    far = __any(far);                                                     // (one lane took the broken piece: the others' pieces go the way that its reference needs)
    auto widened = [&](const u32x4& w, float (&v)[EPV]) __attribute__((always_inline)) {
        const Vec16<T> t = __builtin_bit_cast(Vec16<T>, w);
#pragma unroll
        for (int e = 0; e < EPV; e++) v[e] = Elem<T>::to_f32(t.v[e]);
    };
#pragma unroll
    for (int i = 0; i < kClasses; i++) where[i] = whole0 + i * kThreads + (int)threadIdx.x < whole1 && where[i] < 0 ? whole0 + i * kThreads + threadIdx.x : where[i];
    int p = whole0;                                                       // (the same in all lanes: an address is a scalar and a lane's own offset)
    u32x4 w[kAhead];
    for (; p <= whole1 - kAhead * kThreads; p += kAhead * kThreads) {
#pragma unroll
        for (int i = 0; i < kAhead; i++) w[i] = (base + p + i * kThreads)[threadIdx.x];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            float v[EPV];
            widened(w[i], v);
            take(v, p + i * kThreads + threadIdx.x, most[i % kClasses], where[i % kClasses]);
        }
    }
    if (p < whole1) {
#pragma unroll
        for (int i = 0; i < kAhead; i++) w[i] = (base + p)[min((int)threadIdx.x + i * kThreads, whole1 - 1 - p)];
        auto rest = [&](auto which) __attribute__((always_inline)) {
            constexpr int i = decltype(which)::value;
            if (p + i * kThreads + (int)threadIdx.x < whole1) {
                float v[EPV];
                widened(w[i], v);
                take(v, p + i * kThreads + threadIdx.x, most[i % kClasses], where[i % kClasses]);
            }
        };
        static_assert(kAhead == 4, "a call each");
        rest(std::integral_constant<int, 0>{});
        rest(std::integral_constant<int, 1>{});
        rest(std::integral_constant<int, 2>{});
        rest(std::integral_constant<int, 3>{});
    }
    if (tail && threadIdx.x == 0) {
        float v[EPV];
        broken(p1 - 1, v);
        if (where[0] < 0) where[0] = p1 - 1;
        take(v, p1 - 1, most[0], where[0]);
    }
    const float unslipped = __builtin_amdgcn_exp2f(-slip);
    s.t = unslipped * (s.t - slip * s.l);
    s.l *= unslipped;
    if (a.parts > 1 && threadIdx.x == 0) arrive_claim(a.words + row, seen, a.tag);
    const bool not_a_number = s.l != s.l;
    s = joined(s);
    if (lane == 0) wave_sums[wave] = s;

    // ---- the alternatives of this part
    uint64_t list = 0;
    if (a.top) {
        auto each_of = [&](int q, auto each) __attribute__((always_inline)) {
            float v[EPV];
            if (q >= whole0 && q < whole1) whole(q, v);
            else broken(q, v);
#pragma unroll
            for (int e = 0; e < EPV; e++) {
                const int i = q * EPV - off + e;
                if (i >= 0 && i < (int)a.vocab) each(v[e], (uint32_t)i);
            }
        };
        if (not_a_number) {                                               // (or an infinity: its sums are no numbers either)
            auto look = [&](int q, float& most, int& where) __attribute__((always_inline)) {
                each_of(q, [&](float v, uint32_t) __attribute__((always_inline)) {
                    if (v != v && most == most) { most = v; where = q; }
                });
            };
            if (head && threadIdx.x == kThreads - 1) look(0, most[0], where[0]);
            for (int q = whole0 + threadIdx.x; q < whole1; q += kClasses * kThreads)
#pragma unroll
                for (int i = 0; i < kClasses; i++)
                    if (q + i * kThreads < whole1) look(q + i * kThreads, most[i], where[i]);
            if (tail && threadIdx.x == 0) look(p1 - 1, most[0], where[0]);
        }
        uint64_t keys[kClasses], key = 0;
#pragma unroll
        for (int i = 0; i < kClasses; i++) {
            keys[i] = where[i] >= 0 ? key_of(most[i], (uint32_t)where[i]) : 0;
            key = keys[i] > key ? keys[i] : key;
        }
        uint64_t group = greater<2>(greater<1>(key));
        if (kGroup == 8) group = greater<4>(group);
        if (lane % kGroup == 0) groups[threadIdx.x / kGroup] = group;
        if (threadIdx.x == 0) count = holding = 0;
        __syncthreads();
        if (wave == 0) {
            const uint64_t v = sorted(groups[lane], lane);
            if (lane == a.top - 1) bound = v;
        }
        __syncthreads();
        const uint64_t limit = bound;
        if (key >= limit) {
#pragma unroll
            for (int i = 0; i < kClasses; i++)
                if (keys[i] >= limit && where[i] >= 0) holders[atomicAdd(&holding, 1)] = (uint16_t)(i * kThreads + threadIdx.x);
        }
        __syncthreads();
        // every piece of those classes of lanes whose own maximum reaches the bound, dealt over the workgroup (2^shift items a class), and the two that are broken
        const int turns = (whole1 - whole0 + kClasses * kThreads - 1) / (kClasses * kThreads), shift = turns > 1 ? 32 - __builtin_clz(turns - 1) : 0, items = turns > 0 ? holding << shift : 0;
        const float least = value_of((uint32_t)(limit >> 32));
        auto keep = [&](float v, int q, uint32_t i) __attribute__((always_inline)) {
            if (v < least || key_of(v, (uint32_t)q) < limit) return;
            const int n = atomicAdd(&count, 1);
            if (n < kMost) found[n] = key_of(v, i);
        };
        for (int i0 = 0; i0 < items; i0 += 2 * kThreads) {
            u32x4 w[2];
            int q[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int i = min(i0 + j * kThreads + (int)threadIdx.x, items - 1);
                q[j] = whole0 + holders[i >> shift] + (i & ((1 << shift) - 1)) * (kClasses * kThreads);
                w[j] = base[min(q[j], whole1 - 1)];
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                if (i0 + j * kThreads >= items) break;
                if (i0 + j * kThreads + (int)threadIdx.x >= items || q[j] >= whole1) continue;
                float v[EPV];
                widened(w[j], v);
#pragma unroll
                for (int e = 0; e < EPV; e++) keep(v[e], q[j], (uint32_t)(q[j] * EPV - off + e));
            }
        }
        if ((head && threadIdx.x == 0) || (tail && threadIdx.x == 64)) {
            const int q = threadIdx.x ? p1 - 1 : 0;
            each_of(q, [&](float v, uint32_t i) __attribute__((always_inline)) { keep(v, q, i); });
        }
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
                for (int q = p0 + threadIdx.x; q < p1; q += kThreads)
                    each_of(q, [&](float v, uint32_t i) __attribute__((always_inline)) {
                        const uint64_t k = key_of(v, i);
                        if (k < before && k > mine) mine = k;
                    });
                mine = greater<32>(greater<16>(greater<8>(greater<4>(greater<2>(greater<1>(mine))))));
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
    if (wave == 0) s = joined(lane < kWaves ? wave_sums[lane] : Sums{-INFINITY, 0.f, 0.f});

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
        if (wave == 0) {
            s = Sums{-INFINITY, 0.f, 0.f};
            if (lane < a.parts) s = Sums{load_part(to + 4 * lane), load_part(to + 4 * lane + 1), load_part(to + 4 * lane + 2)};
            s = joined(s);
        }
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

// How a row is dealt: parts of at least 4096 values (two to four pieces a thread), as many as fill the device twice.  (us, twice | four | eight times: 64 rows of 128000 with 20 alternatives 13 | 16 | 30,
// 300 of 32003 f32 with five 15.1 | 15.3 | 18.8, 1000 of 50257 27 | 27 | 35.)
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
    if (rows < 0 || vocab <= 0 || vocab > (1 << 28)) return fail(MHIP_ERR_INVALID_ARGUMENT, "token_log_probs: %lld rows of %lld", (long long)rows, (long long)vocab);
    if (top < 0 || top > kMaxTop || top > vocab) return fail(MHIP_ERR_INVALID_ARGUMENT, "token_log_probs: %d alternatives of %lld (up to 64)", top, (long long)vocab);
    if (dtype != MHIP_BF16 && dtype != MHIP_F16 && dtype != MHIP_F32) return fail(MHIP_ERR_UNSUPPORTED, "token_log_probs: dtype %d (need bf16, f16 or f32)", dtype);
    if (token_dtype != MHIP_I32 && token_dtype != MHIP_I64) return fail(MHIP_ERR_UNSUPPORTED, "token_log_probs: token dtype %d (need i32 or i64)", token_dtype);
    if (rows >= 1 << 24) return fail(MHIP_ERR_UNSUPPORTED, "token_log_probs: %lld rows, more than a launch has threads for", (long long)rows);      // (2^32 of them, 256 a row; rows in parts are few)
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
    hipStream_t st = as_stream(stream);
    // rows that neither are dealt nor fill the device have workgroups of eight waves.  us, four waves | eight: 300 rows of 32003 f32 with five alternatives 15.1 | 13.1, 400 of 50257 bf16 with 20 17.9 | 15.5;
    // but 64 of 128000 13.1 | 14.2, 1000 of 32000 with 20 18.3 | 19.7, 1500 of 32003 18.6 | 20.1
    // Of the others, 16-bit rows that fill the device several times have four classes: a class that reaches the bound is a quarter of the pieces to look at again, each a line from memory, and the others'
    // launch is shorter by what four maxima take: 4096 rows of 50257 with 20 alternatives 100.2 | 89.6, 700 21.7 | 20.2; but 3 10.8 | 11.1, 2000 of 32003 f32 with five 55.4 | 56.5
    const bool wide = a.parts == 1 && rows <= 2 * (int64_t)compute_units() && vocab >= 4096, many = a.parts == 1 && !wide;
    auto go = [&](auto few, auto wider, auto more) { hipLaunchKernelGGL(wide ? wider : many ? more : few, dim3((unsigned)(rows * a.parts)), dim3(wide ? 512 : 256), 0, st, a); };
    if (dtype == MHIP_BF16) go(token_log_probs_kernel<bf16_t, 256, 1>, token_log_probs_kernel<bf16_t, 512, 1>, token_log_probs_kernel<bf16_t, 256, 4>);
    else if (dtype == MHIP_F16) go(token_log_probs_kernel<f16_t, 256, 1>, token_log_probs_kernel<f16_t, 512, 1>, token_log_probs_kernel<f16_t, 256, 4>);
    else go(token_log_probs_kernel<float, 256, 1>, token_log_probs_kernel<float, 512, 1>, token_log_probs_kernel<float, 256, 1>);
    return check_launch("token_log_probs");
}
