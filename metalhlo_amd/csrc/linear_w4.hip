// Linear layers whose weights are held in 4 bits: C = act(x W^T + bias) (+ residual), W[n][k] = (q - z) s with a 4-bit q and, for each n and `group` neighbouring k,
// a scale s and a zero z in the tensors' 16-bit type.
//
//   words   [N / 16][K / 128][64][4]   the operand of v_mfma_f32_16x16x32 as its lanes want it: lane l's word s holds row l % 16 of sixteen and the columns 32 s + 8 (l / 16) + 0 .. 7,
//                                      column i and column i + 4 in the low and the high half of byte i.  A wave reads a kilobyte in one go, and a lane's sixteen bytes feed four products.
//   scales  [N / 16][K / group][16]    pairs of scale and zero; a lane of the result holds four neighbouring rows, whose pairs are sixteen bytes
// both rounded up to whole sixteens and 128s.
//
// A byte 0 .. 15 is that number times 2^-9 as e4m3, across the border of its subnormals: one v_cvt_scalef32_pk per two weights makes 16-bit numbers q, exactly, of bytes that a mask and a shift have made.
// The products of q and x are added over a group in the matrix unit, and so is x itself (an operand of ones, so that each lane of the result has the sum of its own row): what a group
// adds to a result is s (sum q x - z sum x), in fp32 and of numbers that are exact.  Of an infinite x, and of a bf16 x whose sums pass fp32's range, that makes a NaN or an infinity where W x need not have one: results
// that are not finite are added up once more, weight by weight.
//
// Few rows: w4_rows_kernel, whose time is that of reading W.  Many: W is rounded to 16 bits into the workspace and multiplied by mhip_gemm (kManyRows).
#include <algorithm>

#include "arrive.h"

namespace mhip {
namespace {

constexpr int kBlockK = 128;

struct W4Args {
    const void* x;
    const u32x4* words4;
    const uint32_t* scales;           // pairs
    const void *bias, *residual;
    void* c;
    int M, N, K, act;
    int n16, k128;
    int whole;                        // four columns of a row of C lie on 8 bytes, and so do the bias' and the residual's
    int even;                         // rows of x lie on 16 bytes
    int parts, per, chunk;            // of K: workgroups that share it, blocks of one, blocks of x in LDS at a time where that is not known at compile time
    float* sums;                      // [row block][strip][part]
    uint64_t *words, tag;
};

// the eight numbers of a word
template <typename T>
__device__ __forceinline__ u32x4 numbers(uint32_t w) {
    const uint32_t low = w & 0x0F0F0F0Fu, high = (w >> 4) & 0x0F0F0F0Fu;
    if constexpr (std::is_same<T, bf16_t>::value)
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, 512.f, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, 512.f, true)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, 512.f, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, 512.f, true))};
    else
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(low, 512.f, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(low, 512.f, true)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(high, 512.f, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(high, 512.f, true))};
}

template <typename T>
__device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (std::is_same<T, bf16_t>::value) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// the halves of a pair
template <typename T>
__device__ __forceinline__ float low_half(uint32_t w) { return Elem<T>::to_f32(__builtin_bit_cast(T, (uint16_t)w)); }
template <typename T>
__device__ __forceinline__ float high_half(uint32_t w) { return Elem<T>::to_f32(__builtin_bit_cast(T, (uint16_t)(w >> 16))); }

// A workgroup of WN x WK waves has 16 WN columns of C, 16 MT rows and a part of K: wave (wn, wk) the wn-th sixteen columns and every WK-th block of 128.  U blocks of a wave are on their way at a time.
// x lies in LDS: read from memory by each wave for itself it is 4 MT times as many bytes as W's, through an L2 (24 rows, 5120 x 5120, 19.3 us so, 13.5 now).  In two chunks of CU WK blocks of K, ROWS rows
// at most, one multiplied while the next is on its way in registers (one chunk at a time, 64 rows of 4096 x 4096, 18.6 us | 14.5); or, CU = 0, of a few rows all of a part at once (one token of 8192 x 8192,
// two chunks of sixteen blocks 15.8 | so 12.0).
// Where K is dealt over workgroups (parts), the last of them to arrive adds the parts up in order (arrive.h).
template <typename T, int GROUP, int MT, int WN, int WK, int U, int CU, int ROWS>
__global__ __launch_bounds__(64 * WN * WK) void w4_rows_kernel(W4Args g) {
    constexpr int kGroups = kBlockK / GROUP, kSteps = GROUP / 32, kThreads = 64 * WN * WK;
    constexpr bool kWhole = CU == 0;                                       // (CU: see below)
    static_assert(U % (kWhole ? 1 : CU) == 0, "a turn of the words is whole chunks of x");
    constexpr int kChunk = CU * WK, kRowPieces = kWhole ? 1 : kChunk * (kBlockK / 8), kStride = kChunk * (kBlockK * 2) + 16;
    constexpr int kPieces = kWhole ? 4 : (ROWS * kRowPieces + kThreads - 1) / kThreads;      // of x, that a thread has on their way
    extern __shared__ __attribute__((aligned(16))) char smem[];              // x's chunk, then the waves' sums
    __shared__ int last;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % WN, wk = wave / WN;
    const int li = lane & 15, lg = lane >> 4;
    const int strip = blockIdx.x / g.parts, part = blockIdx.x - strip * g.parts, m0 = blockIdx.y * (16 * MT), rows = min(g.M - m0, 16 * MT);
    const int tile = strip * WN + wn, p0 = part * g.per, p1 = min(p0 + g.per, g.k128);
    uint64_t* const word = g.words ? g.words + (int64_t)blockIdx.y * (gridDim.x / g.parts) + strip : nullptr;
    uint64_t seen = 0;
    if (g.parts > 1 && threadIdx.x == 0) seen = arrive_look(word);

    struct Block { u32x4 w, scale[kGroups]; };
    const int64_t at = (int64_t)min(tile, g.n16 - 1) * g.k128;
    const u32x4* wp = g.words4 + at * 64 + lane;
    const uint32_t* sp = g.scales + at * (kGroups * 16) + 4 * lg;
    auto load = [&](Block& b, int kb) __attribute__((always_inline)) {
        b.w = __builtin_nontemporal_load(wp + (int64_t)kb * 64);
#pragma unroll
        for (int j = 0; j < kGroups; j++) b.scale[j] = *reinterpret_cast<const u32x4*>(sp + ((int64_t)kb * kGroups + j) * 16);
    };
    // ---- x: rows sixteen bytes longer than they are, so that sixteen rows' pieces lie in different banks; zeros behind K
    const T* const x = static_cast<const T*>(g.x) + (int64_t)m0 * g.K;
    auto piece = [&](int row, int k) __attribute__((always_inline)) {
        const T* p = x + (int64_t)row * g.K + k;
        u32x4 v = {0, 0, 0, 0};
        if (g.even) {
            if (k < g.K) v = *reinterpret_cast<const u32x4*>(p);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (k + e < g.K) v[e >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, p[e]) << 16 * (e & 1);
        }
        return v;
    };
    u32x4 ahead[kPieces];
    const int stride = kWhole ? g.chunk * (kBlockK * 2) + 16 : kStride;
    int xo[MT];                                                            // (rows behind the last are the last again; nothing is stored of them)
#pragma unroll
    for (int m = 0; m < MT; m++) xo[m] = min(16 * m + li, (kWhole ? rows : ROWS) - 1) * stride + 16 * lg;

    f32x4 acc[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    const uint32_t one = std::is_same<T, bf16_t>::value ? 0x3F803F80u : 0x3C003C00u;
    const u32x4 ones = {one, one, one, one};
    auto multiply = [&](const Block& b, const char* from, int place) __attribute__((always_inline)) {          // `place`: of the block in the chunk
#pragma unroll
        for (int j = 0; j < kGroups; j++) {
            f32x4 part[MT], total[MT];
#pragma unroll
            for (int m = 0; m < MT; m++) part[m] = total[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = j * kSteps; s < (j + 1) * kSteps; s++) {
                const u32x4 q = numbers<T>(b.w[s]);
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    const u32x4 x = *reinterpret_cast<const u32x4*>(from + xo[m] + place * (kBlockK * 2) + 64 * s);
                    part[m] = product<T>(q, x, part[m]);
                    total[m] = product<T>(ones, x, total[m]);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float scale = low_half<T>(b.scale[j][r]), zero = high_half<T>(b.scale[j][r]);
#pragma unroll
                for (int m = 0; m < MT; m++) acc[m][r] = fmaf(scale, fmaf(-zero, total[m][r], part[m][r]), acc[m][r]);
            }
        }
    };
    // ---- a block's words are asked for U blocks ahead, across the chunks of x: a wave's next block is in blk[0] again behind U WK blocks, so that all chunks but a part's last are whole turns of so many (few_of)
    Block blk[U];
#pragma unroll
    for (int u = 0; u < U; u++)
        if (p0 + wk + u * WK < p1) load(blk[u], p0 + wk + u * WK);
    if constexpr (kWhole) {
        for (int c0 = p0; c0 < p1; c0 += g.chunk) {
            const int c1 = min(c0 + g.chunk, p1), pieces = (c1 - c0) * (kBlockK / 8);
            if (c0 > p0) __syncthreads();                                    // (the chunk before has been read)
            for (int i0 = threadIdx.x; i0 < rows * pieces; i0 += kPieces * kThreads) {
                int to[kPieces];
#pragma unroll
                for (int j = 0; j < kPieces; j++) {
                    const int i = min(i0 + j * kThreads, rows * pieces - 1), row = i / pieces, at = i - row * pieces;
                    to[j] = row * stride + at * 16;
                    ahead[j] = piece(row, c0 * kBlockK + at * 8);
                }
#pragma unroll
                for (int j = 0; j < kPieces; j++) *reinterpret_cast<u32x4*>(smem + to[j]) = ahead[j];
            }
            __syncthreads();
            for (int kb = c0 + wk; kb < c1; kb += U * WK) {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (kb + u * WK >= c1) break;
                    multiply(blk[u], smem, kb + u * WK - c0);
                    if (kb + (u + U) * WK < p1) load(blk[u], kb + (u + U) * WK);
                }
            }
        }
    } else {
        auto fetch = [&](int c0) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < kPieces; j++) {
                const int i = threadIdx.x + j * kThreads;
                ahead[j] = piece(min(i / kRowPieces, rows - 1), c0 * kBlockK + i % kRowPieces * 8);
            }
        };
        fetch(p0);
        int which = 0;
        for (int turn = p0; turn < p1; turn += U * WK) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (u % (kWhole ? 1 : CU) == 0) {
                    const int c0 = turn + u * WK;
                    if (c0 >= p1) break;
                    char* const to = smem + which * (ROWS * kStride);         // (whose last readers have passed the barrier of the chunk between)
#pragma unroll
                    for (int j = 0; j < kPieces; j++) {
                        const int i = threadIdx.x + j * kThreads;
                        if (kPieces * kThreads == ROWS * kRowPieces || i < ROWS * kRowPieces) *reinterpret_cast<u32x4*>(to + i / kRowPieces * kStride + i % kRowPieces * 16) = ahead[j];
                    }
                    __syncthreads();
                    if (c0 + kChunk < p1) fetch(c0 + kChunk);
                    which ^= 1;
                }
                const int kb = turn + u * WK + wk;
                if (kb < p1) {
                    multiply(blk[u], smem + (which ^ 1) * (ROWS * kStride), u % (kWhole ? 1 : CU) * WK + wk);
                    if (kb + U * WK < p1) load(blk[u], kb + U * WK);
                }
            }
        }
    }
    if (g.parts > 1 && threadIdx.x == 0) arrive_claim(word, seen, g.tag);

    // ---- sums, as their lanes hold them: lane (li, lg) has row li of C's sixteen and columns 4 lg .. 4 lg + 3.  Item t of the workgroup's is lane t % 64 of row group t / 64 % MT of its tile t / (64 MT)
    constexpr int kItems = WN * MT * 64, kMine = (kItems + kThreads - 1) / kThreads;
    __syncthreads();
    f32x4* sums = reinterpret_cast<f32x4*>(smem);
#pragma unroll
    for (int m = 0; m < MT; m++) sums[(wk * WN + wn) * (MT * 64) + m * 64 + lane] = acc[m];
    __syncthreads();
    f32x4 sum[kMine];
#pragma unroll
    for (int i = 0; i < kMine; i++) {
        const int t = min((int)threadIdx.x + i * kThreads, kItems - 1);
        sum[i] = sums[t];
#pragma unroll
        for (int w = 1; w < WK; w++) sum[i] += sums[w * kItems + t];
    }
    if (g.parts > 1) {
        const int64_t strips = gridDim.x / g.parts, own = ((int64_t)blockIdx.y * strips + strip) * g.parts;
        const __amdgpu_buffer_rsrc_t rs = parts_rsrc(reinterpret_cast<const char*>(g.sums) + own * (kItems * 16));
#pragma unroll
        for (int i = 0; i < kMine; i++)
            if ((int)threadIdx.x + i * kThreads < kItems) store_part(rs, (uint32_t)(part * kItems + (int)threadIdx.x + i * kThreads) * 16, sum[i]);
        if (!arrive_last(word, g.parts, &last)) return;
#pragma unroll
        for (int i = 0; i < kMine; i++) sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int q0 = 0; q0 < g.parts; q0 += 4) {
            f32x4 v[4][kMine];
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int i = 0; i < kMine; i++) v[q][i] = load_part(rs, (uint32_t)(min(q0 + q, g.parts - 1) * kItems + min((int)threadIdx.x + i * kThreads, kItems - 1)) * 16);
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int i = 0; i < kMine; i++)
                    if (q0 + q < g.parts) sum[i] += v[q][i];
        }
    }
    // Four neighbouring results by themselves, from row `first` of sixteen on, by a wave whose lanes share K eight columns at a time: s (q - z) is a number, and x meets it as it is.  (us, one row of 4096 x 14336 with
    // an infinity: 32, of which 10 are the product, and 826 with each lane by itself; a NaN ends it where it is met.)
    auto by_weights = [&](int row, int sixteen, int first) __attribute__((always_inline)) {
        f32x4 y = {0.f, 0.f, 0.f, 0.f};
        const uint32_t* words = reinterpret_cast<const uint32_t*>(g.words4 + (int64_t)sixteen * g.k128 * 64 + first);
        const uint32_t* pairs = g.scales + (int64_t)sixteen * g.k128 * (kGroups * 16) + first;
#pragma unroll 1
        for (int k0 = 0; k0 < g.K; k0 += 512) {
            const int k = k0 + 8 * lane;
            if (k < g.K) {
                const u32x4 eight = piece(row, k);
                const int64_t kb = k / kBlockK;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const uint32_t word = words[(kb * 64 + 16 * (k / 8 % 4) + r) * 4 + k / 32 % 4], pair = pairs[(k / GROUP) * (int64_t)16 + r];
                    const float scale = low_half<T>(pair), zero = high_half<T>(pair);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float q = (float)(word >> (8 * (e & 3) + 4 * (e >> 2)) & 15);
                        y[r] = fmaf(scale * (q - zero), e & 1 ? high_half<T>(eight[e >> 1]) : low_half<T>(eight[e >> 1]), y[r]);
                    }
                }
            }
            if (__any(y[0] != y[0]) && __any(y[1] != y[1]) && __any(y[2] != y[2]) && __any(y[3] != y[3])) break;
        }
#pragma unroll
        for (int r = 0; r < 4; r++) y[r] = wave_sum(y[r]);
        return y;
    };
#pragma unroll
    for (int i = 0; i < kMine; i++) {
        const int t = threadIdx.x + i * kThreads, row = 16 * (t / 64 % MT) + (t & 15), col = (strip * WN + t / (64 * MT)) * 16 + 4 * (t >> 4 & 3);
        const bool mine = t < kItems && row < rows && col < g.N;
        auto wild = [&](int e) __attribute__((always_inline)) { return !(fabsf(sum[i][e]) < INFINITY); };
        for (uint64_t left = __ballot(mine && (wild(0) || wild(1) || wild(2) || wild(3))); left; left &= left - 1) {
            const int l = __builtin_ctzll(left), at = __builtin_amdgcn_readlane(col, l);
            const f32x4 y = by_weights(__builtin_amdgcn_readlane(row, l), at / 16, at % 16);
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (lane == l && wild(e)) sum[i][e] = y[e];
        }
        if (!mine) continue;
        const int64_t place = (int64_t)(m0 + row) * g.N + col;
        T* c = static_cast<T*>(g.c) + place;
        const T *res = static_cast<const T*>(g.residual) + place, *bias = static_cast<const T*>(g.bias) + col;
        Pack4<T> o, r{}, b{};
        const int n = min(g.N - col, 4);
        if (g.whole) {
            if (g.bias) b = *reinterpret_cast<const Pack4<T>*>(bias);
            if (g.residual) r = *reinterpret_cast<const Pack4<T>*>(res);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (g.bias && e < n) b.v[e] = bias[e];
                if (g.residual && e < n) r.v[e] = res[e];
            }
        }
        dispatch_act(g.act, [&](auto act_tag) {
            constexpr int ACT = decltype(act_tag)::value;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float y = apply_act_c<ACT>(g.bias ? sum[i][e] + Elem<T>::to_f32(b.v[e]) : sum[i][e]);
                o.v[e] = Elem<T>::from_f32(g.residual ? y + Elem<T>::to_f32(r.v[e]) : y);
            }
        });
        if (g.whole) {
            *reinterpret_cast<Pack4<T>*>(c) = o;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (e < n) c[e] = o.v[e];
        }
    }
}

// W as 16-bit numbers [N][stride] (zeros behind K), each rounded once: a wave a kilobyte of words.  The product's operands are of the tensors' type: exact ones would be q, and every
// group's sums would have to leave the matrix unit to be scaled, as above, which is no quicker from 129 rows on.  Half a step of each weight is, of independent signs, as much of a result as its own rounding: relative to the
// result's norm, against 64 bits, 1500 rows of 4000 -> 4104 in f16 are off by 2.5e-4 so and by 2.1e-4 with fp32 weights and one rounding.
template <typename T, int GROUP>
__global__ __launch_bounds__(256) void w4_widen_kernel(const u32x4* words, const uint32_t* scales, T* out, int N, int K, int n16, int k128, int stride) {
    constexpr int kGroups = kBlockK / GROUP;
    const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    for (int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); unit < (int64_t)n16 * k128; unit += (int64_t)gridDim.x * 4) {
        const int tile = (int)(unit / k128), kb = (int)(unit - (int64_t)tile * k128), n = tile * 16 + li;
        const u32x4 w = __builtin_nontemporal_load(words + unit * 64 + lane);
        if (n >= N) continue;
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const int k = kb * kBlockK + 32 * s + 8 * lg;
            const uint32_t pair = scales[(unit * kGroups + 32 * s / GROUP) * 16 + li];
            const float scale = low_half<T>(pair), zero = high_half<T>(pair);
            if (k >= stride) continue;
            Vec16<T> v;
#pragma unroll
            for (int e = 0; e < 8; e++) v.v[e] = Elem<T>::from_f32(k + e < K ? ((float)((w[s] >> (8 * (e & 3) + 4 * (e >> 2))) & 15) - zero) * scale : 0.f);
            store16(out + (int64_t)n * stride + k, v);
        }
    }
}

// x [M][K] with rows of `stride` (zeros behind K)
__global__ __launch_bounds__(256) void w4_pad_kernel(const uint16_t* x, uint16_t* out, int64_t all, int K, int stride) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / stride;
        const int k = (int)(i - row * stride);
        out[i] = k < K ? x[row * K + k] : 0;
    }
}

// The words, scales and zeros of a matrix: of each group lo = min(w, 0) and hi = max(w, 0), s = (hi - lo) / 15 rounded to T, z = round(-lo / s), q = round(w / s) + z within 0 .. 15, so that
// zero is held exactly and the ends of the range to half a step.  A wave a kilobyte of words: lane l has the 32 weights that its words will hold.
template <typename S, typename T, int GROUP>
__global__ __launch_bounds__(256) void w4_quantize_kernel(const S* w, int64_t stride_n, int64_t stride_k, u32x4* words, uint32_t* scales, int N, int K, int n16, int k128) {
    constexpr int kGroups = kBlockK / GROUP, kSteps = GROUP / 32;
    const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    const float most = std::is_same<T, bf16_t>::value ? 0x1.FEp127f : 65504.f;
    for (int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); unit < (int64_t)n16 * k128; unit += (int64_t)gridDim.x * 4) {
        const int tile = (int)(unit / k128), kb = (int)(unit - (int64_t)tile * k128), n = tile * 16 + li;
        u32x4 out;
#pragma unroll
        for (int j = 0; j < kGroups; j++) {
            float v[kSteps][8], lo = 0.f, hi = 0.f;
#pragma unroll
            for (int s = 0; s < kSteps; s++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int k = kb * kBlockK + 32 * (j * kSteps + s) + 8 * lg + e;
                    v[s][e] = n < N && k < K ? Elem<S>::to_f32(w[n * stride_n + k * stride_k]) : 0.f;
                    lo = fminf(lo, v[s][e]);
                    hi = fmaxf(hi, v[s][e]);
                }
            lo = fminf(lo, __shfl_xor(lo, 16, 64));
            hi = fmaxf(hi, __shfl_xor(hi, 16, 64));
            lo = fminf(lo, __shfl_xor(lo, 32, 64));
            hi = fmaxf(hi, __shfl_xor(hi, 32, 64));
            const T held = Elem<T>::from_f32(fminf(hi / 15.f - lo / 15.f, most));
            const float scale = Elem<T>::to_f32(held), zero = scale > 0.f ? fminf(rintf(-lo / scale), 15.f) : 0.f;
#pragma unroll
            for (int s = 0; s < kSteps; s++) {
                uint32_t word = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float q = scale > 0.f ? fminf(fmaxf(rintf(v[s][e] / scale) + zero, 0.f), 15.f) : 0.f;
                    word |= (uint32_t)q << (8 * (e & 3) + 4 * (e >> 2));
                }
                out[j * kSteps + s] = word;
            }
            if (lg == 0)
                scales[(unit * kGroups + j) * 16 + li] = (uint32_t)__builtin_bit_cast(uint16_t, held) | (uint32_t)__builtin_bit_cast(uint16_t, Elem<T>::from_f32(zero)) << 16;
        }
        words[unit * 64 + lane] = out;
    }
}

// Rows from which on W is widened in front of a product.
constexpr int64_t kManyRows = 129;

int check_w4(const char* what, const mhip_w4* w, int dtype) {
    if (!w) return fail(MHIP_ERR_INVALID_ARGUMENT, "%s: NULL weights", what);
    if (w->N < 0 || w->K < 0) return fail(MHIP_ERR_INVALID_ARGUMENT, "%s: negative size", what);
    if (w->group != 32 && w->group != 64 && w->group != 128) return fail(MHIP_ERR_UNSUPPORTED, "%s: groups of %lld columns (need 32, 64 or 128)", what, (long long)w->group);
    if (dtype != MHIP_BF16 && dtype != MHIP_F16) return fail(MHIP_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
    if (w->N > (1 << 24) || w->K > (1 << 22)) return fail(MHIP_ERR_UNSUPPORTED, "%s: more than 2^24 rows or 2^22 columns", what);
    return MHIP_OK;
}

// (workgroups of 256; the kernels go on where there is more)
int64_t blocks_for(int64_t n) { return std::min<int64_t>(n, 1 << 20); }
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// The widened W, a copy of x where its rows are off 16 bytes, and what the product itself can use.
struct Wide { int64_t stride, w, x, gemm; };
Wide wide_of(int64_t M, const mhip_w4* w, bool even, int dtype) {
    Wide r{};
    r.stride = even ? w->K : up(w->K, 64);
    r.w = up(w->N * r.stride * 2, 256);
    r.x = even ? 0 : up(M * r.stride * 2, 256);
    r.gemm = mhip_gemm_workspace(M, w->N, r.stride, 1, 0, 1, dtype);
    return r;
}

// How few rows are dealt.  Up to kFew rows: a workgroup four waves that share K of sixteen columns; more: eight waves, four to each sixteen of 32 columns, so that x is read once for these.
// (us, 16 columns | 32 | 64 | 128 a workgroup: 64 rows of 4096 x 4096 22.5 | 14.3 | 14.7 | 21.7, 16 of 4096 x 14336 - | 13.9 | 15.9 | 17.7, 40 of 1000 x 3000 - | 7.0 | 9.7 | 13.8; but 24 of 5120 x 5120
// 19.3 | 15.0 | 13.4 | 15.6)
// Parts: as many as make the device's waves (kWavesWanted, of which few rows have more) busy at once, four blocks for each wave at least, since a part is written and read again (64 rows of 4096 x 4096:
// two blocks a wave 22.7, four 14.7).
constexpr int kFew = 4, kWavesWanted = 2560, kWavesOfFew = 4096, kLdsOfFew = 64 << 10;
struct Few { int mt, wn, wk, strips, blocks, parts, per, chunk; int64_t bytes; };
// Blocks of words that a wave has on their way: what the registers hold; four groups' pairs are as many as their weights.
constexpr int blocks_ahead(int group) { return group == 32 ? 2 : 4; }
Few few_of(int64_t M, int group, int n16, int k128, bool deal) {
    Few f{};
    f.mt = M <= 16 ? 1 : M <= 32 || group == 32 ? 2 : 4;                     // (four sets of sums and four groups' pairs do not fit the registers)
    f.wn = M <= kFew ? 1 : 2;
    f.wk = 4;
    f.strips = (n16 + f.wn - 1) / f.wn;
    f.blocks = (int)((M + 16 * f.mt - 1) / (16 * f.mt));
    f.parts = 1;
    if (deal) {
        const int64_t waves = (int64_t)f.strips * f.blocks * f.wn * f.wk;
        const int most = std::max(k128 / (4 * f.wk), 1);
        f.parts = (int)std::min<int64_t>(std::min<int64_t>(((M <= kFew ? kWavesOfFew : kWavesWanted) + waves / 2) / std::max<int64_t>(waves, 1), most), 64);
        f.parts = std::max(f.parts, 1);
    }
    f.per = (k128 + f.parts - 1) / f.parts;
    f.parts = (k128 + f.per - 1) / f.per;
    const int room = kLdsOfFew / ((int)std::min<int64_t>(M, kFew) * (kBlockK * 2) + 16), turn = blocks_ahead(group) * f.wk;
    f.chunk = room < f.per ? room / turn * turn : f.per;                     // (a whole number of turns of the words: 240 | 112 | 80 | 48 blocks of one to four rows)
    f.bytes = f.parts > 1 ? up((int64_t)f.strips * f.blocks * 8, 16) + (int64_t)f.strips * f.blocks * f.parts * f.wn * f.mt * 1024 : 0;
    return f;
}

template <typename T, int GROUP, int MT, int WN, int WK, int U, int CU, int ROWS>
int launch_rows(hipStream_t st, const W4Args& a, const Few& f) {
    constexpr int kSums = WK * WN * MT * 1024, kLds = std::max(2 * ROWS * (CU * WK * kBlockK * 2 + 16), kSums);
    const int lds = CU == 0 ? std::max(a.M * (f.chunk * (kBlockK * 2) + 16), kSums) : kLds;
    auto kern = w4_rows_kernel<T, GROUP, MT, WN, WK, U, CU, ROWS>;
    if (CU && kLds > 64 << 10) {
        static const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
        if (err != hipSuccess) return fail(MHIP_ERR_LAUNCH, "linear_w4: cannot reserve %d bytes of LDS: %s", kLds, hipGetErrorString(err));
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)(f.strips * f.parts), (unsigned)f.blocks), dim3(64 * WN * WK), lds, st, a);
    return check_launch("linear_w4");
}

template <typename T, int GROUP>
int launch_group(hipStream_t st, const W4Args& a, const Few& f) {
    constexpr int U = blocks_ahead(GROUP);
    if (f.wn == 1) return launch_rows<T, GROUP, 1, 1, 4, U, 0, kFew>(st, a, f);
    if (f.mt == 1) return launch_rows<T, GROUP, 1, 2, 4, U, 2, 16>(st, a, f);
    if constexpr (GROUP != 32) {
        if (f.mt == 4) return launch_rows<T, GROUP, 4, 2, 4, U, 1, 64>(st, a, f);
    }
    return launch_rows<T, GROUP, 2, 2, 4, U, 1, 32>(st, a, f);
}

template <typename F>
int by_group(int64_t group, F&& f) {
    if (group == 32) return f(std::integral_constant<int, 32>{});
    if (group == 64) return f(std::integral_constant<int, 64>{});
    return f(std::integral_constant<int, 128>{});
}

template <typename T>
int run_w4(hipStream_t st, W4Args a, const mhip_w4* w, int dtype, void* workspace, int64_t bytes) {
    if (a.M >= kManyRows && workspace) {
        const Wide wide = wide_of(a.M, w, a.even, dtype);
        if (bytes >= wide.w + wide.x) {
            char* room = static_cast<char*>(workspace);
            T* wt = reinterpret_cast<T*>(room);
            const unsigned units = (unsigned)blocks_for(((int64_t)a.n16 * a.k128 + 3) / 4);
            const int rc = by_group(w->group, [&](auto group) {
                hipLaunchKernelGGL((w4_widen_kernel<T, decltype(group)::value>), dim3(units), dim3(256), 0, st, a.words4, a.scales, wt, a.N, a.K, a.n16, a.k128, (int)wide.stride);
                return check_launch("linear_w4");
            });
            if (rc) return rc;
            const void* x = a.x;
            if (!a.even) {
                x = room + wide.w;
                const int64_t all = a.M * wide.stride;
                hipLaunchKernelGGL(w4_pad_kernel, dim3((unsigned)blocks_for((all + 255) / 256)), dim3(256), 0, st, static_cast<const uint16_t*>(a.x), reinterpret_cast<uint16_t*>(room + wide.w), all, a.K, (int)wide.stride);
                if (const int rc2 = check_launch("linear_w4")) return rc2;
            }
            const int64_t left = std::min(bytes - wide.w - wide.x, wide.gemm);
            return mhip_gemm_ws(st, x, wt, a.bias, a.residual, a.c, a.M, a.N, wide.stride, 1, 0, 0, (int64_t)a.M * a.N, 0, 1, a.act, dtype, left > 0 ? room + wide.w + wide.x : nullptr, left);
        }
    }
    Few f = few_of(a.M, (int)w->group, a.n16, a.k128, true);
    if (f.bytes > 0 && (!workspace || bytes < f.bytes)) f = few_of(a.M, (int)w->group, a.n16, a.k128, false);
    a.parts = f.parts;
    a.per = f.per;
    a.chunk = f.chunk;
    if (f.parts > 1) {
        a.words = static_cast<uint64_t*>(workspace);
        a.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + up((int64_t)f.strips * f.blocks * 8, 16));
        a.tag = launch_tag();
    }
    return by_group(w->group, [&](auto group) { return launch_group<T, decltype(group)::value>(st, a, f); });
}

}  // namespace
}  // namespace mhip

using namespace mhip;

extern "C" int mhip_quantize_w4(void* stream, const void* w, int64_t stride_n, int64_t stride_k, const mhip_w4* out, int w_dtype, int dtype) {
    if (const int rc = check_w4("quantize_w4", out, dtype)) return rc;
    if (w_dtype != MHIP_F32 && w_dtype != MHIP_BF16 && w_dtype != MHIP_F16) return fail(MHIP_ERR_UNSUPPORTED, "quantize_w4: weights of dtype %d", w_dtype);
    if (out->N == 0 || out->K == 0) return MHIP_OK;
    if (!w || !out->words || !out->scales) return fail(MHIP_ERR_INVALID_ARGUMENT, "quantize_w4: NULL tensor");
    if (((uintptr_t)out->words | (uintptr_t)out->scales) & 15) return fail(MHIP_ERR_UNSUPPORTED, "quantize_w4: words and scales must be 16-byte aligned");
    const int n16 = (int)((out->N + 15) / 16), k128 = (int)((out->K + 127) / 128);
    const int64_t blocks = blocks_for(((int64_t)n16 * k128 + 3) / 4);
    auto go = [&](auto source, auto type) {
        using S = decltype(source);
        using T = decltype(type);
        return by_group(out->group, [&](auto group) {
            hipLaunchKernelGGL((w4_quantize_kernel<S, T, decltype(group)::value>), dim3((unsigned)blocks), dim3(256), 0, as_stream(stream), static_cast<const S*>(w), stride_n, stride_k,
                               static_cast<u32x4*>(const_cast<void*>(out->words)), static_cast<uint32_t*>(const_cast<void*>(out->scales)), (int)out->N, (int)out->K, n16, k128);
            return check_launch("quantize_w4");
        });
    };
    auto with = [&](auto type) { return w_dtype == MHIP_F32 ? go(float{}, type) : w_dtype == MHIP_BF16 ? go(bf16_t{}, type) : go(f16_t{}, type); };
    return dtype == MHIP_BF16 ? with(bf16_t{}) : with(f16_t{});
}

extern "C" int64_t mhip_linear_w4_workspace(int64_t M, const mhip_w4* w, int dtype) {
    if (M <= 0 || check_w4("linear_w4_workspace", w, dtype) || w->N == 0 || w->K == 0) return 0;
    if (M < kManyRows) return few_of(M, (int)w->group, (int)((w->N + 15) / 16), (int)((w->K + 127) / 128), true).bytes;
    const Wide even = wide_of(M, w, true, dtype), odd = wide_of(M, w, false, dtype);
    // (whether x lies on 16 bytes is not known here)
    return w->K & 7 ? odd.w + odd.x + odd.gemm : std::max(even.w + even.gemm, odd.w + odd.x + odd.gemm);
}

extern "C" int mhip_linear_w4(void* stream, const void* x, const mhip_w4* w, const void* bias, const void* residual, void* c, int64_t M, int activation, int dtype, void* workspace,
                              int64_t workspace_bytes) {
    if (const int rc = check_w4("linear_w4", w, dtype)) return rc;
    if (M < 0) return fail(MHIP_ERR_INVALID_ARGUMENT, "linear_w4: negative size");
    if (activation < MHIP_ACT_NONE || activation > MHIP_ACT_GELU_ERF) return fail(MHIP_ERR_INVALID_ARGUMENT, "linear_w4: activation %d", activation);
    if (M > (1 << 21)) return fail(MHIP_ERR_UNSUPPORTED, "linear_w4: more than 2^21 rows");
    if (M == 0 || w->N == 0) return MHIP_OK;
    if (w->K == 0) return fail(MHIP_ERR_UNSUPPORTED, "linear_w4: rows of no columns");
    if (!x || !w->words || !w->scales || !c) return fail(MHIP_ERR_INVALID_ARGUMENT, "linear_w4: NULL tensor");
    if (((uintptr_t)w->words | (uintptr_t)w->scales | (uintptr_t)workspace) & 15) return fail(MHIP_ERR_UNSUPPORTED, "linear_w4: words, scales and workspace must be 16-byte aligned");
    const W4Args a{x, static_cast<const u32x4*>(w->words), static_cast<const uint32_t*>(w->scales), bias, residual, c, (int)M, (int)w->N, (int)w->K, activation,
                   (int)((w->N + 15) / 16), (int)((w->K + 127) / 128), !(w->N & 3) && !(((uintptr_t)c | (uintptr_t)bias | (uintptr_t)residual) & 7),
                   !((w->K & 7) || ((uintptr_t)x & 15)), 1, 0, 0, nullptr, nullptr, 0};
    return dtype == MHIP_BF16 ? run_w4<bf16_t>(as_stream(stream), a, w, dtype, workspace, workspace_bytes) : run_w4<f16_t>(as_stream(stream), a, w, dtype, workspace, workspace_bytes);
}
