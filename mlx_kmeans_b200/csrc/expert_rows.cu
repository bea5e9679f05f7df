// expert_rows.cu -- products of a few rows with their experts' matrices (kmc_expert_matmul for single tokens).
//
// With a few rows an expert the matrices' bytes are all there is: each is read once, 2 flops a byte and row.  A CTA
// takes 8 features of an expert that has a row at a time, straight from memory into the B fragment of mma.m16n8k16, the
// expert's rows (16 a pass) being its A fragment: no conversions and multiply-adds, of which four rows an expert already
// cost the CUDA cores more time than the bytes take.  (A tcgen05 tile would be read through shared memory by one CTA per
// 128 features, which leaves SMs idle and costs its set-up.)  The order of the depth is free as long as both operands
// agree, so a lane's fragments are 16 consecutive bytes of a feature and of a row.  A warp has two rounds of 256
// elements of depth in flight; the blocks of 8 features of all experts that have a row are split equally over the CTAs,
// twelve warps an SM, whichever experts were chosen.
// WARPS = 1: a CTA is one warp over the whole depth.  WARPS = 4: four warps share the depth round by round and join
// their float32 sums in shared memory, in a fixed order, the next block's first round under way meanwhile; taken where
// there are too few blocks to go round (see run_rows).
// One row of 8 of 64 experts, 2048 x 2048: 16.5 us for 67 MB (0.62 of the copy bandwidth: one round of loads, ramp and
// tail count); 8 rows of them 62 us for 338 MB (0.83).
// Any size, stride and alignment: 16-byte loads where every row starts on 16 bytes, element by element otherwise.
#include <type_traits>

#include "common.cuh"
#include "experts.cuh"
#include "kmc_internal.h"

namespace kmc {

namespace {

constexpr int kFeatures = 8;
constexpr int kTokens = 16;               // rows of an expert in one pass
constexpr int kChunks = 8;                // of 32 elements of depth, in a round
constexpr int kRound = kChunks * 32;
constexpr int kWarpsPerSm = 12;
constexpr unsigned kFull = 0xffffffffu;

struct RowsArgs {
    const int32_t* offsets;
    const int32_t* rows;
    int64_t x_rows, ldx;
    int pairs, experts, n, d;
};

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 elements of p from k on, zeros past d
template <bool VEC, bool STREAM>
__device__ __forceinline__ uint4 load8(const uint16_t* p, int k, int d) {
    if constexpr (VEC) {                                   // d is a multiple of 8
        if (k >= d) return make_uint4(0u, 0u, 0u, 0u);
        const uint4* q = reinterpret_cast<const uint4*>(p + k);
        if constexpr (STREAM) return __ldcs(q);
        return __ldg(q);
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t lo = k + 2 * i < d ? __ldg(p + k + 2 * i) : 0, hi = k + 2 * i + 1 < d ? __ldg(p + k + 2 * i + 1) : 0;
        w[i] = lo | (hi << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// First position and rows of expert e (0 rows past the last expert)
__device__ __forceinline__ void segment(const RowsArgs& a, int e, int& begin, int& count) {
    begin = count = 0;
    if (e < a.experts) {
        begin = min(max(__ldg(a.offsets + e), 0), a.pairs);
        count = min(max(__ldg(a.offsets + e + 1), 0), a.pairs) - begin;
    }
}

template <typename T, bool VEC, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, kWarpsPerSm / WARPS)
    k_expert_rows(const uint16_t* __restrict__ x, const uint16_t* __restrict__ w, RowsArgs a, T* __restrict__ y) {
    __shared__ float join[2][WARPS][kTokens * kFeatures];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, kl = (lane & 3) * 8;
    pdl_wait();
    const int per = (a.n + kFeatures - 1) / kFeatures;     // blocks of features per expert
    int active = 0, begin, count;
#pragma unroll 4
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
        segment(a, e0 + lane, begin, count);
        active += __popc(__ballot_sync(kFull, count > 0));
    }
    const int64_t blocks = (int64_t)active * per;
    int64_t b = blockIdx.x * blocks / gridDim.x;
    const int64_t b1 = (blockIdx.x + 1) * blocks / gridDim.x;
    // where the CTA is: features f0 .. f0 + 7 of expert e, its rows' positions from p on, `rows` of them left
    int e = -1, f0 = (int)(b - b / per * per) * kFeatures, p = 0, rows = 0;
    auto advance = [&](int skip) {                         // to the skip-th expert with a row after e
        for (int e0 = e + 1;; e0 += 32) {
            segment(a, e0 + lane, begin, count);
            unsigned has = __ballot_sync(kFull, count > 0);
            const int n = __popc(has);
            if (skip >= n && e0 + 32 < a.experts) {
                skip -= n;
                continue;
            }
            for (; skip > 0; skip--) has &= has - 1;
            const int at = has ? __ffs(has) - 1 : 0;
            e = e0 + at;
            p = __shfl_sync(kFull, begin, at);
            rows = __shfl_sync(kFull, count, at);
            return;
        }
    };
    const uint16_t* wp = w;
    auto load = [&](uint4 (&u)[kChunks], int k) {
#pragma unroll
        for (int c = 0; c < kChunks; c++) u[c] = load8<VEC, true>(wp, k + c * 32 + kl, a.d);
    };
    auto place = [&] { wp = w + ((int64_t)e * a.n + min(f0 + g, a.n - 1)) * a.d; };   // past the last: not stored
    uint4 u0[kChunks], u1[kChunks];
    constexpr int STEP = WARPS * kRound;
    if (b < b1) {
        advance((int)(b / per));
        place();
        load(u0, warp * kRound);
    }
    for (int buf = 0; b < b1; buf ^= 1) {
        const int here = min(rows, kTokens), p0 = p, row0 = f0;
        const uint16_t* xs[2];
        bool there[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            int64_t row = -1;
            if (t * 8 + g < here) row = a.rows ? __ldg(a.rows + p + t * 8 + g) : p + t * 8 + g;
            there[t] = row >= 0 && row < a.x_rows;         // otherwise some row, whose results are not stored
            xs[t] = x + (there[t] ? row : 0) * a.ldx;
        }
        float acc[2][4] = {};
        auto multiply = [&](const uint4 (&u)[kChunks], int k) {
            uint4 v[kChunks];
#pragma unroll
            for (int c = 0; c < kChunks; c++) v[c] = load8<VEC, false>(xs[0], k + c * 32 + kl, a.d);
            if (here <= 8) {
#pragma unroll
                for (int c = 0; c < kChunks; c++) {
                    mma_16816<T>(acc[c & 1], v[c].x, 0u, v[c].y, 0u, u[c].x, u[c].y);
                    mma_16816<T>(acc[c & 1], v[c].z, 0u, v[c].w, 0u, u[c].z, u[c].w);
                }
            } else {
                uint4 z[kChunks];
#pragma unroll
                for (int c = 0; c < kChunks; c++) z[c] = load8<VEC, false>(xs[1], k + c * 32 + kl, a.d);
#pragma unroll
                for (int c = 0; c < kChunks; c++) {
                    mma_16816<T>(acc[c & 1], v[c].x, z[c].x, v[c].y, z[c].y, u[c].x, u[c].y);
                    mma_16816<T>(acc[c & 1], v[c].z, z[c].z, v[c].w, z[c].w, u[c].z, u[c].w);
                }
            }
        };
        for (int k = warp * kRound; k < a.d; k += 2 * STEP) {
            if (k + STEP < a.d) load(u1, k + STEP);
            multiply(u0, k);
            if (k + STEP >= a.d) break;
            if (k + 2 * STEP < a.d) load(u0, k + 2 * STEP);
            multiply(u1, k + STEP);
        }
        // on to the expert's further rows, the next features, or the next expert
        if (rows > kTokens) {
            p += kTokens;
            rows -= kTokens;
        } else if (++b < b1) {
            f0 += kFeatures;
            if (f0 >= a.n) {
                f0 = 0;
                advance(0);
            } else {
                segment(a, e, p, rows);                    // (its first row again)
            }
            place();
        }
        if (b < b1) load(u0, warp * kRound);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float v = there[i >> 1] ? acc[0][i] + acc[1][i] : 0.0f;            // a row outside x reads as zeros
            const int t = g + (i >> 1) * 8, f = (lane & 3) * 2 + (i & 1);
            if constexpr (WARPS > 1) join[buf][warp][t * kFeatures + f] = v;
            else if (t < here && row0 + f < a.n) y[(int64_t)(p0 + t) * a.n + row0 + f] = Elem<T>::from(v);
        }
        if constexpr (WARPS > 1) {
            __syncthreads();                               // (two buffers: the next block's sums go to the other one)
            for (int i = threadIdx.x; i < kTokens * kFeatures; i += WARPS * 32) {
                const int t = i / kFeatures, f = row0 + i % kFeatures;
                if (t < here && f < a.n) {
                    float s = join[buf][0][i];
#pragma unroll
                    for (int q = 1; q < WARPS; q++) s += join[buf][q][i];
                    y[(int64_t)(p0 + t) * a.n + f] = Elem<T>::from(s);
                }
            }
        }
    }
    // positions past the last group: zeros
    const int64_t taken = min(max(__ldg(a.offsets + a.experts), 0), a.pairs);
    for (int64_t i = taken * a.n + (int64_t)blockIdx.x * WARPS * 32 + threadIdx.x; i < (int64_t)a.pairs * a.n;
         i += (int64_t)gridDim.x * WARPS * 32)
        y[i] = Elem<T>::from(0.0f);
}

template <typename T>
cudaError_t run_rows(const ExpertCall& c, cudaStream_t st) {
    RowsArgs a;
    a.offsets = c.offsets;
    a.rows = c.rows;
    a.x_rows = c.x_rows;
    a.ldx = c.ldx;
    a.pairs = (int)c.pairs;
    a.experts = c.experts;
    a.n = c.n;
    a.d = c.d;
    auto whole = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const bool vec = c.d % 8 == 0 && c.ldx % 8 == 0 && whole(c.x) && whole(c.w);
    const int64_t blocks = (c.pairs < c.experts ? c.pairs : c.experts) * ((c.n + kFeatures - 1) / kFeatures);
    // Four warps a block divide the last round of blocks more finely and shorten a lone block, at the price of the
    // join: taken where the blocks go round in less than two thirds of the time (1 token, 8 of 64 experts, 2048 x 2048:
    // 16.5 us against 19.2; 4 tokens: 45.6 against 42.9), with at least a round of depth for each of them; and for
    // operands read element by element (1 token, 333 x 515: 5.6 us against 12.5).
    const int64_t slots = kWarpsPerSm * num_sms();
    const double one = (double)((blocks + slots - 1) / slots), four = 0.25 * (double)((4 * blocks + slots - 1) / slots);
    const bool split = !vec || (c.d >= 4 * kRound && 1.5 * four < one);
    const int warps = split ? 4 : 1;
    const int64_t grid = blocks < slots / warps ? blocks : slots / warps;
    auto kern = vec ? (split ? k_expert_rows<T, true, 4> : k_expert_rows<T, true, 1>) : k_expert_rows<T, false, 4>;
    return launch_pdl(kern, dim3((unsigned)grid), dim3(warps * 32), 0, st, static_cast<const uint16_t*>(c.x),
                      static_cast<const uint16_t*>(c.w), a, static_cast<T*>(c.y));
}

}  // namespace

cudaError_t launch_expert_rows(const ExpertCall& c, cudaStream_t st) {
    return c.dtype == 1 ? run_rows<__nv_bfloat16>(c, st) : run_rows<__half>(c, st);
}

}  // namespace kmc
