// combine.cu -- joining the experts' answers (kmc_combine) and its gradient (kmc_combine_grad).
//
//   out_t = sum_j w_tj y_slot(t,j)          dy_slot(t,j) = w_tj dout_t          dw_tj = <dout_t, y_slot(t,j)>
// w = 1 without weights; a pair with slot -1 adds nothing (dw 0), and a row of dy that no pair has is 0.  Which rows those
// are is found from the slots, in a launch before (a caller may drop pairs of a plan by their slots), or from the plan's
// offsets where the caller says that none was dropped.  Sums run in
// float32 in the order j = 0 .. k - 1 (out) or in a fixed tree over the row (dw), and are rounded once when stored; y may
// be float32 where out is 16-bit (a row's gradients by position, from expert_tc.cu).
//
// Memory bound.  Forward: one thread per 16 bytes of out, its k reads of y independent and in flight together; each
// row of y is read once and each row of out written once.  Backward: one warp per pair reads dout_t (the k warps of a
// row run side by side, so it comes from L1 / L2 after the first) and y's row once and writes dy's row.  16384 rows of 8
// choices, 2048 features, bfloat16: both in 281 us, where their bytes (1.74 GB) take 266 at the copy bandwidth.
#include <type_traits>

#include "common.cuh"
#include "experts.cuh"
#include "kmc_internal.h"

namespace kmc {

namespace {

constexpr int kCombineThreads = 256;

struct CombineArgs {
    const int32_t* slot;
    const float* weights;
    const int32_t* taken;                 // device: positions that a pair has (offsets[E]), or nullptr: see pair_of
    int32_t* pair_of;                     // a pair per position, any value where there is none
    int64_t tokens, pairs;
    int choices, width;                   // width: features
};

template <typename T, typename O, int V>
__global__ void __launch_bounds__(kCombineThreads) k_combine(const T* __restrict__ y, CombineArgs a, O* __restrict__ out) {
    pdl_wait();
    const int vecs = a.width / V;
    const int64_t i = (int64_t)blockIdx.x * kCombineThreads + threadIdx.x;
    if (i >= a.tokens * vecs) return;
    const int64_t t = i / vecs;
    const int f = (int)(i - t * vecs) * V;
    const int32_t* slot = a.slot + t * a.choices;
    float acc[V];
#pragma unroll
    for (int v = 0; v < V; v++) acc[v] = 0.0f;
#pragma unroll 4
    for (int j = 0; j < a.choices; j++) {
        const int64_t s = __ldg(slot + j);
        if (s < 0 || s >= a.pairs) continue;
        const float w = a.weights ? __ldg(a.weights + t * a.choices + j) : 1.0f;
        const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(y + s * a.width + f);
#pragma unroll
        for (int v = 0; v < V; v++) acc[v] = fmaf(w, Elem<T>::to(p.v[v]), acc[v]);
    }
    Pack<O, V> r;
#pragma unroll
    for (int v = 0; v < V; v++) r.v[v] = Elem<O>::from(acc[v]);
    *reinterpret_cast<Pack<O, V>*>(out + t * a.width + f) = r;
}

// The pair of each position that has one; the others keep what they held, which has_pair sees through, so nothing is
// cleared first.
__global__ void __launch_bounds__(kCombineThreads) k_pair_of(CombineArgs a) {
    pdl_wait();
    const int64_t p = (int64_t)blockIdx.x * kCombineThreads + threadIdx.x;
    if (p >= a.pairs) return;
    const int64_t s = __ldg(a.slot + p);
    if (s >= 0 && s < a.pairs) a.pair_of[s] = (int32_t)p;
}
// Whether some pair points at position p
__device__ __forceinline__ bool has_pair(const CombineArgs& a, int64_t p) {
    if (a.taken) return p < __ldg(a.taken);
    const int64_t q = __ldcg(a.pair_of + p);
    return q >= 0 && q < a.pairs && __ldg(a.slot + q) == p;
}

template <typename T, int V>
__global__ void __launch_bounds__(kCombineThreads)
    k_combine_grad(const T* __restrict__ dout, const T* __restrict__ y, CombineArgs a, T* __restrict__ dy,
                   float* __restrict__ dw) {
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t p = (int64_t)blockIdx.x * (kCombineThreads / 32) + (threadIdx.x >> 5);
    if (p >= a.pairs) return;
    const int64_t s = __ldg(a.slot + p);
    if (!has_pair(a, p)) {                // its row of dy is 0
        for (int f = lane * V; f < a.width; f += 32 * V) {
            Pack<T, V> z;
#pragma unroll
            for (int v = 0; v < V; v++) z.v[v] = Elem<T>::from(0.0f);
            *reinterpret_cast<Pack<T, V>*>(dy + p * a.width + f) = z;
        }
    }
    const bool got = s >= 0 && s < a.pairs;
    float dot = 0.0f;
    if (got) {
        const float w = a.weights ? __ldg(a.weights + p) : 1.0f;
        const T* g = dout + p / a.choices * a.width;
#pragma unroll 4
        for (int f = lane * V; f < a.width; f += 32 * V) {
            const Pack<T, V> q = *reinterpret_cast<const Pack<T, V>*>(g + f);
            Pack<T, V> r;
            if (dw) {
                const Pack<T, V> u = *reinterpret_cast<const Pack<T, V>*>(y + s * a.width + f);
#pragma unroll
                for (int v = 0; v < V; v++) dot = fmaf(Elem<T>::to(q.v[v]), Elem<T>::to(u.v[v]), dot);
            }
#pragma unroll
            for (int v = 0; v < V; v++) r.v[v] = Elem<T>::from(w * Elem<T>::to(q.v[v]));
            *reinterpret_cast<Pack<T, V>*>(dy + s * a.width + f) = r;
        }
    }
    if (dw) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (lane == 0) dw[p] = dot;
    }
}

template <typename T, typename O, int V>
cudaError_t run_combine(const CombineCall& c, cudaStream_t st) {
    CombineArgs a;
    a.slot = c.slot;
    a.weights = c.weights;
    a.taken = c.taken;
    a.pair_of = c.pair_of;
    a.tokens = c.tokens;
    a.pairs = c.tokens * c.choices;
    a.choices = c.choices;
    a.width = c.width;
    if (c.dout == nullptr) {
        const int64_t blocks = (a.tokens * (a.width / V) + kCombineThreads - 1) / kCombineThreads;
        return launch_pdl(k_combine<T, O, V>, dim3((unsigned)blocks), dim3(kCombineThreads), 0, st,
                          static_cast<const T*>(c.y), a, static_cast<O*>(c.out));
    }
    if constexpr (std::is_same<T, O>::value) {
        if (!a.taken) {
            const int64_t blocks = (a.pairs + kCombineThreads - 1) / kCombineThreads;
            if (cudaError_t e = launch_pdl(k_pair_of, dim3((unsigned)blocks), dim3(kCombineThreads), 0, st, a)) return e;
        }
        const int64_t blocks = (a.pairs + kCombineThreads / 32 - 1) / (kCombineThreads / 32);
        return launch_pdl(k_combine_grad<T, V>, dim3((unsigned)blocks), dim3(kCombineThreads), 0, st,
                          static_cast<const T*>(c.dout), static_cast<const T*>(c.y), a, static_cast<T*>(c.dy),
                          c.dweights);
    }
    return cudaErrorInvalidValue;         // (no gradient of the form with a float32 y)
}

// 16 bytes per access to y where every row starts on a 16-byte boundary, one element otherwise
template <typename T, typename O>
cudaError_t run_combine_type(const CombineCall& c, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    if (c.width % V == 0 && aligned(c.y) && aligned(c.out) && aligned(c.dout) && aligned(c.dy))
        return run_combine<T, O, V>(c, st);
    return run_combine<T, O, 1>(c, st);
}

}  // namespace

cudaError_t launch_combine(const CombineCall& c, cudaStream_t st) {
    switch (c.dtype) {
        case 0: return run_combine_type<float, float>(c, st);
        case 1:
            return c.sum_f32 ? run_combine_type<float, __nv_bfloat16>(c, st) : run_combine_type<__nv_bfloat16, __nv_bfloat16>(c, st);
        default: return c.sum_f32 ? run_combine_type<float, __half>(c, st) : run_combine_type<__half, __half>(c, st);
    }
}

}  // namespace kmc
