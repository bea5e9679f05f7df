// expert_simt.cu -- products of grouped rows with their expert's matrix on the CUDA cores, any size and alignment.
//
//   y_p  = W_e x_row(p)                 rows p of expert e: offsets[e] <= p < offsets[e + 1]
//   dx_p = W_e^T dy_p
//   dW_e = sum_p dy_p x_row(p)^T
// float32 products and sums, one rounding where a result is stored.  64 x 64 output tiles, 16 deep through shared
// memory, 4 x 4 outputs a thread.  Positions past offsets[E] give rows of zeros; a row index outside x reads zeros.
#include "common.cuh"
#include "experts.cuh"
#include "kmc_internal.h"

namespace kmc {

namespace {

constexpr int kT = 64, kDeep = 16, kThreads = 256;

struct SimtArgs {
    const int32_t* offsets;
    const int32_t* rows;
    int64_t x_rows, ldx, pairs;
    int experts, n, d;                    // output columns, depth
    int64_t wn, wd, we;                   // strides of w over output columns, depth, experts
};

__device__ __forceinline__ int64_t offset_of(const SimtArgs& a, int e) {
    const int64_t o = __ldg(a.offsets + e);
    return o < 0 ? 0 : o > a.pairs ? a.pairs : o;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_expert_simt(const T* __restrict__ x, const T* __restrict__ w, SimtArgs a,
                                                          T* __restrict__ y) {
    __shared__ float sx[kDeep][kT + 1], sw[kDeep][kT + 1];
    // the row tile of this CTA: expert e, positions p0 .. p1
    int64_t tile = blockIdx.x, p0 = 0, p1 = 0;
    int e = 0;
    for (; e <= a.experts; e++) {
        const int64_t o0 = e < a.experts ? offset_of(a, e) : offset_of(a, a.experts);
        const int64_t o1 = e < a.experts ? offset_of(a, e + 1) : a.pairs;
        const int64_t t = o1 > o0 ? (o1 - o0 + kT - 1) / kT : 0;
        if (tile < t) {
            p0 = o0 + tile * kT;
            p1 = min(p0 + kT, o1);
            break;
        }
        tile -= t;
    }
    if (p0 >= p1) return;
    const int n0 = blockIdx.y * kT, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    if (e < a.experts) {
        const T* we = w + e * a.we;
        for (int k0 = 0; k0 < a.d; k0 += kDeep) {
            for (int i = threadIdx.x; i < kT * kDeep; i += kThreads) {
                const int r = i / kDeep, k = i % kDeep;
                const int64_t p = p0 + r;
                int64_t row = p < p1 ? (a.rows ? (int64_t)a.rows[p] : p) : -1;
                sx[k][r] = row >= 0 && row < a.x_rows && k0 + k < a.d ? Elem<T>::to(x[row * a.ldx + k0 + k]) : 0.0f;
                sw[k][r] = n0 + r < a.n && k0 + k < a.d ? Elem<T>::to(we[(n0 + r) * a.wn + (k0 + k) * a.wd]) : 0.0f;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kDeep; k++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[i][j] = fmaf(sx[k][ty * 4 + i], sw[k][tx + 16 * j], acc[i][j]);
            __syncthreads();
        }
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const int64_t p = p0 + ty * 4 + i;
            const int n = n0 + tx + 16 * j;
            if (p < p1 && n < a.n) y[p * a.n + n] = Elem<T>::from(acc[i][j]);
        }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_expert_dw_simt(const T* __restrict__ dy, const T* __restrict__ x, SimtArgs a,
                                                             T* __restrict__ dw) {
    __shared__ float sx[kDeep][kT + 1], sg[kDeep][kT + 1];
    const int e = blockIdx.z, n0 = blockIdx.y * kT, d0 = blockIdx.x * kT;
    const int64_t o0 = offset_of(a, e), o1 = offset_of(a, e + 1);
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    for (int64_t k0 = o0; k0 < o1; k0 += kDeep) {
        for (int i = threadIdx.x; i < kT * kDeep; i += kThreads) {
            const int r = i % kT, k = i / kT;
            const int64_t p = k0 + k;
            const int64_t row = p < o1 ? (a.rows ? (int64_t)a.rows[p] : p) : -1;
            sx[k][r] = row >= 0 && row < a.x_rows && d0 + r < a.d ? Elem<T>::to(x[row * a.ldx + d0 + r]) : 0.0f;
            sg[k][r] = p < o1 && n0 + r < a.n ? Elem<T>::to(dy[p * a.n + n0 + r]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kDeep; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = fmaf(sg[k][ty * 4 + i], sx[k][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const int n = n0 + ty * 4 + i, d = d0 + tx + 16 * j;
            if (n < a.n && d < a.d) dw[((int64_t)e * a.n + n) * a.d + d] = Elem<T>::from(acc[i][j]);
        }
}

template <typename T>
cudaError_t run_simt(const ExpertCall& c, cudaStream_t st) {
    SimtArgs a;
    a.offsets = c.offsets;
    a.rows = c.rows;
    a.x_rows = c.x_rows;
    a.ldx = c.ldx;
    a.pairs = c.pairs;
    a.experts = c.experts;
    a.we = (int64_t)c.n * c.d;
    const int64_t tiles = c.pairs / kT + (c.pairs < c.experts ? c.pairs : c.experts) + 1;
    switch (c.kind) {
        case kExpertForward:
            a.n = c.n, a.d = c.d, a.wn = c.d, a.wd = 1;
            k_expert_simt<T><<<dim3((unsigned)tiles, (a.n + kT - 1) / kT), kThreads, 0, st>>>(
                static_cast<const T*>(c.x), static_cast<const T*>(c.w), a, static_cast<T*>(c.y));
            break;
        case kExpertDx:
            a.n = c.d, a.d = c.n, a.wn = 1, a.wd = c.d, a.rows = nullptr, a.x_rows = c.pairs, a.ldx = c.n;
            k_expert_simt<T><<<dim3((unsigned)tiles, (a.n + kT - 1) / kT), kThreads, 0, st>>>(
                static_cast<const T*>(c.dy), static_cast<const T*>(c.w), a, static_cast<T*>(c.dx));
            break;
        default:
            a.n = c.n, a.d = c.d;
            k_expert_dw_simt<T><<<dim3((a.d + kT - 1) / kT, (a.n + kT - 1) / kT, c.experts), kThreads, 0, st>>>(
                static_cast<const T*>(c.dy), static_cast<const T*>(c.x), a, static_cast<T*>(c.dw));
    }
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_expert(const ExpertCall& c, cudaStream_t st) {
    return c.dtype == 1 ? run_simt<__nv_bfloat16>(c, st) : run_simt<__half>(c, st);
}

size_t expert_bytes(const ExpertCall&) { return 0; }

}  // namespace kmc
