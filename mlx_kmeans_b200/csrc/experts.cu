// experts.cu -- products per expert: which kernel a call takes, and the copies of operands that TMA cannot read.
//
// TMA wants a base on 16 bytes and rows a multiple of 16 bytes apart.  An operand that is not so (an odd number of
// columns, a view that starts anywhere) is first copied to the workspace with its rows padded to 8 elements; the
// padding is never read as data (the tensor maps end at the true column).
#include "common.cuh"
#include "experts.cuh"
#include "kmc_internal.h"

namespace kmc {

namespace {

constexpr int kPadThreads = 256;

bool readable(const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }
int64_t padded(int64_t cols) { return (cols + 7) / 8 * 8; }
size_t a256(size_t v) { return (v + 255) & ~size_t(255); }

// rows x cols elements, ld apart, to rows ldp apart: a thread writes 16 bytes
__global__ void __launch_bounds__(kPadThreads)
    k_pad_rows(const uint16_t* __restrict__ src, int64_t rows, int cols, int64_t ld, int ldp, uint16_t* __restrict__ dst) {
    pdl_wait();
    const int vecs = ldp / 8;
    const int64_t i = (int64_t)blockIdx.x * kPadThreads + threadIdx.x;
    if (i >= rows * vecs) return;
    const int64_t r = i / vecs;
    const int c = (int)(i - r * vecs) * 8;
    Pack<uint16_t, 8> p;
#pragma unroll
    for (int j = 0; j < 8; j++) p.v[j] = c + j < cols ? src[r * ld + c + j] : (uint16_t)0;
    *reinterpret_cast<Pack<uint16_t, 8>*>(dst + r * ldp + c) = p;
}

cudaError_t pad(const void** p, int64_t* ld, int64_t rows, int cols, char** ws, cudaStream_t st) {
    if (readable(*p, *ld)) return cudaSuccess;
    const int64_t ldp = padded(cols), blocks = (rows * (ldp / 8) + kPadThreads - 1) / kPadThreads;
    cudaError_t e = launch_pdl(k_pad_rows, dim3((unsigned)blocks), dim3(kPadThreads), 0, st,
                               static_cast<const uint16_t*>(*p), rows, cols, *ld, (int)ldp, reinterpret_cast<uint16_t*>(*ws));
    *p = *ws;
    *ld = ldp;
    *ws += a256((size_t)rows * ldp * 2);
    return e;
}

}  // namespace

size_t expert_bytes(const ExpertCall& c) {
    size_t need = 0;
    if (c.x && !readable(c.x, c.ldx)) need += a256((size_t)c.x_rows * padded(c.d) * 2);
    if (c.w && !readable(c.w, c.d)) need += a256((size_t)c.experts * c.n * padded(c.d) * 2);
    if (c.dy && !readable(c.dy, c.n)) need += a256((size_t)c.pairs * padded(c.n) * 2);
    return need;
}

cudaError_t launch_expert(const ExpertCall& c, cudaStream_t st) {
    if (c.kind != kExpertDx && c.x_rows == 0)              // no row to read: every product is zero
        return c.kind == kExpertForward ? cudaMemsetAsync(c.y, 0, (size_t)c.pairs * c.n * 2, st)
                                        : cudaMemsetAsync(c.dw, 0, (size_t)c.experts * c.n * c.d * 2, st);
    if (c.pairs == 0) return cudaMemsetAsync(c.dw, 0, (size_t)c.experts * c.n * c.d * 2, st);
    Operands o = {c.x, c.w, c.dy, c.ldx, c.d, c.n};
    char* ws = static_cast<char*>(c.ws);
    cudaError_t e = cudaSuccess;
    if (o.x) e = pad(&o.x, &o.ldx, c.x_rows, c.d, &ws, st);
    if (e == cudaSuccess && o.w) e = pad(&o.w, &o.ldw, (int64_t)c.experts * c.n, c.d, &ws, st);
    if (e == cudaSuccess && o.dy) e = pad(&o.dy, &o.lddy, c.pairs, c.n, &ws, st);
    return e == cudaSuccess ? launch_expert_tc(c, o, st) : e;
}

}  // namespace kmc
