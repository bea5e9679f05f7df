// experts.cu -- products per expert: which kernel a call takes, and the copies of operands that TMA cannot read fast.
//
// TMA wants a base on 16 bytes and rows a multiple of 16 bytes apart.  An operand that is not so (an odd number of
// columns, a view that starts anywhere) is first copied to the workspace with its rows padded to 8 elements; the
// padding is never read as data (the tensor maps end at the true column).
//
// Rows of x read by index: with up to 12 rows an expert on average the products' kernel gathers them itself
// (tile::gather4).  A gather of four 128-byte pieces took 36 cycles of the TMA unit however it was issued, so a tile of
// 256 positions spent four times as long on them as on its MMAs (8192 x 8 of 64 experts, 2048 x 2048: 2365 us, from
// grouped rows 529 us), and warps that gather with 16-byte asynchronous copies took 1190 us (the hand-over of a stage
// from copies to tensor cores takes longer than its MMAs).  With more rows an expert, and for dW, x is copied in grouped
// order first: 70 us there, what writing it takes, of 565 in all (32 experts, 2048 x 2048: 6 rows each 57.4 us gathered,
// 60.4 copied; 32 rows each 84.1 and 61.1).
#include "common.cuh"
#include "experts.cuh"
#include "kmc_internal.h"

namespace kmc {

namespace {

constexpr int kTakeThreads = 256;
constexpr int kPieces = 4;

bool readable(const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }
int64_t padded(int64_t cols) { return (cols + 7) / 8 * 8; }
size_t a256(size_t v) { return (v + 255) & ~size_t(255); }
// Forward products of few rows take expert_rows.cu: up to four rows an expert at any size, up to sixteen where all the
// matrices together are small and the tensor-core kernel's set-up counts (device time, 16-bit, rows against tiles:
// 2048 x 2048, 8 of 64 experts: 1 row each 16 us against 19, 4 each 94 against 95, 16 each 225 against 111;
// 512 x 512, 8 experts: 1 to 4 rows each 3 us against 8, 16 each 5 against 9, 32 each 10 against 10).  The rule does not
// look at alignment or at the number of features, and misses the faster side there: rows read element by element, 333 x 515,
// 192 pairs of 32 experts 18.5 against 15.5 and 256 of 64 27.0 against 24.6 (48 of 32 11.5 against 15.4, 128 of 8 11.1
// against 11.5); few features, 64 x 1024, 256 pairs of 8, which go to the tiles, 5.5 against 13.1.
bool by_rows(const ExpertCall& c) {
    if (c.kind != kExpertForward) return false;
    const int64_t used = c.pairs < c.experts ? c.pairs : c.experts;
    return c.pairs <= 4 * used || (c.pairs <= 16 * used && used * c.n * c.d <= (8 << 20));
}
bool takes_x(const ExpertCall& c) {
    return c.x && c.rows && !(c.kind == kExpertForward && c.pairs <= 12 * (int64_t)c.experts);
}

// dst row i (cols elements, ldp apart) = src row idx[i], or row i without idx; zeros for a row outside src and in the
// padding
struct Take {
    const uint16_t* src;
    int64_t src_rows, ld, rows;
    const int32_t* idx;
    int cols, ldp, vec;                   // vec: rows of src can be read 16 bytes at a time
    uint16_t* dst;
};

// One or two copies in a launch (blockIdx.y): a thread writes kPieces times 16 bytes, read as one or element by element.
__global__ void __launch_bounds__(kTakeThreads) k_take(Take t0, Take t1) {
    pdl_wait();
    const Take& t = blockIdx.y == 0 ? t0 : t1;
    const int vecs = t.ldp / 8;
    const int64_t i0 = (int64_t)blockIdx.x * kTakeThreads * kPieces + threadIdx.x, all = t.rows * vecs;
    Pack<uint16_t, 8> p[kPieces];
#pragma unroll
    for (int q = 0; q < kPieces; q++) {
        const int64_t i = i0 + q * kTakeThreads;
        p[q] = {};
        if (i >= all) continue;
        const int64_t r = i / vecs;
        const int c = (int)(i - r * vecs) * 8;
        const int64_t s = t.idx ? (int64_t)__ldg(t.idx + r) : r;
        if (s < 0 || s >= t.src_rows) continue;
        if (t.vec) {
            p[q] = *reinterpret_cast<const Pack<uint16_t, 8>*>(t.src + s * t.ld + c);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (c + j < t.cols) p[q].v[j] = t.src[s * t.ld + c + j];
        }
    }
#pragma unroll
    for (int q = 0; q < kPieces; q++) {
        const int64_t i = i0 + q * kTakeThreads;
        if (i < all) *reinterpret_cast<Pack<uint16_t, 8>*>(t.dst + i * 8) = p[q];
    }
}

// The copies of one call, in the workspace
struct Takes {
    Take t[2] = {};
    int n = 0;
    char* ws;
    void add(const void** p, int64_t* ld, int64_t src_rows, const int32_t* idx, int64_t rows, int cols) {
        Take& k = t[n++];
        k.src = static_cast<const uint16_t*>(*p);
        k.src_rows = src_rows;
        k.ld = *ld;
        k.rows = rows;
        k.idx = idx;
        k.cols = cols;
        k.ldp = (int)padded(cols);
        k.vec = readable(*p, *ld) && cols % 8 == 0;
        k.dst = reinterpret_cast<uint16_t*>(ws);
        *p = ws;
        *ld = k.ldp;
        ws += a256((size_t)rows * k.ldp * 2);
    }
    cudaError_t launch(cudaStream_t st) const {
        if (n == 0) return cudaSuccess;
        int64_t most = 1;
        for (int i = 0; i < n; i++) most = t[i].rows * (t[i].ldp / 8) > most ? t[i].rows * (t[i].ldp / 8) : most;
        const int64_t blocks = (most + kTakeThreads * kPieces - 1) / (kTakeThreads * kPieces);
        if (blocks >= INT32_MAX) return cudaErrorInvalidValue;
        return launch_pdl(k_take, dim3((unsigned)blocks, n), dim3(kTakeThreads), 0, st, t[0], t[1]);
    }
};

}  // namespace

// Positions per tile: 64 where the experts' mean is at most 40 (a stage is then 24 KB and eight are in flight), 256 above
// (2048 x 2048, 32 experts: mean 32 61.4 us against 62.6, mean 64 73.8 against 65.3).
bool expert_few_rows(const ExpertCall& c) { return c.pairs <= (int64_t)c.experts * 40; }

size_t expert_bytes(const ExpertCall& c) {
    size_t need = 0;
    if (by_rows(c)) return 0;
    if (takes_x(c)) need += a256((size_t)c.pairs * padded(c.d) * 2);
    else if (c.x && !readable(c.x, c.ldx)) need += a256((size_t)c.x_rows * padded(c.d) * 2);
    if (c.w && !readable(c.w, c.d)) need += a256((size_t)c.experts * c.n * padded(c.d) * 2);
    if (c.dy && !readable(c.dy, c.n)) need += a256((size_t)c.pairs * padded(c.n) * 2);
    return need;
}

cudaError_t launch_expert(const ExpertCall& c, cudaStream_t st) {
    if (c.kind != kExpertDx && c.x_rows == 0)              // no row to read: every product is zero
        return c.kind == kExpertForward ? cudaMemsetAsync(c.y, 0, (size_t)c.pairs * c.n * 2, st)
                                        : cudaMemsetAsync(c.dw, 0, (size_t)c.experts * c.n * c.d * 2, st);
    if (c.pairs == 0) return cudaMemsetAsync(c.dw, 0, (size_t)c.experts * c.n * c.d * 2, st);
    if (by_rows(c)) return launch_expert_rows(c, st);
    Operands o = {c.x, c.w, c.dy, c.ldx, c.d, c.n, c.rows, c.x_rows};
    Takes copies;
    copies.ws = static_cast<char*>(c.ws);
    if (takes_x(c)) {
        copies.add(&o.x, &o.ldx, c.x_rows, c.rows, c.pairs, c.d);
        o.rows = nullptr;
        o.x_rows = c.pairs;
    } else if (o.x && !readable(o.x, o.ldx)) {
        copies.add(&o.x, &o.ldx, c.x_rows, nullptr, c.x_rows, c.d);
    }
    if (o.w && !readable(o.w, o.ldw)) copies.add(&o.w, &o.ldw, (int64_t)c.experts * c.n, nullptr, (int64_t)c.experts * c.n, c.d);
    if (o.dy && !readable(o.dy, o.lddy)) copies.add(&o.dy, &o.lddy, c.pairs, nullptr, c.pairs, c.n);
    if (cudaError_t e = copies.launch(st)) return e;
    return launch_expert_tc(c, o, st);
}

}  // namespace kmc
