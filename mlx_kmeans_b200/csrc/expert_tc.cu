// expert_tc.cu -- products of grouped rows with their expert's matrix on the tensor cores (tcgen05 + TMEM + TMA).
//
//   forward  y_p  = W_e x_row(p)              positions p of expert e: offsets[e] <= p < offsets[e + 1]
//   dx       dx_p = W_e^T dy_p
//   dW       dW_e = sum_p dy_p x_row(p)^T
// 16-bit operands, float32 accumulation in TMEM, one rounding to 16 bits when a result is stored; dx can be stored in
// float32, for rows whose positions are summed afterwards.
//
// The matrix is the MMA's A operand: features are its M rows, and up to COLS positions its N columns.  N is a run-time
// field of the instruction, so a group of any number of rows costs that number rounded up to 16 (32 for a pair of
// CTAs), not to a tile of 128, and an expert's rows are cut into equal tiles rather than full ones and a rest.  For dx
// the same matrix is read as its transpose (an MN-major A operand); dW takes both operands MN-major, with the positions
// as the depth, so nothing is transposed in memory.
//
// PAIR: two CTAs of a cluster share each MMA (cta_group::2): 256 features x up to 256 positions, each CTA holding 128
// of the features and half of the positions, so a stage of 64 deep is 32 KB a CTA instead of 48 KB for the same work
// (what the L2 can deliver bounds the single-CTA tile).  GATHER (few rows an expert): x's rows are read in place by
// their indices (tile::gather4, four rows an instruction).  A row index past the tensor is filled with zeros by TMA:
// positions past a group's end in dW are loaded that way, so no other group's value (a NaN, say) enters the sum; in
// forward and dx a neighbour's row can only reach columns that are not stored.
//
// Measured (bfloat16, the kernel alone in short bursts): 8192^3 in one group 805 us, 1366 TFLOP/s; 65536 rows of 64
// groups, 2048 x 2048, forward and dx 1110 TFLOP/s, dW 1050 (a forward pass in a row of passes, the copy of x in grouped
// order included and under the power limit: 666 us, 825); 16396 rows of 16 groups, 1536 x 2048, 1000 TFLOP/s, dx with
// float32 results 930, the tensor pipe 53 to 58% busy.  Without its loads the first takes 682 us and without L2 misses
// 755 us, so operands on their way to shared memory bound it (32 KB a stage and CTA, about 45 bytes a cycle), then the
// tensor cores.
//
// Kernel layout (persistent, one CTA per SM): warp 0 loads (TMA), warp 1 issues the MMAs (64 deep a stage; in a pair
// the leader's alone), warps 2-5 store the finished accumulator while the next one is computed (two accumulators in
// TMEM).  Every wait on an mbarrier is bounded; on a timeout the CTA sets the error word, waits for its loads and MMAs
// in flight, and frees TMEM.
#include <cuda.h>

#include <type_traits>

#include "common.cuh"
#include "experts.cuh"
#include "kmc_internal.h"
#include "tcgen05.cuh"

namespace kmc {

namespace {

constexpr int kFeat = 128;                // features per CTA and tile (the MMA's M, or half of it)
constexpr int kDepth = 64;                // depth per stage: one 128-byte swizzle row of 16-bit elements
constexpr int kBox = 64 * kDepth * 2;     // 64 x 64 elements
constexpr int kBlock = 8;                 // position tiles per block of the tile order
constexpr int kTcThreads = 192;
constexpr int kEpiThreads = 128;
constexpr int kEpiBytes = 32 * 80;        // a warp's 32 x 32 results on their way from TMEM to memory
constexpr unsigned kFull = 0xffffffffu;

struct TcArgs {
    const int32_t* offsets;
    const int32_t* rows;
    int64_t x_rows;
    int pairs, experts;
    int feats;                            // M side in all: n (forward, dW), d (dx)
    int cols;                             // dW: N side in all (d); otherwise unused
    int depth;                            // forward: d, dx: n; dW: per expert
    int most;                             // positions per tile at most (forward, dx): COLS, or fewer (see run_tc)
    void* out;
    int64_t ldo;                          // row length of out
    int out_f32;                          // dx: out is float32
    int out_vec;                          // rows of out start on 16-byte boundaries
    int* error;
};

// Loads by index or of the end of a group: rows of x (GATHER), and for dW 16 rows and single rows of dy and x
struct Tails {
    CUtensorMap a16, a_row, b16, b_row;
};

template <int COLS, bool PAIR>
struct TcSmem {
    static constexpr int MINE = PAIR ? COLS / 2 : COLS;       // columns whose operand this CTA holds
    static constexpr int A = kFeat * kDepth * 2;
    static constexpr int B = MINE * kDepth * 2;
    static constexpr int STAGE = A + B;
    static constexpr int BAR = 256;
    static constexpr int EPI = 4 * kEpiBytes;
    static constexpr int EXPERTS = (kGroupMaxExperts + 1) * 4;
    static constexpr int FREE = 227 * 1024 - BAR - EPI - EXPERTS - 2048;   // 1 KB to align, 1 KB of static arrays
    static constexpr int NS = FREE / STAGE > 8 ? 8 : FREE / STAGE;
    static constexpr int base = NS * STAGE + BAR + EPI + 1024;      // + the experts' tile counts
    static_assert(NS >= 2 && 8 * (2 * NS + 5) + 8 <= BAR, "barrier block");
};

// Positions of expert e, with offsets that a caller made wrong kept inside the arrays.
__device__ __forceinline__ void segment(const TcArgs& a, int e, int& begin, int& count) {
    const int o0 = min(max(__ldg(a.offsets + e), 0), a.pairs), o1 = min(max(__ldg(a.offsets + e + 1), 0), a.pairs);
    begin = o0;
    count = o1 > o0 ? o1 - o0 : 0;
}

struct Tile {
    int e, f0, c0;                        // expert, first feature, first column (dW)
    int p0, p1;                           // positions: of the tile (forward, dx), of the expert (dW)
    int ncols;                            // MMA columns (a multiple of Shape::STEP)
    int steps;                            // stages of depth
};

template <int MODE, int COLS, bool PAIR>
struct Shape {
    static constexpr int FEATS = PAIR ? 2 * kFeat : kFeat;    // features per tile
    static constexpr int STEP = PAIR ? 32 : 16;               // granularity of the MMA's N

    static __host__ __device__ __forceinline__ int feature_tiles(const TcArgs& a) { return (a.feats + FEATS - 1) / FEATS; }
    // Rows per tile of an expert with `count` rows: equal tiles of whole STEPs, at most a.most
    static __device__ __forceinline__ int rows(const TcArgs& a, int count) {
        const int tiles = (count + a.most - 1) / a.most;
        return tiles == 0 ? COLS : ((count + tiles - 1) / tiles + STEP - 1) / STEP * STEP;
    }
    // Tiles of expert e per feature tile
    static __device__ __forceinline__ int tiles(const TcArgs& a, int e) {
        int begin, count;
        segment(a, e, begin, count);
        const int size = rows(a, count);
        return (count + size - 1) / size;
    }
    // Tile t; `e` walks up with t, first[e] = tiles of the experts before e (dW: the e-th expert by size).  An expert's tiles go in blocks of kBlock
    // position tiles (dW: column tiles) by all feature tiles, positions fastest, so the tiles that run at the same time
    // read about as many rows of the one operand as of the other, and the L2 serves them.
    static __device__ __forceinline__ Tile at(const TcArgs& a, const int* first, int64_t t, int& e) {
        Tile r;
        const int ft = feature_tiles(a), j = (int)(t / ft);
        int before, here;                                 // position tiles of the experts before, and of this one
        if constexpr (MODE == kExpertDw) {
            here = (a.cols + COLS - 1) / COLS;
            before = j / here * here;
            r.e = first[j / here];
        } else {
            while (j >= first[e + 1]) e++;
            before = first[e];
            here = first[e + 1] - before;
            r.e = e;
        }
        const int in = (int)(t - (int64_t)before * ft), block = in / (kBlock * ft);
        const int left = here - block * kBlock, wide = left < kBlock ? left : kBlock;
        const int k = in - block * kBlock * ft, tile = block * kBlock + k % wide;
        r.f0 = k / wide * FEATS;
        int begin, count;
        segment(a, r.e, begin, count);
        if constexpr (MODE == kExpertDw) {
            r.c0 = tile * COLS;
            r.p0 = begin;
            r.p1 = begin + count;
            r.ncols = min((a.cols - r.c0 + STEP - 1) / STEP * STEP, COLS);
            r.steps = (count + kDepth - 1) / kDepth;
        } else {
            const int size = rows(a, count);
            r.c0 = 0;
            r.p0 = begin + tile * size;
            r.p1 = min(r.p0 + size, begin + count);
            r.ncols = (r.p1 - r.p0 + STEP - 1) / STEP * STEP;
            r.steps = (a.depth + kDepth - 1) / kDepth;
        }
        return r;
    }
};

// Row of x that position p reads, for TMA: x_rows (past the tensor: zeros) where there is none
__device__ __forceinline__ int gather_row(const TcArgs& a, int p, int p1) {
    if (p >= p1) return (int)a.x_rows;
    const int r = a.rows ? __ldg(a.rows + p) : p;
    return r < 0 || r >= a.x_rows ? (int)a.x_rows : r;
}

template <bool PAIR>
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* m, int x, int y, uint32_t bar) {
    if constexpr (PAIR) tma_load_2d_pair(dst, m, x, y, bar);
    else tma_load_2d(dst, m, x, y, bar);
}
template <bool PAIR>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* m, int x, int y, int z, uint32_t bar) {
    if constexpr (PAIR) tma_load_3d_pair(dst, m, x, y, z, bar);
    else tma_load_3d(dst, m, x, y, z, bar);
}
template <bool PAIR>
__device__ __forceinline__ void gather4(uint32_t dst, const CUtensorMap* m, int x, const int (&r)[4], uint32_t bar) {
    if constexpr (PAIR) tma_gather4_pair(dst, m, x, r, bar);
    else tma_gather4(dst, m, x, r, bar);
}

// Stores a warp's 32 features (lanes) x 32 columns of the accumulator.  A lane's values are 2 bytes of 32 different
// rows of out (positions) or 64 bytes of one (dW): written as they are, a tile of 256 columns took 19650 cycles, more
// than its MMAs up to a depth of 2500.  So they go through shared memory and leave as 16-byte pieces of 64-byte runs.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    Pack<T, 2> p;
    p.v[0] = Elem<T>::from(lo);
    p.v[1] = Elem<T>::from(hi);
    return *reinterpret_cast<const uint32_t*>(&p);
}

// Column j is row j of dst (ldo apart), the lanes its 32 consecutive features; rows below `left`, features below
// `feats` exist.
template <typename T>
__device__ __forceinline__ void store_positions(T* dst, int64_t ldo, int left, int feats, bool vec, const float (&v)[32],
                                                unsigned char* stash) {
    const int lane = threadIdx.x & 31;
    if (vec) {
        // word [j / 2][lane] = columns j and j + 1 of the lane's feature; a lane then takes the words of 8 features
        // and separates them into 16 bytes of row j and 16 of row j + 1
        uint32_t* w = reinterpret_cast<uint32_t*>(stash);
#pragma unroll
        for (int j = 0; j < 16; j++) w[j * 36 + lane] = pack2<T>(v[2 * j], v[2 * j + 1]);
        __syncwarp();
        const int g = (lane & 3) * 8;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int j = (lane >> 2) + 8 * i;
            const uint4 a = *reinterpret_cast<const uint4*>(w + j * 36 + g), b = *reinterpret_cast<const uint4*>(w + j * 36 + g + 4);
            const uint4 lo = make_uint4(__byte_perm(a.x, a.y, 0x5410), __byte_perm(a.z, a.w, 0x5410),
                                        __byte_perm(b.x, b.y, 0x5410), __byte_perm(b.z, b.w, 0x5410));
            const uint4 hi = make_uint4(__byte_perm(a.x, a.y, 0x7632), __byte_perm(a.z, a.w, 0x7632),
                                        __byte_perm(b.x, b.y, 0x7632), __byte_perm(b.z, b.w, 0x7632));
            if (g < feats) {                               // feats is a multiple of 8 here
                T* to = dst + (int64_t)(2 * j) * ldo + g;
                if (2 * j < left) *reinterpret_cast<uint4*>(to) = lo;
                if (2 * j + 1 < left) *reinterpret_cast<uint4*>(to + ldo) = hi;
            }
        }
        __syncwarp();
    } else if (lane < feats) {
#pragma unroll
        for (int j = 0; j < 32; j++)
            if (j < left) dst[(int64_t)j * ldo + lane] = Elem<T>::from(v[j]);
    }
}

// The same in float32, 16 columns at a time: 128-byte runs.
__device__ __forceinline__ void store_positions_f32(float* dst, int64_t ldo, int left, int feats, bool vec,
                                                    const float (&v)[32], unsigned char* stash) {
    const int lane = threadIdx.x & 31;
    if (vec) {
        float* w = reinterpret_cast<float*>(stash);
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int j = 0; j < 16; j++) w[j * 36 + lane] = v[16 * h + j];
            __syncwarp();
            const int g = (lane & 7) * 4;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int j = (lane >> 3) + 4 * i;
                if (g < feats && 16 * h + j < left)        // feats is a multiple of 4 here
                    *reinterpret_cast<float4*>(dst + (int64_t)(16 * h + j) * ldo + g) = *reinterpret_cast<const float4*>(w + j * 36 + g);
            }
            __syncwarp();
        }
    } else if (lane < feats) {
#pragma unroll
        for (int j = 0; j < 32; j++)
            if (j < left) dst[(int64_t)j * ldo + lane] = v[j];
    }
}

// The lanes are 32 rows of dst (ldo apart), the columns its consecutive elements; `left` columns and `feats` rows exist.
template <typename T>
__device__ __forceinline__ void store_features(T* dst, int64_t ldo, int left, int feats, bool vec, const float (&v)[32],
                                               unsigned char* stash) {
    const int lane = threadIdx.x & 31;
    if (vec) {
#pragma unroll
        for (int g = 0; g < 4; g++)
            *reinterpret_cast<uint4*>(stash + lane * 80 + g * 16) =
                make_uint4(pack2<T>(v[8 * g], v[8 * g + 1]), pack2<T>(v[8 * g + 2], v[8 * g + 3]),
                           pack2<T>(v[8 * g + 4], v[8 * g + 5]), pack2<T>(v[8 * g + 6], v[8 * g + 7]));
        __syncwarp();
        const int g = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = (lane >> 2) + 8 * i;
            if (r < feats && g * 8 < left)                 // left is a multiple of 8 here
                *reinterpret_cast<uint4*>(dst + r * ldo + g * 8) = *reinterpret_cast<const uint4*>(stash + r * 80 + g * 16);
        }
        __syncwarp();
    } else {                                               // rows of any alignment: a row's 32 elements at a time
        T* mine = reinterpret_cast<T*>(stash + lane * 66);
#pragma unroll
        for (int j = 0; j < 32; j++) mine[j] = Elem<T>::from(v[j]);
        __syncwarp();
        if (lane < left) {
#pragma unroll 8
            for (int r = 0; r < 32; r++)
                if (r < feats) dst[r * ldo + lane] = reinterpret_cast<const T*>(stash + r * 66)[lane];
        }
        __syncwarp();
    }
}

template <typename T, int MODE, int COLS, bool GATHER, bool PAIR>
__global__ void __launch_bounds__(kTcThreads, 1)
    k_expert_tc(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb,
                const __grid_constant__ Tails tails, TcArgs a) {
    static_assert(!GATHER || (MODE == kExpertForward && !PAIR && COLS <= 128), "gathers: one per lane and stage");
    using S = TcSmem<COLS, PAIR>;
    using Sh = Shape<MODE, COLS, PAIR>;
    constexpr int NS = S::NS;
    constexpr int CTAS = PAIR ? 2 : 1;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char* gbars = smem_raw + (base - raw) + NS * S::STAGE;
    const uint32_t bars = base + NS * S::STAGE;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (NS + s); };
    auto accf = [&](int b) { return bars + 8u * (2 * NS + b); };
    auto acce = [&](int b) { return bars + 8u * (2 * NS + 2 + b); };
    const uint32_t drain = bars + 8u * (2 * NS + 4);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbars + 8 * (2 * NS + 5));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gbars + 8 * (2 * NS + 5) + 4);
    unsigned char* stash = gbars + S::BAR;
    int* first = reinterpret_cast<int*>(gbars + S::BAR + S::EPI);
    __shared__ int part[kTcThreads / 32];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = PAIR ? (int)cluster_rank() : 0;       // 0: the pair's leader
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; s++) {
            mbar_init(full(s), 1);                         // the leader's load warp; both CTAs' bytes count on it
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(accf(b), 1);
            mbar_init(acce(b), CTAS * kEpiThreads / 32);   // a lane of each epilogue warp, of both CTAs
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                         "r"(2 * COLS));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                         "r"(2 * COLS));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    }
    pdl_wait();
    int64_t tiles;
    if constexpr (MODE == kExpertDw) {
        // first[i]: the i-th expert by number of rows, most first.  A tile's depth is its expert's rows, and the tiles
        // go to the CTAs in turn: in that order each CTA gets about the same depth in all (in the order of the experts,
        // 10976 rows of 32 experts, 576 x 1904: 63 us).  Beyond kSorted experts, in their own order.
        constexpr int kSorted = 2 * kTcThreads;
        int count[2] = {}, rank[2] = {}, begin;
        for (int i = 0; i < 2; i++) {
            const int x = threadIdx.x + i * kTcThreads;
            if (x < a.experts && a.experts <= kSorted) {
                segment(a, x, begin, count[i]);
                first[x] = count[i];
            }
        }
        __syncthreads();
        if (a.experts <= kSorted)
            for (int y = 0; y < a.experts; y++) {
                const int c = first[y];
                for (int i = 0; i < 2; i++) {
                    const int x = threadIdx.x + i * kTcThreads;
                    rank[i] += c > count[i] || (c == count[i] && y < x) ? 1 : 0;
                }
            }
        __syncthreads();
        for (int x = threadIdx.x, i = 0; x < a.experts; x += kTcThreads, i++) first[a.experts <= kSorted ? rank[i & 1] : x] = x;
        tiles = (int64_t)a.experts * ((a.cols + COLS - 1) / COLS) * Sh::feature_tiles(a);
    } else {
        // first[e]: tiles of the experts before e, by a scan over per-thread runs of experts
        const int run = (a.experts + kTcThreads - 1) / kTcThreads, e0 = min((int)threadIdx.x * run, a.experts);
        const int e1 = min(e0 + run, a.experts);
        int sum = 0;
        for (int e = e0; e < e1; e++) sum += Sh::tiles(a, e);
        int s = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(kFull, s, o);
            if (lane >= o) s += up;
        }
        if (lane == 31) part[warp] = s;
        __syncthreads();
        int at = s - sum;
        for (int w = 0; w < warp; w++) at += part[w];
        for (int e = e0; e < e1; e++) {
            first[e] = at;
            at += Sh::tiles(a, e);
        }
        if (threadIdx.x == kTcThreads - 1) first[a.experts] = at;
    }
    tc_fence_before();
    if constexpr (PAIR) cluster_sync();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    if constexpr (MODE != kExpertDw) tiles = (int64_t)first[a.experts] * Sh::feature_tiles(a);
    const int64_t t0 = blockIdx.x / CTAS, dt = gridDim.x / CTAS;
    int e = 0;

    if (warp == 0) {
        // ---- loads: the whole warp, its lanes sharing the copies of a stage
        int stage = 0;
        uint32_t phase = 0;
        int64_t issued = 0;
        bool ok = true;
        Tile next;
        if (t0 < tiles) next = Sh::at(a, first, t0, e);
        for (int64_t t = t0; t < tiles && ok; t += dt) {
            const Tile w = next;
            if (w.steps == 0) {
                if (t + dt < tiles) next = Sh::at(a, first, t + dt, e);
                continue;
            }
            const int f0 = w.f0 + rank * kFeat;
            const int half = w.ncols / CTAS;               // columns of this CTA's operand
            int r[4];                                      // rows of this lane's gather
            if constexpr (GATHER) {
#pragma unroll
                for (int i = 0; i < 4; i++) r[i] = gather_row(a, w.p0 + lane * 4 + i, w.p1);
            }
            for (int kc = 0; kc < w.steps && ok; kc++) {
                ok = __all_sync(kFull, mbar_wait(empty(stage), phase ^ 1u, abort_flag));
                if (!ok) break;
                const uint32_t sa = base + stage * S::STAGE, sb = sa + S::A;
                const uint32_t bar = PAIR ? cluster_addr(full(stage), 0) : full(stage);
                if constexpr (MODE == kExpertDw) {
                    // A: dy, two boxes of 64 features x 64 positions; B: x, boxes of 64 columns.  The last stage of a
                    // group takes its positions 16 at a time, and the ones past its last whole 16 by gathers of four,
                    // which give zeros past its end (a gather of four takes about as long as a box: the whole stage by
                    // gathers took as long as three others)
                    const int k0 = w.p0 + kc * kDepth, v = min(w.p1 - k0, kDepth), nb = (half + 63) / 64;
                    const int c0 = w.c0 + rank * half;
                    if (lane == 0 && rank == 0)
                        mbar_expect_tx(full(stage), (uint32_t)(CTAS * (2 + nb)) * (uint32_t)((v + 15) / 16 * 16 * 128));
                    __syncwarp();
                    if (v == kDepth) {
                        if (lane < 2) load_2d<PAIR>(sa + lane * kBox, &ma, f0 + lane * 64, k0, bar);
                        else if (lane < 2 + nb) load_2d<PAIR>(sb + (lane - 2) * kBox, &mb, c0 + (lane - 2) * 64, k0, bar);
                    } else {
                        const int i = lane & 7, part = v / 16 * 16 + (i & 3) * 4;
                        for (int h = lane >> 3; h < 2 + nb; h += 4) {
                            const uint32_t to = h < 2 ? sa + h * kBox : sb + (h - 2) * kBox;
                            const int col = h < 2 ? f0 + h * 64 : c0 + (h - 2) * 64;
                            if (i < v / 16) {
                                load_2d<PAIR>(to + i * 2048, h < 2 ? &tails.a16 : &tails.b16, col, k0 + i * 16, bar);
                            } else if (i >= 4 && v % 16 != 0) {
                                int q[4];                  // (x is in grouped order too)
#pragma unroll
                                for (int n = 0; n < 4; n++) q[n] = k0 + part + n < w.p1 ? k0 + part + n : a.pairs;
                                gather4<PAIR>(to + part * 128, h < 2 ? &tails.a_row : &tails.b_row, col, q, bar);
                            }
                        }
                    }
                } else {
                    const int nb = GATHER ? half / 4 : (half + 31) / 32;
                    if (lane == 0) {
                        if (rank == 0) mbar_expect_tx(full(stage), (uint32_t)(CTAS * (S::A + nb * (GATHER ? 512 : 4096))));
                        if constexpr (MODE == kExpertForward) {        // 128 features x 64 deep
                            load_3d<PAIR>(sa, &ma, kc * kDepth, f0, w.e, bar);
                        } else {                                       // two boxes of 64 deep x 64 features
                            load_3d<PAIR>(sa, &ma, f0, kc * kDepth, w.e, bar);
                            load_3d<PAIR>(sa + kBox, &ma, f0 + 64, kc * kDepth, w.e, bar);
                        }
                    }
                    __syncwarp();
                    if (lane < nb) {
                        if constexpr (GATHER) gather4<PAIR>(sb + lane * 512, &tails.b_row, kc * kDepth, r, bar);
                        else load_2d<PAIR>(sb + lane * 4096, &mb, kc * kDepth, w.p0 + rank * half + lane * 32, bar);
                    }
                }
                issued++;
                if (kc == 0 && t + dt < tiles) next = Sh::at(a, first, t + dt, e);
                if (++stage == NS) { stage = 0; phase ^= 1u; }
            }
        }
        // the loads in flight have landed (a timeout) and both CTAs are done with every stage (a pair: the leader's
        // MMAs read this CTA's stages and its commits arrive here) before the CTA ends
        for (int i = 0; i < NS && i < issued; i++) {
            if (--stage < 0) { stage = NS - 1; phase ^= 1u; }
            const uint32_t bar = ok ? empty(stage) : full(stage);
            if (PAIR ? (ok || rank == 0) : !ok)
                for (uint32_t n = 0; n < kSpinLimit && !mbar_try(bar, phase); n++) {}
        }
    } else if (warp == 1) {
        // ---- MMA issuer
        if (lane == 0 && rank == 0) {
            constexpr uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
            constexpr uint32_t amn = MODE != kExpertForward, bmn = MODE == kExpertDw;
            constexpr uint32_t idesc0 = (1u << 4) | (type << 7) | (type << 10) | (amn << 15) | (bmn << 16) |
                                        ((uint32_t)(Sh::FEATS >> 4) << 24);
            int stage = 0;
            uint32_t phase = 0, abuf = 0, aphase = 0;
            bool ok = true;
            // the next tile is worked out while this one's MMAs run: about 1000 cycles (two loads, three divisions)
            // that would otherwise pass between the last MMA of a tile and the first of the next
            Tile next;
            if (t0 < tiles) next = Sh::at(a, first, t0, e);
            for (int64_t t = t0; t < tiles && ok; t += dt) {
                const Tile w = next;
                if (w.steps == 0) {                        // dW of an expert with no rows: nothing to add up
                    if (t + dt < tiles) next = Sh::at(a, first, t + dt, e);
                    continue;
                }
                ok = mbar_wait(acce(abuf), aphase ^ 1u, abort_flag);
                if (!ok) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem + abuf * COLS;
                const uint32_t idesc = idesc0 | ((uint32_t)(w.ncols >> 3) << 17);
                const int deep = MODE == kExpertDw ? w.p1 - w.p0 : a.depth;
                for (int kc = 0; kc < w.steps && ok; kc++) {
                    ok = mbar_wait(full(stage), phase, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t sa = base + stage * S::STAGE, sb = sa + S::A;
                    const uint64_t da = amn ? sw128_desc_mn(sa, kBox) : sw128_desc(sa);
                    const uint64_t db = bmn ? sw128_desc_mn(sb, kBox) : sw128_desc(sb);
#pragma unroll
                    for (int kk = 0; kk < kDepth / 16; kk++) {     // 16 deep: 32 B of a K-major row, 16 MN-major rows
                        const uint64_t oa = (amn ? kk * 2048 : kk * 32) >> 4, ob = (bmn ? kk * 2048 : kk * 32) >> 4;
                        if (kc * kDepth + kk * 16 < deep) {
                            if constexpr (PAIR) mma_f16_pair(d_tmem, da + oa, db + ob, idesc, (kc | kk) != 0);
                            else mma_f16(d_tmem, da + oa, db + ob, idesc, (kc | kk) != 0);
                        }
                    }
                    if constexpr (PAIR) mma_commit_pair(empty(stage));
                    else mma_commit(empty(stage));
                    if (kc == 0 && t + dt < tiles) next = Sh::at(a, first, t + dt, e);
                    if (++stage == NS) { stage = 0; phase ^= 1u; }
                }
                if (!ok) break;
                if constexpr (PAIR) mma_commit_pair(accf(abuf));
                else mma_commit(accf(abuf));
                abuf ^= 1u;
                if (abuf == 0) aphase ^= 1u;
            }
            if (!ok) {                                     // a timeout: the MMAs issued so far end before TMEM is freed
                if constexpr (PAIR) mma_commit_pair(drain);
                else mma_commit(drain);
                for (uint32_t n = 0; n < kSpinLimit && !mbar_try(drain, 0); n++) {}
            }
        }
    } else {
        // ---- epilogue: warp w reads TMEM lane quarter w % 4 (features), 32 columns at a time
        const int q = warp & 3;
        const uint32_t lane_base = tmem + ((uint32_t)(32 * q) << 16);
        T* out = static_cast<T*>(a.out);
        float* out32 = static_cast<float*>(a.out);
        const bool f32 = MODE == kExpertDx && a.out_f32;
        unsigned char* mine = stash + q * kEpiBytes;
        uint32_t abuf = 0, aphase = 0;
        bool ok = true;
        if constexpr (MODE != kExpertDw) {                 // rows past the last group: zeros
            const int64_t taken = min(max(__ldg(a.offsets + a.experts), 0), a.pairs);
            for (int64_t i = taken * a.ldo + (int64_t)blockIdx.x * kEpiThreads + threadIdx.x - 64;
                 i < a.pairs * a.ldo; i += (int64_t)gridDim.x * kEpiThreads) {
                if (f32) out32[i] = 0.0f;
                else out[i] = Elem<T>::from(0.0f);
            }
        }
        for (int64_t t = t0; t < tiles && ok; t += dt) {
            const Tile w = Sh::at(a, first, t, e);
            if (w.steps > 0) {
                ok = mbar_wait(accf(abuf), aphase, abort_flag);
                if (!ok) break;
                tc_fence_after();
            }
            const int f = w.f0 + rank * kFeat + 32 * q;    // the warp's first feature
            for (int c = 0; c < w.ncols && f < a.feats; c += 32) {
                float v[32];
                if (w.steps > 0) {
                    tmem_ld32(lane_base + abuf * COLS + c, v);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j++) v[j] = 0.0f;
                }
                if constexpr (MODE == kExpertDw)
                    store_features<T>(out + ((int64_t)w.e * a.feats + f) * a.ldo + w.c0 + c, a.ldo, a.cols - w.c0 - c,
                                      a.feats - f, a.out_vec, v, mine);
                else if (f32)
                    store_positions_f32(out32 + (int64_t)(w.p0 + c) * a.ldo + f, a.ldo, w.p1 - w.p0 - c, a.feats - f, a.out_vec,
                                        v, mine);
                else
                    store_positions<T>(out + (int64_t)(w.p0 + c) * a.ldo + f, a.ldo, w.p1 - w.p0 - c, a.feats - f, a.out_vec,
                                       v, mine);
            }
            if (w.steps > 0) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (PAIR) mbar_arrive_cluster(cluster_addr(acce(abuf), 0));
                    else mbar_arrive(acce(abuf));
                }
                abuf ^= 1u;
                if (abuf == 0) aphase ^= 1u;
            }
        }
    }

    __syncwarp();
    tc_fence_before();
    if constexpr (PAIR) cluster_sync();
    else __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * COLS));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * COLS));
    }
    if (threadIdx.x == 0 && *abort_flag) *static_cast<volatile int*>(a.error) = 1;
}

// ---------------------------------------------------------------- host side

// rows x cols (x planes) of 16-bit elements, rows ld apart; box of 64 columns x box_rows, 128-byte swizzle, zeros
// outside
bool make_map(CUtensorMap* m, int dtype, const void* base, int64_t cols, int64_t rows, int64_t planes, int64_t ld, int box_rows) {
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)(planes > 0 ? planes : 1)};
    cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)ld * rows * 2};
    cuuint32_t box[3] = {(cuuint32_t)kDepth, (cuuint32_t)box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return encode_tensor_map(m, dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                             planes > 0 ? 3 : 2, const_cast<void*>(base), dims, strides, box, estr,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

template <typename T, int MODE, int COLS, bool GATHER, bool PAIR>
cudaError_t run_tc(const CUtensorMap (&m)[2], const Tails& tails, TcArgs a, cudaStream_t st) {
    auto kern = k_expert_tc<T, MODE, COLS, GATHER, PAIR>;
    using S = TcSmem<COLS, PAIR>;
    static unsigned long long configured = 0;
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(configured >> (dev & 63) & 1ull)) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::base + S::EXPERTS);
        if (e != cudaSuccess) return e;
        configured |= 1ull << (dev & 63);
    }
    const size_t smem = S::base + (size_t)(a.experts + 1) * 4;
    const int grid = PAIR ? num_sms() / 2 * 2 : num_sms();
    // Fewer positions a tile where the results' rows are not on 16-byte boundaries, whose element-wise stores are most of
    // a small call's time, and full tiles would leave CTAs without any: as many as give each CTA (or pair) one tile, 32
    // at least (1554 rows of 12 experts, 515 x 333: 52.8 -> 47.5 us for y, dx and dW).  Not otherwise: every further
    // tile reads its features' matrix again (597 rows of 8 experts, 1072 x 1800: 67.3 -> 75.6 us).
    using Sh = Shape<MODE, COLS, PAIR>;
    const int64_t share = (int64_t)a.pairs * Sh::feature_tiles(a) / (grid / (PAIR ? 2 : 1));
    a.most = a.out_vec || share >= COLS ? COLS : share <= 32 ? 32 : (int)(share + 31) / 32 * 32;
    if constexpr (PAIR) return launch_pdl_clusters(kern, dim3(grid), dim3(kTcThreads), smem, st, 2, m[0], m[1], tails, a);
    return launch_pdl(kern, dim3(grid), dim3(kTcThreads), smem, st, m[0], m[1], tails, a);
}

// A pair's tiles of 256 features, or one CTA's of 128 where there are no more, or (forward, dx: 576 features 46 -> 36 us)
// where those cover a tenth less that does not exist; a pair does the same work about a tenth faster.
template <typename T, int MODE, int COLS, bool GATHER>
cudaError_t run_shape(const CUtensorMap (&m)[2], const Tails& tails, const TcArgs& a, cudaStream_t st) {
    if constexpr (COLS == 256) {
        const int whole = (a.feats + 255) / 256 * 256, half = (a.feats + 127) / 128 * 128;
        if (MODE == kExpertDw ? a.feats > kFeat : whole * 10 <= half * 11) return run_tc<T, MODE, COLS, GATHER, true>(m, tails, a, st);
    }
    return run_tc<T, MODE, COLS, GATHER, false>(m, tails, a, st);
}

template <typename T>
cudaError_t run_kind(const ExpertCall& c, const Operands& o, cudaStream_t st) {
    CUtensorMap m[2];
    Tails tails = {};
    TcArgs a = {};
    a.offsets = c.offsets;
    a.rows = o.rows;
    a.x_rows = o.x_rows;
    a.pairs = (int)c.pairs;
    a.experts = c.experts;
    a.error = c.error;
    const bool few = expert_few_rows(c);
    auto whole = [](const void* p, int cols) { return cols % 8 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    bool ok;
    switch (c.kind) {
        case kExpertForward:
            a.feats = c.n;
            a.depth = c.d;
            a.out = c.y;
            a.out_vec = whole(c.y, c.n);
            a.ldo = c.n;
            ok = make_map(&m[0], c.dtype, o.w, c.d, c.n, c.experts, o.ldw, kFeat) &&
                 make_map(&m[1], c.dtype, o.x, c.d, o.x_rows, 0, o.ldx, 32) &&
                 make_map(&tails.b_row, c.dtype, o.x, c.d, o.x_rows, 0, o.ldx, 1);
            if (!ok) return cudaErrorInvalidValue;
            if (few) return o.rows ? run_shape<T, kExpertForward, 64, true>(m, tails, a, st) : run_shape<T, kExpertForward, 64, false>(m, tails, a, st);
            return run_shape<T, kExpertForward, 256, false>(m, tails, a, st);
        case kExpertDx:
            a.rows = nullptr;
            a.x_rows = c.pairs;
            a.feats = c.d;
            a.depth = c.n;
            a.out = c.dx;
            a.out_f32 = c.dx_f32;
            a.out_vec = c.dx_f32 ? c.d % 4 == 0 && reinterpret_cast<uintptr_t>(c.dx) % 16 == 0 : whole(c.dx, c.d);
            a.ldo = c.d;
            ok = make_map(&m[0], c.dtype, o.w, c.d, c.n, c.experts, o.ldw, kDepth) &&
                 make_map(&m[1], c.dtype, o.dy, c.n, c.pairs, 0, o.lddy, 32);
            if (!ok) return cudaErrorInvalidValue;
            return few ? run_shape<T, kExpertDx, 64, false>(m, tails, a, st) : run_shape<T, kExpertDx, 256, false>(m, tails, a, st);
        default:
            a.feats = c.n;
            a.cols = c.d;
            a.out = c.dw;
            a.out_vec = whole(c.dw, c.d);
            a.ldo = c.d;
            ok = make_map(&m[0], c.dtype, o.dy, c.n, c.pairs, 0, o.lddy, kDepth) &&
                 make_map(&tails.a16, c.dtype, o.dy, c.n, c.pairs, 0, o.lddy, 16) &&
                 make_map(&tails.a_row, c.dtype, o.dy, c.n, c.pairs, 0, o.lddy, 1) &&
                 make_map(&m[1], c.dtype, o.x, c.d, o.x_rows, 0, o.ldx, kDepth) &&
                 make_map(&tails.b16, c.dtype, o.x, c.d, o.x_rows, 0, o.ldx, 16) &&
                 make_map(&tails.b_row, c.dtype, o.x, c.d, o.x_rows, 0, o.ldx, 1);
            if (!ok) return cudaErrorInvalidValue;
            return run_shape<T, kExpertDw, 256, false>(m, tails, a, st);
    }
}

}  // namespace

cudaError_t launch_expert_tc(const ExpertCall& c, const Operands& o, cudaStream_t st) {
    return c.dtype == 1 ? run_kind<__nv_bfloat16>(c, o, st) : run_kind<__half>(c, o, st);
}

}  // namespace kmc
