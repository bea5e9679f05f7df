// group.cu -- the grouping plan of routed rows (kmc_group_rows): a stable counting sort of the (row, choice) pairs by
// expert.
//
// Pair p = t k + j carries expert ids[p]; ids outside [0, E) are left out.  offsets[e] = pairs of experts below e;
// the pairs of expert e, in increasing p, take the positions offsets[e] ..  offsets[e + 1] - 1: slot[p] = position
// (-1: left out) and rows[position] = p / k, the row the position reads (-1 past offsets[E]).
//
// The pairs are cut into chunks of consecutive pairs, one per CTA, and a chunk into one run of consecutive pairs per
// warp, so a position is
//   offsets[e] + pairs of e in earlier chunks + in earlier warps' runs + earlier in the warp's own run,
// counted, never taken from an atomic's order: the plan is the same on every run.  Up to kOneChunk pairs one CTA does
// it all in one launch (which at that size costs more than the work); above, a first kernel counts each chunk's pairs
// per expert and every CTA of the second adds up the chunks before its own.  Latency bounds both: 192 pairs 3.9 us,
// 2^20 pairs of 256 experts 15.9 us (their 12 MB would take 1.9).
#include "common.cuh"
#include "kmc_internal.h"

namespace kmc {

namespace {

constexpr int kGroupThreads = 1024;
constexpr int kGroupWarps = kGroupThreads / 32;
constexpr int64_t kOneChunk = 8192;       // pairs one CTA takes by itself
constexpr int64_t kChunkMin = 4096;       // pairs per chunk otherwise, more where that makes over kMaxChunks of them
constexpr int kMaxChunks = 148;           // one per SM
constexpr int kChunkLoads = (kMaxChunks + 31) / 32;
constexpr int kAhead = 8;                 // ids a thread has in flight
constexpr int kCounters = 32768;          // per-warp counters in shared memory (128 KB): fewer warps work above 1024 experts

struct GroupArgs {
    const int32_t* ids;
    int64_t pairs, chunk;
    int experts, choices, chunks;
    int32_t* counts;                      // experts x chunks (first kernel), when chunks > 1
    int32_t* offsets;
    int32_t* rows;
    int32_t* slot;
};

__global__ void __launch_bounds__(kGroupThreads) k_group_count(GroupArgs a) {
    extern __shared__ int32_t count[];
    pdl_wait();
    for (int e = threadIdx.x; e < a.experts; e += kGroupThreads) count[e] = 0;
    __syncthreads();
    const int64_t p0 = (int64_t)blockIdx.x * a.chunk, p1 = min(p0 + a.chunk, a.pairs);
    for (int64_t b = p0; b < p1; b += kAhead * kGroupThreads) {
        int e[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int64_t p = b + j * kGroupThreads + threadIdx.x;
            e[j] = p < p1 ? __ldg(a.ids + p) : -1;
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++)
            if (e[j] >= 0 && e[j] < a.experts) atomicAdd(count + e[j], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += kGroupThreads)
        a.counts[(int64_t)e * a.chunks + blockIdx.x] = count[e];
}

// Shared memory: before[experts] (first: pairs of e in earlier chunks; then the position of the chunk's first pair of
// e), total[experts] (pairs of e in all), and run[warps][experts] (counts, then next positions, of each warp's run).
__global__ void __launch_bounds__(kGroupThreads) k_group_place(GroupArgs a, int warps) {
    extern __shared__ int32_t sh[];
    int32_t* before = sh;
    int32_t* total = before + a.experts;
    int32_t* run = total + a.experts;
    __shared__ int32_t warp_total[kGroupWarps];
    __shared__ int32_t all;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = a.experts;
    for (int i = threadIdx.x; i < (2 + warps) * E; i += kGroupThreads) sh[i] = 0;
    pdl_wait();
    __syncthreads();

    const int64_t p0 = (int64_t)blockIdx.x * a.chunk, p1 = min(p0 + a.chunk, a.pairs);
    const int64_t per = ((p1 - p0 + warps - 1) / warps + 31) / 32 * 32;
    const int64_t w0 = min(p0 + warp * per, p1), w1 = warp < warps ? min(w0 + per, p1) : w0;
    int ids[kAhead];                      // 256 pairs of the run at a time
    auto load = [&](int64_t b) {
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int64_t p = b + j * 32 + lane;
            const int e = p < w1 ? __ldg(a.ids + p) : -1;
            ids[j] = e < 0 || e > E ? E : e;               // E: left out
        }
    };
    for (int64_t b = w0; b < w1; b += kAhead * 32) {
        load(b);
#pragma unroll
        for (int j = 0; j < kAhead; j++)
            if (ids[j] < E) atomicAdd(run + warp * E + ids[j], 1);
    }
    if (a.chunks > 1) {
        // a warp per expert, four at a time: the counts of all chunks lie side by side and are in flight together (a
        // thread per expert walking down the chunks waited for the L2 once a chunk, 10 us more at 2^20 pairs)
        for (int e0 = warp; e0 < E; e0 += 4 * kGroupWarps) {
            int32_t v[4][kChunkLoads];
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int i = 0; i < kChunkLoads; i++) {
                    const int e = e0 + q * kGroupWarps, c = i * 32 + lane;
                    v[q][i] = e < E && c < a.chunks ? __ldcg(a.counts + (int64_t)e * a.chunks + c) : 0;
                }
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int e = e0 + q * kGroupWarps;
                int32_t sum = 0, below = 0;
#pragma unroll
                for (int i = 0; i < kChunkLoads; i++) {
                    sum += v[q][i];
                    below += i * 32 + lane < (int)blockIdx.x ? v[q][i] : 0;
                }
                sum = __reduce_add_sync(0xffffffffu, sum);
                below = __reduce_add_sync(0xffffffffu, below);
                if (lane == 0 && e < E) {
                    total[e] = sum;
                    before[e] = below;
                }
            }
        }
        __syncthreads();
    } else {
        __syncthreads();
        for (int e = threadIdx.x; e < E; e += kGroupThreads) {
            int32_t sum = 0;
            for (int w = 0; w < warps; w++) sum += run[w * E + e];
            total[e] = sum;
        }
        __syncthreads();
    }

    // exclusive scan of the totals, kGroupThreads experts at a time
    int32_t base = 0;
    for (int e0 = 0; e0 < E; e0 += kGroupThreads) {
        const int e = e0 + threadIdx.x;
        const int32_t v = e < E ? total[e] : 0;
        int32_t s = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t up = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += up;
        }
        if (lane == 31) warp_total[warp] = s;
        __syncthreads();
        if (warp == 0) {
            int32_t t = warp_total[lane];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int32_t up = __shfl_up_sync(0xffffffffu, t, o);
                if (lane >= o) t += up;
            }
            warp_total[lane] = t;
        }
        __syncthreads();
        const int32_t start = base + (warp > 0 ? warp_total[warp - 1] : 0) + s - v;
        base += warp_total[kGroupWarps - 1];
        if (e < E) {
            if (blockIdx.x == 0) a.offsets[e] = start;
            int32_t next = start + before[e], n[kGroupWarps];
#pragma unroll
            for (int w = 0; w < kGroupWarps; w++) n[w] = w < warps ? run[w * E + e] : 0;
#pragma unroll
            for (int w = 0; w < kGroupWarps; w++)
                if (w < warps) {
                    run[w * E + e] = next;
                    next += n[w];
                }
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        all = base;
        if (blockIdx.x == 0) a.offsets[E] = base;
    }
    __syncthreads();

    const int bits = 32 - __clz(E);
    for (int64_t b0 = w0; b0 < w1; b0 += kAhead * 32) {
        if (w1 - w0 > kAhead * 32) load(b0);               // (a shorter run is still in the registers)
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int64_t b = b0 + j * 32, p = b + lane;
            if (b >= w1) break;
            const int e = ids[j];
            // the lanes of the same expert, one ballot per bit of the index (match.any took ten times the instructions)
            unsigned same = 0xffffffffu;
            for (int bit = 0; bit < bits; bit++) {
                const bool one = (e >> bit) & 1;
                const unsigned m = __ballot_sync(0xffffffffu, one);
                same &= one ? m : ~m;
            }
            const int ahead = __popc(same & ((1u << lane) - 1u));
            int32_t pos = -1;
            if (e < E) pos = run[warp * E + e] + ahead;
            __syncwarp();
            if (e < E && ahead == 0) run[warp * E + e] = pos + __popc(same);
            __syncwarp();
            if (p < w1) {
                a.slot[p] = pos;
                if (e < E) a.rows[pos] = (int32_t)((uint32_t)p / (uint32_t)a.choices);
            }
        }
    }
    for (int64_t p = p0 + threadIdx.x; p < p1; p += kGroupThreads)
        if (p >= all) a.rows[p] = -1;     // positions no pair took (each CTA its own chunk's range of them)
}

int64_t group_chunk(int64_t pairs) {
    if (pairs <= kOneChunk) return pairs > 0 ? pairs : 1;
    const int64_t least = (pairs + kMaxChunks - 1) / kMaxChunks;
    return least > kChunkMin ? least : kChunkMin;
}

}  // namespace

size_t group_bytes(int64_t pairs, int experts) {
    const int64_t chunk = group_chunk(pairs), chunks = (pairs + chunk - 1) / chunk;
    return chunks > 1 ? (size_t)chunks * experts * sizeof(int32_t) : 0;
}

cudaError_t launch_group(const int32_t* ids, int64_t pairs, int choices, int experts, int32_t* offsets, int32_t* rows,
                         int32_t* slot, void* ws, cudaStream_t st) {
    GroupArgs a;
    a.ids = ids;
    a.pairs = pairs;
    a.chunk = group_chunk(pairs);
    a.experts = experts;
    a.choices = choices;
    a.chunks = (int)((pairs + a.chunk - 1) / a.chunk);
    a.counts = static_cast<int32_t*>(ws);
    a.offsets = offsets;
    a.rows = rows;
    a.slot = slot;
    int warps = kCounters / experts < kGroupWarps ? kCounters / experts : kGroupWarps;
    const int64_t useful = (a.chunk + 31) / 32;
    if (warps > useful) warps = (int)useful;
    const size_t smem = (size_t)(2 + warps) * experts * sizeof(int32_t);
    static unsigned long long configured = 0;
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(configured >> (dev & 63) & 1ull)) {
        cudaError_t e = cudaFuncSetAttribute(k_group_place, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)((kCounters + 2 * kGroupMaxExperts) * sizeof(int32_t)));
        if (e != cudaSuccess) return e;
        configured |= 1ull << (dev & 63);
    }
    if (a.chunks > 1) {
        cudaError_t e = launch_pdl(k_group_count, dim3(a.chunks), dim3(kGroupThreads), experts * sizeof(int32_t), st, a);
        if (e != cudaSuccess) return e;
    }
    return launch_pdl(k_group_place, dim3(a.chunks > 0 ? a.chunks : 1), dim3(kGroupThreads), smem, st, a, warps);
}

}  // namespace kmc
