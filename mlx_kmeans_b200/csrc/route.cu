// route.cu -- routing of rows to their top-k experts (kmc_route) and the gradient of the weights (kmc_route_grad).
//
// The top-1 label of a Lloyd pass generalised to the k best of E scores with weights.  Row t, logits l_0 .. l_{E-1}:
//   key_i  = l_i (softmax) or sigma(l_i) = 1 / (1 + exp(-l_i)) (sigmoid), plus bias_i; float32, each operation
//            rounded on its own, so the choice is defined bit for bit.  Expert i is available when l_i > -inf and
//            key_i > -inf (a NaN is not) and the row's mask is set.
//   groups   with G > 1 groups of E / G consecutive experts, a group scores the sum of its two best available keys
//            (its best, when it has one); only the top_groups best groups stay (lowest index on ties).
//   ids      the k largest keys in decreasing order, lowest index on ties; -1 where no available expert is left.
//   weights  softmax over the available logits, or (RENORM) over the chosen ones; sigma(l_id), or (RENORM) divided by
//            the sum over the chosen (0 when that sum is 0); times `scale`.
// Gradient, with g = scale dL/dweights on the chosen (the choice itself, and so the bias, has none):
//   softmax  dl_i = p_i ([i chosen] g_i - sum_j g_j p_j) over the available, RENORM: over the chosen, 0 elsewhere
//   sigmoid  dl_i = g_i s_i (1 - s_i), RENORM: (g_i - sum_j g_j s_j / S) s_i (1 - s_i) / S, S = sum of the chosen s_j
//
// LANES lanes of a warp own a row: lane L holds the PER consecutive experts from L PER on (E up to LANES PER), read
// with 16-byte loads where the row allows, their keys as order-preserving 32-bit integers (0: not available).
// E reads and 8 k bytes written per row are little; the choices' instructions bound it (see choose; ALU pipe 79%): 65536
// rows of 128 bfloat16 logits, 8 choices, renormalised 17.9 us and 9.0 us for the gradient, over all experts 21.7 and
// 11.9, where the bytes take 3 each; one row 2.5 us.
#include "common.cuh"
#include "experts.cuh"
#include "kmc_internal.h"

namespace kmc {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kRouteWarps = 8;

// float order as unsigned order (-0 first made +0; no NaN comes here); every finite or infinite value maps above 0
__device__ __forceinline__ unsigned ordered(float f) {
    const unsigned u = __float_as_uint(__fadd_rn(f, 0.0f));
    return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(unsigned u) {
    return __uint_as_float((u & 0x80000000u) ? (u ^ 0x80000000u) : ~u);
}
__device__ __forceinline__ float sigmoid32(float l) { return __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-l))); }

// exp of l - m <= 0 and the quotient of such by their sum (1 at least): the softmax's.  16-bit logits, of which each is
// off by 2^-9 or 2^-12 of itself, take the hardware's exponential of base 2 and its quotient (off by |x| 2^-23 + 2^-21 at
// most, relatively; below 2^-126 it is 0); float32 logits take expf and an IEEE division, and so does the sigmoid, whose
// value decides a choice bit for bit.
template <typename T>
__device__ __forceinline__ float exp_below(float x) {
    if constexpr (sizeof(T) == 2) return __expf(x);
    return expf(x);
}
template <typename T>
__device__ __forceinline__ float share(float p, float total) {
    if constexpr (sizeof(T) == 2) return __fdividef(p, total);
    return __fdiv_rn(p, total);
}

// Over the LANES lanes that share a row (aligned in the warp); every lane of the warp calls them.
template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}
template <int LANES>
__device__ __forceinline__ float row_max(float v) {        // a NaN only if every lane's is
    if constexpr (LANES == 32) {
        float m;
        asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
        return m;
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
    return v;
}
template <int LANES>
__device__ __forceinline__ unsigned row_max(unsigned v) {
    if constexpr (LANES == 32) return __reduce_max_sync(kFull, v);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(kFull, v, o));
    return v;
}
template <int LANES>
__device__ __forceinline__ unsigned row_ballot(bool p) {   // bit i: lane i of the row
    const unsigned m = __ballot_sync(kFull, p);
    if constexpr (LANES == 32) return m;
    return (m >> (threadIdx.x & 31 & ~(LANES - 1))) & ((1u << (LANES & 31)) - 1u);
}

// PER elements per lane as vectors of V (16 bytes, or all PER where that is less), or of half of that
template <typename T, int PER>
struct Vec {
    static constexpr int V = PER * sizeof(T) >= 16 ? 16 / sizeof(T) : PER;
    static constexpr int H = V > 1 ? V / 2 : 1;
    static constexpr size_t BYTES = V * sizeof(T);
    // 2: whole vectors are aligned, 1: halves of one, 0: elements only
    static int level(const void* p, int64_t row_bytes) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(p) | (uintptr_t)row_bytes;
        return at % BYTES == 0 ? 2 : at % (H * sizeof(T)) == 0 ? 1 : 0;
    }
};

template <typename T, int PER, int V>
__device__ __forceinline__ void load_by(const T* row, int i0, int experts, float (&l)[PER]) {
#pragma unroll
    for (int i = 0; i < PER; i += V) {
        if (i0 + i + V <= experts) {
            const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(row + i0 + i);
#pragma unroll
            for (int j = 0; j < V; j++) l[i + j] = Elem<T>::to(p.v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) l[i + j] = i0 + i + j < experts ? Elem<T>::to(row[i0 + i + j]) : -INFINITY;
        }
    }
}
// The lane's PER logits of one row, -inf past the last expert
template <typename T, int PER>
__device__ __forceinline__ void load_row(const T* row, int lane, int experts, int level, float (&l)[PER]) {
    if (level == 2) load_by<T, PER, Vec<T, PER>::V>(row, lane * PER, experts, l);
    else if (level == 1) load_by<T, PER, Vec<T, PER>::H>(row, lane * PER, experts, l);
    else load_by<T, PER, 1>(row, lane * PER, experts, l);
}

template <typename T, int PER, int V>
__device__ __forceinline__ void store_by(T* row, int i0, int experts, const float (&l)[PER]) {
#pragma unroll
    for (int i = 0; i < PER; i += V) {
        if (i0 + i + V <= experts) {
            Pack<T, V> p;
#pragma unroll
            for (int j = 0; j < V; j++) p.v[j] = Elem<T>::from(l[i + j]);
            *reinterpret_cast<Pack<T, V>*>(row + i0 + i) = p;
        } else {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (i0 + i + j < experts) row[i0 + i + j] = Elem<T>::from(l[i + j]);
        }
    }
}
template <typename T, int PER>
__device__ __forceinline__ void store_row(T* row, int lane, int experts, int level, const float (&l)[PER]) {
    if (level == 2) store_by<T, PER, Vec<T, PER>::V>(row, lane * PER, experts, l);
    else if (level == 1) store_by<T, PER, Vec<T, PER>::H>(row, lane * PER, experts, l);
    else store_by<T, PER, 1>(row, lane * PER, experts, l);
}

struct RouteArgs {
    int64_t rows, stride;
    int experts, choices, groups, top_groups, group_size;
    const float* bias;
    const uint8_t* mask;
    float scale;
    int sigmoid, renorm;
    int vec, out_vec;                                      // Vec::level of logits and dlogits
};

// Clears the keys of experts outside the best top_groups groups.  A group that covers a power of two of whole lanes
// merges its lanes' two best keys by xor shuffles; any other split of the experts goes group by group with a masked
// rescan (8 groups of 256 experts: 45 instructions a row against about 500).
template <int PER>
__device__ __forceinline__ void keep_groups(const RouteArgs& a, unsigned (&key)[PER]) {
    const int lane = threadIdx.x & 31, gs = a.group_size, G = a.groups;
    unsigned mine = 0u;                                    // lane g: group g's best key, then its score
    unsigned second = 0u;
    const int lanes = gs / PER;
    if (gs % PER == 0 && (lanes & (lanes - 1)) == 0) {
        unsigned b0 = 0u, b1 = 0u;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            b1 = max(b1, min(b0, key[i]));
            b0 = max(b0, key[i]);
        }
        for (int o = 1; o < lanes; o <<= 1) {
            const unsigned c0 = __shfl_xor_sync(kFull, b0, o), c1 = __shfl_xor_sync(kFull, b1, o);
            b1 = max(max(b1, c1), min(b0, c0));
            b0 = max(b0, c0);
        }
        const int src = lane < G ? lane * lanes : 0;       // G lanes <= 32 PER / PER: in range
        mine = __shfl_sync(kFull, b0, src);
        second = __shfl_sync(kFull, b1, src);
    } else {
        for (int g = 0; g < G; g++) {
            unsigned b0 = 0u, b1 = 0u;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int e = lane * PER + i - g * gs;
                const unsigned v = e >= 0 && e < gs ? key[i] : 0u;
                b1 = max(b1, min(b0, v));
                b0 = max(b0, v);
            }
            const unsigned m0 = __reduce_max_sync(kFull, b0);
            const int first = __ffs(__ballot_sync(kFull, b0 == m0)) - 1;
            const unsigned m1 = __reduce_max_sync(kFull, lane == first ? b1 : b0);
            if (lane == g) {
                mine = m0;
                second = m1;
            }
        }
    }
    const bool some = lane < G && mine != 0u;
    const float best = some ? unordered(mine) : -INFINITY;
    const float score = some && second != 0u ? __fadd_rn(best, unordered(second)) : best;
    int rank = 0;
    for (int g = 0; g < G; g++) {
        const float s = __shfl_sync(kFull, score, g);
        rank += (s > score || (s == score && g < lane)) ? 1 : 0;
    }
    const unsigned keep = __ballot_sync(kFull, some && rank < a.top_groups);
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int g = (lane * PER + i) / gs;
        if (g >= G || !((keep >> g) & 1u)) key[i] = 0u;
    }
}

// The choices of one row by exact keys: lane j gets the j-th.  A choice is the maximum over the lanes' best keys, the
// first lane that has it (the lowest index), and a rescan by that lane.
template <int LANES, int PER>
__device__ __noinline__ int choose_exact(unsigned (&key)[PER], int choices) {
    const int lane = threadIdx.x & (LANES - 1);
    unsigned best = 0u;
    int at = 0, mine = -1;
#pragma unroll
    for (int i = PER - 1; i >= 0; i--)
        if (key[i] >= best) {                              // the lowest of equal keys
            best = key[i];
            at = i;
        }
    for (int j = 0; j < choices; j++) {
        const unsigned top = row_max<LANES>(best);
        const int owner = __ffs(row_ballot<LANES>(best == top)) - 1;
        const int e = __shfl_sync(kFull, lane * PER + at, owner, LANES);
        if (lane == j && top != 0u) mine = e;              // 0: nothing available is left
        if (lane == owner) {
            best = 0u;
            const int gone = at;
#pragma unroll
            for (int i = PER - 1; i >= 0; i--) {
                if (i == gone) key[i] = 0u;
                if (key[i] >= best) {
                    best = key[i];
                    at = i;
                }
            }
        }
    }
    return mine;
}

// The choices of one row.  Key and index share 32 bits: the key's upper bits, then the complement of the index, so one
// maximum finds the best expert, lowest index first, and each lane's words are sorted once (min / max network) and
// popped from the front.  The key's lowest bits are cut off for the index: where two neighbours in the order (the
// first that is not chosen included) agree in all the bits that are left, the rows of the warp are decided by
// choose_exact (`whole`: the cut bits say nothing, as for 16-bit logits without a bias, and equal words are equal keys).
template <int LANES, int PER, bool HALF>
__device__ __forceinline__ int choose(unsigned (&key)[PER], int choices, bool whole) {
    constexpr unsigned INDEX = LANES * PER - 1;
    const int lane = threadIdx.x & (LANES - 1);
    unsigned w[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) w[i] = key[i] ? (key[i] & ~INDEX) | (INDEX - (lane * PER + i)) : 0u;
    auto order = [](unsigned& hi, unsigned& lo) {
        const unsigned m = max(hi, lo);
        lo = min(hi, lo);
        hi = m;
    };
#pragma unroll
    for (int size = 2; size <= PER; size *= 2) {           // bitonic, descending
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int j = i ^ (size - 1);
            if (j > i) order(w[i], w[j]);
        }
#pragma unroll
        for (int d = size / 4; d > 0; d /= 2)
#pragma unroll
            for (int i = 0; i < PER; i++)
                if (!(i & d)) order(w[i], w[i + d]);
    }
    int mine = -1;
    unsigned last = 0u;
    bool close = false;
    for (int j = 0; j < choices; j++) {
        const unsigned top = row_max<LANES>(w[0]);
        if (!(HALF && whole)) close |= top != 0u && ((top ^ last) & ~INDEX) == 0u;
        last = top;
        if (lane == j && top != 0u) mine = (int)(INDEX - (top & INDEX));   // 0: nothing available is left
        if (w[0] == top) {
#pragma unroll
            for (int i = 0; i + 1 < PER; i++) w[i] = w[i + 1];
            w[PER - 1] = 0u;
        }
    }
    if (!(HALF && whole)) {
        const unsigned top = row_max<LANES>(w[0]);         // the first that is not chosen
        close |= top != 0u && ((top ^ last) & ~INDEX) == 0u;
        if (__any_sync(kFull, close)) mine = choose_exact<LANES, PER>(key, choices);
    }
    return mine;
}

template <typename T, int LANES, int PER>
__global__ void __launch_bounds__(kRouteWarps * 32)
    k_route(const T* __restrict__ logits, RouteArgs a, int32_t* __restrict__ ids, float* __restrict__ weights) {
    pdl_wait();
    const int lane = threadIdx.x & (LANES - 1);
    const int64_t slot = (int64_t)blockIdx.x * (kRouteWarps * 32 / LANES) + threadIdx.x / LANES;
    const bool here = slot < a.rows;                       // lanes past the last row go along with it, and store nothing
    const int64_t t = here ? slot : a.rows - 1;
    const T* row = logits + t * a.stride;
    float l[PER];
    load_row<T, PER>(row, lane, a.experts, a.vec, l);
    const bool live = a.mask == nullptr || a.mask[t] != 0;
    float v[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) v[i] = l[i];
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < PER; i++) v[i] = sigmoid32(l[i]);
    }
    if (a.bias != nullptr) {
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (lane * PER + i < a.experts) v[i] = __fadd_rn(v[i], __ldg(a.bias + lane * PER + i));
    }
    unsigned key[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) key[i] = live && l[i] > -INFINITY && v[i] > -INFINITY ? ordered(v[i]) : 0u;
    float m = 0.0f, total = 1.0f;
    if (!a.sigmoid && !a.renorm) {                         // the softmax runs over every available logit
        m = -INFINITY;
#pragma unroll
        for (int i = 0; i < PER; i++) m = l[i] > m ? l[i] : m;
        m = row_max<LANES>(m);
        total = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; i++) total += l[i] > -INFINITY ? exp_below<T>(l[i] - m) : 0.0f;
        total = row_sum<LANES>(total);
    }
    if constexpr (LANES == 32) {
        if (a.groups > 1) keep_groups<PER>(a, key);
    }

    const int mine = choose<LANES, PER, sizeof(T) == 2>(key, a.choices, sizeof(T) == 2 && !a.sigmoid && a.bias == nullptr);
    float w = 0.0f;
    const bool got = mine >= 0;
    const float lm = got ? Elem<T>::to(row[mine]) : -INFINITY;
    if (a.sigmoid) {
        const float s = got ? sigmoid32(lm) : 0.0f;
        if (a.renorm) {
            const float sum = row_sum<LANES>(s);
            w = sum > 0.0f ? s / sum : 0.0f;
        } else {
            w = s;
        }
    } else {
        if (a.renorm) m = row_max<LANES>(lm);
        const float p = got ? exp_below<T>(lm - m) : 0.0f;
        if (a.renorm) total = row_sum<LANES>(p);
        w = got ? share<T>(p, total) : 0.0f;
    }
    if (here && lane < a.choices) {
        ids[t * a.choices + lane] = mine;
        weights[t * a.choices + lane] = a.scale * w;
    }
}

template <typename T, int LANES, int PER>
__global__ void __launch_bounds__(kRouteWarps * 32)
    k_route_grad(const float* __restrict__ dweights, const T* __restrict__ logits, const int32_t* __restrict__ ids,
                 RouteArgs a, T* __restrict__ dlogits) {
    pdl_wait();
    const int lane = threadIdx.x & (LANES - 1);
    const int64_t slot = (int64_t)blockIdx.x * (kRouteWarps * 32 / LANES) + threadIdx.x / LANES;
    const bool here = slot < a.rows;                       // lanes past the last row go along with it, and store nothing
    const int64_t t = here ? slot : a.rows - 1;
    const T* row = logits + t * a.stride;
    T* out = dlogits + t * a.experts;
    int id = lane < a.choices ? ids[t * a.choices + lane] : -1;
    const bool got = id >= 0 && id < a.experts;
    const float g = got ? a.scale * dweights[t * a.choices + lane] : 0.0f;
    const float lm = got ? Elem<T>::to(row[id]) : -INFINITY;

    float p, dot, m = 0.0f, total = 1.0f, slope = 0.0f;
    if (a.sigmoid) {
        const float s = got ? sigmoid32(lm) : 0.0f;
        // 1 - s from exp(l): no cancellation where s is near 1
        slope = got ? s * sigmoid32(-lm) : 0.0f;
        p = s;
        dot = 0.0f;
        if (a.renorm) {
            total = row_sum<LANES>(s);
            // (by every row of the warp, those without a choice too; the quotient first, so that a lone choice's share
            // is 1 and its gradient 0)
            dot = row_sum<LANES>(total > 0.0f ? g * (s / total) : 0.0f);
        }
    } else if (a.renorm) {
        m = row_max<LANES>(lm);
        p = got ? exp_below<T>(lm - m) : 0.0f;
        total = row_sum<LANES>(p);
        p = got ? share<T>(p, total) : 0.0f;
        dot = row_sum<LANES>(g * p);
    }
    float dl[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) dl[i] = 0.0f;
    if (!a.sigmoid && !a.renorm) {
        load_row<T, PER>(row, lane, a.experts, a.vec, dl);
        m = -INFINITY;
#pragma unroll
        for (int i = 0; i < PER; i++) m = dl[i] > m ? dl[i] : m;
        m = row_max<LANES>(m);
        total = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            dl[i] = dl[i] > -INFINITY ? exp_below<T>(dl[i] - m) : 0.0f;
            total += dl[i];
        }
        total = row_sum<LANES>(total);
        p = got ? share<T>(exp_below<T>(lm - m), total) : 0.0f;
        dot = row_sum<LANES>(g * p);
        const bool some = row_ballot<LANES>(got) != 0u;
        const float c = -dot / total;
        // (a row with no choice has a gradient of 0 whatever its logits, +inf and the NaN it makes among them)
#pragma unroll
        for (int i = 0; i < PER; i++) dl[i] = some && dl[i] != 0.0f ? c * dl[i] : 0.0f;
    }
    // the dense row first, then the chosen entries over it
    if (here) store_row<T, PER>(out, lane, a.experts, a.out_vec, dl);
    __syncwarp();
    if (here && got) {
        float v;
        if (a.sigmoid) {
            // (slope / total is at most 1, where (g - dot) / total leaves float32's range at scores around 1e-38)
            v = !a.renorm ? g * slope : total > 0.0f ? (g - dot) * (slope / total) : 0.0f;
        } else {
            v = p * (g - dot);
        }
        out[id] = Elem<T>::from(v);
    }
}

template <typename T, int LANES, int PER>
cudaError_t run_route(const RouteCall& c, RouteArgs a, cudaStream_t st) {
    const int64_t rows = kRouteWarps * 32 / LANES, blocks = (a.rows + rows - 1) / rows;
    a.vec = Vec<T, PER>::level(c.logits, c.stride * (int64_t)sizeof(T));
    a.out_vec = Vec<T, PER>::level(c.dlogits, c.experts * (int64_t)sizeof(T));
    if (c.dweights == nullptr)
        return launch_pdl(k_route<T, LANES, PER>, dim3((unsigned)blocks), dim3(kRouteWarps * 32), 0, st,
                          static_cast<const T*>(c.logits), a, c.ids_out, c.weights);
    return launch_pdl(k_route_grad<T, LANES, PER>, dim3((unsigned)blocks), dim3(kRouteWarps * 32), 0, st, c.dweights,
                      static_cast<const T*>(c.logits), c.ids, a, static_cast<T*>(c.dlogits));
}

template <typename T>
cudaError_t run_route_type(const RouteCall& c, cudaStream_t st) {
    RouteArgs a;
    a.rows = c.rows;
    a.stride = c.stride;
    a.experts = c.experts;
    a.choices = c.choices;
    a.groups = c.groups;
    a.top_groups = c.top_groups;
    a.group_size = c.experts / (c.groups > 0 ? c.groups : 1);
    a.bias = c.bias;
    a.mask = c.mask;
    a.scale = c.scale;
    a.sigmoid = c.sigmoid;
    a.renorm = c.renorm;
    // Few lanes a row where its experts fit and its choices do (lane j holds the j-th): the work that is done once a row
    // is then shared by several rows of a warp.  Groups of experts are compared across a whole warp.
    if (c.groups <= 1) {
        if (c.experts <= 64 && c.choices <= 4) return c.experts <= 32 ? run_route<T, 4, 8>(c, a, st) : run_route<T, 4, 16>(c, a, st);
        if (c.experts <= 64 && c.choices <= 8) return c.experts <= 32 ? run_route<T, 8, 4>(c, a, st) : run_route<T, 8, 8>(c, a, st);
        if (c.experts <= 128 && c.choices <= 8) return run_route<T, 8, 16>(c, a, st);
        if (c.experts <= 128 && c.choices <= 16) return run_route<T, 16, 8>(c, a, st);
        // (sixteen experts a lane take longer for one row: 160 experts, 100 rows 5.3 us at 32 lanes and 7.7 at 16,
        // 8192 rows 13.7 and 12.9, 65536 rows 78.2 and 66.9)
        if (c.experts <= 256 && c.choices <= 16 && c.rows >= 16384) return run_route<T, 16, 16>(c, a, st);
    }
    if (c.experts <= 32) return run_route<T, 32, 1>(c, a, st);
    if (c.experts <= 64) return run_route<T, 32, 2>(c, a, st);
    if (c.experts <= 128) return run_route<T, 32, 4>(c, a, st);
    if (c.experts <= 256) return run_route<T, 32, 8>(c, a, st);
    if (c.experts <= 512) return run_route<T, 32, 16>(c, a, st);
    return run_route<T, 32, 32>(c, a, st);
}

}  // namespace

cudaError_t launch_route(const RouteCall& c, cudaStream_t st) {
    switch (c.dtype) {
        case 0: return run_route_type<float>(c, st);
        case 1: return run_route_type<__nv_bfloat16>(c, st);
        default: return run_route_type<__half>(c, st);
    }
}

}  // namespace kmc
