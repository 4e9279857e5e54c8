// The experts' router (ftcuda/training.h): softmax, top-k, counts and balance loss in one pass over the logits, and its gradient
// in another.
//
//   p = softmax(x_t),  S_t = the k largest x,  w_i = p_{e_i} (over their sum),  c_e = #{(t, i): e_i = e},  P_e = mean_t p_te
//   L = E sum_e f_e P_e,  f_e = c_e / (N k)
//   dL/dx_j = g p_j (s_j - sum_e s_e p_e) with s_e = E f_e / N, and the weights' part: w_i (g_i - sum_i g_i w_i) at the chosen when they are
//   normalised, else p_j (a_j - sum a p) with a = g_i at the chosen
//
// A warp takes a token, a lane some of the experts: the row stays in registers for all that is done with it. A round of top-k is
// a maximum over the warp of keys that order as the logits do. Sums over tokens: each lane keeps its experts' p over all of its
// warp's tokens, a CTA joins its warps and leaves one row of partial sums, and a cluster of eight CTAs adds the rows up; the counts are whole
// numbers in shared memory. One CTA alone (few tokens) finishes by itself, without the second launch.
//
// What bounds it: with few experts latency (16384 x 64 FP32, top 8, as captured graphs: 20.8 us forward, 26.7 with the backward pass, where a kernel that does next to nothing takes 6.2;
// 1.5 us of bytes), with many the forward kernel's chains of dependent whole-number instructions (65535 x 256 BF16, top 8: 45 to 52 us forward at 0.7 TB/s, 66 % of the issue slots used and
// the ALU pipe busy for 62 % of the time), the backward one's latency (31 to 33 us, 2.2 TB/s).
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "ptx.cuh"
#include "training_common.cuh"

namespace ftcuda {
namespace {

namespace cg = cooperative_groups;
using training::Element;

constexpr int kWarps              = 16;  // of the forward kernel's CTA
constexpr int kBackwardWarps      = 8;
constexpr int kCtasPerSm          = 2;
// CTAs of the backward kernel that an SM holds: where a lane has up to 16 bytes of a row few registers are enough, and more rows are on their way
// (65535 x 256 BF16: 36.8 us with four, 32.8 with six; 65536 x 128 FP16: 30.7, 24.6). With more, six are no faster (32768 x 256 FP32: 21.2, 22.7; 16384 x 512
// BF16: 23.0, 24.0).
__host__ __device__ constexpr int backwardCtasPerSm(std::uint64_t bytes) { return bytes <= 16 ? 6 : 4; }
constexpr std::uint32_t kMaxExperts = 1024;
constexpr std::uint32_t kMaxTopK    = 32;
constexpr std::uint32_t kMaxRows    = 512;  // CTAs of the forward kernel at most
constexpr int kFinishCtas         = 8;
constexpr int kFinishThreads      = 512;
constexpr unsigned kAll           = 0xFFFFFFFFU;

// Whole numbers that order as the numbers do: NaN above all, -0 equal to 0. kDead is that of -inf; 0 is below every number.
__device__ __forceinline__ std::uint32_t orderOf(float x) {
    const std::uint32_t bits = __float_as_uint(x + 0.0F);
    const std::uint32_t key  = (bits & 0x80000000U) != 0 ? ~bits : bits | 0x80000000U;
    return x != x ? 0xFFFFFFFFU : key;
}
__device__ __forceinline__ float valueOf(std::uint32_t key) {
    return __uint_as_float((key & 0x80000000U) != 0 ? key & 0x7FFFFFFFU : ~key);  // 0xFFFFFFFF: a NaN again
}
constexpr std::uint32_t kDead = 0x007FFFFFU;

struct RouteParams {
    const void* logits;
    const std::uint8_t* mask;
    std::uint64_t tokens;
    std::int64_t row_stride;
    std::uint32_t experts, top_k;
    std::int32_t normalize;
    float* weights;
    std::int32_t* chosen;
    std::int32_t* counts;
    std::int32_t* routed;
    float* loss;
    float* sums;             // [CTA][experts]
    std::int32_t* hits;      // [CTA][experts]
    std::int32_t* live;      // [CTA]
};

__device__ __forceinline__ float warpSum(float x) {
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2) { x += __shfl_xor_sync(kAll, x, offset); }
    return x;
}

// E sum_e f_e P_e from the sums over all tokens; thread 0's is the result. `shared` has room for a number for each warp.
__device__ __forceinline__ double balance(double part, double* shared) {
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2) { part += __shfl_xor_sync(kAll, part, offset); }
    if ((threadIdx.x & 31) == 0) { shared[threadIdx.x >> 5] = part; }
    __syncthreads();
    double total = 0.0;
    if (threadIdx.x == 0) {
        for (std::uint32_t w = 0; w < blockDim.x / 32; ++w) { total += shared[w]; }
    }
    return total;
}

__device__ __forceinline__ void writeLoss(const RouteParams& p, double total, std::int32_t live) {
    const double n = static_cast<double>(live);
    *p.routed      = live;
    *p.loss        = live == 0 ? 0.0F : static_cast<float>(total * p.experts / (n * p.top_k * n));
}

// Which experts a lane holds, and how they get there. kVector: runs of up to 16 bytes, for rows that are aligned for it and have whole ones.
template<typename T, int kItems, bool kVector> struct Share {
    static constexpr int kMost = 16 / static_cast<int>(sizeof(T));
    static constexpr int kRun  = kVector ? (kItems < kMost ? kItems : kMost) : 1;
    static __device__ __forceinline__ std::uint32_t index(int i, int lane) {
        return static_cast<std::uint32_t>((i / kRun) * 32 * kRun + lane * kRun + i % kRun);
    }
    struct alignas(sizeof(T) * kRun) Run {
        T at[kRun];
    };
    // The lane's part of a row; what lies beyond the last expert is left as it is.
    static __device__ __forceinline__ void load(const T* row, std::uint32_t experts, int lane, T (&out)[kItems]) {
#pragma unroll
        for (int i = 0; i < kItems; i += kRun) {
            if (index(i, lane) < experts) {
                const Run run = *reinterpret_cast<const Run*>(row + index(i, lane));
#pragma unroll
                for (int j = 0; j < kRun; ++j) { out[i + j] = run.at[j]; }
            }
        }
    }
    // The same from a row of FP32 in shared memory that is aligned like the other: four at a time where a run has as many.
    static __device__ __forceinline__ void loadShared(const float* row, std::uint32_t experts, int lane, float (&out)[kItems]) {
        constexpr int kEach = kRun % 4 == 0 ? 4 : kRun % 2 == 0 ? 2 : 1;
        struct alignas(4 * kEach) Part {
            float at[kEach];
        };
#pragma unroll
        for (int i = 0; i < kItems; i += kEach) {
            Part part{};
            if (index(i, lane) < experts) { part = *reinterpret_cast<const Part*>(row + index(i, lane)); }
#pragma unroll
            for (int j = 0; j < kEach; ++j) { out[i + j] = part.at[j]; }
        }
    }
    static __device__ __forceinline__ void store(T* row, std::uint32_t experts, int lane, const T (&in)[kItems]) {
#pragma unroll
        for (int i = 0; i < kItems; i += kRun) {
            if (index(i, lane) < experts) {
                Run run;
#pragma unroll
                for (int j = 0; j < kRun; ++j) { run.at[j] = in[i + j]; }
                *reinterpret_cast<Run*>(row + index(i, lane)) = run;
            }
        }
    }
};

// The k largest logits of a warp's row, the lowest index first among equal ones: lane i gets the key of the i-th, and `first` is the first one's. take()
// gives how many there are above -inf; value() and index() say what a key stands for. A row is -inf beyond the last expert.
template<typename T, int kItems> struct TopK;

// FP32: a round is two reductions, for the key and for the index.
template<int kItems> struct TopK<float, kItems> {
    using Key = std::uint64_t;
    template<typename Place> static __device__ __forceinline__ std::uint32_t take(const float (&x)[kItems], std::uint32_t top_k, int lane, Key& kept, Key& first) {
        std::uint32_t keys[kItems];
#pragma unroll
        for (int i = 0; i < kItems; ++i) { keys[i] = orderOf(x[i]); }
        std::uint32_t round = 0;
        for (; round < top_k; ++round) {
            std::uint32_t best = keys[0];
#pragma unroll
            for (int i = 1; i < kItems; ++i) { best = max(best, keys[i]); }
            best = __reduce_max_sync(kAll, best);
            if (best <= kDead) { break; }
            std::uint32_t at = 0xFFFFFFFFU;
#pragma unroll
            for (int i = kItems - 1; i >= 0; --i) { at = keys[i] == best ? Place::index(i, lane) : at; }
            at = __reduce_min_sync(kAll, at);
#pragma unroll
            for (int i = 0; i < kItems; ++i) { keys[i] = at == Place::index(i, lane) ? 0 : keys[i]; }
            const Key key = static_cast<Key>(best) << 32 | at;
            first         = round == 0 ? key : first;
            kept          = lane == static_cast<int>(round) ? key : kept;
        }
        return round;
    }
    static __device__ __forceinline__ float value(Key key) { return valueOf(static_cast<std::uint32_t>(key >> 32)); }
    static __device__ __forceinline__ std::uint32_t index(Key key) { return static_cast<std::uint32_t>(key); }
};

// 16 bits: a word holds the number's order and, upside down, its index, and one reduction does a round (65535 x 256, top 8: 60 us with all lanes' words
// moved and a question after each round, 52 as here). No two words are equal. Up to eight
// words a lane are sorted first, so that a round only looks at each lane's first one, and the lane it belonged to moves its others up, as many
// as the rounds to come can ask for; more are gone through in each round. No round asks whether anything is left: what comes behind the last one above -inf
// is not above it either.
template<typename T, int kItems> struct TopK {
    using Key = std::int32_t;
    static constexpr bool kSorted       = kItems <= 8;
    static constexpr Key kDead16        = (std::is_same<T, __half>::value ? -0x7C010000 : -0x7F810000) | 0xFFFF;  // the largest of -inf
    static constexpr std::uint32_t kEnd = 8;  // rounds that are written out
    // Adding zero makes -0 the other zero and every NaN the one with all bits but the sign's.
    static __device__ __forceinline__ std::uint32_t bits(T x) {
        const T sum = __hadd(x, Element<T>::narrow(0.0F));
        return *reinterpret_cast<const unsigned short*>(&sum);
    }
    template<bool kMove> static __device__ __forceinline__ Key next(Key (&keys)[kItems], int moved) {
        Key first = keys[0];
        if (!kSorted) {
#pragma unroll
            for (int i = 1; i < kItems; ++i) { first = max(first, keys[i]); }
        }
        const Key key = __reduce_max_sync(kAll, first);
        if (!kMove) { return key; }
        if (kSorted) {
            const bool mine = first == key;
#pragma unroll
            for (int i = 0; i < kItems; ++i) {
                if (i < moved) { keys[i] = mine ? i + 1 < kItems ? keys[i + 1] : INT32_MIN : keys[i]; }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kItems; ++i) { keys[i] = keys[i] == key ? INT32_MIN : keys[i]; }
        }
        return key;
    }
    template<typename Place> static __device__ __forceinline__ std::uint32_t take(const T (&x)[kItems], std::uint32_t top_k, int lane, Key& kept, Key& first) {
        Key keys[kItems];
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const Key word = static_cast<Key>(bits(x[i]) << 16 | (0xFFFFU - Place::index(i, lane)));
            keys[i]        = word ^ (word >> 31 & 0x7FFF0000);  // negative numbers the other way round
        }
        if (kSorted) {
            // Odd-even merging (Batcher's network).
#pragma unroll
            for (int size = 1; size < kItems; size *= 2) {
#pragma unroll
                for (int gap = size; gap > 0; gap /= 2) {
#pragma unroll
                    for (int start = gap % size; start + gap < kItems; start += 2 * gap) {
#pragma unroll
                        for (int i = 0; i < gap; ++i) {
                            if (i + start + gap < kItems && (i + start) / (2 * size) == (i + start + gap) / (2 * size)) {
                                const Key low = keys[i + start], high = keys[i + start + gap];
                                keys[i + start]       = max(low, high);
                                keys[i + start + gap] = min(low, high);
                            }
                        }
                    }
                }
            }
        }
        kept                = INT32_MIN;
        std::uint32_t round = 0;
        const auto note     = [&](Key key) {
            first = round == 0 ? key : first;
            kept  = lane == static_cast<int>(round) ? key : kept;
            ++round;
        };
        for (; round + kEnd < top_k;) { note(next<true>(keys, kItems)); }
#pragma unroll
        for (std::uint32_t left = kEnd; left > 0; --left) {  // as many as there still can be
            if (round + left == top_k) { left == 1 ? note(next<false>(keys, 0)) : note(next<true>(keys, static_cast<int>(left) - 1)); }
        }
        return static_cast<std::uint32_t>(__popc(__ballot_sync(kAll, kept > kDead16)));
    }
    static __device__ __forceinline__ float value(Key key) {
        const unsigned short word = static_cast<unsigned short>((key ^ (key >> 31 & 0x7FFF0000)) >> 16);
        return Element<T>::widen(*reinterpret_cast<const T*>(&word));
    }
    static __device__ __forceinline__ std::uint32_t index(Key key) { return 0xFFFFU - (static_cast<std::uint32_t>(key) & 0xFFFFU); }
};

// e^x, within a few units of the last place for the arguments that a softmax has (|x| 2^-24 more for large ones).
__device__ __forceinline__ float expFast(float x) { return exp2Fast(x * 1.4426950408889634F); }

template<typename T, int kItems, bool kVector> __global__ void __launch_bounds__(kWarps * 32) routeTokens(const RouteParams p) {
    using Place = Share<T, kItems, kVector>;
    using Top   = TopK<T, kItems>;
    extern __shared__ unsigned char memory[];
    auto* const hits = reinterpret_cast<std::int32_t*>(memory);  // [experts]
    auto* const rows = reinterpret_cast<float*>(hits + p.experts);  // [kWarps / 2][experts]
    __shared__ std::int32_t live_total;
    __shared__ double shared[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (std::uint32_t e = threadIdx.x; e < p.experts; e += kWarps * 32) { hits[e] = 0; }
    if (threadIdx.x == 0) { live_total = 0; }
    __syncthreads();
    gridDependencyWait();
    gridDependencyLaunchDependents();

    float sums[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) { sums[i] = 0.0F; }
    std::int32_t live = 0;
    T raw[kItems];  // -inf beyond the last expert
#pragma unroll
    for (int i = 0; i < kItems; ++i) { raw[i] = Element<T>::narrow(-INFINITY); }
    const std::uint64_t step = static_cast<std::uint64_t>(gridDim.x) * kWarps;
    for (std::uint64_t token = static_cast<std::uint64_t>(blockIdx.x) * kWarps + warp; token < p.tokens; token += step) {
        Place::load(static_cast<const T*>(p.logits) + static_cast<std::int64_t>(token) * p.row_stride, p.experts, lane, raw);
        const bool on = p.mask == nullptr || p.mask[token] != 0;
        std::int32_t mine  = -1;
        float value        = 0.0F, weight = 0.0F;
        if (on) {
            typename Top::Key kept = 0, first = 0;
            const std::uint32_t found = Top::template take<Place>(raw, p.top_k, lane, kept, first);
            if (lane < static_cast<int>(found)) {
                mine  = static_cast<std::int32_t>(Top::index(kept));
                value = Top::value(kept);
            }
            const float largest = found != 0 ? Top::value(first) : -INFINITY;
            float x[kItems];
#pragma unroll
            for (int i = 0; i < kItems; ++i) { x[i] = Element<T>::widen(raw[i]); }
            if (largest != -INFINITY) {  // (not a number included)
                float total = 0.0F;
#pragma unroll
                for (int i = 0; i < kItems; ++i) {
                    x[i] = expFast(x[i] - largest);
                    total += x[i];
                }
                total               = warpSum(total);
                const float inverse = 1.0F / total;
#pragma unroll
                for (int i = 0; i < kItems; ++i) { sums[i] += x[i] * inverse; }
                weight = mine >= 0 ? expFast(value - largest) : 0.0F;
                weight /= p.normalize != 0 ? warpSum(weight) : total;
                ++live;
            }
        }
        if (lane < static_cast<int>(p.top_k)) {
            p.weights[token * p.top_k + lane] = weight;
            p.chosen[token * p.top_k + lane]  = mine;
            if (mine >= 0) { atomicAdd(hits + mine, 1); }
        }
    }
    if (lane == 0 && live != 0) { atomicAdd(&live_total, live); }
    // The warps' sums, half of them onto the other half at a time.
#pragma unroll
    for (int half = kWarps / 2; half > 0; half /= 2) {
        if (warp >= half && warp < 2 * half) {
#pragma unroll
            for (int i = 0; i < kItems; ++i) {
                if (Place::index(i, lane) < p.experts) { rows[(warp - half) * p.experts + Place::index(i, lane)] = sums[i]; }
            }
        }
        __syncthreads();
        if (warp < half) {
#pragma unroll
            for (int i = 0; i < kItems; ++i) {
                if (Place::index(i, lane) < p.experts) { sums[i] += rows[warp * p.experts + Place::index(i, lane)]; }
            }
        }
        __syncthreads();
    }
    if (gridDim.x > 1) {
        const std::uint64_t at = static_cast<std::uint64_t>(blockIdx.x) * p.experts;
        if (warp == 0) {
#pragma unroll
            for (int i = 0; i < kItems; ++i) {
                if (Place::index(i, lane) < p.experts) { p.sums[at + Place::index(i, lane)] = sums[i]; }
            }
        }
        for (std::uint32_t e = threadIdx.x; e < p.experts; e += kWarps * 32) { p.hits[at + e] = hits[e]; }
        if (threadIdx.x == 0) { p.live[blockIdx.x] = live_total; }
        return;
    }
    // The only CTA.
    double part = 0.0;
    if (warp == 0) {
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const std::uint32_t e = Place::index(i, lane);
            if (e < p.experts) { part += static_cast<double>(sums[i]) * hits[e]; }
        }
    }
    for (std::uint32_t e = threadIdx.x; e < p.experts; e += kWarps * 32) { p.counts[e] = hits[e]; }
    const double total = balance(part, shared);
    if (threadIdx.x == 0) { writeLoss(p, total, live_total); }
}

// Shared memory of the kernel below, in words: the sums (two words each), those of the groups with their counts, the counts, one more.
__host__ __device__ __forceinline__ std::uint32_t finishWords(std::uint32_t experts) {
    const std::uint32_t groups = experts < kFinishThreads ? kFinishThreads / experts : 1;
    return 2 * experts + 3 * groups * experts + experts + 1;
}

// The rows of partial sums added up: each CTA of the cluster an eighth of them, the first CTA what they come to.
__global__ void __cluster_dims__(kFinishCtas, 1, 1) __launch_bounds__(kFinishThreads) finishRouting(const RouteParams p, std::uint32_t rows) {
    extern __shared__ unsigned char memory[];
    auto* const sums = reinterpret_cast<double*>(memory);                   // [experts]
    auto* const hits = reinterpret_cast<std::int32_t*>(sums) + finishWords(p.experts) - p.experts - 1;  // [experts], then the number of live tokens
    __shared__ double shared[kFinishThreads / 32];
    cg::cluster_group cluster = cg::this_cluster();
    const std::uint32_t rank  = cluster.block_rank();
    gridDependencyWait();
    gridDependencyLaunchDependents();
    const std::uint32_t first = rows * rank / kFinishCtas, last = rows * (rank + 1) / kFinishCtas;
    // Threads beyond the experts take other rows: `groups` of them for each expert, one row in so many each.
    const std::uint32_t groups = max(1U, kFinishThreads / p.experts);
    const std::uint32_t group  = threadIdx.x / p.experts;  // (with more experts than threads, a thread takes several)
    double* const group_sums       = sums + p.experts;
    std::int32_t* const group_hits = reinterpret_cast<std::int32_t*>(group_sums + groups * p.experts);
    if (group < groups || groups == 1) {
        for (std::uint32_t e = threadIdx.x - (groups == 1 ? 0 : group * p.experts); e < p.experts; e += kFinishThreads) {
            double sum         = 0.0;
            std::int32_t count = 0;
#pragma unroll 8
            for (std::uint32_t row = first + (groups == 1 ? 0 : group); row < last; row += groups) {
                sum += static_cast<double>(__ldcg(p.sums + static_cast<std::uint64_t>(row) * p.experts + e));
                count += __ldcg(p.hits + static_cast<std::uint64_t>(row) * p.experts + e);
            }
            group_sums[(groups == 1 ? 0 : group) * p.experts + e] = sum;
            group_hits[(groups == 1 ? 0 : group) * p.experts + e] = count;
        }
    }
    __syncthreads();
    for (std::uint32_t e = threadIdx.x; e < p.experts; e += kFinishThreads) {
        double sum         = 0.0;
        std::int32_t count = 0;
        for (std::uint32_t g = 0; g < groups; ++g) {
            sum += group_sums[g * p.experts + e];
            count += group_hits[g * p.experts + e];
        }
        sums[e] = sum;
        hits[e] = count;
    }
    if (threadIdx.x < 32) {
        std::int32_t live = 0;
        for (std::uint32_t row = first + threadIdx.x; row < last; row += 32) { live += __ldcg(p.live + row); }
        live = __reduce_add_sync(kAll, live);
        if (threadIdx.x == 0) { hits[p.experts] = live; }
    }
    cluster.sync();
    if (rank == 0) {
        double part       = 0.0;
        std::int32_t live = 0;
        for (std::uint32_t e = threadIdx.x; e < p.experts; e += kFinishThreads) {
            double sum         = 0.0;
            std::int32_t count = 0;
#pragma unroll
            for (int r = 0; r < kFinishCtas; ++r) {
                sum += cluster.map_shared_rank(sums, r)[e];
                count += cluster.map_shared_rank(hits, r)[e];
            }
            p.counts[e] = count;
            part += sum * count;
        }
        const double total = balance(part, shared);
        if (threadIdx.x == 0) {
            for (int r = 0; r < kFinishCtas; ++r) { live += cluster.map_shared_rank(hits, r)[p.experts]; }
            writeLoss(p, total, live);
        }
    }
    cluster.sync();  // nobody leaves while its shared memory is read
}

struct RouteGradient {
    const void* logits;
    std::uint64_t tokens;
    std::int64_t row_stride, grad_row_stride;
    std::uint32_t experts, top_k;
    std::int32_t normalize;
    const float* weights;
    const std::int32_t* chosen;
    const std::int32_t* counts;
    const std::int32_t* routed;
    const float* grad_weights;
    const float* grad_loss;
    void* grad_logits;
};

template<typename T, int kItems, bool kVector> __global__ void __launch_bounds__(kBackwardWarps * 32, backwardCtasPerSm(kItems * sizeof(T)) == 6 ? 6 : 1) routeGradient(const RouteGradient p) {
    using Place = Share<T, kItems, kVector>;
    extern __shared__ unsigned char memory[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto* const extra = reinterpret_cast<float*>(memory) + warp * p.experts;  // what the weights add at the chosen experts
    for (std::uint32_t e = lane; e < p.experts; e += 32) { extra[e] = 0.0F; }
    __syncwarp();
    gridDependencyWait();
    gridDependencyLaunchDependents();
    const std::int32_t routed = *p.routed;
    const float gradient      = p.grad_loss != nullptr && routed != 0 ? *p.grad_loss : 0.0F;
    const float unit          = routed != 0 ? static_cast<float>(static_cast<double>(p.experts) / (static_cast<double>(routed) * p.top_k * routed)) : 0.0F;
    float slope[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const std::uint32_t e = Place::index(i, lane);
        slope[i]              = e < p.experts ? gradient * (unit * static_cast<float>(p.counts[e])) : 0.0F;
    }
    // What the next token needs is on its way while this one is worked on.
    const std::uint64_t step = static_cast<std::uint64_t>(gridDim.x) * kBackwardWarps;
    std::uint64_t token      = static_cast<std::uint64_t>(blockIdx.x) * kBackwardWarps + warp;
    T ahead[kItems];  // -inf beyond the last expert
#pragma unroll
    for (int i = 0; i < kItems; ++i) { ahead[i] = Element<T>::narrow(-INFINITY); }
    std::int32_t ahead_mine = -1;
    float ahead_weight = 0.0F, ahead_upstream = 0.0F;
    const auto ask = [&](std::uint64_t t) {
        if (t < p.tokens) {
            Place::load(static_cast<const T*>(p.logits) + static_cast<std::int64_t>(t) * p.row_stride, p.experts, lane, ahead);
            if (lane < static_cast<int>(p.top_k)) {
                ahead_mine     = min(p.chosen[t * p.top_k + lane], static_cast<std::int32_t>(p.experts) - 1);  // (never beyond, whatever stands there)
                ahead_weight   = p.weights[t * p.top_k + lane];
                ahead_upstream = p.grad_weights != nullptr ? p.grad_weights[t * p.top_k + lane] : 0.0F;
            }
        }
    };
    ask(token);
    for (; token < p.tokens; token += step) {
        T* const out            = static_cast<T*>(p.grad_logits) + static_cast<std::int64_t>(token) * p.grad_row_stride;
        const std::int32_t mine = ahead_mine;
        const float weight = mine >= 0 ? ahead_weight : 0.0F, upstream = mine >= 0 ? ahead_upstream : 0.0F;
        T raw[kItems];
#pragma unroll
        for (int i = 0; i < kItems; ++i) { raw[i] = ahead[i]; }
        ask(token + step);
        if (__shfl_sync(kAll, mine, 0) < 0) {  // took no part
#pragma unroll
            for (int i = 0; i < kItems; ++i) { raw[i] = Element<T>::narrow(0.0F); }
            Place::store(out, p.experts, lane, raw);
            continue;
        }
        float x[kItems];
#pragma unroll
        for (int i = 0; i < kItems; ++i) { x[i] = Element<T>::widen(raw[i]); }
        float largest = x[0];
#pragma unroll
        for (int i = 1; i < kItems; ++i) { largest = fmaxf(largest, x[i]); }
#pragma unroll
        for (int offset = 16; offset > 0; offset /= 2) { largest = fmaxf(largest, __shfl_xor_sync(kAll, largest, offset)); }
        float total = 0.0F, mean = 0.0F;
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            x[i] = expFast(x[i] - largest);
            total += x[i];
            mean += x[i] * slope[i];
        }
        total               = warpSum(total);
        const float inverse = 1.0F / total;
        const float inner   = warpSum(weight * upstream);
        // Normalised, the weights are a softmax of their own; otherwise they are the whole softmax's, and shift its mean.
        mean                = warpSum(mean) * inverse + (p.normalize != 0 ? 0.0F : inner);
        const float added   = weight * (upstream - (p.normalize != 0 ? inner : 0.0F));
        if (mine >= 0) { extra[mine] = added; }
        __syncwarp();
        float more[kItems];
        Place::loadShared(extra, p.experts, lane, more);
#pragma unroll
        for (int i = 0; i < kItems; ++i) { raw[i] = Element<T>::narrow(fmaf(x[i] * inverse, slope[i] - mean, more[i])); }
        Place::store(out, p.experts, lane, raw);
        __syncwarp();
        if (mine >= 0) { extra[mine] = 0.0F; }
        __syncwarp();
    }
}

// ---------------------------------------------------------------- host

const char* check(const FtcudaRouting& r) {
    if (training::elementBytes(r.element) == 0) { return "the logits must be FP32, FP16 or BF16"; }
    if (r.experts == 0 || r.experts > kMaxExperts) { return "1 to 1024 experts"; }
    if (r.top_k == 0 || r.top_k > r.experts || r.top_k > kMaxTopK) { return "top_k must be from 1 to the number of experts, and at most 32"; }
    if (r.tokens >= (1ULL << 31)) { return "too many tokens"; }
    if (r.tokens == 0) { return nullptr; }
    if (r.logits == nullptr || !training::aligned(r.logits, training::elementBytes(r.element))) { return "the logits have no address, or one that is not a multiple of their element's size"; }
    if (r.tokens > 1 && (r.row_stride < static_cast<std::int64_t>(r.experts) || r.row_stride >= (1LL << 31))) { return "the logits' rows overlap, or lie too far apart"; }
    return nullptr;
}

// Whether the gradient is written where the backward call reads: but over the logits themselves, which a warp reads before it writes them.
bool overInputs(const FtcudaRouting& r, const float* weights, const std::int32_t* chosen, const std::int32_t* counts, const std::int32_t* routed, const float* grad_weights,
                const float* grad_loss, const void* out, std::int64_t out_stride) {
    const std::uint64_t bytes   = training::elementBytes(r.element), slots = r.tokens * r.top_k;
    const training::Range range = training::rangeOf(out, r.tokens, r.experts, out_stride, bytes);
    const auto met = [&](const void* at, std::uint64_t words) { return at != nullptr && training::meet(range, training::rangeOf(at, 1, words, 0, 4)); };
    if (met(weights, slots) || met(chosen, slots) || met(counts, r.experts) || met(routed, 1) || met(grad_weights, slots) || met(grad_loss, 1)) { return true; }
    const bool same = out == r.logits && (r.tokens == 1 || out_stride == r.row_stride);
    return !same && training::meet(range, training::rangeOf(r.logits, r.tokens, r.experts, r.row_stride, bytes));
}

bool wordAligned(const void* pointer) { return pointer != nullptr && training::aligned(pointer, 4); }

// CTAs of the forward kernel: a warp's worth of tokens at least, the SMs filled at most. 32 tokens and fewer stay in one.
std::uint32_t forwardRows(std::uint64_t tokens, std::uint32_t sms) {
    if (tokens <= 2 * kWarps) { return 1; }
    return static_cast<std::uint32_t>(std::min<std::uint64_t>(ceilDiv(tokens, kWarps), std::min(kMaxRows, sms * kCtasPerSm)));
}

// One of the kernels' instantiations: by type, experts for each lane, and whether the lanes' runs of experts (two, four, or 16 bytes' worth) are whole
// and aligned in every row that the call names. (65535 tokens in BF16, top 8: backward 41 us one by one with 255 experts, 33 in runs of eight with 256; forward 52 either way.)
template<template<typename, int, bool> class Pick, typename Kernel> Kernel choose(std::int32_t element, std::uint32_t experts, bool vector) {
    const auto typed = [&](auto sample) -> Kernel {
        using T          = decltype(sample);
        const auto sized = [&](auto items) -> Kernel { return vector ? Pick<T, decltype(items)::value, true>::kernel : Pick<T, decltype(items)::value, false>::kernel; };
        if (experts <= 32) { return Pick<T, 1, false>::kernel; }
        if (experts <= 64) { return sized(std::integral_constant<int, 2>{}); }
        if (experts <= 128) { return sized(std::integral_constant<int, 4>{}); }
        if (experts <= 256) { return sized(std::integral_constant<int, 8>{}); }
        if (experts <= 512) { return sized(std::integral_constant<int, 16>{}); }
        return sized(std::integral_constant<int, 32>{});
    };
    switch (element) {
        case FTCUDA_ELEMENT_FP32: return typed(float{});
        case FTCUDA_ELEMENT_FP16: return typed(__half{});
        default: return typed(__nv_bfloat16{});
    }
}
template<typename T, int kItems, bool kVector> struct Forward { static constexpr auto kernel = &routeTokens<T, kItems, kVector>; };
template<typename T, int kItems, bool kVector> struct Backward { static constexpr auto kernel = &routeGradient<T, kItems, kVector>; };

// Whether a matrix of [tokens][experts] can be gone through in a lane's runs.
bool wholeRuns(const void* at, std::uint64_t tokens, std::int64_t row_stride, std::uint32_t experts, std::int32_t element) {
    const std::uint64_t bytes = training::elementBytes(element);
    const std::uint64_t items = experts <= 64 ? 2 : experts <= 128 ? 4 : 8;
    const std::uint64_t run   = std::min(items, 16 / bytes);
    return experts % run == 0 && training::aligned(at, run * bytes) && (tokens <= 1 || static_cast<std::uint64_t>(row_stride) % run == 0);
}

}  // namespace
}  // namespace ftcuda

extern "C" uint64_t ftcuda_expert_routing_workspace_bytes(const FtcudaRouting* routing) {
    if (routing == nullptr) { return 0; }
    const std::uint64_t rows = std::min<std::uint64_t>(ftcuda::kMaxRows, ftcuda::ceilDiv(routing->tokens, ftcuda::kWarps) + 1);
    return rows * (8ULL * std::min(routing->experts, ftcuda::kMaxExperts) + 4);
}

extern "C" int ftcuda_expert_routing(const FtcudaRouting* routing, float* weights, int32_t* experts, int32_t* counts, int32_t* routed, float* balance_loss,
                                     void* workspace, uint64_t workspace_bytes, void* stream, char* message, size_t message_capacity) {
    using namespace ftcuda;
    if (routing == nullptr) { return fail(message, message_capacity, 1, "null routing"); }
    const FtcudaRouting& r = *routing;
    if (const char* reason = check(r)) { return fail(message, message_capacity, 1, "%s", reason); }
    if (!wordAligned(counts) || !wordAligned(routed) || !wordAligned(balance_loss) || (r.tokens != 0 && (!wordAligned(weights) || !wordAligned(experts)))) {
        return fail(message, message_capacity, 1, "an output has no address, or one that is not a multiple of four");
    }
    const std::uint64_t needed = ftcuda_expert_routing_workspace_bytes(routing);
    if (!wordAligned(workspace) || workspace_bytes < needed) {
        return fail(message, message_capacity, 1, "workspace of %llu bytes needed, at a multiple of four", static_cast<unsigned long long>(needed));
    }
    int sms = 0;
    if (!training::deviceIsCurrent(r.device, message, message_capacity) || !deviceSmCount(r.device, &sms, message, message_capacity)) { return 1; }
    const std::uint32_t rows = forwardRows(r.tokens, static_cast<std::uint32_t>(sms));
    RouteParams p{};
    p.logits     = r.logits;
    p.mask       = r.mask;
    p.tokens     = r.tokens;
    p.row_stride = r.row_stride;
    p.experts    = r.experts;
    p.top_k      = r.top_k;
    p.normalize  = r.normalize;
    p.weights    = weights;
    p.chosen     = experts;
    p.counts     = counts;
    p.routed     = routed;
    p.loss       = balance_loss;
    p.sums       = static_cast<float*>(workspace);
    p.hits       = reinterpret_cast<std::int32_t*>(p.sums + static_cast<std::uint64_t>(rows) * r.experts);
    p.live       = p.hits + static_cast<std::uint64_t>(rows) * r.experts;
    const auto kernel              = choose<Forward, void (*)(RouteParams)>(r.element, r.experts, wholeRuns(r.logits, r.tokens, r.row_stride, r.experts, r.element));
    const std::size_t shared_bytes = r.experts * 4ULL * (1 + kWarps / 2);
    kernel<<<rows, kWarps * 32, shared_bytes, static_cast<cudaStream_t>(stream)>>>(p);
    cudaError_t error = cudaGetLastError();
    if (error == cudaSuccess) {
        countLaunches(1);
        if (rows > 1) {
            error = training::launchOverlapped(finishRouting, dim3(kFinishCtas), dim3(kFinishThreads), finishWords(r.experts) * 4ULL, static_cast<cudaStream_t>(stream), p, rows);
        }
    }
    if (error != cudaSuccess) { return fail(message, message_capacity, 1, "%s", cudaGetErrorString(error)); }
    return 0;
}

extern "C" int ftcuda_expert_routing_backward(const FtcudaRouting* routing, const float* weights, const int32_t* experts, const int32_t* counts,
                                              const int32_t* routed, const float* grad_weights, const float* grad_loss, void* grad_logits,
                                              int64_t grad_row_stride, void* stream, char* message, size_t message_capacity) {
    using namespace ftcuda;
    if (routing == nullptr) { return fail(message, message_capacity, 1, "null routing"); }
    const FtcudaRouting& r = *routing;
    if (const char* reason = check(r)) { return fail(message, message_capacity, 1, "%s", reason); }
    if (r.tokens == 0) { return 0; }
    if (!wordAligned(weights) || !wordAligned(experts) || !wordAligned(counts) || !wordAligned(routed) || (grad_weights != nullptr && !wordAligned(grad_weights)) ||
        (grad_loss != nullptr && !wordAligned(grad_loss))) {
        return fail(message, message_capacity, 1, "an input has no address, or one that is not a multiple of four");
    }
    if (grad_logits == nullptr || !training::aligned(grad_logits, training::elementBytes(r.element))) {
        return fail(message, message_capacity, 1, "the gradient has no address, or one that is not a multiple of its element's size");
    }
    if (r.tokens > 1 && (grad_row_stride < static_cast<std::int64_t>(r.experts) || grad_row_stride >= (1LL << 31))) {
        return fail(message, message_capacity, 1, "the gradient's rows overlap, or lie too far apart");
    }
    if (overInputs(r, weights, experts, counts, routed, grad_weights, grad_loss, grad_logits, grad_row_stride)) {
        return fail(message, message_capacity, 1, "the gradient lies across something that the call reads");
    }
    int sms = 0;
    if (!training::deviceIsCurrent(r.device, message, message_capacity) || !deviceSmCount(r.device, &sms, message, message_capacity)) { return 1; }
    RouteGradient p{};
    p.logits          = r.logits;
    p.tokens          = r.tokens;
    p.row_stride      = r.row_stride;
    p.grad_row_stride = grad_row_stride;
    p.experts         = r.experts;
    p.top_k           = r.top_k;
    p.normalize       = r.normalize;
    p.weights         = weights;
    p.chosen          = experts;
    p.counts          = counts;
    p.routed          = routed;
    p.grad_weights    = grad_weights;
    p.grad_loss       = grad_loss;
    p.grad_logits     = grad_logits;
    const auto kernel              = choose<Backward, void (*)(RouteGradient)>(r.element, r.experts, wholeRuns(r.logits, r.tokens, r.row_stride, r.experts, r.element) &&
                                                                                                                         wholeRuns(grad_logits, r.tokens, grad_row_stride, r.experts, r.element));
    const std::uint32_t grid       = static_cast<std::uint32_t>(std::min<std::uint64_t>(ceilDiv(r.tokens, kBackwardWarps), static_cast<std::uint64_t>(sms) * backwardCtasPerSm(ceilDiv(r.experts, 32) * training::elementBytes(r.element))));
    const std::size_t shared_bytes = r.experts * 4ULL * kBackwardWarps;
    kernel<<<grid, kBackwardWarps * 32, shared_bytes, static_cast<cudaStream_t>(stream)>>>(p);
    const cudaError_t error = cudaGetLastError();
    if (error != cudaSuccess) { return fail(message, message_capacity, 1, "%s", cudaGetErrorString(error)); }
    countLaunches(1);
    return 0;
}
