// The cross entropy of a product with a large vocabulary (ftcuda/training.h).
//
//   z_tv = h_t . w_v,   lse_t = log sum_v exp z_tv,   l_t = lse_t - z_{t, y_t}
//   dz_tv = g_t (exp(z_tv - lse_t) - [v = y_t]),   dH = dZ W,   dW = dZ^T H
//
// The forward call is one pass over the vocabulary, 2 T V D operations; the backward call goes through the vocabulary piece by
// piece and computes Z of a piece again: dZ of it, then dH += dZ W and dW = dZ^T H, 6 T V D. A piece is as wide as kPieceBytes of dZ allow, so that
// the passes over dH (one for each piece) and the launches weigh little. The step call does both without
// computing Z twice, 6 T V D in all, where kStepBytes have room for all of Z's exponentials, 16 bits each (FP32: for Z):
// a pass over them, two bytes read and two written for each, makes them dZ for an upstream gradient of 1, and what comes from it is multiplied by the one there is.
// dZ waits for that in a memory of its own, with the gathered hidden states and, where the limit has room for it, the weight's copy or planes.
//
// Tokens without a target are left out first: the others' hidden states are gathered into the workspace, which costs one pass over H,
// makes what the padding holds irrelevant (a NaN there would reach dW through 0 * NaN), spares the products those rows, and gives
// the tensor cores an aligned operand whatever H's strides. How many there are only the GPU knows; the kernels read it there.
//
// BF16 and FP16 operands go through loss_products.cu, and FP32 ones as sums of three BF16, which takes six products for each. Where the library's
// own FP32 products in their prepared form (three FP16 products) are ahead, FP32 operands go through those instead, chosen by the same rules as the
// host pipeline's (gemm_choice.hpp), with Z of a piece in the workspace and a pass over it for the statistics or dZ: see libraryPays.
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "gemm_choice.hpp"
#include "loss_products.hpp"
#include "ptx.cuh"
#include "training_common.cuh"

namespace ftcuda {
namespace {

using loss::LiveRows;
using training::Element;

constexpr int kListThreads             = 1024;
constexpr int kGatherThreads           = 256;
constexpr int kSplitCtasPerSm          = 8;
constexpr int kJoinRows                = 32;   // rows of a CTA that joins statistics ...
constexpr int kJoinWarps               = 32;   // ... each of its warps some of the pieces
constexpr int kRowThreads              = 256;  // FP32: threads that go over a row of logits
constexpr std::uint64_t kPieceBytes    = 512ULL << 20;  // of dZ (FP32: of Z), unless ...
constexpr std::uint64_t kLeastColumns  = 8192;          // ... that is fewer columns than these
constexpr std::uint64_t kStepBytes     = 2ULL << 30;    // that the step call's exponentials may take at most
constexpr std::uint64_t kAlign         = 256;
constexpr int kKeptRows                = 32;            // rows of a CTA that turns exponentials into slopes ...
constexpr int kKeptPieces              = 4;             // ... and pieces of the statistics
constexpr int kKeptBatch               = 2;             // packs that a thread asks for at a time

// ---------------------------------------------------------------- kernels

struct ListParams {
    const std::int64_t* target;
    std::int64_t ignore_index, vocabulary;
    std::uint32_t tokens;
    std::int32_t reduction;
    LiveRows rows;
    std::int32_t* slot;        // [tokens]: a token's row, -1 for none
    // where a loss is wanted: written for the tokens that take no part
    float* loss;               // NULL with a reduction
    float* lse;
    // where gradients are
    const float* saved_lse;    // NULL in the step call, which has none yet
    const float* grad_loss;    // NULL: 1
    std::int32_t scale_bits;   // log2 of what the largest |scale| is brought near to; INT_MIN: the scales stay as they are
};

// One CTA: the list of live tokens, and (where gradients are wanted) their scales.
template<bool kScales> __global__ void __launch_bounds__(kListThreads) listTokens(const ListParams p) {
    __shared__ std::uint32_t warp_counts[kListThreads / 32];
    __shared__ std::uint32_t largest_bits;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) { largest_bits = 0; }
    gridDependencyWait();
    gridDependencyLaunchDependents();
    std::uint32_t count = 0, largest = 0;
    for (std::uint32_t base = 0; base < p.tokens; base += kListThreads) {
        const std::uint32_t t = base + threadIdx.x;
        std::int64_t y        = 0;
        bool on               = false;
        if (t < p.tokens) {
            y  = p.target[t];
            on = y != p.ignore_index;
        }
        const unsigned ballot = __ballot_sync(0xFFFFFFFFU, on);
        if (lane == 0) { warp_counts[warp] = __popc(ballot); }
        __syncthreads();
        const std::uint32_t mine   = warp_counts[lane];
        const std::uint32_t before = __reduce_add_sync(0xFFFFFFFFU, lane < warp ? mine : 0);
        const std::uint32_t all    = __reduce_add_sync(0xFFFFFFFFU, mine);
        __syncthreads();
        if (t < p.tokens) {
            const std::uint32_t at = count + before + __popc(ballot & ((1U << lane) - 1));
            p.slot[t]              = on ? static_cast<std::int32_t>(at) : -1;
            if (on) {
                p.rows.token[at]  = static_cast<std::int32_t>(t);
                p.rows.target[at] = y >= 0 && y < p.vocabulary ? static_cast<std::int32_t>(y) : loss::kBadTarget;
                if (kScales && p.reduction == FTCUDA_REDUCTION_NONE) { largest = max(largest, __float_as_uint(p.grad_loss[t]) & 0x7FFFFFFFU); }
            } else {
                if (p.lse != nullptr) { p.lse[t] = 0.0F; }
                if (p.loss != nullptr) { p.loss[t] = 0.0F; }
            }
        }
        count += all;
    }
    const std::uint32_t padded = (max(count, 1U) + loss::kTileRows - 1) / loss::kTileRows * loss::kTileRows;
    if (kScales) {
        float common = 0.0F;
        if (p.reduction != FTCUDA_REDUCTION_NONE) {
            common = p.grad_loss != nullptr ? *p.grad_loss : 1.0F;
            if (p.reduction == FTCUDA_REDUCTION_MEAN) { common /= static_cast<float>(max(count, 1U)); }
        }
        atomicMax(&largest_bits, largest);
        __syncthreads();
        // With one upstream gradient for all, the scale is the power of two alone, so that -1, the slope of a target that has hardly any
        // probability, stays exact (BF16's rounding of -1 / N would be off by the same for every token). With one for each, the largest |scale|
        // becomes a number in [1, 2) 2^scale_bits; not beyond 2^100 times larger, and not where it is 0 or not a number.
        const bool each    = p.reduction == FTCUDA_REDUCTION_NONE;
        const bool rounded = p.scale_bits != INT32_MIN;
        const float top    = __uint_as_float(largest_bits);
        std::int32_t shift = 0;
        if (rounded) { shift = p.scale_bits - (each && top > 0.0F && top <= FLT_MAX ? max(-100, ilogbf(top)) : 0); }
        if (rounded && !each) {
            if (threadIdx.x == 0) { *p.rows.unit = ldexpf(common, -shift); }
            common = 1.0F;
        } else if (threadIdx.x == 0) {
            *p.rows.unit = ldexpf(1.0F, -shift);
        }
        for (std::uint32_t i = threadIdx.x; i < padded; i += kListThreads) {
            float scale = 0.0F, lse2 = 0.0F;
            if (i < count) {
                const std::int32_t t = p.rows.token[i];
                scale                = ldexpf(each ? p.grad_loss[t] : common, shift);
                lse2                 = p.saved_lse != nullptr ? p.saved_lse[t] * loss::kLog2E : 0.0F;
                if (p.rows.target[i] == loss::kBadTarget) { scale = __uint_as_float(0x7FFFFFFFU); }
            }
            p.rows.scale[i] = scale;
            p.rows.lse2[i]  = lse2;
            if (p.rows.own_scale != nullptr) {
                // The same with the row's own |scale| for the largest one.
                const float own        = i < count ? p.grad_loss[p.rows.token[i]] : 0.0F;
                const std::int32_t by  = p.scale_bits - (own != 0.0F && fabsf(own) <= FLT_MAX ? max(-100, ilogbf(own)) : 0);
                p.rows.own_scale[i]    = i < count && p.rows.target[i] == loss::kBadTarget ? scale : ldexpf(own, by);
                p.rows.own_unit[i]     = ldexpf(1.0F, -by);
            }
        }
    }
    for (std::uint32_t i = count + threadIdx.x; i < padded; i += kListThreads) {
        p.rows.token[i]  = -1;
        p.rows.target[i] = -1;
    }
    if (threadIdx.x == 0) { *p.rows.count = count; }
}

// Row i of the copy = hidden state of the i-th live token; zeros behind the last one. Words of `W` where both sides are aligned for it.
template<typename W>
__global__ void __launch_bounds__(kGatherThreads) gatherHidden(const LiveRows rows, std::uint32_t zero_to, const W* hidden, std::int64_t stride, W* copy,
                                                               std::uint64_t pitch, std::uint32_t words) {
    gridDependencyWait();
    gridDependencyLaunchDependents();
    const std::uint32_t live   = *rows.count;
    const std::uint32_t padded = max(zero_to, (max(live, 1U) + loss::kTileRows - 1) / loss::kTileRows * loss::kTileRows);
    const std::uint32_t row    = blockIdx.x;
    if (row >= padded) { return; }
    W* const to = copy + row * pitch;
    if (row < live) {
        const W* const from = hidden + static_cast<std::int64_t>(rows.token[row]) * stride;
#pragma unroll 4
        for (std::uint32_t i = threadIdx.x; i < words; i += kGatherThreads) { to[i] = from[i]; }
    } else {
        for (std::uint32_t i = threadIdx.x; i < words; i += kGatherThreads) { to[i] = W{}; }
    }
}

// A weight that TMA cannot describe, copied with rows at multiples of 16 bytes, eight 16-bit elements (or halves of FP32 ones) a thread: out of the two packs of 16 bytes that they lie across
// where both are between the weight's first and last element, else one by one. (What gets behind a row's last element is never fetched.) 13632 x 2311: 39 us less than
// element by element, 60001 x 3967 286 less.
__global__ void __launch_bounds__(kGatherThreads) copyRows16(const std::uint16_t* matrix, std::int64_t stride, std::uint32_t rows, std::uint16_t* to, std::uint64_t pitch,
                                                             std::uint32_t depth) {
    gridDependencyWait();
    gridDependencyLaunchDependents();
    const std::uintptr_t begin = reinterpret_cast<std::uintptr_t>(matrix), end = reinterpret_cast<std::uintptr_t>(matrix + static_cast<std::int64_t>(rows - 1) * stride + depth);
    const std::uint32_t packs  = (depth + 7) / 8;
    const std::uint64_t all    = static_cast<std::uint64_t>(rows) * packs, step = static_cast<std::uint64_t>(gridDim.x) * kGatherThreads;
    for (std::uint64_t i = static_cast<std::uint64_t>(blockIdx.x) * kGatherThreads + threadIdx.x; i < all; i += step) {
        const std::uint32_t row = static_cast<std::uint32_t>(i / packs), first = static_cast<std::uint32_t>(i - static_cast<std::uint64_t>(row) * packs) * 8;
        const std::uint16_t* const from = matrix + static_cast<std::int64_t>(row) * stride + first;
        const std::uintptr_t at         = reinterpret_cast<std::uintptr_t>(from), low = at & ~std::uintptr_t{15};
        std::uint32_t out[4];
        if (low >= begin && low + 32 <= end) {
            const uint4 a = *reinterpret_cast<const uint4*>(low), b = *reinterpret_cast<const uint4*>(low + 16);
            std::uint32_t words[8]    = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            const std::uint32_t shift = static_cast<std::uint32_t>(at - low);
#pragma unroll
            for (int by = 2; by > 0; by /= 2) {
                if ((shift / 4 & by) != 0) {
#pragma unroll
                    for (int j = 0; j + by < 8; ++j) { words[j] = words[j + by]; }
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) { out[j] = __funnelshift_r(words[j], words[j + 1], shift % 4 * 8); }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const std::uint32_t left = first + 2 * j < depth ? from[2 * j] : 0, right = first + 2 * j + 1 < depth ? from[2 * j + 1] : 0;
                out[j]                   = left | right << 16;
            }
        }
        *reinterpret_cast<uint4*>(to + row * pitch + first) = make_uint4(out[0], out[1], out[2], out[3]);
    }
}

// An FP32 matrix's rows as three BF16 matrices, `plane` elements apart, eight elements a thread. With `gathered`, the rows are those of the live tokens, and
// zeros behind the last one. (16384 x 512: 14.5 us, 22.3 with two elements a thread and a CTA a row.) kWide: the rows begin at multiples of 16 bytes. (The planes' rows do, and have room for whole packs.)
template<bool kWide>
__global__ void __launch_bounds__(kGatherThreads) splitRows(const LiveRows rows, bool gathered, std::uint32_t count, const float* matrix, std::int64_t stride, std::uint16_t* to,
                                                            std::uint64_t pitch, std::uint64_t plane, std::uint32_t depth) {
    gridDependencyWait();
    gridDependencyLaunchDependents();
    const std::uint32_t live   = gathered ? *rows.count : count;
    const std::uint32_t padded = gathered ? (max(live, 1U) + loss::kTileRows - 1) / loss::kTileRows * loss::kTileRows : count;
    const std::uint32_t packs  = (depth + 7) / 8;
    const std::uint64_t all    = static_cast<std::uint64_t>(padded) * packs, step = static_cast<std::uint64_t>(gridDim.x) * kGatherThreads;
    for (std::uint64_t i = static_cast<std::uint64_t>(blockIdx.x) * kGatherThreads + threadIdx.x; i < all; i += step) {
        const std::uint32_t row = static_cast<std::uint32_t>(i / packs), first = static_cast<std::uint32_t>(i - static_cast<std::uint64_t>(row) * packs) * 8;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) { x[j] = 0.0F; }
        if (row < live) {
            const float* const from = matrix + static_cast<std::int64_t>(gathered ? rows.token[row] : static_cast<std::int32_t>(row)) * stride + first;
            if (kWide && first + 8 <= depth) {
                const float4 low = *reinterpret_cast<const float4*>(from), high = *reinterpret_cast<const float4*>(from + 4);
                x[0] = low.x, x[1] = low.y, x[2] = low.z, x[3] = low.w, x[4] = high.x, x[5] = high.y, x[6] = high.z, x[7] = high.w;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) { x[j] = first + j < depth ? from[j] : 0.0F; }
            }
        }
        alignas(16) __nv_bfloat16 parts[3][8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float three[3];
            training::splitPlanes(x[j], three);
#pragma unroll
            for (int p = 0; p < 3; ++p) { parts[p][j] = __float2bfloat16_rn(three[p]); }
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) { *reinterpret_cast<uint4*>(to + p * plane + row * pitch + first) = *reinterpret_cast<const uint4*>(parts[p]); }
    }
}

// Two partial results of a row: sums of 2^(x - base), with the bases.
__device__ __forceinline__ float2 joinPartials(float2 a, float2 b) {
    const float base = fmaxf(a.x, b.x);
    // (A base of -inf belongs to a sum of nothing, or of NaN: taken as it is.)
    const float left  = a.x == -INFINITY ? a.y : a.y * exp2f(a.x - base);
    const float right = b.x == -INFINITY ? b.y : b.y * exp2f(b.x - base);
    return make_float2(base, left + right);
}

struct JoinParams {
    LiveRows rows;
    const float2* partials;  // [piece][capacity]
    std::uint32_t pieces, capacity;
    float* row_loss;         // [capacity]
    float* loss;             // [tokens], or NULL
    float* lse;              // [tokens], or NULL
    bool keep;               // rows.lse2 is wanted
};

__global__ void __launch_bounds__(kJoinWarps * 32) joinStatistics(const JoinParams p) {
    __shared__ float2 shared[kJoinWarps][kJoinRows];
    gridDependencyWait();
    gridDependencyLaunchDependents();
    const std::uint32_t live = *p.rows.count;
    const std::uint32_t row  = blockIdx.x * kJoinRows + (threadIdx.x & 31);
    if (blockIdx.x * kJoinRows >= live) { return; }
    const int warp = threadIdx.x >> 5;
    float2 sum     = make_float2(-INFINITY, 0.0F);
    // Eight pieces at a time: one reference for them and what came before. (Rows up to the next multiple of kTileRows have statistics too.)
    for (std::uint32_t piece = warp; piece < p.pieces; piece += 8 * kJoinWarps) {
        float2 part[8];
        float base = sum.x;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const std::uint32_t at = piece + i * kJoinWarps;
            part[i] = at < p.pieces ? __ldcg(p.partials + static_cast<std::uint64_t>(at) * p.capacity + row) : make_float2(-INFINITY, 0.0F);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) { base = fmaxf(base, part[i].x); }
        float total = sum.x == -INFINITY ? sum.y : sum.y * exp2f(sum.x - base);
#pragma unroll
        for (int i = 0; i < 8; ++i) { total += part[i].x == -INFINITY ? part[i].y : part[i].y * exp2f(part[i].x - base); }
        sum = make_float2(base, total);
    }
    shared[warp][threadIdx.x & 31] = sum;
    __syncthreads();
    if (warp == 0 && row < live) {
        for (int w = 1; w < kJoinWarps; ++w) { sum = joinPartials(sum, shared[w][threadIdx.x]); }
        const float lse2         = sum.x + log2f(sum.y);
        const float lse          = loss::kLn2 * lse2;
        const bool bad           = p.rows.target[row] == loss::kBadTarget;
        const float value        = bad ? __uint_as_float(0x7FFFFFFFU) : lse - p.rows.picked[row];
        const std::int32_t token = p.rows.token[row];
        p.row_loss[row]          = value;
        if (p.lse != nullptr) { p.lse[token] = lse; }
        if (p.keep) { p.rows.lse2[row] = lse2; }
        if (p.loss != nullptr) { p.loss[token] = value; }
    }
}

// One CTA: the live rows' losses added up in 64 bits.
__global__ void __launch_bounds__(kListThreads) sumLosses(const LiveRows rows, const float* row_loss, bool mean, float* loss) {
    __shared__ double shared[kListThreads / 32];
    gridDependencyWait();
    gridDependencyLaunchDependents();
    const std::uint32_t live = *rows.count;
    double sum               = 0.0;
#pragma unroll 4
    for (std::uint32_t i = threadIdx.x; i < live; i += kListThreads) { sum += static_cast<double>(row_loss[i]); }
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2) { sum += __shfl_xor_sync(0xFFFFFFFFU, sum, offset); }
    if ((threadIdx.x & 31) == 0) { shared[threadIdx.x >> 5] = sum; }
    __syncthreads();
    if (threadIdx.x < 32) {
        sum = shared[threadIdx.x];
#pragma unroll
        for (int offset = 16; offset > 0; offset /= 2) { sum += __shfl_xor_sync(0xFFFFFFFFU, sum, offset); }
        if (threadIdx.x == 0) { *loss = static_cast<float>(mean ? sum / static_cast<double>(max(live, 1U)) : sum); }
    }
}

struct RowParams {
    LiveRows rows;
    float* logits;           // of a piece: [rows][pitch]
    std::uint64_t pitch;
    std::uint32_t first, columns;
    float2* partials;        // this piece's: [capacity]
};

// FP32: the statistics of a row's piece, one CTA for each row.
__global__ void __launch_bounds__(kRowThreads) rowStatistics(const RowParams p) {
    __shared__ float2 shared[kRowThreads / 32];
    gridDependencyWait();
    gridDependencyLaunchDependents();
    const std::uint32_t row = blockIdx.x;
    if (row >= *p.rows.count) { return; }
    const float* const z = p.logits + row * p.pitch;  // 16-byte aligned, as the pitch is a multiple of four
    float largest = -INFINITY, base = 0.0F, sum = 0.0F;
    const auto add = [&](const float (&x)[4]) {
        const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        if (top > largest) {  // a new reference for the sum
            const float next = top * loss::kLog2E;
            sum              = largest == -INFINITY ? sum : sum * exp2f(base - next);
            largest          = top;
            base             = next;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) { sum += exp2Fast(fmaf(x[i], loss::kLog2E, -base)); }
    };
#pragma unroll 2
    for (std::uint32_t at = 4 * threadIdx.x; at < p.columns; at += 4 * kRowThreads) {
        float x[4];
        if (at + 4 <= p.columns) {
            const float4 four = *reinterpret_cast<const float4*>(z + at);
            x[0] = four.x, x[1] = four.y, x[2] = four.z, x[3] = four.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) { x[i] = at + i < p.columns ? z[at + i] : -INFINITY; }
        }
        add(x);
    }
    float2 mine = make_float2(largest == -INFINITY ? -INFINITY : base, sum);
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2) {
        mine = joinPartials(mine, make_float2(__shfl_xor_sync(0xFFFFFFFFU, mine.x, offset), __shfl_xor_sync(0xFFFFFFFFU, mine.y, offset)));
    }
    if ((threadIdx.x & 31) == 0) { shared[threadIdx.x >> 5] = mine; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kRowThreads / 32; ++w) { mine = joinPartials(mine, shared[w]); }
        p.partials[row]       = mine;
        const std::int32_t at = p.rows.target[row] - static_cast<std::int32_t>(p.first);
        if (at >= 0 && at < static_cast<std::int32_t>(p.columns)) { p.rows.picked[row] = z[at]; }
    }
}

// FP32: Z of a piece becomes dZ, in place; zeros in the rows behind the live ones.
__global__ void __launch_bounds__(kRowThreads) rowSlopes(const RowParams p) {
    gridDependencyWait();
    gridDependencyLaunchDependents();
    const std::uint32_t row = blockIdx.x;
    float* const z          = p.logits + row * p.pitch;
    const bool on           = row < *p.rows.count;
    const float scale       = on ? p.rows.scale[row] : 0.0F;
    const float lse2        = on ? p.rows.lse2[row] : 0.0F;
    const std::uint32_t hit = on ? static_cast<std::uint32_t>(p.rows.target[row]) - p.first : 0xFFFFFFFFU;  // wraps where there is none
    const auto slope        = [&](float x, std::uint32_t column) {
        return on ? scale * (exp2Fast(fmaf(x, loss::kLog2E, -lse2)) - (column == hit ? 1.0F : 0.0F)) : 0.0F;
    };
#pragma unroll 2
    for (std::uint32_t at = 4 * threadIdx.x; at < p.columns; at += 4 * kRowThreads) {
        // (The pitch has room for a whole quad behind the last column.)
        const float4 x                        = *reinterpret_cast<const float4*>(z + at);
        *reinterpret_cast<float4*>(z + at) = make_float4(slope(x.x, at), slope(x.y, at + 1), slope(x.z, at + 2), slope(x.w, at + 3));
    }
}

struct KeptParams {
    LiveRows rows;
    const float2* partials;  // [piece][capacity]
    std::uint32_t pieces, width, capacity;
    std::uint64_t pitch, plane;
};

// Of a piece's row: what its exponentials are multiplied by to be slopes.
__device__ __forceinline__ float keptFactor(const KeptParams& p, std::uint32_t piece, std::uint32_t row) {
    const float base = p.partials[static_cast<std::uint64_t>(piece) * p.capacity + row].x;
    // (A piece of -inf alone kept zeros; against a sum of nothing, or of NaN, NaN comes out.)
    const float lse2 = p.rows.lse2[row];
    return p.rows.scale[row] * (base == -INFINITY && lse2 > -INFINITY ? 0.0F : exp2f(base - lse2));
}

// (Of 4096 x 32768 in 16 bits 94 us with a pack at a time, 80 with two asked for before the first is written, the rate of a copy.)
// What the product kept becomes dZ, in place: 2^(logit - piece's largest) 2^(that - lse), less the target's one; zeros in the neutral rows. A thread
// takes eight columns of a row at a time, neighbouring threads neighbouring ones.
// kPlanes: from FP32 to the three BF16 matrices at `planes`, T being float; otherwise from FP16 to T.
template<typename T> __global__ void __launch_bounds__(256) keptSlopes(const KeptParams p, void* kept, std::uint16_t* planes) {
    constexpr bool kPlanes = std::is_same<T, float>::value;
    __shared__ float factors[kKeptPieces][kKeptRows];
    gridDependencyWait();
    gridDependencyLaunchDependents();
    const std::uint32_t live   = *p.rows.count;
    const std::uint32_t across = (p.pieces + kKeptPieces - 1) / kKeptPieces;  // CTAs side by side
    const std::uint32_t row0   = blockIdx.x / across * kKeptRows, piece0 = blockIdx.x % across * kKeptPieces;
    const std::uint32_t padded = (max(live, 1U) + loss::kTileRows - 1) / loss::kTileRows * loss::kTileRows;
    if (row0 >= padded) { return; }
    const std::uint32_t pieces = min(p.pieces - piece0, static_cast<std::uint32_t>(kKeptPieces));
    if (threadIdx.x < kKeptPieces * kKeptRows) {
        const std::uint32_t piece = threadIdx.x / kKeptRows, row = row0 + threadIdx.x % kKeptRows;
        if (piece < pieces && row < live) { factors[piece][threadIdx.x % kKeptRows] = keptFactor(p, piece0 + piece, row) * (kPlanes ? 1.0F : 1.0F / loss::kKeptScale); }
    }
    __syncthreads();
    const std::uint32_t each  = p.width / 8;  // packs of a piece's row
    const std::uint32_t packs = pieces * each, all = packs * kKeptRows;
    using From = typename std::conditional<kPlanes, float, __half>::type;
    struct alignas(16) Pack {
        From at[8];
    };
    // A batch is asked for before the first of it is written.
    for (std::uint32_t first = threadIdx.x; first < all; first += kKeptBatch * 256) {
        Pack batch[kKeptBatch];
        const auto place = [&](std::uint32_t i) { return (row0 + i / packs) * p.pitch + piece0 * p.width + i % packs * 8; };
#pragma unroll
        for (int b = 0; b < kKeptBatch; ++b) {
            const std::uint32_t i = first + b * 256;
            if (i < all) { batch[b] = *reinterpret_cast<const Pack*>(static_cast<const From*>(kept) + place(i)); }
        }
#pragma unroll
        for (int b = 0; b < kKeptBatch; ++b) {
            const std::uint32_t i = first + b * 256;
            if (i >= all) { break; }
            const std::uint32_t in_row = i / packs, pack = i - in_row * packs, row = row0 + in_row;
            const std::uint64_t at     = place(i);
            const bool on              = row < live;
            const float factor         = on ? factors[pack / each][in_row] : 0.0F;
            const float scale          = on ? p.rows.scale[row] : 0.0F;
            const std::int32_t hit     = on ? p.rows.target[row] - static_cast<std::int32_t>(piece0 * p.width + pack * 8) : -1;
            if constexpr (kPlanes) {
                alignas(16) __nv_bfloat16 to[3][8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float parts[3];
                    training::splitPlanes(on ? factor * batch[b].at[j] - (j == hit ? scale : 0.0F) : 0.0F, parts);
#pragma unroll
                    for (int plane = 0; plane < 3; ++plane) { to[plane][j] = __float2bfloat16_rn(parts[plane]); }
                }
#pragma unroll
                for (int plane = 0; plane < 3; ++plane) { *reinterpret_cast<uint4*>(planes + plane * p.plane + at) = *reinterpret_cast<const uint4*>(to[plane]); }
            } else {
                alignas(16) T to[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) { to[j] = Element<T>::narrow(on ? factor * __half2float(batch[b].at[j]) - (j == hit ? scale : 0.0F) : 0.0F); }
                *reinterpret_cast<uint4*>(static_cast<__half*>(kept) + at) = *reinterpret_cast<const uint4*>(to);
            }
        }
    }
}

// grad_hidden[t] = unit * upstream * (the sums' parts added up), 0 for a token that takes no part. Few tokens have many parts, and several CTAs each.
template<typename T>
__global__ void __launch_bounds__(kGatherThreads) spreadHidden(const LiveRows rows, const std::int32_t* slot, const float* sums, std::uint64_t part, std::uint64_t pitch,
                                                               std::uint32_t capacity, std::uint32_t splits, std::uint32_t depth, const float* upstream, T* out,
                                                               std::int64_t stride) {
    gridDependencyWait();
    gridDependencyLaunchDependents();
    // (Never beyond, whatever stands there. Without slots every row is its own: the weight's gradient.)
    const std::int32_t row = slot != nullptr ? min(slot[blockIdx.x], static_cast<std::int32_t>(capacity) - 1) : static_cast<std::int32_t>(blockIdx.x);
    const float unit       = (slot != nullptr && row >= 0 && rows.own_unit != nullptr ? rows.own_unit[row] : *rows.unit) * (upstream != nullptr ? *upstream : 1.0F);
    T* const to            = out + static_cast<std::int64_t>(blockIdx.x) * stride;
    const float* const from = sums + static_cast<std::uint64_t>(max(row, 0)) * pitch;
#pragma unroll 2
    for (std::uint32_t i = blockIdx.y * kGatherThreads + threadIdx.x; i < depth; i += gridDim.y * kGatherThreads) {
        float sum = 0.0F;
        if (row >= 0) {
#pragma unroll 8
            for (std::uint32_t s = 0; s < splits; ++s) { sum += from[s * part + i]; }
        }
        to[i] = Element<T>::narrow(unit * sum);
    }
}

// ---------------------------------------------------------------- host: layout of the workspace

// Offsets in two memories: one that the step call keeps from the loss to the gradients, and one of the call's own. What lies where in the kept one goes by sizes alone, so
// that the weight may be at another address when the gradients are made (saved-tensor hooks of torch hand back a copy): a copy of the weight for TMA, which depends on
// its address, is the last thing there, and the memory's size says whether there is one.
struct Layout {
    bool library;                 // FP32 through the library's products
    bool planes;                  // ... or as three BF16 matrices
    std::uint64_t capacity;       // rows, a multiple of kTileRows
    std::uint64_t copy_pitch;     // of the hidden states' copy, elements
    std::uint64_t weight_pitch;   // of the weight's copy or planes, 0: none
    bool weight_kept;             // ... which are in the kept memory
    bool weight_made;             // ... since the loss: the gradients need not make them
    std::uint64_t columns;        // of a piece
    std::uint64_t piece_pitch;    // of Z or dZ, elements
    std::uint64_t pieces;         // partial statistics of a row
    std::uint32_t splits;         // of the sums for dH
    std::uint32_t weight_splits;  // ... for dW, 1: it needs none
    std::uint32_t weight_rows;    // rows of a part of those
    std::uint64_t sums_pitch;
    std::uint64_t count, unit, slot, hidden, piece;  // kept
    std::uint64_t weight;
    std::uint64_t token, target, scale, lse2, picked, row_loss, partials, exponentials, sums, weight_sums, product, product_bytes;
    std::uint64_t own_scale, own_unit, own_piece;  // where rows have scales of their own
    std::uint64_t kept_bytes, bytes;
};

std::uint64_t roundUp(std::uint64_t x, std::uint64_t unit) { return (x + unit - 1) / unit * unit; }

bool isFp32(const FtcudaLinearCrossEntropy& q) { return q.element == FTCUDA_ELEMENT_FP32; }

// Whether TMA can fetch the weight as it is.
bool weightFits(const FtcudaLinearCrossEntropy& q) {
    return training::aligned(q.weight, 16) && (q.vocabulary == 1 || q.weight_row_stride % (16 / static_cast<std::int64_t>(training::elementBytes(q.element))) == 0);
}

std::uint64_t weightStride(const FtcudaLinearCrossEntropy& q) {
    return q.vocabulary == 1 ? roundUp(q.depth, 8) : static_cast<std::uint64_t>(q.weight_row_stride);
}

// One FP32 product by the first family that takes it, in its prepared form where that is faster. `slopes`: A is dZ. What a slope is off by already,
// as its logit is a rounded sum, is over 2^-24 of it; next to the largest of 768 slopes that share a scale, one of under
// 2^-26 of that may be rounded at 2^-50 of it (the other operand's elements have to be within 2^26 of one another all the same). Without
// that, the small probabilities of every vocabulary would send these products to the form that is half as fast.
struct Product {
    FtcudaGemmLaunch launch;
    std::uint64_t bytes;
};
int configureProduct(const FtcudaGemmDesc& desc, bool slopes, int sms, std::uint64_t bytes_left, Product& product, char* message, std::size_t capacity) {
    const GemmCandidates candidates = gemmCandidates(desc.m, desc.n, desc.k, desc.b_row_stride == 1 && desc.n > 1, static_cast<std::uint64_t>(sms));
    for (int i = 0; i < candidates.count; ++i) {
        const int kernel = candidates.kernels[i];
        if (ftcuda_gemm_supports(kernel, &desc, nullptr, 0) != 0) { continue; }
        if (const int status = ftcuda_gemm_configure(kernel, &desc, &product.launch, message, capacity)) { return status; }
        product.bytes = ftcuda_gemm_workspace_bytes(&product.launch);
        if (product.bytes > bytes_left) { continue; }
        if ((kernel == FTCUDA_GEMM_TF32X3 || kernel == FTCUDA_GEMM_TF32X3_SPLITK) && preparedFormPays(desc.m, desc.n, desc.k)) {
            Product prepared;
            if (ftcuda_gemm_prepare(&product.launch, &desc, &prepared.launch, nullptr, 0) == 0) {
                prepared.bytes = ftcuda_gemm_workspace_bytes(&prepared.launch);
                reinterpret_cast<LaunchState*>(&prepared.launch)->prepared.absolute_a = slopes ? 1 : 0;
                if (prepared.bytes <= bytes_left) { product = prepared; }
            }
        }
        return 0;
    }
    return fail(message, capacity, 1, "no FP32 product takes the problem");
}

// The two memories that a call has.
struct Memory {
    unsigned char* kept;
    unsigned char* own;
    unsigned char* weight(const Layout& l) const { return (l.weight_kept ? kept : own) + l.weight; }
};

// The three FP32 products of a piece of `columns` columns from `first` on.
FtcudaGemmDesc describeLogits(const FtcudaLinearCrossEntropy& q, const Layout& l, const Memory& memory, std::uint64_t first, std::uint64_t columns) {
    FtcudaGemmDesc d{};
    d.a            = reinterpret_cast<const float*>(memory.kept + l.hidden);
    d.b            = l.weight_pitch != 0 ? reinterpret_cast<const float*>(memory.weight(l)) + first * l.weight_pitch
                                         : static_cast<const float*>(q.weight) + static_cast<std::int64_t>(first) * q.weight_row_stride;
    d.d            = reinterpret_cast<float*>(memory.kept + l.piece);
    d.alpha        = 1.0F;
    d.m            = q.tokens;
    d.n            = columns;
    d.k            = q.depth;
    d.a_row_stride = static_cast<std::int64_t>(l.copy_pitch);
    d.a_col_stride = 1;
    d.b_row_stride = 1;
    d.b_col_stride = l.weight_pitch != 0 ? static_cast<std::int64_t>(l.weight_pitch) : q.vocabulary == 1 ? static_cast<std::int64_t>(q.depth) : q.weight_row_stride;
    d.d_row_stride = static_cast<std::int64_t>(l.piece_pitch);
    d.d_col_stride = 1;
    d.device       = q.device;
    return d;
}
FtcudaGemmDesc describeHidden(const FtcudaLinearCrossEntropy& q, const Layout& l, const Memory& memory, std::uint64_t first, std::uint64_t columns) {
    FtcudaGemmDesc d = describeLogits(q, l, memory, first, columns);
    d.a              = d.d;
    d.d              = reinterpret_cast<float*>(memory.own + l.sums);
    d.n              = q.depth;
    d.k              = columns;
    d.a_row_stride   = static_cast<std::int64_t>(l.piece_pitch);
    d.b_row_stride   = d.b_col_stride;
    d.b_col_stride   = 1;
    d.d_row_stride   = static_cast<std::int64_t>(l.sums_pitch);
    if (first != 0) {
        d.beta         = 1.0F;
        d.c            = d.d;
        d.c_row_stride = d.d_row_stride;
        d.c_col_stride = 1;
    }
    return d;
}
FtcudaGemmDesc describeWeight(const FtcudaLinearCrossEntropy& q, const Layout& l, const Memory& memory, std::uint64_t first, std::uint64_t columns, void* grad_weight,
                              std::int64_t stride) {
    FtcudaGemmDesc d = describeLogits(q, l, memory, first, columns);
    d.b              = d.a;
    d.a              = d.d;
    d.d              = static_cast<float*>(grad_weight) + static_cast<std::int64_t>(first) * stride;
    d.m              = columns;
    d.n              = q.depth;
    d.k              = q.tokens;
    d.a_row_stride   = 1;
    d.a_col_stride   = static_cast<std::int64_t>(l.piece_pitch);
    d.b_row_stride   = static_cast<std::int64_t>(l.copy_pitch);
    d.b_col_stride   = 1;
    d.d_row_stride   = stride;
    return d;
}

// What a call computes: the loss, the gradients from a loss that is known (and logits computed again), or one of the two halves of a step.
enum class Form { kLoss, kGradients, kStepLoss, kStepGradients };
constexpr bool isStep(Form form) { return form == Form::kStepLoss || form == Form::kStepGradients; }

// Whether FP32 operands are better off with the library's products. Measured (library / three BF16 matrices, microseconds):
//   large products that take the prepared form; a step of 2048 x 2048 x 32000 2501 / 3231, 4096 x 1024 x 16000 1476 / 1666, 700 x 2048 x 20000 743 / 837, 1200 x 1200 x 9000
//   379 / 407, but 1024 x 1024 x 4096 165 / 150, 768 x 768 x 30000 558 / 521, 512 x 2048 x 32000 963 / 971, 256 x 1024 x 32000 424 / 324, and 2048 x 512 x 8000 349 / 281;
//   few tokens, which read the weight once and would have it split for nothing else: a step of 64 x 4096 x 32000 790 / 916, 32 x 2048 x 128 41 / 77, 64 x 1024 x 32000 275 / 282,
//   8 x 512 x 16000 94 / 107, but 64 x 512 x 8000 77 / 73, 48 x 512 x 16000 118 / 109, 20 x 512 x 5000 73 / 63, 96 x 1024 x 32000 333 / 289;
//   the loss alone, more of both: 96 x 4096 x 32000 225 / 505, 128 x 1024 x 20000 67 / 117, 300 x 2048 x 50000 442 / 580, 512 x 4096 x 32000 641 / 785, but 256 x 1024 x 32000 151 / 146,
//   768 x 768 x 30000 193 / 179.
bool libraryPays(const FtcudaLinearCrossEntropy& q, Form form) {
    if (!isFp32(q)) { return false; }
    const bool large = q.depth >= 768 && q.tokens * q.depth >= 1400000 && preparedFormPays(q.tokens, q.vocabulary, q.depth);
    if (form == Form::kLoss) { return large || q.tokens <= 128 || q.depth >= 2048; }
    return large || q.tokens <= 8 || (q.tokens <= 64 && q.depth >= 1024);
}

// Whether the hidden states' gradient needs slopes of its own: with one scale for all rows, those whose upstream gradient is 2^-16 of the largest would keep four bits of a probability
// of 2^-17 in FP16, and nothing of one of 2^-22. (Both slopes come out of one product: 2000 x 2048 x 50257 1.23 -> 1.26 ms, 4096 x 1024 x 32000 0.84 -> 0.92.)
bool rowsHaveScales(const FtcudaLinearCrossEntropy& q, Form form) {
    return form == Form::kGradients && q.element == FTCUDA_ELEMENT_FP16 && q.reduction == FTCUDA_REDUCTION_NONE;
}

// What a logit takes of the workspace while it is there, in bytes: its slope, and in the step call its exponential as well where that cannot
// be in the same place.
std::uint64_t logitBytes(const FtcudaLinearCrossEntropy& q, Form form) {
    if (!isFp32(q)) { return rowsHaveScales(q, form) ? 4 : 2; }
    return libraryPays(q, form) ? 4 : isStep(form) ? 2 * loss::kPlanes + 4 : 2 * loss::kPlanes;
}

// What the step call holds of all logits at once, in bytes.
std::uint64_t stepBytes(const FtcudaLinearCrossEntropy& q) {
    return roundUp(std::max<std::uint64_t>(q.tokens, 1), loss::kTileRows) * roundUp(q.vocabulary, 256) * logitBytes(q, Form::kStepLoss);
}

// Hands out offsets of a memory.
struct Room {
    std::uint64_t at = 0;
    std::uint64_t take(std::uint64_t size) {
        const std::uint64_t here = at;
        at += roundUp(size, kAlign);
        return here;
    }
};

constexpr std::uint64_t kAny = ~std::uint64_t{0};

// `kept_bytes`: of the memory that a step's loss left for these gradients; kAny in the other calls.
int layOut(const FtcudaLinearCrossEntropy& q, Form form, std::uint64_t kept_bytes, int sms, Layout& l, char* message, std::size_t capacity) {
    const bool gradients      = form != Form::kLoss && form != Form::kStepLoss;
    const bool statistics     = form != Form::kGradients && form != Form::kStepGradients;
    l                         = Layout{};
    l.library                 = libraryPays(q, form);
    l.planes                  = isFp32(q) && !l.library;
    const std::uint64_t bytes = logitBytes(q, form), element = l.planes ? 2 * loss::kPlanes : training::elementBytes(q.element);
    l.capacity                = roundUp(std::max<std::uint64_t>(q.tokens, 1), loss::kTileRows);
    l.copy_pitch              = roundUp(q.depth, 8);
    const std::uint64_t fill  = roundUp(q.vocabulary, 256);
    l.columns                 = isStep(form) ? fill : std::min(fill, std::max(kLeastColumns, kPieceBytes / (l.capacity * bytes) / 256 * 256));
    l.columns                 = roundUp(ceilDiv(fill, ceilDiv(fill, l.columns)), 256);  // pieces of about one size
    l.piece_pitch             = l.columns;
    l.pieces                  = l.library ? ceilDiv(q.vocabulary, l.columns) : loss::statisticsPieces(static_cast<std::uint32_t>(q.vocabulary), static_cast<std::uint32_t>(l.capacity), sms);
    l.sums_pitch              = roundUp(q.depth, 8);
    l.weight_rows             = static_cast<std::uint32_t>(roundUp(std::min(l.columns, q.vocabulary), loss::kTileRows));
    const loss::GradientSplits splits = l.library || !gradients ? loss::GradientSplits{1, 1}
                                                  : loss::gradientSplits(static_cast<std::uint32_t>(std::max<std::uint64_t>(q.tokens, 1)), static_cast<std::uint32_t>(q.depth),
                                                                         static_cast<std::uint32_t>(std::min(l.columns, q.vocabulary)), l.planes, sms);
    l.splits                  = splits.hidden;
    l.weight_splits           = splits.weight;
    Room kept, own;
    l.count  = kept.take(4);
    l.unit   = kept.take(4);
    l.slot   = kept.take(4 * l.capacity);
    l.hidden = kept.take(element * l.capacity * l.copy_pitch);
    if (form != Form::kLoss || l.library) { l.piece = kept.take(element * l.capacity * l.piece_pitch); }
    // (The prepared products split the weight whatever its rows' alignment; the others would copy it for each product, element by element: a step of 8 x 3967 x 60001 FP32
    // 3166 us, 1309 with one copy; 1000 x 2311 x 20000, prepared, the loss 384, with a copy 411.)
    const bool split_anyway = l.library && preparedFormPays(q.tokens, q.vocabulary, q.depth);
    // What waits for the gradients is no more than the logits' limit with the weight's copy either: a larger one is made again. (256 x 4096 x 131072 FP32 4.74 ms with 3.2 GB of planes
    // waiting, 5.65 made again, 300 x 4096 x 90000 4.95 and 5.57; in a step of 600 x 512 x 16384, where they wait, another splitting would take 14 us of 269.)
    Room with_copy          = kept;
    const std::uint64_t at  = with_copy.take(element * q.vocabulary * l.copy_pitch);
    const bool may_keep     = isStep(form) && stepBytes(q) + element * q.vocabulary * l.copy_pitch <= kStepBytes, keeps = may_keep && kept_bytes == with_copy.at;
    if (l.planes || (keeps && !split_anyway) || (!split_anyway && !weightFits(q))) {
        l.weight_pitch = l.copy_pitch;
        l.weight_kept  = keeps || (may_keep && kept_bytes == kAny);
        l.weight_made  = form == Form::kStepGradients && l.weight_kept;
        l.weight       = l.weight_kept ? at : own.take(element * q.vocabulary * l.copy_pitch);
        if (l.weight_kept) { kept = with_copy; }
    }
    l.kept_bytes = kept.at;
    if (kept_bytes != kAny && kept_bytes != l.kept_bytes) {
        return fail(message, capacity, 1, "the kept memory has %llu bytes, which is not what the loss of this problem leaves", static_cast<unsigned long long>(kept_bytes));
    }
    if (form != Form::kStepGradients) {
        l.token  = own.take(4 * l.capacity);
        l.target = own.take(4 * l.capacity);
        l.scale  = own.take(4 * l.capacity);
        l.lse2   = own.take(4 * l.capacity);
    }
    if (statistics) {
        l.picked   = own.take(4 * l.capacity);
        l.row_loss = own.take(4 * l.capacity);
        l.partials = own.take(8 * l.capacity * l.pieces);
    }
    if (l.planes && isStep(form) && statistics) { l.exponentials = own.take(4 * l.capacity * l.piece_pitch); }
    if (gradients) {
        l.sums = own.take(4 * l.capacity * l.sums_pitch * l.splits);
        if (rowsHaveScales(q, form)) {
            l.own_scale = own.take(4 * l.capacity);
            l.own_unit  = own.take(4 * l.capacity);
            l.own_piece = own.take(element * l.capacity * l.piece_pitch);
        }
        if (l.weight_splits > 1) { l.weight_sums = own.take(4 * static_cast<std::uint64_t>(l.weight_rows) * l.sums_pitch * l.weight_splits); }
    }
    if (l.library && q.tokens != 0) {
        // The most that any product of any piece wants. (The addresses are not known yet, but how they are aligned is.)
        l.product            = own.at;
        auto* const stand_in = reinterpret_cast<unsigned char*>(std::uintptr_t{1} << 40);
        const Memory memory{stand_in, stand_in};
        for (std::uint64_t first = 0; first < q.vocabulary; first += l.columns) {
            const std::uint64_t columns = std::min(l.columns, q.vocabulary - first);
            if (first != 0 && columns == l.columns && first != l.columns) { continue; }  // like the piece before
            Product product;
            if (form != Form::kStepGradients) {
                if (configureProduct(describeLogits(q, l, memory, first, columns), false, sms, ~std::uint64_t{0}, product, message, capacity) != 0) { return 1; }
                l.product_bytes = std::max(l.product_bytes, product.bytes);
            }
            if (!gradients) { continue; }
            if (configureProduct(describeHidden(q, l, memory, first, columns), true, sms, ~std::uint64_t{0}, product, message, capacity) != 0) { return 1; }
            l.product_bytes = std::max(l.product_bytes, product.bytes);
            if (configureProduct(describeWeight(q, l, memory, first, columns, stand_in, static_cast<std::int64_t>(q.depth)), true, sms, ~std::uint64_t{0}, product, message, capacity) != 0) { return 1; }
            l.product_bytes = std::max(l.product_bytes, product.bytes);
        }
        own.take(l.product_bytes);
    }
    l.bytes = own.at;
    return 0;
}

const char* check(const FtcudaLinearCrossEntropy& q) {
    const std::uint64_t bytes = training::elementBytes(q.element);
    if (bytes == 0) { return "the operands must be FP32, FP16 or BF16"; }
    if (q.reduction < FTCUDA_REDUCTION_NONE || q.reduction > FTCUDA_REDUCTION_SUM) { return "unknown reduction"; }
    if (q.vocabulary == 0 || q.vocabulary >= (1ULL << 24)) { return "1 to 2^24 - 1 columns of the vocabulary"; }
    if (q.depth == 0 || q.depth >= (1ULL << 20)) { return "a depth of 1 to 2^20 - 1"; }
    if (q.tokens >= (1ULL << 24)) { return "at most 2^24 - 1 tokens"; }
    if (q.weight == nullptr || !training::aligned(q.weight, bytes)) { return "the weight has no address, or one that is not a multiple of its element's size"; }
    if (q.vocabulary > 1 && (q.weight_row_stride < static_cast<std::int64_t>(q.depth) || q.weight_row_stride >= (1LL << 31))) { return "the weight's rows overlap, or lie too far apart"; }
    if (q.tokens == 0) { return nullptr; }
    if (q.hidden == nullptr || !training::aligned(q.hidden, bytes)) { return "the hidden states have no address, or one that is not a multiple of their element's size"; }
    if (q.tokens > 1 && (q.hidden_row_stride < static_cast<std::int64_t>(q.depth) || q.hidden_row_stride >= (1LL << 31))) { return "the hidden states' rows overlap, or lie too far apart"; }
    if (q.target == nullptr || !training::aligned(q.target, 8)) { return "the targets have no address, or one that is not a multiple of eight"; }
    return nullptr;
}

// ---------------------------------------------------------------- host: the calls

class Call final {
  public:
    Call(const FtcudaLinearCrossEntropy& problem, char* message, std::size_t capacity) : q_(problem), message_(message), capacity_(capacity) {}

    // Everything that is the same in both directions; 0 or a failure that has its message. The halves of a step have their kept memory; the other calls' is the workspace's beginning.
    int begin(Form form, void* kept_memory, std::uint64_t kept_bytes, void* workspace, std::uint64_t workspace_bytes, void* stream) {
        if (!training::deviceIsCurrent(q_.device, message_, capacity_) || !deviceSmCount(q_.device, &sms_, message_, capacity_)) { return 1; }
        if (layOut(q_, form, form == Form::kStepGradients ? kept_bytes : kAny, sms_, l_, message_, capacity_) != 0) { return 1; }
        if (!isStep(form)) {
            if (workspace == nullptr || workspace_bytes < l_.kept_bytes + l_.bytes || !training::aligned(workspace, kAlign)) {
                return fail(message_, capacity_, 1, "workspace of %llu bytes needed, at a multiple of 256", static_cast<unsigned long long>(l_.kept_bytes + l_.bytes));
            }
            memory_ = Memory{static_cast<unsigned char*>(workspace), static_cast<unsigned char*>(workspace) + l_.kept_bytes};
        } else {
            if (kept_memory == nullptr || kept_bytes != l_.kept_bytes || !training::aligned(kept_memory, kAlign)) {
                return fail(message_, capacity_, 1, "kept memory of %llu bytes needed, no more and no less, at a multiple of 256", static_cast<unsigned long long>(l_.kept_bytes));
            }
            if (workspace == nullptr || workspace_bytes < l_.bytes || !training::aligned(workspace, kAlign)) {
                return fail(message_, capacity_, 1, "workspace of %llu bytes needed, at a multiple of 256", static_cast<unsigned long long>(l_.bytes));
            }
            memory_ = Memory{static_cast<unsigned char*>(kept_memory), static_cast<unsigned char*>(workspace)};
        }
        int* status              = nullptr;
        volatile int* host       = nullptr;
        if (!deviceStatusWord(q_.device, &status, &host, message_, capacity_)) { return 1; }
        if (const int code = takeDeviceStatus(host)) {
            return fail(message_, capacity_, 1, "an earlier kernel reported a timed-out wait (code %d)", code);
        }
        stream_      = static_cast<cudaStream_t>(stream);
        rows_.count  = kept<std::uint32_t>(l_.count);
        rows_.unit   = kept<float>(l_.unit);
        rows_.token  = own<std::int32_t>(l_.token);
        rows_.target = own<std::int32_t>(l_.target);
        rows_.scale  = own<float>(l_.scale);
        rows_.lse2   = own<float>(l_.lse2);
        rows_.picked = own<float>(l_.picked);
        own_scales_  = rowsHaveScales(q_, form);
        if (own_scales_) {
            rows_.own_scale = own<float>(l_.own_scale);
            rows_.own_unit  = own<float>(l_.own_unit);
        }
        products_    = loss::ProductCall{l_.planes || q_.element == FTCUDA_ELEMENT_BF16, l_.planes, static_cast<std::uint32_t>(l_.capacity), static_cast<std::uint32_t>(q_.depth), rows_,
                                      {memory_.kept + l_.hidden, l_.copy_pitch, l_.capacity * l_.copy_pitch}, status, sms_, stream_, message_, capacity_, false};
        if (message_ != nullptr && capacity_ != 0) { message_[0] = '\0'; }
        return 0;
    }

    cudaError_t forward(float* loss, float* lse) {
        ListParams list = listParams();
        list.loss       = q_.reduction == FTCUDA_REDUCTION_NONE ? loss : nullptr;
        list.lse        = lse;
        // (The first kernel of a call is an ordinary launch: it starts when what came before in the stream is done.)
        listTokens<false><<<1, kListThreads, 0, stream_>>>(list);
        cudaError_t error = started();
        if (error == cudaSuccess) { error = gather(); }
        float2* const partials = own<float2>(l_.partials);
        if (!l_.library) {
            if (error == cudaSuccess) { error = loss::launchStatistics(products_, weight(0), static_cast<std::uint32_t>(q_.vocabulary), partials); }
        } else {
            std::uint64_t piece = 0;
            for (std::uint64_t first = 0; first < q_.vocabulary && error == cudaSuccess; first += l_.columns, ++piece) {
                const std::uint64_t columns = std::min(l_.columns, q_.vocabulary - first);
                error                       = multiply(describeLogits(q_, l_, memory_, first, columns), false);
                if (error == cudaSuccess) {
                    error = training::launchOverlapped(rowStatistics, dim3(static_cast<unsigned>(q_.tokens)), dim3(kRowThreads), 0, stream_, rowParams(first, columns, partials + piece * l_.capacity));
                }
            }
        }
        return error == cudaSuccess ? join(loss, lse, false) : error;
    }

    // The loss and, for an upstream gradient of 1, the slopes, with the logits computed once.
    cudaError_t stepLoss(float* loss) {
        ListParams list = listParams();
        list.scale_bits = scaleBits();
        listTokens<true><<<1, kListThreads, 0, stream_>>>(list);
        cudaError_t error = started();
        if (error == cudaSuccess) { error = gather(); }
        float2* const partials        = own<float2>(l_.partials);
        const std::uint32_t columns   = static_cast<std::uint32_t>(q_.vocabulary);
        void* const exponentials      = l_.planes ? memory_.own + l_.exponentials : memory_.kept + l_.piece;
        if (error == cudaSuccess && !l_.library) { error = loss::launchKept(products_, weight(0), columns, partials, exponentials, l_.piece_pitch); }
        if (l_.library) {
            if (error == cudaSuccess) { error = multiply(describeLogits(q_, l_, memory_, 0, columns), false); }
            if (error == cudaSuccess) { error = training::launchOverlapped(rowStatistics, dim3(static_cast<unsigned>(q_.tokens)), dim3(kRowThreads), 0, stream_, rowParams(0, columns, partials)); }
        }
        if (error == cudaSuccess) { error = join(loss, nullptr, true); }
        if (error != cudaSuccess) { return error; }
        if (l_.library) {
            return training::launchOverlapped(rowSlopes, dim3(static_cast<unsigned>(q_.tokens)), dim3(kRowThreads), 0, stream_, rowParams(0, columns, nullptr));
        } else {
            const KeptParams params{rows_, partials, static_cast<std::uint32_t>(l_.pieces), loss::statisticsWidth(columns, static_cast<std::uint32_t>(l_.capacity), sms_), static_cast<std::uint32_t>(l_.capacity),
                                    l_.piece_pitch, slopesPlane()};
            const dim3 grid(static_cast<unsigned>(ceilDiv(l_.pieces, kKeptPieces) * (l_.capacity / kKeptRows)));  // (of x, which takes any number)
            const auto kernel = l_.planes ? keptSlopes<float> : q_.element == FTCUDA_ELEMENT_FP16 ? keptSlopes<__half> : keptSlopes<__nv_bfloat16>;
            return training::launchOverlapped(kernel, grid, dim3(256), 0, stream_, params, exponentials, kept<std::uint16_t>(l_.piece));
        }
    }

    // The gradients from the slopes that stepLoss left in the kept memory, for an upstream gradient of *upstream (NULL: 1).
    cudaError_t stepGradients(const float* upstream, void* grad_hidden, std::int64_t hidden_stride, void* grad_weight, std::int64_t weight_stride, std::int32_t grad_element) {
        const bool copies = l_.weight_pitch != 0 && !l_.weight_made;
        products_.starts  = !copies;
        cudaError_t error = copies ? copyWeight(true) : cudaSuccess;
        if (error == cudaSuccess) { error = multiplySlopes(0, q_.vocabulary, grad_hidden != nullptr, grad_weight, weight_stride, grad_element, upstream); }
        if (error == cudaSuccess && grad_hidden != nullptr) { error = spreadTyped(hiddenParts(hidden_stride, upstream), grad_hidden, grad_element); }
        if (error != cudaSuccess || !l_.library || grad_weight == nullptr || upstream == nullptr) { return error; }
        // (The library's products take a factor from the host alone.)
        FtcudaGradient all{};
        all.data = all.out = grad_weight;
        all.rows           = q_.vocabulary;
        all.cols           = q_.depth;
        all.row_stride = all.out_row_stride = weight_stride;
        all.element = all.out_element = grad_element;
        return ftcuda_gradient_scale(&all, 1, upstream, q_.device, stream_, message_, capacity_) == 0 ? cudaSuccess : cudaErrorUnknown;
    }

    cudaError_t backward(const float* lse, const float* grad_loss, void* grad_hidden, std::int64_t hidden_stride, void* grad_weight, std::int64_t weight_stride) {
        ListParams list = listParams();
        list.saved_lse  = lse;
        list.grad_loss  = grad_loss;
        list.scale_bits = scaleBits();
        listTokens<true><<<1, kListThreads, 0, stream_>>>(list);
        cudaError_t error = started();
        if (error == cudaSuccess) { error = gather(); }
        for (std::uint64_t first = 0; first < q_.vocabulary && error == cudaSuccess; first += l_.columns) {
            const std::uint64_t columns = std::min(l_.columns, q_.vocabulary - first);
            error                       = slopes(first, columns, grad_hidden != nullptr, grad_weight != nullptr);
            if (error == cudaSuccess) { error = multiplySlopes(first, columns, grad_hidden != nullptr, grad_weight, weight_stride, q_.element, nullptr); }
        }
        return error == cudaSuccess && grad_hidden != nullptr ? spreadTyped(hiddenParts(hidden_stride, nullptr), grad_hidden, q_.element) : error;
    }

  private:
    template<typename T> T* kept(std::uint64_t offset) const { return reinterpret_cast<T*>(memory_.kept + offset); }
    template<typename T> T* own(std::uint64_t offset) const { return reinterpret_cast<T*>(memory_.own + offset); }

    static cudaError_t started() {
        const cudaError_t error = cudaGetLastError();
        if (error == cudaSuccess) { countLaunches(1); }
        return error;
    }

    // Elements between the planes of the slopes.
    std::uint64_t slopesPlane() const { return l_.capacity * l_.piece_pitch; }

    // FP16's exponents do not hold small probabilities unless the largest slope is near 2^13.
    std::int32_t scaleBits() const { return isFp32(q_) ? INT32_MIN : q_.element == FTCUDA_ELEMENT_FP16 ? 13 : 0; }

    ListParams listParams() const {
        ListParams list{};
        list.target       = q_.target;
        list.ignore_index = q_.ignore_index;
        list.vocabulary   = static_cast<std::int64_t>(q_.vocabulary);
        list.tokens       = static_cast<std::uint32_t>(q_.tokens);
        list.reduction    = q_.reduction;
        list.rows         = rows_;
        list.slot         = kept<std::int32_t>(l_.slot);
        return list;
    }

    RowParams rowParams(std::uint64_t first, std::uint64_t columns, float2* partials) const {
        return RowParams{rows_, kept<float>(l_.piece), l_.piece_pitch, static_cast<std::uint32_t>(first), static_cast<std::uint32_t>(columns), partials};
    }

    // An operand as three BF16 matrices, `rows` rows of it at most. `starts`: the first kernel of a call.
    cudaError_t split(bool starts, bool gathered, std::uint64_t rows, const float* from, std::int64_t stride, unsigned char* to, std::uint64_t pitch) const {
        const std::uint64_t threads = rows * ceilDiv(q_.depth, 8), most = static_cast<std::uint64_t>(sms_) * kSplitCtasPerSm;
        const dim3 grid(static_cast<unsigned>(std::min(most, ceilDiv(threads, kGatherThreads))));
        const auto kernel = training::aligned(from, 16) && stride % 4 == 0 ? splitRows<true> : splitRows<false>;
        return training::launchKernel(!starts, kernel, grid, dim3(kGatherThreads), 0, stream_, rows_, gathered, static_cast<std::uint32_t>(rows), from, stride,
                                      reinterpret_cast<std::uint16_t*>(to), pitch, rows * pitch, static_cast<std::uint32_t>(q_.depth));
    }

    // The live hidden states, and the weight where TMA cannot fetch it as it is.
    cudaError_t gather() const {
        cudaError_t error = cudaSuccess;
        if (l_.planes) {
            error = split(false, true, l_.capacity, static_cast<const float*>(q_.hidden), q_.tokens <= 1 ? 0 : q_.hidden_row_stride, memory_.kept + l_.hidden, l_.copy_pitch);
        } else {
            const std::uint64_t bytes = training::elementBytes(q_.element);
            // The library's products go over all rows, the others over whole tiles of live ones.
            const std::uint32_t zero_to = l_.library ? static_cast<std::uint32_t>(q_.tokens) : 0;
            const auto run = [&](auto word) {
                using W                   = decltype(word);
                const std::uint64_t ratio = sizeof(W) / bytes;
                return training::launchOverlapped(gatherHidden<W>, dim3(static_cast<unsigned>(l_.capacity)), dim3(kGatherThreads), 0, stream_, rows_, zero_to,
                                                  static_cast<const W*>(q_.hidden), static_cast<std::int64_t>(q_.hidden_row_stride / static_cast<std::int64_t>(ratio)),
                                                  kept<W>(l_.hidden), l_.copy_pitch / ratio, static_cast<std::uint32_t>(q_.depth / ratio));
            };
            const std::uint64_t row = q_.depth * bytes;
            const bool wide         = row % 16 == 0 && training::aligned(q_.hidden, 16) && (q_.tokens <= 1 || static_cast<std::uint64_t>(q_.hidden_row_stride) * bytes % 16 == 0);
            error                   = wide ? run(uint4{}) : bytes == 4 ? run(std::uint32_t{}) : run(std::uint16_t{});
        }
        return error == cudaSuccess && l_.weight_pitch != 0 ? copyWeight(false) : error;
    }

    // The weight's planes, or its copy for TMA.
    cudaError_t copyWeight(bool starts) const {
        if (l_.planes) {
            return split(starts, false, q_.vocabulary, static_cast<const float*>(q_.weight), q_.vocabulary == 1 ? 0 : q_.weight_row_stride, memory_.weight(l_), l_.weight_pitch);
        }
        const std::uint64_t words = training::elementBytes(q_.element) / 2;
        const std::uint64_t ctas  = std::min(ceilDiv(q_.vocabulary * ceilDiv(words * q_.depth, 8), kGatherThreads), static_cast<std::uint64_t>(sms_) * kSplitCtasPerSm);
        return training::launchKernel(!starts, copyRows16, dim3(static_cast<unsigned>(ctas)), dim3(kGatherThreads), 0, stream_, static_cast<const std::uint16_t*>(q_.weight),
                                      q_.vocabulary == 1 ? std::int64_t{0} : static_cast<std::int64_t>(words) * q_.weight_row_stride, static_cast<std::uint32_t>(q_.vocabulary),
                                      reinterpret_cast<std::uint16_t*>(memory_.weight(l_)), words * l_.weight_pitch, static_cast<std::uint32_t>(words * q_.depth));
    }

    // The weight from row `first` on, as the 16-bit products fetch it.
    loss::Matrix16 weight(std::uint64_t first) const {
        const bool copied         = l_.weight_pitch != 0;
        const std::uint64_t pitch = copied ? l_.weight_pitch : weightStride(q_);
        const void* const from    = copied ? memory_.weight(l_) : q_.weight;
        return loss::Matrix16{static_cast<const unsigned char*>(from) + 2 * first * pitch, pitch, q_.vocabulary * pitch};
    }

    // One FP32 product.
    cudaError_t multiply(const FtcudaGemmDesc& desc, bool slopes) const {
        Product product;
        if (configureProduct(desc, slopes, sms_, l_.product_bytes, product, message_, capacity_) != 0 ||
            ftcuda_gemm_launch(&product.launch, memory_.own + l_.product, l_.product_bytes, stream_, message_, capacity_) != 0) {
            return cudaErrorUnknown;  // the message says which
        }
        return cudaSuccess;
    }

    // The statistics of all rows joined: the loss, and (keep) rows_.lse2.
    cudaError_t join(float* loss, float* lse, bool keep) const {
        JoinParams join{};
        join.rows     = rows_;
        join.partials = own<float2>(l_.partials);
        join.pieces   = static_cast<std::uint32_t>(l_.pieces);
        join.capacity = static_cast<std::uint32_t>(l_.capacity);
        join.row_loss = own<float>(l_.row_loss);
        join.loss     = q_.reduction == FTCUDA_REDUCTION_NONE ? loss : nullptr;
        join.lse      = lse;
        join.keep     = keep;
        const cudaError_t error = training::launchOverlapped(joinStatistics, dim3(static_cast<unsigned>(l_.capacity / kJoinRows)), dim3(kJoinWarps * 32), 0, stream_, join);
        if (error != cudaSuccess || q_.reduction == FTCUDA_REDUCTION_NONE) { return error; }
        return training::launchOverlapped(sumLosses, dim3(1), dim3(kListThreads), 0, stream_, rows_, static_cast<const float*>(own<float>(l_.row_loss)),
                                          q_.reduction == FTCUDA_REDUCTION_MEAN, loss);
    }

    // dZ of a piece of the vocabulary, to the workspace.
    cudaError_t slopes(std::uint64_t first, std::uint64_t columns, bool for_hidden, bool for_weight) const {
        const std::uint32_t first32 = static_cast<std::uint32_t>(first), columns32 = static_cast<std::uint32_t>(columns);
        if (!l_.library) {
            return loss::launchSlopes(products_, weight(first), first32, columns32, own_scales_ && !for_weight ? nullptr : memory_.kept + l_.piece,
                                      own_scales_ && for_hidden ? memory_.own + l_.own_piece : nullptr, l_.piece_pitch, slopesPlane());
        }
        const cudaError_t error = multiply(describeLogits(q_, l_, memory_, first, columns), false);
        if (error != cudaSuccess) { return error; }
        return training::launchOverlapped(rowSlopes, dim3(static_cast<unsigned>(q_.tokens)), dim3(kRowThreads), 0, stream_, rowParams(first, columns, nullptr));
    }

    // What dZ of a piece is multiplied with.
    cudaError_t multiplySlopes(std::uint64_t first, std::uint64_t columns, bool hidden, void* grad_weight, std::int64_t weight_stride, std::int32_t grad_element,
                               const float* upstream) const {
        if (!l_.library) {
            loss::Gradients gradients{};
            gradients.sums                  = hidden ? own<float>(l_.sums) : nullptr;
            gradients.sums_pitch            = l_.sums_pitch;
            gradients.own_slopes            = own_scales_ ? memory_.own + l_.own_piece : nullptr;
            gradients.splits                = l_.splits;
            gradients.accumulate            = first != 0;
            gradients.weight_gradient_fp32  = grad_element == FTCUDA_ELEMENT_FP32;
            gradients.weight_gradient_pitch = weight_stride;
            gradients.upstream              = upstream;
            if (l_.weight_splits > 1 && grad_weight != nullptr) {
                gradients.weight_sums   = own<float>(l_.weight_sums);
                gradients.weight_splits = l_.weight_splits;
                gradients.weight_rows   = l_.weight_rows;
            }
            if (grad_weight != nullptr) {
                gradients.weight_gradient =
                    static_cast<unsigned char*>(grad_weight) + static_cast<std::int64_t>(training::elementBytes(grad_element) * first) * weight_stride;
            }
            const cudaError_t error = loss::launchGradients(products_, weight(first), static_cast<std::uint32_t>(columns), loss::Matrix16{memory_.kept + l_.piece, l_.piece_pitch, slopesPlane()}, gradients);
            if (error != cudaSuccess || gradients.weight_sums == nullptr) { return error; }
            return spreadTyped(Spread{columns, nullptr, gradients.weight_sums, l_.weight_rows, l_.weight_splits, weight_stride, upstream}, gradients.weight_gradient, grad_element);
        }
        cudaError_t error = cudaSuccess;
        if (hidden) { error = multiply(describeHidden(q_, l_, memory_, first, columns), true); }
        if (error == cudaSuccess && grad_weight != nullptr) { error = multiply(describeWeight(q_, l_, memory_, first, columns, grad_weight, weight_stride), true); }
        return error;
    }

    // Parts of sums to be added up.
    struct Spread {
        std::uint64_t rows;
        const std::int32_t* slot;
        const float* sums;
        std::uint64_t capacity;
        std::uint32_t splits;
        std::int64_t stride;
        const float* upstream;
    };
    Spread hiddenParts(std::int64_t stride, const float* upstream) const {
        return Spread{q_.tokens, kept<std::int32_t>(l_.slot), own<float>(l_.sums), l_.capacity, l_.splits, stride, upstream};
    }

    cudaError_t spreadTyped(const Spread& parts, void* out, std::int32_t element) const {
        switch (element) {
            case FTCUDA_ELEMENT_FP32: return spread(parts, static_cast<float*>(out));
            case FTCUDA_ELEMENT_FP16: return spread(parts, static_cast<__half*>(out));
            default: return spread(parts, static_cast<__nv_bfloat16*>(out));
        }
    }

    template<typename T> cudaError_t spread(const Spread& parts, T* out) const {
        // (64 x 2048 in 16 parts: 14 us with a CTA for each token, 5 with eight; 4096 x 512 in one: 14, and 20 with two.)
        const std::uint64_t each = std::min(ceilDiv(q_.depth, kGatherThreads), std::max<std::uint64_t>(1, static_cast<std::uint64_t>(sms_) * 4 / parts.rows));
        return training::launchOverlapped(spreadHidden<T>, dim3(static_cast<unsigned>(parts.rows), static_cast<unsigned>(each)), dim3(kGatherThreads), 0, stream_, rows_, parts.slot,
                                          parts.sums, parts.capacity * l_.sums_pitch, l_.sums_pitch, static_cast<std::uint32_t>(parts.capacity), parts.splits,
                                          static_cast<std::uint32_t>(q_.depth), parts.upstream, out, parts.stride);
    }

    const FtcudaLinearCrossEntropy& q_;
    char* message_;
    std::size_t capacity_;
    int sms_ = 0;
    Layout l_{};
    Memory memory_{};
    cudaStream_t stream_ = nullptr;
    LiveRows rows_{};
    bool own_scales_ = false;
    loss::ProductCall products_{};
};

// What a call came to. A failure below may have left its own message.
int finish(cudaError_t error, char* message, std::size_t capacity) {
    if (error == cudaSuccess) { return 0; }
    if (message != nullptr && capacity != 0 && message[0] != '\0') { return 1; }
    return fail(message, capacity, 1, "%s", cudaGetErrorString(error));
}

bool wordAligned(const void* pointer) { return pointer != nullptr && training::aligned(pointer, 4); }

// nullptr, or why the step call does not take the problem.
const char* checkStep(const FtcudaLinearCrossEntropy& q) {
    if (q.reduction == FTCUDA_REDUCTION_NONE) { return "without reduction the upstream gradients differ from token to token"; }
    if (q.tokens == 0) { return "there are no tokens"; }
    if (stepBytes(q) > kStepBytes) { return "the exponentials of all logits take more than 2 GiB"; }
    return nullptr;
}

// Memory from an operand's first byte up to its last one.
struct Extent {
    std::uintptr_t begin, end;
};
Extent extentOf(const void* at, std::uint64_t rows, std::uint64_t cols, std::int64_t stride, std::uint64_t bytes) {
    const std::uintptr_t begin = reinterpret_cast<std::uintptr_t>(at);
    if (at == nullptr || rows == 0) { return {0, 0}; }
    return {begin, begin + ((rows - 1) * static_cast<std::uint64_t>(rows > 1 ? stride : 0) + cols) * bytes};
}
bool meet(const Extent& a, const Extent& b) { return a.begin < b.end && b.begin < a.end; }

// nullptr, or what is wrong with where the gradients go. The weight's stride comes out as one that rows can have.
const char* checkGradients(const FtcudaLinearCrossEntropy& q, std::uint64_t bytes, const void* grad_hidden, std::int64_t hidden_stride, const void* grad_weight,
                           std::int64_t& weight_stride) {
    const std::int64_t depth = static_cast<std::int64_t>(q.depth);
    if ((grad_hidden != nullptr && !training::aligned(grad_hidden, bytes)) || (grad_weight != nullptr && !training::aligned(grad_weight, bytes))) {
        return "a gradient's address is not a multiple of its element's size";
    }
    if (grad_hidden != nullptr && q.tokens > 1 && (hidden_stride < depth || hidden_stride >= (1LL << 31))) {
        return "the rows of the hidden states' gradient overlap, or lie too far apart";
    }
    if (grad_weight != nullptr && q.vocabulary > 1 && (weight_stride < depth || weight_stride >= (1LL << 31))) {
        return "the rows of the weight's gradient overlap, or lie too far apart";
    }
    if (q.vocabulary == 1) { weight_stride = depth; }
    const Extent hidden_out = extentOf(grad_hidden, q.tokens, q.depth, hidden_stride, bytes), weight_out = extentOf(grad_weight, q.vocabulary, q.depth, weight_stride, bytes);
    const Extent in[]       = {extentOf(q.hidden, q.tokens, q.depth, q.hidden_row_stride, training::elementBytes(q.element)),
                               extentOf(q.weight, q.vocabulary, q.depth, q.weight_row_stride, training::elementBytes(q.element)), extentOf(q.target, 1, q.tokens, 0, 8)};
    bool apart = !meet(hidden_out, weight_out);
    for (const Extent& operand : in) { apart = apart && !meet(hidden_out, operand) && !meet(weight_out, operand); }
    return apart ? nullptr : "a gradient lies across the other one or an operand";
}

const char* checkAddress(const void* loss, const char* reason) { return wordAligned(loss) ? nullptr : reason; }
constexpr const char* kNoLoss     = "the loss has no address, or one that is not a multiple of four";
constexpr const char* kNoUpstream = "the loss's gradient has no address, or one that is not a multiple of four";

// What a call needs: 0, or a failure with its message.
int layOutChecked(const FtcudaLinearCrossEntropy* problem, Form form, std::uint64_t kept_bytes, Layout& layout, char* message, std::size_t capacity) {
    if (problem == nullptr) { return fail(message, capacity, 1, "null problem"); }
    const char* reason = check(*problem);
    if (reason == nullptr && isStep(form)) { reason = checkStep(*problem); }
    if (reason != nullptr) { return fail(message, capacity, 1, "%s", reason); }
    int sms = 0;
    return deviceSmCount(problem->device, &sms, message, capacity) && layOut(*problem, form, kept_bytes, sms, layout, message, capacity) == 0 ? 0 : 1;
}

// Of a step with both memories in one workspace, the kept one first: how much that is, and how much both are.
int stepBytesInOne(const FtcudaLinearCrossEntropy* problem, std::uint64_t& kept_bytes, std::uint64_t& bytes, char* message, std::size_t capacity) {
    Layout first, second;
    if (layOutChecked(problem, Form::kStepLoss, kAny, first, message, capacity) != 0) { return 1; }
    if (layOutChecked(problem, Form::kStepGradients, first.kept_bytes, second, message, capacity) != 0) { return 1; }
    kept_bytes = first.kept_bytes;
    bytes      = first.kept_bytes + std::max(first.bytes, second.bytes);
    return 0;
}

// The halves of a step; what they are given is checked but for the memories.
int stepLoss(const FtcudaLinearCrossEntropy& problem, float* loss, void* kept, std::uint64_t kept_bytes, void* workspace, std::uint64_t workspace_bytes, void* stream, char* message,
             std::size_t capacity) {
    Call call(problem, message, capacity);
    if (const int status = call.begin(Form::kStepLoss, kept, kept_bytes, workspace, workspace_bytes, stream)) { return status; }
    return finish(call.stepLoss(loss), message, capacity);
}
int stepGradients(const FtcudaLinearCrossEntropy& problem, const float* grad_loss, std::int32_t grad_element, void* grad_hidden, std::int64_t hidden_stride, void* grad_weight,
                  std::int64_t weight_stride, void* kept, std::uint64_t kept_bytes, void* workspace, std::uint64_t workspace_bytes, void* stream, char* message,
                  std::size_t capacity) {
    if (grad_hidden == nullptr && grad_weight == nullptr) { return 0; }
    Call call(problem, message, capacity);
    if (const int status = call.begin(Form::kStepGradients, kept, kept_bytes, workspace, workspace_bytes, stream)) { return status; }
    return finish(call.stepGradients(grad_loss, grad_hidden, hidden_stride, grad_weight, weight_stride, grad_element), message, capacity);
}

// The kept part at the beginning of a workspace for both; 0, or a failure with its message. `exactly`: a size that another problem's would be is refused.
int splitWorkspace(const FtcudaLinearCrossEntropy& problem, void* workspace, std::uint64_t workspace_bytes, bool exactly, std::uint64_t& kept_bytes, char* message,
                   std::size_t capacity) {
    if (!training::deviceIsCurrent(problem.device, message, capacity)) { return 1; }
    std::uint64_t bytes = 0;
    if (stepBytesInOne(&problem, kept_bytes, bytes, message, capacity) != 0) { return 1; }
    if (workspace == nullptr || workspace_bytes < bytes || (exactly && workspace_bytes != bytes) || !training::aligned(workspace, kAlign)) {
        return fail(message, capacity, 1, "workspace of %llu bytes needed, %sat a multiple of 256", static_cast<unsigned long long>(bytes), exactly ? "no more and no less, " : "");
    }
    return 0;
}

}  // namespace
}  // namespace ftcuda

extern "C" int ftcuda_linear_cross_entropy_workspace_bytes(const FtcudaLinearCrossEntropy* problem, int backward, uint64_t* workspace_bytes, char* message,
                                                           size_t message_capacity) {
    using namespace ftcuda;
    if (workspace_bytes == nullptr) { return fail(message, message_capacity, 1, "null argument"); }
    Layout layout;
    if (layOutChecked(problem, backward != 0 ? Form::kGradients : Form::kLoss, kAny, layout, message, message_capacity) != 0) { return 1; }
    *workspace_bytes = layout.kept_bytes + layout.bytes;
    return 0;
}

extern "C" int ftcuda_linear_cross_entropy_step_workspace_bytes(const FtcudaLinearCrossEntropy* problem, uint64_t* workspace_bytes, char* message, size_t message_capacity) {
    using namespace ftcuda;
    if (workspace_bytes == nullptr) { return fail(message, message_capacity, 1, "null argument"); }
    std::uint64_t kept_bytes = 0;
    return stepBytesInOne(problem, kept_bytes, *workspace_bytes, message, message_capacity);
}

extern "C" int ftcuda_linear_cross_entropy_step_loss_bytes(const FtcudaLinearCrossEntropy* problem, uint64_t* kept_bytes, uint64_t* workspace_bytes, char* message,
                                                           size_t message_capacity) {
    using namespace ftcuda;
    if (kept_bytes == nullptr || workspace_bytes == nullptr) { return fail(message, message_capacity, 1, "null argument"); }
    Layout layout;
    if (layOutChecked(problem, Form::kStepLoss, kAny, layout, message, message_capacity) != 0) { return 1; }
    *kept_bytes      = layout.kept_bytes;
    *workspace_bytes = layout.bytes;
    return 0;
}

extern "C" int ftcuda_linear_cross_entropy_step_gradients_bytes(const FtcudaLinearCrossEntropy* problem, uint64_t kept_bytes, uint64_t* workspace_bytes, char* message,
                                                                size_t message_capacity) {
    using namespace ftcuda;
    if (workspace_bytes == nullptr) { return fail(message, message_capacity, 1, "null argument"); }
    Layout layout;
    if (layOutChecked(problem, Form::kStepGradients, kept_bytes, layout, message, message_capacity) != 0) { return 1; }
    *workspace_bytes = layout.bytes;
    return 0;
}

extern "C" int ftcuda_linear_cross_entropy_step(const FtcudaLinearCrossEntropy* problem, float* loss, int32_t grad_element, void* grad_hidden, int64_t grad_hidden_row_stride,
                                                void* grad_weight, int64_t grad_weight_row_stride, void* workspace, uint64_t workspace_bytes, void* stream,
                                                char* message, size_t message_capacity) {
    using namespace ftcuda;
    if (problem == nullptr) { return fail(message, message_capacity, 1, "null problem"); }
    const char* reason = check(*problem);
    if (reason == nullptr) { reason = checkStep(*problem); }
    if (reason == nullptr && grad_element != problem->element && grad_element != FTCUDA_ELEMENT_FP32) { reason = "the gradients are of the operands' type, or FP32"; }
    if (reason == nullptr) { reason = checkAddress(loss, kNoLoss); }
    if (reason == nullptr) { reason = checkGradients(*problem, training::elementBytes(grad_element), grad_hidden, grad_hidden_row_stride, grad_weight, grad_weight_row_stride); }
    if (reason != nullptr) { return fail(message, message_capacity, 1, "%s", reason); }
    std::uint64_t kept = 0;
    if (const int status = splitWorkspace(*problem, workspace, workspace_bytes, false, kept, message, message_capacity)) { return status; }
    void* const own = static_cast<unsigned char*>(workspace) + kept;
    if (const int status = stepLoss(*problem, loss, workspace, kept, own, workspace_bytes - kept, stream, message, message_capacity)) { return status; }
    return stepGradients(*problem, nullptr, grad_element, grad_hidden, grad_hidden_row_stride, grad_weight, grad_weight_row_stride, workspace, kept, own, workspace_bytes - kept, stream,
                         message, message_capacity);
}

extern "C" int ftcuda_linear_cross_entropy_step_loss(const FtcudaLinearCrossEntropy* problem, float* loss, void* workspace, uint64_t workspace_bytes, void* stream, char* message,
                                                     size_t message_capacity) {
    using namespace ftcuda;
    if (problem == nullptr) { return fail(message, message_capacity, 1, "null problem"); }
    const char* reason = check(*problem);
    if (reason == nullptr) { reason = checkStep(*problem); }
    if (reason == nullptr) { reason = checkAddress(loss, kNoLoss); }
    if (reason != nullptr) { return fail(message, message_capacity, 1, "%s", reason); }
    std::uint64_t kept = 0;
    if (const int status = splitWorkspace(*problem, workspace, workspace_bytes, false, kept, message, message_capacity)) { return status; }
    return stepLoss(*problem, loss, workspace, kept, static_cast<unsigned char*>(workspace) + kept, workspace_bytes - kept, stream, message, message_capacity);
}

extern "C" int ftcuda_linear_cross_entropy_step_gradients(const FtcudaLinearCrossEntropy* problem, const float* grad_loss, void* grad_hidden, int64_t grad_hidden_row_stride,
                                                          void* grad_weight, int64_t grad_weight_row_stride, void* workspace, uint64_t workspace_bytes, void* stream,
                                                          char* message, size_t message_capacity) {
    using namespace ftcuda;
    if (problem == nullptr) { return fail(message, message_capacity, 1, "null problem"); }
    const char* reason = check(*problem);
    if (reason == nullptr) { reason = checkStep(*problem); }
    if (reason == nullptr) { reason = checkAddress(grad_loss, kNoUpstream); }
    if (reason == nullptr) {
        reason = checkGradients(*problem, training::elementBytes(problem->element), grad_hidden, grad_hidden_row_stride, grad_weight, grad_weight_row_stride);
    }
    if (reason != nullptr) { return fail(message, message_capacity, 1, "%s", reason); }
    std::uint64_t kept = 0;
    if (const int status = splitWorkspace(*problem, workspace, workspace_bytes, true, kept, message, message_capacity)) { return status; }
    return stepGradients(*problem, grad_loss, problem->element, grad_hidden, grad_hidden_row_stride, grad_weight, grad_weight_row_stride, workspace, kept,
                         static_cast<unsigned char*>(workspace) + kept, workspace_bytes - kept, stream, message, message_capacity);
}

extern "C" int ftcuda_linear_cross_entropy_step_loss_kept(const FtcudaLinearCrossEntropy* problem, float* loss, void* kept, uint64_t kept_bytes, void* workspace,
                                                          uint64_t workspace_bytes, void* stream, char* message, size_t message_capacity) {
    using namespace ftcuda;
    if (problem == nullptr) { return fail(message, message_capacity, 1, "null problem"); }
    const char* reason = check(*problem);
    if (reason == nullptr) { reason = checkStep(*problem); }
    if (reason == nullptr) { reason = checkAddress(loss, kNoLoss); }
    if (reason != nullptr) { return fail(message, message_capacity, 1, "%s", reason); }
    return stepLoss(*problem, loss, kept, kept_bytes, workspace, workspace_bytes, stream, message, message_capacity);
}

extern "C" int ftcuda_linear_cross_entropy_step_gradients_kept(const FtcudaLinearCrossEntropy* problem, const float* grad_loss, void* grad_hidden, int64_t grad_hidden_row_stride,
                                                               void* grad_weight, int64_t grad_weight_row_stride, void* kept, uint64_t kept_bytes, void* workspace,
                                                               uint64_t workspace_bytes, void* stream, char* message, size_t message_capacity) {
    using namespace ftcuda;
    if (problem == nullptr) { return fail(message, message_capacity, 1, "null problem"); }
    const char* reason = check(*problem);
    if (reason == nullptr) { reason = checkStep(*problem); }
    if (reason == nullptr) { reason = checkAddress(grad_loss, kNoUpstream); }
    if (reason == nullptr) {
        reason = checkGradients(*problem, training::elementBytes(problem->element), grad_hidden, grad_hidden_row_stride, grad_weight, grad_weight_row_stride);
    }
    if (reason != nullptr) { return fail(message, message_capacity, 1, "%s", reason); }
    return stepGradients(*problem, grad_loss, problem->element, grad_hidden, grad_hidden_row_stride, grad_weight, grad_weight_row_stride, kept, kept_bytes, workspace, workspace_bytes,
                         stream, message, message_capacity);
}

extern "C" int ftcuda_linear_cross_entropy(const FtcudaLinearCrossEntropy* problem, float* loss, float* lse, void* workspace, uint64_t workspace_bytes, void* stream,
                                           char* message, size_t message_capacity) {
    using namespace ftcuda;
    if (problem == nullptr) { return fail(message, message_capacity, 1, "null problem"); }
    if (const char* reason = check(*problem)) { return fail(message, message_capacity, 1, "%s", reason); }
    const bool empty = problem->tokens == 0;
    if (!(empty && problem->reduction == FTCUDA_REDUCTION_NONE) && !wordAligned(loss)) { return fail(message, message_capacity, 1, "%s", kNoLoss); }
    if (!empty && !wordAligned(lse)) { return fail(message, message_capacity, 1, "lse has no address, or one that is not a multiple of four"); }
    Call call(*problem, message, message_capacity);
    if (const int status = call.begin(Form::kLoss, nullptr, 0, workspace, workspace_bytes, stream)) { return status; }
    if (empty) {
        return finish(problem->reduction == FTCUDA_REDUCTION_NONE ? cudaSuccess : cudaMemsetAsync(loss, 0, sizeof(float), static_cast<cudaStream_t>(stream)), message,
                      message_capacity);
    }
    return finish(call.forward(loss, lse), message, message_capacity);
}

extern "C" int ftcuda_linear_cross_entropy_backward(const FtcudaLinearCrossEntropy* problem, const float* lse, const float* grad_loss, void* grad_hidden,
                                                    int64_t grad_hidden_row_stride, void* grad_weight, int64_t grad_weight_row_stride, void* workspace,
                                                    uint64_t workspace_bytes, void* stream, char* message, size_t message_capacity) {
    using namespace ftcuda;
    if (problem == nullptr) { return fail(message, message_capacity, 1, "null problem"); }
    if (const char* reason = check(*problem)) { return fail(message, message_capacity, 1, "%s", reason); }
    const std::uint64_t bytes = training::elementBytes(problem->element);
    const bool empty          = problem->tokens == 0;
    if (!empty && (!wordAligned(lse) || !wordAligned(grad_loss))) { return fail(message, message_capacity, 1, "lse or the loss's gradient has no address, or one that is not a multiple of four"); }
    if (const char* reason = checkGradients(*problem, bytes, grad_hidden, grad_hidden_row_stride, grad_weight, grad_weight_row_stride)) {
        return fail(message, message_capacity, 1, "%s", reason);
    }
    Call call(*problem, message, message_capacity);
    if (const int status = call.begin(Form::kGradients, nullptr, 0, workspace, workspace_bytes, stream)) { return status; }
    if (empty) {
        if (grad_weight == nullptr) { return 0; }
        return finish(cudaMemset2DAsync(grad_weight, static_cast<std::size_t>(grad_weight_row_stride) * bytes, 0, problem->depth * bytes, problem->vocabulary,
                                        static_cast<cudaStream_t>(stream)), message, message_capacity);
    }
    if (grad_hidden == nullptr && grad_weight == nullptr) { return 0; }
    return finish(call.backward(lse, grad_loss, grad_hidden, grad_hidden_row_stride, grad_weight, grad_weight_row_stride), message, message_capacity);
}
