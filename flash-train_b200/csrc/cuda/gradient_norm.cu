// The norm over many gradients and their clipping (ftcuda/training.h).
//
//   n = (sum of all x^2)^(1/2)  or  max |x|,     out = x * min(1, max_norm / (n + 1e-6))
//
// Two passes over the gradients, since the factor depends on every element: the first reads them, the second
// reads and writes them. Both are bound by HBM. A pass is one launch for up to kDense tensors, whose
// table travels in the kernel's parameters (no copy to the device, so that a captured graph holds it). The tensors are cut into
// chunks of kChunk elements, and every CTA takes a contiguous run of about as many chunks as any other, whatever tensors they are
// of: one of a thousand small tensors costs what its bytes cost. Runs instead of single chunks spare the search for a chunk's tensor.
// The second pass walks every run backwards, as what the first pass read last is still in L2.
//
// The first pass leaves one partial sum for each CTA; every CTA of the second adds them all up again, always in the same order, rather
// than wait for one that does it (a few thousand bytes out of L2), so two launches are all that a clip takes.
//
// Measured beside a copy's 6.55 TB/s: the norm of 453 million FP32 elements in large tensors 255 us, 7.1 TB/s (some of it out of L2); the clip of 906 million from BF16
// to FP32 1.24 ms, 5.9 TB/s over two readings and a writing; that of 75 million in 1024 tensors of odd sizes, to an output that is aligned otherwise, 165 us, 5.5 TB/s.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>
#include <vector>

#include "ptx.cuh"
#include "training_common.cuh"

namespace ftcuda {
namespace {

using training::Element;
using training::Range;
using training::rangeOf;
using training::sideBySide;

constexpr int kThreads            = 256;
constexpr int kSumCtasPerSm       = 4;
constexpr int kScaleCtasPerSm     = 4;
constexpr int kSumBatch           = 4;  // packs of 16 bytes that a thread asks for at a time, twice over
constexpr int kScaleBatch         = 4;
constexpr int kScaleShifted       = 3;  // ... or pairs of packs, where the two sides' alignment differs
constexpr int kScaleSingles       = 8;  // ... or single elements, where their types' sizes do as well
constexpr std::uint32_t kChunk    = 16 * kThreads;  // elements
// Tensors of one launch: what nearly fills the 32764 bytes that a kernel's parameters may take; and few of them, whose table is quicker
// to hand over.
constexpr std::uint32_t kDense    = 1152;           // dense ones
constexpr std::uint32_t kRows     = 608;            // with rows apart among them
constexpr std::uint32_t kFew      = 64;
constexpr std::uint64_t kMostGradients = 1ULL << 20;
constexpr std::uint64_t kMostLaunches  = (kMostGradients + kRows - 1) / kRows;
constexpr std::uint64_t kMostChunks    = 1ULL << 30;  // of all gradients, so that their numbers fit 32 bits: 2^42 elements
constexpr std::uint64_t kMaxGrid  = 2048;           // CTAs of one launch at most (and room for their sums)

struct Entry {
    const void* data;
    void* out;
    std::uint64_t rows, cols;
    std::int64_t row_stride, out_row_stride;
    std::uint64_t first;  // chunks of the tensors before
    std::int32_t element, out_element;
};

// Where rows lie apart.
template<std::uint32_t kCapacity, bool kWithRows> struct RowTable {
    std::uint64_t rows[kCapacity];
    std::int64_t row_stride[kCapacity], out_row_stride[kCapacity];
};
template<std::uint32_t kCapacity> struct RowTable<kCapacity, false> {};

template<std::uint32_t kCapacity, bool kWithRows> struct Table : RowTable<kCapacity, kWithRows> {
    static constexpr std::uint32_t kTensors = kCapacity;
    const void* data[kCapacity];
    void* out[kCapacity];
    std::uint64_t shape[kCapacity];  // cols, the element's type and the output's: 48, 8, 8 bits
    std::uint32_t first[kCapacity];
    std::uint32_t chunks, count;

    __host__ __device__ __forceinline__ void set(std::uint32_t i, const Entry& entry) {
        data[i]  = entry.data;
        out[i]   = entry.out;
        shape[i] = entry.cols | static_cast<std::uint64_t>(entry.element) << 48 | static_cast<std::uint64_t>(entry.out_element) << 56;
        first[i] = static_cast<std::uint32_t>(entry.first);
        if constexpr (kWithRows) {
            this->rows[i]           = entry.rows;
            this->row_stride[i]     = entry.row_stride;
            this->out_row_stride[i] = entry.out_row_stride;
        }
    }
    __device__ __forceinline__ Entry get(std::uint32_t i) const {
        Entry entry;
        entry.data           = data[i];
        entry.out            = out[i];
        entry.cols           = shape[i] & 0xFFFFFFFFFFFFULL;
        entry.element        = static_cast<std::int32_t>(shape[i] >> 48 & 0xFF);
        entry.out_element    = static_cast<std::int32_t>(shape[i] >> 56);
        entry.first          = first[i];
        entry.rows           = 1;
        entry.row_stride     = 0;
        entry.out_row_stride = 0;
        if constexpr (kWithRows) {
            entry.rows           = this->rows[i];
            entry.row_stride     = this->row_stride[i];
            entry.out_row_stride = this->out_row_stride[i];
        }
        return entry;
    }
};
using FewTable   = Table<kFew, true>;
using RowsTable  = Table<kRows, true>;
using DenseTable = Table<kDense, false>;
static_assert(sizeof(RowsTable) + 64 <= 32764 && sizeof(DenseTable) + 64 <= 32764, "kernel parameters");

// Largest and smallest sum of squares that FP32 holds as well as 64 bits would: with a sum of up to 16 squares in here, none overflowed, and what
// underflowed in one (2^-150) is under 2^-60 of the sum.
constexpr float kLargestSum  = 0x1p+120F;
constexpr float kSmallestSum = 0x1p-90F;

struct Sum2 {
    double total = 0.0;
    // n <= 16 neighbouring elements.
    template<int n> __device__ __forceinline__ void add(const float (&x)[n]) {
        float sum = 0.0F;
#pragma unroll
        for (int i = 0; i < n; ++i) { sum = fmaf(x[i], x[i], sum); }
        if (sum >= kSmallestSum && sum <= kLargestSum) {
            total += static_cast<double>(sum);
        } else {
#pragma unroll
            for (int i = 0; i < n; ++i) { total = fma(static_cast<double>(x[i]), static_cast<double>(x[i]), total); }
        }
    }
    __device__ __forceinline__ void join(double other) { total += other; }
    __device__ __forceinline__ double norm() const { return sqrt(total); }
};

// |x| as a whole number orders the finite numbers, the infinities above them and NaN above all.
struct SumInf {
    double total = 0.0;  // of magnitudes that are FP32 numbers: exact
    template<int n> __device__ __forceinline__ void add(const float (&x)[n]) {
        std::uint32_t largest = 0;
#pragma unroll
        for (int i = 0; i < n; ++i) { largest = max(largest, __float_as_uint(x[i]) & 0x7FFFFFFFU); }
        join(static_cast<double>(__uint_as_float(largest)));
    }
    __device__ __forceinline__ void join(double other) { total = other > total || other != other ? other : total; }
    __device__ __forceinline__ double norm() const { return total; }
};

template<typename T, int n> struct alignas(sizeof(T) * n) Pack {
    T at[n];
};

// Elements up to the first one at a multiple of 16 bytes.
template<typename T> __device__ __forceinline__ std::uint32_t misaligned(const T* at) {
    return static_cast<std::uint32_t>((16 - (reinterpret_cast<std::uintptr_t>(at) & 15)) & 15) / static_cast<std::uint32_t>(sizeof(T));
}

// Goes over `count` packs with all threads of the CTA, from the last one back with kBack, kBatch at a time for each: the next batch is asked
// for (by `load`) before `use` is called for the packs of the one at hand, so that loads are always on their way.
template<int kBatch, bool kBack, typename Load, typename Use>
__device__ __forceinline__ void stream(const Load& load, std::uint64_t count, const Use& use) {
    using P = decltype(load(std::int64_t{0}));
    constexpr std::int64_t kStep  = kBack ? -kBatch * kThreads : kBatch * kThreads;
    constexpr std::int64_t kEach  = kBack ? -kThreads : kThreads;
    const std::uint64_t batches   = count / (kBatch * kThreads);
    std::int64_t at               = kBack ? static_cast<std::int64_t>(count) - 1 - threadIdx.x : threadIdx.x;
    if (batches != 0) {
        P now[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) { now[i] = load(at + i * kEach); }
#pragma unroll 1
        for (std::uint64_t batch = 1; batch < batches; ++batch) {
            P next[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) { next[i] = load(at + kStep + i * kEach); }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) { use(at + i * kEach, now[i]); }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) { now[i] = next[i]; }
            at += kStep;
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) { use(at + i * kEach, now[i]); }
        at += kStep;
    }
#pragma unroll 1
    for (; kBack ? at >= 0 : at < static_cast<std::int64_t>(count); at += kEach) {
        const P one = load(at);
        use(at, one);
    }
}

// Written once and not read again here: leaves what the first pass read in L2.
template<typename Q> __device__ __forceinline__ void storeStreaming(Q* to, const Q& value) {
    if constexpr (sizeof(Q) == 16) {
        __stcs(reinterpret_cast<uint4*>(to), *reinterpret_cast<const uint4*>(&value));
    } else if constexpr (sizeof(Q) == 8) {
        __stcs(reinterpret_cast<uint2*>(to), *reinterpret_cast<const uint2*>(&value));
    } else if constexpr (sizeof(Q) == 4) {
        __stcs(reinterpret_cast<unsigned int*>(to), *reinterpret_cast<const unsigned int*>(&value));
    } else {
        __stcs(reinterpret_cast<unsigned short*>(to), *reinterpret_cast<const unsigned short*>(&value));
    }
}

// `count` neighbouring elements: packs of 16 bytes, and the ends one by one.
template<typename T, typename Sum> __device__ __forceinline__ void sumRow(const T* row, std::uint64_t count, Sum& sum) {
    constexpr int kEach         = 16 / sizeof(T);
    using P                     = Pack<T, kEach>;
    const std::uint32_t head    = static_cast<std::uint32_t>(min(count, static_cast<std::uint64_t>(misaligned(row))));
    const std::uint64_t packs   = (count - head) / kEach;
    const std::uint64_t rest    = head + packs * kEach;
    const std::uint32_t ends    = head + static_cast<std::uint32_t>(count - rest);
    if (threadIdx.x < ends) {
        const float x[1] = {Element<T>::widen(row[threadIdx.x < head ? threadIdx.x : rest + (threadIdx.x - head)])};
        sum.add(x);
    }
    const P* const from = reinterpret_cast<const P*>(row + head);
    stream<kSumBatch, false>([&](std::int64_t at) { return from[at]; }, packs, [&](std::int64_t, const P& pack) {
        float x[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j) { x[j] = Element<T>::widen(pack.at[j]); }
        sum.add(x);
    });
}

// out = row * factor. Packs of four elements (eight where both sides have 16 bits) where both sides are aligned for them at the same element: a
// warp's accesses are neighbours on both sides then. Otherwise shifted packs, or one element at a time.
template<typename T, typename U>
__device__ __forceinline__ void scaleRow(const T* row, U* out, std::uint64_t count, float factor) {
    constexpr int kEach      = 16 / (sizeof(T) > sizeof(U) ? sizeof(T) : sizeof(U));
    using P                  = Pack<T, kEach>;
    using Q                  = Pack<U, kEach>;
    const std::uint32_t head = static_cast<std::uint32_t>(min(count, static_cast<std::uint64_t>(sizeof(T) >= sizeof(U) ? misaligned(row) : misaligned(out))));
    const bool both          = reinterpret_cast<std::uintptr_t>(row + head) % sizeof(P) == 0 && reinterpret_cast<std::uintptr_t>(out + head) % sizeof(Q) == 0;
    if (both) {
        const std::uint64_t packs = (count - head) / kEach;
        const std::uint64_t rest  = head + packs * kEach;
        const std::uint32_t ends  = head + static_cast<std::uint32_t>(count - rest);
        if (threadIdx.x < ends) {
            const std::uint64_t at = threadIdx.x < head ? threadIdx.x : rest + (threadIdx.x - head);
            out[at]                = Element<U>::narrow(Element<T>::widen(row[at]) * factor);
        }
        Q* const to = reinterpret_cast<Q*>(out + head);
        const P* const from = reinterpret_cast<const P*>(row + head);
        stream<kScaleBatch, true>([&](std::int64_t at) { return from[at]; }, packs, [&](std::int64_t at, const P& pack) {
            Q o;
#pragma unroll
            for (int j = 0; j < kEach; ++j) { o.at[j] = Element<U>::narrow(Element<T>::widen(pack.at[j]) * factor); }
            storeStreaming(to + at, o);
        });
    } else if (sizeof(T) == sizeof(U) && row != static_cast<const void*>(out)) {
        // Packs of both sides, the input's shifted: pack k of the output lies across two of the input's, whose words are moved down by `shift` bytes. The second one
        // of them a neighbour reads as well.
        const std::uint32_t first  = misaligned(row);
        const std::uint32_t start  = misaligned(out) >= first ? misaligned(out) : misaligned(out) + kEach;
        const std::uint64_t whole  = count > first ? (count - first) / kEach : 0;
        const std::uint64_t packs  = whole > 1 ? whole - 1 : 0;
        const std::uint64_t rest   = start + packs * kEach;
        const std::uint32_t ends   = packs != 0 ? start + static_cast<std::uint32_t>(count - rest) : static_cast<std::uint32_t>(count);  // fewer than four packs
        const std::uint32_t shift  = (start - first) * static_cast<std::uint32_t>(sizeof(T));
        const uint4* const from    = reinterpret_cast<const uint4*>(row + first);
        Q* const to                = reinterpret_cast<Q*>(out + start);
        if (threadIdx.x < ends) {
            const std::uint64_t at = packs == 0 || threadIdx.x < start ? threadIdx.x : rest + (threadIdx.x - start);
            out[at]                = Element<U>::narrow(Element<T>::widen(row[at]) * factor);
        }
        struct Two {
            uint4 low, high;
        };
        stream<kScaleShifted, true>([&](std::int64_t at) { return Two{from[at], from[at + 1]}; }, packs, [&](std::int64_t at, const Two& two) {
            std::uint32_t words[8] = {two.low.x, two.low.y, two.low.z, two.low.w, two.high.x, two.high.y, two.high.z, two.high.w};
#pragma unroll
            for (int by = 2; by > 0; by /= 2) {
                if ((shift / 4 & by) != 0) {
#pragma unroll
                    for (int i = 0; i + by < 8; ++i) { words[i] = words[i + by]; }
                }
            }
            std::uint32_t moved[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { moved[i] = __funnelshift_r(words[i], words[i + 1], shift % 4 * 8); }
            const P pack = *reinterpret_cast<const P*>(moved);
            Q o;
#pragma unroll
            for (int j = 0; j < kEach; ++j) { o.at[j] = Element<U>::narrow(Element<T>::widen(pack.at[j]) * factor); }
            storeStreaming(to + at, o);
        });
    } else {
        stream<kScaleSingles, true>([&](std::int64_t at) { return row[at]; }, count, [&](std::int64_t at, const T& x) { storeStreaming(out + at, Element<U>::narrow(Element<T>::widen(x) * factor)); });
    }
}

// The tensor that chunk `chunk` is of.
template<typename TableT> __device__ __forceinline__ std::uint32_t findEntry(const TableT& table, std::uint64_t chunk) {
    std::uint32_t low = 0, high = table.count;  // first[low] <= chunk < first[high]
    while (high - low > 1) {
        const std::uint32_t middle = (low + high) / 2;
        if (table.first[middle] <= chunk) {
            low = middle;
        } else {
            high = middle;
        }
    }
    return low;
}

// Neighbouring elements in the chunks from `begin` up to `end` of one tensor: of a dense one all of them, of a row of others the first chunk's
// (kBack: the last one's).
struct Stretch {
    std::uint64_t row, col, count, chunks;
};

template<bool kBack> __device__ __forceinline__ Stretch stretchOf(const Entry& entry, std::uint64_t begin, std::uint64_t end) {
    Stretch s;
    if (entry.rows == 1) {
        s.row    = 0;
        s.col    = (begin - entry.first) * kChunk;
        s.chunks = end - begin;
    } else {
        const std::uint64_t local = (kBack ? end - 1 : begin) - entry.first, per_row = (entry.cols + kChunk - 1) / kChunk;
        s.row                     = local / per_row;
        s.col                     = (local - s.row * per_row) * kChunk;
        s.chunks                  = 1;
    }
    s.count = min(s.chunks * kChunk, entry.cols - s.col);
    return s;
}

// Joined over the CTA, the same order in every call; the result in thread 0.
template<typename Sum> __device__ __forceinline__ void joinBlock(Sum& sum, double* shared) {
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2) { sum.join(__shfl_down_sync(0xFFFFFFFFU, sum.total, offset)); }
    if ((threadIdx.x & 31) == 0) { shared[threadIdx.x >> 5] = sum.total; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int warp = 1; warp < kThreads / 32; ++warp) { sum.join(shared[warp]); }
    }
}

template<typename Sum, typename TableT> __global__ void __launch_bounds__(kThreads, kSumCtasPerSm) gradientSums(const __grid_constant__ TableT table, double* partials) {
    __shared__ double shared[kThreads / 32];
    gridDependencyWait();
    gridDependencyLaunchDependents();
    const std::uint64_t all = table.chunks, begin = all * blockIdx.x / gridDim.x, end = all * (blockIdx.x + 1) / gridDim.x;
    Sum sum;
    if (begin < end) {
        std::uint32_t index = findEntry(table, begin);
#pragma unroll 1
        for (std::uint64_t chunk = begin; chunk < end;) {
            while (index + 1 < table.count && table.first[index + 1] <= chunk) { ++index; }
            const Entry entry         = table.get(index);
            const std::uint64_t last  = index + 1 < table.count ? min(end, static_cast<std::uint64_t>(table.first[index + 1])) : end;
            const Stretch s           = stretchOf<false>(entry, chunk, last);
            const std::int64_t offset = static_cast<std::int64_t>(s.row) * entry.row_stride + static_cast<std::int64_t>(s.col);
            switch (entry.element) {
                case FTCUDA_ELEMENT_FP32: sumRow(static_cast<const float*>(entry.data) + offset, s.count, sum); break;
                case FTCUDA_ELEMENT_FP16: sumRow(static_cast<const __half*>(entry.data) + offset, s.count, sum); break;
                default: sumRow(static_cast<const __nv_bfloat16*>(entry.data) + offset, s.count, sum); break;
            }
            chunk += s.chunks;
        }
    }
    joinBlock(sum, shared);
    if (threadIdx.x == 0) { partials[blockIdx.x] = sum.total; }
}

// All partial sums joined; every CTA and every launch comes to the same number.
template<typename Sum> __device__ __forceinline__ double joinPartials(const double* partials, std::uint32_t count, double* shared) {
    Sum sum;
    for (std::uint32_t at = threadIdx.x; at < count; at += kThreads) { sum.join(__ldcg(partials + at)); }
    joinBlock(sum, shared);
    return sum.norm();
}

template<typename Sum> __global__ void __launch_bounds__(kThreads) gradientNorm(const double* partials, std::uint32_t count, float* norm) {
    __shared__ double shared[kThreads / 32];
    gridDependencyWait();
    gridDependencyLaunchDependents();
    const double total = joinPartials<Sum>(partials, count, shared);
    if (threadIdx.x == 0) { *norm = static_cast<float>(total); }
}

template<typename T> __device__ __forceinline__ void scaleStretch(const Entry& entry, const Stretch& s, float factor) {
    const T* const row        = static_cast<const T*>(entry.data) + static_cast<std::int64_t>(s.row) * entry.row_stride + static_cast<std::int64_t>(s.col);
    const std::int64_t offset = static_cast<std::int64_t>(s.row) * entry.out_row_stride + static_cast<std::int64_t>(s.col);
    switch (entry.out_element) {
        case FTCUDA_ELEMENT_FP32: scaleRow(row, static_cast<float*>(entry.out) + offset, s.count, factor); break;
        case FTCUDA_ELEMENT_FP16: scaleRow(row, static_cast<__half*>(entry.out) + offset, s.count, factor); break;
        default: scaleRow(row, static_cast<__nv_bfloat16*>(entry.out) + offset, s.count, factor); break;
    }
}

// The CTA's run of chunks, from the last one back.
template<typename TableT> __device__ __forceinline__ void scaleRun(const TableT& table, float factor) {
    const std::uint64_t all = table.chunks, begin = all * blockIdx.x / gridDim.x, end = all * (blockIdx.x + 1) / gridDim.x;
    if (begin == end) { return; }
    std::uint32_t index = findEntry(table, end - 1);
#pragma unroll 1
    for (std::uint64_t chunk = end; chunk > begin;) {
        while (table.first[index] >= chunk) { --index; }
        const Entry entry  = table.get(index);
        const Stretch s    = stretchOf<true>(entry, max(begin, entry.first), chunk);
        chunk -= s.chunks;
        if (factor == 1.0F && entry.out == entry.data) { continue; }
        switch (entry.element) {
            case FTCUDA_ELEMENT_FP32: scaleStretch<float>(entry, s, factor); break;
            case FTCUDA_ELEMENT_FP16: scaleStretch<__half>(entry, s, factor); break;
            default: scaleStretch<__nv_bfloat16>(entry, s, factor); break;
        }
    }
}

template<typename Sum, typename TableT>
__global__ void __launch_bounds__(kThreads, kScaleCtasPerSm) gradientScale(const __grid_constant__ TableT table, const double* partials, std::uint32_t count,
                                                                           double max_norm, float* norm) {
    __shared__ double shared[kThreads / 32];
    __shared__ float shared_factor;
    gridDependencyWait();
    gridDependencyLaunchDependents();
    const double total = joinPartials<Sum>(partials, count, shared);
    if (threadIdx.x == 0) {
        const double ratio = max_norm / (total + 1e-6);
        shared_factor      = ratio >= 1.0 ? 1.0F : static_cast<float>(ratio);  // a ratio that is not a number stays one
        if (norm != nullptr && blockIdx.x == 0) { *norm = static_cast<float>(total); }
    }
    __syncthreads();
    scaleRun(table, shared_factor);
}

// The factor as the caller gives it.
template<typename TableT> __global__ void __launch_bounds__(kThreads, kScaleCtasPerSm) gradientMultiply(const __grid_constant__ TableT table, const float* factor) {
    gridDependencyWait();
    gridDependencyLaunchDependents();
    scaleRun(table, *factor);
}

// ---------------------------------------------------------------- host

// nullptr, or what is wrong with a gradient (`out` looked at for a clip alone).
const char* checkGradient(const FtcudaGradient& g, bool clip) {
    if (g.rows == 0 || g.cols == 0) { return nullptr; }
    const std::uint64_t bytes = training::elementBytes(g.element);
    if (bytes == 0) { return "the element type is none of FP32, FP16 and BF16"; }
    if (g.data == nullptr) { return "no address"; }
    if (!training::aligned(g.data, bytes)) { return "the address is not a multiple of the element's size"; }
    if (g.rows >= (1ULL << 40) || g.cols >= (1ULL << 40)) { return "an extent is too large"; }
    if (g.rows > 1 && (g.row_stride < static_cast<std::int64_t>(g.cols) || g.row_stride >= (1LL << 40))) { return "rows overlap, or lie too far apart"; }
    if (g.rows > (1ULL << 44) / (g.rows > 1 ? static_cast<std::uint64_t>(g.row_stride) : g.cols)) { return "too many elements, or too far apart"; }
    if (!clip) { return nullptr; }
    const std::uint64_t out_bytes = training::elementBytes(g.out_element);
    if (out_bytes == 0) { return "the output's element type is none of FP32, FP16 and BF16"; }
    if (g.out == nullptr) { return "no address for the output"; }
    if (!training::aligned(g.out, out_bytes)) { return "the output's address is not a multiple of its element's size"; }
    if (g.rows > 1 && (g.out_row_stride < static_cast<std::int64_t>(g.cols) || g.out_row_stride >= (1LL << 40))) { return "the output's rows overlap, or lie too far apart"; }
    if (g.rows > 1 && g.rows > (1ULL << 44) / static_cast<std::uint64_t>(g.out_row_stride)) { return "the output's rows lie too far apart"; }
    return nullptr;
}

Range inputOf(const FtcudaGradient& g) { return rangeOf(g.data, g.rows, g.cols, g.row_stride, training::elementBytes(g.element)); }
Range outputOf(const FtcudaGradient& g) { return rangeOf(g.out, g.rows, g.cols, g.out_row_stride, training::elementBytes(g.out_element)); }

// An operand by where it begins, and which: gradient 2 i is read, 2 i + 1 written.
struct Operand {
    std::uint64_t begin;
    std::uint64_t which;
};

// nullptr, or why the gradients cannot be clipped at once: no byte may be written that another operand reads or writes. What is read outside of
// all that is written is left out before anything is sorted.
const char* checkOverlap(const FtcudaGradient* gradients, std::uint64_t count) {
    std::uint64_t lowest = ~std::uint64_t{0}, highest = 0;
    for (std::uint64_t i = 0; i < count; ++i) {
        if (gradients[i].rows == 0 || gradients[i].cols == 0) { continue; }
        const Range out = outputOf(gradients[i]);
        lowest          = std::min(lowest, out.begin);
        highest         = std::max(highest, out.end);
    }
    std::vector<Operand> operands;
    operands.reserve(2 * count);
    for (std::uint64_t i = 0; i < count; ++i) {
        const FtcudaGradient& g = gradients[i];
        if (g.rows == 0 || g.cols == 0) { continue; }
        operands.push_back({reinterpret_cast<std::uintptr_t>(g.out), 2 * i + 1});
        if (g.data == g.out) {
            if (g.element != g.out_element || inputOf(g).stride != outputOf(g).stride) { return "a gradient that is its own output has another type or stride there"; }
            continue;
        }
        const Range in = inputOf(g);
        if (in.begin < highest && in.end > lowest) { operands.push_back({in.begin, 2 * i}); }
    }
    const auto before = [](const Operand& a, const Operand& b) { return a.begin < b.begin; };
    if (!std::is_sorted(operands.begin(), operands.end(), before)) { std::sort(operands.begin(), operands.end(), before); }
    const auto range = [&](const Operand& o) { return (o.which & 1) != 0 ? outputOf(gradients[o.which / 2]) : inputOf(gradients[o.which / 2]); };
    for (std::size_t i = 0; i < operands.size(); ++i) {
        const Range a = range(operands[i]);
        for (std::size_t j = i + 1; j < operands.size() && operands[j].begin < a.end; ++j) {
            if (((operands[i].which | operands[j].which) & 1) != 0 && !sideBySide(a, range(operands[j]))) {
                return "an output overlaps another gradient or output";
            }
        }
    }
    return nullptr;
}

// The gradient as the kernels see it: rows that follow one another are one.
Entry entryOf(const FtcudaGradient& g, bool clip) {
    Entry entry{g.data, clip ? g.out : nullptr, g.rows, g.cols, g.row_stride, g.out_row_stride, 0, g.element, g.out_element};
    if (g.rows == 1 || (g.row_stride == static_cast<std::int64_t>(g.cols) && (!clip || g.out_row_stride == g.row_stride))) {
        entry.cols = g.rows * g.cols;
        entry.rows = 1;
    }
    return entry;
}

std::uint64_t chunksOf(const Entry& entry) { return entry.rows * ceilDiv(entry.cols, kChunk); }

// As many gradients from `begin` on as one launch takes; returns where the next one begins.
template<typename TableT> std::uint64_t fillTable(TableT& table, const FtcudaGradient* gradients, std::uint64_t begin, std::uint64_t count, bool clip) {
    table.count          = 0;
    std::uint64_t chunks = 0, i = begin;
    for (; i < count && table.count < TableT::kTensors; ++i) {
        if (gradients[i].rows == 0 || gradients[i].cols == 0) { continue; }
        Entry entry                = entryOf(gradients[i], clip);
        const std::uint64_t wanted = chunksOf(entry);
        entry.first = chunks;
        table.set(table.count++, entry);
        chunks += wanted;
    }
    table.chunks = static_cast<std::uint32_t>(chunks);
    return i;
}

// Launches that `count` gradients can take.
std::uint64_t launchesFor(std::uint64_t count) { return count <= kFew ? 1 : ceilDiv(count, kRows); }

// CTAs for that many chunks: the SMs filled once, or a chunk each.
std::uint32_t gridFor(std::uint64_t chunks, int sms, int per_sm) {
    const std::uint64_t most = std::min<std::uint64_t>(kMaxGrid, static_cast<std::uint64_t>(sms) * static_cast<std::uint64_t>(per_sm));
    return static_cast<std::uint32_t>(std::max<std::uint64_t>(1, std::min(chunks, most)));
}

struct Call {
    const FtcudaGradient* gradients;
    std::uint64_t count;
    bool clip;
    double max_norm;
    float* norm;
    double* partials;
    int sms;
    cudaStream_t stream;
};

template<typename Sum, typename TableT> cudaError_t enqueue(const Call& call) {
    TableT table;
    std::uint64_t starts[kMostLaunches + 1] = {0};
    std::uint32_t partials = 0, launches = 0;
    for (std::uint64_t at = 0; launches == 0 || at < call.count; ++launches) {
        if (launches == kMostLaunches) { return cudaErrorInvalidValue; }  // (not with the counts and sizes that the checks allow)
        at                       = fillTable(table, call.gradients, at, call.count, call.clip);
        starts[launches + 1]     = at;
        const std::uint32_t grid = gridFor(table.chunks, call.sms, kSumCtasPerSm);
        // The first launch of a call is an ordinary one: it starts when what came before in the stream is done.
        if (launches == 0) {
            gradientSums<Sum, TableT><<<grid, kThreads, 0, call.stream>>>(table, call.partials);
            const cudaError_t error = cudaGetLastError();
            if (error != cudaSuccess) { return error; }
            countLaunches(1);
        } else {
            const cudaError_t error = training::launchOverlapped(gradientSums<Sum, TableT>, dim3(grid), dim3(kThreads), 0, call.stream, table, call.partials + partials);
            if (error != cudaSuccess) { return error; }
        }
        partials += grid;
    }
    if (!call.clip) {
        return training::launchOverlapped(gradientNorm<Sum>, dim3(1), dim3(kThreads), 0, call.stream, static_cast<const double*>(call.partials), partials, call.norm);
    }
    for (std::uint32_t l = launches; l-- > 0;) {
        if (launches > 1) { fillTable(table, call.gradients, starts[l], starts[l + 1], call.clip); }
        const cudaError_t error = training::launchOverlapped(gradientScale<Sum, TableT>, dim3(gridFor(table.chunks, call.sms, kScaleCtasPerSm)), dim3(kThreads), 0,
                                                             call.stream, table, static_cast<const double*>(call.partials), partials, call.max_norm,
                                                             l == 0 ? call.norm : static_cast<float*>(nullptr));
        if (error != cudaSuccess) { return error; }
    }
    return cudaSuccess;
}

template<typename TableT> cudaError_t enqueueMultiply(const FtcudaGradient* gradients, std::uint64_t count, const float* factor, int sms, cudaStream_t stream) {
    TableT table;
    for (std::uint64_t at = 0; at < count;) {
        const bool first         = at == 0;
        at                       = fillTable(table, gradients, at, count, true);
        const std::uint32_t grid = gridFor(table.chunks, sms, kScaleCtasPerSm);
        if (first) {  // an ordinary launch: it starts when what came before in the stream is done
            gradientMultiply<TableT><<<grid, kThreads, 0, stream>>>(table, factor);
            const cudaError_t error = cudaGetLastError();
            if (error != cudaSuccess) { return error; }
            countLaunches(1);
        } else {
            const cudaError_t error = training::launchOverlapped(gradientMultiply<TableT>, dim3(grid), dim3(kThreads), 0, stream, table, factor);
            if (error != cudaSuccess) { return error; }
        }
    }
    return cudaSuccess;
}

// The table that a list of gradients takes: the small one, the one for many dense tensors, or the one that can have rows apart.
template<typename Few, typename Dense, typename Rows>
cudaError_t withTable(const FtcudaGradient* gradients, std::uint64_t count, bool clip, const Few& few, const Dense& dense, const Rows& rows) {
    if (count <= kFew) { return few(); }
    for (std::uint64_t i = 0; i < count; ++i) {
        if (gradients[i].rows != 0 && gradients[i].cols != 0 && entryOf(gradients[i], clip).rows != 1) { return rows(); }
    }
    return dense();
}

// What every call minds about its gradients; 0, or a failure with its message.
int checkGradients(const FtcudaGradient* gradients, std::uint64_t count, bool written, char* message, std::size_t capacity) {
    if (gradients == nullptr && count != 0) { return fail(message, capacity, 1, "null gradients"); }
    if (count > kMostGradients) { return fail(message, capacity, 1, "too many gradients"); }
    std::uint64_t chunks = 0;
    for (std::uint64_t i = 0; i < count; ++i) {
        const char* reason = checkGradient(gradients[i], written);
        if (reason == nullptr && gradients[i].rows != 0 && gradients[i].cols != 0) {
            chunks += chunksOf(entryOf(gradients[i], written));  // (at most 2^44 each)
            if (chunks > kMostChunks) { reason = "too many elements, or rows apart, in all"; }
        }
        if (reason != nullptr) { return fail(message, capacity, 1, "gradient %llu: %s", static_cast<unsigned long long>(i), reason); }
    }
    if (!written) { return 0; }
    try {
        if (const char* reason = checkOverlap(gradients, count)) { return fail(message, capacity, 1, "%s", reason); }
    } catch (const std::bad_alloc&) { return fail(message, capacity, 1, "out of host memory"); }
    return 0;
}

int runCall(const FtcudaGradient* gradients, std::uint64_t count, int norm_kind, bool clip, double max_norm, float* norm, std::int32_t device, void* workspace,
            std::uint64_t workspace_bytes, void* stream, char* message, std::size_t capacity) {
    if (norm == nullptr || !training::aligned(norm, 4)) { return fail(message, capacity, 1, "the norm has no address, or one that is not a multiple of four"); }
    if (norm_kind != FTCUDA_NORM_2 && norm_kind != FTCUDA_NORM_INF) { return fail(message, capacity, 1, "unknown kind of norm %d", norm_kind); }
    if (clip && !(max_norm >= 0.0)) { return fail(message, capacity, 1, "max_norm must not be negative"); }
    const std::uint64_t needed = ftcuda_gradient_norm_workspace_bytes(count);
    if (workspace == nullptr || workspace_bytes < needed || !training::aligned(workspace, 8)) {
        return fail(message, capacity, 1, "workspace of %llu bytes needed, at a multiple of eight", static_cast<unsigned long long>(needed));
    }
    if (const int status = checkGradients(gradients, count, clip, message, capacity)) { return status; }
    int sms = 0;
    if (!training::deviceIsCurrent(device, message, capacity) || !deviceSmCount(device, &sms, message, capacity)) { return 1; }
    const Call call{gradients, count, clip, max_norm, norm, static_cast<double*>(workspace), sms, static_cast<cudaStream_t>(stream)};
    const auto run = [&](auto sum) {
        using Sum = decltype(sum);
        return withTable(gradients, count, clip, [&] { return enqueue<Sum, FewTable>(call); }, [&] { return enqueue<Sum, DenseTable>(call); },
                         [&] { return enqueue<Sum, RowsTable>(call); });
    };
    const cudaError_t error = norm_kind == FTCUDA_NORM_2 ? run(Sum2{}) : run(SumInf{});
    if (error != cudaSuccess) { return fail(message, capacity, 1, "%s", cudaGetErrorString(error)); }
    return 0;
}

}  // namespace
}  // namespace ftcuda

extern "C" uint64_t ftcuda_gradient_norm_workspace_bytes(uint64_t count) {
    return ftcuda::launchesFor(count == 0 ? 1 : count) * ftcuda::kMaxGrid * sizeof(double);
}

extern "C" int ftcuda_gradient_norm(const FtcudaGradient* gradients, uint64_t count, int norm_kind, float* norm, int32_t device, void* workspace,
                                    uint64_t workspace_bytes, void* stream, char* message, size_t message_capacity) {
    return ftcuda::runCall(gradients, count, norm_kind, false, 0.0, norm, device, workspace, workspace_bytes, stream, message, message_capacity);
}

extern "C" int ftcuda_gradient_clip(const FtcudaGradient* gradients, uint64_t count, int norm_kind, double max_norm, float* norm, int32_t device,
                                    void* workspace, uint64_t workspace_bytes, void* stream, char* message, size_t message_capacity) {
    return ftcuda::runCall(gradients, count, norm_kind, true, max_norm, norm, device, workspace, workspace_bytes, stream, message, message_capacity);
}

extern "C" int ftcuda_gradient_scale(const FtcudaGradient* gradients, uint64_t count, const float* factor, int32_t device, void* stream, char* message,
                                     size_t message_capacity) {
    using namespace ftcuda;
    if (factor == nullptr || !training::aligned(factor, 4)) { return fail(message, message_capacity, 1, "the factor has no address, or one that is not a multiple of four"); }
    if (const int status = checkGradients(gradients, count, true, message, message_capacity)) { return status; }
    int sms = 0;
    if (!training::deviceIsCurrent(device, message, message_capacity) || !deviceSmCount(device, &sms, message, message_capacity)) { return 1; }
    const auto queue        = static_cast<cudaStream_t>(stream);
    const cudaError_t error = withTable(gradients, count, true, [&] { return enqueueMultiply<FewTable>(gradients, count, factor, sms, queue); },
                                        [&] { return enqueueMultiply<DenseTable>(gradients, count, factor, sms, queue); },
                                        [&] { return enqueueMultiply<RowsTable>(gradients, count, factor, sms, queue); });
    if (error != cudaSuccess) { return fail(message, message_capacity, 1, "%s", cudaGetErrorString(error)); }
    return 0;
}
