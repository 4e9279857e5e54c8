// The products of the linear cross entropy on BF16 or FP16 operands, or on FP32 ones as sums of three BF16 (loss_products.hpp), each with
// its epilogue (linear_cross_entropy.cu has the whole).
//
//   statistics   Z = H W^T; of a tile of Z nothing is kept but the rows' maxima and sums of exponentials
//   kept         the same, and the exponentials go to memory in FP16, each against its row's maximum in 64 or 128 columns
//   slopes       Z once more; dZ = scale (exp(Z - lse) - onehot), rounded to the operands' type, goes to memory for a piece of the vocabulary
//   gradients    dH (+)= dZ W and dW = dZ^T H of that piece, in one launch
//
// dZ is rounded to 16 bits because the tensor cores take it as an operand of the type that W and H have; half a step (2^-9, 2^-12
// of each value) is what the gradients' own rounding comes to as well. Its scale brings the largest possible value near 1 (BF16) or 2^14 (FP16, whose
// exponents would not hold the small probabilities otherwise). With an upstream gradient for each token FP16's range holds only those near the largest at one
// scale, which dW's sums over tokens need; dH's rows have a scale each, and a dZ of their own.
//
// One kernel does all four. A pair of CTAs (tcgen05 cta_group::2, a cluster of two) takes tiles of 256 rows and up to 256 columns, K in
// blocks of 64; a CTA brings its 128 rows of A and its half of B, each as the matrix lies in memory: an operand whose
// neighbours run along K is a K-major operand, one whose neighbours run along its rows an MN-major one, so nothing is ever transposed.
//
//   warps 0, 2   TMA producers of A and of B (one thread each, in both CTAs; the bytes of both count on the first CTA's barrier)
//   warp 1       MMA issuer (one thread, in the first CTA, for both CTAs' tensor cores)
//   warps 4-11   epilogue, 32 rows x half of the columns each
//
// An FP32 product is six BF16 ones (kTermsA, kTermsB say which planes), a K block's one after another in the same accumulator: a sixth of
// the rate that the tensor cores have for BF16, with no scaling and no case that it is not exact enough for.
//
// Tensor memory holds two accumulators of 256 columns: one is filled while the other is read. What the epilogue reads goes to registers at once
// and the accumulator back to the issuer, every kSumBlocks blocks of K, or kFp32Blocks where the operands are FP32: the tensor cores cut off
// below the last bit of the sum so far, which makes a sum of many steps short by about 2^-23 for each, while the parts are added to nearest. (Sums of
// positive terms over 131072 columns and over 16384 tokens came out 8.9e-5 and 1.1e-4 too small when read at the end alone, now 1.8e-5 and 4.2e-5; the loss
// of 257 x 4096 x 131072 was off by 1.3e-6, now by 3.2e-7. A step of 4096 x 4096 x 65536 takes 4.40 ms for 4.38.) A thread has one row, so maxima, sums and
// the target's column need no exchange between threads, and its output is 256 neighbouring bytes, written 32 at a time.
//
// A K block is 512 cycles of MMAs, and the threads that feed them must need less. One producer for both operands, with its parameters read again for
// every block, took 660; an issuer under `if (lane == 0)` as much, as the compiler moves every descriptor into uniform registers where the
// branch may diverge. With a producer for each operand and the issuing warp in step (one thread elected for the instructions alone) the
// tensor pipe is busy for 90 % of the time instead of 73: statistics of 8192 x 4096 x 65536 1237 -> 1347 TFLOP/s in a seconds-long loop (power-limited, at
// 1233 MHz instead of 1410; the library's product 1358 beside it), 1384 -> 1540 in a burst. 16 row tiles walked together instead of 8 give 3 %.
//
// Every wait is bounded, as in the other kernels (ptx.cuh).
#include "loss_products.hpp"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gemm_kernels.hpp"
#include "ptx.cuh"
#include "training_common.cuh"

namespace ftcuda {
namespace loss {
namespace {

constexpr std::uint32_t kBlockK = 64;  // 128 bytes, one swizzle row
constexpr std::uint32_t kTileN  = 256;
constexpr std::uint32_t kItemBlocks  = 12;  // of an item: what it costs beside its own
constexpr std::uint32_t kMostSplits  = 96;
constexpr std::uint32_t kMostWeightSplits = 16;
constexpr std::uint32_t kLaunchBlocks = 12;          // of one more launch
constexpr std::uint32_t kStreamSplits = 16;          // where the weight streams through; 96 are no faster there (1 x 512 x 131072 BF16: 183 us, 189)
constexpr std::uint64_t kStreamTokens = 400;         // at which the tensor cores take as long as HBM does (times an FP32 product's terms)
constexpr std::uint64_t kStreamBytes  = 64ULL << 20;  // half of L2
constexpr std::uint32_t kSumBlocks   = 16;
constexpr std::uint32_t kFp32Blocks  = 2;
constexpr std::uint32_t kTerms       = 6;         // of an FP32 product: which plane of A and of B, four bits for each term
constexpr std::uint32_t kTermsA      = 0x201100;
constexpr std::uint32_t kTermsB      = 0x021010;
constexpr int kStages           = 5;  // seven are no faster; what is left is the stores' L1
constexpr int kThreads          = 384;
constexpr int kOperandBytes     = 128 * 128;  // a CTA's share of A, and of a B of 256 columns
constexpr int kStageBytes       = 2 * kOperandBytes;
constexpr int kBarrierOffset    = kStages * kStageBytes;
constexpr int kScratchOffset    = kBarrierOffset + 256;
constexpr int kScratchRow       = 33;  // words: rows of 32 numbers that neither rows nor columns have bank conflicts in
constexpr int kScratchBytes     = 32 * kScratchRow * 4;  // of an epilogue warp
constexpr std::uint32_t kBoxBytes = 64 * 128;  // 64 rows of 128 bytes: one box of an MN-major operand

constexpr int kRegsLight = 72;   // producer, issuer (warpgroup 0)
constexpr int kRegsDrain = 216;  // epilogue (warpgroups 1, 2)
static_assert(128 * kRegsLight + 256 * kRegsDrain <= 168 * kThreads, "the CTA's register pool is what it was launched with");
constexpr int kProducerA     = 0;
constexpr int kIssuerWarp    = 1;
constexpr int kProducerB     = 2;
constexpr int kFirstEpilogue = 4;
constexpr std::uint32_t kTmemColumns = 512;

enum Mode : int { kStatistics, kKept, kSlopes, kGradients };
constexpr int smemBytes(int mode) { return kScratchOffset + 1024 + (mode == kGradients ? 8 * kScratchBytes : 0); }
static_assert(smemBytes(kGradients) <= 232448, "shared memory of one CTA");

struct Barriers {
    std::uint64_t full[kStages];  // used in the pair's first CTA
    std::uint64_t empty[kStages];
    std::uint64_t sum_full[2];
    std::uint64_t sum_empty[2];   // used in the pair's first CTA
    std::uint64_t flush;
    std::uint32_t tmem_base;
    int abort_flag;
};
static_assert(sizeof(Barriers) <= 256, "barrier block");

struct Problem {
    std::uint32_t rows;          // 0: the live rows
    std::uint32_t blocks;        // K blocks; 0: those of the live rows
    std::uint32_t columns, tile_n, tiles_n;
    std::uint32_t splits, blocks_per_split;
    std::uint32_t a_along_rows, b_along_rows;  // MN-major
};

struct ProductParams {
    Problem problem[2];
    std::uint32_t problems, band;
    std::uint32_t instruction;  // the operands' type
    std::uint32_t bf16, capacity;
    std::uint32_t terms;        // products for each block of K: 1, or kTerms
    std::uint32_t chunk;        // blocks of K between two readings of a sum
    std::uint32_t first;        // column of the vocabulary that column 0 is
    LiveRows rows;
    float2* partials;
    void* slopes;               // or what is kept
    void* own_slopes;
    std::uint64_t slopes_pitch, slopes_plane;
    float* sums;
    float* weight_sums;         // NULL: the weight's gradient is written as it is
    std::uint64_t sums_pitch;
    std::uint32_t weight_rows;
    std::uint32_t accumulate;
    std::uint32_t weight_problem;  // which of the problems is the weight's gradient
    void* weight_gradient;
    std::int64_t weight_gradient_pitch;
    std::uint32_t weight_fp32;
    std::uint32_t weight_vector;   // elements of it that one aligned store takes: 16, 8, or 1
    const float* upstream;         // NULL: 1
    int* status;
};

struct ProductMaps {
    CUtensorMap a[2], b[2];
};

struct Item {
    std::uint32_t problem, row, col, split, first_block, blocks;
};

// The launch's tiles, from the number of live rows.
struct Work {
    std::uint32_t tiles_m[2], blocks[2], items[2];
    // Every pair takes its share of the first problem's items and then of the second's. Where the first ones do not come out even, the
    // pairs from `late` on, which have one less of them, take `early` items of the second problem each meanwhile.
    std::uint32_t late, early;
};

// How long that takes, an item of the first problem taking `first`, one of the second `second`.
__host__ __device__ __forceinline__ std::uint64_t makespan(std::uint32_t first_items, std::uint32_t first, std::uint32_t second_items, std::uint32_t second, std::uint32_t pairs,
                                                           std::uint32_t early) {
    const std::uint32_t own = first_items / pairs, late = first_items % pairs, others = pairs - late;
    const std::uint64_t all   = static_cast<std::uint64_t>(early) * others;
    const std::uint32_t taken = all < second_items ? static_cast<std::uint32_t>(all) : second_items, rest = second_items - taken;
    const std::uint32_t before = (taken + others - 1) / others;
    const std::uint64_t most  = static_cast<std::uint64_t>(own + (late != 0 ? 1 : 0)) * first + static_cast<std::uint64_t>((rest + pairs - 1) / pairs) * second;
    const std::uint64_t least = static_cast<std::uint64_t>(own) * first + static_cast<std::uint64_t>(before + (rest > late ? (rest - late + pairs - 1) / pairs : 0)) * second;
    return most > least ? most : least;
}

// The better one of the two numbers of early items next to an even share.
__host__ __device__ __forceinline__ std::uint32_t earlyItems(std::uint32_t first_items, std::uint32_t first, std::uint32_t second_items, std::uint32_t second, std::uint32_t pairs) {
    if (second_items == 0 || first_items % pairs == 0) { return 0; }
    const std::uint32_t fewer = first / second;
    return makespan(first_items, first, second_items, second, pairs, fewer + 1) < makespan(first_items, first, second_items, second, pairs, fewer) ? fewer + 1 : fewer;
}

__device__ __forceinline__ Work workOf(const ProductParams& p, std::uint32_t live, std::uint32_t pairs) {
    live = max(live, 1U);
    Work w;
    w.items[1] = 0;
#pragma unroll
    for (std::uint32_t i = 0; i < 2; ++i) {
        if (i < p.problems) {
            const Problem& problem = p.problem[i];
            w.tiles_m[i]           = ((problem.rows != 0 ? problem.rows : live) + kTileRows - 1) / kTileRows;
            w.blocks[i]            = problem.blocks != 0 ? problem.blocks : (live + kBlockK - 1) / kBlockK;
            w.items[i]             = w.tiles_m[i] * problem.tiles_n * problem.splits;
        }
    }
    w.late  = w.items[0] % pairs;
    // (An item costs about kItemBlocks blocks' time beside its own.)
    const std::uint32_t first = p.problem[0].splits == 1 ? w.blocks[0] : p.problem[0].blocks_per_split;
    w.early                   = 0;
    if (w.items[1] != 0) {
        const std::uint32_t second = p.problem[1].splits == 1 ? w.blocks[1] : p.problem[1].blocks_per_split;
        w.early                    = earlyItems(w.items[0], first * p.terms + kItemBlocks, w.items[1], second * p.terms + kItemBlocks, pairs);
    }
    return w;
}

// The number of a pair's n-th item, or kNoItem.
constexpr std::uint32_t kNoItem = 0xFFFFFFFFU;
__device__ __forceinline__ std::uint32_t itemOf(const Work& work, std::uint32_t pair, std::uint32_t pairs, std::uint32_t n) {
    const std::uint32_t own = work.items[0] / pairs + (pair < work.late ? 1 : 0);
    if (n < own) { return pair + n * pairs; }
    n -= own;
    const std::uint32_t others = work.early * (pairs - work.late);  // taken early
    std::uint32_t item         = others + pair + n * pairs;
    if (pair >= work.late) {
        item = n < work.early ? pair - work.late + n * (pairs - work.late) : others + pair + (n - work.early) * pairs;
    }
    return item < work.items[1] ? work.items[0] + item : kNoItem;
}

__device__ __forceinline__ Item decode(const ProductParams& p, const Work& work, std::uint32_t item) {
    Item w;
    w.problem              = item < work.items[0] ? 0 : 1;
    const Problem& problem = p.problem[w.problem];
    if (w.problem != 0) { item -= work.items[0]; }
    const std::uint32_t tiles_m = w.problem != 0 ? work.tiles_m[1] : work.tiles_m[0];
    const std::uint32_t blocks  = w.problem != 0 ? work.blocks[1] : work.blocks[0];
    const std::uint32_t tiles   = tiles_m * problem.tiles_n;
    w.split                     = item / tiles;
    const std::uint32_t tile    = item - w.split * tiles;
    const std::uint32_t band    = tile / (p.band * problem.tiles_n);
    const std::uint32_t first   = band * p.band;
    const std::uint32_t rows    = min(p.band, tiles_m - first);
    const std::uint32_t rest    = tile - band * p.band * problem.tiles_n;
    w.row                       = (first + rest % rows) * kTileRows;
    w.col                       = rest / rows * problem.tile_n;
    w.first_block               = w.split * problem.blocks_per_split;
    // (Few live rows may leave a part nothing.)
    w.blocks                    = problem.splits == 1 ? blocks : w.first_block < blocks ? min(blocks - w.first_block, problem.blocks_per_split) : 0;
    return w;
}

struct Ring {
    std::uint32_t slot = 0, round = 0;
    __device__ __forceinline__ void next() {
        if (++slot == kStages) {
            slot = 0;
            ++round;
        }
    }
};

__device__ __forceinline__ std::uint32_t pack16(float low, float high, bool bf16) {
    if (bf16) {
        const __nv_bfloat162 pair = __floats2bfloat162_rn(low, high);
        return *reinterpret_cast<const std::uint32_t*>(&pair);
    }
    const __half2 pair = __floats2half2_rn(low, high);
    return *reinterpret_cast<const std::uint32_t*>(&pair);
}

// This thread's row of FP32 numbers as three BF16 matrices with room for whole tiles.
__device__ __forceinline__ void storePlanes(const ProductParams& p, std::uint32_t row, std::uint32_t col, std::uint32_t pieces, float scale, bool on, const float (&v)[128]) {
    unsigned char* const out = static_cast<unsigned char*>(p.slopes) + (static_cast<std::uint64_t>(row) * p.slopes_pitch + col) * 2;
#pragma unroll
    for (int j = 0; j < 128; j += 16) {
        if (j < 64 || pieces == 4) {
            std::uint32_t packed[kPlanes][8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float low[kPlanes], high[kPlanes];
                training::splitPlanes(on ? scale * v[j + 2 * i] : 0.0F, low);
                training::splitPlanes(on ? scale * v[j + 2 * i + 1] : 0.0F, high);
#pragma unroll
                for (std::uint32_t plane = 0; plane < kPlanes; ++plane) { packed[plane][i] = pack16(low[plane], high[plane], true); }
            }
#pragma unroll
            for (std::uint32_t plane = 0; plane < kPlanes; ++plane) { storeGlobal8(out + 2 * (plane * p.slopes_plane + j), packed[plane]); }
        }
    }
}

// This thread's row of a 16-bit matrix that has room for whole tiles; what lies beyond the columns is never fetched.
__device__ __forceinline__ void storeRow(const ProductParams& p, void* to, std::uint32_t row, std::uint32_t col, std::uint32_t pieces, float scale, bool on, bool bf16,
                                         const float (&v)[128]) {
    unsigned char* const out = static_cast<unsigned char*>(to) + (static_cast<std::uint64_t>(row) * p.slopes_pitch + col) * 2;
#pragma unroll
    for (int j = 0; j < 128; j += 16) {
        if (j < 64 || pieces == 4) {
            std::uint32_t packed[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) { packed[i] = on ? pack16(scale * v[j + 2 * i], scale * v[j + 2 * i + 1], bf16) : 0; }
            storeGlobal8(out + 2 * j, packed);
        }
    }
}

// What a warp does with 32 rows (`row`: this thread's) and 32 * pieces columns from `col` on, held in v.
template<bool kKeep>
__device__ __forceinline__ void finishStatistics(const ProductParams& p, const Item& w, std::uint32_t row, std::uint32_t col, std::uint32_t pieces,
                                                 std::uint32_t half, std::uint32_t live, float (&v)[128]) {
    const std::uint32_t columns = p.problem[0].columns;
    const std::int32_t at       = row < live ? p.rows.target[row] - static_cast<std::int32_t>(col) : -1;
    const bool here             = at >= 0 && at < static_cast<std::int32_t>(32 * pieces);
    // Rarely: a target lies among these columns.
    if (__any_sync(0xFFFFFFFFU, here)) {
        float picked = 0.0F;
#pragma unroll
        for (int j = 0; j < 128; ++j) { picked = j == at ? v[j] : picked; }
        if (here) { p.rows.picked[row] = picked; }
    }
    if (col + 32 * pieces > columns) {
#pragma unroll
        for (int j = 0; j < 128; ++j) { v[j] = col + j < columns ? v[j] : -INFINITY; }
    }
    // (Four chains each: there are two warps a scheduler to hide what an instruction takes.)
    float tops[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int j = 4; j < 128; ++j) {
        if (j < 64 || pieces == 4) { tops[j % 4] = fmaxf(tops[j % 4], v[j]); }
    }
    const float largest = fmaxf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), -INFINITY);  // not NaN
    const bool none  = largest == -INFINITY;  // and no reference to subtract; sums of nothing (or of NaN) come out
    const float base = none ? 0.0F : largest * kLog2E;
    float sum[4] = {0.0F, 0.0F, 0.0F, 0.0F};
#pragma unroll
    for (int j = 0; j < 128; ++j) {
        if (j < 64 || pieces == 4) {
            const float e = exp2Fast(fmaf(v[j], kLog2E, -base));
            sum[j % 4] += e;
            if (kKeep) { v[j] = e; }
        }
    }
    const std::uint32_t piece = 2 * (w.col / p.problem[0].tile_n) + half;
    p.partials[static_cast<std::uint64_t>(piece) * p.capacity + row] = make_float2(none ? -INFINITY : base, (sum[0] + sum[1]) + (sum[2] + sum[3]));
    if (kKeep && p.terms == 1) { storeRow(p, p.slopes, row, col, pieces, kKeptScale, true, false, v); }
    if (kKeep && p.terms != 1) {
        float* const out = static_cast<float*>(p.slopes) + static_cast<std::uint64_t>(row) * p.slopes_pitch + col;
#pragma unroll
        for (int j = 0; j < 128; j += 8) {
            if (j < 64 || pieces == 4) {
                float o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) { o[i] = v[j + i]; }
                storeGlobal8(out + j, o);
            }
        }
    }
}

__device__ __forceinline__ void finishSlopes(const ProductParams& p, std::uint32_t row, std::uint32_t col, std::uint32_t pieces, std::uint32_t live,
                                             float (&v)[128]) {
    const bool on            = row < live;
    const float scale        = on ? p.rows.scale[row] : 0.0F;
    const float lse2         = on ? p.rows.lse2[row] : 0.0F;
    const std::int32_t at    = on ? p.rows.target[row] - static_cast<std::int32_t>(p.first + col) : -1;
    const bool here          = at >= 0 && at < static_cast<std::int32_t>(32 * pieces);
#pragma unroll
    for (int j = 0; j < 128; ++j) { v[j] = exp2Fast(fmaf(v[j], kLog2E, -lse2)); }
    if (__any_sync(0xFFFFFFFFU, here)) {
#pragma unroll
        for (int j = 0; j < 128; ++j) { v[j] = j == at ? v[j] - 1.0F : v[j]; }
    }
    if (p.terms == 1) {
        if (p.slopes != nullptr) { storeRow(p, p.slopes, row, col, pieces, scale, on, p.bf16 != 0, v); }
        if (p.own_slopes != nullptr) { storeRow(p, p.own_slopes, row, col, pieces, on ? p.rows.own_scale[row] : 0.0F, on, p.bf16 != 0, v); }
    } else {
        storePlanes(p, row, col, pieces, scale, on, v);
    }
}

__device__ __forceinline__ void finishSums(const ProductParams& p, const Item& w, float* sums, std::uint32_t rows, bool accumulate, std::uint32_t row, std::uint32_t col,
                                           std::uint32_t pieces, float (&v)[128]) {
    float* const at = sums + (static_cast<std::uint64_t>(w.split) * rows + row) * p.sums_pitch + col;
#pragma unroll
    for (int j = 0; j < 128; j += 8) {
        if ((j < 64 || pieces == 4) && col + j < p.sums_pitch) {
            float o[8];
            if (accumulate) {
                loadGlobal8(at + j, o);
#pragma unroll
                for (int i = 0; i < 8; ++i) { o[i] += v[j + i]; }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) { o[i] = v[j + i]; }
            }
            storeGlobal8(at + j, o);
        }
    }
}

// A gradient whose rows no aligned store fits (an odd depth, say): 32 columns at a time are turned in shared memory, so that a warp writes neighbours. (A thread writing
// its own row element by element touches 32 rows with every store: a step of 72 x 2311 x 13632 FP16 took 502 us so and takes 140, of 1000 x 1001 x 20000 BF16 412 and 158.)
__device__ __forceinline__ void finishWeightTurned(const ProductParams& p, const Problem& problem, std::uint32_t row, std::uint32_t col, std::uint32_t pieces, float unit,
                                                   float* scratch, float (&v)[128]) {
    const std::uint32_t lane = threadIdx.x & 31, row0 = row - lane;
    const std::uint32_t rows = row0 < problem.rows ? min(32U, problem.rows - row0) : 0;
#pragma unroll
    for (std::uint32_t q = 0; q < 4; ++q) {
        if (q < pieces) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 32; ++j) { scratch[lane * kScratchRow + j] = unit * v[q * 32 + j]; }
            __syncwarp();
            const std::uint32_t at = col + q * 32 + lane;
            if (at < problem.columns) {
                for (std::uint32_t i = 0; i < rows; ++i) {
                    const float x            = scratch[i * kScratchRow + lane];
                    const std::int64_t place = static_cast<std::int64_t>(row0 + i) * p.weight_gradient_pitch + at;
                    if (p.weight_fp32 != 0) {
                        static_cast<float*>(p.weight_gradient)[place] = x;
                    } else {
                        static_cast<std::uint16_t*>(p.weight_gradient)[place] = static_cast<std::uint16_t>(pack16(x, 0.0F, p.bf16 != 0));
                    }
                }
            }
        }
    }
}

__device__ __forceinline__ void finishWeight(const ProductParams& p, const Problem& problem, std::uint32_t row, std::uint32_t col, std::uint32_t pieces,
                                             float unit, float (&v)[128]) {
    if (row >= problem.rows) { return; }
    if (p.weight_fp32 != 0) {
        float* const at = static_cast<float*>(p.weight_gradient) + static_cast<std::int64_t>(row) * p.weight_gradient_pitch + col;
#pragma unroll
        for (int j = 0; j < 128; j += 8) {
            if (j < 64 || pieces == 4) {
                float o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) { o[i] = unit * v[j + i]; }
                if (col + j < problem.columns) { storeGlobal8(at + j, o); }
            }
        }
        return;
    }
    unsigned char* const at = static_cast<unsigned char*>(p.weight_gradient) + (static_cast<std::int64_t>(row) * p.weight_gradient_pitch + col) * 2;
#pragma unroll
    for (int j = 0; j < 128; j += 16) {
        if (j < 64 || pieces == 4) {
            std::uint32_t packed[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) { packed[i] = pack16(unit * v[j + 2 * i], unit * v[j + 2 * i + 1], p.bf16 != 0); }
            if (p.weight_vector == 16) {
                if (col + j < problem.columns) { storeGlobal8(at + 2 * j, packed); }
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (col + j + 8 * i < problem.columns) {
                        *reinterpret_cast<uint4*>(at + 2 * j + 16 * i) = make_uint4(packed[4 * i], packed[4 * i + 1], packed[4 * i + 2], packed[4 * i + 3]);
                    }
                }
            }
        }
    }
}

template<int kMode>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
lossProduct(const __grid_constant__ ProductMaps maps, const __grid_constant__ ProductParams p) {
    extern __shared__ unsigned char smem_raw[];
    const std::uint32_t align_offset = (1024 - (smemAddress(smem_raw) & 1023)) & 1023;
    unsigned char* smem              = smem_raw + align_offset;
    Barriers* bars                   = reinterpret_cast<Barriers*>(smem + kBarrierOffset);
    volatile int* abort_flag         = &bars->abort_flag;
    const int warp                   = __shfl_sync(0xFFFFFFFFU, static_cast<int>(threadIdx.x >> 5), 0);  // known to be the warp's
    const int lane                   = threadIdx.x & 31;
    const std::uint32_t rank         = clusterCtaRank();
    const std::uint32_t pair         = blockIdx.x >> 1;
    const std::uint32_t pairs        = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbarrierInit(&bars->full[s], 1);
            mbarrierInit(&bars->empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbarrierInit(&bars->sum_full[s], 1);
            mbarrierInit(&bars->sum_empty[s], 16);
        }
        mbarrierInit(&bars->flush, 1);
        bars->abort_flag = 0;
        fenceBarrierInit();
        for (std::uint32_t i = 0; i < p.problems; ++i) {
            prefetchTensorMap(&maps.a[i]);
            prefetchTensorMap(&maps.b[i]);
        }
    }
    if (warp == kIssuerWarp) { tmemAllocatePair(&bars->tmem_base, kTmemColumns); }
    tcgen05FenceBeforeSync();
    __syncthreads();
    clusterBarrierArrive();
    clusterBarrierWait();
    tcgen05FenceAfterSync();
    const std::uint32_t tmem_base = bars->tmem_base;

    // Launched with programmatic stream serialization: what is above overlaps the predecessor's tail.
    gridDependencyWait();
    gridDependencyLaunchDependents();
    const std::uint32_t live = min(*p.rows.count, p.capacity);  // (never beyond, whatever stands there)
    const Work work          = workOf(p, live, pairs);

    if (warp >= kFirstEpilogue) {
        registersGrow<kRegsDrain>();
        const int e                   = warp - kFirstEpilogue;                    // 0..7
        const std::uint32_t half      = static_cast<std::uint32_t>(e >> 2);
        const std::uint32_t in_tile   = static_cast<std::uint32_t>(32 * (warp & 3));  // the tensor-memory lanes a warp can read
        const std::uint32_t tmem_row  = tmem_base + (in_tile << 16);
        const std::uint32_t sum_empty[2] = {mapToRank(&bars->sum_empty[0], 0), mapToRank(&bars->sum_empty[1], 0)};
        const float unit              = kMode != kGradients ? 1.0F : *p.rows.unit * (p.upstream != nullptr ? *p.upstream : 1.0F);
        std::uint32_t sums = 0;
        bool ok = true;
        for (std::uint32_t n = 0, item; ok && (item = itemOf(work, pair, pairs, n)) != kNoItem; ++n) {
            const Item w                 = decode(p, work, item);
            const Problem& problem       = p.problem[w.problem];
            const std::uint32_t pieces   = problem.tile_n / 64;  // of 32 columns, for this warp
            const std::uint32_t row      = w.row + rank * 128 + in_tile + lane;
            const std::uint32_t col      = w.col + half * 32 * pieces;
            float v[128];
#pragma unroll
            for (int j = 0; j < 128; ++j) { v[j] = 0.0F; }
            for (std::uint32_t kb = 0; kb < w.blocks; kb += min(p.chunk, w.blocks - kb), ++sums) {
                const std::uint32_t which = sums & 1;
                ok = mbarrierWait(&bars->sum_full[which], (sums >> 1) & 1, abort_flag);
                if (!ok) { break; }
                tcgen05FenceAfterSync();
#pragma unroll
                for (std::uint32_t q = 0; q < 4; ++q) {
                    if (q < pieces) {
                        float part[32];
                        tmemLoad32(tmem_row + which * kTileN + half * 32 * pieces + q * 32, part);
#pragma unroll
                        for (int j = 0; j < 32; ++j) { v[q * 32 + j] += part[j]; }
                    }
                }
                tcgen05FenceBeforeSync();
                __syncwarp();
                if (lane == 0) { mbarrierArriveCluster(sum_empty[which]); }
            }
            if (!ok) { break; }
            if (kMode == kStatistics) {
                finishStatistics<false>(p, w, row, col, pieces, half, live, v);
            } else if (kMode == kKept) {
                finishStatistics<true>(p, w, row, col, pieces, half, live, v);
            } else if (kMode == kSlopes) {
                finishSlopes(p, row, col, pieces, live, v);
            } else if (w.problem == p.weight_problem && p.weight_sums != nullptr) {
                finishSums(p, w, p.weight_sums, p.weight_rows, false, row, col, pieces, v);
            } else if (w.problem == p.weight_problem) {
                if (p.weight_vector != 1) {
                    finishWeight(p, problem, row, col, pieces, unit, v);
                } else {
                    finishWeightTurned(p, problem, row, col, pieces, unit, reinterpret_cast<float*>(smem + kScratchOffset + e * kScratchBytes), v);
                }
            } else {
                finishSums(p, w, p.sums, p.capacity, p.accumulate != 0, row, col, pieces, v);
            }
        }
        if (!ok) { *abort_flag = 1; }
    } else {
        registersShrink<kRegsLight>();
        if (warp == kProducerA || warp == kProducerB) {
            bool ok = true;
            if (lane == 0) {
                const bool second        = warp == kProducerB;
                const bool arms          = !second && rank == 0;
                unsigned char* const to  = smem + (second ? kOperandBytes : 0);
                const std::uint32_t full = mapToRank(&bars->full[0], 0);
                Ring ring;
                std::uint32_t filled = 0;
                for (std::uint32_t n = 0, item; ok && (item = itemOf(work, pair, pairs, n)) != kNoItem; ++n) {
                    // What does not change within an item is in registers before its K blocks: this loop has 512 cycles a block.
                    const Item w                 = decode(p, work, item);
                    const Problem& problem       = p.problem[w.problem];
                    const CUtensorMap* const map = second ? &maps.b[w.problem] : &maps.a[w.problem];
                    const std::uint32_t rows     = second ? problem.tile_n / 2 : 128;
                    const std::int32_t row       = static_cast<std::int32_t>((second ? w.col : w.row) + rank * rows);
                    const bool along             = (second ? problem.b_along_rows : problem.a_along_rows) != 0;
                    const bool two               = along && rows == 128;  // boxes: an MN-major one has 64 rows
                    const std::int32_t first     = static_cast<std::int32_t>(w.first_block * kBlockK);
                    const std::int32_t step_x = along ? 0 : static_cast<std::int32_t>(kBlockK), step_y = along ? static_cast<std::int32_t>(kBlockK) : 0;
                    const std::uint32_t bytes    = 2 * (kOperandBytes + problem.tile_n / 2 * 128);
                    std::int32_t x = along ? row : first, y = along ? first : row;
                    const std::uint32_t terms = p.terms, loads = w.blocks * terms, planes = terms == 1 ? 0 : second ? kTermsB : kTermsA;
                    std::uint32_t term        = 0;
                    for (std::uint32_t load = 0; load < loads; ++load, ++filled, ring.next()) {
                        const std::int32_t plane = static_cast<std::int32_t>(planes >> (4 * term) & 0xF);
                        ok = mbarrierWait(&bars->empty[ring.slot], (ring.round & 1) ^ 1, abort_flag);
                        if (!ok) { break; }
                        // The bytes of both CTAs count on the first CTA's barrier, which that CTA arms. (The other's
                        // may land first: the phase cannot complete before it has been armed.)
                        if (arms) { mbarrierArriveExpectTx(&bars->full[ring.slot], bytes); }
                        tmaLoad3dPair(to + ring.slot * kStageBytes, map, full + ring.slot * 8, x, y, plane);
                        if (two) { tmaLoad3dPair(to + ring.slot * kStageBytes + kBoxBytes, map, full + ring.slot * 8, x + 64, y, plane); }
                        if (++term == terms) {
                            term = 0;
                            x += step_x;
                            y += step_y;
                        }
                    }
                }
                // Neither CTA leaves before the last commits have arrived on its barriers.
                for (std::uint32_t i = 0; i < kStages && i < filled && ok; ++i) {
                    const std::uint32_t use = filled - 1 - i;
                    ok = mbarrierWait(&bars->empty[use % kStages], (use / kStages) & 1, abort_flag);
                }
                if (!ok) { *abort_flag = 1; }
            }
            __syncwarp();
        } else if (warp == kIssuerWarp && rank == 0) {
            // The whole warp goes through the loop and one thread issues: descriptors that are the warp's stay in uniform registers.
            const bool leads               = electOne();
            const std::uint64_t stage_step = kStageBytes >> 4;
            const std::uint32_t base       = smemAddress(smem);
            Ring ring;
            std::uint32_t sums = 0;
            bool ok            = true;
            for (std::uint32_t n = 0, item; ok && (item = itemOf(work, pair, pairs, n)) != kNoItem; ++n) {
                const Item w           = decode(p, work, item);
                const Problem& problem = p.problem[w.problem];
                const bool a_mn = problem.a_along_rows != 0, b_mn = problem.b_along_rows != 0;
                // Sixteen of K are 32 bytes of a K-major tile's rows, or sixteen rows of an MN-major one.
                const std::uint64_t a0 = a_mn ? umaDescriptorMn128(base, kBoxBytes) : umaDescriptorK128(base);
                const std::uint64_t b0 = b_mn ? umaDescriptorMn128(base + kOperandBytes, kBoxBytes) : umaDescriptorK128(base + kOperandBytes);
                const std::uint64_t a_step = a_mn ? 16 * 128 >> 4 : 2, b_step = b_mn ? 16 * 128 >> 4 : 2;
                const std::uint32_t instruction =
                    p.instruction | umaInstructionF16(kTileRows, problem.tile_n) | (a_mn ? kUmaAMnMajor : 0) | (b_mn ? kUmaBMnMajor : 0);
                for (std::uint32_t kb = 0, blocks; kb < w.blocks && ok; kb += blocks, ++sums) {
                    blocks                    = min(p.chunk, w.blocks - kb);
                    const std::uint32_t loads = blocks * p.terms;
                    const std::uint32_t which = sums & 1;
                    const std::uint32_t d     = tmem_base + which * kTileN;
                    ok = mbarrierWait(&bars->sum_empty[which], ((sums >> 1) & 1) ^ 1, abort_flag);
                    if (!ok) { break; }
                    tcgen05FenceAfterSync();
                    for (std::uint32_t load = 0; load < loads; ++load, ring.next()) {
                        ok = mbarrierWait(&bars->full[ring.slot], ring.round & 1, abort_flag);
                        if (!ok) { break; }
                        tcgen05FenceAfterSync();
                        const std::uint64_t a = a0 + ring.slot * stage_step, b = b0 + ring.slot * stage_step;
                        if (leads) {
#pragma unroll
                            for (std::uint32_t step = 0; step < kBlockK / 16; ++step) {
                                umaF16Pair(d, a + step * a_step, b + step * b_step, instruction, load != 0 || step != 0 ? 1U : 0U);
                            }
                            umaCommitPair(&bars->empty[ring.slot]);
                        }
                        __syncwarp();
                    }
                    if (!ok) { break; }
                    if (leads) { umaCommitPair(&bars->sum_full[which]); }
                    __syncwarp();
                }
            }
            if (!ok && leads) {
                *abort_flag = 1;
                // Let MMAs already issued finish before tensor memory is freed.
                umaCommitPair(&bars->flush);
                int never = 0;
                mbarrierWait(&bars->flush, 0, &never);
            }
            __syncwarp();
        }
    }

    __syncthreads();
    if (*abort_flag != 0) {
        if (threadIdx.x == 0) {
            if (p.status != nullptr) { *p.status = 2; }
            // Copies that were armed but never consumed may still be landing (their bytes count on the
            // first CTA's barriers; the second waits for the first below).
            int never = 0;
            for (int s = 0; s < kStages && rank == 0; ++s) {
                mbarrierWait(&bars->full[s], 0, &never);
                mbarrierWait(&bars->full[s], 1, &never);
            }
        }
        __syncthreads();
    }
    tcgen05FenceBeforeSync();
    clusterBarrierArrive();
    clusterBarrierWait();
    if (warp == kIssuerWarp) {
        tcgen05FenceAfterSync();
        tmemFreePair(tmem_base, kTmemColumns);
    }
}

// ---------------------------------------------------------------- host

std::uint32_t divideUp(std::uint32_t x, std::uint32_t y) { return (x + y - 1) / y; }

// 128 columns where that is all there are: B's tile is half as wide then.
std::uint32_t tileColumns(std::uint32_t columns) { return columns <= 128 ? 128 : kTileN; }

// Of the logits: and where that does not give a pair of SMs two tiles.
std::uint32_t logitTileColumns(std::uint32_t columns, std::uint32_t capacity, int sms) {
    const std::uint64_t tiles = static_cast<std::uint64_t>(capacity / kTileRows) * divideUp(columns, kTileN);
    return 2 * tiles <= static_cast<std::uint64_t>(std::max(1, sms / 2)) ? 128 : tileColumns(columns);
}

// An operand whose rows (of the product) are `rows` and whose depth is `k`: neighbours along K, or along the rows.
bool encodeOperand(CUtensorMap* map, const ProductCall& call, Matrix16 matrix, bool along_rows, std::uint32_t rows, std::uint32_t k, std::uint32_t tile_rows) {
    const std::uint64_t planes = call.planes ? kPlanes : 1, apart = call.planes ? matrix.plane * 2 : matrix.pitch * 2;
    return along_rows ? encodeMap16(map, call.bf16, matrix.at, rows, k, planes, matrix.pitch * 2, apart, 64, call.message, call.message_capacity)
                      : encodeMap16(map, call.bf16, matrix.at, k, rows, planes, matrix.pitch * 2, apart, tile_rows, call.message, call.message_capacity);
}

template<int kMode> cudaError_t launch(const ProductCall& call, const ProductMaps& maps, const ProductParams& p, std::uint64_t items) {
    cudaError_t error = cudaFuncSetAttribute(lossProduct<kMode>, cudaFuncAttributeMaxDynamicSharedMemorySize, smemBytes(kMode));
    if (error != cudaSuccess) { return error; }
    const std::uint64_t pairs = std::max<std::uint64_t>(1, std::min<std::uint64_t>(static_cast<std::uint64_t>(call.sms) / 2, items));
    return training::launchKernel(!call.starts, lossProduct<kMode>, dim3(static_cast<unsigned>(2 * pairs)), dim3(kThreads), smemBytes(kMode), call.stream, maps, p);
}

ProductParams paramsFor(const ProductCall& call) {
    ProductParams p{};
    p.problems       = 1;
    p.band           = 16;
    p.instruction    = call.bf16 ? kUmaBf16 : 0;
    p.bf16           = call.bf16 ? 1 : 0;
    p.terms          = call.planes ? kTerms : 1;
    p.chunk          = call.planes ? kFp32Blocks : kSumBlocks;
    p.capacity       = call.capacity;
    p.rows           = call.rows;
    p.status         = call.status;
    p.weight_problem = 2;
    return p;
}

// Z = H W^T over `columns` rows of the weight.
bool describeLogits(const ProductCall& call, Matrix16 weight, std::uint32_t columns, ProductMaps& maps, ProductParams& p) {
    Problem& problem          = p.problem[0];
    problem.columns           = columns;
    problem.tile_n            = logitTileColumns(columns, call.capacity, call.sms);
    problem.tiles_n           = divideUp(columns, problem.tile_n);
    problem.blocks            = divideUp(call.depth, kBlockK);
    problem.splits            = 1;
    problem.blocks_per_split  = problem.blocks;
    return encodeOperand(&maps.a[0], call, call.hidden, false, call.capacity, call.depth, 128) &&
           encodeOperand(&maps.b[0], call, weight, false, columns, call.depth, problem.tile_n / 2);
}

}  // namespace

std::uint32_t statisticsWidth(std::uint32_t columns, std::uint32_t capacity, int sms) { return logitTileColumns(columns, capacity, sms) / 2; }
std::uint32_t statisticsPieces(std::uint32_t columns, std::uint32_t capacity, int sms) { return 2 * divideUp(columns, logitTileColumns(columns, capacity, sms)); }

cudaError_t launchStatistics(const ProductCall& call, Matrix16 weight, std::uint32_t vocabulary, float2* partials) {
    ProductMaps maps;
    ProductParams p = paramsFor(call);
    p.partials      = partials;
    if (!describeLogits(call, weight, vocabulary, maps, p)) { return cudaErrorInvalidValue; }
    return launch<kStatistics>(call, maps, p, static_cast<std::uint64_t>(call.capacity / kTileRows) * p.problem[0].tiles_n);
}

cudaError_t launchKept(const ProductCall& call, Matrix16 weight, std::uint32_t vocabulary, float2* partials, void* kept, std::uint64_t kept_pitch) {
    ProductMaps maps;
    ProductParams p = paramsFor(call);
    p.partials      = partials;
    p.slopes        = kept;
    p.slopes_pitch  = kept_pitch;
    if (!describeLogits(call, weight, vocabulary, maps, p)) { return cudaErrorInvalidValue; }
    return launch<kKept>(call, maps, p, static_cast<std::uint64_t>(call.capacity / kTileRows) * p.problem[0].tiles_n);
}

cudaError_t launchSlopes(const ProductCall& call, Matrix16 weight, std::uint32_t first, std::uint32_t columns, void* slopes, void* own_slopes, std::uint64_t slopes_pitch,
                         std::uint64_t slopes_plane) {
    ProductMaps maps;
    ProductParams p = paramsFor(call);
    p.first         = first;
    p.slopes        = slopes;
    p.own_slopes    = own_slopes;
    p.slopes_pitch  = slopes_pitch;
    p.slopes_plane  = slopes_plane;
    if (!describeLogits(call, weight, columns, maps, p)) { return cudaErrorInvalidValue; }
    return launch<kSlopes>(call, maps, p, static_cast<std::uint64_t>(call.capacity / kTileRows) * p.problem[0].tiles_n);
}

// The sum over the columns is cut into as many parts as let both gradients' items end soonest (all tokens taken for live), a part's way through memory and
// back counted as well. Where the weight streams through (too large for L2, and too few tokens to be bound by anything else), into as many as make two items
// for each pair of SMs, so that all of them fetch it. Measured, a step, always the latter / as here: 700 x 700 x 3000 FP32 133 / 104 us, 1024 x 600 x 9000 FP32 250 / 224,
// 4096 x 512 x 32768 BF16 471 / 445; with 16 parts at most, 256 x 104 x 99422 FP32 331, with up to 96 267; 257 x 4096 x 131072 BF16 920, and 1016 where the items alone decide, 64 x 2048 x 50257 205 and 218.
// The weight's gradient is cut over the tokens where its items are few and long (many tokens, a small vocabulary), against a launch that adds the parts up: a step of
// 7424 x 432 x 1526 FP32 320 us, 228 so, of 16384 x 1024 x 500 BF16 224 and 183, of 4000 x 200 x 900 FP16 70 and 56.
GradientSplits gradientSplits(std::uint32_t tokens, std::uint32_t depth, std::uint32_t columns, bool planes, int sms) {
    const std::uint32_t across = divideUp(depth, tileColumns(depth)), tiles = divideUp(tokens, kTileRows) * across;
    const std::uint32_t pairs  = static_cast<std::uint32_t>(std::max(1, sms / 2));
    const std::uint32_t blocks = divideUp(columns, kBlockK), rows = divideUp(tokens, kBlockK), terms = planes ? kTerms : 1;
    if (static_cast<std::uint64_t>(tokens) * terms <= kStreamTokens && static_cast<std::uint64_t>(columns) * depth * 2 * (planes ? kPlanes : 1) > kStreamBytes) {
        const std::uint32_t wanted = std::min({std::max(1U, blocks / 8), kStreamSplits, std::max(1U, 2 * pairs / tiles)});
        return {divideUp(blocks, divideUp(blocks, wanted)), 1};
    }
    const std::uint32_t weight_items = divideUp(columns, kTileRows) * across;
    const std::uint64_t apart  = static_cast<std::uint64_t>(tokens) * depth >> 19;  // a block's 512 cycles are the time of 2^21 bytes or so
    const std::uint64_t weight_apart = (static_cast<std::uint64_t>(columns) * depth >> 19) + 1;
    GradientSplits best        = {1, 1};
    std::uint64_t least        = ~std::uint64_t{0};
    const std::uint32_t most   = 2 * weight_items <= pairs ? std::min(rows, kMostWeightSplits) : 1;
    for (std::uint32_t parts = 1; parts <= most; parts *= 2) {
        const std::uint32_t weight = divideUp(rows, parts) * terms + kItemBlocks;
        const std::uint64_t extra  = parts == 1 ? 0 : parts * weight_apart + kLaunchBlocks;
        std::uint32_t before       = 0;
        // (All numbers up to eight, then about every eighth part more: the host has this to do in every call.)
        for (std::uint32_t wanted = 1; wanted <= std::min(blocks, kMostSplits); wanted += std::max(1U, wanted / 8)) {
            const std::uint32_t each = divideUp(blocks, wanted), splits = divideUp(blocks, each);  // none of them empty
            if (splits == before) { continue; }
            before                   = splits;
            const std::uint32_t part = each * terms + kItemBlocks, items = weight_items * parts;
            std::uint64_t time       = makespan(tiles * splits, part, items, weight, pairs, earlyItems(tiles * splits, part, items, weight, pairs)) + splits * apart + extra;
            time += parts == 1 ? 0 : time / 8;  // (what is cut has to be well ahead: 5000 x 300 x 4000 FP32 289 us as one, 299 in two parts)
            if (time < least) {
                least = time;
                best  = {splits, parts};
            }
        }
    }
    return best;
}

cudaError_t launchGradients(const ProductCall& call, Matrix16 weight, std::uint32_t columns, Matrix16 slopes, const Gradients& gradients) {
    ProductMaps maps;
    ProductParams p = paramsFor(call);
    p.problems      = 0;
    p.upstream      = gradients.upstream;
    std::uint64_t items        = 0;
    const std::uint32_t tile_n = tileColumns(call.depth), tiles_n = divideUp(call.depth, tile_n);
    bool encoded = true;
    if (gradients.sums != nullptr) {
        Problem& problem          = p.problem[p.problems];
        problem.columns           = call.depth;
        problem.tile_n            = tile_n;
        problem.tiles_n           = tiles_n;
        problem.blocks            = divideUp(columns, kBlockK);
        problem.blocks_per_split  = divideUp(problem.blocks, gradients.splits);
        problem.splits            = divideUp(problem.blocks, problem.blocks_per_split);
        problem.b_along_rows      = 1;
        p.sums                    = gradients.sums;
        p.sums_pitch              = gradients.sums_pitch;
        p.accumulate              = gradients.accumulate ? 1 : 0;
        const Matrix16 own = gradients.own_slopes != nullptr ? Matrix16{gradients.own_slopes, slopes.pitch, slopes.plane} : slopes;
        encoded = encodeOperand(&maps.a[p.problems], call, own, false, call.capacity, columns, 128) &&
                  encodeOperand(&maps.b[p.problems], call, weight, true, call.depth, columns, 64);
        items += static_cast<std::uint64_t>(call.capacity / kTileRows) * tiles_n * problem.splits;
        ++p.problems;
    }
    if (encoded && gradients.weight_gradient != nullptr) {
        Problem& problem          = p.problem[p.problems];
        problem.rows              = columns;
        problem.columns           = call.depth;
        problem.tile_n            = tile_n;
        problem.tiles_n           = tiles_n;
        problem.splits            = gradients.weight_sums != nullptr ? gradients.weight_splits : 1;
        problem.blocks_per_split  = divideUp(call.capacity / kBlockK, problem.splits);
        p.weight_sums             = gradients.weight_sums;
        p.weight_rows             = gradients.weight_rows;
        p.sums_pitch              = gradients.sums_pitch;
        problem.a_along_rows      = 1;
        problem.b_along_rows      = 1;
        p.weight_problem          = p.problems;
        p.weight_gradient         = gradients.weight_gradient;
        p.weight_gradient_pitch   = gradients.weight_gradient_pitch;
        p.weight_fp32             = gradients.weight_gradient_fp32 ? 1 : 0;
        const std::uint32_t bytes = gradients.weight_gradient_fp32 ? 4 : 2;
        const auto fits = [&](std::uint32_t n) {
            return call.depth % n == 0 && gradients.weight_gradient_pitch % n == 0 && training::aligned(gradients.weight_gradient, bytes * n);
        };
        p.weight_vector = !gradients.weight_gradient_fp32 && fits(16) ? 16 : fits(8) ? 8 : 1;
        encoded = encodeOperand(&maps.a[p.problems], call, slopes, true, columns, call.capacity, 128) &&
                  encodeOperand(&maps.b[p.problems], call, call.hidden, true, call.depth, call.capacity, 64);
        items += static_cast<std::uint64_t>(divideUp(columns, kTileRows)) * tiles_n * problem.splits;
        ++p.problems;
    }
    if (!encoded) { return cudaErrorInvalidValue; }
    if (p.problems == 0) { return cudaSuccess; }
    return launch<kGradients>(call, maps, p, items);
}

}  // namespace loss
}  // namespace ftcuda
