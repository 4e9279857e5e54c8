// The products of the linear cross entropy on the tensor cores (loss_products.cu), as linear_cross_entropy.cu calls them.
#ifndef FTCUDA_LOSS_PRODUCTS_HPP_
#define FTCUDA_LOSS_PRODUCTS_HPP_

#include <cuda_runtime_api.h>

#include <cstddef>
#include <cstdint>

namespace ftcuda {
namespace loss {

constexpr std::uint32_t kTileRows = 256;  // rows of a CTA pair's tile; the live tokens' arrays are filled up to a multiple of it
constexpr float kLog2E            = 1.4426950408889634F;
constexpr float kLn2              = 0.6931471805599453F;

// The tokens that have a target, in their order. Behind the last one, up to a multiple of kTileRows (one at least), stand
// neutral rows: hidden state 0, target -1, scale 0.
struct LiveRows {
    std::uint32_t* count;
    float* unit;            // what a sum of products of slopes is multiplied by in the end
    std::int32_t* token;    // the token a row is of
    std::int32_t* target;   // its column, -1 for none, kBadTarget for one outside of the vocabulary
    float* scale;           // upstream gradient of the row's loss over `unit`
    float* lse2;            // log2 of the row's sum of exponentials
    float* picked;          // the logit of the target
    float* own_scale;       // FP16, an upstream gradient for each token: the row's scale for the hidden states' gradient, and ...
    float* own_unit;        // ... what its sum is multiplied by in the end; NULL where `scale` and `unit` do for both gradients
};
constexpr std::int32_t kBadTarget = -2;

// A matrix of 16-bit elements in memory, rows of neighbours; or an FP32 matrix as three of them, whose sum it is (kPlanes).
struct Matrix16 {
    const void* at;
    std::uint64_t pitch;  // elements between rows
    std::uint64_t plane;  // elements between matrices; any for one
};

// An FP32 number is the sum of three BF16 ones to within its own rounding: x = h + m + l, h = bf16(x), m = bf16(x - h), l = bf16(x - h - m), whatever
// its exponent. Of the nine products of two such sums, six are 2^-16 or more of the whole.
constexpr std::uint32_t kPlanes = 3;

struct ProductCall {
    bool bf16;
    bool planes;              // FP32 operands, as kPlanes BF16 matrices each; the slopes come and go the same way, all other results are FP32
    std::uint32_t capacity;   // rows that the live arrays have room for, a multiple of kTileRows
    std::uint32_t depth;      // elements of a hidden state
    LiveRows rows;
    Matrix16 hidden;          // [capacity][depth]: the live rows' hidden states
    int* status;
    int sms;
    cudaStream_t stream;
    char* message;
    std::size_t message_capacity;
    bool starts;              // a call with this product: an ordinary launch, which waits for all that came before in the stream
};

// Columns of the vocabulary that one partial result of the statistics covers, and how many of those there are.
std::uint32_t statisticsWidth(std::uint32_t columns, std::uint32_t capacity, int sms);
std::uint32_t statisticsPieces(std::uint32_t columns, std::uint32_t capacity, int sms);

// For every live row and piece of columns: {largest logit times log2 e, sum of 2^(logit log2 e - that)} to
// partials[piece][capacity]; and the target's logit to rows.picked.
cudaError_t launchStatistics(const ProductCall& call, Matrix16 weight, std::uint32_t vocabulary, float2* partials);

// The same, and kept[row][column] = 2^(logit log2 e - its piece's largest): FP32 for FP32 operands, else times kKeptScale in FP16 whatever the
// operands' type: against the largest of its piece a number needs no more range, and BF16 would round 2^3 times as much. The pitch is a multiple of 256.
constexpr float kKeptScale = 8192.0F;
cudaError_t launchKept(const ProductCall& call, Matrix16 weight, std::uint32_t vocabulary, float2* partials, void* kept, std::uint64_t kept_pitch);

// slopes[row][column - first] = scale (2^(logit log2 e - lse2) - [column is the target]) for `columns` columns from `first` on;
// `weight` starts at row `first`. The pitch is a multiple of 256. own_slopes: the same with rows.own_scale. Either may be NULL.
cudaError_t launchSlopes(const ProductCall& call, Matrix16 weight, std::uint32_t first, std::uint32_t columns, void* slopes, void* own_slopes, std::uint64_t slopes_pitch,
                         std::uint64_t slopes_plane);

// How many parts the sums are cut into: over `columns` columns for the gradient of the hidden states (over fewer columns
// launchGradients may fill fewer of them, never more), and over the tokens for that of the weight.
struct GradientSplits {
    std::uint32_t hidden, weight;
};
GradientSplits gradientSplits(std::uint32_t tokens, std::uint32_t depth, std::uint32_t columns, bool planes, int sms);

struct Gradients {
    // hidden: sums[split][capacity][pitch] (+)= slopes (own_slopes, where there are some) times weight; NULL when not wanted.
    float* sums;
    const void* own_slopes;
    std::uint64_t sums_pitch;  // a multiple of 8
    std::uint32_t splits;
    bool accumulate;
    // weight: rows of the piece = unit * slopes^T times hidden; NULL when not wanted.
    void* weight_gradient;
    std::int64_t weight_gradient_pitch;
    bool weight_gradient_fp32;  // or of the operands' type
    const float* upstream;      // a number that the weight's gradient is multiplied by as well; NULL: 1
    // With weight_splits > 1 its parts are left in weight_sums[split][weight_rows][sums_pitch] instead, without either factor.
    float* weight_sums;
    std::uint32_t weight_splits, weight_rows;  // rows: a multiple of kTileRows
};
cudaError_t launchGradients(const ProductCall& call, Matrix16 weight, std::uint32_t columns, Matrix16 slopes, const Gradients& gradients);

}  // namespace loss
}  // namespace ftcuda

#endif
