/*
 * ftcuda/training.h -- what a training step does around its products: the loss over a large
 * vocabulary, the experts' router, the gradients' norm.
 *
 * Same manner as ftcuda/ftcuda.h: plain pointers, integers and fixed-size structs; no C++ types, no
 * exceptions; 0 = success, nonzero = failure with a NUL-terminated reason in the caller's message
 * buffer (when one is given). Every call checks its arguments on the host, enqueues on `stream` and returns
 * without synchronising; nothing is allocated, so calls can be captured into a CUDA graph. The workspace
 * belongs to one call at a time: calls that can overlap on the GPU need one each. `device` must be the calling
 * thread's current device. The reference has none of these operators.
 */
#ifndef FTCUDA_TRAINING_H_
#define FTCUDA_TRAINING_H_

#include <ftcuda/ftcuda.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types, with the values of FTrainNumericType (flash_train/common.h). */
enum {
    FTCUDA_ELEMENT_FP32 = 4,
    FTCUDA_ELEMENT_FP16 = 7,
    FTCUDA_ELEMENT_BF16 = 8,
};

/* ---- the cross entropy of a product with a large vocabulary ---- */

enum {
    FTCUDA_REDUCTION_NONE = 0, /* a loss for each token */
    FTCUDA_REDUCTION_MEAN = 1, /* their sum over the number of tokens that have a target; 0 where none has */
    FTCUDA_REDUCTION_SUM  = 2,
};

/*
 * logits[t][v] = hidden[t] . weight[v],  loss[t] = log(sum_v exp(logits[t][v])) - logits[t][target[t]].
 * The two calls below never have all logits in memory: a piece of the vocabulary's gradients of them at a time is in the backward call, and a piece of FP32 logits in the forward
 * call where FP32 operands go through the library's products. A step call has a number for each logit: its exponential, then its gradient (FP32 operands that go through the library's
 * products: the logit, then its gradient), which are kept from the loss to the gradients; at most 2 GiB.
 *   - hidden [tokens][depth], weight [vocabulary][depth]: unit stride along the depth, the others any that keep rows apart; both
 *     of one type. BF16 and FP16 are multiplied by the tensor cores with FP32 sums; FP32 to FP32's precision, as sums of three BF16 matrices (which
 *     the workspace then holds, six bytes an element of the weight) or by the library's FP32 products, whichever is faster for the sizes.
 *   - target [tokens]: INT64. A token whose target is ignore_index takes no part: its loss and gradient are 0, whatever its hidden
 *     state holds, and but for the library's FP32 products nothing is computed for it. Any other target outside of [0, vocabulary) makes the token's loss
 *     NaN, and the gradients too.
 *   - infinities and NaN in what takes part reach the token's loss and the gradients as NaN (a logit of -inf is a probability of 0).
 *   - a gradient's rounding: with BF16 and FP16 operands the logits' gradients are rounded to that type before they are
 *     multiplied, at a scale that keeps FP16's range, and the products' sums once at the end. Without reduction that scale is each token's own for its row of the hidden states'
 *     gradient; the weight's gradient, a sum over tokens, has one for all of them, at which a logit's gradient is off by up to 2^-38 of the largest upstream one in FP16. In the step call their exponentials are FP16 before that,
 *     against the largest of 64 or 128 neighbours.
 * Sums are in an order that depends on the sizes and on which tokens take part alone: equal calls give equal bits.
 */
typedef struct {
    const void* hidden;
    const void* weight;
    const int64_t* target;
    uint64_t tokens, vocabulary, depth;
    int64_t hidden_row_stride, weight_row_stride;
    int64_t ignore_index;
    int32_t element;
    int32_t reduction;
    int32_t device;
} FtcudaLinearCrossEntropy;

/* Bytes of workspace that the forward (backward = 0) or the backward call needs. */
FTCUDA_API int ftcuda_linear_cross_entropy_workspace_bytes(const FtcudaLinearCrossEntropy* problem, int backward, uint64_t* workspace_bytes, char* message,
                                                           size_t message_capacity);

/* loss: FP32, one number, or [tokens] without reduction; lse: FP32 [tokens], the logarithm of each token's sum (0 for a token that takes no
 * part), which the backward call wants back. The workspace starts at a multiple of 256. */
FTCUDA_API int ftcuda_linear_cross_entropy(const FtcudaLinearCrossEntropy* problem, float* loss, float* lse, void* workspace, uint64_t workspace_bytes,
                                           void* stream, char* message, size_t message_capacity);

/*
 * The gradients of hidden and weight, each of the operands' type and dense along the depth; either may be NULL (not wanted).
 * grad_loss: FP32 on the device, in the loss's shape. They are written, not added to. From its first byte to its last one, a gradient's memory may
 * not meet the other's or an operand's (refused).
 */
FTCUDA_API int ftcuda_linear_cross_entropy_backward(const FtcudaLinearCrossEntropy* problem, const float* lse, const float* grad_loss, void* grad_hidden,
                                                    int64_t grad_hidden_row_stride, void* grad_weight, int64_t grad_weight_row_stride,
                                                    void* workspace, uint64_t workspace_bytes, void* stream, char* message,
                                                    size_t message_capacity);

/* ---- the norm over many tensors, and clipping ---- */

/*
 * One gradient: `rows` rows of `cols` neighbouring elements, `row_stride` elements apart (a dense tensor of any rank is one
 * row). `out` is where ftcuda_gradient_clip writes it, in the same shape; it may be `data` itself (same
 * type, same stride), and ftcuda_gradient_norm does not look at it. No alignment beyond the element's own is needed.
 */
typedef struct {
    const void* data;
    void* out;
    uint64_t rows, cols;
    int64_t row_stride, out_row_stride;
    int32_t element, out_element;
} FtcudaGradient;

enum {
    FTCUDA_NORM_2   = 0, /* sqrt(sum x^2) */
    FTCUDA_NORM_INF = 1, /* max |x|       */
};

/* Bytes of workspace that either call needs for `count` gradients. */
FTCUDA_API uint64_t ftcuda_gradient_norm_workspace_bytes(uint64_t count);

/*
 * *norm (one FP32 number on the device) = the norm over all elements of all gradients; 0 for none. Squares are summed in 64 bits
 * (in 32 within a few neighbouring elements, where none is so large or small that its square would leave FP32's range), in an
 * order that depends on the sizes alone, so equal calls give equal bits. NaN and infinities propagate.
 * Any number of gradients; a tensor that is listed twice counts twice.
 */
FTCUDA_API int ftcuda_gradient_norm(const FtcudaGradient* gradients, uint64_t count, int norm_kind, float* norm, int32_t device,
                                    void* workspace, uint64_t workspace_bytes, void* stream, char* message,
                                    size_t message_capacity);

/*
 * The norm as above, and out = data * min(1, max_norm / (norm + 1e-6)), the factor rounded to FP32 once and the product rounded
 * once to the output's type. Where that factor is 1, gradients that are their own `out` are left alone, without being
 * written. A norm that is not a number makes every element NaN; an infinite one makes the finite elements 0 and the others NaN (all of them NaN where
 * max_norm is infinite too). max_norm >= 0.
 * No element may be written that another gradient reads or writes (refused where addresses, sizes and strides
 * show it).
 */
FTCUDA_API int ftcuda_gradient_clip(const FtcudaGradient* gradients, uint64_t count, int norm_kind, double max_norm, float* norm,
                                    int32_t device, void* workspace, uint64_t workspace_bytes, void* stream, char* message,
                                    size_t message_capacity);

/*
 * out = data * *factor (one FP32 on the device), rounded once. Where the factor is 1, gradients that are their own `out` are left alone, without
 * being written. Needs no workspace; the rest as for ftcuda_gradient_clip.
 */
FTCUDA_API int ftcuda_gradient_scale(const FtcudaGradient* gradients, uint64_t count, const float* factor, int32_t device, void* stream,
                                     char* message, size_t message_capacity);

/*
 * The loss, and the gradients for an upstream gradient of 1, in one call that computes the logits once: three quarters of the work of the
 * two calls above. Their exponentials (FP32: the logits, or exponentials and slopes, 10 bytes each) are in the workspace meanwhile. With a reduction only, and
 * only where they take at most 2 GiB; ftcuda_linear_cross_entropy_step_workspace_bytes answers with a failure where that is not so.
 * grad_element: the operands' type, or FP32, for a caller that multiplies by an upstream gradient afterwards and wants nothing rounded (or, with
 * FP16, lost) before. Either gradient may be NULL.
 */
FTCUDA_API int ftcuda_linear_cross_entropy_step_workspace_bytes(const FtcudaLinearCrossEntropy* problem, uint64_t* workspace_bytes, char* message,
                                                                size_t message_capacity);
FTCUDA_API int ftcuda_linear_cross_entropy_step(const FtcudaLinearCrossEntropy* problem, float* loss, int32_t grad_element, void* grad_hidden,
                                                int64_t grad_hidden_row_stride, void* grad_weight, int64_t grad_weight_row_stride,
                                                void* workspace, uint64_t workspace_bytes, void* stream, char* message,
                                                size_t message_capacity);

/*
 * The step call in two: the loss first, and the gradients when the upstream gradient (*grad_loss, FP32 on the device) is known, of the operands' type: FP32
 * sums times the upstream gradient, rounded to 16 bits once, behind that. In between the workspace keeps what they are made of, for the same problem, and so does the weight; the hidden states and the targets are not looked at again.
 * The second call may be made any number of times, with the workspace_bytes that ftcuda_linear_cross_entropy_step_workspace_bytes says, no more and no less.
 */
FTCUDA_API int ftcuda_linear_cross_entropy_step_loss(const FtcudaLinearCrossEntropy* problem, float* loss, void* workspace, uint64_t workspace_bytes,
                                                     void* stream, char* message, size_t message_capacity);
FTCUDA_API int ftcuda_linear_cross_entropy_step_gradients(const FtcudaLinearCrossEntropy* problem, const float* grad_loss, void* grad_hidden,
                                                          int64_t grad_hidden_row_stride, void* grad_weight, int64_t grad_weight_row_stride,
                                                          void* workspace, uint64_t workspace_bytes, void* stream, char* message,
                                                          size_t message_capacity);

/*
 * The same two calls with what is kept in a memory of its own, so that each call's workspace is free again behind it. `kept` and the workspaces start at multiples of 256;
 * kept_bytes is what ftcuda_linear_cross_entropy_step_loss_bytes says for the problem of the loss, no more and no less, in both calls. When the gradients are made
 * the weight's values have to be the same; its address and strides need not.
 */
FTCUDA_API int ftcuda_linear_cross_entropy_step_loss_bytes(const FtcudaLinearCrossEntropy* problem, uint64_t* kept_bytes, uint64_t* workspace_bytes, char* message,
                                                           size_t message_capacity);
FTCUDA_API int ftcuda_linear_cross_entropy_step_gradients_bytes(const FtcudaLinearCrossEntropy* problem, uint64_t kept_bytes, uint64_t* workspace_bytes, char* message,
                                                                size_t message_capacity);
FTCUDA_API int ftcuda_linear_cross_entropy_step_loss_kept(const FtcudaLinearCrossEntropy* problem, float* loss, void* kept, uint64_t kept_bytes, void* workspace,
                                                          uint64_t workspace_bytes, void* stream, char* message, size_t message_capacity);
FTCUDA_API int ftcuda_linear_cross_entropy_step_gradients_kept(const FtcudaLinearCrossEntropy* problem, const float* grad_loss, void* grad_hidden,
                                                               int64_t grad_hidden_row_stride, void* grad_weight, int64_t grad_weight_row_stride, void* kept,
                                                               uint64_t kept_bytes, void* workspace, uint64_t workspace_bytes, void* stream, char* message,
                                                               size_t message_capacity);

/* ---- the experts' router ---- */

/*
 * Each token's softmax over its experts' logits p = softmax(logits[t]), its top_k experts, and what they add up to:
 *   experts[t][i]  the i-th largest logit's index; among equal ones (-0 equals 0) the lowest index comes first. Not a number
 *                  counts as larger than anything. Logits of -inf are never chosen: the slots they would take say -1.
 *   weights[t][i]  p of that expert, 0 in a slot of -1; with `normalize` divided by the sum over the token's slots
 *   counts[e]      how many slots say e: the sizes of the grouped products' groups
 *   *routed        how many tokens took part: those that the mask does not take out and that have a logit above -inf. The others
 *                  have -1 and 0 in all slots, and no part in anything below.
 *   *balance_loss  experts * sum_e f_e P_e with f_e = counts[e] / (routed * top_k) and P_e the mean of p[e] over the routed
 *                  tokens; 0 where none is. For a gradient f_e is a constant.
 * logits: [tokens][experts], unit stride along the experts, row_stride elements between tokens; 1 to 1024 experts, top_k at most 32
 * and at most `experts`. mask: one byte for each token, nonzero = takes part; NULL = all do. Everything is computed in FP32
 * whatever the logits' type, sums over tokens in an order that depends on the sizes alone.
 */
typedef struct {
    const void* logits;
    const uint8_t* mask;
    uint64_t tokens;
    int64_t row_stride;
    uint32_t experts;
    uint32_t top_k;
    int32_t normalize;
    int32_t element;
    int32_t device;
} FtcudaRouting;

/* Bytes of workspace that ftcuda_expert_routing needs; at most about 5 MB. */
FTCUDA_API uint64_t ftcuda_expert_routing_workspace_bytes(const FtcudaRouting* routing);

/* weights: FP32 [tokens][top_k]; experts: INT32 [tokens][top_k]; counts: INT32 [experts]; all dense, on the device, none may be NULL. */
FTCUDA_API int ftcuda_expert_routing(const FtcudaRouting* routing, float* weights, int32_t* experts, int32_t* counts, int32_t* routed,
                                     float* balance_loss, void* workspace, uint64_t workspace_bytes, void* stream, char* message,
                                     size_t message_capacity);

/*
 * grad_logits (of the logits' type, grad_row_stride elements between tokens) from grad_weights (FP32 [tokens][top_k], dense) and *grad_loss (one FP32 on the
 * device), either of which may be NULL, meaning zero; the other arguments as the forward call took and left them (an expert's number beyond the last one
 * is taken for the last one). grad_logits may be the logits themselves, with their stride; otherwise it may not meet what the call reads (refused). Needs no workspace.
 */
FTCUDA_API int ftcuda_expert_routing_backward(const FtcudaRouting* routing, const float* weights, const int32_t* experts, const int32_t* counts,
                                              const int32_t* routed, const float* grad_weights, const float* grad_loss,
                                              void* grad_logits, int64_t grad_row_stride, void* stream, char* message,
                                              size_t message_capacity);

#ifdef __cplusplus
}
#endif

#endif
