/*
 * ftcuda/training.h -- what a training step does around its products: the gradients' norm.
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
 * written. A norm that is not a number makes every element NaN; an infinite one makes the finite elements 0 and the others NaN. max_norm >= 0.
 * No element may be written that another gradient reads or writes (refused where addresses, sizes and strides
 * show it).
 */
FTCUDA_API int ftcuda_gradient_clip(const FtcudaGradient* gradients, uint64_t count, int norm_kind, double max_norm, float* norm,
                                    int32_t device, void* workspace, uint64_t workspace_bytes, void* stream, char* message,
                                    size_t message_capacity);

#ifdef __cplusplus
}
#endif

#endif
