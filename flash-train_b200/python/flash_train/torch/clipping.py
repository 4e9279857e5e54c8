"""clip_grad_norm_ over a model's parameters, with the arguments of torch.nn.utils.clip_grad_norm_."""
import torch

from ._flash_train_torch import clip_grads, grad_norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Scales the `.grad` of the parameters (one tensor, or an iterable of them; those without a gradient are passed over) in
    place so that their common norm is at most `max_norm`, and returns the norm from before, an FP32 number on their device.

    Does not wait for the GPU, unless `error_if_nonfinite` asks for a RuntimeError, before anything is changed, when the norm is
    infinite or not a number. A parameter that is listed twice is refused, as its gradient would be scaled twice.
    """
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    gradients = [p.grad for p in parameters if p.grad is not None]
    with torch.no_grad():
        if error_if_nonfinite and gradients:
            norm = grad_norm(gradients, norm_type)
            if not torch.isfinite(norm):
                raise RuntimeError(f"the gradients' norm of order {norm_type} is not finite; they were not clipped")
        return clip_grads(gradients, float(max_norm), float(norm_type))
