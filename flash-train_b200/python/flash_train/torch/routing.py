"""The experts' router in front of a grouped product."""
import typing

import torch

from ._flash_train_torch import _expert_routing


class ExpertRouting(typing.NamedTuple):
    weights: torch.Tensor       # (..., top_k) FP32, differentiable
    experts: torch.Tensor       # (..., top_k) INT32; -1 in a slot that nothing takes
    counts: torch.Tensor        # (experts,) INT32: the rows of each group of a grouped product
    balance_loss: torch.Tensor  # () FP32, differentiable


def expert_routing(logits, top_k, *, normalize=True, mask=None) -> ExpertRouting:
    """Softmax over the last dimension of `logits` (FP32, FP16 or BF16; up to 1024 experts), the `top_k` (up to 32) experts of each
    token with their weights, how many slots each expert got, and the balance loss.

    weights: the softmax at the chosen experts, with `normalize` divided by their sum. Among equal logits the lower index comes
    first; experts whose logit is -inf are never chosen (their slots: -1, weight 0).
    mask: truth values, one for each token; tokens that are False (or whose logits are all -inf) have -1 and 0 in all slots, are not
    counted and get a gradient of zero.
    balance_loss: E * sum_e f_e P_e, f_e the share of all filled and unfilled slots of the routed tokens that went to expert e, P_e the mean of its softmax over the
    routed tokens; 1 when both are even. Its gradient goes through P_e alone.

    Logits of any leading shape; the experts of a token must be neighbours in memory. Gradients of `weights` and `balance_loss`
    reach `logits`; there is no second derivative.
    """
    return ExpertRouting(*_expert_routing(logits, top_k, normalize, mask))
