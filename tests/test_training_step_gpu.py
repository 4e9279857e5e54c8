"""A training step of a layer of experts with the operators as they are used together: router, grouped products, loss, gradients, clipping.

Every operator is held against the formula in 64 bits on what went into it in this run, so that each bound is the operator's own, and what
goes from one to the next (shapes, types, slots that nothing takes, padding, groups without a row) is what it is in use."""
import math

import pytest
import torch

from test_expert_routing_gpu import check_forward, check_gradient
from test_expert_routing_gpu import oracle as routing_oracle
from test_gradient_norm_gpu import check_clipped, check_norm, exact_norm
from test_linear_cross_entropy_gpu import STEP, Oracle, check, ft  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


def check_product(got, a, b, what):
    """FP32 sums of a.shape[1] products, one after another at worst, of operands split to 2^-22 at worst."""
    value, size = a.double() @ b.double(), a.double().abs() @ b.double().abs()
    check(got, value, (a.shape[1] + 8) * 2 * STEP * size, what)


def step(ft, capi, tokens, depth, experts, k, width, vocabulary, dtype, seed, closed=0, padding=0, normalize=True):  # noqa: F811
    generator = torch.Generator(device="cuda").manual_seed(seed)

    def draw(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=generator) * scale).requires_grad_()

    binding = capi.GroupedGemmBinding()
    products = []

    def grouped(a, b, rows, out):
        """out[group] = a[group] @ b[group]; each operand (tensor, rows, columns, row strides, column strides, offsets)."""

        def operand(tensor, rows, cols, row_strides=None, col_strides=None):
            return {"address": tensor.data_ptr(), "rows": rows, "cols": cols, "row_strides": row_strides, "col_strides": col_strides}

        empty = {"address": 0, "rows": out[1], "cols": out[2]}
        plan = binding.make_plan(operand(*a), operand(*b), empty, operand(*out))
        size = plan.workspace_bytes(0)
        workspace = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
        plan.execute(0, workspace.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()  # (the Plan goes out of scope)

    class Product(torch.autograd.Function):
        @staticmethod
        def forward(context, a, b):
            context.save_for_backward(a, b)
            return ft.gemm(a, b)

        @staticmethod
        def backward(context, gradient):
            a, b = context.saved_tensors
            gradient = gradient.contiguous()
            out = ft.gemm(gradient, b.t().contiguous()), ft.gemm(a.t().contiguous(), gradient)
            products.extend([(out[0], gradient, b.t()), (out[1], a.t(), gradient)])
            return out

    class Experts(torch.autograd.Function):
        """rows of each group times the group's matrix."""

        @staticmethod
        def forward(context, rows, matrices, counts):
            context.save_for_backward(rows, matrices)
            context.counts = counts
            n, d, w = len(counts), matrices.shape[1], matrices.shape[2]
            out = torch.empty(rows.shape[0], w, device="cuda")
            grouped((rows, counts, [d] * n), (matrices, [d] * n, [w] * n), counts, (out, counts, [w] * n))
            return out

        @staticmethod
        def backward(context, gradient):
            rows, matrices = context.saved_tensors
            counts = context.counts
            n, d, w = len(counts), matrices.shape[1], matrices.shape[2]
            gradient = gradient.contiguous()
            grad_rows, grad_matrices = torch.empty_like(rows), torch.full_like(matrices, math.nan)
            grouped((gradient, counts, [w] * n), (matrices, [w] * n, [d] * n, [1] * n, [w] * n), counts, (grad_rows, counts, [d] * n))
            grouped((rows, [d] * n, counts, [1] * n, [d] * n), (gradient, counts, [w] * n), counts, (grad_matrices, [d] * n, [w] * n))
            return grad_rows, grad_matrices, None

    hidden, router = draw(tokens, depth), draw(depth, experts, scale=2 * depth ** -0.5)
    up, down = draw(experts, depth, width, scale=depth ** -0.5), draw(experts, width, depth, scale=width ** -0.5)
    head = (torch.randn(vocabulary, depth, device="cuda", generator=generator) * depth ** -0.5).to(dtype).requires_grad_()
    target = torch.randint(0, vocabulary, (tokens,), device="cuda", generator=generator)
    mask = torch.ones(tokens, dtype=torch.bool, device="cuda")
    if padding:
        mask[-padding:] = False
        target[-padding:] = -100
    logits = Product.apply(hidden, router)
    shut = logits.clone()
    if closed:
        shut[:, :closed] = -math.inf  # experts that take nothing: groups without a row
    routing = ft.expert_routing(shut, k, normalize=normalize, mask=mask)
    slots = routing.experts.flatten()
    order = torch.argsort(torch.where(slots < 0, experts, slots), stable=True)
    counts = routing.counts.tolist()
    assert sum(counts) == int((slots >= 0).sum())
    order = order[:sum(counts)]
    rows = hidden[order // k]
    first = Experts.apply(rows, up, counts)
    second = Experts.apply(torch.relu(first), down, counts)
    mixed = second * routing.weights.flatten()[order, None]
    out = (hidden + torch.zeros_like(hidden).index_add(0, order // k, mixed)).to(dtype)
    kept = [logits, shut, routing.weights, rows, first, second, out]
    for tensor in kept:
        tensor.retain_grad()
    loss = ft.linear_cross_entropy(out, head, target) + 0.01 * routing.balance_loss
    loss.backward()

    # Forward: the router, the experts' products, the loss.
    check_product(logits.detach(), hidden.detach(), router.detach(), "router's logits")
    expected = routing_oracle(shut.detach(), k, normalize, mask)
    check_forward(routing, shut, expected)
    begin = 0
    for e, count in enumerate(counts):
        end = begin + count
        for got, a, b in ((first[begin:end], rows[begin:end], up[e]), (second[begin:end], torch.relu(first[begin:end]), down[e]),
                          (rows.grad[begin:end], first.grad[begin:end], up[e].t()), (up.grad[e], rows[begin:end].t(), first.grad[begin:end]),
                          (down.grad[e], torch.relu(first[begin:end]).t(), second.grad[begin:end])):
            if got.numel() and a.shape[1]:
                check_product(got.detach(), a.detach(), b.detach(), f"expert {e}")
            else:
                assert not got.any()  # a gradient over no rows is zero
        begin = end
    for got, a, b in products:
        check_product(got, a, b, "a gradient of the router")
    oracle = Oracle(out.detach(), head.detach(), target)
    live = int(oracle.live.sum())
    total = oracle.loss.sum() / live
    balance = 0.01 * routing.balance_loss.double().item()
    check(loss.detach(), total + balance, oracle.loss_error.sum() / live + 4 * STEP * (total + balance), "loss")

    # Backward: the loss's gradients, the router's, and all ways to the hidden states together.
    dh, dh_bound, dw, dw_bound = oracle.gradients(torch.full((tokens,), 1.0 / live, device="cuda", dtype=torch.float64), dtype)
    check(out.grad, dh, dh_bound, "gradient of the loss's hidden states")
    check(head.grad, dw, dw_bound, "gradient of the vocabulary")
    check_gradient(shut.grad, shut.detach(), k, normalize, expected, routing.weights.grad, 0.01)
    ways = [out.grad.double(), products[0][0].double(), torch.zeros_like(hidden).double().index_add(0, order // k, rows.grad.double())]
    check(hidden.grad, sum(ways), (k + 3) * 2 * STEP * (sum(way.abs() for way in ways[:2]) + torch.zeros_like(ways[0]).index_add(0, order // k, rows.grad.double().abs())),
          "gradient of the hidden states")
    assert not hidden.grad[~mask].any() if padding else True

    # The norm over all of them, and the clipping.
    parameters = [hidden, router, up, down, head]
    before = [p.grad.clone() for p in parameters]
    norm = exact_norm(before)
    check_norm(ft.clip_grad_norm_(parameters, norm / 3), norm)
    for p, gradient in zip(parameters, before):
        check_clipped(p.grad, gradient, norm, norm / 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens, depth, experts, k, width, vocabulary, closed, padding, normalize", [
    (200, 64, 8, 2, 96, 1000, 0, 0, True),
    (300, 160, 16, 4, 130, 5003, 3, 45, False),  # products with K >= 128, experts without a row, padding
    (1, 64, 4, 1, 64, 300, 0, 0, True),          # one token: most groups are empty
    (2048, 256, 64, 8, 128, 8191, 0, 100, True),
])
def test_a_step(ft, capi, tokens, depth, experts, k, width, vocabulary, closed, padding, normalize, dtype):  # noqa: F811
    step(ft, capi, tokens, depth, experts, k, width, vocabulary, dtype, seed=tokens, closed=closed, padding=padding, normalize=normalize)
