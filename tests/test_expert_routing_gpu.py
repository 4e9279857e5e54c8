"""expert_routing and its gradient against the definition in 64 bits."""
import gc
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24  # half a step of FP32
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ft(native_library):
    if not torch.cuda.is_available():
        pytest.fail("the GPU tests need a CUDA device")
    from conftest import load_build_module

    load_build_module().build_torch_binding(verbose=False)
    import flash_train.torch

    return flash_train.torch


@pytest.fixture
def memory_given_back():
    """What a large test took goes back to the device, so that no later test's small tensor sits in a piece of it and keeps the rest."""
    yield
    gc.collect()
    torch.cuda.empty_cache()


def oracle(logits, k, normalize=True, mask=None):
    """The definition, in 64 bits on the CPU. Slots are filled one after another by the largest logit left, the lowest index among equals."""
    x = logits.detach().double().cpu()
    tokens, n = x.shape
    live = (x > -math.inf).any(1) | torch.isnan(x).any(1)
    if mask is not None:
        live &= mask.cpu()
    experts = torch.full((tokens, k), -1, dtype=torch.int64)
    order = torch.where(torch.isnan(x), torch.full_like(x, math.inf), x)  # tests with NaN have no +inf in the same row
    left = order.clone()
    rows = torch.arange(tokens)
    for slot in range(k):
        best = left.max(1).values
        first = (left == best[:, None]).int().argmax(1)
        taken = live & (best > -math.inf)
        experts[taken, slot] = first[taken]
        left[rows[taken], first[taken]] = -math.inf
    p = torch.softmax(x, 1)
    p[~live] = 0.0
    filled = experts >= 0
    weights = torch.where(filled, p.gather(1, experts.clamp(min=0)), 0.0)
    if normalize:
        total = weights.sum(1, keepdim=True)
        weights = torch.where(filled, weights / total, 0.0)
    counts = torch.bincount(experts[filled], minlength=n)
    routed = int(live.sum())
    shares = counts.double() / max(1, routed * k)
    loss = n * (shares * p.sum(0)).sum().item() / max(1, routed)
    return {"p": p, "weights": weights, "experts": experts, "counts": counts, "routed": routed, "shares": shares, "loss": loss}


def spread(logits):
    finite = logits.detach().float()
    finite = finite[torch.isfinite(finite)]
    return (finite.max() - finite.min()).item() if finite.numel() else 0.0


def relative(logits):
    """Of a softmax value: the rounded difference from the largest logit (its size times half a step), the exponential (two steps), a
    sum of up to 32 in a lane and five levels over the warp, a division and two products."""
    return (spread(logits) + 4 + 32 + 5 + 6) * STEP


def check_forward(routing, logits, expected, tokens_in_a_row=64):
    tolerance = relative(logits)
    assert routing.experts.dtype == torch.int32 and routing.counts.dtype == torch.int32
    assert torch.equal(routing.experts.cpu().long(), expected["experts"])
    assert torch.equal(routing.counts.cpu().long(), expected["counts"])
    error = (routing.weights.detach().double().cpu() - expected["weights"]).abs()
    # (2^-126: exponentials below the smallest normal number are not held to a relative error.)
    assert (error <= 2 * tolerance * expected["weights"] + 2.0 ** -126).all(), error.max()
    # Sums over a warp's tokens one after another, then over 16 warps in four levels.
    assert abs(routing.balance_loss.item() - expected["loss"]) <= (tolerance + (tokens_in_a_row + 8) * STEP) * expected["loss"]


def check_gradient(got, logits, k, normalize, expected, grad_weights, grad_loss):
    p, w, e = expected["p"], expected["weights"], expected["experts"].clamp(min=0)
    n = p.shape[1]
    slope = grad_loss * n * expected["shares"] / max(1, expected["routed"])
    g = torch.where(expected["experts"] >= 0, grad_weights.double().cpu(), 0.0)
    dot = (g * w).sum(1, keepdim=True)
    size = (g.abs() * w).sum(1, keepdim=True)
    if normalize:
        value = p * (slope - (p @ slope)[:, None])
        scale = p * (slope.abs() + (p @ slope.abs())[:, None])
        value.scatter_add_(1, e, w * (g - dot))
        scale.scatter_add_(1, e, w * (g.abs() + size))
    else:
        value = p * (slope - (p @ slope)[:, None] - dot)
        scale = p * (slope.abs() + (p @ slope.abs())[:, None] + size)
        value.scatter_add_(1, e, w * g)
        scale.scatter_add_(1, e, w * g.abs())
    # Each term is a product of up to three values of that relative error and the sums' own.
    bound = 4 * relative(logits) * scale + 2.0 ** -126
    finfo = torch.finfo(got.dtype)
    if got.dtype != torch.float32:
        bound = bound + finfo.eps / 2 * value.abs() + finfo.smallest_normal * finfo.eps / 2
    error = (got.double().cpu() - value).abs()
    assert got.dtype == logits.dtype and (error <= bound).all(), (error - bound).max()


def make(tokens, experts, dtype, seed=0, scale=2.0):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(tokens, experts, device="cuda", generator=generator).mul_(scale).to(dtype)


def run_and_check(ft, logits, k, normalize=True, mask=None, grad_loss=0.37, seed=1):
    leaf = logits.detach().requires_grad_()
    routing = ft.expert_routing(leaf, k, normalize=normalize, mask=mask)
    expected = oracle(logits, k, normalize, mask)
    check_forward(routing, logits, expected)
    generator = torch.Generator(device="cuda").manual_seed(seed)
    grad_weights = torch.randn(routing.weights.shape, device="cuda", generator=generator)
    loss_grad = torch.tensor(grad_loss, device="cuda")
    got, = torch.autograd.grad((routing.weights, routing.balance_loss), leaf, (grad_weights, loss_grad))
    check_gradient(got, logits, k, normalize, expected, grad_weights, loss_grad.double().item())
    return routing, got


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens, experts, k", [(1, 1, 1), (1, 8, 2), (32, 8, 8), (33, 60, 4), (500, 64, 8), (77, 65, 6), (129, 128, 1), (40, 160, 32),
                                                (1000, 256, 8), (50, 257, 5), (64, 512, 10), (35, 1000, 8), (20, 1024, 32)])
def test_against_the_definition(ft, tokens, experts, k, dtype, normalize):
    run_and_check(ft, make(tokens, experts, dtype), k, normalize)


def test_more_tokens_than_warps(ft):
    run_and_check(ft, make(20011, 37, torch.float32), 3)


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_logits_go_to_the_lowest_index(ft, dtype):
    logits = (make(300, 96, torch.float32) * 0.5).round().to(dtype)  # a handful of values, many of each
    logits[0] = 0.0
    logits[1, ::2], logits[1, 1::2] = 0.0, -0.0
    run_and_check(ft, logits, 7)
    assert ft.expert_routing(logits[:2], 4).experts.tolist() == [[0, 1, 2, 3]] * 2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [9, 700])
def test_mask(ft, dtype, tokens):
    logits = make(tokens, 48, dtype)
    mask = torch.rand(tokens, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)) < 0.6
    mask[3] = False
    routing, gradient = run_and_check(ft, logits, 4, mask=mask)
    assert (routing.experts[~mask] == -1).all() and not routing.weights[~mask].any() and not gradient[~mask].any()
    logits = torch.where(mask[:, None], logits, torch.full_like(logits, math.nan))  # what is masked is not looked at
    again = ft.expert_routing(logits, 4, mask=mask)
    assert torch.equal(again.weights, routing.weights) and torch.equal(again.balance_loss, routing.balance_loss)


@pytest.mark.parametrize("tokens", [5, 100])
def test_nobody_takes_part(ft, tokens):
    logits = make(tokens, 16, torch.float32).requires_grad_()
    routing = ft.expert_routing(logits, 2, mask=torch.zeros(tokens, dtype=torch.bool, device="cuda"))
    assert (routing.experts == -1).all() and not routing.weights.any() and not routing.counts.any() and routing.balance_loss.item() == 0.0
    gradient, = torch.autograd.grad((routing.weights.sum() + routing.balance_loss), logits)
    assert not gradient.any()


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_closed_experts(ft, dtype, normalize):
    """-inf closes an expert; a token may have fewer than k open ones, or none. The type's lowest value is a logit like any other."""
    logits = make(200, 40, dtype, scale=1.0)
    logits[:, 5:9] = -math.inf
    logits[3] = -math.inf
    logits[4, 2:] = -math.inf
    logits[199, :39] = -math.inf
    routing, gradient = run_and_check(ft, logits, 5, normalize)
    assert routing.experts[3].tolist() == [-1] * 5 and sorted(routing.experts[4].tolist()) == [-1, -1, -1, 0, 1]
    assert routing.experts[199].tolist() == [39, -1, -1, -1, -1] and not gradient[3].any()
    lowest = torch.full((2, 6), torch.finfo(dtype).min, device="cuda", dtype=dtype)
    lowest[1, 4] = 1.0
    low = ft.expert_routing(lowest, 2, normalize=normalize)
    assert low.experts.tolist() == [[0, 1], [4, 0]] and torch.allclose(low.weights[0], torch.full((2,), 0.5 if normalize else 1 / 6, device="cuda"))
    assert low.weights[1].tolist() == [1.0, 0.0]


@pytest.mark.parametrize("dtype", TYPES)
def test_not_a_number_shows(ft, dtype):
    logits = make(40, 33, dtype)
    logits[7, 20] = math.nan
    leaf = logits.detach().requires_grad_()
    routing = ft.expert_routing(leaf, 3)
    expected = oracle(logits, 3)
    assert torch.equal(routing.experts.cpu().long(), expected["experts"]) and routing.experts[7, 0].item() == 20
    assert torch.isnan(routing.weights[7]).all() and torch.isfinite(routing.weights[6]).all() and math.isnan(routing.balance_loss.item())
    gradient, = torch.autograd.grad(routing.weights.sum(), leaf)
    assert torch.isnan(gradient[7]).all() and torch.isfinite(gradient[8]).all()


def test_large_logits(ft):
    run_and_check(ft, make(64, 32, torch.float32, scale=3000.0), 4)


def test_gradient_against_differences(ft):
    """Central differences of the FP32 result. With a step h their own error is h^2 / 6 times a third derivative, which for a
    softmax of weights g is at most 6 |g|, and the results' rounding over h."""
    base = torch.tensor([[0.9, -0.4, 0.3, 1.6, -1.2, 0.0]], device="cuda").repeat(2, 1)  # far enough apart for the same choice
    base[1] = base[1].flip(0)
    grad_weights = torch.tensor([[0.7, -0.3], [0.2, 1.1]], device="cuda")
    h = 2.0 ** -5
    for normalize in (True, False):
        def value(logits):
            routing = ft.expert_routing(logits, 2, normalize=normalize)
            return (routing.weights * grad_weights).sum() + 0.5 * routing.balance_loss

        leaf = base.clone().requires_grad_()
        gradient, = torch.autograd.grad(value(leaf), leaf)
        for t in range(2):
            for e in range(6):
                step = torch.zeros_like(base)
                step[t, e] = h
                difference = (value(base + step).item() - value(base - step).item()) / (2 * h)
                size = grad_weights.abs().sum().item() + 0.5 * 6
                assert abs(difference - gradient[t, e].item()) <= size * (h * h + 64 * STEP / h)


def test_either_gradient_alone_and_none(ft):
    logits = make(70, 24, torch.float32).requires_grad_()
    routing = ft.expert_routing(logits, 3)
    expected = oracle(logits, 3)
    grad_weights = torch.ones_like(routing.weights) * 0.5
    first, = torch.autograd.grad(routing.weights, logits, grad_weights, retain_graph=True)
    check_gradient(first, logits, 3, True, expected, grad_weights, 0.0)
    second, = torch.autograd.grad(routing.balance_loss, logits, retain_graph=True)
    check_gradient(second, logits, 3, True, expected, torch.zeros_like(grad_weights), 1.0)
    assert not routing.experts.requires_grad and not routing.counts.requires_grad
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(routing.balance_loss, logits, create_graph=True)
    assert not ft.expert_routing(logits.detach(), 3).weights.requires_grad


def test_shapes_strides_and_types_of_gradients(ft):
    wide = make(90, 100, torch.bfloat16)
    window = wide[:, 30:70]
    run_and_check(ft, window, 4)
    run_and_check(ft, make(91, 33, torch.float16)[1::2, 1:], 4)
    cube = make(60, 32, torch.float32).view(3, 20, 32).requires_grad_()
    mask = torch.rand(3, 20, device="cuda") < 0.5
    routing = ft.expert_routing(cube, 2, mask=mask)
    flat = ft.expert_routing(cube.view(60, 32), 2, mask=mask.view(60))
    assert routing.weights.shape == (3, 20, 2) and torch.equal(routing.weights.view(60, 2), flat.weights) and torch.equal(routing.counts, flat.counts)
    gradient, = torch.autograd.grad(routing.weights.sum(2).t().sum() + routing.balance_loss.double(), cube)
    assert gradient.shape == cube.shape
    one = ft.expert_routing(cube[0, 0].detach(), 2)
    assert one.weights.shape == (2,)
    empty = ft.expert_routing(torch.empty(0, 8, device="cuda"), 2)
    assert empty.weights.shape == (0, 2) and not empty.counts.any() and empty.balance_loss.item() == 0.0


def test_equal_calls_give_equal_bits(ft):
    logits = make(30000, 64, torch.bfloat16)
    assert len({ft.expert_routing(logits, 8).balance_loss.item() for _ in range(5)}) == 1


def test_another_stream_and_a_graph(ft):
    logits = make(3000, 64, torch.float32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = ft.expert_routing(logits, 4)
    torch.cuda.current_stream().wait_stream(side)
    check_forward(on_side, logits, oracle(logits, 4))
    held = logits.clone().requires_grad_()
    grad_weights = torch.randn(3000, 4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        routing = ft.expert_routing(held, 4)
        gradient, = torch.autograd.grad((routing.weights, routing.balance_loss), held, (grad_weights, torch.ones((), device="cuda")))
    for seed in (1, 2):
        with torch.no_grad():
            held.copy_(make(3000, 64, torch.float32, seed))
        graph.replay()
        expected = oracle(held, 4)
        check_forward(routing, held, expected)
        check_gradient(gradient, held, 4, True, expected, grad_weights, 1.0)


def test_refusals(ft):
    x = make(10, 8, torch.float32)
    for call, reason in [
        (lambda: ft.expert_routing(x.cpu(), 2), "device tensor"), (lambda: ft.expert_routing(x.double(), 2), "FP32, FP16 or BF16"), (lambda: ft.expert_routing(x, 0), "top_k"),
        (lambda: ft.expert_routing(x, 9), "top_k"), (lambda: ft.expert_routing(make(2, 1025, torch.float32), 2), "1024"),
        (lambda: ft.expert_routing(x.t(), 2), "neighbours"), (lambda: ft.expert_routing(x[:1].expand(10, 8), 2), "rows overlap"),
        (lambda: ft.expert_routing(x, 2, mask=torch.ones(9, dtype=torch.bool, device="cuda")), "each token"),
        (lambda: ft.expert_routing(x, 2, mask=torch.ones(10, device="cuda")), "truth values"),
        (lambda: ft.expert_routing(x, 2, mask=torch.ones(10, dtype=torch.bool)), "truth values"),
    ]:
        with pytest.raises(RuntimeError, match=reason):
            call()


def test_another_device_than_the_current_one(ft, capi):
    x, out = make(10, 16, torch.float32), torch.empty(1 << 20, device="cuda")
    r = capi.Routing(logits=x.data_ptr(), mask=None, tokens=10, row_stride=16, experts=16, top_k=2, normalize=1, element=4, device=1)
    weights, experts, counts, routed, loss, workspace, gw, gl, gx = (out.data_ptr() + 65536 * i for i in range(9))
    with pytest.raises(capi.FTrainError, match="device 1 must be current"):
        capi.expert_routing(r, weights, experts, counts, routed, loss, workspace, 65536)
    with pytest.raises(capi.FTrainError, match="device 1 must be current"):
        capi.expert_routing_backward(r, weights, experts, counts, routed, gw, gl, gx, 16)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("experts, k", [(40, 3), (256, 8), (1000, 20)])
def test_gradient_over_the_logits_themselves(ft, capi, dtype, experts, k):
    """grad_logits may be the logits, with their stride."""
    tokens, code = 3001, {torch.float32: 4, torch.float16: 7, torch.bfloat16: 8}[dtype]
    x = make(tokens, experts, dtype, seed=8)
    routing = ft.expert_routing(x, k)
    r = capi.Routing(logits=x.data_ptr(), mask=None, tokens=tokens, row_stride=experts, experts=experts, top_k=k, normalize=1, element=code, device=0)
    routed = torch.tensor(tokens, dtype=torch.int32, device="cuda")
    gw, gl = torch.randn(tokens, k, device="cuda"), torch.tensor(0.5, device="cuda")
    apart = torch.empty_like(x)
    for to in (apart, x):
        capi.expert_routing_backward(r, routing.weights.data_ptr(), routing.experts.data_ptr(), routing.counts.data_ptr(), routed.data_ptr(), gw.data_ptr(), gl.data_ptr(),
                                     to.data_ptr(), experts, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(apart, x) and torch.isfinite(x).all() and x.any()


def test_slots_that_nothing_takes_with_many_rounds(ft):
    """More slots than experts that can be chosen, below and above the rounds that are written out one by one."""
    for dtype in TYPES:
        for experts, k in ((40, 32), (256, 8), (256, 9), (600, 20)):
            x = make(77, experts, dtype, seed=k)
            x[:, torch.randperm(experts, device="cuda")[: experts - 5]] = -math.inf
            x[5] = -math.inf
            x[6, 3:] = -math.inf
            run_and_check(ft, x, k)


def test_logits_past_32_bits(ft, memory_given_back):
    """More than 2^32 logits: the last tokens come out as they do alone, and every slot is counted."""
    tokens, experts, k = (1 << 22) + 1001, 1024, 4
    x = torch.empty(tokens, experts, device="cuda", dtype=torch.bfloat16)
    for piece in x.split(1 << 18):
        piece.copy_(torch.randn(piece.shape, device="cuda"))
    x.requires_grad_()
    tail = x.detach()[-3000:].clone().requires_grad_()
    routing, alone = ft.expert_routing(x, k), ft.expert_routing(tail, k)
    assert torch.equal(routing.experts[-3000:], alone.experts) and torch.equal(routing.weights[-3000:], alone.weights)
    assert torch.equal(routing.counts.long(), torch.bincount(routing.experts.flatten(), minlength=experts))
    # Sums over 900 tokens of a warp one after another, whose softmax values are all about 1 / 1024: the loss is 1 within their rounding and what chance leaves.
    assert abs(routing.balance_loss.item() - 1.0) < 1e-2
    upstream = torch.randn(tokens, k, device="cuda")
    grad, = torch.autograd.grad(routing.weights, x, upstream)
    expected, = torch.autograd.grad(alone.weights, tail, upstream[-3000:].contiguous())
    assert torch.equal(grad[-3000:], expected)
