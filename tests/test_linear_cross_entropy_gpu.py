"""linear_cross_entropy and its gradients against the definition in 64 bits."""
import gc
import math

import pytest
import torch
import torch.nn.functional as F

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


def make(tokens, depth, vocabulary, dtype, seed=0, spread=2.0):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    hidden = torch.randn(tokens, depth, device="cuda", generator=generator).to(dtype)
    weight = (torch.randn(vocabulary, depth, device="cuda", generator=generator) * spread * depth ** -0.5).to(dtype)
    target = torch.randint(0, vocabulary, (tokens,), device="cuda", generator=generator)
    return hidden, weight, target


class Oracle:
    """The definition in 64 bits, and how far FP32 sums and the stated roundings can be from it.

    A logit is a sum of `depth` products: with n terms added one after another (the tensor cores add 8 or 16 at a time, and cut off
    instead of rounding: two half steps each) it is off by at most (n / 8 + 8) 2^-23 of the sum of the products' magnitudes. That
    allows as well for the products of split FP32 operands. An exponential is off by its argument's error, by two steps of its
    own and by the argument's rounding, whose size is that of the logits (in powers of two)."""

    def __init__(self, hidden, weight, target, ignore_index=-100):
        self.live = target != ignore_index
        self.h = torch.where(self.live[:, None], hidden.double(), 0.0)
        self.w = weight.double()
        self.target = torch.where(self.live, target, 0)
        z = self.h @ self.w.T
        self.lse = torch.logsumexp(z, 1)
        self.loss = torch.where(self.live, self.lse - z.gather(1, self.target[:, None])[:, 0], 0.0)
        depth = hidden.shape[1]
        z_error = (depth / 8 + 8) * 2 * STEP * (self.h.abs() @ self.w.abs().T).amax(1)
        size = z.abs().amax(1) + self.lse.abs()
        self.relative = 2 * z_error + (32 + 4 * size) * 2 * STEP  # of an exponential against the sum
        self.loss_error = torch.where(self.live, self.relative + 4 * size * STEP, 0.0)
        self.z = z

    def gradients(self, grad, dtype, step=True):
        """For upstream gradients `grad` of each token: (dH, its bound, dW, its bound), the roundings of the results to `dtype` among them."""
        grad = torch.where(self.live, grad.double(), 0.0)
        slope = torch.exp(self.z - self.lse[:, None])
        error = slope * self.relative[:, None]
        if step and dtype != torch.float32:
            # In the step call an exponential is in FP16 for a while, at 2^13 for the largest of its piece of the vocabulary: one more rounding, of half
            # a step (2^-11 relative, or 2^-25 of what is at most 2^13 where it is subnormal).
            error += 2.0 ** -11 * slope + 2.0 ** -38
        slope.scatter_add_(1, self.target[:, None], torch.full_like(self.lse, -1.0)[:, None])
        half_step = torch.finfo(dtype).eps / 2
        # The slopes' rounding; and the smallest that FP16 holds at its scale of 2^13 for the largest gradient.
        error += (half_step + 4 * STEP) * slope.abs()
        slope *= grad[:, None]
        error *= grad.abs()[:, None]
        # Below 2^-126, FP32's smallest normal number, exponentials come out as 0, and so may operands of the products: with p < 2^-126 the
        # slope g p is off by |g p| < 2^-126 |g|, with |g p| < 2^-126 by less than that.
        error += (grad.abs()[:, None] + 1.0) * 2.0 ** -126
        if dtype == torch.float16:
            error += grad.abs().max() * 2.0 ** -38
        if dtype == torch.float32:  # large products: small slopes to 2^-50 of the largest that shares their scale (at most 1 times the largest gradient)
            error += grad.abs().max() * 2.0 ** -50
        vocabulary, tokens = self.w.shape[0], self.h.shape[0]
        finfo = torch.finfo(dtype)
        out = []
        for a, e, b, terms in ((slope, error, self.w, vocabulary), (slope.T, error.T, self.h, tokens)):
            value = a @ b
            bound = (e + (terms / 8 + 24) * 2 * STEP * a.abs()) @ b.abs() + half_step * value.abs() * 1.01 + finfo.smallest_normal * finfo.eps
            out += [value, bound]
        return out


def check(got, value, bound, what):
    error = (got.double() - value).abs() - bound
    assert torch.isfinite(got).all() and (error <= 0).all(), f"{what}: {error.max().item():.3g} beyond a bound of {bound.max().item():.3g}"


def run(ft, hidden, weight, target, reduction="mean", upstream=None, **options):
    h, w = hidden.detach().requires_grad_(), weight.detach().requires_grad_()
    loss = ft.linear_cross_entropy(h, w, target, reduction=reduction, **options)
    upstream = torch.ones_like(loss) if upstream is None else upstream
    return loss.detach(), *torch.autograd.grad(loss, (h, w), upstream)


def run_and_check(ft, hidden, weight, target, reduction="mean", scale=1.0, ignore_index=-100):
    tokens = hidden.shape[0]
    oracle = Oracle(hidden, weight, target, ignore_index)
    count = max(1, int(oracle.live.sum()))
    if reduction == "none":
        upstream = torch.randn(tokens, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)) * scale
        each = upstream
    else:
        upstream = torch.tensor(scale, device="cuda")
        each = torch.full((tokens,), scale / (count if reduction == "mean" else 1), device="cuda", dtype=torch.float64)
    loss, grad_hidden, grad_weight = run(ft, hidden, weight, target, reduction, upstream, ignore_index=ignore_index)
    assert loss.dtype == torch.float32 and grad_hidden.dtype == hidden.dtype and grad_weight.dtype == weight.dtype
    if reduction == "none":
        check(loss, oracle.loss, oracle.loss_error, "loss")
    else:
        divisor = count if reduction == "mean" else 1
        total = oracle.loss.sum() / divisor
        check(loss, total, oracle.loss_error.sum() / divisor + 2 * STEP * total.abs(), "loss")
    dh, dh_bound, dw, dw_bound = oracle.gradients(each, hidden.dtype)
    check(grad_hidden, dh, dh_bound, "hidden's gradient")
    check(grad_weight, dw, dw_bound, "weight's gradient")
    assert not grad_hidden[~oracle.live].any()
    return loss, grad_hidden, grad_weight


SIZES = [(1, 64, 128), (1, 1, 1), (2, 8, 1), (5, 16, 2), (1, 4096, 300), (3, 100, 17), (33, 65, 131), (64, 128, 129), (255, 72, 257), (256, 64, 256), (257, 200, 1000),
         (300, 512, 2049), (513, 33, 700), (1000, 1024, 3000), (90, 130, 20011), (2000, 1100, 9000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens, depth, vocabulary", SIZES)
def test_against_the_definition(ft, tokens, depth, vocabulary, dtype):
    hidden, weight, target = make(tokens, depth, vocabulary, dtype)
    run_and_check(ft, hidden, weight, target, scale=64.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_reductions(ft, dtype, reduction):
    hidden, weight, target = make(170, 96, 450, dtype, seed=2)
    target[::3] = -100
    target[5:20] = 7
    run_and_check(ft, hidden, weight, target, reduction)
    target[target == 7] = -1
    run_and_check(ft, hidden, weight, target.clamp(min=-1), reduction, ignore_index=-1)


@pytest.mark.parametrize("dtype", TYPES)
def test_upstream_gradients_of_any_size(ft, dtype):
    """The slopes' scale follows the largest upstream gradient; small ones beside it, and zeros, keep their own precision in BF16 and FP32."""
    hidden, weight, target = make(100, 64, 300, dtype, seed=3)
    for scale in ((1e-30, 1e-3, 1.0, 1e4) if dtype != torch.float16 else (1e-3, 1.0, 50.0)):
        run_and_check(ft, hidden, weight, target, "none", scale)
    zero = torch.zeros(100, device="cuda")
    _, grad_hidden, grad_weight = run(ft, hidden, weight, target, "none", zero)
    assert not grad_hidden.any() and not grad_weight.any()
    bad = zero.clone()
    bad[3] = math.inf
    _, grad_hidden, _ = run(ft, hidden, weight, target, "none", bad)
    assert not torch.isfinite(grad_hidden[3]).any() and not grad_hidden[4].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_what_padding_holds_does_not_matter(ft, dtype):
    hidden, weight, target = make(600, 80, 333, dtype, seed=4)
    target[100:400] = -100
    target[599] = -100
    expected = run_and_check(ft, hidden, weight, target)
    hidden[target == -100] = math.nan
    hidden[150] = math.inf
    got = run(ft, hidden, weight, target)
    assert all(torch.equal(a, b) for a, b in zip(got[:1] + got[2:], expected[:1] + expected[2:])) and torch.equal(got[1], expected[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [0, 1, 300])
def test_no_target_at_all(ft, dtype, tokens):
    hidden, weight, target = make(tokens, 72, 200, dtype, seed=5)
    hidden.fill_(math.nan)
    target.fill_(-100)
    for reduction in ("mean", "sum", "none"):
        loss, grad_hidden, grad_weight = run(ft, hidden, weight, target, reduction)
        assert not loss.any() and loss.shape == (target.shape if reduction == "none" else ()) and not grad_hidden.any() and not grad_weight.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_target_outside_of_the_vocabulary_shows(ft, dtype):
    hidden, weight, target = make(40, 64, 100, dtype, seed=6)
    for bad in (100, -1, -101, 1 << 40, -(1 << 63)):
        wrong = target.clone()
        wrong[11] = bad
        loss, grad_hidden, grad_weight = run(ft, hidden, weight, wrong, "none")
        assert torch.isnan(loss[11]) and torch.isfinite(loss).sum() == 39
        assert torch.isnan(grad_hidden[11]).all() and torch.isfinite(grad_hidden[12]).all() and torch.isnan(grad_weight).all()
        assert torch.isnan(ft.linear_cross_entropy(hidden, weight, wrong))


@pytest.mark.parametrize("dtype", TYPES)
def test_large_logits(ft, dtype):
    """Only differences to the largest logit are exponentials' arguments."""
    hidden, weight, target = make(70, 64, 500, dtype, seed=7, spread=200.0)
    run_and_check(ft, hidden, weight, target)


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_and_nan_show(ft, dtype):
    hidden, weight, target = make(50, 64, 300, dtype, seed=8)
    hidden[3, 5] = math.nan
    loss = ft.linear_cross_entropy(hidden, weight, target, reduction="none")
    assert torch.isnan(loss[3]) and torch.isfinite(loss).sum() == 49
    # A logit of -inf is a column of probability zero; all of them leave nothing.
    hidden = hidden.abs().nan_to_num(1.0) + 0.01
    weight[7] = -math.inf
    target[target == 7] = 8
    target[0] = 7
    loss = ft.linear_cross_entropy(hidden.to(dtype), weight, target, reduction="none")
    keep = torch.arange(300, device="cuda") != 7
    rest = target - (target > 7).long()
    without = ft.linear_cross_entropy(hidden.to(dtype), weight[keep], rest, reduction="none")
    assert loss[0].item() == math.inf and torch.allclose(loss[1:], without[1:], rtol=0, atol=1e-4)


@pytest.mark.parametrize("dtype, tokens, vocabulary", [(torch.bfloat16, 4096, 140001), (torch.float16, 4500, 131072), (torch.float32, 4096, 70001)])
def test_several_pieces_of_the_vocabulary(ft, memory_given_back, dtype, tokens, vocabulary):
    hidden, weight, target = make(tokens, 40, vocabulary, dtype, seed=10)
    target[::7] = -100
    target[1], target[2] = 0, vocabulary - 1
    loss, grad_hidden, grad_weight = run(ft, hidden, weight, target, "sum", torch.tensor(2.0, device="cuda"))
    # In 64 bits, some rows at a time; each result's 2-norm against that of its error: the slopes' rounding and the results' own.
    total, dw, worst = 0.0, torch.zeros(vocabulary, 40, device="cuda", dtype=torch.float64), 0.0
    w = weight.double()
    tolerance = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2e-6}[dtype] * 1.5
    for part in torch.arange(tokens, device="cuda").split(500):
        h, y = hidden[part].double(), target[part]
        live = y != -100
        log_p = torch.log_softmax(h @ w.T, 1)
        total -= log_p.gather(1, y.clamp(min=0)[:, None])[live].sum().item()
        slope = log_p.exp_()
        slope[torch.arange(len(part), device="cuda"), y.clamp(min=0)] -= 1.0
        slope *= 2.0 * live[:, None]
        dh = slope @ w
        assert (grad_hidden[part].double() - dh).norm() <= tolerance * dh.norm()
        dw += slope.T @ h
    assert abs(loss.item() - total) <= 2e-6 * total
    assert (grad_weight.double() - dw).norm() <= tolerance * dw.norm()
    edges = [0, 255, 256, vocabulary - 1]
    assert (grad_weight[edges].double() - dw[edges]).norm() <= 2 * tolerance * dw[edges].norm()


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(ft, dtype):
    hidden, weight, target = make(130, 80, 300, dtype, seed=11)
    wide_h = torch.zeros(260, 101, device="cuda", dtype=dtype)
    wide_w = torch.zeros(301, 97, device="cuda", dtype=dtype)
    odd_h, odd_w = wide_h[::2, 3:83], wide_w[1:, 1:81]
    odd_h.copy_(hidden)
    odd_w.copy_(weight)
    padded_w = torch.zeros(300, 96, device="cuda", dtype=dtype)[:, :80]
    padded_w.copy_(weight)
    expected = run_and_check(ft, hidden, weight, target)
    run_and_check(ft, odd_h, odd_w, target)
    for h, w in ((odd_h, weight), (hidden, padded_w)):
        got = run(ft, h, w, target)
        assert all(torch.allclose(a.float(), b.float(), rtol=1e-6, atol=0) or torch.equal(a, b) for a, b in zip(got, expected))


def test_leading_dimensions(ft):
    hidden, weight, target = make(60, 64, 200, torch.bfloat16, seed=12)
    flat = run(ft, hidden, weight, target, "none", torch.arange(60, device="cuda").float())
    cube = run(ft, hidden.view(3, 20, 64), weight, target.view(3, 20), "none", torch.arange(60, device="cuda").float().view(3, 20))
    assert cube[0].shape == (3, 20) and cube[1].shape == (3, 20, 64)
    assert torch.equal(cube[0].view(-1), flat[0]) and torch.equal(cube[1].view(60, 64), flat[1]) and torch.equal(cube[2], flat[2])
    one = ft.linear_cross_entropy(hidden[0], weight, target[0])
    assert abs(one.item() - flat[0][0].item()) <= 1e-5


@pytest.mark.parametrize("dtype", TYPES)
def test_either_operand_alone(ft, dtype):
    hidden, weight, target = make(100, 64, 300, dtype, seed=13)
    _, both_h, both_w = run(ft, hidden, weight, target)
    h = hidden.clone().requires_grad_()
    ft.linear_cross_entropy(h, weight, target).backward()
    assert torch.equal(h.grad, both_h)
    w = weight.clone().requires_grad_()
    ft.linear_cross_entropy(hidden, w, target).backward()
    assert torch.equal(w.grad, both_w)
    assert not ft.linear_cross_entropy(hidden, weight, target).requires_grad
    loss = ft.linear_cross_entropy(h, w, target)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(loss, h, create_graph=True)


def test_gradient_against_differences(ft):
    """Central differences of the FP32 loss, summed. Their own error: a third derivative of at most 6 max|w|^3 (max|h|^3 for each of the tokens)
    times h^2 / 6, and the loss's rounding over h."""
    hidden, weight, target = make(3, 8, 11, torch.float32, seed=14, spread=1.0)
    _, grad_hidden, grad_weight = run(ft, hidden, weight, target, "sum")
    step = 2.0 ** -5

    def value(h, w):
        return ft.linear_cross_entropy(h, w, target, reduction="sum").item()

    total = value(hidden, weight)
    for matrix, gradient, other, copies in ((hidden, grad_hidden, weight, 1), (weight, grad_weight, hidden, 3)):
        bound = copies * other.abs().max().item() ** 3 * step ** 2 + 32 * STEP * total / step
        for i in range(matrix.shape[0]):
            for j in range(matrix.shape[1]):
                change = torch.zeros_like(matrix)
                change[i, j] = step
                up, down = ((value(matrix + change, weight), value(matrix - change, weight)) if matrix is hidden else
                            (value(hidden, matrix + change), value(hidden, matrix - change)))
                assert abs((up - down) / (2 * step) - gradient[i, j].item()) <= bound


def test_like_torch(ft):
    hidden, weight, target = make(200, 128, 1000, torch.float32, seed=15)
    target[::5] = -100
    h, w = hidden.clone().requires_grad_(), weight.clone().requires_grad_()
    expected = F.cross_entropy(h @ w.t(), target)
    expected.backward()
    loss, grad_hidden, grad_weight = run(ft, hidden, weight, target)
    assert torch.allclose(loss, expected.detach(), rtol=1e-5) and torch.allclose(grad_hidden, h.grad, rtol=1e-3, atol=1e-6)
    assert torch.allclose(grad_weight, w.grad, rtol=1e-3, atol=1e-6)


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_calls_give_equal_bits(ft, dtype):
    hidden, weight, target = make(700, 256, 5000, dtype, seed=16)
    first = run(ft, hidden, weight, target)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(ft, hidden, weight, target), first))


@pytest.mark.parametrize("dtype", TYPES)
def test_another_stream_and_a_graph(ft, dtype):
    hidden, weight, target = make(300, 128, 900, dtype, seed=17)
    expected = run(ft, hidden, weight, target)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = run(ft, hidden, weight, target)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(on_side, expected))
    held = hidden.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(ft, held, weight, target)
    for fraction in (2, 3):  # other hidden states and other numbers of live tokens
        held.copy_(make(300, 128, 900, dtype, seed=17 + fraction)[0])
        target[::fraction] = -100
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(captured, run(ft, held, weight, target)))


@pytest.mark.parametrize("dtype", TYPES)
def test_a_thread_of_its_own(ft, dtype):
    """A thread that has called nothing of CUDA before, as each of an autograd engine's is once: its memory comes out of the allocator's cache."""
    import threading

    hidden, weight, target = make(600, 1024, 3000, dtype, seed=18)
    expected = run(ft, hidden, weight, target)
    got = []
    thread = threading.Thread(target=lambda: got.extend(run(ft, hidden, weight, target)))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert len(got) == 3 and all(torch.equal(a, b) for a, b in zip(got, expected))


def test_refusals(ft):
    h, w, y = make(10, 16, 20, torch.float32)
    for call, reason in [
        (lambda: ft.linear_cross_entropy(h.cpu(), w, y), "device tensors"), (lambda: ft.linear_cross_entropy(h.double(), w.double(), y), "FP32, FP16 or BF16"),
        (lambda: ft.linear_cross_entropy(h.half(), w, y), "one type"), (lambda: ft.linear_cross_entropy(h, w[:, :8], y), "columns"),
        (lambda: ft.linear_cross_entropy(h, w, y.int()), "INT64"), (lambda: ft.linear_cross_entropy(h, w, y[:9]), "each hidden state"),
        (lambda: ft.linear_cross_entropy(h, w, y, reduction="max"), "reduction"), (lambda: ft.linear_cross_entropy(h, w.t().contiguous().t(), y), "contiguous along"),
        (lambda: ft.linear_cross_entropy(h[:1].expand(10, 16), w, y), "rows overlap"), (lambda: ft.linear_cross_entropy(h, w.view(20, 4, 4), y), "rank two"),
        (lambda: ft.linear_cross_entropy(h, w[:0], y), "empty"),
    ]:
        with pytest.raises(RuntimeError, match=reason):
            call()


# ---- the step in one call: what torch runs wherever there is a reduction and room for the exponentials

def split_in_two(capi, hidden, weight, target, upstream, reduction=1):
    """The loss and the gradients through the two calls of the C interface, the logits computed in each."""
    tokens, depth = hidden.shape
    element = {torch.float32: capi.ELEMENT_FP32, torch.float16: capi.ELEMENT_FP16, torch.bfloat16: capi.ELEMENT_BF16}[hidden.dtype]
    q = capi.LinearCrossEntropy(hidden.data_ptr(), weight.data_ptr(), target.data_ptr(), tokens, weight.shape[0], depth, depth, depth, -100, element, reduction, 0)
    size = max(capi.linear_cross_entropy_workspace_bytes(q, False), capi.linear_cross_entropy_workspace_bytes(q, True))
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    loss, lse = torch.empty((), device="cuda"), torch.empty(tokens, device="cuda")
    grad_hidden, grad_weight = torch.full_like(hidden, math.nan), torch.full_like(weight, math.nan)
    stream = torch.cuda.current_stream().cuda_stream
    capi.linear_cross_entropy(q, loss.data_ptr(), lse.data_ptr(), workspace.data_ptr(), size, stream)
    capi.linear_cross_entropy_backward(q, lse.data_ptr(), upstream.data_ptr(), grad_hidden.data_ptr(), depth, grad_weight.data_ptr(), depth, workspace.data_ptr(),
                                       size, stream)
    torch.cuda.synchronize()
    return loss, grad_hidden, grad_weight


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens, depth, vocabulary", SIZES)
def test_the_two_calls_against_the_definition(ft, capi, tokens, depth, vocabulary, dtype):
    hidden, weight, target = make(tokens, depth, vocabulary, dtype)
    target[1::4] = -100
    oracle = Oracle(hidden, weight, target)
    count = max(1, int(oracle.live.sum()))
    upstream = torch.tensor(48.0, device="cuda")
    loss, grad_hidden, grad_weight = split_in_two(capi, hidden, weight, target, upstream)
    total = oracle.loss.sum() / count
    check(loss, total, oracle.loss_error.sum() / count + 2 * STEP * total.abs(), "loss")
    dh, dh_bound, dw, dw_bound = oracle.gradients(torch.full((tokens,), 48.0 / count, device="cuda", dtype=torch.float64), dtype, step=False)
    check(grad_hidden, dh, dh_bound, "hidden's gradient")
    check(grad_weight, dw, dw_bound, "weight's gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factor", [1.0, 2.0 ** -3, 0.3, 1e-20, 0.0])
def test_any_upstream_gradient_of_the_step(ft, dtype, factor):
    """BF16 gradients wait rounded, and are rounded again where the factor is no power of two; the others are rounded once."""
    hidden, weight, target = make(200, 96, 700, dtype, seed=20)
    one = run(ft, hidden, weight, target)
    got = run(ft, hidden, weight, target, upstream=torch.tensor(factor, device="cuda"))
    oracle = Oracle(hidden, weight, target)
    dh, dh_bound, dw, dw_bound = oracle.gradients(torch.full((200,), factor / 200, device="cuda", dtype=torch.float64), dtype)
    again = torch.finfo(dtype).eps / 2
    for g, value, bound in ((got[1], dh, dh_bound), (got[2], dw, dw_bound)):
        check(g, value, bound + again * value.abs() * 1.01, "gradient")
    if dtype != torch.float16 and math.log2(factor or 1.0) % 1.0 == 0.0 and factor:
        assert torch.equal(got[1], one[1] * factor) and torch.equal(got[2], one[2] * factor)


@pytest.mark.parametrize("dtype", TYPES)
def test_two_backward_passes(ft, dtype):
    """The gradients that wait in the graph are given away only where no other pass can come."""
    hidden, weight, target = make(90, 64, 300, dtype, seed=21)
    h, w = hidden.clone().requires_grad_(), weight.clone().requires_grad_()
    loss = ft.linear_cross_entropy(h, w, target)
    first = torch.autograd.grad(loss, (h, w), torch.tensor(4.0, device="cuda"), retain_graph=True)
    kept = [g.clone() for g in first]
    for g in first:
        g.fill_(math.nan)
    second = torch.autograd.grad(loss, (h, w), torch.tensor(8.0, device="cuda"), retain_graph=True)
    only = torch.autograd.grad(loss, w, torch.tensor(4.0, device="cuda"), retain_graph=True)[0]
    third = torch.autograd.grad(loss, (h, w), torch.tensor(4.0, device="cuda"))
    # (Below FP16's smallest normal number each rounding is half of 2^-24, the first of them doubled here.)
    tiny = 1.5 * 2.0 ** -24 if dtype == torch.float16 else 0.0
    assert all(((a.float() * 2 - b.float()).abs() <= tiny).all() and torch.equal(a, c) for a, b, c in zip(kept, second, third)) and torch.equal(only, kept[1])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, (h, w))
    # The loss in two places of one graph, and accumulation into what is there.
    loss = ft.linear_cross_entropy(h, w, target)
    (loss + 3 * loss).backward()
    assert torch.equal(h.grad, kept[0]) and torch.equal(w.grad, kept[1])
    ft.linear_cross_entropy(h, w, target).mul(4).backward()
    assert torch.equal(w.grad, kept[1] + kept[1])


def test_a_loss_scale_keeps_small_fp16_gradients(ft):
    hidden, weight, target = make(500, 64, 4000, torch.float16, seed=22)
    _, _, grad_weight = run(ft, hidden * 2.0 ** -6, weight, target, upstream=torch.tensor(2.0 ** 16, device="cuda"))
    oracle = Oracle(hidden * 2.0 ** -6, weight, target)
    _, _, dw, dw_bound = oracle.gradients(torch.full((500,), 2.0 ** 16 / 500, device="cuda", dtype=torch.float64), torch.float16)
    check(grad_weight, dw, dw_bound, "weight's gradient")
    assert (dw.abs().median() / 2 ** 16) < torch.finfo(torch.float16).smallest_normal  # unscaled, most would have been lost


def test_what_the_step_refuses(ft, capi):
    hidden, weight, target = make(10, 16, 20, torch.bfloat16)

    def problem(**change):
        fields = dict(hidden=hidden.data_ptr(), weight=weight.data_ptr(), target=target.data_ptr(), tokens=10, vocabulary=20, depth=16, hidden_row_stride=16,
                      weight_row_stride=16, ignore_index=-100, element=8, reduction=1, device=0)
        return capi.LinearCrossEntropy(**{**fields, **change})

    for change, reason in (({"reduction": 0}, "without reduction"), ({"tokens": 0}, "no tokens"), ({"tokens": 1 << 20, "vocabulary": 1 << 20}, "2 GiB")):
        with pytest.raises(capi.FTrainError, match=reason):
            capi.linear_cross_entropy_step_workspace_bytes(problem(**change))
    size = capi.linear_cross_entropy_step_workspace_bytes(problem())
    workspace, out = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty(4096, device="cuda")
    with pytest.raises(capi.FTrainError, match="operands' type"):
        capi.linear_cross_entropy_step(problem(), out.data_ptr(), 7, 0, 0, 0, 0, workspace.data_ptr(), size)
    with pytest.raises(capi.FTrainError, match="workspace of"):
        capi.linear_cross_entropy_step(problem(), out.data_ptr(), 8, 0, 0, 0, 0, workspace.data_ptr(), size - 1)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_tokens_of_a_small_vocabulary(ft, memory_given_back, dtype):
    """More rows of 32 than a grid's second dimension takes (FP32: more logits than the step call takes)."""
    hidden, weight, target = make(32 * 65535 + 1, 8, 3, dtype, seed=14)
    target[::5] = -100
    run_and_check(ft, hidden, weight, target, scale=1024.0)


def test_another_device_than_the_current_one(ft, capi):
    hidden, weight, target = make(10, 16, 20, torch.bfloat16)
    q = capi.LinearCrossEntropy(hidden=hidden.data_ptr(), weight=weight.data_ptr(), target=target.data_ptr(), tokens=10, vocabulary=20, depth=16, hidden_row_stride=16,
                                weight_row_stride=16, ignore_index=-100, element=8, reduction=1, device=1)
    out = torch.empty(1 << 20, device="cuda")
    loss, lse, grad_loss, dh, dw, workspace = (out.data_ptr() + 65536 * i for i in range(6))
    with pytest.raises(capi.FTrainError, match="device 1 must be current"):
        capi.linear_cross_entropy(q, loss, lse, workspace, 1 << 21)
    with pytest.raises(capi.FTrainError, match="device 1 must be current"):
        capi.linear_cross_entropy_backward(q, lse, grad_loss, dh, 16, dw, 16, workspace, 1 << 21)
    with pytest.raises(capi.FTrainError, match="device 1 must be current"):
        capi.linear_cross_entropy_step(q, loss, 8, dh, 16, dw, 16, workspace, 1 << 21)


def test_two_calls_at_once(ft):
    """Two streams, each with its own workspace from the allocator; and in one process two threads' backward passes."""
    cases = [make(700, 256, 5000, torch.bfloat16, seed=30), make(300, 128, 9001, torch.float16, seed=31), make(400, 96, 3001, torch.float32, seed=32)]
    alone = [run(ft, *case) for case in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        together = []
        for case, stream in zip(cases, streams):
            with torch.cuda.stream(stream):
                together.append(run(ft, *case))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for one, other in zip(alone, together) for a, b in zip(one, other))


@pytest.mark.parametrize("dtype", TYPES)
def test_two_graphs_with_a_pool_in_common(ft, dtype):
    """Captured one after the other into one memory pool, so that the second one's workspace may be the first one's; replayed in turn and after new inputs."""
    hidden, weight, target = make(300, 96, 2000, dtype, seed=33)
    inputs = [tuple(x.clone() for x in (hidden, weight, target)) for _ in range(2)]
    leaves = [(h.requires_grad_(), w.requires_grad_(), t) for h, w, t in inputs]
    pool, graphs, results = torch.cuda.graph_pool_handle(), [], []
    for h, w, t in leaves:
        torch.autograd.grad(ft.linear_cross_entropy(h, w, t), (h, w))
    torch.cuda.synchronize()
    for h, w, t in leaves:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            loss = ft.linear_cross_entropy(h, w, t)
            results.append((loss.detach(), *torch.autograd.grad(loss, (h, w))))
        graphs.append(graph)
    for seed in (40, 41):
        for i, (h, w, t) in enumerate(leaves):
            fresh = make(300, 96, 2000, dtype, seed=seed + 10 * i)
            with torch.no_grad():
                h.copy_(fresh[0]), w.copy_(fresh[1])
            t.copy_(fresh[2])
            t[::3 + i] = -100
            graphs[i].replay()
            got = [x.clone() for x in results[i]]
            expected = run(ft, h.detach(), w.detach(), t)
            assert all(torch.equal(a, b) for a, b in zip(got, expected))


@pytest.mark.parametrize("dtype, tokens, vocabulary, reduction", [(torch.bfloat16, 16, 530001, "sum"), (torch.float16, 16, 530001, "none"), (torch.float32, 80, 270001, "sum"),
                                                                  (torch.float32, 20, 530001, "none")])
def test_a_weight_past_32_bits(ft, memory_given_back, dtype, tokens, vocabulary, reduction):
    """More than 2^31 elements (or 2^32 bytes of them), against the formula piece by piece: the sums over the vocabulary, and rows of the weight's gradient from both ends."""
    depth = 4096
    hidden, _, _ = make(tokens, depth, 2, dtype, seed=50)
    weight = torch.empty(vocabulary, depth, device="cuda", dtype=dtype)
    for piece in weight.split(65536):
        piece.copy_(torch.randn(piece.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(piece.shape[0])) * depth ** -0.5)
    target = torch.randint(0, vocabulary, (tokens,), device="cuda")
    target[0], target[1], target[2] = 0, vocabulary - 1, vocabulary // 2
    loss, grad_hidden, grad_weight = run(ft, hidden, weight, target, reduction)
    h = hidden.double()
    z = torch.cat([h @ piece.double().T for piece in weight.split(65536)], 1)
    size = max((h.abs() @ piece.double().abs().T).max().item() for piece in weight.split(65536))
    lse = torch.logsumexp(z, 1)
    # The bounds of Oracle, with the largest of all tokens for each.
    relative = 2 * (depth / 8 + 8) * 2 * STEP * size + (32 + 4 * (z.abs().max() + lse.abs().max()).item()) * 2 * STEP
    expected = lse - z.gather(1, target[:, None])[:, 0]
    if reduction == "sum":
        check(loss, expected.sum(), tokens * relative + 2 * STEP * expected.sum(), "loss")
    else:
        check(loss, expected, torch.full_like(expected, relative), "loss")
    slope = torch.exp(z - lse[:, None])
    half_step = torch.finfo(dtype).eps / 2
    error = slope * (relative + 2.0 ** -11 * (dtype != torch.float32) + half_step + 4 * STEP) + 2.0 ** -38 * (dtype != torch.float32) + 2.0 ** -49 * (dtype == torch.float32)
    slope[torch.arange(tokens), target] -= 1.0
    error[torch.arange(tokens), target] += half_step + 4 * STEP
    value, bound = torch.zeros_like(h), torch.zeros_like(h)
    for s, e, piece in zip(slope.split(65536, 1), error.split(65536, 1), weight.split(65536)):
        value += s @ piece.double()
        bound += (e + (vocabulary / 8 + 24) * 2 * STEP * s.abs()) @ piece.double().abs()
    finfo = torch.finfo(dtype)
    check(grad_hidden, value, bound + 1.01 * half_step * value.abs() + finfo.smallest_normal * finfo.eps, "hidden's gradient")
    for rows in (slice(0, 3000), slice(vocabulary // 2 - 1500, vocabulary // 2 + 1500), slice(vocabulary - 3000, vocabulary)):
        value = slope[:, rows].T @ h
        bound = (error[:, rows].T + (tokens / 8 + 24) * 2 * STEP * slope[:, rows].T.abs()) @ h.abs()
        check(grad_weight[rows], value, bound + 1.01 * half_step * value.abs() + finfo.smallest_normal * finfo.eps, "weight's gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens, depth, vocabulary", [(1, 64, 128), (64, 1024, 700), (300, 96, 1500), (900, 1600, 2000), (1537, 200, 4001)])
def test_the_step_in_two(ft, capi, tokens, depth, vocabulary, dtype):
    """The loss first and gradients twice, with operands and gradients whose rows lie apart: as the step in one where the upstream gradient is 1, and for another one
    against the definition."""
    hidden, weight, target = make(tokens, depth, vocabulary, dtype, seed=60)
    target[2::5] = -100
    wide = torch.full((tokens, depth + 24), math.nan, device="cuda", dtype=dtype)
    wide[:, :depth] = hidden
    q = capi.LinearCrossEntropy(hidden=wide.data_ptr(), weight=weight.data_ptr(), target=target.data_ptr(), tokens=tokens, vocabulary=vocabulary, depth=depth,
                                hidden_row_stride=depth + 24, weight_row_stride=depth, ignore_index=-100, element={torch.float32: 4, torch.float16: 7, torch.bfloat16: 8}[dtype],
                                reduction=1, device=0)
    stream = torch.cuda.current_stream().cuda_stream
    size = capi.linear_cross_entropy_step_workspace_bytes(q)
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    losses, upstreams = torch.full((2,), math.nan, device="cuda"), torch.tensor([1.0, 37.5], device="cuda")
    out = [(torch.full((tokens, depth + 8), 7.0, device="cuda", dtype=dtype), torch.full((vocabulary, depth + 16), 7.0, device="cuda", dtype=dtype)) for _ in range(3)]
    capi.linear_cross_entropy_step(q, losses.data_ptr(), q.element, out[0][0].data_ptr(), depth + 8, out[0][1].data_ptr(), depth + 16, workspace.data_ptr(), size, stream)
    workspace.fill_(255)
    capi.linear_cross_entropy_step_loss(q, losses.data_ptr() + 4, workspace.data_ptr(), size, stream)
    for i in (1, 2):
        capi.linear_cross_entropy_step_gradients(q, upstreams.data_ptr() + 4 * (i - 1), out[i][0].data_ptr(), depth + 8, out[i][1].data_ptr(), depth + 16, workspace.data_ptr(),
                                                 size, stream)
    torch.cuda.synchronize()
    assert torch.equal(losses[0], losses[1]) and torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    assert all((x[:, depth:] == 7).all() for pair in out for x in pair)  # nothing beside the rows
    oracle = Oracle(hidden, weight, target)
    live = max(1, int(oracle.live.sum()))
    dh, dh_bound, dw, dw_bound = oracle.gradients(torch.full((tokens,), 37.5 / live, device="cuda", dtype=torch.float64), dtype)
    # (FP32 by the library's products: one more rounding, by the factor.)
    check(out[2][0][:, :depth], dh, dh_bound + 2 * STEP * dh.abs(), "hidden's gradient")
    check(out[2][1][:, :depth], dw, dw_bound + 2 * STEP * dw.abs(), "weight's gradient")


@pytest.mark.parametrize("dtype", TYPES)
def test_what_changes_between_the_passes(ft, dtype):
    """An operand that is overwritten between the passes is noticed, as torch's own operators do."""
    for which in range(3):
        operands = make(100, 64, 300, dtype, seed=61)
        h, w = operands[0].clone().requires_grad_(), operands[1].clone().requires_grad_()
        loss = ft.linear_cross_entropy(h, w, operands[2])
        with torch.no_grad():
            (h, w, operands[2])[which].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(loss, (h, w))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens, depth, vocabulary, offset, gap", [(5, 1027, 517, 1, 0), (5, 131, 90, 2, 3), (70, 1025, 300, 3, 2), (130, 127, 1001, 5, 4), (300, 2051, 700, 7, 1),
                                                                    (40, 1024, 600, 1, 7), (513, 259, 777, 6, 0), (1, 9, 3, 3, 1)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_weight_at_any_address(ft, dtype, tokens, depth, vocabulary, offset, gap, reduction):
    """Rows at any distance from any element on, in a buffer whose other elements are NaN: copies take whole packs where they can, and nothing of the others is used."""
    hidden, weight, target = make(tokens, depth, vocabulary, dtype, seed=70 + offset)
    buffer = torch.full((offset + vocabulary * (depth + gap),), math.nan, device="cuda", dtype=dtype)
    view = buffer[offset:].view(vocabulary, depth + gap)[:, :depth]
    view.copy_(weight)
    run_and_check(ft, hidden, view, target, reduction)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens, depth, vocabulary, live", [(3000, 72, 300, 1.0), (3000, 72, 300, 0.02), (2000, 257, 129, 0.5), (5000, 128, 1000, 0.0), (6000, 40, 5, 1.0)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_many_tokens_of_few_classes(ft, dtype, tokens, depth, vocabulary, live, reduction):
    """The weight's gradient is summed up in parts over the tokens, of which few live ones leave some empty; together with the other gradient and alone."""
    hidden, weight, target = make(tokens, depth, vocabulary, dtype, seed=80)
    target[torch.rand(tokens, device="cuda", generator=torch.Generator(device="cuda").manual_seed(81)) >= live] = -100
    _, _, grad_weight = run_and_check(ft, hidden, weight, target, reduction, scale=16.0)
    w = weight.clone().requires_grad_()
    loss = ft.linear_cross_entropy(hidden, w, target, reduction=reduction)
    upstream = torch.randn(tokens, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)) * 16.0 if reduction == "none" else torch.tensor(16.0, device="cuda")
    alone, = torch.autograd.grad(loss, w, upstream)
    assert torch.equal(alone, grad_weight)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens, depth, vocabulary, offset, gap", [(70, 1024, 300, 1, 0), (300, 96, 1501, 3, 0), (40, 136, 700, 0, 5), (90, 1027, 601, 0, 5), (130, 129, 515, 1, 0),
                                                                    (64, 1024, 300, 0, 8), (8, 130, 400, 0, 6),
                                                                    (64, 1024, 300, 1, 0), (8, 131, 400, 2, 0)])
def test_a_weight_that_comes_back_from_elsewhere(ft, dtype, tokens, depth, vocabulary, offset, gap):
    """What a saved-tensor hook hands back is another copy: a weight at an odd address or with rows at an odd distance comes back dense and aligned, and one that TMA takes with
    rows that it does not."""
    hidden, weight, target = make(tokens, depth, vocabulary, dtype, seed=90)
    target[::6] = -100
    buffer = torch.full((offset + vocabulary * (depth + gap),), math.nan, device="cuda", dtype=dtype)
    view = buffer[offset:].view(vocabulary, depth + gap)[:, :depth]
    view.copy_(weight)
    expected = run(ft, hidden, view, target)
    h, w = hidden.clone().requires_grad_(), view.detach().requires_grad_()
    with torch.autograd.graph.save_on_cpu():
        loss = ft.linear_cross_entropy(h, w, target)
    grad_hidden, grad_weight = torch.autograd.grad(loss, (h, w))
    assert torch.equal(loss.detach(), expected[0])
    oracle = Oracle(hidden, weight, target)
    each = torch.full((tokens,), 1.0 / int(oracle.live.sum()), device="cuda", dtype=torch.float64)
    dh, dh_bound, dw, dw_bound = oracle.gradients(each, dtype)
    check(grad_hidden, dh, dh_bound, "hidden's gradient")
    check(grad_weight, dw, dw_bound, "weight's gradient")


@pytest.mark.parametrize("dtype, tokens, depth, vocabulary", [(torch.bfloat16, 2048, 512, 32768), (torch.float16, 600, 512, 50000), (torch.float32, 400, 512, 32768), (torch.float32, 1200, 1200, 9000)])
def test_what_waits_in_the_graph(ft, memory_given_back, dtype, tokens, depth, vocabulary):
    """From the forward pass to the backward one: the slopes (FP32 operands: three halves each, or one number where they go through the library's products), the hidden states, a
    copy of an FP32 weight; not what one of the passes needs for itself."""
    hidden, weight, target = make(tokens, depth, vocabulary, dtype, seed=98)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    before = torch.cuda.memory_allocated()
    loss = ft.linear_cross_entropy(h, w, target)
    kept = torch.cuda.memory_allocated() - before
    rows, columns, bytes = -(-tokens // 256) * 256, -(-vocabulary // 256) * 256, {torch.float32: 6, torch.float16: 2, torch.bfloat16: 2}[dtype]
    pitch = -(-depth // 8) * 8
    limit = rows * columns * bytes + rows * pitch * bytes + (vocabulary * pitch * 6 if dtype == torch.float32 else 0)
    assert kept <= limit + (4 << 20)  # (the lists, and what the allocator rounds up to)
    loss.backward()


def test_what_the_kept_memory_has_to_be(ft, capi):
    hidden, weight, target = make(10, 16, 20, torch.bfloat16)
    buffer = torch.zeros(20 * 17, device="cuda", dtype=torch.bfloat16)

    def problem(weight, stride=16):
        return capi.LinearCrossEntropy(hidden=hidden.data_ptr(), weight=weight.data_ptr(), target=target.data_ptr(), tokens=10, vocabulary=20, depth=16, hidden_row_stride=16,
                                       weight_row_stride=stride, ignore_index=-100, element=8, reduction=1, device=0)

    q, odd = problem(weight), problem(buffer, 17)
    kept, size = capi.linear_cross_entropy_step_loss_bytes(q)
    with_copy, _ = capi.linear_cross_entropy_step_loss_bytes(odd)
    assert with_copy > kept
    memory, out = torch.empty(1 << 20, dtype=torch.uint8, device="cuda"), torch.empty(4096, device="cuda")
    loss, at = out.data_ptr(), memory.data_ptr()
    for bytes, where, workspace, reason in ((kept - 1, at, size, "kept memory of"), (kept + 256, at, size, "kept memory of"), (kept, at + 128, size, "kept memory of"),
                                            (kept, 0, size, "kept memory of"), (kept, at, size - 1, "workspace of")):
        with pytest.raises(capi.FTrainError, match=reason):
            capi.linear_cross_entropy_step_loss_kept(q, loss, where, bytes, at + (1 << 19), workspace)
    for p in (q, odd):  # either size is one that a loss can have left, whatever the weight's address is by now
        for bytes in (kept, with_copy):
            assert capi.linear_cross_entropy_step_gradients_bytes(p, bytes) > 0
        with pytest.raises(capi.FTrainError, match="kept memory has"):
            capi.linear_cross_entropy_step_gradients_bytes(p, kept + 256)
        with pytest.raises(capi.FTrainError, match="kept memory has"):
            capi.linear_cross_entropy_step_gradients_kept(p, loss, loss + 1024, 16, loss + 2048, 16, at, with_copy + 256, at + (1 << 19), 1 << 19)
    # With both in one workspace its size says what was kept.
    whole = capi.linear_cross_entropy_step_workspace_bytes(q)
    for bytes in (whole - 1, whole + 1, capi.linear_cross_entropy_step_workspace_bytes(odd)):
        with pytest.raises(capi.FTrainError, match="no more and no less"):
            capi.linear_cross_entropy_step_gradients(q, loss, loss + 1024, 16, loss + 2048, 16, at, bytes)


@pytest.mark.parametrize("dtype, depth, vocabulary", [(torch.float32, 4096, 90001), (torch.bfloat16, 4097, 262145)])
def test_a_large_copy_of_the_weight_does_not_wait_in_the_graph(ft, capi, memory_given_back, dtype, depth, vocabulary):
    """Three halves for each element of an FP32 weight, or the copy of one that TMA does not take: beyond the 2 GiB they are made again for the gradients."""
    hidden, _, target = make(100, depth, vocabulary, dtype, seed=99)
    target[::5] = -100
    weight = torch.empty(vocabulary, depth, device="cuda", dtype=dtype)
    for piece in weight.split(65536):
        piece.copy_(torch.randn(piece.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(piece.shape[0])) * depth ** -0.5)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    before = torch.cuda.memory_allocated()
    loss = ft.linear_cross_entropy(h, w, target)
    assert torch.cuda.memory_allocated() - before <= 256 * (vocabulary + 255) * (6 if dtype == torch.float32 else 2) + (16 << 20)
    grad_hidden, grad_weight = torch.autograd.grad(loss, (h, w))
    loss2, hidden2, weight2 = split_in_two(capi, hidden.detach(), weight.detach(), target, torch.ones((), device="cuda"))
    # Either form is off by its slopes' rounding (two of them in the step) and its results' own.
    tolerance = {torch.float32: 2e-6, torch.bfloat16: 2.0 ** -8}[dtype] * 3
    assert abs(loss.item() - loss2.item()) <= 2e-6 * loss2.item()
    assert (grad_hidden - hidden2).float().norm() <= tolerance * hidden2.float().norm() and (grad_weight - weight2).float().norm() <= tolerance * weight2.float().norm()


@pytest.mark.parametrize("dtype, tokens, vocabulary", [(torch.bfloat16, 8192, 131072), (torch.float32, 3000, 65536)])
def test_where_there_is_no_room_for_the_exponentials(ft, memory_given_back, dtype, tokens, vocabulary):
    """With less memory left than the step wants, the gradients come from the form that goes through the vocabulary piece by piece."""
    hidden, weight, target = make(tokens, 64, vocabulary, dtype, seed=97)
    target[::5] = -100
    expected = run(ft, hidden, weight, target)
    torch.cuda.synchronize()
    gc.collect()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    total = torch.cuda.get_device_properties(0).total_memory
    before = torch.cuda.memory_reserved()
    torch.cuda.set_per_process_memory_fraction((before + 1.25 * 2 ** 30) / total)
    try:
        for _ in range(3):  # the first of these asks for the room, the others remember
            got = run(ft, hidden, weight, target)
            assert torch.cuda.max_memory_reserved() <= before + 1.25 * 2 ** 30
            tolerance = 2e-6 if dtype == torch.float32 else torch.finfo(dtype).eps
            assert abs(got[0].item() - expected[0].item()) <= 1e-6 * expected[0].item()
            assert all((a.double() - b.double()).norm() <= 2 * tolerance * b.double().norm() for a, b in zip(got[1:], expected[1:]))
            del got
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    # With the memory back, the step is asked for again in the end: equal bits.
    for _ in range(70):
        got = run(ft, hidden, weight, target)
    assert all(torch.equal(a, b) for a, b in zip(got, expected))


@pytest.mark.parametrize("tokens, depth, vocabulary", [(200, 96, 700), (300, 200, 5001)])
def test_fp16_rows_of_small_upstream_gradients(ft, tokens, depth, vocabulary):
    """A token's row of the hidden states' gradient is as exact beside upstream gradients that are 2^22 times larger as it is alone: against its own bound, which has
    no part of any other token's."""
    hidden, weight, target = make(tokens, depth, vocabulary, torch.float16, seed=95)
    target[::9] = -100
    oracle = Oracle(hidden, weight, target)
    upstream = torch.randn(tokens, device="cuda").sign() * torch.exp2(14.0 - torch.arange(tokens, device="cuda") % 23)
    upstream[3], upstream[4] = 0.0, 2.0 ** -30
    _, grad_hidden, grad_weight = run(ft, hidden, weight, target, "none", upstream)
    dh, dh_bound, dw, dw_bound = oracle.gradients(upstream, torch.float16, step=False)
    # oracle's bound allows 2^-38 of the largest upstream gradient in every slope; of the token's own it is 2^-38 as well.
    extra = ((upstream.abs().max() - upstream.abs()) * 2.0 ** -38).double()[:, None] * oracle.w.abs().sum(0)[None, :]
    check(grad_hidden, dh, dh_bound - extra, "hidden's gradient")
    check(grad_weight, dw, dw_bound, "weight's gradient")
    assert not grad_hidden[3].any()
    h, w = hidden.clone().requires_grad_(), weight.clone().requires_grad_()
    loss = ft.linear_cross_entropy(h, w, target, reduction="none")
    for alone, both in ((h, grad_hidden), (w, grad_weight)):
        assert torch.equal(torch.autograd.grad(loss, alone, upstream, retain_graph=True)[0], both)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factor", [2.0 ** -3, 0.3, 1e-20, 700.0])
def test_an_upstream_gradient_is_multiplied_in_before_the_rounding(ft, dtype, factor):
    """One rounding to the results' type, whatever the factor. (FP32 as three BF16 matrices: the factor and the sum, a step each, are in the bound for sums.)"""
    hidden, weight, target = make(200, 96, 700, dtype, seed=20)
    _, grad_hidden, grad_weight = run(ft, hidden, weight, target, upstream=torch.tensor(factor, device="cuda"))
    oracle = Oracle(hidden, weight, target)
    dh, dh_bound, dw, dw_bound = oracle.gradients(torch.full((200,), factor / 200, device="cuda", dtype=torch.float64), dtype)
    check(grad_hidden, dh, dh_bound, "hidden's gradient")
    check(grad_weight, dw, dw_bound, "weight's gradient")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens, depth, vocabulary", [(1, 64, 128), (300, 96, 1500), (70, 1025, 300), (1537, 200, 4001), (3000, 72, 300), (2000, 257, 129)])
def test_fp32_gradients_of_16_bit_operands(ft, capi, tokens, depth, vocabulary, dtype):
    """The step in one with gradients in FP32: an odd depth, sums in parts over the tokens, rows apart; nothing is rounded to 16 bits."""
    hidden, weight, target = make(tokens, depth, vocabulary, dtype, seed=96)
    target[2::5] = -100
    q = capi.LinearCrossEntropy(hidden=hidden.data_ptr(), weight=weight.data_ptr(), target=target.data_ptr(), tokens=tokens, vocabulary=vocabulary, depth=depth,
                                hidden_row_stride=depth, weight_row_stride=depth, ignore_index=-100, element=7 if dtype == torch.float16 else 8, reduction=2, device=0)
    size = capi.linear_cross_entropy_step_workspace_bytes(q)
    workspace = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    loss = torch.empty((), device="cuda")
    grad_hidden, grad_weight = (torch.full((rows, depth + 3), 7.0, device="cuda") for rows in (tokens, vocabulary))
    capi.linear_cross_entropy_step(q, loss.data_ptr(), capi.ELEMENT_FP32, grad_hidden.data_ptr(), depth + 3, grad_weight.data_ptr(), depth + 3, workspace.data_ptr(), size,
                                   torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    oracle = Oracle(hidden, weight, target)
    dh, dh_bound, dw, dw_bound = oracle.gradients(torch.ones(tokens, device="cuda", dtype=torch.float64), dtype)
    # The bounds but for the results' rounding to 16 bits, in whose place comes FP32's; (the smallest FP16 number is in them, and matters to none of these).
    half_step = torch.finfo(dtype).eps / 2
    check(grad_hidden[:, :depth], dh, dh_bound - (1.01 * half_step - STEP) * dh.abs(), "hidden's gradient")
    check(grad_weight[:, :depth], dw, dw_bound - (1.01 * half_step - STEP) * dw.abs(), "weight's gradient")
    assert (grad_hidden[:, depth:] == 7).all() and (grad_weight[:, depth:] == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens, depth, vocabulary", [(5, 131, 90), (70, 1025, 300), (300, 127, 1501)])
def test_the_step_in_two_over_a_weight_that_is_copied(ft, capi, tokens, depth, vocabulary, dtype):
    """One workspace, a weight at an odd address with rows at an odd distance, gradients twice: as torch's graph makes them."""
    hidden, weight, target = make(tokens, depth, vocabulary, dtype, seed=100)
    target[2::5] = -100
    buffer = torch.full((3 + vocabulary * (depth + 1),), math.nan, device="cuda", dtype=dtype)
    view = buffer[3:].view(vocabulary, depth + 1)[:, :depth]
    view.copy_(weight)
    loss, expected_hidden, expected_weight = run(ft, hidden, view, target, upstream=torch.tensor(37.5, device="cuda"))
    q = capi.LinearCrossEntropy(hidden=hidden.data_ptr(), weight=view.data_ptr(), target=target.data_ptr(), tokens=tokens, vocabulary=vocabulary, depth=depth,
                                hidden_row_stride=depth, weight_row_stride=depth + 1, ignore_index=-100, element={torch.float32: 4, torch.float16: 7, torch.bfloat16: 8}[dtype],
                                reduction=1, device=0)
    stream = torch.cuda.current_stream().cuda_stream
    size = capi.linear_cross_entropy_step_workspace_bytes(q)
    workspace = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    numbers = torch.tensor([math.nan, 37.5], device="cuda")
    capi.linear_cross_entropy_step_loss(q, numbers.data_ptr(), workspace.data_ptr(), size, stream)
    for _ in range(2):
        grad_hidden, grad_weight = torch.full_like(hidden, math.nan), torch.full_like(weight, math.nan)
        capi.linear_cross_entropy_step_gradients(q, numbers.data_ptr() + 4, grad_hidden.data_ptr(), depth, grad_weight.data_ptr(), depth, workspace.data_ptr(), size, stream)
        torch.cuda.synchronize()
        assert torch.equal(numbers[0], loss) and torch.equal(grad_hidden, expected_hidden) and torch.equal(grad_weight, expected_weight)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_logits_computed_again_on_demand(ft, memory_given_back, dtype):
    """recompute=True keeps one number a token, and gives the gradients that a definition of its own bounds."""
    hidden, weight, target = make(1000, 128, 9001, dtype, seed=101)
    target[::6] = -100
    h, w = hidden.clone().requires_grad_(), weight.clone().requires_grad_()
    before = torch.cuda.memory_allocated()
    loss = ft.linear_cross_entropy(h, w, target, reduction="sum", recompute=True)
    assert torch.cuda.memory_allocated() - before <= 4 * 1000 + 4096
    grad_hidden, grad_weight = torch.autograd.grad(loss, (h, w), torch.tensor(3.0, device="cuda"))
    oracle = Oracle(hidden, weight, target)
    dh, dh_bound, dw, dw_bound = oracle.gradients(torch.full((1000,), 3.0, device="cuda", dtype=torch.float64), dtype, step=False)
    check(loss.detach(), oracle.loss.sum(), oracle.loss_error.sum() + 2 * STEP * oracle.loss.sum(), "loss")
    check(grad_hidden, dh, dh_bound, "hidden's gradient")
    check(grad_weight, dw, dw_bound, "weight's gradient")
    assert torch.equal(ft.linear_cross_entropy(hidden, weight, target, recompute=True), ft.linear_cross_entropy(hidden, weight, target))
