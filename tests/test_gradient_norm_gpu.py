"""grad_norm, clip_grads and clip_grad_norm_ against the definition in 64 bits."""
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


def exact_norm(gradients, norm_type=2.0):
    if norm_type == math.inf:
        return max((g.double().abs().max().item() for g in gradients if g.numel()), default=0.0)
    return math.sqrt(math.fsum((g.double() ** 2).sum().item() for g in gradients))


# Squares are added up in FP32 over at most eight elements, eight roundings of which the root halves the effect; one more for the result.
NORM_TOLERANCE = 5 * STEP


def check_norm(norm, expected):
    assert norm.shape == () and norm.dtype == torch.float32
    assert abs(norm.item() - expected) <= NORM_TOLERANCE * expected, (norm.item(), expected)


def check_clipped(out, gradient, norm, max_norm):
    """The factor carries the norm's error and a rounding, the product a rounding, and the result that of its type."""
    factor = min(1.0, max_norm / (norm + 1e-6))
    expected = gradient.double() * factor
    relative = NORM_TOLERANCE + 2 * STEP + (torch.finfo(out.dtype).eps / 2 if out.dtype != torch.float32 else 0.0)
    smallest = torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps / 2  # half a step among the subnormal numbers
    error = (out.double() - expected).abs() - relative * expected.abs()
    assert error.max().item() <= smallest if error.numel() else True


def make(shapes, dtype, seed=0, scale=1.0):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(shape, device="cuda", generator=generator).mul_(scale).to(dtype) for shape in shapes]


SHAPES = {
    "one element": [(1,)],
    "a few": [(7,), (33, 5), (1,), (4096,), (4097,), (3, 5, 7)],
    "empty among them": [(0,), (5, 0, 3), (17,), (0,)],
    "a chunk and its neighbours": [(4095,), (4096,), (4097,), (8192,), (12289,)],
    "large": [(1023, 2049), (11,), (4096, 1024)],
}


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shapes", SHAPES.values(), ids=SHAPES.keys())
def test_norm(ft, shapes, dtype, norm_type):
    gradients = make(shapes, dtype)
    check_norm(ft.grad_norm(gradients, norm_type), exact_norm(gradients, norm_type))


@pytest.mark.parametrize("count", [63, 64, 65, 480, 481, 1500])
def test_any_number_of_tensors_of_mixed_types(ft, count):
    gradients = [make([(1 + 37 * i % 301,)], TYPES[i % 3], seed=i)[0] for i in range(count)]
    expected = exact_norm(gradients)
    check_norm(ft.grad_norm(gradients), expected)
    outs = [torch.full_like(g, float("nan")) for g in gradients]
    check_norm(ft.clip_grads(gradients, 0.5, out=outs), expected)
    for g, out in zip(gradients, outs):
        check_clipped(out, g, expected, 0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out_dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 1])
def test_clip_into_buffers_of_any_type_and_alignment(ft, dtype, out_dtype, shift):
    shapes = [(4096,), (5,), (127, 65), (3 * 4096 + 1,), (8191,)]
    gradients = make(shapes, dtype, seed=3)
    norm = exact_norm(gradients)
    sizes = [math.prod(s) for s in shapes]
    flat = torch.full((sum(sizes) + shift,), 7.0, device="cuda", dtype=out_dtype)
    outs = [piece.view(shape) for piece, shape in zip(flat[shift:].split(sizes), shapes)]
    kept = [g.clone() for g in gradients]
    check_norm(ft.clip_grads(gradients, 2.0, out=outs), norm)
    for g, k, out in zip(gradients, kept, outs):
        assert torch.equal(g, k)
        check_clipped(out, g, norm, 2.0)
    assert (flat[:shift] == 7.0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_clip_in_place_from_any_address(ft, dtype, shift):
    storage = make([(70001,)], dtype, seed=5)[0]
    before = storage.clone()
    gradients = [storage[shift:shift + 20000], storage[20010:20011], storage[30001:60000]]
    originals = [g.clone() for g in gradients]
    norm = exact_norm(originals)
    version = storage._version
    check_norm(ft.clip_grads(gradients, 1.0), norm)
    assert storage._version > version
    for g, original in zip(gradients, originals):
        check_clipped(g, original, norm, 1.0)
    for untouched in (slice(0, shift), slice(20000 + shift, 20010), slice(20011, 30001), slice(60000, None)):
        assert torch.equal(storage[untouched], before[untouched])


def test_windows_transposes_and_channels_last(ft):
    matrix = make([(300, 96)], torch.float32, seed=8)[0]
    before = matrix.clone()
    left, right = matrix[:, :31], matrix[:, 31:90]
    picture = make([(2, 5, 7, 9)], torch.float32, seed=9)[0].to(memory_format=torch.channels_last)
    turned = make([(40, 60)], torch.bfloat16, seed=10)[0].t()
    gradients = [left, right, picture, turned]
    originals = [g.clone() for g in gradients]
    norm = exact_norm(originals)
    check_norm(ft.grad_norm(gradients), norm)
    check_norm(ft.clip_grads(gradients, 0.25), norm)
    for g, original in zip(gradients, originals):
        check_clipped(g, original, norm, 0.25)
    assert torch.equal(matrix[:, 90:], before[:, 90:])


def test_a_factor_of_one_changes_nothing(ft):
    gradients = make([(1000,), (17, 3)], torch.float32, scale=1e-3)
    kept = [g.clone() for g in gradients]
    norm = exact_norm(gradients)
    check_norm(ft.clip_grads(gradients, 10.0), norm)
    outs = [torch.zeros_like(g) for g in gradients]
    ft.clip_grads(gradients, math.inf, out=outs)
    for g, k, out in zip(gradients, kept, outs):
        assert torch.equal(g, k) and torch.equal(out, k)


def test_zeros_and_a_limit_of_zero(ft):
    zeros = [torch.zeros(5000, device="cuda"), torch.zeros(3, device="cuda", dtype=torch.bfloat16)]
    assert ft.clip_grads(zeros, 1.0).item() == 0.0 and not any(z.any() for z in zeros)
    ones = [torch.ones(9, device="cuda")]
    assert ft.clip_grads(ones, 0.0).item() == 3.0 and not ones[0].any()
    assert ft.grad_norm([torch.empty(0, device="cuda")]).item() == 0.0


@pytest.mark.parametrize("magnitude", [1e-42, 1e-30, 1e-20, 1e19, 1e30, 3e38])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_squares_outside_of_fp32(ft, dtype, magnitude):
    """Squares of these under- or overflow in FP32."""
    gradients = [torch.full((n,), magnitude, device="cuda").to(dtype) for n in (1, 5, 100)]
    gradients[2][::3] = 0
    expected = exact_norm(gradients)
    if expected <= torch.finfo(torch.float32).max:
        got = ft.grad_norm(gradients).item()
        assert abs(got - expected) <= NORM_TOLERANCE * expected + 2.0 ** -150  # half a step of the smallest numbers
    else:
        assert ft.grad_norm(gradients).item() == math.inf
    assert ft.grad_norm(gradients, math.inf).item() == exact_norm(gradients, math.inf)


def test_large_and_small_in_one_tensor(ft):
    gradient = torch.full((10000,), 1e-25, device="cuda")
    gradient[1234] = 1e25
    check_norm(ft.grad_norm([gradient]), exact_norm([gradient]))


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_infinities_and_nan(ft, norm_type):
    base = make([(9000,), (50,)], torch.float32)
    for bad in (math.inf, -math.inf, math.nan):
        gradients = [g.clone() for g in base]
        gradients[0][8191] = bad
        norm = ft.clip_grads(gradients, 1.0, norm_type)
        if math.isnan(bad):
            assert math.isnan(norm.item()) and all(torch.isnan(g).all() for g in gradients)
        else:
            assert norm.item() == math.inf
            assert torch.isnan(gradients[0][8191]) and torch.isnan(gradients[0]).sum() == 1 and not gradients[1].any()


def test_equal_calls_give_equal_bits(ft):
    gradients = make([(1 << 20,), (777777,), (13,)], torch.bfloat16)
    norms = {ft.grad_norm(gradients).item() for _ in range(5)}
    assert len(norms) == 1


def test_many_elements_past_32_bits(ft, memory_given_back):
    gradient = torch.zeros((1 << 32) + 5, device="cuda", dtype=torch.bfloat16)
    gradient[-1], gradient[1 << 31] = 3.0, 4.0
    assert ft.clip_grads([gradient], 2.5).item() == 5.0
    assert gradient[-1].item() == 1.5 and gradient[1 << 31].item() == 2.0 and gradient.count_nonzero().item() == 2


def test_the_same_gradient_twice(ft):
    g = make([(100,)], torch.float32)[0]
    check_norm(ft.grad_norm([g, g]), math.sqrt(2) * exact_norm([g]))
    with pytest.raises(RuntimeError, match="overlaps"):
        ft.clip_grads([g, g], 1.0)


def test_clip_grad_norm_like_torch(ft):
    torch.manual_seed(0)
    layers = [torch.nn.Sequential(torch.nn.Linear(65, 33), torch.nn.GELU(), torch.nn.Linear(33, 9)).cuda() for _ in range(2)]
    layers[1].load_state_dict(layers[0].state_dict())
    x = torch.randn(20, 65, device="cuda")
    for layer in layers:
        layer(x).square().sum().backward()
        layer[2].bias.grad = None
    expected = torch.nn.utils.clip_grad_norm_(layers[0].parameters(), 0.1)
    got = ft.clip_grad_norm_(layers[1].parameters(), 0.1)
    assert abs(got.item() - expected.item()) <= 1e-5 * expected.item()  # torch sums in FP32
    for a, b in zip(layers[0].parameters(), layers[1].parameters()):
        if a.grad is not None:
            assert torch.allclose(a.grad, b.grad, rtol=2e-5, atol=0)
    assert ft.clip_grad_norm_([], 1.0).item() == 0.0
    single = torch.nn.Parameter(torch.ones(4, device="cuda"))
    single.grad = torch.full_like(single, math.inf)
    with pytest.raises(RuntimeError, match="not finite"):
        ft.clip_grad_norm_(single, 1.0, error_if_nonfinite=True)
    assert torch.isinf(single.grad).all()


def test_another_stream_and_a_graph(ft):
    gradients = make([(300000,), (77,)], torch.float32)
    norm = exact_norm(gradients)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check_norm(ft.grad_norm(gradients), norm)
    torch.cuda.current_stream().wait_stream(side)
    outs = [torch.empty_like(g) for g in gradients]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ft.clip_grads(gradients, 1.0, out=outs)
    for factor in (1.0, 3.0):
        for g in gradients:
            g.mul_(factor)
        graph.replay()
        check_norm(captured, exact_norm(gradients))
        for g, out in zip(gradients, outs):
            check_clipped(out, g, exact_norm(gradients), 1.0)


def test_refusals(ft):
    g = torch.ones(8, device="cuda")
    for call, reason in [
        (lambda: ft.grad_norm([torch.ones(8)]), "device tensor"), (lambda: ft.grad_norm([g.double()]), "FP32, FP16 or BF16"),
        (lambda: ft.grad_norm([g], 1.0), "norm_type"), (lambda: ft.clip_grads([g], -1.0), "max_norm"), (lambda: ft.clip_grads([g], math.nan), "max_norm"),
        (lambda: ft.clip_grads([g], 1.0, out=[]), "one tensor for each"), (lambda: ft.clip_grads([g], 1.0, out=[torch.ones(7, device="cuda")]), "shape"),
        (lambda: ft.grad_norm([torch.ones(4, 6, 8, device="cuda")[:, ::2, ::2]]), "neighbouring"), (lambda: ft.grad_norm([g[:1].expand(5)]), "neighbouring"),
        (lambda: ft.clip_grads([torch.ones(4, 6, device="cuda")], 1.0, out=[torch.ones(6, 4, device="cuda").t()]), "neighbouring"),
        (lambda: ft.clip_grads([torch.nn.Parameter(g)], 1.0), "require a gradient"),
    ]:
        with pytest.raises(RuntimeError, match=reason):
            call()


@pytest.mark.parametrize("count", [1, 70, 600])
def test_scale_by_a_number_on_the_device(ft, capi, count):
    elements = {torch.float32: capi.ELEMENT_FP32, torch.bfloat16: capi.ELEMENT_BF16, torch.float16: capi.ELEMENT_FP16}
    gradients = [make([(1 + 53 * i % 777,)], TYPES[i % 3], seed=i)[0] for i in range(count)]
    outs = [torch.empty_like(g, dtype=TYPES[(i // 3) % 3]) for i, g in enumerate(gradients)]
    described = [capi.Gradient(g.data_ptr(), o.data_ptr(), 1, g.numel(), 0, 0, elements[g.dtype], elements[o.dtype]) for g, o in zip(gradients, outs)]
    factor = torch.tensor(0.7, device="cuda")
    capi.gradient_scale(described, factor.data_ptr(), 0, torch.cuda.current_stream().cuda_stream)
    for g, o in zip(gradients, outs):
        assert torch.equal(o, (g.float() * factor).to(o.dtype))


@pytest.mark.parametrize("count, apart", [(608, True), (609, True), (1152, False), (1153, False), (1300, True)])
def test_lists_that_fill_a_launch(ft, count, apart):
    """Dense tensors, or windows of wider matrices among them; every one is clipped once."""
    gradients, wide = [], []
    for i in range(count):
        matrix = make([(3, 5 + i % 9)], TYPES[i % 3], seed=i)[0]
        wide.append((matrix, matrix.clone()))
        gradients.append(matrix[:, :4] if apart and i % 2 else matrix)
    originals = [g.clone() for g in gradients]
    norm = exact_norm(originals)
    check_norm(ft.grad_norm(gradients), norm)
    check_norm(ft.clip_grads(gradients, 1.0), norm)
    for i, (g, original) in enumerate(zip(gradients, originals)):
        check_clipped(g, original, norm, 1.0)
        if apart and i % 2:
            assert torch.equal(wide[i][0][:, 4:], wide[i][1][:, 4:])


def test_another_device_than_the_current_one(ft, capi):
    g, out = torch.ones(100, device="cuda"), torch.empty(1 << 16, device="cuda")
    gradients = [capi.Gradient(data=g.data_ptr(), out=g.data_ptr(), rows=1, cols=100, row_stride=0, out_row_stride=0, element=4, out_element=4)]
    with pytest.raises(capi.FTrainError, match="device 1 must be current"):
        capi.gradient_scale(gradients, out.data_ptr(), device=1)
    assert (g == 1).all()


def test_what_would_leave_autograd_is_refused(ft):
    """A penalty on a gradient's norm would otherwise train on nothing."""
    x = torch.ones(5, device="cuda", requires_grad=True)
    gradient, = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    for call in (lambda: ft.grad_norm([gradient]), lambda: ft.grad_norm([x]), lambda: ft.clip_grads([gradient], 1.0), lambda: ft.clip_grads([gradient], 1.0, out=[torch.empty(5, device="cuda")])):
        with pytest.raises(RuntimeError, match="must not require a gradient: the norm is not differentiable"):
            call()
    with torch.no_grad():
        check_norm(ft.grad_norm([gradient, x]), exact_norm([gradient.detach(), x.detach()]))
    check_norm(ft.grad_norm([gradient.detach()]), exact_norm([gradient.detach()]))
    loss = (x * 2).sum()
    loss.backward()
    x.grad.requires_grad_()  # clip_grad_norm_ works in place and records nothing
    check_norm(ft.clip_grad_norm_([x], 1.0), math.sqrt(20.0))
