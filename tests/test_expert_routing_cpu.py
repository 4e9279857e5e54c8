"""What ftcuda_expert_routing and its gradient refuse: checked before anything touches a device, so made-up addresses do."""
import pytest

OUTPUTS = (0x1000000, 0x2000000, 0x3000000, 0x3100000, 0x3200000)
WORKSPACE = (0x4000000, 16 << 20)


def routing(capi, **change):
    fields = dict(logits=0x10000000, mask=None, tokens=100, row_stride=64, experts=64, top_k=8, normalize=1, element=4, device=0)
    return capi.Routing(**{**fields, **change})


def refuse(capi, reason, call, *arguments):
    with pytest.raises(capi.FTrainError) as info:
        call(*arguments)
    assert reason in info.value.message, info.value.message


@pytest.mark.parametrize("change, reason", [
    ({"element": 1}, "FP32, FP16 or BF16"), ({"experts": 0}, "1 to 1024"), ({"experts": 1025, "row_stride": 1025}, "1 to 1024"), ({"top_k": 0}, "top_k"),
    ({"top_k": 65}, "top_k"), ({"top_k": 33}, "top_k"), ({"tokens": 1 << 31}, "too many tokens"), ({"logits": None}, "no address"),
    ({"logits": 0x10000002}, "multiple"), ({"row_stride": 63}, "rows overlap"), ({"row_stride": -64}, "rows overlap"), ({"row_stride": 0}, "rows overlap"),
])
def test_problems_that_cannot_be(capi, change, reason):
    r = routing(capi, **change)
    refuse(capi, reason, capi.expert_routing, r, *OUTPUTS, *WORKSPACE)
    refuse(capi, reason, capi.expert_routing_backward, r, *OUTPUTS[:4], 0, 0, 0x5000000, 64)


def test_addresses_that_cannot_be(capi):
    r = routing(capi)
    for i in range(5):
        for bad in (0, OUTPUTS[i] + 2):
            refuse(capi, "an output has no address", capi.expert_routing, r, *OUTPUTS[:i], bad, *OUTPUTS[i + 1:], *WORKSPACE)
    needed = capi.expert_routing_workspace_bytes(r)
    for workspace in ((0, needed), (0x4000002, needed), (0x4000000, needed - 1)):
        refuse(capi, "workspace of", capi.expert_routing, r, *OUTPUTS, *workspace)
    for i in range(4):
        refuse(capi, "an input has no address", capi.expert_routing_backward, r, *OUTPUTS[:i], 0, *OUTPUTS[i + 1:4], 0, 0, 0x5000000, 64)
    for gradients in ((0x6000001, 0), (0, 0x6000002)):
        refuse(capi, "an input has no address", capi.expert_routing_backward, r, *OUTPUTS[:4], *gradients, 0x5000000, 64)
    refuse(capi, "the gradient has no address", capi.expert_routing_backward, r, *OUTPUTS[:4], 0, 0, 0, 64)
    refuse(capi, "the gradient has no address", capi.expert_routing_backward, r, *OUTPUTS[:4], 0, 0, 0x5000002, 64)
    refuse(capi, "gradient's rows overlap", capi.expert_routing_backward, r, *OUTPUTS[:4], 0, 0, 0x5000000, 63)


def test_the_workspace_is_bounded(capi):
    assert capi.expert_routing_workspace_bytes(routing(capi, tokens=0)) > 0
    assert capi.expert_routing_workspace_bytes(routing(capi, tokens=(1 << 31) - 1, experts=1024, row_stride=1024)) <= 5 << 20


def test_a_gradient_across_what_is_read(capi):
    r, wide = routing(capi, element=8), routing(capi, row_stride=192)
    across = [(r, OUTPUTS[:4], 0, 0, 0x10000000 + 2, 64), (r, OUTPUTS[:4], 0, 0, 0x10000000 - 12798, 64), (r, OUTPUTS[:4], 0, 0, 0x10000000, 65),
              (r, OUTPUTS[:4], 0, 0, 0x10000000 + 128 * 99 + 126, 64), (wide, OUTPUTS[:4], 0, 0, 0x10000000 + 4 * 63, 192), (wide, OUTPUTS[:4], 0, 0, 0x10000000 + 4 * 129, 192),
              (wide, OUTPUTS[:4], 0, 0, 0x10000000 + 4 * 64, 191)]
    for i in range(4):  # the last byte of an input, and one in the gradient's middle
        across += [(r, OUTPUTS[:4], 0, 0, OUTPUTS[i] + (3200, 3200, 256, 4)[i] - 2, 64), (r, OUTPUTS[:4], 0, 0, OUTPUTS[i] - 6400, 64)]
    across += [(r, OUTPUTS[:4], 0x6000000, 0, 0x6000000 + 3198, 64), (r, OUTPUTS[:4], 0, 0x6000000, 0x6000000 - 12798, 64)]
    for problem, inputs, grad_weights, grad_loss, out, stride in across:
        refuse(capi, "lies across", capi.expert_routing_backward, problem, *inputs, grad_weights, grad_loss, out, stride)


def test_a_gradient_over_or_beside_the_logits_reaches_the_device_check(capi):
    import torch

    if torch.cuda.is_available():
        pytest.skip("would launch on made-up addresses")
    r, wide = routing(capi, element=8), routing(capi, row_stride=192)
    for problem, out, stride in ((r, 0x10000000, 64), (r, 0x10000000 + 12800, 64), (r, 0x10000000 - 12800, 64), (wide, 0x10000000, 192), (wide, 0x10000000 + 4 * 64, 192),
                                 (wide, 0x10000000 + 4 * 128, 192), (wide, 0x10000000 - 4 * 64, 192), (routing(capi, tokens=1), 0x10000000, 7)):
        with pytest.raises(capi.FTrainError) as info:
            capi.expert_routing_backward(problem, *OUTPUTS[:4], 0, 0, out, stride)
        assert "across" not in info.value.message
