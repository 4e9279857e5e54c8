"""What ftcuda_linear_cross_entropy and its gradients refuse: checked before anything touches a device, so made-up addresses do."""
import pytest


def problem(capi, **change):
    fields = dict(hidden=0x10000000, weight=0x20000000, target=0x30000000, tokens=100, vocabulary=1000, depth=64, hidden_row_stride=64,
                  weight_row_stride=64, ignore_index=-100, element=8, reduction=1, device=0)
    return capi.LinearCrossEntropy(**{**fields, **change})


def refuse(capi, reason, call, *arguments):
    with pytest.raises(capi.FTrainError) as info:
        call(*arguments)
    assert reason in info.value.message, info.value.message


@pytest.mark.parametrize("change, reason", [
    ({"element": 1}, "FP32, FP16 or BF16"), ({"reduction": 3}, "reduction"), ({"reduction": -1}, "reduction"), ({"vocabulary": 0}, "vocabulary"),
    ({"vocabulary": 1 << 24}, "vocabulary"), ({"depth": 0}, "depth"), ({"depth": 1 << 20}, "depth"), ({"tokens": 1 << 24}, "tokens"),
    ({"weight": None}, "the weight has no address"), ({"weight": 0x20000001}, "the weight has no address"), ({"weight_row_stride": 63}, "weight's rows overlap"),
    ({"weight_row_stride": -64}, "weight's rows overlap"), ({"hidden": None}, "hidden states have no address"), ({"hidden": 0x10000001}, "hidden states have no address"),
    ({"hidden_row_stride": 0}, "hidden states' rows overlap"), ({"target": None}, "targets"), ({"target": 0x30000004}, "targets"),
])
def test_problems_that_cannot_be(capi, change, reason):
    q = problem(capi, **change)
    refuse(capi, reason, capi.linear_cross_entropy, q, 0x40000000, 0x50000000, 0x60000000, 1 << 40)
    refuse(capi, reason, capi.linear_cross_entropy_backward, q, 0x40000000, 0x50000000, 0x70000000, 64, 0x80000000, 64, 0x60000000, 1 << 40)
    refuse(capi, reason, capi.linear_cross_entropy_workspace_bytes, q, False)


def test_addresses_that_cannot_be(capi):
    q = problem(capi)
    for loss, lse in ((0, 0x50000000), (0x40000002, 0x50000000), (0x40000000, 0), (0x40000000, 0x50000001)):
        refuse(capi, "has no address", capi.linear_cross_entropy, q, loss, lse, 0x60000000, 1 << 40)
    for lse, grad in ((0, 0x50000000), (0x40000000, 0), (0x40000000, 0x50000002)):
        refuse(capi, "has no address", capi.linear_cross_entropy_backward, q, lse, grad, 0x70000000, 64, 0x80000000, 64, 0x60000000, 1 << 40)
    back = capi.linear_cross_entropy_backward
    refuse(capi, "a gradient's address", back, q, 0x40000000, 0x50000000, 0x70000001, 64, 0x80000000, 64, 0x60000000, 1 << 40)
    refuse(capi, "a gradient's address", back, q, 0x40000000, 0x50000000, 0x70000000, 64, 0x80000001, 64, 0x60000000, 1 << 40)
    refuse(capi, "hidden states' gradient overlap", back, q, 0x40000000, 0x50000000, 0x70000000, 63, 0x80000000, 64, 0x60000000, 1 << 40)
    refuse(capi, "weight's gradient overlap", back, q, 0x40000000, 0x50000000, 0x70000000, 64, 0x80000000, 63, 0x60000000, 1 << 40)


@pytest.mark.parametrize("grad_hidden, grad_weight", [(0x10000000, 0x80000000), (0x70000000, 0x20000000), (0x10000000 + 12798, 0), (0, 0x20000000 + 127998),
                                                      (0x70000000, 0x70000000 + 12798), (0x70000000, 0x30000000), (0x30000000 - 12798, 0)])
def test_gradients_across_other_memory(capi, grad_hidden, grad_weight):
    q = problem(capi)
    refuse(capi, "lies across", capi.linear_cross_entropy_backward, q, 0x40000000, 0x50000000, grad_hidden, 64, grad_weight, 64, 0x60000000, 1 << 40)
    refuse(capi, "lies across", capi.linear_cross_entropy_step, q, 0x40000000, 8, grad_hidden, 64, grad_weight, 64, 0x60000000, 1 << 40)


@pytest.mark.parametrize("change, reason", [
    ({"reduction": 0}, "without reduction"), ({"tokens": 0}, "no tokens"), ({"tokens": 1 << 16, "vocabulary": 1 << 15}, "2 GiB"), ({"element": 1}, "FP32, FP16 or BF16"),
    ({"hidden": None}, "hidden states have no address"), ({"weight_row_stride": 1}, "weight's rows overlap"),
])
def test_what_the_step_does_not_take(capi, change, reason):
    q = problem(capi, **change)
    refuse(capi, reason, capi.linear_cross_entropy_step, q, 0x40000000, 8, 0x70000000, 64, 0x80000000, 64, 0x60000000, 1 << 40)
    refuse(capi, reason, capi.linear_cross_entropy_step_workspace_bytes, q)


def test_where_the_step_does_not_write(capi):
    q, step = problem(capi), capi.linear_cross_entropy_step
    refuse(capi, "operands' type", step, q, 0x40000000, 7, 0x70000000, 64, 0x80000000, 64, 0x60000000, 1 << 40)
    refuse(capi, "the loss has no address", step, q, 0, 8, 0x70000000, 64, 0x80000000, 64, 0x60000000, 1 << 40)
    refuse(capi, "the loss has no address", step, q, 0x40000001, 8, 0x70000000, 64, 0x80000000, 64, 0x60000000, 1 << 40)
    refuse(capi, "a gradient's address", step, q, 0x40000000, 4, 0x70000002, 64, 0x80000000, 64, 0x60000000, 1 << 40)
    refuse(capi, "hidden states' gradient overlap", step, q, 0x40000000, 8, 0x70000000, 63, 0x80000000, 64, 0x60000000, 1 << 40)
    refuse(capi, "weight's gradient overlap", step, q, 0x40000000, 8, 0x70000000, 64, 0x80000000, -64, 0x60000000, 1 << 40)


@pytest.mark.parametrize("change, reason", [
    ({"reduction": 0}, "without reduction"), ({"tokens": 0}, "no tokens"), ({"tokens": 1 << 16, "vocabulary": 1 << 15}, "2 GiB"), ({"element": 1}, "FP32, FP16 or BF16"),
    ({"target": 0x30000004}, "targets"), ({"weight": None}, "the weight has no address"),
])
def test_what_the_step_in_two_does_not_take(capi, change, reason):
    q = problem(capi, **change)
    refuse(capi, reason, capi.linear_cross_entropy_step_loss, q, 0x40000000, 0x60000000, 1 << 40)
    refuse(capi, reason, capi.linear_cross_entropy_step_gradients, q, 0x40000000, 0x70000000, 64, 0x80000000, 64, 0x60000000, 1 << 40)


def test_where_the_step_in_two_does_not_write(capi):
    q = problem(capi)
    refuse(capi, "the loss has no address", capi.linear_cross_entropy_step_loss, q, 0, 0x60000000, 1 << 40)
    refuse(capi, "the loss has no address", capi.linear_cross_entropy_step_loss, q, 0x40000002, 0x60000000, 1 << 40)
    step = capi.linear_cross_entropy_step_gradients
    refuse(capi, "gradient has no address", step, q, 0, 0x70000000, 64, 0x80000000, 64, 0x60000000, 1 << 40)
    refuse(capi, "gradient has no address", step, q, 0x40000001, 0x70000000, 64, 0x80000000, 64, 0x60000000, 1 << 40)
    refuse(capi, "a gradient's address", step, q, 0x40000000, 0x70000001, 64, 0x80000000, 64, 0x60000000, 1 << 40)
    refuse(capi, "weight's gradient overlap", step, q, 0x40000000, 0x70000000, 64, 0x80000000, 63, 0x60000000, 1 << 40)
    refuse(capi, "lies across", step, q, 0x40000000, 0x70000000, 64, 0x20000000, 64, 0x60000000, 1 << 40)


@pytest.mark.parametrize("change, reason", [
    ({"reduction": 0}, "without reduction"), ({"tokens": 0}, "no tokens"), ({"tokens": 1 << 16, "vocabulary": 1 << 15}, "2 GiB"), ({"element": 1}, "FP32, FP16 or BF16"),
    ({"target": 0x30000004}, "targets"), ({"weight": None}, "the weight has no address"),
])
def test_what_the_step_with_a_kept_memory_does_not_take(capi, change, reason):
    q = problem(capi, **change)
    refuse(capi, reason, capi.linear_cross_entropy_step_loss_bytes, q)
    refuse(capi, reason, capi.linear_cross_entropy_step_gradients_bytes, q, 1 << 20)
    refuse(capi, reason, capi.linear_cross_entropy_step_loss_kept, q, 0x40000000, 0x50000000, 1 << 20, 0x60000000, 1 << 40)
    refuse(capi, reason, capi.linear_cross_entropy_step_gradients_kept, q, 0x40000000, 0x70000000, 64, 0x80000000, 64, 0x50000000, 1 << 20, 0x60000000, 1 << 40)


def test_where_the_step_with_a_kept_memory_does_not_write(capi):
    q = problem(capi)
    loss, step = capi.linear_cross_entropy_step_loss_kept, capi.linear_cross_entropy_step_gradients_kept
    refuse(capi, "the loss has no address", loss, q, 0, 0x50000000, 1 << 20, 0x60000000, 1 << 40)
    refuse(capi, "gradient has no address", step, q, 0x40000001, 0x70000000, 64, 0x80000000, 64, 0x50000000, 1 << 20, 0x60000000, 1 << 40)
    refuse(capi, "a gradient's address", step, q, 0x40000000, 0x70000001, 64, 0x80000000, 64, 0x50000000, 1 << 20, 0x60000000, 1 << 40)
    refuse(capi, "lies across", step, q, 0x40000000, 0x70000000, 64, 0x20000000, 64, 0x50000000, 1 << 20, 0x60000000, 1 << 40)
