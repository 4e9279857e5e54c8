"""What ftcuda_gradient_norm and ftcuda_gradient_clip refuse. The checks come before anything touches a device, so made-up addresses do."""
import pytest

MIB = 1 << 20


def gradient(capi, data=0x10000000, out=0x10000000, rows=1, cols=1000, row_stride=0, out_row_stride=0, element=4, out_element=4):
    return capi.Gradient(data, out, rows, cols, row_stride, out_row_stride, element, out_element)


def refuse(capi, gradients, reason, clip=True, max_norm=1.0, norm=0x2000, workspace=0x4000, workspace_bytes=MIB, norm_kind=0):
    with pytest.raises(capi.FTrainError) as info:
        if clip:
            capi.gradient_clip(gradients, max_norm, norm, workspace, workspace_bytes, norm_kind)
        else:
            capi.gradient_norm(gradients, norm, workspace, workspace_bytes, norm_kind)
    assert reason in info.value.message, info.value.message


@pytest.mark.parametrize("clip", [True, False])
@pytest.mark.parametrize("change, reason", [
    ({"element": 1}, "element type"), ({"data": 0}, "no address"), ({"data": 0x10000002}, "multiple of the element"),
    ({"rows": 3, "row_stride": 999}, "rows overlap"), ({"rows": 3, "row_stride": -5}, "rows overlap"),
    ({"rows": 1 << 39, "cols": 1 << 39, "row_stride": 1 << 39}, "too many elements"), ({"rows": 1 << 41}, "too large"),
])
def test_gradients_that_cannot_be(capi, clip, change, reason):
    refuse(capi, [gradient(capi), gradient(capi, **{"out": 0x20000000, **change})], reason, clip)


@pytest.mark.parametrize("change, reason", [
    ({"out_element": 0}, "output's element type"), ({"out": 0}, "no address for the output"), ({"out": 0x20000001, "out_element": 8}, "multiple of its element"),
    ({"rows": 3, "row_stride": 1000, "out_row_stride": 1}, "output's rows overlap"),
])
def test_outputs_that_cannot_be(capi, change, reason):
    refuse(capi, [gradient(capi, **change)], reason)


def test_calls_that_cannot_be(capi):
    good = [gradient(capi)]
    for clip in (True, False):
        refuse(capi, good, "norm has no address", clip, norm=0)
        refuse(capi, good, "norm has no address", clip, norm=0x2002)
        refuse(capi, good, "unknown kind of norm", clip, norm_kind=2)
        refuse(capi, good, "workspace of", clip, workspace=0)
        refuse(capi, good, "workspace of", clip, workspace=0x4004)
        refuse(capi, good, "workspace of", clip, workspace_bytes=capi.gradient_norm_workspace_bytes(1) - 1)
    refuse(capi, good, "max_norm", max_norm=-0.5)
    refuse(capi, good, "max_norm", max_norm=float("nan"))


def test_outputs_that_overlap_are_refused(capi):
    at = 0x10000000
    twice = [gradient(capi, at, at), gradient(capi, at, at)]
    refuse(capi, twice, "overlaps")
    # The last element of one is the first of the next.
    refuse(capi, [gradient(capi, at, at), gradient(capi, at + 999 * 4, at + 999 * 4)], "overlaps")
    # An output over another gradient's input, and one over its own input but not at the same place.
    refuse(capi, [gradient(capi, at, 0x20000000), gradient(capi, 0x30000000, at + 400)], "overlaps")
    refuse(capi, [gradient(capi, at, at + 4)], "overlaps")
    # In place with another type or stride.
    refuse(capi, [gradient(capi, at, at, element=8, out_element=4)], "its own output")
    refuse(capi, [gradient(capi, at, at, rows=4, cols=10, row_stride=20, out_row_stride=10)], "its own output")
    # Windows of one matrix: overlapping by a column, and of different strides.
    window = dict(rows=100, cols=10, row_stride=64, out_row_stride=64)
    refuse(capi, [gradient(capi, at, at, **window), gradient(capi, at + 9 * 4, at + 9 * 4, **window)], "overlaps")
    refuse(capi, [gradient(capi, at, at, **window), gradient(capi, at + 60 * 4, at + 60 * 4, **window)], "overlaps")
    refuse(capi, [gradient(capi, at, at, **window), gradient(capi, at + 10 * 4, at + 10 * 4, rows=100, cols=10, row_stride=63, out_row_stride=63)], "overlaps")


def test_what_is_sound_reaches_the_device_check(capi):
    """Nothing in these lists is refused: the call ends where it asks for a device, which there is none of here (or which runs elsewhere)."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("would launch on made-up addresses")
    at = 0x10000000
    window = dict(rows=100, cols=10, row_stride=64, out_row_stride=64)
    lists = [[gradient(capi, at, at, **window), gradient(capi, at + 10 * 4, at + 10 * 4, **window)],
             [gradient(capi, at, at), gradient(capi, at + 4000, at + 4000)], [gradient(capi, at, 0x20000000), gradient(capi, at, 0x30000000)],
             [gradient(capi, cols=0, data=0, out=0)]]
    for gradients in lists:
        with pytest.raises(capi.FTrainError) as info:
            capi.gradient_clip(gradients, 1.0, 0x2000, 0x4000, MIB)
        assert "overlap" not in info.value.message and "gradient" not in info.value.message


def test_the_workspace_grows_with_the_launches(capi):
    sizes = [capi.gradient_norm_workspace_bytes(n) for n in (0, 1, 64, 65, 480, 481, 5000)]
    assert sizes == sorted(sizes) and sizes[0] == sizes[1] > 0 and sizes[-1] <= MIB


def test_scaling_refuses_the_same(capi):
    good = gradient(capi)
    for gradients, factor, reason in (([good], 0, "the factor"), ([good], 0x2002, "the factor"), ([gradient(capi, element=2)], 0x2000, "element type"),
                                      ([good, good], 0x2000, "overlaps"), ([gradient(capi, out=0)], 0x2000, "no address for the output")):
        with pytest.raises(capi.FTrainError) as info:
            capi.gradient_scale(gradients, factor)
        assert reason in info.value.message
