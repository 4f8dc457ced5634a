"""Further refusals and results of the transformer operators' host paths."""
import math

import pytest
import torch

import transformer_cases as cases


@pytest.fixture(scope="module", autouse=True)
def _backend():
    import catch_b200  # noqa: F401


@pytest.mark.parametrize("dev", ["cpu", "blackwell"])
@pytest.mark.parametrize("change, message", [
    (dict(query_offset=-(1 << 63)), "2\\^30"),
    (dict(query_offset=-(1 << 30)), "2\\^30"),
    (dict(scale=1e39), "finite"),
    (dict(scale=-1e300), "finite"),
])
def test_softmax_arguments_out_of_range(dev, change, message):
    from catch_b200.fusion import relative_bias_softmax

    with pytest.raises(RuntimeError, match=message):
        relative_bias_softmax(torch.zeros(1, 1, 2, 3).to(dev), torch.zeros(4, 1).to(dev), **change)


def test_softmax_sizes_out_of_range():
    """Sizes of tensors that hold nothing (a length of zero) or the same element throughout."""
    from catch_b200.fusion import relative_bias_softmax

    one, table = torch.zeros(1, 1, 1, 1), torch.zeros(4, 1)
    far = (1 << 30) - 1
    with pytest.raises(RuntimeError, match="apart"):  # distances that pass 32 bits
        relative_bias_softmax(one.expand(1, 1, 1, far), table, query_offset=-far)
    with pytest.raises(RuntimeError, match="apart"):
        relative_bias_softmax(one.expand(1, 1, far, 1), table, query_offset=far)
    with pytest.raises(RuntimeError, match="heads"):
        relative_bias_softmax(one.expand(1, 1 << 31, 1, 1), torch.zeros(1, 1).expand(4, 1 << 31))
    with pytest.raises(RuntimeError, match="batch"):
        relative_bias_softmax(one[:, :, :0].expand(1 << 31, 1, 0, 1), table)
