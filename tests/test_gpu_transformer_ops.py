"""The transformer operators' kernels against their 64-bit forms."""
import pytest
import torch

from transformer_op_checks import OPS_CHECKS, run_check

pytestmark = pytest.mark.gpu
DEV = "blackwell"


@pytest.fixture(scope="module", autouse=True)
def _backend():
    import catch_b200  # noqa: F401

    assert torch.b200.backend_name() == "cuda"
    torch.b200.set_flag("op_trycatch", False)
    yield
    torch.b200.set_flag("op_trycatch", True)


@pytest.mark.parametrize("name", list(OPS_CHECKS))
def test_against_64_bits(name):
    run_check(name, DEV)


def test_smallest_calls_launch_kernels():
    from catch_b200 import _C
    from catch_b200.fusion import qk_norm_rotary, relative_bias_softmax, top_logits_distillation

    q = torch.randn(1, 1, 1, 8).to(DEV)
    cos, sin = torch.ones(1, 4).to(DEV), torch.zeros(1, 4).to(DEV)
    z, t, i = torch.randn(2, 5).to(DEV), torch.randn(2, 2).to(DEV), torch.zeros(2, 2, dtype=torch.long).to(DEV)
    for call in (lambda: qk_norm_rotary(q, q, None, None, cos, sin), lambda: relative_bias_softmax(q, torch.zeros(4, 1).to(DEV)),
                 lambda: top_logits_distillation(z, t, i)):
        _C._reset_kernel_launch_count()
        call()
        assert _C._kernel_launch_count() >= 1
