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


def _calls(dev="cpu"):
    """Each operator as a function of one tensor, and that tensor."""
    from catch_b200.fusion import qk_norm_rotary, relative_bias_softmax, top_logits_distillation

    torch.manual_seed(0)
    cos, sin = (t.to(dev) for t in cases.tables(4, 4))
    q, k, w = torch.randn(1, 3, 2, 8).to(dev), torch.randn(1, 3, 1, 8).to(dev), torch.ones(8).to(dev)
    s, t = torch.randn(1, 2, 3, 4).to(dev), torch.randn(8, 2).to(dev)
    z, te, idx = torch.randn(3, 7).to(dev), torch.randn(3, 2).to(dev), torch.tensor([[0, 3], [1, -1], [-1, -1]]).to(dev)
    return {
        "rotary queries": (lambda x: qk_norm_rotary(x, k, w, w, cos, sin)[0], q),
        "rotary keys": (lambda x: qk_norm_rotary(q, x, w, None, cos, sin)[1], k),
        "rotary weight": (lambda x: qk_norm_rotary(q, k, x, w, cos, sin)[0], w),
        "softmax scores": (lambda x: relative_bias_softmax(x, t, max_distance=8), s),
        "softmax table": (lambda x: relative_bias_softmax(s, x, max_distance=8), t),
        "distillation": (lambda x: top_logits_distillation(x, te, idx, temperature=2.0), z),
    }


CALLS = ["rotary queries", "rotary keys", "rotary weight", "softmax scores", "softmax table", "distillation"]


@pytest.mark.parametrize("dev", ["cpu", "blackwell"])
@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(name, dev):
    import torch.autograd.forward_ad as fwd

    f, x = _calls(dev)[name]
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(fwd.make_dual(x, torch.ones_like(x)))
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            f(fwd.make_dual(x, torch.ones_like(x)))
        f(x)  # without a tangent
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jacfwd(f)(x)


@pytest.mark.parametrize("what", ["cos", "mask", "teacher"])
def test_forward_mode_is_refused_for_constants(what):
    import torch.autograd.forward_ad as fwd
    from catch_b200.fusion import qk_norm_rotary, relative_bias_softmax, top_logits_distillation

    cos, sin = cases.tables(4, 4)
    q, z = torch.randn(1, 3, 2, 8), torch.randn(3, 7)
    with fwd.dual_level():
        dual = lambda x: fwd.make_dual(x, torch.ones_like(x))  # noqa: E731
        with pytest.raises(RuntimeError, match="forward-mode"):
            if what == "cos":
                qk_norm_rotary(q, q, None, None, dual(cos), sin)
            elif what == "mask":
                relative_bias_softmax(q, torch.zeros(4, 3), dual(torch.zeros(1, 1, 2, 8)))
            else:
                top_logits_distillation(z, dual(torch.randn(3, 2)), torch.zeros(3, 2, dtype=torch.long))
