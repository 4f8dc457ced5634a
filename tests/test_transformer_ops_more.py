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


# --------------------------------------------------------------- what lies between autograd and the kernels sees the operators
@pytest.mark.parametrize("dev", ["cpu", "blackwell"])
@pytest.mark.parametrize("name", CALLS)
def test_function_transforms(name, dev):
    f, x = _calls(dev)[name]
    g = torch.randn(f(x).shape).to(dev)
    total = lambda x: (f(x) * g).sum()  # noqa: E731
    leaf = x.clone().requires_grad_()
    (want,) = torch.autograd.grad(total(leaf), leaf)
    assert torch.equal(torch.func.grad(total)(x), want)
    value, pull = torch.func.vjp(f, x)
    assert torch.equal(value, f(x)) and torch.equal(pull(g)[0], want)
    many = torch.stack([x, 0.5 * x, -x])
    assert torch.equal(torch.func.vmap(f)(many), torch.stack([f(v) for v in many]))
    each = torch.stack([torch.func.grad(total)(v) for v in many])
    assert torch.allclose(torch.func.vmap(torch.func.grad(total))(many), each, rtol=2.0 ** -20, atol=2.0 ** -20)


@pytest.mark.parametrize("dev", ["cpu", "blackwell"])
def test_dispatch_modes_see_the_operators(dev):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(func.name())
            return func(*args, **(kwargs or {}))

    for name, (f, x) in _calls(dev).items():
        want = f(x)
        leaf = x.clone().requires_grad_()
        with Seen() as seen:
            y = f(leaf)
            (d,) = torch.autograd.grad(y.sum(), leaf)
        assert torch.equal(y, want) and d.shape == x.shape
        op = {"rot": "qk_norm_rotary", "sof": "relative_bias_softmax", "dis": "top_logits_distillation"}[name[:3]]
        ours = [n for n in seen.names if n.startswith("catch_b200::" + op)]
        assert any(not n.endswith("_backward") for n in ours) and any(n.endswith("_backward") for n in ours), (name, seen.names)


@pytest.mark.parametrize("dev", ["cpu", "blackwell"])
@pytest.mark.parametrize("name", CALLS)
def test_fake_tensors_have_the_shapes(name, dev):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.utils._pytree import tree_map

    f, x = _calls(dev)[name]
    leaf = x.clone().requires_grad_()
    y = f(leaf)
    (d,) = torch.autograd.grad(y.sum(), leaf)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        fake = mode.from_tensor(x).requires_grad_()
        fy = f(fake)
        (fd,) = torch.autograd.grad(fy.sum(), fake)
    for a, b in ((fy, y), (fd, d)):
        assert a.shape == b.shape and a.dtype == b.dtype and a.device == b.device and a.stride() == b.stride()


def test_meta_tensors_have_the_shapes_and_are_checked():
    ops = torch.ops.catch_b200
    m = dict(device="meta")
    q, k, c, w = torch.randn(2, 5, 4, 8, **m), torch.randn(2, 5, 2, 8, **m), torch.randn(7, 3, **m), torch.randn(8, **m).bfloat16()
    yq, yk = ops.qk_norm_rotary(q, k, w, None, c, c)
    assert yq.shape == q.shape and yk.shape == k.shape
    dq, dk, dw, none = ops.qk_norm_rotary_backward(yq, yk, q, k, w, None, c, c, None, 1e-6, False)
    assert dq.shape == q.shape and dk.shape == k.shape and dw.shape == w.shape and dw.dtype == w.dtype and none is None
    s, t = torch.randn(2, 3, 5, 6, **m).bfloat16(), torch.randn(8, 3, **m)
    p, st = ops.relative_bias_softmax(s, t)
    assert p.shape == s.shape and p.dtype == s.dtype and st.shape == (2, 3, 5, 2) and st.dtype == torch.float32
    ds, dt = ops.relative_bias_softmax_backward(p, s, st, t, None, 1.0, True, 128, 0, True)
    assert ds.shape == s.shape and dt.shape == t.shape
    z, te, i = torch.randn(4, 9, **m).half(), torch.randn(4, 2, **m), torch.zeros(4, 2, dtype=torch.long, **m)
    for reduction, shape in ((0, (4,)), (1, ()), (2, ())):
        assert ops.top_logits_distillation(z, te, i, 1.0, reduction).shape == shape
        loss, stats, count = ops.top_logits_distillation_stats(z, te, i, 1.0, reduction)
        assert loss.shape == shape and loss.dtype == torch.float32 and stats.shape == (4, 2)
        dz = ops.top_logits_distillation_backward(loss, z, stats, count, te, i, 1.0, reduction)
        assert dz.shape == z.shape and dz.dtype == z.dtype
    with pytest.raises(RuntimeError, match="differ in batch, length or head_dim"):
        ops.qk_norm_rotary(q, k[:, :4], None, None, c, c)
    with pytest.raises(RuntimeError, match="buckets, heads"):
        ops.relative_bias_softmax(s, t[:, :2])
    with pytest.raises(RuntimeError, match="shape of its logits"):
        ops.top_logits_distillation(z, te, i[:, :1])


def test_the_loss_with_its_statistics_is_differentiable():
    z, te, idx = torch.randn(3, 7, requires_grad=True), torch.randn(3, 2), torch.tensor([[0, 3], [1, -1], [-1, -1]])
    for reduction in (0, 1, 2):
        plain = torch.ops.catch_b200.top_logits_distillation(z, te, idx, 2.0, reduction)
        loss, stats, count = torch.ops.catch_b200.top_logits_distillation_stats(z, te, idx, 2.0, reduction)
        assert not stats.requires_grad and not count.requires_grad
        assert torch.equal(torch.autograd.grad(loss.sum(), z)[0], torch.autograd.grad(plain.sum(), z)[0])


@pytest.mark.parametrize("name", CALLS)
def test_traced_by_the_compiler(name):
    f, x = _calls()[name]
    g = torch.randn(f(x).shape)
    total = lambda x: (f(x) * g).sum()  # noqa: E731
    got = torch.compile(total, backend="aot_eager", fullgraph=True)
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    total(a).backward()
    got(b).backward()
    assert torch.allclose(a.grad, b.grad, rtol=2.0 ** -20, atol=2.0 ** -20)


def test_selective_checkpointing_keeps_the_results():
    from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts

    def policy(ctx, op, *args, **kwargs):
        return CheckpointPolicy.MUST_SAVE if "relative_bias_softmax" in op.name() else CheckpointPolicy.PREFER_RECOMPUTE

    from catch_b200.fusion import relative_bias_softmax

    torch.manual_seed(1)
    s, t = torch.randn(1, 2, 3, 4, requires_grad=True), torch.randn(8, 2, requires_grad=True)
    body = lambda s, t: relative_bias_softmax(s.sin(), t, max_distance=8).square().sum()  # noqa: E731
    want = torch.autograd.grad(body(s, t), (s, t))
    y = checkpoint(body, s, t, use_reentrant=False, context_fn=lambda: create_selective_checkpoint_contexts(policy))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (s, t)), want))


# ------------------------------------------------------------------------------------------------ derivatives of derivatives
@pytest.mark.parametrize("dev", ["cpu", "blackwell"])
@pytest.mark.parametrize("name", CALLS)
def test_second_derivatives_are_refused_however_they_are_asked_for(name, dev):
    import torch.autograd.forward_ad as fwd

    f, x = _calls(dev)[name]
    g = torch.randn(f(x).shape).to(dev)
    total = lambda x: (f(x) * g).sum()  # noqa: E731
    refused = lambda: pytest.raises(RuntimeError, match="gradient of the gradient|forward-mode")  # noqa: E731
    with refused():
        torch.func.grad(lambda x: torch.func.grad(total)(x).square().sum())(x)
    with refused():
        torch.func.jvp(torch.func.grad(total), (x,), (torch.ones_like(x),))
    with refused():
        torch.func.hessian(total)(x)
    with refused():
        torch.func.jacrev(torch.func.grad(total))(x)
    with refused():  # of the gradient with respect to the factor that it starts from
        torch.func.jvp(lambda g: torch.func.vjp(f, x)[1](g)[0], (g,), (g,))
    leaf = x.clone().requires_grad_()
    (d,) = torch.autograd.grad(total(leaf), leaf, create_graph=True)
    with refused():
        torch.autograd.grad(d.sum(), leaf, allow_unused=True)
    start = g.clone().requires_grad_()
    (d,) = torch.autograd.grad(f(leaf), leaf, start, create_graph=True)
    with refused():
        torch.autograd.grad(d.sum(), start)
    with fwd.dual_level(), refused():
        torch.autograd.grad(f(leaf), leaf, fwd.make_dual(g, torch.ones_like(g)))
    # the value beside the gradient can be differentiated once more
    both = lambda x: sum(t.sum() for t in torch.func.vjp(f, x)[:1])  # noqa: E731
    assert torch.allclose(torch.func.grad(both)(x), torch.autograd.grad(f(leaf).sum(), leaf)[0], rtol=2.0 ** -20, atol=2.0 ** -20)


def test_results_of_the_backward_forms_refuse_derivatives():
    ops = torch.ops.catch_b200
    cos, sin = cases.tables(4, 4)
    q, w = torch.randn(1, 3, 2, 8, requires_grad=True), torch.ones(8, requires_grad=True)
    s, z = torch.randn(1, 2, 3, 4, requires_grad=True), torch.randn(3, 7, requires_grad=True)
    t, te, idx = torch.randn(8, 2), torch.randn(3, 2), torch.zeros(3, 2, dtype=torch.long)
    p, st = ops.relative_bias_softmax(s.detach(), t)
    loss, stats, count = ops.top_logits_distillation_stats(z.detach(), te, idx, 1.0, 1)
    calls = [lambda: ops.qk_norm_rotary_backward(q.detach(), q.detach(), q, q, w, None, cos, sin, None, 1e-6, False)[:3],
             lambda: ops.relative_bias_softmax_backward(p, s, st, t, None, 1.0, True, 128, 0, True),
             lambda: (ops.top_logits_distillation_backward(torch.ones(()), z, stats, count, te, idx, 1.0, 1),)]
    for call in calls:
        with torch.no_grad():
            plain = call()
        assert not any(r.requires_grad for r in plain)
        for r, want in zip(call(), plain):
            assert torch.equal(r.detach(), want)
            with pytest.raises(RuntimeError, match="gradient of the gradient"):
                r.sum().backward()


@pytest.mark.parametrize("dev", ["cpu", "blackwell"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_the_early_gradient_can_be_left_out(dev, reduction):
    from catch_b200.fusion import top_logits_distillation

    z, te, idx = torch.randn(3, 7).to(dev).requires_grad_(), torch.randn(3, 2).to(dev), torch.tensor([[0, 3], [1, -1], [-1, -1]]).to(dev)
    with_it, without = (top_logits_distillation(z, te, idx, temperature=2.0, reduction=reduction, early_gradient=e) for e in (True, False))
    assert torch.equal(with_it, without)
    for factor in (1.0, 0.3):
        a, b = (torch.autograd.grad(factor * y.sum(), z, retain_graph=True)[0] for y in (with_it, without))
        assert torch.equal(a, b)


def test_an_encoder_takes_configurations_from_before_there_were_position_types():
    from types import SimpleNamespace

    from catch_b200.models.bert import BertConfig, BertForSequenceClassification

    new = ("position_embedding_type", "relative_attention_num_buckets", "relative_attention_max_distance", "rotary_base")
    c = BertConfig(vocab_size=50, hidden_size=16, num_hidden_layers=1, num_attention_heads=2, intermediate_size=32, max_position_embeddings=10)
    old = SimpleNamespace(**{k: v for k, v in vars(c).items() if k not in new})
    torch.manual_seed(0)
    a = BertForSequenceClassification(c).eval()
    b = BertForSequenceClassification(old).eval()
    b.load_state_dict(a.state_dict())
    ids = torch.randint(0, 50, (2, 7))
    assert torch.equal(a(ids), b(ids))


def numbers_of_rows(dev):
    """The third result is the number of rows with entries for a mean, 1 otherwise, and nothing else."""
    ops = torch.ops.catch_b200
    for n, kept, want in ((4, [[0, -1], [-1, -1], [2, 3], [-1, 1]], 3), (2, [[-1, -1], [-5, -1]], 0), (0, [], 0)):
        z, te = torch.randn(n, 5).to(dev), torch.randn(n, 2).to(dev)
        idx = torch.tensor(kept, dtype=torch.long).view(n, 2).to(dev)
        for reduction in (0, 1, 2):
            loss, stats, count = ops.top_logits_distillation_stats(z, te, idx, 2.0, reduction)
            assert count.shape == (1,) and float(count) == (want if reduction == 1 else 1), (n, reduction, count)
            assert bool(torch.isfinite(loss.cpu()).all())
            leaf = z.clone().requires_grad_()
            (dz,) = torch.autograd.grad(ops.top_logits_distillation(leaf, te, idx, 2.0, reduction).sum(), leaf)
            g = torch.ones(loss.shape).to(dev)
            assert torch.equal(ops.top_logits_distillation_backward(g, z, stats, count, te, idx, 2.0, reduction).cpu(), dz.cpu())
            # the same numbers on the host
            host = ops.top_logits_distillation_stats(z.cpu(), te.cpu(), idx.cpu(), 2.0, reduction)
            assert torch.equal(host[2], count.cpu())


@pytest.mark.parametrize("dev", ["cpu", "blackwell"])
def test_numbers_of_rows(dev):
    numbers_of_rows(dev)


def infinities_and_nan(dev):
    """Kept scores and logits that are infinite or no number give what torch's softmax gives for the row: NaN throughout."""
    from catch_b200.fusion import relative_bias_softmax, top_logits_distillation

    for bad in (math.inf, math.nan):
        for Lk in (5, 64, 1100):
            s = torch.randn(1, 1, 3, Lk)
            s[0, 0, 1, 2] = bad
            m = torch.ones(1, 1, 3, Lk, dtype=torch.bool)
            m[..., 0] = False
            p = relative_bias_softmax(s.to(dev), torch.zeros(4, 1).to(dev), m.to(dev), max_distance=8).cpu()
            want = torch.softmax(s.masked_fill(~m, -math.inf), -1)
            assert torch.equal(p.isnan(), want.isnan()) and bool(want[0, 0, 1].isnan().all())
            assert torch.allclose(p, want, rtol=1e-5, atol=1e-7, equal_nan=True)
        z = torch.randn(3, 70)
        z[1, 7] = bad
        idx = torch.tensor([[0, 7], [3, 4], [5, 6]])
        loss = top_logits_distillation(z.to(dev), torch.zeros(3, 2).to(dev), idx.to(dev), reduction="none").cpu()
        want = math.log(0.5) - torch.log_softmax(z, 1).gather(1, idx).mean(1)
        assert torch.allclose(loss, want, rtol=1e-5, atol=1e-6, equal_nan=True) and bool(loss[1].isnan())


@pytest.mark.parametrize("dev", ["cpu", "blackwell"])
def test_infinities_and_nan(dev):
    infinities_and_nan(dev)
