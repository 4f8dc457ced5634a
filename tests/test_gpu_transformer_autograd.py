"""The transformer operators' gradients under the ways in which autograd may run a backward pass."""
import pytest
import torch

import transformer_cases as cases
from test_transformer_ops_more import CALLS, _calls as calls
from transformer_cases import check

pytestmark = pytest.mark.gpu
DEV = "blackwell"


@pytest.fixture(scope="module", autouse=True)
def _backend():
    import catch_b200  # noqa: F401

    assert torch.b200.backend_name() == "cuda"
    torch.b200.set_flag("op_trycatch", False)
    yield
    torch.b200.set_flag("op_trycatch", True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("factor", [1.0, 0.5])
@pytest.mark.parametrize("start, width", [(0, 101), (3, 120), (1, 101)])
def test_logits_that_come_back_in_another_layout(dtype, factor, start, width):
    """A hook on saved tensors may hand them back with other strides and another place within 16 bytes."""
    from catch_b200.fusion import top_logits_distillation

    N, V = 9, 97
    torch.manual_seed(1)
    z = torch.randn(N, V).to(dtype)
    t, idx = cases.teacher_of(N, V, 5, 3)

    def shifted(x):  # the same values, `start` elements behind a boundary, rows `width` apart
        if x.shape != (N, V):
            return x
        return torch.zeros(N, width, dtype=x.dtype, device=x.device)[:, start:start + V].copy_(x)

    for first in (z.to(DEV), shifted(z.to(DEV))):
        leaf = first.detach().requires_grad_()
        for unpack in (lambda x: x.clone(memory_format=torch.contiguous_format), shifted):
            with torch.autograd.graph.saved_tensors_hooks(lambda x: x, unpack):
                loss = top_logits_distillation(leaf, t.to(DEV), idx.to(DEV), temperature=2.0)
                (dz,) = torch.autograd.grad(loss, leaf, torch.tensor(factor).to(DEV))
            check(dz, *cases.distill_reference(z, t, idx, 2.0, "mean", factor)[1], "gradient")


@pytest.mark.parametrize("name", CALLS)
def test_function_transforms(name):
    """As on the host; the same sums may be taken in another order where a slice lies elsewhere within 16 bytes."""
    f, x = calls(DEV)[name]
    g = torch.randn(f(x).shape).to(DEV)
    total = lambda x: (f(x) * g).sum()  # noqa: E731
    leaf = x.clone().requires_grad_()
    (want,) = torch.autograd.grad(total(leaf), leaf)
    near = lambda a, b: torch.allclose(a.cpu(), b.cpu(), rtol=2.0 ** -18, atol=2.0 ** -18)  # noqa: E731
    assert near(torch.func.grad(total)(x), want)
    value, pull = torch.func.vjp(f, x)
    assert near(value, f(x)) and near(pull(g)[0], want)
    many = torch.stack([x, 0.5 * x, -x])
    assert near(torch.func.vmap(f)(many), torch.stack([f(v) for v in many]))
    assert near(torch.func.vmap(torch.func.grad(total))(many), torch.stack([torch.func.grad(total)(v) for v in many]))


def test_dispatch_modes_see_the_operators():
    from test_transformer_ops_more import test_dispatch_modes_see_the_operators as on_host

    on_host(DEV)


@pytest.mark.parametrize("name", CALLS)
def test_fake_tensors_have_the_shapes(name):
    from test_transformer_ops_more import test_fake_tensors_have_the_shapes as on_host

    on_host(name, DEV)


@pytest.mark.parametrize("name", CALLS)
def test_second_derivatives_are_refused(name):
    from test_transformer_ops_more import test_second_derivatives_are_refused_however_they_are_asked_for as on_host

    on_host(name, DEV)


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(name):
    from test_transformer_ops_more import test_forward_mode_is_refused as on_host

    on_host(name, DEV)


def test_an_index_out_of_range_in_a_backward_raises_there_and_not_later():
    """In synchronous mode; the flag on the device is shared by all operators that look things up."""
    ops = torch.ops.catch_b200
    cos, sin = torch.ones(4, 2).to(DEV), torch.zeros(4, 2).to(DEV)
    q, far = torch.randn(1, 3, 2, 8).to(DEV), torch.tensor([[0, 1, 4]]).to(DEV)
    z, te = torch.randn(2, 5).to(DEV), torch.randn(2, 2).to(DEV)
    good, bad = torch.tensor([[0, 1], [2, -1]]).to(DEV), torch.tensor([[0, 1], [2, 5]]).to(DEV)
    loss, stats, count = ops.top_logits_distillation_stats(z, te, good, 1.0, 1)
    rotary = lambda pos: ops.qk_norm_rotary_backward(q, q, q, q, None, None, cos, sin, pos, 1e-6, False)  # noqa: E731
    distill = lambda idx: ops.top_logits_distillation_backward(loss, z, stats, count, te, idx, 1.0, 1)  # noqa: E731
    rows, first = torch.randn(5, 3).to(DEV), torch.tensor([0, 4]).to(DEV)
    torch.b200.set_flag("async_disable", True)
    try:
        for call, name in ((lambda: rotary(far), "qk_norm_rotary_backward"), (lambda: distill(bad), "top_logits_distillation_backward")):
            with pytest.raises(IndexError, match=name):
                call()
            assert torch.equal(rows.index_select(0, first).cpu(), rows.cpu()[[0, 4]])  # nothing is left behind
        rotary(torch.tensor([[-1, 0, 3]]).to(DEV))
        distill(good)
    finally:
        torch.b200.set_flag("async_disable", False)
    # a forward that ran before the mode was switched on
    leaf = z.clone().requires_grad_()
    late = ops.top_logits_distillation(leaf, te, bad, 1.0, 0)
    torch.b200.set_flag("async_disable", True)
    try:
        with pytest.raises(IndexError, match="top_logits_distillation_backward"):
            torch.autograd.grad(late.sum(), leaf)
        assert torch.equal(rows.index_select(0, first).cpu(), rows.cpu()[[0, 4]])
    finally:
        torch.b200.set_flag("async_disable", False)


def test_large_products_in_half_precision():
    """Queries times keys of 64 x 40 x 40 = 102400, beyond fp16; scaled by 1 / sqrt(64) they are 12800, the same for every key, so that
    the probabilities are those of the bias alone."""
    from catch_b200.models.bert import BertConfig, BertSelfAttention, FusedBertSelfAttention

    torch.manual_seed(2)
    c = BertConfig(hidden_size=128, num_attention_heads=2, attention_probs_dropout_prob=0.0, position_embedding_type="relative_bias")
    att = BertSelfAttention(c)
    with torch.no_grad():
        for p in (att.query, att.key):
            p.weight.zero_()
            p.bias.fill_(40.0)
        att.relative_bias.copy_(torch.randn(32, 2))
    x = torch.randn(2, 9, 128)
    want = att(x).detach()
    att.__class__ = FusedBertSelfAttention
    att.to(DEV)
    with torch.autocast(DEV, dtype=torch.float16):
        y = att(x.to(DEV))
    assert y.dtype == torch.float16
    y.float().sum().backward()
    # (values, probabilities and the product's result are rounded to 2^-11 each; means of nine values of size one)
    assert float((y.detach().cpu().float() - want).abs().max()) <= 4 * 2.0 ** -11 * float(want.abs().max().clamp(min=1.0))
    assert all(bool(torch.isfinite(p.grad.cpu()).all()) for p in att.parameters())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V, width, step", [(4096, 4096, 64), (1001, 1001, 37), (999, 1005, 5), (7, 1000, 1)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_the_gradient_takes_the_memory_of_the_logits(dtype, V, width, step, reduction):
    """Whatever the distance of the logits' rows, such as that of each sequence's last token."""
    from catch_b200.fusion import top_logits_distillation

    N = 9
    torch.manual_seed(V)
    whole = torch.randn(N, step, width).to(dtype).to(DEV)
    z = whole[:, step // 2, width - V:].detach().requires_grad_()
    assert z.stride(0) == step * width
    t, idx = cases.teacher_of(N, V, 5, 3)
    t, idx = t.to(DEV), idx.to(DEV)
    g = torch.rand(N).to(DEV) if reduction == "none" else torch.ones(()).to(DEV)
    torch.b200.synchronize()
    before = torch.b200.memory_allocated()
    loss = top_logits_distillation(z, t, idx, temperature=2.0, reduction=reduction)
    gradient = N * (V + 8) * z.element_size() + 16
    assert torch.b200.memory_allocated() - before <= gradient + 8 * 512  # (the allocator's blocks are multiples of 512 bytes)
    for factor in (1, 2):
        (dz,) = torch.autograd.grad(loss, z, factor * g, retain_graph=True)
        assert dz.untyped_storage().nbytes() <= gradient
        check(dz, *cases.distill_reference(z, t, idx, 2.0, reduction, (factor * g).cpu())[1], "gradient")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_without_the_early_gradient_the_forward_holds_none(dtype, reduction):
    from catch_b200.fusion import top_logits_distillation

    N, V = 64, 40000
    z = torch.randn(N, V).to(dtype)
    t, idx = cases.teacher_of(N, V, 5, 3)
    leaf = z.to(DEV).requires_grad_()
    args = (leaf, t.to(DEV), idx.to(DEV))
    for early in (True, False):
        torch.b200.synchronize()
        before = torch.b200.memory_allocated()
        loss = top_logits_distillation(*args, temperature=2.0, reduction=reduction, early_gradient=early)
        assert (torch.b200.memory_allocated() - before >= z.numel() * z.element_size()) == early
        for factor in (1.0, 0.3):
            (dz,) = torch.autograd.grad(loss, leaf, torch.tensor(factor).to(DEV), retain_graph=True)
            check(dz, *cases.distill_reference(z, t, idx, 2.0, reduction, factor)[1], "gradient")
            del dz
        del loss


def test_second_derivatives_of_scores_that_are_laid_out_anew():
    """The copy that the backward reads must not hide the scores from whoever differentiates once more."""
    from catch_b200.fusion import relative_bias_softmax

    wide = torch.randn(1, 2, 3, 9).to(DEV)
    s = wide[..., 1:6].detach().requires_grad_()
    y = relative_bias_softmax(s, torch.randn(8, 2).to(DEV), max_distance=8)
    (d,) = torch.autograd.grad(y.square().sum(), s, create_graph=True)
    with pytest.raises(RuntimeError, match="gradient of the gradient"):
        torch.autograd.grad((d * s.detach()).sum() + s.sum(), s)
    t = torch.randn(8, 2).to(DEV)
    (d,) = torch.autograd.grad(relative_bias_softmax(s, t, max_distance=8), s, torch.ones(1, 2, 3, 5).to(DEV), create_graph=True)
    with pytest.raises(RuntimeError, match="gradient of the gradient"):
        torch.autograd.grad(d.sum() + s.sum(), s)


def test_statistics_may_begin_anywhere():
    """A caller (or a hook on saved tensors) may keep them as a part of something else: on no boundary of a pair of numbers."""
    ops = torch.ops.catch_b200

    def elsewhere(t):
        return torch.cat([torch.zeros(1, device=DEV), t.flatten()])[1:].view(t.shape)

    s, t, g = torch.randn(2, 2, 5, 9).to(DEV), torch.randn(8, 2).to(DEV), torch.randn(2, 2, 5, 9).to(DEV)
    p, st = ops.relative_bias_softmax(s, t, None, 1.0, True, 12, 0)
    assert elsewhere(st).data_ptr() % 8 == 4 and elsewhere(st).is_contiguous()
    a, b = (ops.relative_bias_softmax_backward(g, s, x, t, None, 1.0, True, 12, 0, True) for x in (st, elsewhere(st)))
    assert torch.equal(a[0].cpu(), b[0].cpu()) and torch.equal(a[1].cpu(), b[1].cpu())
    z, te, idx = torch.randn(5, 33).to(DEV), torch.randn(5, 3).to(DEV), torch.randint(0, 33, (5, 3)).to(DEV)
    loss, st, count = ops.top_logits_distillation_stats(z, te, idx, 1.0, 1)
    a, b = (ops.top_logits_distillation_backward(torch.ones(()).to(DEV), z, x, count, te, idx, 1.0, 1) for x in (st, elsewhere(st)))
    assert torch.equal(a.cpu(), b.cpu())


def test_threads_with_tables_of_different_sizes():
    """The same kernel at once with more and with less shared memory."""
    import threading

    ops = torch.ops.catch_b200
    s, g, t = (torch.randn(1, 1, 1, 2048).bfloat16().to(DEV), torch.randn(1, 1, 1, 2048).bfloat16().to(DEV), torch.randn(32, 1).to(DEV))
    forward = lambda d: ops.relative_bias_softmax(s, t, None, 1.0, True, d, 9000)  # noqa: E731
    backward = lambda d, st: ops.relative_bias_softmax_backward(g, s, st, t, None, 1.0, True, d, 9000, True)  # noqa: E731
    want = {d: (forward(d)[0].cpu(), *(x.cpu() for x in backward(d, forward(d)[1]))) for d in (8192, 4096)}
    errors = []

    def work(d):
        try:
            with torch.b200.stream(torch.b200.queue_from_pool()):
                for _ in range(30000):
                    p, st = forward(d)
                for _ in range(5000):
                    grads = backward(d, st)
                assert all(torch.equal(a.cpu(), b) for a, b in zip((p, *grads), want[d]))
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    torch.b200.synchronize()
    threads = [threading.Thread(target=work, args=(d,)) for d in (8192, 4096, 8192, 4096)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not errors, errors


def test_numbers_of_rows():
    from test_transformer_ops_more import numbers_of_rows

    numbers_of_rows(DEV)


def test_infinities_and_nan():
    from test_transformer_ops_more import infinities_and_nan

    infinities_and_nan(DEV)


@pytest.mark.parametrize("how", ["checkpoint", "reentrant checkpoint", "on the host"])
def test_recomputed_and_offloaded_tensors(how):
    """The three operators in a row, their saved tensors recomputed or kept on the host meanwhile."""
    from catch_b200.fusion import qk_norm_rotary, relative_bias_softmax, top_logits_distillation
    from torch.utils.checkpoint import checkpoint

    torch.manual_seed(4)
    B, L, H, D, V = 2, 11, 3, 16, 77
    qkv, w, table = torch.randn(B, L, 3 * H, D), torch.ones(D), torch.randn(8, H)
    head = torch.randn(H * D, V + 6)
    cos, sin = (t.to(DEV) for t in cases.tables(L, D))
    t, idx = (x.to(DEV) for x in cases.teacher_of(B * L, V, 5, 1))

    def body(qkv, w, table, head):
        q, k = qk_norm_rotary(qkv[:, :, :H], qkv[:, :, H:2 * H], w, w, cos, sin)
        p = relative_bias_softmax(torch.matmul(q.permute(0, 2, 1, 3), k.permute(0, 2, 3, 1)), table, scale=0.25, max_distance=12)
        y = torch.matmul(p, qkv[:, :, 2 * H:].permute(0, 2, 1, 3)).permute(0, 2, 1, 3).reshape(B * L, H * D)
        return top_logits_distillation(torch.matmul(y, head)[:, 3:3 + V], t, idx, temperature=2.0)

    def leaves():
        return [x.to(DEV).requires_grad_() for x in (qkv, w, table, head)]

    plain, other = leaves(), leaves()
    (body(*plain)).backward()
    for factor in (1.0, 0.5):
        for x in other:
            x.grad = None
        if how == "on the host":
            with torch.autograd.graph.save_on_cpu():
                (factor * body(*other)).backward()
        else:
            (factor * checkpoint(body, *other, use_reentrant=how.startswith("reentrant"))).backward()
        for a, b in zip(plain, other):
            assert torch.allclose(factor * a.grad.cpu(), b.grad.cpu(), rtol=2.0 ** -18, atol=2.0 ** -18 * float(a.grad.cpu().abs().max()))
