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


def test_gradients_against_differences():
    from transformer_op_checks import differences

    differences(DEV)


@pytest.mark.parametrize("position", ["absolute", "relative_bias", "rotary"])
@pytest.mark.parametrize("fused, dtype", [(False, None), (True, torch.bfloat16)])
def test_a_student_learns_from_a_teacher(position, fused, dtype):
    from transformer_op_checks import student_step

    student_step(DEV, position, fused, dtype)


def _inputs(seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, cos, sin = r(2, 9, 3, 16).bfloat16(), r(2, 9, 3, 16).bfloat16(), r(9, 8), r(9, 8)
    s, t = r(2, 3, 9, 24).bfloat16(), r(8, 3)
    z, te = r(5, 301).bfloat16(), r(5, 7)
    idx = torch.stack([torch.randperm(301, generator=g)[:7] for _ in range(5)])
    return dict(q=q, k=k, w=1 + 0.1 * r(16), cos=cos, sin=sin, gq=r(2, 9, 3, 16).bfloat16(), gk=r(2, 9, 3, 16).bfloat16(), s=s, t=t,
                gp=r(2, 3, 9, 24).bfloat16(), z=z, te=te, idx=idx, g=torch.tensor(0.5))


def _all(x):
    """Every operator forward and backward through the _backward forms, as a capturing thread may call them."""
    ops = torch.ops.catch_b200
    y = ops.qk_norm_rotary(x["q"], x["k"], x["w"], x["w"], x["cos"], x["sin"])
    d = ops.qk_norm_rotary_backward(x["gq"], x["gk"], x["q"], x["k"], x["w"], x["w"], x["cos"], x["sin"], None, 1e-6, False)
    p, st = ops.relative_bias_softmax(x["s"], x["t"], None, 0.5, True, 12, 0)
    ds = ops.relative_bias_softmax_backward(x["gp"], x["s"], st, x["t"], None, 0.5, True, 12, 0, True)
    loss, stats, count = ops.top_logits_distillation_stats(x["z"], x["te"], x["idx"], 2.0, 1)
    dz = ops.top_logits_distillation_backward(x["g"], x["z"], stats, count, x["te"], x["idx"], 2.0, 1)
    return [*y, *d, p, *ds, loss, dz]


def test_captured_calls_replay_on_new_data_and_two_graphs_do_not_meet():
    first, second = ({k: v.to(DEV) for k, v in _inputs(i).items()} for i in (1, 2))
    with torch.no_grad():
        _all(first)
        graphs = []
        for x in (first, second):
            g = torch.b200.Graph()
            with torch.b200.graph(g):
                out = _all(x)
            graphs.append((g, out))
        for seed in (3, 4):
            fresh = [_inputs(seed), _inputs(seed + 10)]
            for x, new in zip((first, second), fresh):
                for k, v in new.items():
                    x[k].copy_(v)
            side = torch.b200.queue_from_pool()
            torch.b200.synchronize()
            with torch.b200.stream(side):  # both graphs under way at once, on two queues
                graphs[0][0].replay()
            graphs[1][0].replay()
            torch.b200.synchronize()
            for (_, out), x in zip(graphs, (first, second)):
                for i, (a, b) in enumerate(zip(out, _all(x))):
                    assert torch.equal(a.cpu(), b.cpu()), i


def test_a_backward_through_autograd_is_not_captured():
    from catch_b200.fusion import qk_norm_rotary, relative_bias_softmax, top_logits_distillation

    x = {k: v.to(DEV) for k, v in _inputs(5).items()}
    s, z, q = (x[n].clone().requires_grad_() for n in ("s", "z", "q"))
    calls = [lambda: (relative_bias_softmax(s, x["t"]), s, x["gp"]),
             lambda: (top_logits_distillation(z, x["te"], x["idx"]), z, x["g"]),
             lambda: (qk_norm_rotary(q, x["k"], None, None, x["cos"], x["sin"])[0], q, x["gq"])]
    for call in calls:
        kept = call()  # an eager graph of the same leaf lives meanwhile
        g = torch.b200.Graph()
        with pytest.raises(RuntimeError, match="cannot be captured"):
            with torch.b200.graph(g):
                y, leaf, grad = call()
                torch.autograd.grad(y, leaf, grad)
        assert not g.valid
        (d,) = torch.autograd.grad(kept[0], kept[1], kept[2])  # and still works
        assert bool(torch.isfinite(d.float().cpu()).all())


def test_the_same_inputs_give_the_same_bits():
    torch.manual_seed(0)
    ops = torch.ops.catch_b200
    s, g, t = (torch.randn(6, 5, 200, 333).to(DEV), torch.randn(6, 5, 200, 333).to(DEV), torch.randn(32, 5).to(DEV))
    q, gq, w, cos = torch.randn(4, 300, 6, 64).to(DEV), torch.randn(4, 300, 6, 64).to(DEV), torch.randn(64).to(DEV), torch.randn(300, 32).to(DEV)
    z, te, idx = torch.randn(700, 999).to(DEV), torch.randn(700, 8).to(DEV), torch.randint(0, 999, (700, 8)).to(DEV)

    def run():
        p, st = ops.relative_bias_softmax(s, t, None, 1.0, True, 64, 0)
        loss, stats, count = ops.top_logits_distillation_stats(z, te, idx, 1.0, 1)
        return [p, *ops.relative_bias_softmax_backward(g, s, st, t, None, 1.0, True, 64, 0, True),
                *ops.qk_norm_rotary_backward(gq, gq, q, q, w, w, cos, cos, None, 1e-6, False), loss]

    first = [x.cpu() for x in run()]
    for _ in range(3):
        assert all(torch.equal(a, b.cpu()) for a, b in zip(first, run()))


def test_calls_on_two_queues_and_from_two_threads():
    import threading

    x = [{k: v.to(DEV) for k, v in _inputs(20 + i).items()} for i in range(2)]
    want = [[t.cpu() for t in _all(v)] for v in x]
    torch.b200.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.no_grad(), torch.b200.stream(torch.b200.queue_from_pool()):
                for _ in range(20):
                    out = _all(x[i])
                got[i] = [t.cpu() for t in out]
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_an_index_out_of_range_raises_in_synchronous_mode():
    from catch_b200.fusion import qk_norm_rotary, top_logits_distillation

    cos, sin = torch.ones(4, 2).to(DEV), torch.zeros(4, 2).to(DEV)
    q = torch.randn(1, 3, 2, 8).to(DEV)
    z, te = torch.randn(2, 5).to(DEV), torch.randn(2, 2).to(DEV)
    torch.b200.set_flag("async_disable", True)
    try:
        with pytest.raises(IndexError, match="qk_norm_rotary"):
            qk_norm_rotary(q, q, None, None, cos, sin, torch.tensor([[0, 1, 4]]).to(DEV))
        with pytest.raises(IndexError, match="top_logits_distillation"):
            top_logits_distillation(z, te, torch.tensor([[0, 1], [2, 5]]).to(DEV))
        y, _ = qk_norm_rotary(q, q, None, None, cos, sin, torch.tensor([[-1, 0, 3]]).to(DEV))  # padding
        assert float(y[0, 0].abs().max()) == 0 and float(y[0, 1].abs().max()) > 0
        top_logits_distillation(z, te, torch.tensor([[0, -1], [-100, 4]]).to(DEV))
    finally:
        torch.b200.set_flag("async_disable", False)


# Offsets that pass 32 bits: zeros but for the last rows, which are compared with a call on those rows alone.
def test_scores_beyond_two_to_the_31():
    ops = torch.ops.catch_b200
    B, H, Lq, Lk = 3, 8, 9001, 10240  # 2.2e9 scores of 16 bits
    s = torch.zeros(B, H, Lq, Lk, dtype=torch.bfloat16, device=DEV)
    tail = torch.randn(H, 5, Lk).bfloat16().to(DEV)
    s[-1, :, -5:].copy_(tail)
    t = torch.randn(32, H).to(DEV)
    p, st = ops.relative_bias_softmax(s, t, None, 1.0, True, 128, 0)
    part, part_st = ops.relative_bias_softmax(tail.unsqueeze(0).contiguous(), t, None, 1.0, True, 128, Lq - 5)
    assert torch.equal(p[-1, :, -5:].cpu(), part[0].cpu()) and torch.equal(st[-1, :, -5:].cpu(), part_st[0].cpu())
    ds, _ = ops.relative_bias_softmax_backward(p, s, st, t, None, 1.0, True, 128, 0, False)
    part_ds, _ = ops.relative_bias_softmax_backward(part, tail.unsqueeze(0).contiguous(), part_st, t, None, 1.0, True, 128, Lq - 5, False)
    assert torch.equal(ds[-1, :, -5:].cpu(), part_ds[0].cpu())


def test_logits_and_heads_beyond_two_to_the_31():
    ops = torch.ops.catch_b200
    N, V = 17000, 131072  # 2.2e9 logits of 16 bits
    z = torch.zeros(N, V, dtype=torch.bfloat16, device=DEV)
    tail = torch.randn(3, V).bfloat16().to(DEV)
    z[-3:].copy_(tail)
    te, idx = torch.randn(N, 4).to(DEV), torch.randint(0, V, (N, 4)).to(DEV)
    g = torch.rand(N).to(DEV)
    loss, st, n = ops.top_logits_distillation_stats(z, te, idx, 1.0, 0)
    part, part_st, m = ops.top_logits_distillation_stats(tail, te[-3:], idx[-3:], 1.0, 0)
    assert torch.equal(loss[-3:].cpu(), part.cpu())
    dz = ops.top_logits_distillation_backward(g, z, st, n, te, idx, 1.0, 0)
    part_dz = ops.top_logits_distillation_backward(g[-3:], tail, part_st, m, te[-3:], idx[-3:], 1.0, 0)
    assert torch.equal(dz[-3:].cpu(), part_dz.cpu())
    del z, dz
    B, L, H, D = 2, 131101, 64, 128  # 2.1e9 elements of queries
    q = torch.zeros(B, L, H, D, dtype=torch.bfloat16, device=DEV)
    end = torch.randn(4, H, D).bfloat16().to(DEV)
    q[-1, -4:].copy_(end)
    k = torch.zeros(B, L, 1, D, dtype=torch.bfloat16, device=DEV)
    cos, sin = torch.randn(L, D // 2).to(DEV), torch.randn(L, D // 2).to(DEV)
    y, _ = ops.qk_norm_rotary(q, k, None, None, cos, sin)
    few, kf = end.unsqueeze(0), k[-1:, -4:]
    part, _ = ops.qk_norm_rotary(few, kf, None, None, cos[-4:], sin[-4:])
    assert torch.equal(y[-1, -4:].cpu(), part[0].cpu())
    dq = ops.qk_norm_rotary_backward(y, k, q, k, None, None, cos, sin, None, 1e-6, False)[0]
    part_dq = ops.qk_norm_rotary_backward(part, kf, few, kf, None, None, cos[-4:], sin[-4:], None, 1e-6, False)[0]
    assert torch.equal(dq[-1, -4:].cpu(), part_dq[0].cpu())


def test_the_guide_executes():
    from transformer_op_checks import guide

    guide()
