"""Query / key norm with rotation, softmax with a relative position bias and distillation from a teacher's top logits:
refusals and results of the host paths, on the host-simulated device and on CPU tensors."""
import math

import pytest
import torch

import transformer_cases as cases
from transformer_op_checks import OPS_CHECKS, run_check


@pytest.fixture(scope="module", autouse=True)
def _backend():
    import catch_b200  # noqa: F401


@pytest.mark.parametrize("name", [c for c in OPS_CHECKS if not OPS_CHECKS[c][2]])
def test_host_path(name):
    run_check(name, "blackwell")


@pytest.mark.parametrize("name", ["rotary f32 half", "softmax f32 none", "distill f32 mean"])
def test_cpu_tensors(name):
    run_check(name, "cpu")


def _rotary_args(**change):
    cos, sin = cases.tables(8, 6)
    a = dict(q=torch.randn(2, 5, 4, 8), k=torch.randn(2, 5, 2, 8), q_weight=torch.ones(8), k_weight=None, cos=cos, sin=sin)
    a.update(change)
    return a


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.randn(2, 5, 8)), "batch, length, heads, head_dim"),
    (dict(k=torch.randn(2, 4, 2, 8)), "differ in batch, length or head_dim"),
    (dict(k=torch.randn(2, 5, 2, 8).bfloat16()), "both float32"),
    (dict(q=torch.randn(2, 5, 4, 8).double(), k=torch.randn(2, 5, 2, 8).double()), "float32, bfloat16 or float16"),
    (dict(q=torch.randn(2, 5, 4, 7), k=torch.randn(2, 5, 2, 7), q_weight=None), "even"),
    (dict(q=torch.randn(1, 1, 1, 514), k=torch.randn(1, 1, 1, 514), q_weight=None), "at most 512"),
    (dict(cos=torch.ones(8, 5), sin=torch.ones(8, 5)), "rotate 10 dimensions of 8"),
    (dict(cos=torch.ones(8, 2)), "cos and sin"),
    (dict(cos=torch.ones(8, 2).double(), sin=torch.ones(8, 2).double()), "floating tables"),
    (dict(cos=torch.ones(4, 2), sin=torch.ones(4, 2)), "5 tokens, but cos and sin have 4 positions"),
    (dict(q_weight=torch.ones(4)), "weights are floating"),
    (dict(q_weight=torch.ones(8, dtype=torch.long)), "weights are floating"),
    (dict(positions=torch.zeros(2, 5)), "int64 or int32"),
    (dict(positions=torch.zeros(3, 5, dtype=torch.long)), r"\[batch, length\] or \[length\]"),
    (dict(eps=-1.0), "eps"),
    (dict(cos=torch.ones(8, 2, requires_grad=True), sin=torch.ones(8, 2)), "constants"),
    (dict(q_weight=torch.ones(8, device="meta")), "same device"),
])
def test_rotary_refusals(change, message):
    from catch_b200.fusion import qk_norm_rotary

    with pytest.raises(RuntimeError, match=message):
        qk_norm_rotary(**_rotary_args(**change))


@pytest.mark.parametrize("change, message", [
    (dict(scores=torch.randn(4, 5, 6)), "batch, heads, queries, keys"),
    (dict(scores=torch.randn(2, 3, 5, 6).double()), "float32, bfloat16 or float16"),
    (dict(table=torch.randn(8, 4)), "buckets, heads"),
    (dict(table=torch.randint(0, 3, (8, 3))), "floating"),
    (dict(table=torch.randn(7, 3)), "even number"),
    (dict(table=torch.randn(2, 3)), "between 4"),
    (dict(table=torch.randn(600, 3)), "between 4"),
    (dict(max_distance=2), "above 2"),
    (dict(max_distance=10000), "at most"),
    (dict(query_offset=1 << 40), "2\\^30"),
    (dict(scale=math.inf), "finite"),
    (dict(mask=torch.zeros(2, 1, 5, 6, dtype=torch.long)), "bool"),
    (dict(mask=torch.zeros(2, 1, 5, 7)), "broadcast"),
    (dict(mask=torch.zeros(1, 2, 1, 5, 6)), "four dimensions"),
    (dict(mask=torch.zeros(2, 1, 1, 6, requires_grad=True)), "no gradient"),
    (dict(mask=torch.zeros(2, 1, 1, 6, device="meta")), "same device"),
])
def test_softmax_refusals(change, message):
    from catch_b200.fusion import relative_bias_softmax

    a = dict(scores=torch.randn(2, 3, 5, 6), table=torch.randn(8, 3))
    a.update(change)
    with pytest.raises(RuntimeError, match=message):
        relative_bias_softmax(**a)


@pytest.mark.parametrize("change, error, message", [
    (dict(logits=torch.randn(3, 4, 5)), RuntimeError, "rows, vocabulary"),
    (dict(logits=torch.randn(4, 9).double()), RuntimeError, "float32, bfloat16 or float16"),
    (dict(teacher_logits=torch.randn(3, 2)), RuntimeError, "rows, kept"),
    (dict(teacher_index=torch.zeros(4, 3, dtype=torch.long)), RuntimeError, "shape of its logits"),
    (dict(teacher_index=torch.zeros(4, 2)), RuntimeError, "int64 or int32"),
    (dict(logits=torch.randn(4, 0)), RuntimeError, "vocabulary of 0"),
    (dict(logits=torch.randn(1, 2000), teacher_logits=torch.zeros(1, 1025), teacher_index=torch.zeros(1, 1025, dtype=torch.long)), RuntimeError, "at most 1024"),
    (dict(temperature=0.0), RuntimeError, "temperature"),
    (dict(temperature=math.nan), RuntimeError, "temperature"),
    (dict(reduction="batchmean"), ValueError, "reduction"),
    (dict(teacher_logits=torch.randn(4, 2, requires_grad=True)), RuntimeError, "detach"),
    (dict(teacher_index=torch.zeros(4, 2, dtype=torch.long, device="meta")), RuntimeError, "same device"),
])
def test_distillation_refusals(change, error, message):
    from catch_b200.fusion import top_logits_distillation

    a = dict(logits=torch.randn(4, 9), teacher_logits=torch.randn(4, 2), teacher_index=torch.zeros(4, 2, dtype=torch.long))
    a.update(change)
    with pytest.raises(error, match=message):
        top_logits_distillation(**a)


def test_the_gradient_of_the_gradient_raises():
    from catch_b200.fusion import qk_norm_rotary, relative_bias_softmax, top_logits_distillation

    cos, sin = cases.tables(4, 4)
    q, s, z = (torch.randn(sh, requires_grad=True) for sh in ((1, 3, 2, 8), (1, 2, 3, 4), (3, 7)))
    outs = [(qk_norm_rotary(q, q.detach(), None, None, cos, sin)[0], q),
            (relative_bias_softmax(s, torch.randn(8, 2)), s),
            (top_logits_distillation(z, torch.randn(3, 2), torch.zeros(3, 2, dtype=torch.long)), z)]
    for y, leaf in outs:
        (g,) = torch.autograd.grad(y.sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="gradient of the gradient"):
            g.sum().backward()


@pytest.mark.parametrize("buckets, bidirectional, max_distance", [(32, True, 128), (32, False, 128), (64, True, 256), (4, True, 8),
                                                                 (2, False, 2), (256, False, 2048), (512, True, 8192), (18, True, 60)])
def test_bucket_borders_are_exact(buckets, bidirectional, max_distance):
    """With zero scores and one bucket's entry raised, the keys of that bucket show in the probabilities."""
    from catch_b200.fusion import relative_bias_softmax

    far = min(max_distance + 3, 600)
    want = torch.tensor([cases.bucket_of(j - far, buckets, bidirectional, max_distance) for j in range(2 * far + 1)])
    table = torch.arange(buckets, dtype=torch.float32)[:, None] / buckets  # all different
    p = relative_bias_softmax(torch.zeros(1, 1, 1, 2 * far + 1), table, bidirectional=bidirectional, max_distance=max_distance, query_offset=far)
    p = p.flatten().double().log()
    got = ((p - p[far]) * buckets).round().long() + want[far]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dev", ["cpu", "blackwell"])
def test_gradients_against_differences(dev):
    from transformer_op_checks import differences

    differences(dev)


@pytest.mark.parametrize("position", ["absolute", "relative_bias", "rotary"])
@pytest.mark.parametrize("fused", [False, True])
def test_a_student_learns_from_a_teacher(position, fused):
    from transformer_op_checks import student_step

    student_step("blackwell", position, fused)


def test_position_types_of_the_encoder():
    from catch_b200.models.bert import BertConfig, BertForSequenceClassification

    small = dict(vocab_size=50, hidden_size=16, num_hidden_layers=1, num_attention_heads=2, intermediate_size=32, max_position_embeddings=10)
    names = {t: set(BertForSequenceClassification(BertConfig(position_embedding_type=t, **small)).state_dict()) for t in
             ("absolute", "relative_bias", "rotary")}
    assert names["absolute"] == set(BertForSequenceClassification(BertConfig(**small)).state_dict())
    base = names["absolute"] - {"embeddings.position_embeddings.weight"}
    assert names["relative_bias"] == base | {"layers.0.attention.relative_bias"}
    assert names["rotary"] == base | {"layers.0.attention.query_norm", "layers.0.attention.key_norm"}
    with pytest.raises(ValueError, match="position_embedding_type"):
        BertForSequenceClassification(BertConfig(position_embedding_type="learned", **small))
    with pytest.raises(RuntimeError, match="12 tokens, but cos and sin have 10 positions"):
        BertForSequenceClassification(BertConfig(position_embedding_type="rotary", **small))(torch.zeros(1, 12, dtype=torch.long))


def test_an_index_out_of_range_raises_in_synchronous_mode():
    from catch_b200.fusion import qk_norm_rotary, top_logits_distillation

    cos, sin = cases.tables(4, 4)
    q = torch.randn(1, 3, 2, 8)
    torch.b200.set_flag("async_disable", True)
    try:
        with pytest.raises(IndexError, match="qk_norm_rotary"):
            qk_norm_rotary(q, q, None, None, cos, sin, torch.tensor([[0, 1, 4]]))
        with pytest.raises(IndexError, match="top_logits_distillation"):
            top_logits_distillation(torch.randn(2, 5), torch.randn(2, 2), torch.tensor([[0, 1], [2, 5]]))
        y, _ = qk_norm_rotary(q, q, None, None, cos, sin, torch.tensor([[-1, 0, 3]]))  # padding
        assert y[0, 0].abs().max() == 0 and y[0, 1].abs().max() > 0
        top_logits_distillation(torch.randn(2, 5), torch.randn(2, 2), torch.tensor([[0, -1], [-100, 4]]))
    finally:
        torch.b200.set_flag("async_disable", False)


def test_the_guide_executes():
    from pathlib import Path

    from transformer_op_checks import GUIDE, guide

    assert GUIDE in (Path(__file__).resolve().parent.parent / "docs" / "training.md").read_text()
    guide()
