"""Checks of the transformer operators against their 64-bit forms: each entry of OPS_CHECKS is (function, arguments, needs a GPU);
the tests run them on the host-simulated device and on a GPU."""
import math

import torch

import transformer_cases as cases
from transformer_cases import check

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _grad(out, leaves, grads):
    return torch.autograd.grad(out, leaves, grads)


def rotary(dev, dtype=F32, B=2, L=7, Hq=4, Hk=2, D=16, R=16, interleaved=False, positions=None, packed=False, weights=F32, P=None,
           pos_dtype=torch.int64, table_dtype=F32, transposed=False, eps=1e-6, zero_row=False, grad_strided=False):
    from catch_b200.fusion import qk_norm_rotary

    torch.manual_seed(D * 31 + L)
    if packed:
        qkv = torch.randn(B, L, (Hq + 2 * Hk) * D).to(dtype).to(dev).requires_grad_()
        parts = qkv.view(B, L, Hq + 2 * Hk, D)
        q, k = parts[:, :, :Hq], parts[:, :, Hq:Hq + Hk]
    elif transposed:  # [B, H, L, D] memory
        q = torch.randn(B, Hq, L, D).to(dtype).to(dev).requires_grad_().transpose(1, 2)
        k = torch.randn(B, Hk, L, D).to(dtype).to(dev).requires_grad_().transpose(1, 2)
    else:
        q, k = torch.randn(B, L, Hq, D), torch.randn(B, L, Hk, D)
        if zero_row:
            q[0, 0] = 0
        q, k = q.to(dtype).to(dev).requires_grad_(), k.to(dtype).to(dev).requires_grad_()
    qw = kw = None
    if weights is not None:
        qw, kw = ((1 + 0.3 * torch.randn(D)).to(weights).to(dev).requires_grad_() for _ in range(2))
    cos, sin = (t.to(table_dtype) for t in cases.tables(P or max(L, 1), R))
    pos = None
    if positions == "rows":
        pos = torch.randint(0, cos.shape[0], (B, L), dtype=pos_dtype)
    elif positions == "line":
        pos = torch.randint(0, cos.shape[0], (L,), dtype=pos_dtype)
    elif positions == "outside":  # padding tokens and one beyond the tables
        pos = torch.randint(0, cos.shape[0], (B, L), dtype=pos_dtype)
        pos[:, 0], pos[-1, -1] = -1, cos.shape[0]
    yq, yk = qk_norm_rotary(q, k, qw, kw, cos.to(dev), sin.to(dev), None if pos is None else pos.to(dev), eps=eps, interleaved=interleaved)
    assert yq.is_contiguous() and yk.is_contiguous() and yq.dtype == dtype
    if grad_strided:
        gq = torch.randn(B, Hq, L, D).to(dtype).to(dev).transpose(1, 2)
    else:
        gq = torch.randn(B, L, Hq, D).to(dtype).to(dev)
    gk = torch.randn(B, L, Hk, D).to(dtype).to(dev)
    leaves = [q, k] + ([qw, kw] if weights is not None else [])
    got = _grad((yq, yk), leaves, (gq, gk))
    for n, (x, w, y, g) in enumerate(((q, qw, yq, gq), (k, kw, yk, gk))):
        ry, rdx, rdw = cases.rotary_reference(x, w, cos, sin, pos, eps, interleaved, g)
        check(y, *ry, f"output {n}")
        check(got[n], *rdx, f"input gradient {n}")
        if w is not None:
            assert got[2 + n].dtype == weights
            check(got[2 + n], *rdw, f"weight gradient {n}")


def softmax(dev, dtype=F32, B=2, H=3, Lq=9, Lk=13, mask=None, buckets=8, max_distance=20, bidirectional=True, offset=0, scale=0.5,
            table_dtype=F32, layout=None, grad_layout=None):
    from catch_b200.fusion import relative_bias_softmax

    torch.manual_seed(Lq * 7 + Lk)
    s = torch.randn(B, H, Lq, Lk) * 3
    g = torch.randn(B, H, Lq, Lk)
    m = None
    if mask == "key bool":
        m = torch.rand(B, 1, 1, Lk) < 0.7
    elif mask == "full bool":  # the first two rows leave nothing; scores and gradients hold junk where nothing is kept
        m = torch.rand(B, H, Lq, Lk) < 0.6
        m[..., :2, :] = False
        s = torch.where(m, s, torch.tensor([math.nan, math.inf, -math.inf, 1e30])[torch.randint(0, 4, s.shape)])
        g = torch.where(m, g, torch.tensor([math.nan, math.inf])[torch.randint(0, 2, s.shape)])
    elif mask == "key float":
        m = torch.where(torch.rand(B, 1, 1, Lk) < 0.7, 0.0, -10000.0)
    elif mask == "lowest":  # the type's lowest value, on whole rows too: those are as if nothing were masked
        m = torch.where(torch.rand(B, 1, Lq, Lk) < 0.7, 0.0, torch.finfo(dtype).min).to(dtype)
        m[:, :, 0] = torch.finfo(dtype).min
        s[:, :, 0] = s[:, :, 0].sign() * 0  # (there the scores vanish against the mask)
    elif mask == "inf":
        m = torch.where(torch.rand(1, H, Lq, Lk) < 0.7, torch.randn(1, H, Lq, Lk), torch.tensor(-math.inf)).to(dtype)
        m[:, :, 1] = -math.inf
        s = torch.where((m == -math.inf).expand_as(s), torch.tensor(math.nan), s)
    elif mask == "line":
        m = torch.where(torch.rand(Lk) < 0.7, torch.randn(Lk), torch.tensor(-math.inf))
    elif mask == "column":
        m = (torch.rand(Lq, 1) < 0.7)
    elif mask == "transposed":  # keys are not its innermost dimension in memory
        m = (torch.rand(B, 1, Lk, Lq) < 0.7).transpose(2, 3)
    t = torch.randn(buckets, H).to(table_dtype)
    sd = s.to(dtype).to(dev)
    if layout == "heads last":
        sd = s.to(dtype).permute(0, 2, 1, 3).contiguous().to(dev).permute(0, 2, 1, 3)
    elif layout == "slice":  # a part of a wider buffer, rows that begin anywhere
        wide = torch.zeros(B, H, Lq, Lk + 3, dtype=dtype)
        wide[..., 1:1 + Lk] = s.to(dtype)
        sd = wide.to(dev)[..., 1:1 + Lk]
    elif layout == "expanded":
        sd = s[:1].to(dtype).to(dev).expand(B, H, Lq, Lk)
        s = s[:1].expand(B, H, Lq, Lk)
    elif layout == "offset":  # contiguous, but not from a 16-byte boundary on
        sd = torch.cat([torch.zeros(1, dtype=dtype), s.to(dtype).flatten()]).to(dev)[1:].view(B, H, Lq, Lk)
    sd, td = sd.detach().requires_grad_(), t.to(dev).requires_grad_()
    probs = relative_bias_softmax(sd, td, None if m is None else m.to(dev), scale=scale, bidirectional=bidirectional,
                                  max_distance=max_distance, query_offset=offset)
    assert probs.dtype == dtype
    gd = g.to(dtype).to(dev)
    if grad_layout == "transposed":
        gd = g.to(dtype).transpose(2, 3).contiguous().to(dev).transpose(2, 3)
    elif grad_layout == "expanded":
        gd = g.to(dtype)[:, :, :, :1].to(dev).expand(B, H, Lq, Lk)
        g = g[:, :, :, :1].expand(B, H, Lq, Lk)
    ds, dt = _grad(probs, (sd, td), gd)
    ref = cases.softmax_reference(s.to(dtype), t, m, g.to(dtype), scale, bidirectional, max_distance, offset)
    check(probs, *ref[0], "probabilities")
    check(ds, *ref[1], "score gradient")
    assert dt.dtype == table_dtype
    check(dt, *ref[2], "table gradient")


def distill(dev, dtype=F32, N=6, V=37, K=5, T=2.0, reduction="mean", factor=1.0, absent=None, layout=None, index_dtype=torch.int64,
            teacher_dtype=F32, repeated=False, spread=3.0, infinite=False):
    from catch_b200.fusion import top_logits_distillation

    torch.manual_seed(V + K)
    z = (torch.randn(N, V) * spread).to(dtype)
    t, idx = cases.teacher_of(N, V, min(K, V), V, teacher_dtype)
    if repeated and K > 1:
        idx[:, K // 2:] = idx[:, : K - K // 2]
        idx[0] = idx[0, 0]
    if absent == "some":
        idx[torch.rand(idx.shape) < 0.4] = -1
        idx[0] = -100
        if N > 2:
            t[2] = -math.inf
        t[-1, -1] = -math.inf
    elif absent == "all":
        idx[:] = -1
    if infinite:  # words that the student may not choose
        z[:, ::3] = -math.inf
        for r in range(N):
            idx[r] = torch.where(idx[r] % 3 == 0, torch.full_like(idx[r], -1), idx[r])
        idx[0, 0] = 1
    zd = z.to(dev)
    if layout == "slice":  # a padded vocabulary
        wide = torch.zeros(N, V + 11, dtype=dtype)
        wide[:, 3:3 + V] = z
        zd = wide.to(dev)[:, 3:3 + V]
    elif layout == "transposed":
        zd = z.t().contiguous().to(dev).t()
    elif layout == "offset":
        zd = torch.cat([torch.zeros(1, dtype=dtype), z.flatten()]).to(dev)[1:].view(N, V)
    elif layout == "expanded":
        zd = z[:1].to(dev).expand(N, V)
        z = z[:1].expand(N, V)
    zd = zd.detach().requires_grad_()
    g = torch.rand(N) * factor if reduction == "none" else torch.tensor(float(factor))
    loss = top_logits_distillation(zd, t.to(dev), idx.to(index_dtype).to(dev), temperature=T, reduction=reduction)
    assert loss.dtype == F32
    ref = cases.distill_reference(z, t, idx, T, reduction, g)
    check(loss, *ref[0], "loss")
    for again in range(2):  # a retained graph gives the same gradient, with another factor one that fits it
        (dz,) = torch.autograd.grad(loss, zd, g.to(dev), retain_graph=True)
        check(dz, *ref[1], f"gradient {again}")
        assert dz.dtype == dtype
    (twice,) = torch.autograd.grad(loss, zd, 2 * g.to(dev), retain_graph=True)
    check(twice, ref[1][0] * 2, ref[1][1] * 2, "gradient of twice the loss")
    check(dz, *ref[1], "the earlier gradient is left alone")
    with torch.no_grad():
        check(top_logits_distillation(zd, t.to(dev), idx.to(index_dtype).to(dev), temperature=T, reduction=reduction), *ref[0], "loss alone")


def _entries():
    e = {}

    def add(name, fn, gpu=False, **kw):
        assert name not in e
        e[name] = (fn, kw, gpu)

    for t, n in ((F32, "f32"), (BF16, "bf16"), (F16, "f16")):
        add(f"rotary {n} half", rotary, dtype=t)
        add(f"rotary {n} interleaved partial", rotary, dtype=t, interleaved=True, R=8, Hq=3, Hk=1)
        add(f"rotary {n} packed", rotary, dtype=t, packed=True, positions="rows", P=50)
        add(f"rotary {n} odd dims", rotary, dtype=t, D=36, R=10, B=1, L=5)
        add(f"rotary {n} wide", rotary, dtype=t, D=256, R=256, B=1, L=3, Hq=2, Hk=2)
        add(f"rotary {n} outside", rotary, dtype=t, positions="outside", P=9)
        add(f"softmax {n} none", softmax, dtype=t)
        add(f"softmax {n} key float", softmax, dtype=t, mask="key float")
        add(f"softmax {n} full bool", softmax, dtype=t, mask="full bool")
        add(f"softmax {n} inf", softmax, dtype=t, mask="inf")
        add(f"softmax {n} lowest", softmax, dtype=t, mask="lowest")
        add(f"softmax {n} one query", softmax, dtype=t, Lq=1, Lk=41, offset=40, bidirectional=False)
        add(f"softmax {n} vectors", softmax, dtype=t, Lq=16, Lk=64, mask="key bool")
        add(f"distill {n} mean", distill, dtype=t)
        add(f"distill {n} sum", distill, dtype=t, reduction="sum", factor=0.25)
        add(f"distill {n} none", distill, dtype=t, reduction="none", absent="some", factor=3.0)
        add(f"distill {n} odd rows", distill, dtype=t, V=101, N=4, layout="slice")
        add(f"distill {n} scaled", distill, dtype=t, factor=1024.0)
    add("rotary line int32", rotary, positions="line", pos_dtype=torch.int32, P=30)
    add("rotary no weights", rotary, weights=None)
    add("rotary bf16 weights and tables", rotary, dtype=BF16, weights=BF16, table_dtype=BF16)
    add("rotary f16 weights", rotary, dtype=F16, weights=F16)
    add("rotary heads outer", rotary, transposed=True, D=8, R=4)
    add("rotary strided gradient", rotary, grad_strided=True)
    add("rotary no rotation", rotary, R=0)
    add("rotary smallest head", rotary, D=2, R=2)
    add("rotary largest head", rotary, D=512, R=2, B=1, L=2, Hq=1, Hk=1)
    add("rotary odd largest", rotary, D=510, R=254, B=1, L=2, Hq=1, Hk=1, interleaved=True)
    add("rotary one token", rotary, L=1, B=1, Hq=1, Hk=1)
    add("rotary no tokens", rotary, L=0)
    add("rotary no batch", rotary, B=0)
    add("rotary zero head", rotary, zero_row=True)
    add("rotary f16 two lanes", rotary, dtype=F16, D=20, R=20)
    add("softmax one key", softmax, Lk=1, Lq=3)
    add("softmax one by one", softmax, B=1, H=1, Lq=1, Lk=1)
    add("softmax no queries", softmax, Lq=0)
    add("softmax no batch", softmax, B=0)
    add("softmax line mask", softmax, mask="line")
    add("softmax column mask", softmax, mask="column")
    add("softmax transposed mask", softmax, mask="transposed")
    add("softmax heads last", softmax, layout="heads last")
    add("softmax slice", softmax, dtype=BF16, layout="slice")
    add("softmax offset", softmax, dtype=BF16, layout="offset")
    add("softmax expanded", softmax, layout="expanded")
    add("softmax transposed gradient", softmax, grad_layout="transposed")
    add("softmax expanded gradient", softmax, grad_layout="expanded")
    add("softmax bf16 table", softmax, dtype=BF16, table_dtype=BF16, Lq=20, Lk=30)
    add("softmax far offset", softmax, offset=1000)
    add("softmax negative offset", softmax, offset=-50)
    add("softmax negative scale", softmax, scale=-1.5)
    add("softmax two buckets", softmax, buckets=2, max_distance=2, bidirectional=False)
    add("softmax 514 keys", softmax, dtype=F32, B=1, H=2, Lq=40, Lk=514, buckets=32, max_distance=64, mask="key bool")
    add("softmax 1030 keys", softmax, dtype=BF16, B=1, H=1, Lq=33, Lk=1030, buckets=32, max_distance=128, mask="full bool")
    add("softmax 300 keys far reach", softmax, dtype=F16, B=2, H=2, Lq=300, Lk=300, buckets=64, max_distance=1000)
    add("softmax long row", softmax, dtype=BF16, B=1, H=2, Lq=5, Lk=9001, buckets=32, max_distance=128, offset=8996, mask="inf")
    add("softmax long reach", softmax, dtype=F32, B=1, H=1, Lq=3, Lk=5000, buckets=256, max_distance=8192, bidirectional=False, offset=4997)
    add("softmax narrow keys far reach", softmax, dtype=BF16, B=1, H=2, Lq=700, Lk=11, buckets=32, max_distance=512)
    add("softmax many rows", softmax, dtype=BF16, B=70, H=2, Lq=33, Lk=24, buckets=32, max_distance=128, mask="key float")
    add("distill one word", distill, V=1, K=1, N=3)
    add("distill two words", distill, V=2, K=2, N=5)
    add("distill one row", distill, N=1)
    add("distill no rows", distill, N=0)
    add("distill nothing kept", distill, K=0)
    add("distill all absent", distill, absent="all")
    add("distill all kept", distill, V=40, K=40)
    add("distill repeated", distill, repeated=True, K=7)
    add("distill int32 bf16 teacher", distill, index_dtype=torch.int32, teacher_dtype=BF16)
    add("distill transposed", distill, layout="transposed")
    add("distill offset", distill, dtype=BF16, layout="offset")
    add("distill expanded", distill, layout="expanded")
    add("distill forbidden words", distill, infinite=True)
    add("distill cold", distill, T=0.05)
    add("distill hot", distill, T=50.0)
    add("distill 5000 words", distill, dtype=BF16, V=5003, K=200, N=9, absent="some", repeated=True)
    add("distill many kept", distill, V=3001, K=1024, N=3, repeated=True)
    add("distill wide", distill, dtype=BF16, V=70001, K=64, N=3)
    add("distill many rows", distill, V=33, K=4, N=1500, absent="some")
    return e


OPS_CHECKS = _entries()


def run_check(name, dev):
    fn, kw, _ = OPS_CHECKS[name]
    fn(dev, **kw)


# ------------------------------------------------------------------------------------------ gradients against differences
def against_differences(f, x, grad, step, what):
    """``f`` (a number from fp32 tensors, summed in 64 bits) along three directions: the central difference is off by step^2 / 6 times
    the third derivative and by the rounding of f's fp32 results over the step; the functions here are sums of some hundred terms of
    size one with derivatives of size one, so 2^-8 relative to the gradient's length covers both at a step of 2^-7."""
    g = torch.Generator().manual_seed(5)
    for _ in range(3):
        v = torch.randn(x.shape, generator=g)
        v = v / v.norm()
        dev = v.to(x.device)
        slope = (f(x + step * dev) - f(x - step * dev)) / (2 * step)
        want = float((grad.detach().cpu().double() * v.double()).sum())
        assert abs(slope - want) <= 2.0 ** -8 * max(1.0, float(grad.detach().cpu().double().norm())), (what, slope, want)


def differences(dev):
    from catch_b200.fusion import qk_norm_rotary, relative_bias_softmax, top_logits_distillation

    torch.manual_seed(8)
    h = 2.0 ** -7
    total = lambda t, g: float((t.detach().cpu().double() * g.double()).sum())  # noqa: E731
    q, k, w = torch.randn(1, 3, 2, 8).to(dev), torch.randn(1, 3, 1, 8).to(dev), (1 + 0.2 * torch.randn(8)).to(dev)
    cos, sin = (t.to(dev) for t in cases.tables(3, 6))
    gq, gk = torch.randn(1, 3, 2, 8), torch.randn(1, 3, 1, 8)
    rot = lambda q, k, w: (lambda y: total(y[0], gq) + total(y[1], gk))(qk_norm_rotary(q, k, w, w, cos, sin))  # noqa: E731
    leaves = [t.clone().requires_grad_() for t in (q, k, w)]
    y = qk_norm_rotary(leaves[0], leaves[1], leaves[2], leaves[2], cos, sin)
    grads = torch.autograd.grad(y, leaves, (gq.to(dev), gk.to(dev)))
    for i, (t, g) in enumerate(zip((q, k, w), grads)):
        against_differences(lambda x: rot(*[x if j == i else o for j, o in enumerate((q, k, w))]), t, g, h, f"rotary {i}")
    s, t = torch.randn(2, 2, 5, 6).to(dev), torch.randn(4, 2).to(dev)
    m = torch.ones(2, 1, 5, 6, dtype=torch.bool)
    m[:, :, :, 4:] = False
    m[0, 0, 1] = False
    gp = torch.randn(2, 2, 5, 6)
    soft = lambda s, t: relative_bias_softmax(s, t, m.to(dev), scale=0.7, max_distance=6)  # noqa: E731
    sl, tl = s.clone().requires_grad_(), t.clone().requires_grad_()
    ds, dt = torch.autograd.grad(soft(sl, tl), (sl, tl), gp.to(dev))
    against_differences(lambda x: total(soft(x, t), gp), s, ds, h, "scores")
    against_differences(lambda x: total(soft(s, x), gp), t, dt, h, "table")
    z = torch.randn(4, 11).to(dev)
    te, idx = cases.teacher_of(4, 11, 3, 2)
    idx[0, 1] = -1
    loss = lambda z: top_logits_distillation(z, te.to(dev), idx.to(dev), temperature=1.5, reduction="sum")  # noqa: E731
    zl = z.clone().requires_grad_()
    (dz,) = torch.autograd.grad(loss(zl), zl)
    against_differences(lambda x: float(loss(x)), z, dz, h, "logits")


# -------------------------------------------------------------------------------------------------------- together
def _student(position, layers=2):
    from catch_b200.models.bert import BertConfig, BertForSequenceClassification

    torch.manual_seed(3)
    c = BertConfig(vocab_size=97, hidden_size=32, num_hidden_layers=layers, num_attention_heads=4, intermediate_size=64,
                   max_position_embeddings=40, num_labels=24, hidden_dropout_prob=0.0, attention_probs_dropout_prob=0.0,
                   position_embedding_type=position)
    m = BertForSequenceClassification(c)
    with torch.no_grad():
        for n, p in m.named_parameters():
            if "relative_bias" in n or n.endswith("_norm"):  # (not the places where their gradients would say nothing)
                p.add_(0.3 * torch.randn_like(p))
    return m


def student_step(dev, position, fused=False, dtype=None):
    """An encoder with the model's own switch for positions learns from a teacher's top logits: loss and gradients of one step, on
    ``dev`` and with plain modules on the host."""
    from catch_b200.fusion import top_logits_distillation
    from catch_b200.models.bert import fuse_bert

    torch.manual_seed(4)
    ids = torch.randint(0, 97, (3, 17))
    keep = torch.ones(3, 17)
    keep[1, 9:] = 0
    te, idx = cases.teacher_of(3, 24, 5, 1)

    def step(model, d, autocast):
        with torch.autocast(d.split(":")[0], dtype=dtype or torch.bfloat16, enabled=autocast):
            logits = model(ids.to(d), attention_mask=keep.to(d))
        loss = top_logits_distillation(logits, te.to(d), idx.to(d), temperature=2.0)
        loss.backward()
        return float(loss.detach()), {n: p.grad.detach().cpu().double() for n, p in model.named_parameters() if p.grad is not None}

    ref_loss, ref = step(_student(position), "cpu", False)
    model = _student(position).to(dev)
    got_loss, got = step(fuse_bert(model) if fused else model, dev, dtype is not None)
    assert set(got) == set(ref) and any("relative_bias" in n or n.endswith("_norm") for n in got) == (position != "absolute")
    # products of the device: TF32 (2^-11 a factor) or 16 bits (2^-8), through some twenty products in a row either way
    tol = 20 * 2 * (2.0 ** -11 if dtype is None else 2.0 ** -8)
    assert abs(got_loss - ref_loss) <= tol * abs(ref_loss)
    for n in ref:
        assert (got[n] - ref[n]).norm() <= tol * ref[n].norm() + 1e-6, (n, float((got[n] - ref[n]).norm() / ref[n].norm()))


GUIDE = """import torch, catch_b200
from catch_b200.fusion import qk_norm_rotary, relative_bias_softmax, top_logits_distillation

B, L, heads, dim, vocabulary = 2, 64, 4, 32, 1000
qkv = torch.randn(B, L, 3 * heads, dim).bfloat16().to("blackwell").requires_grad_()    # one packed projection
q, k, v = qkv[:, :, :heads], qkv[:, :, heads:2 * heads], qkv[:, :, 2 * heads:]          # slices, no copies

# norm of every query / key head and rotation by position, one pass over both
angle = torch.arange(L)[:, None] * 10000.0 ** (-torch.arange(0, dim, 2) / dim)
norm = torch.ones(dim).to("blackwell").requires_grad_()
q, k = qk_norm_rotary(q, k, norm, norm, angle.cos().to("blackwell"), angle.sin().to("blackwell"))

# scale + learned relative position bias + mask + softmax over the scores; the bias is never stored as a matrix
scores = torch.matmul(q.permute(0, 2, 1, 3), k.permute(0, 2, 3, 1))
table = torch.zeros(32, heads).to("blackwell").requires_grad_()
keep = torch.ones(B, 1, 1, L, dtype=torch.bool).to("blackwell")
probs = relative_bias_softmax(scores, table, keep, scale=dim ** -0.5, max_distance=128)
context = torch.matmul(probs, v.permute(0, 2, 1, 3))

# a student's logits against the teacher's 16 largest of every row
logits = torch.matmul(context.permute(0, 2, 1, 3).reshape(B * L, heads * dim),
                      torch.randn(heads * dim, vocabulary).bfloat16().to("blackwell"))
best, where = torch.randn(B * L, vocabulary).topk(16)
loss = top_logits_distillation(logits, best.to("blackwell"), where.to("blackwell"), temperature=2.0)
loss.backward()
"""


def guide():
    """The code of the training guide on positions and distillation, run as written."""
    names = {}
    exec(compile(GUIDE, "guide", "exec"), names)
    for leaf in ("qkv", "norm", "table"):
        assert bool(torch.isfinite(names[leaf].grad.float().cpu()).all()) and float(names[leaf].grad.float().cpu().abs().sum()) > 0
