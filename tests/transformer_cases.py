"""Plain 64-bit forms of the transformer operators with the error that each result may have, shared by the tests on the
host-simulated device and on a GPU.

A bound counts roundings: ``half_step(dtype)`` is the relative error of one rounding to the result's type, U that of one fp32
operation.  ``terms`` is the sum of the magnitudes that were added to give a result: every fp32 operation on the way is off by at
most U times that, so an operator with n operations in a row is off by n U terms at most.  The n used (SLACK) is 64: the longest chain
here is a reduction of a row over lanes and warps (some terms a lane, then at most 10 levels) behind an exponential of about 8 U."""
import math

import torch

U = 2.0 ** -24
SLACK = 64
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(out, ref, terms, what, slack=SLACK):
    assert out.shape == ref.shape, (what, out.shape, ref.shape)
    o, ref, terms = out.detach().cpu().double(), ref.detach().double(), terms.detach().double()
    # a result in the type's subnormal range is off by half the smallest subnormal
    tiny = torch.finfo(out.dtype).tiny * torch.finfo(out.dtype).eps / 2
    bound = half_step(out.dtype) * ref.abs() + slack * U * terms * (1 + half_step(out.dtype)) + tiny
    bad = ~((o - ref).abs() <= bound)
    if bool(bad.any()):
        i = int(torch.where(bad, ((o - ref).abs() / bound).nan_to_num(math.inf), 0.0).flatten().argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {o.numel()} are off; worst at {i}: {o.flatten()[i].item()!r} "
                             f"for {ref.flatten()[i].item()!r}, {bound.flatten()[i].item():.3g} allowed")


# ------------------------------------------------------------------------------------------------- norm and rotation
def rotate(n, cos, sin, R, interleaved, sign=1.0):
    out = n.clone()
    for i in range(R // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
        c, s = cos[..., i], sign * sin[..., i]
        out[..., a] = n[..., a] * c - n[..., b] * s
        out[..., b] = n[..., b] * c + n[..., a] * s
    return out


def rotate_terms(n, cos, sin, R, interleaved):
    """The magnitudes that rotate() adds: |a cos| + |b sin| and |b cos| + |a sin|."""
    out = n.abs().clone()
    for i in range(R // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
        c, s = cos[..., i].abs(), sin[..., i].abs()
        out[..., a] = n[..., a].abs() * c + n[..., b].abs() * s
        out[..., b] = n[..., b].abs() * c + n[..., a].abs() * s
    return out


def rotary_reference(x, w, cos, sin, positions, eps, interleaved, dy):
    """((y, terms), (dx, terms), (dw, terms)) for one of q and k, all on the host in 64 bits."""
    x, dy = x.detach().cpu().double(), dy.detach().cpu().double()
    cos, sin = cos.detach().cpu().double(), sin.detach().cpu().double()
    B, L, H, D = x.shape
    R = 2 * cos.shape[1]
    pos = torch.arange(L).expand(B, L) if positions is None else positions.cpu().long().expand(B, L)
    inside = ((pos >= 0) & (pos < cos.shape[0]))[:, :, None, None]
    at = pos.clamp(0, cos.shape[0] - 1)
    c, s = cos[at][:, :, None], sin[at][:, :, None]
    r = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    weight = torch.ones(D, dtype=torch.float64) if w is None else w.detach().cpu().double()
    n = x * r * weight
    keep = lambda t: torch.where(inside, t, torch.zeros_like(t))  # noqa: E731
    y = keep(rotate(n, c, s, R, interleaved))
    y_terms = keep(rotate_terms(n, c, s, R, interleaved))
    g = rotate(dy, c, s, R, interleaved, -1.0)
    g_terms = rotate_terms(dy, c, s, R, interleaved)
    dw = keep(g * x * r).sum((0, 1, 2))
    dw_terms = keep(g_terms * x.abs() * r).sum((0, 1, 2))
    dot = (g * weight * x).mean(-1, keepdim=True)
    dot_terms = (g_terms * weight.abs() * x.abs()).mean(-1, keepdim=True)
    dx = keep(r * (g * weight - x * r * r * dot))
    dx_terms = keep(r * (g_terms * weight.abs() + x.abs() * r * r * dot_terms))
    return (y, y_terms), (dx, dx_terms), (dw, dw_terms)


def tables(P, R, seed=0):
    if R == 0:
        return torch.zeros(P, 0), torch.zeros(P, 0)
    angle = torch.arange(P)[:, None] * 10000.0 ** (-torch.arange(0, R, 2) / R) + 0.1 * seed
    return angle.cos(), angle.sin()


# ---------------------------------------------------------------------------------------------------- biased softmax
def bucket_of(rel, buckets, bidirectional, max_distance):
    n = buckets // 2 if bidirectional else buckets
    d, up = (abs(rel), n if rel > 0 else 0) if bidirectional else (max(0, -rel), 0)
    exact, far = n // 2, n - n // 2
    if d < exact:
        return up + d
    return up + exact + max(k for k in range(far) if k == 0 or d ** far >= max_distance ** k * exact ** (far - k))


def softmax_reference(scores, table, mask, dprobs, scale, bidirectional, max_distance, offset):
    """((probs, terms), (dscores, terms), (dtable, terms))"""
    s, t, g = scores.detach().cpu().double(), table.detach().cpu().double(), dprobs.detach().cpu().double()
    B, H, Lq, Lk = s.shape
    of = {rel: bucket_of(rel, t.shape[0], bidirectional, max_distance) for rel in range(-(Lq - 1) - offset, Lk - offset)}
    bucket = torch.tensor([[of[j - i - offset] for j in range(Lk)] for i in range(Lq)], dtype=torch.long).view(Lq, Lk)
    bias = t[bucket].permute(2, 0, 1)
    a = s * scale + bias
    size = s.abs() * abs(scale) + bias.abs()
    if mask is not None:
        mask = mask.cpu()
        if mask.dtype == torch.bool:
            a = a.masked_fill(~mask, -math.inf)
        else:
            m = mask.double()
            a = (a + m).masked_fill(m == -math.inf, -math.inf)
            size = size + m.masked_fill(m == -math.inf, 0.0).abs()
    gone = a == -math.inf
    top = a.amax(-1, keepdim=True)
    e = torch.exp(a - top).masked_fill(gone, 0.0)
    total = e.sum(-1, keepdim=True)
    p = torch.where(total == 0, torch.zeros_like(e), e / total)
    # an error of the exponent counts as it is: |a| and the row's largest |a| each take part in it
    grow = 1 + size.masked_fill(gone, 0.0) + size.masked_fill(gone, 0.0).amax(-1, keepdim=True)
    grow = torch.where(p > 0, grow, torch.ones_like(grow)).clamp(max=1e6)
    g = g.masked_fill(p == 0, 0.0)
    dot = (p * g).sum(-1, keepdim=True)
    d = p * (g - dot)
    worst = torch.where(p > 0, grow, torch.zeros_like(grow)).amax(-1, keepdim=True)
    d_terms = p * (g.abs() + (p * g.abs()).sum(-1, keepdim=True)) * worst
    dt, dt_terms = torch.zeros_like(t), torch.zeros_like(t)
    dt.index_add_(0, bucket.flatten(), d.sum(0).permute(1, 2, 0).reshape(-1, H))
    dt_terms.index_add_(0, bucket.flatten(), d_terms.sum(0).permute(1, 2, 0).reshape(-1, H))
    # results below the smallest normal fp32 number may be flushed
    return (p, p * grow + 2.0 ** -126 / U), (d * scale, d_terms * abs(scale) + 2.0 ** -126 / U * (1 + (g.abs().amax() if g.numel() else 0.0))), (dt, dt_terms + 2.0 ** -120 / U)


# ------------------------------------------------------------------------------------------------------- distillation
def distill_reference(logits, teacher, index, T, reduction, factor):
    """((loss, terms), (dlogits, terms)); factor: the gradient of the loss, a number or one for each row."""
    z, t, idx = logits.detach().cpu().double(), teacher.detach().cpu().double(), index.cpu().long()
    N, V = z.shape
    loss, terms = torch.zeros(N, dtype=torch.float64), torch.zeros(N, dtype=torch.float64)
    logq = torch.log_softmax(z / T, 1)
    spread = torch.zeros(N, V, dtype=torch.float64)
    real = torch.zeros(N, dtype=torch.bool)
    for r in range(N):
        there = (idx[r] >= 0) & (idx[r] < V) & (t[r] != -math.inf)
        real[r] = bool(there.any())
        if not real[r]:
            continue
        p = torch.softmax(t[r][there] / T, 0)
        lq = logq[r][idx[r][there]]
        size = 1 + t[r][there].abs().amax() / T + z[r].abs().masked_fill(z[r].isinf(), 0).amax() / T
        loss[r] = T * T * (p * (p.log() - lq)).sum()
        terms[r] = T * T * (p * (p.log().abs() + lq.abs() + size)).sum()
        spread[r].index_add_(0, idx[r][there], p)
    count = max(1, int(real.sum())) if reduction == "mean" else 1
    f = torch.as_tensor(factor, dtype=torch.float64).expand(N) * T / count * real
    q = logq.exp()
    size = 1 + 2 * z.abs().masked_fill(z.isinf(), 0).amax() / T + t.abs().masked_fill(t.isinf(), 0).amax() / T if t.numel() else torch.tensor(1.0)
    d = f[:, None] * torch.where(real[:, None], q - spread, torch.zeros_like(q))
    d_terms = f.abs()[:, None] * (q.nan_to_num() + spread) * size + 2.0 ** -126 / U
    if reduction != "none":
        loss, terms = loss.sum() / count, terms.sum() / count
    return (loss, terms), (d, d_terms)


def teacher_of(N, V, K, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    idx = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(N)]) if N else torch.zeros(0, K, dtype=torch.long)
    return (torch.randn(N, K, generator=g) * 3).sort(1, descending=True).values.to(dtype), idx
