"""The transformer operators' kernels from row to row: sizes at which every block, group of lanes or item goes on to further rows, heads
or sequences, against the 64-bit forms.

Sums over rows are longer here than in transformer_op_checks, so the number of fp32 operations behind a result (``slack``) is counted for
each kind of sum.  Table gradient: a lane adds at most two results a row (SLACK covers the 30 rows of a group), a thread of the last step one
number for each of the blocks of a head (at most 148 x 8 over at least 2 heads, 592).  Loss of a mean or a sum: a thread of the last block adds
one row in 32 (N / 32).  Weight gradient: as in transformer_op_checks, some 16 heads a lane and 10 blocks a thread."""
import math

import pytest
import torch

import transformer_cases as cases
from transformer_cases import SLACK, check

pytestmark = pytest.mark.gpu
DEV = "blackwell"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TABLE_SLACK = SLACK + 592


@pytest.fixture(scope="module", autouse=True)
def _backend():
    import catch_b200  # noqa: F401

    assert torch.b200.backend_name() == "cuda"
    torch.b200.set_flag("op_trycatch", False)
    yield
    torch.b200.set_flag("op_trycatch", True)


def _mask(kind, dtype, B, Lq, Lk, offset):
    if kind == "causal":
        ahead = torch.arange(Lk) > torch.arange(Lq)[:, None] + offset
        return torch.zeros(Lq, Lk).masked_fill(ahead, -math.inf).to(dtype).view(1, 1, Lq, Lk)
    if kind == "padding":
        return torch.where(torch.arange(Lk) < torch.randint(Lk // 2, Lk + 1, (B, 1, 1, 1)), 0.0, -10000.0)
    if kind == "key bool":
        return torch.arange(Lk) < torch.randint(Lk // 2, Lk + 1, (B, 1, 1, 1))
    if kind == "random":  # some rows leave nothing
        return (torch.rand(B, 1, Lq, Lk) < 0.8) & (torch.rand(B, 1, Lq, 1) < 0.95)
    return None


@pytest.mark.parametrize("dtype, B, H, Lq, Lk, mask, bidirectional, layout", [
    (BF16, 3, 12, 233, 2048, None, True, None),            # whole rows over several warps
    (BF16, 3, 12, 233, 2048, "causal", False, None),
    (F16, 2, 4, 600, 4096, "key bool", True, None),
    (BF16, 4, 6, 300, 1024, "padding", True, "heads last"),
    (BF16, 4, 6, 300, 1024, "random", True, None),
    (F32, 2, 3, 500, 1024, None, True, None),
    (F32, 2, 3, 500, 1500, "key bool", False, None),       # ... whose last vectors are not all filled
    (BF16, 2, 4, 500, 1032, "causal", True, None),
    (BF16, 1, 3, 900, 5000, "key bool", True, None),       # four vectors a lane
    (BF16, 2, 3, 500, 1031, "random", True, None),         # rows that begin anywhere, over several warps
    (F32, 2, 3, 500, 1031, None, False, None),
    (BF16, 32, 12, 128, 128, "padding", True, None),       # several rows to a warp: sums move from row to row
    (BF16, 200, 12, 37, 64, None, True, None),             # and begin anew with a sequence
    (F16, 200, 12, 37, 64, "random", False, "heads last"),
    (F32, 90, 5, 67, 100, "padding", True, None),
    (BF16, 30, 7, 100, 200, "causal", True, None),
    (F32, 4, 7, 389, 517, "random", True, None),           # rows that begin anywhere, within a warp
    (BF16, 9, 7, 101, 333, None, True, None),
    (BF16, 300, 6, 31, 19, "key bool", False, None),
    (BF16, 2, 2, 350, 9000, "causal", True, None),         # beyond the registers
    (F32, 2, 2, 350, 5003, "random", False, None),
])
def test_softmax_from_row_to_row(dtype, B, H, Lq, Lk, mask, bidirectional, layout):
    from catch_b200.fusion import relative_bias_softmax

    torch.manual_seed(Lq + Lk)
    buckets, max_distance, scale, offset = 32, 128, 0.25, max(0, Lk - Lq) // 2
    s, g = torch.randn(B, H, Lq, Lk).to(dtype), torch.randn(B, H, Lq, Lk).to(dtype)
    t, m = torch.randn(buckets, H), _mask(mask, dtype, B, Lq, Lk, offset)
    if layout == "heads last":
        sd = s.permute(0, 2, 1, 3).contiguous().to(DEV).permute(0, 2, 1, 3).detach().requires_grad_()
    else:
        sd = s.to(DEV).requires_grad_()
    td = t.to(DEV).requires_grad_()
    probs = relative_bias_softmax(sd, td, None if m is None else m.to(DEV), scale=scale, bidirectional=bidirectional,
                                  max_distance=max_distance, query_offset=offset)
    ds, dt = torch.autograd.grad(probs, (sd, td), g.to(DEV))
    ref = cases.softmax_reference(s, t, m, g, scale, bidirectional, max_distance, offset)
    check(probs, *ref[0], "probabilities")
    check(ds, *ref[1], "score gradient")
    check(dt, *ref[2], "table gradient", slack=TABLE_SLACK)


@pytest.mark.parametrize("dtype, B, L, Hq, Hk, D, R, interleaved", [
    (BF16, 5, 2101, 10, 5, 64, 64, False),    # items of eight heads and of two, of five
    (F16, 5, 1101, 11, 3, 128, 64, True),     # of eight and of three, of three
    (F32, 3, 2101, 9, 9, 64, 64, False),      # of eight and of one
    (BF16, 7, 1601, 10, 5, 80, 32, True),     # lanes without a part of the head
    (BF16, 4, 701, 17, 2, 256, 256, False),
    (F16, 3, 1201, 5, 12, 36, 10, False),     # narrow vectors
    (BF16, 3, 401, 9, 10, 100, 50, False),    # single elements
])
@pytest.mark.parametrize("packed", [True, False])
def test_rotary_from_head_to_head(dtype, B, L, Hq, Hk, D, R, interleaved, packed):
    from catch_b200.fusion import qk_norm_rotary

    torch.manual_seed(D + L)
    x = torch.randn(B, L, Hq + 2 * Hk, D).to(dtype)
    if packed:
        xd = x.to(DEV).requires_grad_()
        q, k = xd[:, :, :Hq], xd[:, :, Hq:Hq + Hk]
    else:
        q, k = (t.contiguous().to(DEV).requires_grad_() for t in (x[:, :, :Hq], x[:, :, Hq:Hq + Hk]))
    qw, kw = ((1 + 0.3 * torch.randn(D)).to(DEV).requires_grad_() for _ in range(2))
    cos, sin = cases.tables(L, R)
    pos = torch.randint(-1, L, (B, L))
    gq, gk = torch.randn(B, L, Hq, D).to(dtype), torch.randn(B, L, Hk, D).to(dtype)
    yq, yk = qk_norm_rotary(q, k, qw, kw, cos.to(DEV), sin.to(DEV), pos.to(DEV), interleaved=interleaved)
    got = torch.autograd.grad((yq, yk), (q, k, qw, kw), (gq.to(DEV), gk.to(DEV)))
    for n, (xs, w, y, g) in enumerate(((x[:, :, :Hq], qw, yq, gq), (x[:, :, Hq:Hq + Hk], kw, yk, gk))):
        ry, rdx, rdw = cases.rotary_reference(xs, w, cos, sin, pos, 1e-6, interleaved, g)
        check(y, *ry, f"output {n}")
        check(got[n], *rdx, f"input gradient {n}")
        check(got[2 + n], *rdw, f"weight gradient {n}")


@pytest.mark.parametrize("dtype, N, V, K, layout", [
    (BF16, 2600, 20011, 40, None),      # two or three rows to a block of 128 threads
    (BF16, 1300, 33000, 64, "padded"),
    (F32, 2500, 9001, 16, None),
    (BF16, 12000, 40, 7, None),         # five to a block of two warps
    (F32, 11000, 33, 5, "padded"),
    (BF16, 700, 70001, 300, None),      # to a block of 512
])
@pytest.mark.parametrize("reduction, factor", [("mean", 1.0), ("sum", 1.0), ("mean", 0.3), ("none", 2.0)])
def test_distillation_from_row_to_row(dtype, N, V, K, layout, reduction, factor):
    from catch_b200.fusion import top_logits_distillation

    torch.manual_seed(V + K)
    T = 2.0
    z = (torch.randn(N, V) * 2).to(dtype)
    t = torch.randn(N, K) * 3
    idx = (torch.randint(0, V, (N, 1)) + torch.arange(K) * max(1, V // K)) % V
    idx[::3, K // 2:] = idx[::3, : K - K // 2]      # the same word more than once
    idx[torch.rand(N, K) < 0.3] = -1
    idx[torch.rand(N) < 0.2] = -100                 # rows without any
    if layout == "padded":
        wide = torch.zeros(N, V + 5, dtype=dtype)
        wide[:, :V] = z
        zd = wide.to(DEV)[:, :V].detach().requires_grad_()
    else:
        zd = z.to(DEV).requires_grad_()
    g = torch.rand(N) * factor if reduction == "none" else torch.tensor(factor)
    loss = top_logits_distillation(zd, t.to(DEV), idx.to(DEV), temperature=T, reduction=reduction)
    (dz,) = torch.autograd.grad(loss, zd, g.to(DEV))
    ref = cases.distill_reference(z, t, idx, T, reduction, g)
    slack = SLACK + (0 if reduction == "none" else N // 32)
    check(loss, *ref[0], "loss", slack=slack)
    check(dz, *ref[1], "gradient")
    with torch.no_grad():
        check(top_logits_distillation(zd, t.to(DEV), idx.to(DEV), temperature=T, reduction=reduction), *ref[0], "loss alone", slack=slack)


@pytest.mark.parametrize("mask_dtype", [F32, BF16, torch.bool])
def test_mask_bytes_beyond_two_to_the_31(mask_dtype):
    """One row of 2^29 keys and some: an additive fp32 mask has more than 2^31 bytes then."""
    ops = torch.ops.catch_b200
    n, last, some = (1 << 29) + 1000, 700, 6
    s = torch.zeros(1, 1, 1, n, dtype=BF16, device=DEV)
    m = torch.zeros(1, 1, 1, n, dtype=mask_dtype, device=DEV) if mask_dtype == torch.bool else \
        torch.full((1, 1, 1, n), -math.inf, dtype=mask_dtype, device=DEV)
    for part in (m[..., -last:], m[..., 8:8 + some]):
        part.fill_(True if mask_dtype == torch.bool else 0.0)
    t = torch.zeros(4, 1, device=DEV)
    p, st = ops.relative_bias_softmax(s, t, m, 1.0, False, 8, n - 1)
    want = torch.zeros(n, dtype=BF16)
    want[-last:] = want[8:8 + some] = 1.0 / (last + some)
    assert torch.equal(p.cpu().flatten(), want)
    g = torch.zeros(1, 1, 1, n, dtype=BF16, device=DEV)
    g[..., -1].fill_(1.0)
    ds, _ = ops.relative_bias_softmax_backward(g, s, st, t, m, 1.0, False, 8, n - 1, False)
    q = 1.0 / (last + some)
    ds = ds.cpu().flatten()
    assert int((ds != 0).sum()) == last + some
    assert abs(float(ds[-1]) - q * (1 - q)) <= q * 2.0 ** -8 and abs(float(ds[-2]) + q * q) <= q * q * 2.0 ** -7


@pytest.mark.parametrize("N, K", [(1, 1), (33, 1), (40, 2), (1000, 5), (700, 6), (300, 33), (5000, 64), (3000, 130), (16411, 17), (9, 1024), (70000, 3)])
@pytest.mark.parametrize("index_dtype", [torch.int64, torch.int32])
def test_the_number_of_rows_with_entries(N, K, index_dtype):
    """Exactly, wherever in a row its only entry stands."""
    torch.manual_seed(N + K)
    V = 50
    idx = torch.full((N, K), -1, dtype=index_dtype)
    kind, at = torch.randint(0, 4, (N,)), torch.randint(0, K, (N,))
    rows = torch.arange(N)
    idx[rows, at] = torch.where(kind == 0, -7, torch.randint(0, V, (N,))).to(index_dtype)     # none
    idx[kind == 1] = torch.randint(0, V, (int((kind == 1).sum()), K)).to(index_dtype)         # all
    te = torch.randn(N, K)
    te[rows[kind == 2], at[kind == 2]] = -math.inf                                            # one that the teacher excludes
    want = ((idx >= 0) & (te != -math.inf)).any(1).sum()
    z = torch.randn(N, V)
    loss, stats, count = torch.ops.catch_b200.top_logits_distillation_stats(z.to(DEV), te.to(DEV), idx.to(DEV), 1.0, 1)
    assert float(count[0]) == float(want)
    each = torch.ops.catch_b200.top_logits_distillation(z.to(DEV), te.to(DEV), idx.to(DEV), 1.0, 0).cpu().double()
    assert abs(float(loss) - float(each.sum()) / max(1, int(want))) <= (SLACK + N // 32) * cases.U * float(each.abs().sum()) / max(1, int(want))
