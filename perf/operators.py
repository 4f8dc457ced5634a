"""Cases of the transformer operators in ``catch_b200.fusion`` and their plain forms.

Three operators of an encoder's training step: the norm and rotation of queries and keys (``qk_norm_rotary``), the
softmax over scores with a learned relative position bias (``relative_bias_softmax``), and the distillation loss against
a teacher's top logits (``top_logits_distillation``).  ``run`` makes the framework's calls where ``own`` is true and
computes the same in elementary torch operations, in 32 bits or more, where it is false.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


# ---------------------------------------------------------------------------------------------------------- the cases
def _rotary(name, B, L, Hq, Hk, D, R, dtype, train, packed=False, interleaved=False, given=False, weights=True):
    """q [B, L, Hq, D], k [B, L, Hk, D]; the first R dimensions rotate; ``packed``: q and k are slices of one projection's
    result; ``given``: positions come as a tensor (packed documents that each begin at zero)."""
    return {"name": name, "op": "rotary", "B": B, "L": L, "Hq": Hq, "Hk": Hk, "D": D, "R": R, "dtype": dtype,
            "train": train, "packed": packed, "interleaved": interleaved, "given": given, "weights": weights}


def _softmax(name, B, H, Lq, Lk, dtype, train, mask, buckets=32, max_distance=128, bidirectional=True):
    """scores [B, H, Lq, Lk]; ``mask``: none, "key" (additive, -10000 on padded keys, [B, 1, 1, Lk]), "bool" ([B, 1, Lq, Lk], some
    rows leave no key) or "inf" (additive -inf above the diagonal, [1, 1, Lq, Lk], in the scores' type)."""
    return {"name": name, "op": "softmax", "B": B, "H": H, "Lq": Lq, "Lk": Lk, "dtype": dtype, "train": train,
            "mask": mask, "buckets": buckets, "max_distance": max_distance, "bidirectional": bidirectional}


def _distill(name, N, V, K, dtype, train, temperature, reduction, padded=False):
    """logits [N, V], the teacher's top K; ``padded``: some rows have fewer entries, some none at all (index -1)."""
    return {"name": name, "op": "distill", "N": N, "V": V, "K": K, "dtype": dtype, "train": train,
            "temperature": temperature, "reduction": reduction, "padded": padded}


def listed():
    return [
        # one new token for each of eight sequences: the smallest call, where the launch is what costs
        _rotary("rotary one token", 8, 1, 12, 12, 64, 64, "bf16", False, given=True),
        # a training batch of the base-size encoder in models/bert.py (32 x 128 tokens, 12 heads of 64)
        _rotary("rotary encoder batch", 32, 128, 12, 12, 64, 64, "bf16", True),
        # long sequences with shared key heads, read out of the packed projection without a copy
        _rotary("rotary long shared keys", 8, 2048, 32, 8, 128, 128, "bf16", True, packed=True),
        # ragged length, partial rotation of adjacent pairs, packed documents, half precision
        _rotary("rotary ragged partial", 3, 1021, 10, 5, 80, 32, "f16", True, interleaved=True, given=True),
        # one query over a long row of keys: a step of generation
        _softmax("bias softmax one query", 4, 12, 1, 1537, "f16", False, "none", bidirectional=False),
        # the scores of one layer of the base-size encoder, with its additive padding mask
        _softmax("bias softmax encoder", 32, 12, 128, 128, "bf16", True, "key"),
        # long sequences: the scores of one layer fill 200 MB
        _softmax("bias softmax long", 2, 12, 2048, 2048, "bf16", True, "inf", bidirectional=False),
        # odd lengths, rows that a mask leaves empty, 32-bit scores, a longer reach of the bias
        _softmax("bias softmax ragged", 3, 7, 389, 517, "f32", True, "bool", buckets=64, max_distance=256),
        # a classifier over 1000 classes learning from its teacher's five best
        _distill("distill classifier", 128, 1000, 5, "f16", True, 4.0, "mean"),
        # masked-word prediction over the encoder's vocabulary of 30522 words, 64 logits kept
        _distill("distill encoder vocabulary", 4096, 30522, 64, "bf16", True, 2.0, "mean"),
        # a large vocabulary
        _distill("distill large vocabulary", 4096, 131072, 128, "bf16", True, 1.0, "mean"),
        # odd vocabulary in 32 bits, a loss for each row, rows with few or no kept logits
        _distill("distill ragged rows", 777, 50021, 37, "f32", True, 1.5, "none", padded=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rotary", "softmax", "distill"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    train = rng.random() < 0.75
    if op == "rotary":
        D = rng.choice((32, 40, 64, 64, 72, 80, 96, 100, 128, 128, 192, 256))
        R = rng.choice((D, D, D // 4 * 2, 16))
        Hk = rng.randint(1, 12)
        Hq = Hk * rng.choice((1, 1, 2, 3, 4))
        tokens = _log(rng, 1, max(2, min(20000, 80_000_000 // ((Hq + Hk) * D * (2 if dtype == "f32" else 1)))))
        B = min(tokens, rng.randint(1, 16))
        c = _rotary("", B, max(1, tokens // B), Hq, Hk, D, R, dtype, train, rng.random() < 0.4, rng.random() < 0.4,
                    rng.random() < 0.5, rng.random() < 0.8)
    elif op == "softmax":
        H = rng.randint(1, 16)
        Lk = _log(rng, 4, 4096)  # over a single key the answer is one and its gradient zero
        Lq = 1 if rng.random() < 0.2 else rng.choice((Lk, Lk, _log(rng, 1, 2048)))
        B = _log(rng, 1, max(1.0, min(64.0, 90e6 / (H * Lq * Lk * (2 if dtype == "f32" else 1)))))
        H = max(1, min(H, int(90e6 / (B * Lq * Lk * (2 if dtype == "f32" else 1)))))
        c = _softmax("", B, H, Lq, Lk, dtype, train, rng.choice(("none", "key", "bool", "inf")), rng.choice((16, 32, 64)),
                     rng.choice((64, 128, 128, 256)), rng.random() < 0.6)
    else:
        V = _log(rng, 8, 131072)
        N = _log(rng, 4, min(8192, max(2, 500_000_000 // (V * (2 if dtype == "f32" else 1)))))
        c = _distill("", N, V, min(V, _log(rng, 2, 256)), dtype, train, rng.choice((1.0, 1.5, 2.0, 4.0)),
                     rng.choice(("mean", "mean", "sum", "none")), rng.random() < 0.4)
    del c["name"]
    return c


# --------------------------------------------------------------------------------------------------------- the inputs
def _normal(g, shape, scale=1.0):
    """Normal values on the host, in 32 bits.  Beyond four million they repeat in shifted runs: drawing them all would take
    most of the time of a measurement."""
    n, block = math.prod(shape), 1 << 22
    if n <= block:
        return torch.randn(shape, generator=g) * scale
    base = torch.randn(block, generator=g) * scale
    shifts = torch.randint(0, block, (-(-n // block),), generator=g).tolist()
    return torch.cat([base.roll(s) for s in shifts])[:n].view(shape)


def _rotary_inputs(c, g):
    B, L, Hq, Hk, D, R, t = c["B"], c["L"], c["Hq"], c["Hk"], c["D"], c["R"], _DTYPES[c["dtype"]]
    x = {}
    if c["packed"]:  # what one projection gives for queries, keys and values
        x["qkv"] = _normal(g, (B, L, (Hq + 2 * Hk) * D), 1.5).to(t)
    else:
        x["q"], x["k"] = _normal(g, (B, L, Hq, D), 1.5).to(t), _normal(g, (B, L, Hk, D), 0.7).to(t)
    if c["weights"]:
        x["qw"], x["kw"] = 1 + 0.2 * torch.randn(D, generator=g), 1 + 0.2 * torch.randn(D, generator=g)
    P = max(L, 2048)
    angle = torch.arange(P, dtype=torch.float64)[:, None] * (10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R))
    x["cos"], x["sin"] = angle.cos().float(), angle.sin().float()
    if c["given"]:
        x["positions"] = (torch.arange(L) + torch.randint(0, P, (B, 1), generator=g)) % P
    if c["train"]:
        x["dq"], x["dk"] = _normal(g, (B, L, Hq, D)).to(t), _normal(g, (B, L, Hk, D)).to(t)
    return x


def _softmax_inputs(c, g):
    B, H, Lq, Lk, t = c["B"], c["H"], c["Lq"], c["Lk"], _DTYPES[c["dtype"]]
    x = {"scores": _normal(g, (B, H, Lq, Lk), 16.0).to(t), "table": torch.randn((c["buckets"], H), generator=g)}
    if c["mask"] == "key":
        lengths = torch.randint(max(1, Lk // 2), Lk + 1, (B, 1, 1, 1), generator=g)
        x["mask"] = torch.where(torch.arange(Lk) < lengths, 0.0, -10000.0)
    elif c["mask"] == "bool":
        x["mask"] = torch.rand((B, 1, Lq, Lk), generator=g) < 0.8
        x["mask"] &= torch.rand((B, 1, Lq, 1), generator=g) < 0.95  # the others leave nothing
    elif c["mask"] == "inf":
        ahead = torch.arange(Lk) > torch.arange(Lq)[:, None] + max(0, Lk - Lq)
        x["mask"] = torch.zeros(Lq, Lk).masked_fill(ahead, -math.inf).to(t).view(1, 1, Lq, Lk)
    if c["train"]:
        x["dprobs"] = _normal(g, (B, H, Lq, Lk)).to(t)
    return x


def _distill_inputs(c, g):
    N, V, K = c["N"], c["V"], c["K"]
    x = {"logits": _normal(g, (N, V), 2.5).to(_DTYPES[c["dtype"]])}
    x["index"] = (torch.randint(0, V, (N, 1), generator=g) + torch.arange(K) * (V // K)) % V
    x["teacher"] = 8.0 - torch.cumsum(torch.rand((N, K), generator=g) * (6.0 / K), 1)  # falling, as a sorted top K
    if c["padded"]:
        kept = torch.randint(0, K + 1, (N, 1), generator=g)
        kept[0] = K
        x["index"] = torch.where(torch.arange(K) < kept, x["index"], -1)
    if c["train"]:
        # the loss is where backward() begins; half precision trains with a loss scale
        x["g"] = (torch.rand(N, generator=g) if c["reduction"] == "none" else torch.ones(())) * (1024 if c["dtype"] == "f16" else 1)
    return x


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator().manual_seed(seed)
    x = {"rotary": _rotary_inputs, "softmax": _softmax_inputs, "distill": _distill_inputs}[c["op"]](c, g)
    device = "cuda"
    if own:  # the framework's operators take tensors of its own device
        import catch_b200  # noqa: F401

        device = "blackwell"
    x = {k: v.to(device) for k, v in x.items()}
    if "qkv" in x:
        B, L, D, Hq, Hk = c["B"], c["L"], c["D"], c["Hq"], c["Hk"]
        parts = x.pop("qkv").view(B, L, Hq + 2 * Hk, D)
        x["q"], x["k"] = parts[:, :, :Hq], parts[:, :, Hq:Hq + Hk]
    if own and c["train"]:
        x.update({k: x[k].detach().requires_grad_() for k in ("q", "k", "qw", "kw", "scores", "table", "logits") if k in x})
    return c, x


# ----------------------------------------------------------------------------------------------- the framework's calls
def _own_rotary(c, x):
    from catch_b200.fusion import qk_norm_rotary

    out = qk_norm_rotary(x["q"], x["k"], x.get("qw"), x.get("kw"), x["cos"], x["sin"], x.get("positions"),
                         interleaved=c["interleaved"])
    if not c["train"]:
        return out
    leaves = [x[n] for n in ("q", "k", "qw", "kw") if n in x]
    return (*(o.detach() for o in out), *torch.autograd.grad(out, leaves, (x["dq"], x["dk"])))


def _own_softmax(c, x):
    from catch_b200.fusion import relative_bias_softmax

    probs = relative_bias_softmax(x["scores"], x["table"], x.get("mask"), scale=0.125, bidirectional=c["bidirectional"],
                                  max_distance=c["max_distance"], query_offset=max(0, c["Lk"] - c["Lq"]))
    if not c["train"]:
        return (probs,)
    return (probs.detach(), *torch.autograd.grad(probs, (x["scores"], x["table"]), x["dprobs"]))


def _own_distill(c, x):
    from catch_b200.fusion import top_logits_distillation

    loss = top_logits_distillation(x["logits"], x["teacher"], x["index"], temperature=c["temperature"], reduction=c["reduction"])
    if not c["train"]:
        return (loss,)
    return (loss.detach(), *torch.autograd.grad(loss, (x["logits"],), x["g"]))


# ------------------------------------------------------------------------------------------------------ the plain forms
def _turn(n, cos, sin, R, interleaved):
    """The first R dimensions of n turned by the angles whose cosines and sines are given."""
    if interleaved:
        a, b = n[..., 0:R:2], n[..., 1:R:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = n[..., : R // 2], n[..., R // 2: R]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, n[..., R:]), -1)


def _plain_head(c, x, name, cos, sin):
    t, w = x[name].float(), x.get(name + "w")
    r = torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6)
    n = t * r
    y = _turn(n if w is None else n * w, cos, sin, c["R"], c["interleaved"]).to(x[name].dtype)
    if not c["train"]:
        return y, None, None
    back = _turn(x["d" + name].float(), cos, -sin, c["R"], c["interleaved"])
    dw = None if w is None else (back * n).sum((0, 1, 2), dtype=torch.float64).float()
    back = back if w is None else back * w
    return y, (r * (back - n * (back * n).mean(-1, keepdim=True))).to(x[name].dtype), dw


def _plain_rotary(c, x):
    at = x["positions"] if "positions" in x else torch.arange(c["L"], device=x["cos"].device)[None]
    cos, sin = x["cos"][at][:, :, None], x["sin"][at][:, :, None]
    (yq, dq, dqw), (yk, dk, dkw) = _plain_head(c, x, "q", cos, sin), _plain_head(c, x, "k", cos, sin)
    if not c["train"]:
        return yq, yk
    return (yq, yk, dq, dk, dqw, dkw) if c["weights"] else (yq, yk, dq, dk)


def _bucket(rel, buckets, max_distance, bidirectional):
    """Distances below half of a side's buckets have one each, farther ones share them by logarithm; in 64 bits, with
    a nudge for the distances that lie on a border exactly."""
    n = buckets // 2 if bidirectional else buckets
    d = rel.abs() if bidirectional else (-rel).clamp(min=0)
    exact = n // 2
    far = torch.log(d.clamp(min=1).double() / exact) / math.log(max_distance / exact) * (n - exact)
    far = (exact + torch.floor(far + 1e-9)).clamp(max=n - 1).long()
    b = torch.where(d < exact, d, far)
    return torch.where(rel > 0, b + n, b) if bidirectional else b


def _plain_softmax(c, x):
    s, table = x["scores"], x["table"]
    B, H, Lq, Lk = s.shape
    rel = torch.arange(Lk, device=s.device)[None] - torch.arange(Lq, device=s.device)[:, None] - max(0, Lk - Lq)
    bucket = _bucket(rel, c["buckets"], c["max_distance"], c["bidirectional"])
    a = s.float() * 0.125 + table[bucket].permute(2, 0, 1)
    mask = x.get("mask")
    if mask is not None:
        a = torch.where(mask, a, -math.inf) if mask.dtype == torch.bool else a + mask.float()
    top = a.amax(-1, keepdim=True)
    e = torch.exp(a - torch.where(top == -math.inf, 0.0, top))
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-30)  # a row with nothing left gives zeros
    if not c["train"]:
        return (p.to(s.dtype),)
    d = x["dprobs"].float()
    d = p * (d - (p * d).sum(-1, keepdim=True))
    # sums over diagonals: with rows in reverse and Lq columns of zeros behind each, a reshape to rows one column shorter
    # puts every diagonal into one column
    lines = torch.nn.functional.pad(d.sum(0, dtype=torch.float64).flip(1), (0, Lq)).reshape(H, -1)
    lines = lines[:, : Lq * (Lk + Lq - 1)].view(H, Lq, Lk + Lq - 1).sum(1)
    first = torch.cat((bucket[1:, 0].flip(0), bucket[0]))  # the bucket of each diagonal
    dt = torch.zeros(table.shape, dtype=torch.float64, device=s.device).index_add_(0, first, lines.t())
    return p.to(s.dtype), (d * 0.125).to(s.dtype), dt.float()


def _plain_distill(c, x):
    z, index, T = x["logits"].float() / c["temperature"], x["index"], c["temperature"]
    valid = index >= 0
    at = index.clamp(min=0)
    t = torch.where(valid, x["teacher"] / T, -math.inf)
    top = t.amax(-1, keepdim=True)
    e = torch.exp(t - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True).clamp(min=1e-30)
    p = e / total
    logp = torch.where(valid, t - top - torch.log(total), 0.0)
    m = z.amax(-1, keepdim=True)
    lse = m + torch.log(torch.exp(z - m).sum(-1, keepdim=True))
    rows = (T * T * (p * (logp - (z.gather(1, at) - lse))).double().sum(-1))
    real = valid.any(-1)
    count = real.sum().clamp(min=1) if c["reduction"] == "mean" else 1
    loss = (rows if c["reduction"] == "none" else rows.sum() / count).float()
    if not c["train"]:
        return (loss,)
    g = torch.where(real, x["g"], 0.0)[:, None] * (T / count)
    d = torch.exp(z - lse) * g
    d.scatter_add_(1, at, -p * g)
    return loss, d.to(x["logits"].dtype)


def run(state):
    c, x = state
    if own:
        return {"rotary": _own_rotary, "softmax": _own_softmax, "distill": _own_distill}[c["op"]](c, x)
    return {"rotary": _plain_rotary, "softmax": _plain_softmax, "distill": _plain_distill}[c["op"]](c, x)


# ---------------------------------------------------------------------------------------- what cannot be done without
def work(case):
    c, e = case, _BYTES[case["dtype"]]
    if c["op"] == "rotary":
        n = c["B"] * c["L"] * (c["Hq"] + c["Hk"]) * c["D"]
        passes = 4 if c["train"] else 2  # x and dy read, y and dx written
        side = c["L"] * c["R"] * 4 + (c["B"] * c["L"] * 8 if c["given"] else 0)
        return {"bytes": passes * n * e + side, "flops": n * (20 if c["train"] else 8)}
    if c["op"] == "softmax":
        n = c["B"] * c["H"] * c["Lq"] * c["Lk"]
        passes = 4 if c["train"] else 2  # scores and their results' gradient read, probabilities and gradient written
        side = {"none": 0, "key": c["B"] * c["Lk"] * 4, "bool": c["B"] * c["Lq"] * c["Lk"], "inf": c["Lq"] * c["Lk"] * e}[c["mask"]]
        return {"bytes": passes * n * e + side + c["buckets"] * c["H"] * 8, "flops": n * (14 if c["train"] else 6)}
    n = c["N"] * c["V"]
    return {"bytes": (2 if c["train"] else 1) * n * e + c["N"] * c["K"] * 12, "flops": n * (7 if c["train"] else 4)}


# ------------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_rotary(c, x):
    """Each pair of dimensions as a complex number, turned by a product with e^(i angle); gradients by automatic
    differentiation."""
    B, L, R = c["B"], c["L"], c["R"]
    if "positions" in x:
        pos = x["positions"]
    else:
        pos = torch.arange(L, device=x["cos"].device).expand(B, L)
    unit = torch.complex(x["cos"].double(), x["sin"].double())[pos].view(B, L, 1, R // 2)
    leaves, outs = [], []
    for name in ("q", "k"):
        t = x[name].double().contiguous().requires_grad_(c["train"])
        w = x[name + "w"].double().requires_grad_(c["train"]) if c["weights"] else None
        n = t / (t.pow(2).sum(-1, keepdim=True) / c["D"] + 1e-6).sqrt()
        if w is not None:
            n = n * w
        head, tail = n[..., :R], n[..., R:]
        pairs = head.unflatten(-1, (R // 2, 2)) if c["interleaved"] else head.unflatten(-1, (2, R // 2)).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
        turned = turned.flatten(-2) if c["interleaved"] else turned.transpose(-1, -2).flatten(-2)
        outs.append(torch.cat((turned, tail), -1))
        leaves.append((t, w))
    if not c["train"]:
        return outs
    wanted = [l[0] for l in leaves] + ([l[1] for l in leaves] if c["weights"] else [])
    grads = torch.autograd.grad(outs, wanted, (x["dq"].double(), x["dk"].double()))
    return [o.detach() for o in outs] + list(grads)


def _exact_softmax(c, x):
    """The bias of every distance from integers alone (a distance passes a border where d^m reaches its product), a
    matrix of those, torch's own softmax where something is left, automatic differentiation."""
    H, Lq, Lk, dev = c["H"], c["Lq"], c["Lk"], x["scores"].device
    n = c["buckets"] // 2 if c["bidirectional"] else c["buckets"]
    exact, far = n // 2, n - n // 2

    def bucket(rel):
        d = abs(rel) if c["bidirectional"] else max(0, -rel)
        up = n if c["bidirectional"] and rel > 0 else 0
        if d < exact:
            return up + d
        passed = [k for k in range(far) if d ** far >= c["max_distance"] ** k * exact ** (far - k)]
        return up + exact + passed[-1]

    offset = max(0, Lk - Lq)
    of = torch.tensor([bucket(max(-4096, min(4096, r))) for r in range(-(Lq - 1) - offset, Lk - offset)], device=dev)
    table = x["table"].double().requires_grad_(c["train"])
    lines = table.t()[:, of]  # [H, Lq + Lk - 1]
    bias = lines.unfold(1, Lk, 1).flip(1)  # row i begins at distance -i - offset
    s = x["scores"].double().requires_grad_(c["train"])
    a = s / 8 + bias
    left = torch.ones((1, 1, 1, 1), dtype=torch.bool, device=dev)
    if c["mask"] == "bool":
        left = x["mask"]
    elif c["mask"] == "inf":
        left = x["mask"] == 0
    elif c["mask"] == "key":
        a = a + x["mask"].double()
    left = left.expand(a.shape[0], 1, Lq, Lk)
    any_left = left.any(-1, keepdim=True)
    p = torch.softmax(a.masked_fill(~left & any_left, -math.inf), -1) * any_left
    if not c["train"]:
        return (p,)
    return (p.detach(), *torch.autograd.grad(p, (s, table), x["dprobs"].double()))


def _exact_distill(c, x):
    """Row by row of the definition: the teacher's distribution spread over the vocabulary, minus the student's."""
    N, V, T = c["N"], c["V"], c["temperature"]
    keep = x["index"] >= 0
    weight = torch.exp((x["teacher"].double() - x["teacher"].double().max()) / T) * keep
    share = weight / weight.sum(1, keepdim=True).clamp(min=1e-300)
    entropy = torch.special.entr(share).sum(1)
    rows = keep.any(1)
    count = max(1, int(rows.sum())) if c["reduction"] == "mean" else 1
    loss, grad, step = [], [], max(1, 60_000_000 // V)
    for lo in range(0, N, step):
        part = slice(lo, min(N, lo + step))
        logq = torch.log_softmax(x["logits"][part].double() / T, 1)
        full = torch.zeros_like(logq).scatter_add_(1, x["index"][part].clamp(min=0), share[part])
        loss.append(T * T * (-entropy[part] - (full * logq).sum(1)) * rows[part])
        if c["train"]:
            g = x["g"].double().expand(N)[part] * rows[part] / count
            grad.append((logq.exp_().sub_(full) * (T * g)[:, None]).to(torch.float32 if N * V > 60_000_000 else torch.float64))
    loss = torch.cat(loss)
    loss = loss if c["reduction"] == "none" else loss.sum() / count
    return (loss, torch.cat(grad)) if c["train"] else (loss,)


def exact(case, seed):
    c, x = prepare(case, seed)
    return {"rotary": _exact_rotary, "softmax": _exact_softmax, "distill": _exact_distill}[c["op"]](c, x)
