"""Device time of the transformer operators (queries / keys with norm and rotation, softmax with a relative position
bias, distillation against a teacher's top logits), forward and backward, at fixed sizes.

    python benchmarks/transformer_ops.py [--only rotary|softmax|distill]

Inputs alternate between three sets, so that those beyond 40 MB are not in L2 when they are read again.  Bytes are what a
direction has to move: each tensor it reads and writes once; the rate is set against the copy bandwidth of 6566 GB/s.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import catch_b200  # noqa: F401,E402

DEV, COPY = "blackwell", 6565.8
bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
OPS = torch.ops.catch_b200


def timed(fn, sets, iters):
    for s in sets:
        fn(*s)
    torch.b200.synchronize()
    begin, end = (torch.b200.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for i in range(iters):
        fn(*sets[i % len(sets)])
    end.record()
    torch.b200.synchronize()
    return begin.elapsed_time(end) / iters * 1e3


def report(name, us, bytes_):
    rate = bytes_ / us / 1e3
    print(f"{name:64s} {us:9.1f} us {rate:7.0f} GB/s  {rate / COPY:.2f} of copy", flush=True)


def rotary(iters):
    for B, L, Hq, Hk, D, R, dt, inter in ((8, 2048, 32, 8, 128, 128, bf16, False), (256, 128, 12, 12, 64, 64, bf16, False),
                                          (8, 2048, 16, 16, 64, 64, f32, False), (24, 1021, 10, 5, 80, 32, f16, True)):
        cos, sin, w = torch.randn(2048, R // 2).to(DEV), torch.randn(2048, R // 2).to(DEV), torch.ones(D).to(DEV)
        sets = []
        for _ in range(3):
            x = torch.randn(B, L, Hq + 2 * Hk, D).to(dt).to(DEV)
            sets.append((x[:, :, :Hq], x[:, :, Hq:Hq + Hk], torch.randn(B, L, Hq, D).to(dt).to(DEV), torch.randn(B, L, Hk, D).to(dt).to(DEV)))
        n = B * L * (Hq + Hk) * D * dt.itemsize
        name = f"rotary {B}x{L} heads {Hq}+{Hk} of {D} rotated {R} {str(dt)[6:]}"
        report(name + " forward", timed(lambda q, k, *_: OPS.qk_norm_rotary(q, k, w, w, cos, sin, None, 1e-6, inter), sets, iters), 2 * n)
        report(name + " backward", timed(lambda q, k, gq, gk: OPS.qk_norm_rotary_backward(gq, gk, q, k, w, w, cos, sin, None, 1e-6, inter),
                                         sets, iters), 3 * n)


def softmax(iters):
    for B, H, Lq, Lk, dt, mask in ((2, 12, 2048, 2048, bf16, None), (2, 12, 2048, 2048, bf16, "causal"), (128, 12, 128, 128, bf16, "padding"),
                                   (16, 12, 512, 512, bf16, None), (12, 7, 389, 517, f32, "random"),
                                   (1, 12, 1024, 8192, bf16, None), (1, 12, 1024, 16384, bf16, None), (1, 12, 1024, 8192, f32, None)):
        m = None
        if mask == "causal":
            m = torch.zeros(Lq, Lk).masked_fill(torch.arange(Lk) > torch.arange(Lq)[:, None], -float("inf")).to(dt).view(1, 1, Lq, Lk).to(DEV)
        elif mask == "padding":
            m = torch.where(torch.arange(Lk) < Lk - 28, 0.0, -10000.0).expand(B, 1, 1, Lk).contiguous().to(DEV)
        elif mask == "random":
            m = (torch.rand(B, 1, Lq, Lk) < 0.8).to(DEV)
        table = torch.randn(32, H).to(DEV)
        sets = []
        for _ in range(3):
            s = torch.randn(B, H, Lq, Lk).to(dt).to(DEV)
            sets.append((s, torch.randn(B, H, Lq, Lk).to(dt).to(DEV), OPS.relative_bias_softmax(s, table, m, 0.125, True, 128, 0)[1]))
        n = B * H * Lq * Lk * dt.itemsize
        name = f"softmax {B}x{H}x{Lq}x{Lk} {str(dt)[6:]} mask {mask}"
        report(name + " forward", timed(lambda s, *_: OPS.relative_bias_softmax(s, table, m, 0.125, True, 128, 0), sets, iters), 2 * n)
        for need, what in ((False, " backward, scores"), (True, " backward, scores and table")):
            report(name + what, timed(lambda s, g, st: OPS.relative_bias_softmax_backward(g, s, st, table, m, 0.125, True, 128, 0, need),
                                      sets, iters), 3 * n)


def distill(iters):
    from catch_b200.fusion import top_logits_distillation

    for N, V, K, dt, absent in ((4096, 30522, 64, bf16, 0.0), (4096, 131072, 128, bf16, 0.0), (777, 50021, 37, f32, 0.0), (8192, 1000, 5, bf16, 0.0),
                                (4096, 30522, 64, bf16, 0.85), (16384, 4000, 128, bf16, 0.85)):
        index = (torch.randint(0, V, (N, 1)) + torch.arange(K) * (V // K)) % V
        index[torch.rand(N) < absent] = -1
        teacher, index = torch.randn(N, K).to(DEV), index.to(DEV)
        sets = [(torch.randn(N, V).to(dt).to(DEV),) for _ in range(2)]
        grad = [(z.clone().requires_grad_(),) for (z,) in sets]
        n = N * V * dt.itemsize
        name = f"distill {N}x{V} kept {K} {str(dt)[6:]}" + (f" {absent:.0%} of the rows empty" if absent else "")
        loss = lambda z, early=True: top_logits_distillation(z, teacher, index, temperature=2.0, early_gradient=early)  # noqa: E731
        report(name + " loss", timed(loss, sets, iters), n)
        report(name + " loss and gradient", timed(loss, grad, iters), 2 * n)
        one = torch.ones(()).to(DEV)
        report(name + " with backward(), factor 1", timed(lambda z: torch.autograd.grad(loss(z), (z,), one), grad, iters), 2 * n)
        half = 0.5 * one
        report(name + " with backward(), factor 0.5", timed(lambda z: torch.autograd.grad(loss(z), (z,), half), grad, iters), 2 * n)
        report(name + " the same, early_gradient=False", timed(lambda z: torch.autograd.grad(loss(z, False), (z,), half), grad, iters), 2 * n)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--only", choices=("rotary", "softmax", "distill"))
    ap.add_argument("--iters", type=int, default=20)
    a = ap.parse_args()
    for fn in (rotary, softmax, distill):
        if a.only in (None, fn.__name__):
            fn(a.iters)
