"""Trains a projection of noisy features and searches its rows.

Features carry their class in a few hidden directions, under noise that
dominates plain distances. A two-layer projection is trained by the softmax
over inner products with one row per class -- ``linear``, ``softmax_xent`` and
their gradients, bf16 operands with fp32 master weights -- and the KNN graph of
the projected rows (``brute_force_knn_device``) then links rows of one class.

    python examples/train_search_rows.py --rows 20000 --steps 60
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch

import knng_gpu_b200 as kg


def make_features(rows, width, classes, seed):
    """Rows = class centre in 16 hidden directions + strong noise in all others."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    labels = torch.randint(0, classes, (rows,), generator=gen, device="cuda")
    centres = torch.randn((classes, 16), generator=gen, device="cuda")
    noise = torch.randn((rows, width - 16), generator=gen, device="cuda") * 2.0
    hidden = centres[labels] + 0.2 * torch.randn((rows, 16), generator=gen, device="cuda")
    turn = torch.linalg.qr(torch.randn((width, width), generator=gen, device="cuda")).Q
    return (torch.cat([hidden, noise], 1) @ turn).contiguous(), labels


def same_class_share(rows, labels, k):
    """Share of the KNN graph's edges that stay within a class."""
    ids, _, _ = kg.brute_force_knn_device(rows.contiguous(), k, kg.L2Squared())
    return float((labels[ids.long()] == labels[:, None]).float().mean())


def run(rows=20000, width=128, hidden=256, out=64, classes=500, batch=4096, steps=60, rate=6e-3, scale=4.0, k=10,
        seed=0, report=print):
    features, labels = make_features(rows, width, classes, seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed + 1)

    def matrix(r, c):
        return torch.randn((r, c), generator=gen, device="cuda") * c ** -0.5

    # fp32 master weights, updated by Adam; the operators read bf16 copies.
    master = {"w1": matrix(hidden, width), "b1": torch.zeros(hidden, device="cuda"),
              "w2": matrix(out, hidden), "classes": 0.5 * matrix(classes, out)}
    first = {n: torch.zeros_like(t) for n, t in master.items()}
    second = {n: torch.zeros_like(t) for n, t in master.items()}
    x16 = features.bfloat16()
    before = same_class_share(features, labels, k)
    losses = []
    for step in range(steps):
        pick = torch.randint(0, rows, (batch,), generator=gen, device="cuda")
        x, y = x16[pick], labels[pick]
        p = {n: t.bfloat16() for n, t in master.items()}
        h, pre = kg.linear(x, p["w1"], p["b1"], activation="gelu", save_pre=True)
        z = kg.linear(h, p["w2"])
        loss, lse = kg.softmax_xent(z, p["classes"], y, scale=scale)
        dloss = torch.full((batch,), 1.0 / batch, device="cuda")
        dz, dclasses = kg.softmax_xent_backward(dloss, z, p["classes"], y, lse, scale=scale)
        dh, dw2, _ = kg.linear_backward(dz, h, p["w2"])
        _, dw1, db1 = kg.linear_backward(dh, x, p["w1"], pre=pre, activation="gelu", need_dx=False, need_db=True)
        for name, grad in (("w1", dw1), ("b1", db1), ("w2", dw2), ("classes", dclasses)):
            g = grad.float()
            first[name].mul_(0.9).add_(g, alpha=0.1)
            second[name].mul_(0.99).addcmul_(g, g, value=0.01)
            m = first[name] / (1 - 0.9 ** (step + 1))
            v = second[name] / (1 - 0.99 ** (step + 1))
            master[name] -= rate * m / (v.sqrt() + 1e-8)
        losses.append(loss.mean())
        if step % 20 == 19:
            report(f"step {step + 1}: loss {float(losses[-1]):.3f}")
    p = {n: t.bfloat16() for n, t in master.items()}
    h = kg.linear(x16, p["w1"], p["b1"], activation="gelu")
    searched = kg.linear(h, p["w2"], out_dtype=torch.float32)
    after = same_class_share(searched, labels, k)
    report(f"neighbours of the same class: features {before:.3f}, projected rows {after:.3f}")
    return {"before": before, "after": after, "first_loss": float(losses[0]), "last_loss": float(losses[-1])}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--rows", type=int, default=20000)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--classes", type=int, default=500)
    a = ap.parse_args()
    run(rows=a.rows, steps=a.steps, classes=a.classes)
