"""An additive model over binned features, trained by gradients beside a boosted one.

    python examples/additive_student.py

1. A table's columns are cut into bins (``select_borders``, ``quantize``), as for a boosted model.
2. The student holds a row of class scores for every (feature, bin); a table row's scores are the sum of its
   bins' (``lookup_rows``).
3. It is trained on the labels: their log probability and the entropy (``class_logprobs``), the
   gradient by the scores (``logprob_gradients``), that by the held rows (``lookup_gradients``) and a
   step with states in 8 bits (``AdamW``).

torch is imported first: one HIP runtime serves the process.
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import catboost_rs_amd as cb  # noqa: E402
from examples.distill_classes import table  # noqa: E402


def binned(x, border_count=32):
    """Indices [rows][features] i32 of every value's (feature, bin), and how many there are."""
    borders = cb.select_borders(x, border_count)
    sizes = [len(b) + 1 for b in borders]
    starts = np.concatenate([[0], np.cumsum(sizes)])
    bins = [cb.quantize(column, b).astype(np.int32) + int(start) for column, b, start in zip(x, borders, starts)]
    return np.stack(bins, 1), int(starts[-1])


def loss_and_gradient(held, index, label, entropy_weight=0.01):
    """Mean of -log p(label) - entropy_weight * entropy over the rows, and its gradient by the held rows."""
    scores = cb.lookup_rows(held, index)
    got = cb.class_logprobs(scores, label)
    rows = len(label)
    g = torch.full_like(got.logprob, -1.0 / rows)
    h = torch.full_like(got.entropy, -entropy_weight / rows)
    grad = cb.logprob_gradients(scores, label, g, got.stats, entropy_grad=h)
    loss = -(got.logprob.mean() + entropy_weight * got.entropy.mean())
    return loss, cb.lookup_gradients(grad, index, held.shape[0])


def main(rows=20_000, features=12, classes=10, steps=60):
    x, y = table(rows, features, classes)
    index, entries = binned(x)
    index = torch.from_numpy(index).cuda()
    label = torch.from_numpy(y.astype(np.int32)).cuda()
    held = torch.zeros(entries, classes, device="cuda")
    optimizer = cb.AdamW([held], lr=0.05, weight_decay=0.0, state="f8")
    losses = []
    for _ in range(steps):
        loss, grad = loss_and_gradient(held, index, label)
        optimizer.step([grad])
        losses.append(loss)
    losses = torch.stack(losses).tolist()
    top = cb.class_logprobs(cb.lookup_rows(held, index), label, k=1)
    right = (top.top_index[:, 0] == label).float().mean().item()
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}; the label is the most probable class on {right:.1%} of the rows; "
          f"mean entropy {top.entropy.mean().item():.3f}")
    return losses, held


if __name__ == "__main__":
    main()
