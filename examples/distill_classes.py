"""A boosted model teaches a linear one, which then answers by drawing classes.

    python examples/distill_classes.py

1. A MultiClass model is trained on a generated table (``Trainer``) and applied to it
   (``apply_oblivious``): raw scores [classes][rows].
2. ``top_classes`` keeps the teacher's k largest scores of every row and its log-sum-exp: what a
   student needs, in a fraction of the memory of the scores.
3. A linear student in torch is trained on ``distill_gradients`` alone; it never sees a label.
4. ``sample_classes`` draws an answer of the student for every row, within a nucleus.

torch is imported first: one HIP runtime serves the process.
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import catboost_rs_amd as cb  # noqa: E402


def table(rows, features, classes, seed=0):
    """Normal features, and a class drawn by a linear score of them."""
    g = np.random.default_rng(seed)
    x = g.standard_normal((features, rows)).astype(np.float32)
    score = g.standard_normal((classes, features)).astype(np.float32) @ x
    return x, np.argmax(score + g.gumbel(size=score.shape), 0).astype(np.float64)


def teacher_scores(x, y, classes, trees=40, depth=5):
    """Raw scores [classes][rows] of a boosted model trained on the table."""
    borders = cb.select_borders(x, 32)
    tr = cb.Trainer.from_floats(x, borders, y, loss="MultiClass", leaf_method="Newton", approx_dim=classes, depth=depth,
                                learning_rate=0.3)
    try:
        splits, leaves = tr.fit(trees)
    finally:
        tr.close()
    split_borders = [borders[f][b] for tree in splits for f, b in tree]
    return cb.apply_oblivious(x, splits[:, :, 0].ravel(), split_borders, np.arange(trees + 1) * depth,
                              leaves.transpose(0, 2, 1).ravel() * 1.0, np.arange(trees + 1) << depth, approx_dim=classes)


def main(rows=20_000, features=12, classes=10, k=3, temperature=2.0, steps=60):
    x, y = table(rows, features, classes)
    raw = teacher_scores(x, y, classes)
    teacher = torch.from_numpy(raw.astype(np.float32)).cuda().t()      # [rows][classes] over [classes][rows]
    values, index, lse = cb.top_classes(teacher, k, temperature=temperature)

    inputs = torch.from_numpy(x).cuda()
    weight = torch.zeros(classes, features, device="cuda")
    losses = []
    for _ in range(steps):
        scores = (weight @ inputs).t()                                  # class-major, as the teacher's
        loss, grad = cb.distill_gradients(scores, values, index, top_lse=lse, temperature=temperature)
        weight -= (2.0 / rows) * (grad.t() @ inputs.t())
        losses.append(loss.mean())
    losses = torch.stack(losses).tolist()

    scores = (weight @ inputs).t()
    uniform = torch.rand(rows, device="cuda", dtype=torch.float64)
    drawn, logprob = cb.sample_classes(scores, uniform, top_p=0.9)
    best, _ = cb.sample_classes(scores, uniform, temperature=0.0)
    agree = (best == index[:, 0]).float().mean().item()
    print(f"distillation loss {losses[0]:.4f} -> {losses[-1]:.4f}; the student's first class is the teacher's on "
          f"{agree:.1%} of the rows; mean log probability of a drawn class {logprob.mean().item():.3f}")
    return losses, agree, drawn


if __name__ == "__main__":
    main()
