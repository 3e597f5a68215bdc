"""Train a byte model, let a narrower one learn from its largest logits, and search for the
student's best continuations.

    python examples/distill_bytes.py [--steps N]

Runs the operators behind the logits together: the teacher's largest logits of each row, the
distilled loss with its gradient in the student's training, and a beam search over the
student's carried states.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from asca_amd.ssm import SsmModel  # noqa: E402
from examples.ssm_bytes import TEXT, batches  # noqa: E402


def main(steps: int = 150, batch: int = 16, seq: int = 96) -> tuple[list[float], list[bytes]]:
    big, small = SsmModel(vocab=256, d=128, n_layers=2), SsmModel(vocab=256, d=64, n_layers=1)
    for m in (big, small):
        m.set_params(m.init(0))
    for _, (ids, tgt) in zip(range(steps), batches(np.random.default_rng(1), batch, seq)):
        big.forward_backward(ids, tgt, batch)
        big.clip(1.0)
        big.adamw(lr=3e-3)
    losses = []
    for k, (ids, tgt) in zip(range(steps), batches(np.random.default_rng(2), batch, seq)):
        t = big.teacher(ids, batch, 16, temperature=2.0)
        losses.append(small.forward_backward(ids, tgt, batch, t, alpha=0.7))
        t.free()
        small.clip(1.0)
        small.adamw(lr=3e-3)
        if k % 20 == 0 or k == steps - 1:
            print(f"step {k:4d}  distilled loss {losses[-1]:.4f}", flush=True)
    prompts = np.stack([np.frombuffer(TEXT[a:a + 20], np.uint8) for a in (0, 7)])
    found, scores = small.beam_search(prompts, beams=4, steps=30)
    for p, rows, sc in zip(prompts, found, scores):
        for r, x in zip(rows, sc):
            print(f"{x:8.3f}  {bytes(p).decode()}|{bytes(r.astype(np.uint8)).decode('latin1')}", flush=True)
    out = [bytes(p) + bytes(r[0].astype(np.uint8)) for p, r in zip(prompts, found)]
    for m in (big, small):
        m.close()
    return losses, out


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=150)
    main(ap.parse_args().steps)
