"""Train a small state space byte model on a repeating text, then let it go on.

    python examples/ssm_bytes.py [--steps N]

Runs the state space block's operators together: the scan, the convolution and the
fused norms with their backwards, gradient clipping and AdamW in training; prompts of
different lengths and single rows on carried states in serving.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from asca_amd.ssm import SsmModel  # noqa: E402

TEXT = b"a constant state carries the whole past; "


def batches(rng, batch: int, seq: int):
    text = np.frombuffer(TEXT * (seq // len(TEXT) + 3), np.uint8)
    while True:
        at = rng.integers(0, len(TEXT), batch)
        rows = np.stack([text[a:a + seq + 1] for a in at])
        yield rows[:, :-1].reshape(-1), rows[:, 1:].reshape(-1)


def main(steps: int = 200, batch: int = 16, seq: int = 96) -> tuple[list[float], bytes]:
    m = SsmModel(vocab=256, d=128, n_layers=2)
    m.set_params(m.init(0))
    losses = []
    for k, (ids, tgt) in zip(range(steps), batches(np.random.default_rng(1), batch, seq)):
        losses.append(m.forward_backward(ids, tgt, batch))
        norm, factor = m.clip(1.0)
        m.adamw(lr=3e-3)
        if k % 20 == 0 or k == steps - 1:
            print(f"step {k:4d}  loss {losses[-1]:.4f}  gradient norm {norm:.3f} scaled by {factor:.3f}", flush=True)
    # two prompts of different lengths, then one byte at a time
    prompts = [TEXT[:20], TEXT[:33]]
    ids = np.zeros((2, 33), np.uint8)
    for row, p in zip(ids, prompts):
        row[:len(p)] = np.frombuffer(p, np.uint8)
    st = m.new_state(2)
    nxt = m.prompt(ids, st, [len(p) for p in prompts]).argmax(1)
    out = [bytearray(p) for p in prompts]
    for _ in range(60):
        for o, b in zip(out, nxt):
            o.append(int(b))
        nxt = m.step(nxt, st).argmax(1)
    for o in out:
        print(bytes(o).decode("latin1"), flush=True)
    m.close()
    return losses, [bytes(o) for o in out]


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=200)
    main(ap.parse_args().steps)
