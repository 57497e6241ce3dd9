"""A small model of tokens trained on the HIP device:  python -m vernondsl_amd.examples.token_model

Characters of this file are the tokens; the model predicts each one from the one before it: embedding,
residual MLP blocks with layer norm, and the output layer with its cross entropy (tied to the embedding),
forward and backward recorded once and replayed as one hipGraph.  The weights live on the host in f32,
take a step of gradient descent with momentum there, and are written back in bf16.
"""
from __future__ import annotations

import argparse
import json

import numpy as np

from vernondsl_amd import graph, rng
from vernondsl_amd.rhi import Device, Queue


def text_tokens():
    """This file's characters as ids, and how many there are of each kind."""
    with open(__file__, "rb") as f:
        data = np.frombuffer(f.read(), np.uint8)
    kinds, ids = np.unique(data, return_inverse=True)
    return ids.astype(np.int32), len(kinds)


def initial(name, shape):
    """Xavier-normal matrices, a smaller embedding, norms of gain 1 and offset 0."""
    if len(shape) == 1:
        return np.full(shape, 1.0 if name.endswith("gamma") else 0.0, np.float32)
    std = 0.02 if name == "E" else np.sqrt(2.0 / sum(shape))
    seed = sum(ord(c) << (k % 16) for k, c in enumerate(name))
    return rng.normal(seed, shape[0] * shape[1], 0.0, std).reshape(shape).astype(np.float32)


def train(steps=60, tokens=512, dim=128, hidden=512, layers=2, rate=0.3, momentum=0.9):
    """Trains for `steps` steps and returns the loss of each."""
    ids, vocab = text_tokens()
    g, grads = graph.token_mlp_train_graph(tokens, vocab, dim, hidden, layers)
    dev = Device(0)
    q = Queue(dev)
    exe = g.compile(dev)
    weights = {n: initial(n, g.values[n].shape) for n in grads}
    speed = {n: np.zeros_like(w) for n, w in weights.items()}

    def write(n):
        exe.write(q, n, rng.f32_to_bf16(weights[n]) if g.values[n].dtype == "bf16" else weights[n])

    for n in weights:
        write(n)
    step, losses = None, []
    for k in range(steps):
        at = (np.arange(tokens) + k * tokens) % (len(ids) - 1)
        exe.write(q, "ids", ids[at])
        exe.write(q, "labels", ids[at + 1])
        if step is None:
            step = exe.capture(q)
        step.launch(q)
        losses.append(float(exe.read(q, "loss")[0]))
        for n, d in grads.items():
            speed[n] = momentum * speed[n] + exe.read(q, d.name)
            weights[n] -= rate * (1.0 - momentum) * speed[n]
            write(n)
    step.destroy()
    exe.free()
    q.destroy()
    dev.close()
    return losses


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=60)
    losses = train(ap.parse_args(argv).steps)
    print(json.dumps({"steps": len(losses), "first_loss": losses[0], "last_loss": losses[-1]}), flush=True)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
