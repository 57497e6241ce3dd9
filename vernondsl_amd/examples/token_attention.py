"""A small model of tokens that see each other, trained and then served on the HIP device:
python -m vernondsl_amd.examples.token_attention

Characters of this file are the tokens.  Training: packed sequences of the text, each token predicting the next one, attention
with rotary positions before every MLP, forward and backward one hipGraph (token_transformer_train_graph).  Serving: prompts
that arrive together are continued token by token over a paged cache (token_transformer_serve_graph): each step takes a chunk
of one prompt beside the next tokens of the others, and is one hipGraph too.
"""
from __future__ import annotations

import argparse
import json

import numpy as np

from vernondsl_amd import graph, kernels, rng
from vernondsl_amd.examples.token_model import initial
from vernondsl_amd.rhi import Device, Queue

MODEL = dict(dim=128, heads=4, kv_heads=2, head_dim=32, hidden=256, layers=2)


def text_tokens():
    """This file's characters as ids, and their kinds."""
    with open(__file__, "rb") as f:
        data = np.frombuffer(f.read(), np.uint8)
    kinds, ids = np.unique(data, return_inverse=True)
    return ids.astype(np.int32), kinds


def train(dev, q, steps=60, seqs=4, length=128, rate=0.3, momentum=0.9):
    """Trains for `steps` steps; returns the weights (f32, on the host) and the loss of each step."""
    ids, kinds = text_tokens()
    tokens = seqs * length
    g, grads = graph.token_transformer_train_graph(tokens, seqs, len(kinds), **MODEL)
    exe = g.compile(dev)
    weights = {n: initial(n, g.values[n].shape) for n in grads}
    speed = {n: np.zeros_like(w) for n, w in weights.items()}

    def write(n):
        exe.write(q, n, rng.f32_to_bf16(weights[n]) if g.values[n].dtype == "bf16" else weights[n])

    for n in weights:
        write(n)
    exe.write(q, "freqs", kernels.rope_frequencies(MODEL["head_dim"]))
    exe.write(q, "starts", np.arange(seqs + 1, dtype=np.int32) * length)
    exe.write(q, "positions", np.tile(np.arange(length, dtype=np.int32), seqs))
    step, losses = None, []
    for k in range(steps):
        first = rng.uniform(k, seqs) * (len(ids) - length - 1)
        at = (first.astype(np.int64)[:, None] + np.arange(length)).reshape(-1)
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
    return weights, losses


class Server:
    """Serves up to `seqs` sequences from a pool of pages, `rows` new tokens a step."""

    def __init__(self, dev, q, weights, vocab, rows=16, seqs=4, page=16, pages=40, pages_per_seq=16, model=None):
        self.q, self.rows, self.seqs, self.page = q, rows, seqs, page
        model = model or MODEL
        g = graph.token_transformer_serve_graph(rows, seqs, pages, page, pages_per_seq, vocab, **model)
        self.exe = g.compile(dev)
        for n, w in weights.items():
            self.exe.write(q, n, rng.f32_to_bf16(w) if g.values[n].dtype == "bf16" else w)
        self.exe.write(q, "freqs", kernels.rope_frequencies(model["head_dim"]))
        self.free = list(range(pages))
        self.table = np.full((seqs, pages_per_seq), -1, np.int32)
        self.lengths = np.zeros(seqs, np.int32)
        self.graph = None

    def step(self, new):
        """new: {sequence: its next tokens}, `rows` of them at most.  Returns {sequence: the logits of its last one}."""
        ids, positions = np.full(self.rows, -1, np.int32), np.zeros(self.rows, np.int32)
        starts, last = np.zeros(self.seqs + 1, np.int32), {}
        at = 0
        for s in range(self.seqs):
            tokens = new.get(s, [])
            ids[at:at + len(tokens)] = tokens
            positions[at:at + len(tokens)] = self.lengths[s] + np.arange(len(tokens))
            self.lengths[s] += len(tokens)
            while np.count_nonzero(self.table[s] >= 0) * self.page < self.lengths[s]:
                self.table[s, np.count_nonzero(self.table[s] >= 0)] = self.free.pop()
            at += len(tokens)
            starts[s + 1] = at
            if len(tokens):
                last[s] = at - 1
        for name, x in (("ids", ids), ("positions", positions), ("starts", starts), ("lengths", self.lengths), ("table", self.table)):
            self.exe.write(self.q, name, x)
        if self.graph is None:
            self.graph = self.exe.capture(self.q)
        self.graph.launch(self.q)
        logits = self.exe.read(self.q, "logits")
        return {s: logits[r] for s, r in last.items()}

    def close(self):
        if self.graph is not None:
            self.graph.destroy()
        self.exe.free()


def answer(server, prompts, count):
    """The `count` likeliest next tokens of each prompt, one after the other: prompts are taken in chunks beside the others' tokens."""
    todo = {s: list(p) for s, p in enumerate(prompts)}
    out = {s: [] for s in todo}
    while any(len(o) < count for o in out.values()):
        new, room = {}, server.rows
        for s in sorted(todo, key=lambda s: len(todo[s])):  # single tokens first
            take = todo[s][:room] if len(out[s]) < count else []
            if take:
                new[s], room = take, room - len(take)
        for s, logits in server.step(new).items():
            todo[s] = todo[s][len(new[s]):]
            if not todo[s]:
                out[s].append(int(np.argmax(logits)))
                todo[s] = [out[s][-1]]
    return [out[s] for s in sorted(out)]


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--tokens", type=int, default=24)
    a = ap.parse_args(argv)
    dev = Device(0)
    q = Queue(dev)
    weights, losses = train(dev, q, a.steps)
    ids, kinds = text_tokens()
    server = Server(dev, q, weights, len(kinds))
    prompts = [ids[k:k + n] for k, n in ((0, 40), (300, 5), (700, 19))]
    answers = answer(server, prompts, a.tokens)
    server.close()
    q.destroy()
    dev.close()
    text = ["".join(chr(kinds[t]) for t in [*p, *x]) for p, x in zip(prompts, answers)]
    print(json.dumps({"steps": len(losses), "first_loss": losses[0], "last_loss": losses[-1], "texts": text}), flush=True)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
