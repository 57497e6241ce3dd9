"""graph64's ops and those of a transformer in 64 bits on the host: rotary positions, attention and its gradient, the paged cache."""
import numpy as np

import attention64
import graph64
from vernondsl_amd import graph, kernels


class _One:
    def __init__(self, op, prepare=()):
        self.ops, self.prepare_ops = [op] if op else [], list(prepare)


def _split(x, a):
    h, kv, d = a["heads"], a["kv_heads"], a["dim"]
    return [p.reshape(len(x), -1, d) for p in np.split(x, [h * d, (h + kv) * d], axis=1)]


def _scale(a):
    return a["scale"] if a["scale"] is not None else a["dim"] ** -0.5


def run(g, feeds):
    """{value name: array} after all of g's ops.  Caches are those of the feeds, updated in place."""
    v = graph64.run(_One(None, g.prepare_ops), feeds)
    for n in feeds:
        if "cache" in n:
            v[n] = feeds[n]
    for op in g.ops:
        a, ins = op.attrs, [v[i.name] for i in op.inputs]
        out = [o.name for o in op.outputs]
        if op.kind == "rope":
            x, positions, freqs = ins
            v[out[0]] = attention64.rope(x, positions, 2 * np.pi * freqs.sum(0), a["heads"], a["dim"], a["first"], a["interleaved"], a["inverse"],
                                         a["magnitude"])
        elif op.kind == "attention":
            o, lse, _, _ = attention64.packed(*_split(ins[0], a), ins[1], _scale(a), a["causal"])
            v[out[0]], v[out[1]] = o.reshape(len(o), -1), lse
        elif op.kind == "attention_bwd":
            dout, qkv, starts, o, lse = ins
            parts = _split(qkv, a)
            grads, _ = attention64.packed_grad(*parts, o.reshape(parts[0].shape), lse, dout.reshape(parts[0].shape), starts, _scale(a), a["causal"])
            v[out[0]] = np.concatenate([d.reshape(len(dout), -1) for d in grads], 1)
        elif op.kind == "cache_append":
            qkv, k_cache, v_cache, starts, lengths, table = ins
            _, k, x = _split(qkv, a)
            page = k_cache.shape[2]
            for s, at, m, pos in attention64.cache_positions(starts, lengths, len(qkv)):
                for i in range(m):
                    to = table[s, (pos + i) // page], slice(None), (pos + i) % page
                    k_cache[to], v_cache[to] = k[at + i], x[at + i]
        elif op.kind == "paged_attention":
            qkv, k_cache, v_cache, starts, lengths, table = ins
            o, *_ = attention64.paged(_split(qkv, a)[0], k_cache, v_cache, starts, lengths, table, _scale(a))
            v[out[0]] = o.reshape(len(o), -1)
        else:
            v.update({n: x for n, x in graph64.run(_One(op), {i.name: v[i.name] for i in op.inputs}).items() if n not in feeds})
    return v


def plain_transformer(tokens, seqs, vocab, dim, heads, kv_heads, head_dim, hidden, layers, tied=True, causal=True, **flags):
    """token_transformer_train_graph's forward pass in a graph without its fused forms, and the loss."""
    g = graph.Graph(**flags)
    ids, labels, positions = (g.input(n, (tokens,), "i32") for n in ("ids", "labels", "positions"))
    starts, freqs = g.input("starts", (seqs + 1,), "i32"), g.input("freqs", (2, head_dim // 2), "f32")
    table, h = graph._transformer(g, ids, positions, freqs, vocab, dim, heads, kv_heads, head_dim, hidden, layers,
                                  lambda qkv, k: g.attention(qkv, starts, heads, kv_heads, causal=causal))
    return g, g.linear_cross_entropy(h, table if tied else g.param("W_out", (vocab, dim), "bf16"), labels)


def weights(g, seed):
    """Values of g's params: matrices of unit rows, gains about 1."""
    r = np.random.default_rng(seed)
    made = {o.name for op in g.prepare_ops for o in op.outputs}
    out = {}
    for v in g.values.values():
        if v.kind == "param" and v.name not in made:
            x = r.standard_normal(v.shape) * (v.shape[-1] ** -0.5 if len(v.shape) == 2 else 0.2) + (1.0 if v.name.endswith("gamma") else 0.0)
            out[v.name] = x.astype(np.float32)
    return out


def packed_inputs(r, tokens, lengths, vocab, head_dim, front=0):
    starts = np.concatenate([[front], front + np.cumsum(lengths)]).astype(np.int32)
    positions = np.zeros(tokens, np.int32)
    ids, labels = (np.full(tokens, -1, np.int32) for _ in range(2))
    for a, b in zip(starts[:-1], starts[1:]):
        positions[a:b] = np.arange(b - a) + r.integers(0, 1000)
        ids[a:b], labels[a:b] = r.integers(0, vocab, b - a), r.integers(-1, vocab, b - a)
    return {"ids": ids, "labels": labels, "positions": positions, "starts": starts, "freqs": kernels.rope_frequencies(head_dim)}
