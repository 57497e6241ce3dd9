"""A transformer's training step, and the serving of it, on the device (embedding, norms, rotary positions, attention, MLPs, cross
entropy; captured graphs) against the same in 64 bits with the graphs' bf16 roundings left out.

A rounding moves a tensor by at most 2^-8 of its norm.  Forward, a value passes in each layer those of the norm, the
projection, the rotation, the weights and the output of the attention, the norm and the activation: 7, and the last norm's.
Backward, besides, the gradients that each product takes: into the two MLP layers and through GELU', the attention's dout and
ds and weights, the projection's, the output's: 8 a layer, and G.  As if they all pointed one way: (7 layers + 1) 2^-8 of the logits,
(15 layers + 3) 2^-8 of a gradient."""
import numpy as np
import pytest

import attention_graph64 as ag
from vernondsl_amd import graph, kernels, rng
from vernondsl_amd.examples import token_attention

pytestmark = pytest.mark.gpu


def write_weights(exe, q, g, w):
    """Writes w rounded to the params' types, and returns what they then are."""
    out = {}
    for n, x in w.items():
        bf16 = g.values[n].dtype == "bf16"
        exe.write(q, n, rng.f32_to_bf16(x) if bf16 else x)
        out[n] = rng.bf16_to_f32(rng.f32_to_bf16(x)) if bf16 else x
    return out


# whole packed tiles; ragged rows in front of, between and behind ragged sequences, an odd group; heads of an odd size, untied
@pytest.mark.parametrize("tokens,lengths,front,model,layers,tied", [
    (256, [256], 0, dict(vocab=512, dim=256, heads=4, kv_heads=2, head_dim=64, hidden=512), 1, True),
    (300, [100, 0, 1, 130, 40], 9, dict(vocab=300, dim=64, heads=6, kv_heads=2, head_dim=32, hidden=128), 2, True),
    (77, [40, 37], 0, dict(vocab=77, dim=96, heads=3, kv_heads=3, head_dim=40, hidden=160), 2, False)])
def test_training_step_matches_64_bits(dev, q, tokens, lengths, front, model, layers, tied):
    g, grads = graph.token_transformer_train_graph(tokens, len(lengths), layers=layers, tied=tied, **model)
    plain, loss = ag.plain_transformer(tokens, len(lengths), layers=layers, tied=tied, **model)
    plain_grads = plain.backward(loss)
    feeds = ag.packed_inputs(np.random.default_rng(tokens), tokens, lengths, model["vocab"], model["head_dim"], front)
    exe = g.compile(dev)
    w = write_weights(exe, q, g, ag.weights(plain, 11))
    for n, x in feeds.items():
        exe.write(q, n, x)
    exe.run(q)
    names = ["loss"] + [d.name for d in grads.values()]
    eager = {n: exe.read(q, n) for n in names}
    want = ag.run(plain, {**w, **feeds})
    rel = (15 * layers + 3) * 2.0 ** -8
    assert abs(float(eager["loss"][0]) - want[loss.name][0]) <= rel * abs(want[loss.name][0])
    for n, d in grads.items():
        x = want[plain_grads[n].name]
        assert np.linalg.norm(eager[d.name].astype(np.float64) - x) <= rel * np.linalg.norm(x), n
    step = exe.capture(q)
    for k in range(3):
        for n in names:
            exe.t[n].buffer.fill_u32(q, 0x7FC07FC0)
        q.sync()
        step.launch(q)
        q.sync()
        for n in names:
            assert np.array_equal(exe.read(q, n), eager[n]), f"replay differs from the eager run in {n}"
    # another packing of the same rows, through the same recording: what the eager run of it gives
    other = ag.packed_inputs(np.random.default_rng(1), tokens, [0] * (len(lengths) - 1) + [tokens - 3], model["vocab"], model["head_dim"])
    for n, x in other.items():
        exe.write(q, n, x)
    exe.run(q)
    eager = {n: exe.read(q, n) for n in names}
    step.launch(q)
    q.sync()
    for n in names:
        assert np.array_equal(exe.read(q, n), eager[n])
    step.destroy()
    exe.free()


def test_serving_matches_64_bits(dev, q):
    """Three texts in chunks and single tokens side by side, each step one replay: every token's logits against the whole forward
    pass of its text."""
    model = dict(dim=128, heads=8, kv_heads=2, head_dim=64, hidden=256, layers=2)
    vocab, texts = 100, [np.random.default_rng(s).integers(0, 100, n).astype(np.int32) for s, n in enumerate((60, 33, 5))]
    tokens = sum(map(len, texts))
    plain, loss = ag.plain_transformer(tokens, 3, vocab, **model)
    w = ag.weights(plain, 4)
    server = token_attention.Server(dev, q, w, vocab, rows=24, seqs=3, page=16, pages=9, pages_per_seq=4, model=model)
    w = {n: rng.bf16_to_f32(rng.f32_to_bf16(x)) if plain.values[n].dtype == "bf16" else x for n, x in w.items()}
    starts = np.concatenate([[0], np.cumsum([len(t) for t in texts])]).astype(np.int32)
    feeds = {"ids": np.concatenate(texts), "labels": np.zeros(tokens, np.int32), "starts": starts, "freqs": kernels.rope_frequencies(64),
             "positions": np.concatenate([np.arange(len(t)) for t in texts]).astype(np.int32)}
    v = ag.run(plain, {**w, **feeds})
    want = v[loss.producer.inputs[0].name] @ w["E"].astype(np.float64).T
    rel = (7 * model["layers"] + 1) * 2.0 ** -8
    done, plan = [0, 0, 0], [[20, 1, 0], [1, 20, 2], [18, 5, 1], [1, 1, 1], [12, 6, 1], [0, 0, 0], [8, 0, 0]]
    for counts in plan:
        new = {s: texts[s][done[s]:done[s] + n] for s, n in enumerate(counts) if n}
        for s, logits in server.step(new).items():
            done[s] += counts[s]
            x = want[starts[s] + done[s] - 1]
            assert np.linalg.norm(logits - x) <= rel * np.linalg.norm(x), (counts, s)
    assert done == [60, 33, 5]
    server.close()


def test_example_runs(dev, q):
    weights, losses = token_attention.train(dev, q, steps=3)
    assert len(losses) == 3 and np.all(np.isfinite(losses)) and all(np.all(np.isfinite(w)) for w in weights.values())
    ids, kinds = token_attention.text_tokens()
    server = token_attention.Server(dev, q, weights, len(kinds))
    prompts = [ids[:40], ids[100:103]]
    together = token_attention.answer(server, prompts, 6)
    server.close()
    assert [len(a) for a in together] == [6, 6] and all(0 <= t < len(kinds) for a in together for t in a)
