"""Graphs that reach a param through every operand that has a gradient (position tables, computed and shared output
weights, factorised tables, frozen and untied tables, norms without offset), on the device against 64 bits without the
graph's bf16 roundings.

No gradient passes more than 12 tensors that are rounded to bf16, each of which moves by at most 2^-8 of its norm: 12 * 2^-8
in norm if they all pointed one way."""
import numpy as np
import pytest

import graph64
from vernondsl_amd import rng

pytestmark = pytest.mark.gpu
REL = 12 * 2.0 ** -8
FLAGS = {**graph64.FLAGS, "fused": dict(prepare_transposes=True, fuse_gelu_backward=True, pack_weights=True, fuse_mse=True,
                                        store_gelu_deriv=True, k_major_grads=True)}


@pytest.mark.parametrize("flags", FLAGS)
@pytest.mark.parametrize("name", graph64.GRAPHS)
def test_gradients_match_64_bits(dev, q, name, flags):
    g, loss = graph64.GRAPHS[name](**FLAGS[flags])
    grads = g.backward(loss)
    feeds = graph64.inputs(g, 11)
    exe = g.compile(dev)
    for n, x in feeds.items():
        if g.values[n].dtype == "bf16":
            exe.write(q, n, rng.f32_to_bf16(x))
            feeds[n] = rng.bf16_to_f32(rng.f32_to_bf16(x))
        else:
            exe.write(q, n, x)
    exe.run(q)
    names = [loss.name] + [d.name for d in grads.values()]
    eager = {n: exe.read(q, n) for n in names}
    plain, ploss = graph64.GRAPHS[name]()  # the same gradients from the ops of the plain form
    pgrads = plain.backward(ploss)
    v = graph64.run(plain, feeds)
    want = float(v[ploss.name][0])
    assert abs(float(eager[loss.name][0]) - want) <= REL * abs(want)
    assert set(grads) == set(pgrads)
    for p, d in grads.items():
        ref = v[pgrads[p].name]
        assert np.linalg.norm(eager[d.name].astype(np.float64) - ref) <= REL * np.linalg.norm(ref), p
    step = exe.capture(q)
    for _ in range(3):
        for n in names:
            exe.t[n].buffer.fill_u32(q, 0x7FC07FC0)
        q.sync()
        step.launch(q)
        q.sync()
        for n in names:
            assert np.array_equal(exe.read(q, n), eager[n]), n
    step.destroy()
    exe.free()
