"""How the cross entropy's gradients are laid out, on the host: pieces of the vocabulary and splits of dx's sum over a
piece's columns.  The 256 x 256 tiles' loop needs at least one stage of 64 columns in every split that is launched (its
copies run two stages ahead of it, so a split without columns would read past the weights)."""
import ctypes as C
import random

import pytest

from vernondsl_amd import _lib

WIDE = 2


def plan(n, vocab, dim, piece):
    v = (C.c_int64 * 7)()
    _lib.call("vdsl_debug_linear_xent_plan", n, vocab, dim, piece, v)
    return dict(zip(("pieces", "piece", "last", "grads", "splits", "last_splits", "dw_splits"), v))


def check(n, vocab, dim, piece):
    p = plan(n, vocab, dim, piece)
    assert (p["pieces"] - 1) * p["piece"] + p["last"] == vocab and 0 < p["last"] <= p["piece"]
    assert p["pieces"] == 1 or p["piece"] % 256 == 0
    assert 1 <= p["last_splits"] <= p["splits"]
    if p["pieces"] == 1:
        assert p["last_splits"] == p["splits"]
    if p["grads"] == WIDE:
        assert p["last_splits"] <= -(-p["last"] // 64), "a split of the last piece has no columns"
        assert p["splits"] <= -(-p["piece"] // 64) and p["dw_splits"] <= -(-n // 64)
    return p


# the vocabulary's remainder is 8 to 64 columns and dx's sum is split
@pytest.mark.parametrize("n,dim,vocab,piece", [(4096, 1536, 18440, 2304), (2048, 1024, 141336, 6144), (1352, 4064, 28167, 2444),
                                               (1024, 5504, 18440, 2304), (1024, 5504, 18496, 2304)])
def test_short_last_piece_has_no_empty_split(n, dim, vocab, piece):
    p = check(n, vocab, dim, piece)
    assert p["grads"] == WIDE and p["pieces"] > 2 and p["splits"] > 1 and p["last"] <= 64 and p["last_splits"] == 1


def test_no_empty_split_over_the_range():
    r = random.Random(3)
    seen = 0
    for _ in range(20000):
        n, dim, vocab = (round(2 ** r.uniform(a, b)) for a, b in ((8, 14), (6, 13), (10, 18)))
        p = check(n, vocab, dim, r.choice([0, round(2 ** r.uniform(8, 14))]))
        seen += p["grads"] == WIDE and p["splits"] > p["last_splits"]
    assert seen  # pieces that do not fill all splits are among them


def test_plan_refusals():
    v = (C.c_int64 * 7)()
    for a in ((4, 0, 64, 0), (4, 9, 4, 0), (-1, 9, 64, 0), (4, 9, 64, -1)):
        with pytest.raises(_lib.VdslError):
            _lib.call("vdsl_debug_linear_xent_plan", *a, v)
    with pytest.raises(_lib.VdslError):
        _lib.call("vdsl_debug_linear_xent_plan", 4, 9, 64, 0, None)
