"""Beam selection over logits masked by the lowest f32: offers like others, whose
scores in 64 bits may lie below the lowest f32 and are held at it.

Beside 2^128 what a score and a sum add is rounded off in 64 bits, so masked tokens
tie and go to the lowest beam, then token."""
import numpy as np
import pytest

from test_gpu_beam import TOL, Case, oracle

pytestmark = pytest.mark.gpu

LOWEST = np.finfo(np.float32).min


def masked(seed, batch, beams, vocab, live, left):
    """`live` beams with scores, `left` tokens each that are not masked."""
    rng = np.random.default_rng(seed)
    logits = np.full((batch, beams, vocab), LOWEST, np.float32)
    scores = np.full((batch, beams), -np.inf, np.float32)
    scores[:, live] = rng.uniform(-6, 0, (batch, len(live)))
    for r in range(batch):
        for b in range(beams):
            logits[r, b, rng.choice(vocab, left, replace=False)] = 2.5 * rng.standard_normal(left)
    return logits, scores


def check(c):
    p, t, s, _ = [o.download() for o in c.out]
    want, _ = oracle(c.logits, c.scores, c.finished, c.select, np.float64(np.float32(c.factor)), c.end)
    assert np.array_equal(p, want[0]) and np.array_equal(t, want[1])
    full, low = want[0] >= 0, want[2] < -1e30
    assert np.all(s[~full] == -np.inf) and np.all(s[full & low] == LOWEST)
    some = full & ~low
    assert np.all(np.abs(s[some].astype(np.float64) - want[2][some]) <= TOL + 2.0 ** -24 * np.abs(want[2][some]))
    return s


@pytest.mark.parametrize("factor", [1.0, 1.25, 3.0])
@pytest.mark.parametrize("beams,vocab,select,live,left", [
    (8, 248321, 16, [5, 6, 7], 3),  # 1944 lists, 243 a beam
    (8, 248321, 16, [0, 7], 5), (4, 300, 8, [1, 3], 2), (64, 20000, 64, [52, 53, 60, 63], 7), (64, 20000, 64, [0, 63], 1),
    (1, 50257, 16, [0], 1), (32, 32000, 64, [30], 40),
])
def test_masked_by_the_lowest_value(dev, beams, vocab, select, live, left, factor):
    print(f"[beam] {beams} {vocab} {select} {live} {factor}", flush=True)
    logits, scores = masked(vocab + left, 1, beams, vocab, live, left)
    c = Case(logits, scores, select=select, factor=factor)
    c.run()
    check(c)


@pytest.mark.parametrize("factor", [1.0, 2.0])
def test_the_next_step_goes_on_from_them(dev, factor):
    """Beams held at the lowest score still offer their tokens, behind all others'."""
    logits, scores = masked(3, 2, 4, 3000, [1, 2], 1)
    c = Case(logits, scores, select=4, factor=factor)
    c.run()
    held = check(c)
    assert (held == LOWEST).sum() == 4
    rng = np.random.default_rng(4)
    d = Case((2.5 * rng.standard_normal((2, 4, 3000))).astype(np.float32), held, select=64, factor=factor)
    d.run()
    check(d)
