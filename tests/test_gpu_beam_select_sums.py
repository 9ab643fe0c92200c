"""The log sums behind beam search's scores: as exact as their exponentials however
many terms a part of a row has and however they lie, so that beams whose scores are
close keep their order."""
import numpy as np
import pytest

from tests.test_gpu_beam_select import DTYPES, call_select

pytestmark = pytest.mark.gpu


def log_sum(x):
    """log sum exp of a row in f64, and how far the kernel's may be from it. Its terms'
    relative errors, in units of 2^-24: t = x - max is rounded once, t log2 e once (|t|
    each, as errors of the exponent), the exponential is off by one in its last place (2),
    and the sum of a lane's 16 terms of a tile rounds each at most 4 times; all else is
    f64. The sum's error is the terms' mean by weight, the log's is the same number."""
    t = x.astype(np.float64) - np.float64(x.max())
    p = np.exp(t)
    units = 2 * (p * -t).sum() / p.sum() + 2 + 4
    return np.float64(x.max()) + np.log(p.sum()), 1.01 * units * 2.0 ** -24


def rows_of_all_kinds(vocab, dtype):
    """Plateaus (whose terms all round the same way), normal, rising (the maximum moves
    with every tile) and falling rows, far from 0 too; the largest logit is at token 77."""
    i = np.arange(vocab)
    rng = np.random.default_rng(vocab)
    kinds = {"plateau": np.where(i < 1024, 0.0, -6.3), "near": np.full(vocab, -0.1), "farther": np.full(vocab, -1.3),
             "deep": np.full(vocab, -9.1), "normal": 2.5 * rng.standard_normal(vocab), "rising": 12 * i / vocab,
             "falling": -12 * i / vocab, "steps": np.floor(i / 1024) * 0.37, "large": 900 - 3 * rng.random(vocab),
             "low": -900 - rng.standard_normal(vocab), "two thirds": np.where(i % 3 == 0, -2.7, -0.4)}
    if dtype == "f32":
        kinds["past f16"] = 1e6 + rng.integers(-8, 0, vocab)
    out = {}
    for name, row in kinds.items():
        row = row.astype(DTYPES[dtype])
        row[77] = row.max()
        row[77] = np.nextafter(row[77], DTYPES[dtype](np.inf))
        out[name] = row
    return out


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("groups,vocab", [(1, 128256), (15, 700), (300, 128256), (2052, 32003)])
def test_log_sums(sdk, groups, vocab, dtype):
    """In 126 parts of a row, one short one, 13 of ten tiles, and one of 32. Scores that
    all but cancel the log sum show it to its last digits."""
    kinds = rows_of_all_kinds(vocab, dtype)
    sums = {name: log_sum(row) for name, row in kinds.items()}
    names = [list(kinds)[g % len(kinds)] for g in range(max(groups, len(kinds)))]
    for first in range(0, len(names), groups):
        some = names[first:first + groups]
        logits = np.stack([kinds[name] for name in some])[:, None]
        scores = np.array([[sums[name][0] - np.float64(kinds[name][77])] for name in some]).astype(np.float32)
        parents, tokens, new_scores, _ = call_select(sdk, logits, scores, None, 5, 1)
        assert (parents == 0).all() and (tokens == 77).all()
        for g, name in enumerate(some):
            total, off = sums[name]
            want = np.float64(scores[g, 0]) + (np.float64(kinds[name][77]) - total)
            far = abs(new_scores[g, 0] - want)
            assert far <= off + 1e-12 + 2.0 ** -24 * abs(want), f"{name}: off by {far:.3g}, {off:.3g} allowed"


def close_beams(rng, beams, vocab, dtype):
    """Logits [beams, vocab], a plateau and a few larger ones, and scores whose best
    candidates differ by a few millionths, and those candidates' scores in f64."""
    logits = np.empty((beams, vocab), DTYPES[dtype])
    scores, best, offs = np.empty(beams, np.float32), np.empty(beams), np.empty(beams)
    for b, place in enumerate(rng.permutation(beams)):
        logits[b] = -rng.uniform(5, 8) if b % 4 else -4 - rng.random(vocab)
        logits[b, :1024] = 0
        logits[b, 1000 + b] = 0.01
        total, offs[b] = log_sum(logits[b])
        scores[b] = total - 3.4e-6 * place
        best[b] = np.float64(scores[b]) + np.float64(logits[b, 1000 + b]) - total
    gaps = -np.diff(np.sort(best)[::-1])
    assert (gaps > 2 * offs.max()).all()    # (of this test's inputs)
    return logits, scores, best


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("groups,beams,vocab", [(1, 64, 128256), (513, 4, 32003)])
def test_beams_close_to_each_other(sdk, groups, beams, vocab, dtype):
    """In their order, whether a group is alone or among many, which takes its rows in
    fewer parts."""
    logits, scores, best = close_beams(np.random.default_rng(beams), beams, vocab, dtype)
    want = np.argsort(-best)
    for count in {1, groups}:
        x = np.broadcast_to(logits, (count, beams, vocab))
        s = np.broadcast_to(scores, (count, beams))
        parents, tokens, _, _ = call_select(sdk, x, s, None, 5, beams)
        assert (parents == want).all(), f"{count} groups"
        assert (tokens == 1000 + want).all(), f"{count} groups"
