"""Beam search's choice against the plain model: the candidates and their order
exactly, but where two beams' scores are closer than the log sums are known; scores
within the roundings that tests/beam_model.py counts."""
import ctypes
import threading

import numpy as np
import pytest

from tests import beam_model

pytestmark = pytest.mark.gpu

DTYPES = {"f16": np.float16, "f32": np.float32}


def call_select(sdk, logits, scores, ended, end_token, keep, device=True, flags=True):
    groups = logits.shape[0]
    dtype = "f16" if logits.dtype == np.float16 else "f32"

    def give(a):
        return None if a is None else sdk.from_numpy(a, device=device)

    outs = [sdk.from_numpy(np.full((groups, keep), 9, d), device=device)
            for d in (np.uint32, np.uint32, np.float32, np.uint32)]
    sdk.call(f"tensor_beam_select_{dtype}", give(logits), give(scores), give(ended), end_token, *outs[:3],
             outs[3] if flags else None)
    return [o.download() for o in outs]


def check(got, logits, scores, ended, end_token, keep, what=""):
    parents, tokens, new_scores, new_ended = got
    want_p, want_t, want_s, _ = beam_model.select(logits, scores, ended, end_token, keep)
    table = beam_model.scores_of(logits, scores, ended, end_token)
    units = beam_model.tolerance(logits, scores, ended)
    assert np.array_equal(new_ended, (tokens == end_token).astype(np.uint32)), what
    for g in range(logits.shape[0]):
        # with the rounding of the f64 sums of scores that are this large
        off = units[g] * 2.0 ** -24 + 1e-12
        there = want_s[g] > -np.inf
        assert np.array_equal(new_scores[g] > -np.inf, there), f"{what} group {g}"
        assert (parents[g][~there] == 0).all() and (tokens[g][~there] == end_token).all(), f"{what} group {g}"
        finite = there & np.isfinite(want_s[g])
        assert np.array_equal(new_scores[g][there & ~finite], want_s[g][there & ~finite]), f"{what} group {g}"
        bound = off + 2.0 ** -24 * np.abs(want_s[g][finite])
        assert (np.abs(new_scores[g][finite] - want_s[g][finite]) <= bound).all(), f"{what} group {g}"
        differ = np.flatnonzero((parents[g] != want_p[g]) | (tokens[g] != want_t[g]))
        for i in differ:   # another beam's candidate of all but the same score
            score = table[g, parents[g, i], tokens[g, i]]
            assert abs(score - want_s[g, i]) <= 2 * off and parents[g, i] != want_p[g, i], \
                f"{what} group {g}: place {i} is ({parents[g, i]}, {tokens[g, i]}), not ({want_p[g, i]}, {want_t[g, i]})"
        pairs = list(zip(parents[g][there], tokens[g][there]))
        assert len(set(pairs)) == len(pairs), f"{what} group {g}: a candidate twice"


def run(sdk, rng, groups, beams, vocab, keep, dtype, ended=False, spread=2.5, logits=None, device=True, what=""):
    if logits is None:
        logits = (spread * rng.standard_normal((groups, beams, vocab))).astype(DTYPES[dtype])
    scores = np.sort(-8 - 2 * np.abs(rng.standard_normal((groups, beams))))[:, ::-1].astype(np.float32).copy()
    flags = (rng.random((groups, beams)) < 0.4).astype(np.uint32) if ended else None
    end = int(rng.integers(vocab))
    got = call_select(sdk, logits, scores, flags, end, keep, device)
    check(got, logits, scores, flags, end, keep, f"{what} {groups}x{beams}x{vocab} keep {keep} {dtype}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 63, 511, 512, 513, 1000, 1025, 5003, 32003])
def test_vocabularies(sdk, vocab, dtype):
    """Rows that start anywhere in memory, of less than a vector to many parts."""
    rng = np.random.default_rng(vocab)
    run(sdk, rng, 2, 3, vocab, min(6, 3 * vocab), dtype)
    run(sdk, rng, 3, 1, vocab, 1, dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("beams,keep", [(1, 64), (2, 5), (4, 4), (5, 11), (8, 16), (16, 32), (33, 64), (64, 64), (64, 1)])
def test_beams_and_kept(sdk, beams, keep, dtype):
    rng = np.random.default_rng(100 * beams + keep)
    run(sdk, rng, 2, beams, 1501, keep, dtype)
    run(sdk, rng, 3, beams, 2000, keep, dtype, ended=True, what="ended")


def test_large_vocabulary(sdk):
    """More candidates per lane than a wave takes at once, and one row alone."""
    rng = np.random.default_rng(7)
    run(sdk, rng, 1, 2, 300001, 64, "f32")
    run(sdk, rng, 1, 1, 300001, 64, "f16")


def test_many_groups(sdk):
    run(sdk, np.random.default_rng(8), 700, 4, 130, 8, "f16", ended=True)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("order", ["rising", "falling", "flat", "two values", "zeros of both signs", "rising by lanes"])
def test_orders_that_fill_the_lists(sdk, order, dtype):
    """Every logit larger than all before it, or none, or all alike: equal ones are
    taken in the order of beams, then of tokens."""
    vocab = 6001
    i = np.arange(vocab)
    row = {"rising": i / 512, "falling": -i / 512, "flat": 0 * i, "two values": np.where(i % 37 == 5, 1, 0),
           "zeros of both signs": np.where(i % 3 == 0, -0.0, 0.0), "rising by lanes": i % 512 / 64.0}[order]
    logits = np.broadcast_to(row, (2, 3, vocab)).astype(DTYPES[dtype])
    for scores in (np.zeros((2, 3)), np.array([[0, -1, -2], [-3, -0.5, -0.5]])):
        scores = scores.astype(np.float32)
        got = call_select(sdk, logits, scores, None, 5, 40)
        want = beam_model.select(logits, scores, None, 5, 40)
        # rows alike have the same log sum, so that beams' equal scores are equal here too
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), order
        check(got, logits, scores, None, 5, 40, order)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_masked_logits(sdk, dtype):
    """Rows of which few tokens are allowed, one or none: the rest of the outputs is
    the end token without a score."""
    rng = np.random.default_rng(11)
    logits = rng.standard_normal((4, 3, 2500)).astype(DTYPES[dtype])
    logits[0][rng.random((3, 2500)) < 0.997] = -np.inf
    logits[1] = -np.inf
    logits[2, :2] = -np.inf
    logits[2, 2, np.arange(2500) != 1777] = -np.inf
    logits[3, 0] = -np.inf
    run(sdk, rng, 4, 3, 2500, 20, dtype, logits=logits)
    run(sdk, rng, 4, 3, 2500, 20, dtype, logits=logits, ended=True)


def test_lowest_values(sdk):
    """Masks by the type's lowest number are candidates, after all others."""
    for dtype in (np.float16, np.float32):
        logits = np.full((1, 2, 700), np.finfo(dtype).min, dtype)
        logits[0, 0, 10:14] = [1, 3, 2, 3]
        logits[0, 1, 699] = 0
        scores = np.array([[-1, -2]], np.float32)
        got = call_select(sdk, logits, scores, None, 0, 8)
        check(got, logits, scores, None, 0, 8)
        assert got[0][0].tolist()[:5] == [0, 0, 1, 0, 0] and got[1][0].tolist()[:5] == [11, 13, 699, 12, 10]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_special_logits_and_scores(sdk, dtype):
    """NaN in a row or a score: no candidates of that beam. +inf: those logits share
    the probability. Scores of -inf: none; of +inf: in their order."""
    rng = np.random.default_rng(12)
    base = rng.standard_normal((6, 3, 1500)).astype(DTYPES[dtype])
    base[0, 1, 700] = np.nan
    base[1, 0, [3, 900, 1400]] = np.inf
    base[2, 2, 5], base[2, 2, 1200] = np.inf, np.nan
    base[3] = np.nan
    base[4, 0, :1024] = -np.inf
    scores = -np.abs(rng.standard_normal((6, 3))).astype(np.float32)
    scores[4, 1], scores[5, 0], scores[5, 2] = -np.inf, np.nan, np.inf
    ended = np.zeros((6, 3), np.uint32)
    ended[2, 2] = 7       # any flag but 0; its logits are not looked at
    ended[3, 1] = 1
    for flags in (None, ended):
        got = call_select(sdk, base, scores, flags, 1499, 10)
        check(got, base, scores, flags, 1499, 10, dtype)


def test_ended_beams_without_a_score(sdk):
    logits = np.zeros((1, 3, 40), np.float32)
    scores = np.array([[-np.inf, np.nan, -2]], np.float32)
    got = call_select(sdk, logits, scores, np.ones((1, 3), np.uint32), 39, 3)
    assert got[0].tolist() == [[2, 0, 0]] and got[1].tolist() == [[39, 39, 39]]
    assert got[2].tolist() == [[-2, -np.inf, -np.inf]] and got[3].tolist() == [[1, 1, 1]]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_scores_in_place_and_without_flags(sdk, dtype):
    rng = np.random.default_rng(13)
    logits = rng.standard_normal((2, 4, 900)).astype(DTYPES[dtype])
    scores = -np.abs(rng.standard_normal((2, 4))).astype(np.float32)
    ended = np.array([[0, 1, 0, 0], [1, 0, 0, 1]], np.uint32)
    for device in (True, False):
        s, e = sdk.from_numpy(scores, device=device), sdk.from_numpy(ended, device=device)
        p, t = (sdk.from_numpy(np.zeros((2, 4), np.uint32), device=device) for _ in range(2))
        sdk.call(f"tensor_beam_select_{dtype}", sdk.from_numpy(logits, device=device), s, e, 17, p, t, s, e)
        check([x.download() for x in (p, t, s, e)], logits, scores, ended, 17, 4)
    got = call_select(sdk, logits, scores, ended, 17, 4, flags=False)
    assert (got[3] == 9).all()
    got[3] = (got[1] == 17).astype(np.uint32)
    check(got, logits, scores, ended, 17, 4)


def test_host_operands(sdk):
    run(sdk, np.random.default_rng(14), 2, 3, 4001, 7, "f16", ended=True, device=False)
    run(sdk, np.random.default_rng(15), 2, 3, 4001, 7, "f32", device=False)


def test_no_groups(sdk):
    e = [sdk.tensor(d, (0, 3)) for d in ("u32", "u32", "f32")]
    sdk.call("tensor_beam_select_f32", sdk.tensor("f32", (0, 2, 9)), sdk.tensor("f32", (0, 2)), None, 1, *e, None)


def test_the_same_again(sdk):
    """Results do not depend on which waves are first."""
    rng = np.random.default_rng(16)
    logits = (2.5 * rng.standard_normal((2, 8, 50021))).astype(np.float16)
    scores = -np.abs(rng.standard_normal((2, 8))).astype(np.float32)
    first = call_select(sdk, logits, scores, None, 3, 16)
    for _ in range(5):
        again = call_select(sdk, logits, scores, None, 3, 16)
        assert all(np.array_equal(a, b) for a, b in zip(first, again))


def test_recorded(sdk):
    """Two recorded calls of one stream, replayed with eager ones in between, on
    logits that have changed meanwhile."""
    hip = sdk.lib
    stream = ctypes.c_void_p(sdk.stream())
    rng = np.random.default_rng(17)
    logits = [(2.5 * rng.standard_normal((2, 4, 9001))).astype(np.float32) for _ in range(4)]
    scores = -np.abs(rng.standard_normal((2, 4))).astype(np.float32)
    x, s = [sdk.from_numpy(logits[i]) for i in range(2)], sdk.from_numpy(scores)
    outs = [[sdk.tensor(d, (2, 4)) for d in ("u32", "u32", "f32", "u32")] for _ in range(2)]
    calls = [("tensor_beam_select_f32", x[i], s, None, 3, *outs[i]) for i in range(2)]
    runs = []
    for call in calls:
        sdk.call(*call)
        sdk.synchronize()
        graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
        assert hip.hipStreamBeginCapture(stream, 2) == 0
        try:
            sdk.call(*call)
        finally:
            assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
        assert hip.hipGraphDestroy(graph) == 0
        runs.append(exe)
    for replay in range(4):
        for i in range(2):
            x[i].upload(logits[(replay + i) % 4])
        for exe in runs:
            assert hip.hipGraphLaunch(exe, stream) == 0
        call_select(sdk, logits[3], scores, None, 1, 4)
        for i in range(2):
            check([o.download() for o in outs[i]], logits[(replay + i) % 4], scores, None, 3, 4, f"replay {replay}")
    sdk.synchronize()
    for exe in runs:
        assert hip.hipGraphExecDestroy(exe) == 0


def test_largest_vocabulary(sdk):
    """2^26 tokens: the last of them, equal ones far apart, and sums of as many terms."""
    vocab = 2 ** 26
    logits = np.random.default_rng(18).random((1, 1, vocab), np.float32).astype(np.float16)
    logits[0, 0, [vocab - 1, 5, vocab // 2 + 1]] = [4, 3, 3]
    scores = np.array([[-1]], np.float32)
    got = call_select(sdk, logits, scores, None, vocab - 1, 3)
    assert got[0].tolist() == [[0, 0, 0]] and got[1].tolist() == [[vocab - 1, 5, vocab // 2 + 1]]
    assert got[3].tolist() == [[1, 0, 0]]
    total = sum(np.exp(part.astype(np.float64)).sum() for part in np.array_split(logits[0, 0], 64))
    # as beam_model.tolerance counts for 128 parts of 512 tiles each
    off = (3 * 4 + 2 + (8 + 6) * 2 * 513) * 2.0 ** -24
    assert (np.abs(got[2][0] - (np.array([4, 3, 3]) - 1 - np.log(total))) <= off + 2.0 ** -24 * 20).all()


def test_more_groups_than_one_launch_takes(sdk):
    """Of 2^22 + 3 groups each its own choice."""
    groups = 2 ** 22 + 3
    rng = np.random.default_rng(19)
    logits = rng.integers(-8, 9, (groups, 1, 3)).astype(np.float16)
    scores = rng.integers(-9, 0, (groups, 1)).astype(np.float32)
    ended = (rng.random((groups, 1)) < 0.1).astype(np.uint32)
    parents, tokens, new_scores, new_ended = call_select(sdk, logits, scores, ended, 2, 1)
    over = ended[:, 0] != 0
    want = np.where(over, 2, logits[:, 0].argmax(-1))
    assert (parents == 0).all() and np.array_equal(tokens[:, 0], want) and np.array_equal(new_ended[:, 0], want == 2)
    x = logits[:, 0].astype(np.float64)
    s = np.where(over, scores[:, 0], scores[:, 0] + x.max(-1) - np.log(np.exp(x).sum(-1)))
    # (3 |t| + 2 + (8 + 6) * 2) units at 16 at most, and the score's rounding
    assert (np.abs(new_scores[:, 0] - s) <= (3 * 16 + 2 + 28 + 16) * 2.0 ** -24).all()


def test_threads(sdk):
    errors = []

    def work(seed):
        try:
            rng = np.random.default_rng(seed)
            for i in range(6):
                run(sdk, rng, 2, 4, 3001 + seed, 8, ("f16", "f32")[i % 2], ended=i % 3 == 0, device=i % 4 != 3,
                    what=f"thread {seed}")
        except BaseException as e:      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
