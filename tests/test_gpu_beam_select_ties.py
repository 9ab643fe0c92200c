"""Rows of which many logits equal the bound of a part's candidates (masks by the type's
lowest number, flat rows): the first of them are chosen, and the choice takes hardly longer."""
import time

import numpy as np
import pytest

from tests import beam_model
from tests.test_gpu_beam_select import DTYPES, call_select

pytestmark = pytest.mark.gpu


def rows_with_ties(vocab, dtype):
    i = np.arange(vocab)
    low = np.finfo(DTYPES[dtype]).min
    rng = np.random.default_rng(vocab)
    kinds = [np.zeros(vocab), np.where(i % 2, 1.0, low), np.where(i % 64 < 3, 2.0, 1.0), np.where(i < vocab // 2, low, -5.0),
             np.where(i < vocab // 2, -5.0, low), np.where(rng.random(vocab) < 0.01, 3.0, low), rng.integers(-2, 2, vocab),
             np.where(i // 512 % 2, 0.0, -0.0), np.where(i == vocab - 1, 1.0, low), (i // 3000 % 5) * 1.0,
             np.where(i // 4 % 2, -np.inf, 0.5), np.where(i >= vocab - 1100, 0.25, -i / vocab)]
    return [np.asarray(k, np.float64).astype(DTYPES[dtype]) for k in kinds]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("vocab", [900, 1030, 20011, 70003])
@pytest.mark.parametrize("keep", [1, 3, 8, 23, 24, 64])
def test_the_first_of_equal_logits(sdk, keep, vocab, dtype):
    """In one part (2100 rows of which all are like the first ones) and in many."""
    kinds = rows_with_ties(vocab, dtype)
    wants = [beam_model.select(row[None, None], np.zeros((1, 1), np.float32), None, 7, keep) for row in kinds]
    for groups in (len(kinds), 2100 if vocab == 20011 else 60):
        logits = np.stack([kinds[g % len(kinds)] for g in range(groups)])[:, None]
        parents, tokens, _, _ = call_select(sdk, logits, np.zeros((groups, 1), np.float32), None, 7, keep)
        assert (parents == 0).all()
        for g in range(groups):
            assert np.array_equal(tokens[g], wants[g % len(kinds)][1][0]), f"row {g} of {groups}, kind {g % len(kinds)}"


def milliseconds(sdk, logits, keep):
    """Of one call, the quickest of several runs."""
    groups, beams, _ = logits.shape
    x, s = sdk.from_numpy(logits), sdk.from_numpy(np.zeros((groups, beams), np.float32))
    outs = [sdk.tensor(d, (groups, keep)) for d in ("u32", "u32", "f32")]
    dtype = "f16" if logits.dtype == np.float16 else "f32"
    best = np.inf
    for _ in range(6):
        sdk.synchronize()
        start = time.perf_counter()
        for _ in range(20):
            sdk.call(f"tensor_beam_select_{dtype}", x, s, None, 5, *outs, None)
        sdk.synchronize()
        best = min(best, (time.perf_counter() - start) / 20 * 1e3)
    return best


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_equal_logits_take_hardly_longer(sdk, dtype):
    """All but three logits at the type's lowest number, and all alike: few of the many
    that reach the bound are looked at (all of them took 8 to 11 times as long as usual;
    1.3 and 1.7 times are measured, of which ties of all beams in the choice are most)."""
    rng = np.random.default_rng(3)
    ordinary = np.broadcast_to((2.5 * rng.standard_normal((1, 8, 128256))).astype(DTYPES[dtype]), (32, 8, 128256))
    masked = np.full(ordinary.shape, np.finfo(DTYPES[dtype]).min, DTYPES[dtype])
    masked[:, :, [5, 70000, 128000]] = 1
    usual = milliseconds(sdk, ordinary, 8)
    for what, logits in (("masked", masked), ("flat", np.zeros_like(masked))):
        took = milliseconds(sdk, logits, 8)
        print(f"{dtype} {what}: {took * 1e3:.1f} us, ordinary {usual * 1e3:.1f}")
        assert took < 2.2 * usual, what
