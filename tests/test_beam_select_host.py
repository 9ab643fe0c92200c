"""Beam search's choice without a GPU: what the call refuses, and the plain model
against direct sums."""
import math

import numpy as np
import pytest

from tests import beam_model


def tensors(sdk, groups=2, beams=3, vocab=9, keep=3, dtype="f32", device=False):
    give = {"logits": (dtype, (groups, beams, vocab)), "scores": ("f32", (groups, beams)),
            "ended": ("u32", (groups, beams)), "parents": ("u32", (groups, keep)), "tokens": ("u32", (groups, keep)),
            "new_scores": ("f32", (groups, keep)), "new_ended": ("u32", (groups, keep))}
    return {n: sdk.tensor(d, s, device=device) for n, (d, s) in give.items()}


def refuse(sdk, t, end=1, dtype="f32"):
    ok, message = sdk.try_call(f"tensor_beam_select_{dtype}", t["logits"], t["scores"], t["ended"], end, t["parents"],
                               t["tokens"], t["new_scores"], t["new_ended"])
    assert ok == 0
    return message


@pytest.fixture(scope="module")
def plain_sdk():
    from inference_c_amd import Sdk
    return Sdk()


@pytest.mark.parametrize("name", ["logits", "scores", "parents", "tokens", "new_scores"])
def test_missing_operands(plain_sdk, name):
    t = tensors(plain_sdk)
    t[name] = None
    assert refuse(plain_sdk, t).startswith("beam select requires rank-3 F32 logits")


@pytest.mark.parametrize("name,dtype,shape", [("logits", "f16", (2, 3, 9)), ("logits", "f32", (6, 9)),
                                              ("scores", "f16", (2, 3)), ("scores", "f32", (6,)),
                                              ("ended", "f32", (2, 3)), ("parents", "i32", (2, 3)),
                                              ("tokens", "u32", (2, 3, 1)), ("new_scores", "u32", (2, 3)),
                                              ("new_ended", "f32", (2, 3))])
def test_types_and_ranks(plain_sdk, name, dtype, shape):
    t = tensors(plain_sdk)
    t[name] = plain_sdk.tensor(dtype, shape, device=False)
    assert refuse(plain_sdk, t).startswith("beam select requires rank-3 F32 logits")
    if name == "logits" and dtype == "f32":
        assert refuse(plain_sdk, tensors(plain_sdk), dtype="f16").startswith("beam select requires rank-3 F16 logits")


@pytest.mark.parametrize("sizes,end", [(dict(beams=65), 1), (dict(beams=0), 1), (dict(keep=0), 1), (dict(keep=65), 1),
                                       (dict(vocab=0), 0), (dict(), 9), (dict(), 2 ** 32 - 1)])
def test_sizes(plain_sdk, sizes, end):
    assert refuse(plain_sdk, tensors(plain_sdk, **sizes), end).startswith("beam select requires 1 to 64 beams")


@pytest.mark.parametrize("name,shape", [("scores", (3, 2)), ("ended", (2, 4)), ("parents", (1, 3)), ("tokens", (2, 4)),
                                        ("new_scores", (3, 3)), ("new_ended", (2, 2))])
def test_shapes(plain_sdk, name, shape):
    t = tensors(plain_sdk)
    t[name] = plain_sdk.tensor(t[name].dtype, shape, device=False)
    assert refuse(plain_sdk, t).startswith("beam select: scores and ended flags must be")


@pytest.mark.parametrize("a,b", [("parents", "tokens"), ("parents", "new_ended"), ("tokens", "new_ended"),
                                 ("parents", "ended"), ("tokens", "ended")])
def test_outputs_apart(plain_sdk, a, b):
    t = tensors(plain_sdk)
    t[b] = t[a]
    assert refuse(plain_sdk, t).startswith("beam select: outputs must be tensors of their own")


def test_without_device(plain_sdk):
    if plain_sdk.available:
        pytest.skip("a HIP device is present")
    assert refuse(plain_sdk, tensors(plain_sdk)).startswith("HIP device unavailable")


def test_the_plain_choice_by_direct_sums():
    """Scores by fsum, candidates by Python's sort."""
    rng = np.random.default_rng(3)
    logits = rng.integers(-3, 4, (3, 3, 11)).astype(np.float64)   # (with ties)
    logits[0, 1, 4] = -np.inf
    logits[1, 0] = -np.inf
    scores = np.array([[-1, -2, -1.5], [-1, -1, -3], [0, -np.inf, np.nan]])
    ended = np.array([[0, 0, 0], [0, 1, 0], [0, 0, 1]])
    got = beam_model.select(logits, scores, ended, 7, 9)
    for g in range(3):
        found = []
        for b in range(3):
            if math.isnan(scores[g, b]) or scores[g, b] == -math.inf:
                continue
            if ended[g, b]:
                found.append((-scores[g, b], b, 0.0, 7))
                continue
            total = math.fsum(math.exp(x) for x in logits[g, b])
            for v, x in enumerate(logits[g, b]):
                if x > -math.inf:
                    found.append((-(scores[g, b] + x - math.log(total)), b, -x, v))
        found.sort(key=lambda f: (round(f[0], 10), f[1:]))
        want = found[:9] + [(math.inf, 0, 0.0, 7)] * (9 - len(found))
        assert got[0][g].tolist() == [w[1] for w in want] and got[1][g].tolist() == [w[3] for w in want]
        assert np.allclose(np.nan_to_num(got[2][g], neginf=-99), [-99 if w[0] == math.inf else -w[0] for w in want],
                           rtol=0, atol=1e-13)
        assert got[3][g].tolist() == [int(w[3] == 7) for w in want]
