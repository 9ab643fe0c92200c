"""Copies and reorders from several host threads, of sequences that all differ: every
target ends with exactly the sequences that its thread asked for, a copy beside
reorders has all of its sequences from before or all from after one, and reorders that
cancel out leave their cache as it was."""
import threading

import numpy as np
import pytest

from tests.kv_model import Model, u32s
from tests.test_gpu_kv_cache import check_read
from tests.test_gpu_kv_sequences import KEEP, copied, filled

pytestmark = pytest.mark.gpu

DIMS = (64, 32)


def in_threads(work, count):
    errors = []

    def body(i):
        try:
            work(i)
        except BaseException as e:      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=body, args=(i,)) for i in range(count)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]


def test_copies_from_one_cache_into_one_each(sdk):
    source = filled(sdk, 6, 2, 200, DIMS, [130, 64, 199, 7, 0, 191], 31, marks=True)

    def work(i):
        rng = np.random.default_rng(i)
        target, model = sdk.kv_cache(5, 2, 220, *DIMS), Model(5, 2, *DIMS)
        for step in range(30):
            which = [int(s) if s < 6 else KEEP for s in rng.integers(0, 8, 5)]
            sdk.call("tensor_kv_cache_copy", source.cache, u32s(which), target)
            model = copied(source.model, which, model)
            if step % 10 == 9:
                check_read(sdk, target, model, f"thread {i}, step {step}")

    in_threads(work, 4)
    source.check("the source")


def test_copies_beside_reorders(sdk):
    beams = filled(sdk, 8, 2, 200, DIMS, [130] * 4 + [75] * 4, 32, marks=True)
    before = beams.model
    after = copied(before, [1, 0, 3, 2, 7, 6, 5, 4], before)

    def work(i):
        swap = sdk.from_numpy(np.array([[1, 0, 3, 2], [3, 2, 1, 0]], np.uint32))
        target = sdk.kv_cache(8, 2, 200, *DIMS)
        for step in range(40):
            sdk.call("tensor_kv_cache_reorder", beams.cache, swap)
            if step % 4 == i:
                which = [(b + i + step) % 8 for b in range(8)]
                sdk.call("tensor_kv_cache_copy", beams.cache, u32s(which), target)
                wants = [copied(m, which, Model(8, 2, *DIMS)) for m in (before, after)]
                try:
                    check_read(sdk, target, wants[0])
                except AssertionError:
                    check_read(sdk, target, wants[1], f"thread {i}, step {step}: neither before nor after a reorder")

    in_threads(work, 4)
    beams.check("after an even number of swaps")


def test_reorders_of_a_cache_each(sdk):
    def work(i):
        rng = np.random.default_rng(50 + i)
        pair = filled(sdk, 6, 2, 200, DIMS, [100 + i] * 3 + [64 - i] * 3, 40 + i)
        for step in range(30):
            parents = rng.integers(0, 3, (2, 3)).astype(np.uint32) if step % 6 == 0 else \
                np.stack([rng.permutation(3) for _ in range(2)]).astype(np.uint32)
            sdk.call("tensor_kv_cache_reorder", pair.cache, sdk.from_numpy(parents))
            which = [g * 3 + int(p) for g in range(2) for p in parents[g]]
            pair.model = copied(pair.model, which, pair.model)
        pair.check(f"thread {i}")

    in_threads(work, 4)
