"""Padded query rows of attention over the cache: what they hold has no effect on any
bit of the rows that are there, nor on the weights."""
import numpy as np
import pytest

from tests.test_gpu_kv_attention import attend as attend_plain
from tests.test_gpu_kv_cache import DTYPES
from tests.test_gpu_kv_shared import pair_of

pytestmark = pytest.mark.gpu


def paddings(rng, q, counts):
    """The rows q with padding of several kinds."""
    there = np.arange(q.shape[2]) < np.array(counts)[:, None]
    where = np.broadcast_to(there[:, None, :, None], q.shape)
    for kind in (0.0, 30.0, 1000.0, np.nan, np.inf):
        with np.errstate(over="ignore", invalid="ignore"):
            yield kind, np.where(where, q, (kind * rng.standard_normal(q.shape)).astype(q.dtype))


def same(results):
    (_, first), *others = results
    for kind, other in others:
        for a, b in zip(first, other):
            assert (a is None and b is None) or np.array_equal(a.view(np.uint8), b.view(np.uint8)), f"padding of {kind}"


@pytest.mark.parametrize("weighted", [False, True], ids=["", "weights"])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("lengths,heads,n,counts", [
    ([40, 30, 3, 20], 8, 3, [3, 1, 0, 2]), ([900, 700, 800, 100], 8, 11, [11, 2, 0, 7]),
    ([3000, 2900], 16, 700, [333, 700])], ids=["few", "rows", "tiles"])
def test_over_own_tokens(sdk, lengths, heads, n, counts, dtype, weighted):
    own = pair_of(sdk, 4, (128, 128), lengths, 3)
    q = own.rng.standard_normal((len(lengths), heads, n, 128)).astype(DTYPES[dtype])
    w0 = np.zeros((len(lengths), 4, max(lengths)), np.float32) if weighted else None
    same([(kind, attend_plain(sdk, own.cache, x, 0.3, True, counts, w0, 128)) for kind, x in paddings(own.rng, q, counts)])
