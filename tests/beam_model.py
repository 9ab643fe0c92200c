"""A plain 64-bit model of beam search's choice (tensor_beam_select,
include/tensor_ops_ext.h) and of the caches it works with, for the tests."""
import numpy as np

from tests.kv_model import Model


def log_sum(x):
    """log sum exp of a row without NaN, and its largest element."""
    top = x.max()
    if top == -np.inf:
        return -np.inf, top
    with np.errstate(invalid="ignore"):
        t = np.where(x == top, 0.0, x - top)
    return np.log(np.exp(t).sum()), top


def scores_of(logits, scores, ended, end_token):
    """Scores [groups, beams, vocab] in f64, -inf where there is no candidate."""
    x, scores = logits.astype(np.float64), scores.astype(np.float64)
    out = np.full(x.shape, -np.inf)
    for g, b in np.ndindex(x.shape[:2]):
        if np.isnan(scores[g, b]):
            continue
        if ended is not None and ended[g, b]:
            out[g, b, end_token] = scores[g, b]
            continue
        row = x[g, b]
        if np.isnan(row).any() or row.max() == -np.inf:
            continue
        total, top = log_sum(row)
        with np.errstate(invalid="ignore"):
            out[g, b] = scores[g, b] + (np.where(row == top, 0.0, row - top) - total)
        out[g, b][np.isnan(out[g, b])] = -np.inf
        out[g, b][row == -np.inf] = -np.inf
    return out


def select(logits, scores, ended, end_token, keep):
    """(parents, tokens, new scores in f64, new ended)."""
    groups, beams, vocab = logits.shape
    table = scores_of(logits, scores, ended, end_token)
    parents = np.zeros((groups, keep), np.uint32)
    tokens = np.full((groups, keep), end_token, np.uint32)
    best = np.full((groups, keep), -np.inf)
    beam, token = np.divmod(np.arange(beams * vocab), vocab)
    for g in range(groups):
        s, x = table[g].reshape(-1), logits[g].reshape(-1).astype(np.float64)
        order = np.lexsort((token, -x, beam, -s))[:keep]
        order = order[s[order] > -np.inf]
        parents[g, :len(order)] = beam[order]
        tokens[g, :len(order)] = token[order]
        best[g, :len(order)] = s[order]
    return parents, tokens, best, (tokens == end_token).astype(np.uint32)


def tolerance(logits, scores, ended):
    """How far a new score may be from the model's, in units of 2^-24 for each
    group. The kernel's log sums: t = x - max rounds (|t|), the exponent's two products
    round (2 |t|), the exponential is off by 1 in its last place (2), each as a relative
    error of its term, of which the sum has the weighted mean; a lane adds up its terms of
    at most (vocab / 512 + 1) tiles of 8 in f32, and rescales twice a tile (6 more each),
    all of at most 1 relative; the rest is f64. Then the score rounds to f32."""
    x = logits.astype(np.float64)
    out = np.zeros(x.shape[0])
    tiles = x.shape[2] // 512 + 2
    for g, b in np.ndindex(x.shape[:2]):
        if ended is not None and ended[g, b]:
            continue
        row = x[g, b][np.isfinite(x[g, b])]
        if row.size == 0:
            continue
        t = row - row.max()
        p = np.exp(t)
        out[g] = max(out[g], 3 * (p * -t).sum() / p.sum() + 2 + (8 + 6) * tiles)
    return out


class Joined:
    """What attention sees of a sequence: its prefix's tokens, then its own."""

    def __init__(self, prefix, own):
        self.parts = prefix, own

    def held(self):
        return np.concatenate([p.held() for p in self.parts])


def joined(prefix, own, members):
    """The model of attention over `own`'s sequences behind their prefixes."""
    model = Model(*own.shape)
    on = [p for p, m in enumerate(members) for _ in range(m)]
    for b in range(own.shape[0]):
        for h in range(own.shape[1]):
            model.k[b][h] = Joined(prefix.k[on[b]][h], own.k[b][h])
            model.v[b][h] = Joined(prefix.v[on[b]][h], own.v[b][h])
            model.marked[b][h] = np.concatenate([prefix.marked[on[b]][h], own.marked[b][h]])
    return model
