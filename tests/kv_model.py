"""A plain 64-bit model of the 8-bit key/value cache (include/tensor_kv_cache.h)
and of attention over it, for the tests."""
import ctypes

import numpy as np

BLOCK = 64


def u32s(values):
    return (ctypes.c_uint32 * len(values))(*[int(v) for v in values])


def to_f16(x):
    with np.errstate(over="ignore"):
        return np.asarray(x).astype(np.float16)


def quantise(rows):
    """Codes and f32 scale of exact rows (f64)."""
    a = float(np.abs(rows).max()) if rows.size else 0.0
    if a == 0.0:
        return np.zeros(rows.shape, np.int64), np.float32(0.0)
    return np.rint(127.0 * rows / a).astype(np.int64), np.float32(a / 127.0)


class Head:
    """Keys or values (f16 rows) of one sequence and head."""

    def __init__(self, dim):
        self.dim, self.blocks, self.open = dim, [], np.zeros((0, dim), np.float16)

    def append(self, rows):
        self.open = np.concatenate([self.open, rows])
        while len(self.open) >= BLOCK:
            self.blocks.append(quantise(self.open[:BLOCK].astype(np.float64)))
            self.open = self.open[BLOCK:]

    def held(self):
        """Exact values, f64."""
        parts = [c.astype(np.float64) * float(s) for c, s in self.blocks]
        return np.concatenate(parts + [self.open.astype(np.float64)])

    def f32(self):
        return self.held().astype(np.float32)     # (one rounding of an exact product)

    def truncate(self, n):
        rows = self.f32()[n // BLOCK * BLOCK:n]
        if n // BLOCK < len(self.blocks):
            self.blocks, self.open = self.blocks[:n // BLOCK], rows.astype(np.float16)
        else:
            self.open = self.open[:n - len(self.blocks) * BLOCK]

    def hold_anew(self, values):
        """The head that holds these exact values."""
        new = Head(self.dim)
        whole = len(values) // BLOCK * BLOCK
        new.blocks = [quantise(values[i:i + BLOCK]) for i in range(0, whole, BLOCK)]
        new.open = values[whole:].astype(np.float32).astype(np.float16)
        return new


class Model:
    def __init__(self, batch, heads, dim, vdim):
        self.shape = (batch, heads, dim, vdim)
        self.k = [[Head(dim) for _ in range(heads)] for _ in range(batch)]
        self.v = [[Head(vdim) for _ in range(heads)] for _ in range(batch)]
        self.marked = [[np.zeros(0, bool) for _ in range(heads)] for _ in range(batch)]

    def length(self, b):
        return len(self.marked[b][0])

    def append(self, key, value, counts=None):
        key, value = to_f16(key), to_f16(value)
        for b in range(self.shape[0]):
            n = key.shape[2] if counts is None else counts[b]
            for h in range(self.shape[1]):
                k, v = key[b, h, :n].copy(), value[b, h, :n].copy()
                bad = ~(np.isfinite(k).all(-1) & np.isfinite(v).all(-1))
                k[bad] = 0
                v[bad] = 0
                self.k[b][h].append(k)
                self.v[b][h].append(v)
                self.marked[b][h] = np.concatenate([self.marked[b][h], bad])

    def truncate(self, lengths):
        for b in range(self.shape[0]):
            for h in range(self.shape[1]):
                self.k[b][h].truncate(lengths[b])
                self.v[b][h].truncate(lengths[b])
                self.marked[b][h] = self.marked[b][h][:lengths[b]]

    def read(self, dtype, rows, into_k, into_v):
        """The outputs of a read into copies of the given arrays."""
        out = []
        for heads, into in ((self.k, into_k), (self.v, into_v)):
            into = into.copy()
            for b in range(self.shape[0]):
                for h in range(self.shape[1]):
                    x = heads[b][h].f32()
                    x[self.marked[b][h]] = np.nan
                    into[b, h, :len(x)] = x.astype(dtype)
            out.append(into)
        return out

    def evict(self, weights, first, recent, keep):
        """(the target's model, kept indices per [b][h])."""
        batch, heads, dim, vdim = self.shape
        new = Model(batch, heads, dim, vdim)
        kept = [[None] * heads for _ in range(batch)]
        for b in range(batch):
            n = self.length(b)
            for h in range(heads):
                if n <= keep:
                    index = np.arange(n)
                else:
                    middle = np.arange(first, n - recent)
                    want = keep - first - recent
                    if weights is None:
                        picked = middle[len(middle) - want:]
                    else:
                        w = weights[b, h, middle].astype(np.float64)
                        order = sorted(range(len(middle)), key=lambda i: (np.isnan(w[i]), -w[i] if w[i] == w[i] else 0, i))
                        picked = np.sort(middle[order[:want]])
                    index = np.concatenate([np.arange(first), picked, np.arange(n - recent, n)]).astype(np.int64)
                kept[b][h] = index
                new.k[b][h] = self.k[b][h].hold_anew(self.k[b][h].held()[index])
                new.v[b][h] = self.v[b][h].hold_anew(self.v[b][h].held()[index])
                new.marked[b][h] = self.marked[b][h][index]
        return new, kept

    def attention(self, q, scale, causal, counts=None):
        """(out, tolerance, weights, weights' tolerance), all f64; padded rows NaN
        in `out` and to be compared apart.

        Tolerances, from the roundings that the kernels make (u = 2^-24):
          scores   s = sum of dim products: each add rounds, and the f32 q's pieces, the
                   block factor and the scaling round: at most (dim + 16) u times
                   A = scale * sum |q k|; it enters p = exp(s - max) as a relative
                   error, for the row's own p and for its sum;
          f16      P is rounded to f16, 2^-11 relative, in the product and in the
                   sum, or by 2^-25 absolute, P's largest being 2^4 to 2^12 times
                   a value scale down to 2^-3 of the unit (2^-26); the output is
                   rounded, 2^-11;
          f32      P is a pair (2^-22, or 2^-25 absolute with its largest 2^12 and
                   the same 2^-3: 2^-34), the output 2^-24;
          sums     over T keys in f32: at most T u each, for values and for P."""
        batch, heads, dim, vdim = self.shape
        hq, n = q.shape[1], q.shape[2]
        half = q.dtype == np.float16
        q = q.astype(np.float64)
        u = 2.0 ** -24
        out = np.full((batch, hq, n, vdim), np.nan)
        tol = np.zeros(out.shape)
        longest = max(self.length(b) for b in range(batch))
        weights, wtol = np.zeros((batch, heads, longest)), np.zeros((batch, heads, longest))
        for b in range(batch):
            count, length = n if counts is None else counts[b], self.length(b)
            i = np.arange(count)
            seen = np.maximum(length - count + i + 1, 0) if causal else np.full(count, length)
            hidden = np.arange(length)[None, :] >= seen[:, None]
            for j in range(hq):
                h = j // (hq // heads)
                k, v = self.k[b][h].held(), self.v[b][h].held()
                with np.errstate(invalid="ignore", over="ignore"):
                    s = q[b, j, :count] @ k.T * scale
                    size = np.where(hidden, 0.0, np.abs(q[b, j, :count]) @ np.abs(k).T * abs(scale))
                s[:, self.marked[b][h]] = np.nan
                s[hidden] = -np.inf
                has_nan = np.isnan(s).any(-1)
                top = np.where(np.isnan(s), -np.inf, s).max(-1, initial=-np.inf)
                zero = ~np.isfinite(top)
                plain = ~zero & ~has_nan
                out[b, j, :count][zero] = 0.0
                if not plain.any():
                    continue
                s, big_a, n_seen = s[plain], size[plain].max(-1)[:, None], seen[plain][:, None]
                p = np.exp(s - top[plain][:, None])
                total = p.sum(-1, keepdims=True)
                p /= total
                o, mass = p @ v, p @ np.abs(v)
                out[b, j, :count][plain] = o
                in_sight = np.cumsum(np.abs(v), axis=0)[seen[plain] - 1]
                rel = 2 * (dim + 16) * u * (big_a + 1) + 2 * n_seen * u
                if half:
                    t = (rel + 2.0 ** -10) * mass + 2.0 ** -11 * np.abs(o) \
                        + 2.0 ** -26 * (in_sight + n_seen * np.abs(o)) / total + 2.0 ** -24
                else:
                    t = (rel + 2.0 ** -21) * mass + 4 * u * np.abs(o) + 2.0 ** -34 * in_sight / total + 1e-40
                tol[b, j, :count][plain] = t
                weights[b, h, :length] += p.sum(0)
                w = rel + 16 * u   # (f16 too: these go by the sum before P's rounding)
                wtol[b, h, :length] += (w * p).sum(0)
        return out, tol, weights, wtol
