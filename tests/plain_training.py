"""Plain restatements, in numpy with at least 64 bits, of the operators at the two ends of a training step: log probabilities with entropies and
alternatives, and norms of gradients; with bounds on how far a rounded computation may be off."""
import numpy as np

NAN, INF = float("nan"), float("inf")


def wide(kind):
    return np.float64 if kind == np.float32 else np.longdouble


class Rows(object):
    """Everything about logits as rows [positions, classes] of float32 or float64.

    Bounds count halves of the type's eps (`unit`), for sums whose longest chain of additions is `chain`: d = x - m is off by |d|; exp(d) by that,
    relatively, and four more (two units in the last place); S by the mean of these over p, which is D1 = sum p |d|, and chain; T alike with
    e d for e, which the error of d changes by a relative |d| + 1; a logarithm by its argument's and four of its own."""

    def __init__(self, x, labels=None, top_k=0, chain=64):
        kind = x.dtype
        self.unit = np.finfo(kind).eps / 2
        self.x, self.labels, self.top_k = x, labels, top_k
        n, k = x.shape
        w = wide(kind)
        self.bad = ~(x < INF).all(1)                                       # a NaN or an infinity
        self.nothing = (x == -INF).all(1)
        with np.errstate(invalid="ignore", over="ignore"):
            m = np.where(np.isnan(x), -INF, x).max(1, keepdims=True).astype(w)
            self.d = np.where((self.bad | self.nothing)[:, None], -INF, x.astype(w) - m)
            e = np.exp(self.d)
        s = np.where(self.nothing | self.bad, 1, e.sum(1))
        self.p = e / s[:, None]
        d0 = np.where(self.d == -INF, 0, self.d)
        self.log_s = np.log(s)
        self.l = self.d - self.log_s[:, None]
        self.entropy = self.log_s - (self.p * d0).sum(1)
        self.entropy[self.nothing], self.entropy[self.bad] = 0, NAN
        d1, d2 = (self.p * abs(d0)).sum(1), (self.p * d0 * d0).sum(1)
        off_s = chain + 6 + d1                                             # of S, relatively, and so of log S
        self.off_l = self.unit * (abs(d0) + abs(np.where(self.d == -INF, 0, self.l)) + (off_s + 4 * abs(self.log_s) + 4)[:, None])
        self.off_entropy = self.unit * (off_s + 4 * abs(self.log_s) + 4 + (d1 * (chain + 8) + d1 + d2) + d1 * off_s + abs(np.where(self.bad, 0, self.entropy)))
        v = np.where(np.isnan(x), -INF, x)
        order = np.argsort(-v, axis=1, kind="stable")[:, :top_k]
        chosen = np.take_along_axis(v, order, 1)
        self.top_index = np.where(chosen == -INF, -1, order).astype(np.int32)

    def _of(self, values, at, where, otherwise):
        got = np.take_along_axis(values, np.where(where, at, 0), 1)
        return np.where(where, got, otherwise)

    def label(self):
        """(log probabilities of the labels, bounds)"""
        at = self.labels[:, None]
        known = (at >= 0) & (at < self.x.shape[1])
        v = self._of(np.where(self.nothing[:, None], -INF, np.where(self.bad[:, None], NAN, self.l)), at, known, 0)
        return v[:, 0], self._of(self.off_l, at, known, 0)[:, 0]

    def top(self):
        some = self.top_index >= 0
        v = self._of(np.where(self.bad[:, None], NAN, self.l), self.top_index, some, -INF)
        return v, self._of(self.off_l, self.top_index, some, 0)

    def gradient(self, g_label=None, g_entropy=None, g_top=None):
        """(dlogits, bounds)"""
        n, k = self.x.shape
        up, size = np.zeros(self.p.shape, self.p.dtype), np.zeros(self.p.shape, self.p.dtype)
        rows = np.arange(n)
        if g_label is not None:
            known = (self.labels >= 0) & (self.labels < k)
            g = np.where(known, g_label, 0)
            np.add.at(up, (rows, np.where(known, self.labels, 0)), g)
            np.add.at(size, (rows, np.where(known, self.labels, 0)), abs(g))
        if g_top is not None:
            some = self.top_index >= 0
            np.add.at(up, (rows[:, None], np.where(some, self.top_index, 0)), np.where(some, g_top, 0))
            np.add.at(size, (rows[:, None], np.where(some, self.top_index, 0)), np.where(some, abs(g_top), 0))
            size_top = np.where(some, abs(g_top), 0).sum(1)
        taken = up.sum(1)
        size_taken = (abs(g) if g_label is not None else 0) + (size_top if g_top is not None else 0)
        ge = np.zeros(n, self.p.dtype) if g_entropy is None else g_entropy.astype(self.p.dtype)
        l = np.where(self.p > 0, self.l, 0)
        h = np.where(self.bad, 0, self.entropy)
        dx = up - self.p * (taken[:, None] + ge[:, None] * (l + h[:, None]))
        dx[self.nothing], dx[self.bad] = 0, NAN
        inner = np.reshape(size_taken, (-1, 1)) + abs(ge)[:, None] * (abs(l) + abs(h)[:, None])
        off = self.p * (inner * (self.off_l + (12 + self.top_k) * self.unit) + abs(ge)[:, None] * (self.off_l + self.off_entropy[:, None]))
        # (dx = (-p inner + g_label) + g_top: an addition is off by a unit of what it gives, which where label and alternative are one class is
        # up to p inner + |g_label| + |g_top| although their sum may be far less: label 5, -0.3539, as alternative 0.3001 of a position of ten)
        off = off + 2 * self.unit * (size + abs(np.where(np.isnan(dx), 0, dx)))
        # (what is below the normal numbers may be flushed)
        return dx, off + np.finfo(self.x.dtype).tiny * (1 + inner)


def norm(tensors, order=2):
    """The norm of all values of a list of arrays, in 80 bits (whose exponent takes squares of any float64)."""
    flat = np.concatenate([t.reshape(-1).astype(np.longdouble) for t in tensors] + [np.zeros(1, np.longdouble)])
    if np.isnan(flat).any():
        return np.longdouble(NAN)
    return abs(flat).max() if order == INF else np.sqrt((flat * flat).sum())


def clipped(tensors, limit, order=2):
    """(norm as it is returned, scaled tensors rounded once)"""
    kind = np.float64 if any(t.dtype == np.float64 for t in tensors) else np.float32
    with np.errstate(over="ignore"):
        n = norm(tensors, order).astype(kind)
    scale = np.longdouble(limit) / np.longdouble(n) if np.isfinite(n) and n > limit else np.longdouble(1)
    return n, [t if scale == 1 else (t.astype(np.longdouble) * scale).astype(t.dtype) for t in tensors]
