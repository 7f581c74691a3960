"""CPU restatement, in 64 bits, of the decoding operators: beam selection and the paged 8-bit key/value cache with its
attention.  Test infrastructure only."""
from __future__ import annotations

import math

import numpy as np

PAGE = 64
EXP_MIN, EXP_MAX = -64, 119


def select(logits, scores, eos=-1):
    """logits [B, K, V], scores [B, K] -> (scores, tokens, parents) of the K that go on, and of the best 2K.  Values that are equal
    in 64 bits: the lowest beam first, within a beam the largest logit (values that differ by less than 64 bits tell are equal,
    their logits are not), then the lowest word."""
    x = np.asarray(logits, np.float64)
    s = np.asarray(scores, np.float64)
    B, K, V = x.shape
    out = [np.zeros((B, n), t) for n in (K, 2 * K) for t in (np.float64, np.int64, np.int64)]
    for b in range(B):
        value, logit = np.full((K, V), -np.inf), np.zeros((K, V))
        for k in range(K):
            top = x[b, k].max()
            if np.isfinite(top) and np.isfinite(s[b, k]) and not np.isnan(x[b, k]).any():
                value[k] = s[b, k] + (x[b, k] - (top + math.log(np.exp(x[b, k] - top).sum())))
                logit[k] = x[b, k]
        flat = value.reshape(-1)
        order = np.lexsort((-logit.reshape(-1), np.repeat(np.arange(K), V), -flat))[:2 * K]  # stable: then by word
        go = [i for i in order if i % V != eos][:K]
        for j, picks in ((0, go), (3, order)):
            out[j][b], out[j + 1][b], out[j + 2][b] = flat[picks], [i % V for i in picks], [i // V for i in picks]
    return tuple(out)


def round_e4m3(x):
    """Nearest e4m3 value, ties to even, saturating at 448; NaN for what is not finite."""
    x = np.asarray(x, np.float64)
    mag = np.minimum(np.abs(x), 448.0)
    with np.errstate(divide="ignore", invalid="ignore"):
        step = np.exp2(np.maximum(np.floor(np.log2(mag)), -6) - 3)
        q = np.where(mag > 0, np.rint(mag / step) * step, 0.0)
    return np.where(np.isfinite(x), np.copysign(q, x), np.nan)


def exponent(x):
    """Smallest e with max|x| <= 448 * 2**e over the finite x, clamped."""
    x = np.abs(np.asarray(x, np.float64))
    x = x[np.isfinite(x)]
    most = x.max() if x.size else 0.0
    if most == 0:
        return EXP_MIN
    part, e = math.frexp(most)
    return min(EXP_MAX, max(EXP_MIN, e - 9 + (part > 0.875)))


class Cache:
    """Every page is a list of up to 64 rows per layer, head and tensor, with its exponent."""

    def __init__(self, num_seqs, max_len, kv_heads, head_dim, num_layers=1, num_pages=None):
        self.M = -(-max_len // PAGE)
        self.P = num_seqs * self.M if num_pages is None else num_pages
        self.H, self.D, self.L, self.S = kv_heads, head_dim, num_layers, num_seqs
        self.table = np.full((num_seqs, self.M), -1, np.int64)
        self.lens, self.starts = np.zeros(num_seqs, np.int64), np.zeros(num_seqs, np.int64)
        self.data = np.zeros((num_layers, self.P, kv_heads, 2, PAGE, head_dim))
        self.exps = np.zeros((num_layers, self.P, kv_heads, 2), np.int64)
        self.status = 0

    @property
    def refs(self):
        return np.bincount(self.table[self.table >= 0], minlength=self.P)

    def extend(self, n, every=1):
        slots = np.arange(0, self.S, every)
        n = np.broadcast_to(np.asarray(n), slots.shape)
        refs = self.refs
        bad = (4 if (n < 0).any() else 0) | (2 if (self.lens[slots] + n > self.M * PAGE).any() else 0)
        plan = []
        if not bad:
            free = [p for p in range(self.P) if refs[p] == 0]
            opened = {}
            for s, c in zip(slots, n):
                if c > 0 and self.lens[s] % PAGE:
                    opened.setdefault(self.table[s, self.lens[s] // PAGE], []).append(s)
            for s, c in zip(slots, n):
                at = self.lens[s] // PAGE
                if c > 0 and self.lens[s] % PAGE:
                    page = self.table[s, at]
                    if refs[page] > 1 and not (len(opened[page]) == refs[page] and opened[page][0] == s):
                        plan.append((s, at, page))
                for j in range(-(-self.lens[s] // PAGE), -(-(self.lens[s] + c) // PAGE)):
                    plan.append((s, j, None))
            if len(plan) > len(free):
                bad = 1
        self.starts[slots] = self.lens[slots]
        self.status |= bad
        if bad:
            return
        for (s, j, source), page in zip(plan, free):
            if source is not None:
                self.data[:, page], self.exps[:, page] = self.data[:, source], self.exps[:, source]
            self.table[s, j] = page
        self.lens[slots] += n

    def reorder(self, parents):
        parents = np.asarray(parents)
        B, K = parents.shape
        table, lens = self.table.copy(), self.lens.copy()
        for b in range(B):
            for k in range(K):
                p, s = parents[b, k], b * K + k
                if p == -1:
                    self.table[s], self.lens[s] = -1, 0
                elif 0 <= p < K:
                    self.table[s], self.lens[s] = table[b * K + p], lens[b * K + p]
                else:
                    self.status |= 8
        self.starts = self.lens.copy()

    def compact(self):
        used = np.flatnonzero(self.refs > 0)
        n = len(used)
        name = np.arange(self.P)
        high = used[used >= n]
        holes = np.setdiff1d(np.arange(n), used)
        name[high] = holes
        self.data[:, holes], self.exps[:, holes] = self.data[:, high], self.exps[:, high]
        self.table = np.where(self.table >= 0, name[self.table], -1)
        return n

    def write(self, k, v, layer=0, every=1):
        for i, s in enumerate(range(0, self.S, every)):
            end = min(self.lens[s], self.starts[s] + k.shape[1])
            for w, x in ((0, k), (1, v)):
                for h in range(self.H):
                    at = self.starts[s]
                    while at < end:
                        j, t0 = at // PAGE, at % PAGE
                        t1 = min(PAGE, t0 + end - at)
                        rows = np.asarray(x[i, at - self.starts[s]:at - self.starts[s] + t1 - t0, h], np.float64)
                        page = self.table[s, j]
                        held = self.data[layer, page, h, w]
                        e = exponent(rows)
                        if t0:
                            old = self.exps[layer, page, h, w]
                            e = max(e, old)
                            held[:t0] = round_e4m3(held[:t0] * 2.0 ** -float(e)) * 2.0 ** float(e)
                        held[t0:t1] = round_e4m3(rows * 2.0 ** -float(e)) * 2.0 ** float(e)
                        self.exps[layer, page, h, w] = e
                        at += t1 - t0

    def tokens(self, s, layer, h, w):
        """[lens[s], D]: what is held of a sequence."""
        n = self.lens[s]
        pages = self.table[s, :-(-n // PAGE)]
        return self.data[layer, pages, h, w].reshape(-1, self.D)[:n]

    def read(self, first, count, layer, every=1):
        slots = list(range(0, self.S, every))
        first = np.broadcast_to(np.asarray(first), (len(slots),))
        out = np.zeros((2, len(slots), count, self.H, self.D))
        for i, s in enumerate(slots):
            for h in range(self.H):
                for w in range(2):
                    x = self.tokens(s, layer, h, w)[first[i]:first[i] + count]
                    out[w, i, :len(x), h] = x
        return out[0], out[1]

    def attend(self, q, layer=0, scale=None, every=1, magnitude=False):
        """``magnitude``: of the values' magnitudes instead, sum p |v| / sum p, which the rounding of p is relative to."""
        q = np.asarray(q, np.float64)
        S, n, heads, D = q.shape
        scale = D ** -0.5 if scale is None else scale
        out = np.zeros(q.shape)
        for i, s in enumerate(range(0, self.S, every)):
            for j in range(heads):
                h = j // (heads // self.H)
                k, v = self.tokens(s, layer, h, 0), self.tokens(s, layer, h, 1)
                v = np.abs(v) if magnitude else v
                for r in range(min(n, self.lens[s] - self.starts[s])):
                    t = self.starts[s] + r + 1
                    a = scale * (k[:t] @ q[i, r, j])
                    p = np.exp(a - a.max())
                    out[i, r, j] = p @ v[:t] / p.sum()
        return out
