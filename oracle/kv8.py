"""The paged 8-bit K/V cache in numpy, from its definition (include/decide_cuda.h, dc_kv8_*): loops over sequences, pages and heads, float64
throughout, codes by table lookup. Test infrastructure; shares nothing with the kernels."""
from __future__ import annotations

import math

import numpy as np

NO_KEYS = 0xFFFFFFFF


class Violation(Exception):
    """What the device reports through the status word."""


def _decode_table() -> np.ndarray:
    t = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = (8 + m) * 2.0 ** (e - 10) if e else m * 2.0 ** -9
        if c & 127 == 127:
            x = math.nan
        t[c] = -x if c & 128 else x
    return t


DECODE = _decode_table()


def encode(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3 code of |x| <= 448, ties to the even code; the sign of zero is kept."""
    size = np.abs(x)
    up = np.searchsorted(DECODE[:127], size)            # least code whose value is >= size
    up = np.minimum(up, 126)
    down = np.maximum(up - 1, 0)
    over, under = DECODE[up] - size, size - DECODE[down]
    code = np.where(over < under, up, np.where(under < over, down, np.where(up % 2 == 0, up, down)))
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def scale_for(amax: float) -> float:
    """Least power of two, 2^-60 or more, with 448 * scale >= amax."""
    s = 2.0 ** -60
    while 448 * s < amax:
        s *= 2
    return s


class Cache:
    """k, v: uint8 codes [layers, n_pages, nkv, page, hd]; scales [layers, n_pages, nkv] float64; table, lens, refs as Python ints."""

    def __init__(self, layers, n_pages, nkv, hd, n_seqs, max_pages, page):
        self.k, self.v = (np.zeros((layers, n_pages, nkv, page, hd), np.uint8) for _ in range(2))
        self.k_scale, self.v_scale = (np.full((layers, n_pages, nkv), 2.0 ** -60) for _ in range(2))
        self.table = np.zeros((n_seqs, max_pages), np.int64)
        self.lens, self.refs = np.zeros(n_seqs, np.int64), np.zeros(n_pages, np.int64)
        self.page, self.max_pages, self.n_pages = page, max_pages, n_pages

    def pages(self, length):
        return -(-int(length) // self.page)

    def held(self, j):
        if self.lens[j] > self.max_pages * self.page:
            raise Violation("length")
        ids = self.table[j, :self.pages(self.lens[j])]
        if (ids >= self.n_pages).any() or (ids < 0).any():
            raise Violation("page")
        return ids

    def _take(self, count):
        free = np.flatnonzero(self.refs == 0)
        if len(free) < count:
            raise Violation("pool")
        self.refs[free[:count]] = 1
        return free[:count]

    def extend(self, add):
        if any(n + a > self.max_pages * self.page for n, a in zip(self.lens, add)):
            raise Violation("length")
        if sum(self.pages(n + a) - self.pages(n) for n, a in zip(self.lens, add)) > (self.refs == 0).sum():
            raise Violation("pool")
        for j, a in enumerate(add):
            have, want = self.pages(self.lens[j]), self.pages(self.lens[j] + a)
            self.table[j, have:want] = self._take(want - have)
            self.lens[j] += a

    def fork(self, src, dst, deep):
        n_seqs = len(self.lens)
        if any(not 0 <= s < n_seqs for s in [*src, *dst]) or len(set(dst)) < len(dst) or set(src) & set(dst):
            raise Violation("sequence")
        for s in [*src, *dst]:
            self.held(s)
        refs = self.refs.copy()
        for d in dst:
            np.subtract.at(refs, self.held(d), 1)
        if (refs < 0).any():
            raise Violation("refs")
        copied = [self.pages(self.lens[s]) if deep else int(self.lens[s] % self.page != 0) for s in src]
        if sum(copied) > (refs == 0).sum():
            raise Violation("pool")
        self.refs = refs
        ids = [self._take(c) for c in copied]       # all of them before the sharing below, in the order of the forks
        for s, d, new, c in zip(src, dst, ids, copied):
            old = self.held(s)
            shared = len(old) - c
            np.add.at(self.refs, old[:shared], 1)
            self.table[d, :len(old)] = np.concatenate([old[:shared], new])
            for o, p in zip(old[shared:], new):
                for a in (self.k, self.v, self.k_scale, self.v_scale):
                    a[:, p] = a[:, o]
            self.lens[d] = self.lens[s]

    def free(self, seqs):
        for j in seqs:
            if not 0 <= j < len(self.lens):
                raise Violation("sequence")
            for p in self.held(j):
                if self.refs[p] == 0:
                    raise Violation("refs")
                self.refs[p] -= 1
            self.lens[j] = 0

    def compact(self):
        used = self.refs > 0
        live = int(used.sum())
        src, dst = np.flatnonzero(used[live:]) + live, np.flatnonzero(~used[:live])
        where = np.arange(self.n_pages)
        for s, d in zip(src, dst):
            for a in (self.k, self.v, self.k_scale, self.v_scale):
                a[:, d] = a[:, s]
            self.refs[d], self.refs[s], where[s] = self.refs[s], 0, d
        for j in range(len(self.lens)):
            self.table[j, :self.pages(self.lens[j])] = where[self.held(j)]
        return live

    def append(self, layer, k, v, row_start):
        """k, v: float64 [rows, nkv, hd]."""
        for j in range(len(self.lens)):
            r0, r1 = row_start[j], row_start[j + 1]
            if r1 < r0 or r1 > len(k) or r1 - r0 > self.lens[j]:
                raise Violation("offsets")
            ids = self.held(j)
            begin = int(self.lens[j]) - (r1 - r0)
            for b in range(begin // self.page, len(ids)):
                lo, hi = max(begin, b * self.page), min(int(self.lens[j]), (b + 1) * self.page)
                if lo >= hi:
                    continue
                p, o = int(ids[b]), lo - b * self.page
                if self.refs[p] != 1:
                    raise Violation("shared")
                for codes, scales, new in ((self.k, self.k_scale, k), (self.v, self.v_scale, v)):
                    for h in range(codes.shape[2]):
                        x = new[r0 + lo - begin:r0 + hi - begin, h]
                        before = scales[layer, p, h] if o else 0.0
                        if not np.isfinite(x).all() or math.isnan(before):
                            scales[layer, p, h] = math.nan
                            codes[layer, p, h, o:o + hi - lo] = 0
                            continue
                        scale = max(before, scale_for(np.abs(x).max()))
                        if o and scale > before:
                            codes[layer, p, h, :o] = encode(DECODE[codes[layer, p, h, :o]] * before / scale)
                        codes[layer, p, h, o:o + hi - lo] = encode(x / scale)
                        scales[layer, p, h] = scale

    def tokens(self, layer, j, head, codes, scales):
        """The sequence's values [len, hd], the scales of its tokens, and the codes' values."""
        ids = self.held(j)
        n = int(self.lens[j])
        c = DECODE[codes[layer, ids, head]].reshape(-1, codes.shape[-1])[:n]
        s = np.repeat(scales[layer, ids, head], self.page)[:n]
        return c, s

    def attention(self, layer, q, gate, q_start, qpos, half_step, bf16, weight=2 * 2.0 ** -11, least=2.0 ** -25):
        """Returns (y, tolerance) [rows, nq * hd] in float64; NaN rows where a scale that is attended is NaN.

        The tolerance is what the kernel's arithmetic may be off by, term by term:
          scores: products are exact, the fp32 sum of hd of them is off by at most 2^-22 sum |q k| for each of its hd / 16 + 2 steps,
            and the argument of the exponential by 2^-22 of its size (in log2 units) twice;
          the exponential itself by 2^-22, each join of two partial sums by 2^-23 (32 of them are plenty), so a weight is off by a factor
            1 + w, and numerator and denominator each by as much;
          weights in fp16: off by 2^-11 in the product, and in the total at most as much (`weight`: both together); small ones by `least` of the row's
            largest term in absolute size in the product;
          bf16 queries: elements under 2^-28 of the row's largest are off by 2^-39 of it;
          the gate's sigmoid by 2^-20; the output by half a step of its type (`half_step` of its size; fp16 below 2^-14: 2^-25)."""
        rows, nq = q.shape[0], q.shape[1]
        hd, nkv = self.k.shape[-1], self.k.shape[2]
        y, tol = np.zeros((rows, nq * hd)), np.zeros((rows, nq * hd))
        for j in range(len(self.lens)):
            n = int(self.lens[j])
            count = q_start[j + 1] - q_start[j]
            for h in range(nq):
                kc, ks = self.tokens(layer, j, h // (nq // nkv), self.k, self.k_scale)
                vc, vs = self.tokens(layer, j, h // (nq // nkv), self.v, self.v_scale)
                for i in range(count):
                    r = q_start[j] + i
                    pos = n - count + i if qpos is None else int(qpos[r])
                    see = 0 if pos == NO_KEYS or n == 0 or pos < 0 else min(pos, n - 1) + 1
                    if see == 0:
                        continue
                    k, v = kc[:see] * ks[:see, None], vc[:see] * vs[:see, None]
                    cols = slice(h * hd, (h + 1) * hd)
                    s = k @ q[r, h] * hd ** -0.5
                    if np.isnan(s).any() or np.isnan(vs[:see]).any():
                        y[r, cols], tol[r, cols] = math.nan, 0
                        continue
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out = p @ v
                    size = np.abs(k) @ np.abs(q[r, h]) * hd ** -0.5
                    arg = np.abs(s) / math.log(2) + np.abs(np.log2(vs[:see]))
                    w = ((hd / 16 + 2) * 2.0 ** -22 * size.max() + 2 * 2.0 ** -22 * 2 * arg.max() * math.log(2) + 2.0 ** -22 + 32 * 2.0 ** -23)
                    if bf16:
                        w += 2.0 ** -39 * np.abs(q[r, h]).max() * np.abs(k).sum(1).max() * hd ** -0.5
                    mass = p @ np.abs(v)
                    t = (2 * w + weight) * mass + least * (p * vs[:see]).max() * np.abs(vc[:see]).sum(0)
                    if gate is not None:
                        g = 1 / (1 + np.exp(-gate[r, cols]))
                        out, t = out * g, t * g + 2.0 ** -20 * np.abs(out) * g
                    y[r, cols], tol[r, cols] = out, t + half_step * (np.abs(out) + t) + 2.0 ** -25
        return y, tol
