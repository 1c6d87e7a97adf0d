"""Rows whose top-p border is a rounding: writes sampling_borders.npz.

In each row the weights of the first n tokens make half of the whole but for an ulp: with
top_p = 0.5 the target lies between the two sums that sample_tokens forms of them, the scan
over the bins (which reaches it) and the bin's start plus its tokens' weights (which does
not).  Found by a model of both sums in exact arithmetic.  `python make_sampling_borders.py`.
"""
import math
from fractions import Fraction as F
from pathlib import Path

import numpy as np

C = 8 / math.log(2)  # bins of a natural logarithm, T = 1
POLY = [699.1093111382294, 38597.3698262215, 1783466.322640276, 61751342.16030201, 1425413776.8902755,
        4503599627370496.0 + 16451499093.0]
BINS, WAVE = 384, 64


def fma(a, b, c):
    return float(F(a) * F(b) + F(c))


def weight(x):
    """(bin, whole-number weight) of a logit."""
    b = math.floor(x * C)
    f = fma(x, C, -float(b))
    y = fma(f, POLY[0], POLY[1])
    for c in POLY[2:]:
        y = fma(y, f, c)
    return b, int(F(y) - 2 ** 52)


def scale(j):
    s = (0.91700404320467123 if j & 1 else 1.0) * (0.84089641525371454 if j & 2 else 1.0)
    return math.ldexp(s * (0.70710678118654752 if j & 4 else 1.0), -(j >> 3) - 34)


SCALES = [scale(j) for j in range(BINS)]


def scan(w):
    """Mass before each bin, and of all: in a wave by doubling steps, waves in turn."""
    waves = []
    for v in range(0, BINS, WAVE):
        ws, ss = w[v:v + WAVE], SCALES[v:v + WAVE]
        m = [float(F(a) * F(s)) for a, s in zip(ws, ss)]
        m = [m[0]] + [fma(ws[i], ss[i], m[i - 1]) for i in range(1, WAVE)]
        step = 2
        while step < WAVE:
            m = [m[i] + m[i - step] if i >= step else m[i] for i in range(WAVE)]
            step *= 2
        waves.append(m)
    out = [0.0]
    for v, m in enumerate(waves):
        before = 0.0
        for x in waves[:v]:
            before += x[-1]
        out += [before + x for x in m]
    return out


def histogram(row):
    first, w = weight(float(max(row)))[0], [0] * BINS
    for x in row:
        b, y = weight(float(x))
        if first - b < BINS:
            w[first - b] += y
    return w


def both_sums(row, bin):
    w = histogram(row)
    m = scan(w)
    return m[bin], m[bin + 1], fma(w[bin], SCALES[bin], m[bin]), m[BINS]


def find(rng, n):
    head = np.float32(np.sort(-rng.random(n) * 2.4)[::-1])
    head[0] = 0
    bin = -weight(float(head[-1]))[0]
    _, up_to, fine, _ = both_sums(head, bin)
    if not fine < up_to:
        return None
    rest = 2 * F(up_to) - sum(F(a) * F(s) for a, s in zip(histogram(head), SCALES))
    tail = []
    while rest > F(2) ** -44:
        x = np.float32(min(head[-1] - 0.2, math.log(float(rest)) - 0.3 * rng.random() - 0.01))
        b, y = weight(float(x))
        if F(y) * F(SCALES[-b]) <= rest:
            tail.append(x)
            rest -= F(y) * F(SCALES[-b])
    if rest > F(2) ** -60:
        tail.append(np.float32(math.log(float(rest))))
    row = np.concatenate([head, np.float32(tail)])
    before, up_to, fine, all_of = both_sums(row, bin)
    return row if before < fine < 0.5 * all_of <= up_to else None


def main():
    rng, rows, heads = np.random.default_rng(0), [], []
    for n in [128, 128, 127, 64, 65, 20] + list(range(30, 125, 9)):
        row = None
        while row is None:
            row = find(rng, n)
        rows.append(row)
        heads.append(n)
    out = np.full((len(rows), max(map(len, rows))), -np.inf, np.float32)
    for o, r in zip(out, rows):
        o[:len(r)] = r
    np.savez_compressed(Path(__file__).with_name("sampling_borders.npz"), rows=out, heads=np.int32(heads))


if __name__ == "__main__":
    main()
