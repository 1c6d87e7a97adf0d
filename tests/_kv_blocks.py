"""The block-scaled cache and the batch tables restated in numpy (float64
where values are computed), for the tests of their kernels."""
from __future__ import annotations

import numpy as np

INT8, FP8 = 0, 1
QMAX = {INT8: 127.0, FP8: 448.0}


def places(bs, D):
    """Byte of (token, dim) inside a (block, head): K layout, V layout."""
    k, v = np.zeros((bs, D), np.int64), np.zeros((bs, D), np.int64)
    E = D // 16
    for t in range(bs):
        base, w = t // 16 * 16 * D, t % 16
        for d in range(D):
            h, r = divmod(d, D // 2)
            k[t, d] = base + (r // 8) * 256 + w * 16 + h * 8 + r % 8
            m, u = divmod(d, E)
            v[t, d] = base + (u // 4) * 1024 + (w // 4) * 256 + m * 16 + (u % 4) * 4 + w % 4
    return k, v


def e4m3_values():
    out = np.zeros(256)
    for b in range(256):
        s, e, m = b >> 7, (b >> 3) & 15, b & 7
        x = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out[b] = np.nan if e == 15 and m == 7 else (-x if s else x)
    return out


E4M3 = e4m3_values()


def values(codes, fmt):
    """float64 values of raw codes (any shape, uint8 bytes)."""
    codes = np.asarray(codes).view(np.uint8)
    return E4M3[codes] if fmt == FP8 else codes.view(np.int8).astype(np.float64)


def scale_for(amax, fmt):
    if amax == 0:
        return 0.0
    amax, s = min(amax, 65504.0), 2.0 ** -24
    while amax > QMAX[fmt] * s:
        s *= 2
    return s


_E4M3_POS = E4M3[:127]  # ascending, code = index


def nearest(y, fmt):
    """The code value nearest to y, ties to the even code."""
    y = np.asarray(y, np.float64)
    if fmt == INT8:
        return np.rint(y)
    a = np.abs(y)
    i = np.clip(np.searchsorted(_E4M3_POS, a), 1, 126)
    lo, hi = _E4M3_POS[i - 1], _E4M3_POS[i]
    pick_hi = (a - lo > hi - a) | ((a - lo == hi - a) & (i % 2 == 0))
    return np.copysign(np.where(pick_hi, hi, lo), y)


def limit(s, fmt):
    return (63.0 if s >= 1024 else 127.0) if fmt == INT8 else (240.0 if s >= 256 else 448.0)


def bytes_of(vals, fmt):
    """Raw bytes of code values."""
    vals = np.asarray(vals, np.float64)
    if fmt == INT8:
        return vals.astype(np.int8).view(np.uint8)
    return np.where(np.signbit(vals), 128, 0).astype(np.uint8) | np.searchsorted(_E4M3_POS, np.abs(vals)).astype(np.uint8)


class Cache:
    """Codes [nb, hkv, bs, D] (raw bytes, logical order) and scales of K and V."""

    def __init__(self, nb, hkv, bs, D, fmt):
        self.nb, self.hkv, self.bs, self.D, self.fmt = nb, hkv, bs, D, fmt
        self.codes = [np.zeros((nb, hkv, bs, D), np.uint8) for _ in "kv"]
        self.scale = [np.zeros((nb, hkv)) for _ in "kv"]

    def fill(self, rng, lo=-6, hi=-3):
        """Random finite codes, scales 2^lo .. 2^hi."""
        for c, s in zip(self.codes, self.scale):
            b = rng.integers(0, 256, c.shape, dtype=np.uint8)
            if self.fmt == FP8:
                b[(b & 127) == 127] = 8
            else:
                b[b == 128] = 0
            c[...] = b
            s[...] = 2.0 ** rng.integers(lo, hi + 1, s.shape)

    def raw(self):
        """K and V bytes in the kernels' layout [nb, hkv, bs * D]."""
        out = []
        for c, p in zip(self.codes, places(self.bs, self.D)):
            r = np.zeros((self.nb, self.hkv, self.bs * self.D), np.uint8)
            r[:, :, p.reshape(-1)] = c.reshape(self.nb, self.hkv, -1)
            out.append(r)
        return out

    def stored(self, which, blk):
        """float64 [hkv, bs, D] of a block."""
        return values(self.codes[which][blk], self.fmt) * self.scale[which][blk][:, None, None]

    def write_run(self, rows, blk, off):
        """rows = (k, v) float64 [n, hkv, D] at offsets off .. of block blk."""
        for which, x in enumerate(rows):
            for h in range(self.hkv):
                r = x[:, h]
                old = self.scale[which][blk, h] if off > 0 else 0.0
                s = max(old, scale_for(np.max(np.abs(r)), self.fmt))
                c = self.codes[which][blk, h]
                if s > old and off > 0:
                    c[:off] = bytes_of(nearest(values(c[:off], self.fmt) * (old / s), self.fmt), self.fmt)
                lim = limit(s, self.fmt)
                y = r if s == 0 else np.clip(r / s, -lim, lim)  # zeros of either sign keep it
                c[off:off + len(r)] = bytes_of(nearest(y, self.fmt), self.fmt)
                self.scale[which][blk, h] = s


def rotate(qkv, bias, pos, hq, hkv, D, cos, sin):
    """(q fp16 [T, hq, D], k, v fp16 [T, hkv, D]) in fp32 without contraction."""
    T = qkv.shape[0]
    x = qkv if bias is None else (qkv.astype(np.float32) + bias.astype(np.float32)).astype(np.float16)
    x = x.astype(np.float32).reshape(T, hq + 2 * hkv, D)
    c, s = cos[pos][:, None], sin[pos][:, None]
    a, b = x[:, :hq + hkv, :D // 2], x[:, :hq + hkv, D // 2:]
    with np.errstate(invalid="ignore", over="ignore"):
        r = np.concatenate([a * c - b * s, b * c + a * s], -1).astype(np.float16)
    return r[:, :hq], r[:, hq:], x[:, hq + hkv:].astype(np.float16)


def runs(slots, bs, nb):
    """[(first row, n, block, offset)] of a call's slots."""
    out, t = [], 0
    while t < len(slots):
        if slots[t] < 0 or slots[t] // bs >= nb:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t + n - 1] + 1 and slots[t + n] % bs != 0:
            n += 1
        out.append((t, n, slots[t] // bs, slots[t] % bs))
        t += n
    return out


def write(cache, qkv, bias, pos, slots, hq, cos, sin):
    """The operator: cache updated, q (fp16) returned."""
    q, k, v = rotate(qkv, bias, pos, hq, cache.hkv, cache.D, cos, sin)
    for t, n, blk, off in runs(slots, cache.bs, cache.nb):
        cache.write_run((k[t:t + n].astype(np.float64), v[t:t + n].astype(np.float64)), blk, off)
    return q


def attention(cache, table, q, scale, keys):
    """float64 attention of query rows q [n, hq, D] over the first keys[i] keys of
    a table; returns (out, bound): bound is the largest error that the kernels'
    roundings allow:
      fp16 output            2^-11 |o|, and half its subnormal spacing, 2^-25
      fp16 probabilities     2^-11 sum p|v|, and for those below fp16's normal
                             range 2^-25 a key relative to the largest, of values
                             up to twice the largest |v|
      fp32 scores            an error d of a score changes p by the factor
                             1 + d; at most D + 8 roundings of 2^-24, of the sum
                             of |products|, on either side of the maximum
    """
    hq, D = q.shape[1:]
    G, bs = hq // cache.hkv, cache.bs
    out = np.zeros(q.shape)
    bound = np.full(q.shape, 2.0 ** -25)
    ids = [b if 0 <= b < cache.nb else 0 for b in table]
    most = min(max(keys), len(table) * bs) if len(keys) else 0
    if most <= 0:
        return out, bound
    need = -(-most // bs)
    k = np.concatenate([cache.stored(0, b) for b in ids[:need]], 1)
    v = np.concatenate([cache.stored(1, b) for b in ids[:need]], 1)
    for i in range(len(q)):
        n = min(keys[i], len(table) * bs)
        if n <= 0:
            continue
        for h in range(hq):
            kk, vv, x = k[h // G, :n], v[h // G, :n], q[i, h].astype(np.float64)
            s = kk @ x * scale
            p = np.exp(s - s.max())
            L = p.sum()
            o = p @ vv / L
            a = p @ np.abs(vv) / L
            dev = 2 * (D + 8) * 2.0 ** -24 * abs(scale) * np.max(np.abs(kk) @ np.abs(x))
            out[i, h] = o
            bound[i, h] += 2.0 ** -11 * np.abs(o) + (2.0 ** -11 + 2 * dev + 2.0 ** -18) * a + \
                n * 2.0 ** -24 * np.max(np.abs(vv)) / L
    return out, bound


def tables(past, new, rows, bs, thr, table, ring, head, count):
    """build_batch_tables, one sequence after another.  table and ring are
    updated; returns the outputs in a dict."""
    S, mb, cap = len(past), table.shape[1], len(ring)
    o = {n: np.zeros(S, np.int32) for n in ("q_start", "q_len", "ctx_len")}
    o |= {"positions": np.zeros(rows, np.int32), "slot_mapping": np.full(rows, -1, np.int32),
          "decode_token": np.full(rows, -1, np.int32), "decode_seq": np.zeros(rows, np.int32),
          "prefill_seq": np.full(S, -1, np.int32)}
    at = asked = taken = nd = npf = refused = 0
    back = []
    for s in range(S):
        p, n = int(past[s]), max(int(new[s]), 0)
        o["q_start"][s] = min(at, 1 << 30)
        have, want = -(-max(p, 0) // bs), -(-(max(p, 0) + n) // bs)
        if new[s] < 0:
            back += [int(x) for x in table[s, :min(have, mb)]]
        elif n > 0:
            fits = p >= 0 and want <= mb and at + n <= rows
            need = want - have
            asked += need if fits else 0
            if fits and (need == 0 or asked <= count):
                o["q_len"][s], o["ctx_len"][s] = n, p + n
                for b in range(have, want):
                    table[s, b] = ring[(head + taken) % cap]
                    taken += 1
                for i in range(n):
                    o["positions"][at + i] = p + i
                    o["slot_mapping"][at + i] = table[s, (p + i) // bs] * bs + (p + i) % bs
                if n <= thr:
                    for i in range(n):
                        o["decode_token"][nd], o["decode_seq"][nd] = at + i, s
                        nd += 1
                else:
                    o["prefill_seq"][npf] = s
                    npf += 1
            else:
                refused += 1
                o["ctx_len"][s] = p
            at += n
        else:
            o["ctx_len"][s] = p
    for i, b in enumerate(back):
        ring[(head + count + i) % cap] = b
    o["counts"] = np.array([min(at, 1 << 30), nd, npf, refused], np.int32)
    o["state"] = np.array([(head + taken) % cap, count - taken + len(back)], np.int32)
    return o
