"""Decode attention over shared prefixes in an INT8 cache whose V scales differ widely: keys
without weight, keys that an item does not attend to and rows of zeros take no bits from the
values that an item does attend to."""
import numpy as np
import pytest

from tests._util import say
from tests.test_shared_prefix_gpu import U16, U32, Case, torch  # noqa: F401  (torch: the fixture)

pytestmark = pytest.mark.gpu
Q0 = 16.0  # dim 0 of every query head; of keys it is 0 but where a test sets a key's score by it
FORMS = {"tiles of 16": (2, [40, 9, 300]), "tiles of 128": (4, [30, 1, 70] + [5] * 33)}


class Scales(Case):
    """V rows of random codes and scales in [small, 2 small)."""

    def __init__(self, torch, form, D, cache, small, prefix=700, per=None, seed=1):  # noqa: F811
        per, own = per or FORMS[form][0], FORMS[form][1]
        super().__init__(torch, [(prefix, own), (None, [500])], 2 * per, 2, D, 16, cache, seed, amp=1.0)
        g = torch.Generator(device="cuda").manual_seed(seed)
        k, v, ks, vs = self.planes
        k[..., 0] = 0
        there = ~torch.isnan(vs.float())
        v.copy_(torch.randint(-127, 128, v.shape, generator=g, device="cuda").to(torch.int8))
        rand = small * (1 + torch.rand(vs.shape, generator=g, device="cuda"))
        vs.copy_(torch.where(there, rand.to(vs.dtype), vs))
        self.q[:, :self.hq * D].view(self.rows, self.hq, D)[..., 0] = Q0

    def cell(self, item, pos):
        """(block, row) of a key that the item attends to."""
        first = self.firsts[item]
        if first is not None and pos < self.prefix[np.searchsorted(self.starts, item, "right") - 1]:
            item = first
        return int(self.table[self.seqs[item], pos // self.bs]), pos % self.bs

    def put(self, item, pos, score, v_scale=None, zero=False):
        """A key whose score is `score` for all query heads; with zero, a V row of zeros as the
        cache's writers store it."""
        b, off = self.cell(item, pos)
        k, v, ks, vs = self.planes
        k[b, :, off] = 0
        if score:
            k[b, :, off, 0] = 127 if score > 0 else -127
            ks[b, :, off] = abs(score) / (self.scale * Q0 * 127)
        if zero:
            v[b, :, off] = 0
            vs[b, :, off] = 1.0
        else:
            vs[b, :, off] = v_scale

    def close(self, out, items=None):
        """Every item within a bound that knows only what its keys weigh.

        A score is off by D products and sums and three roundings of its own products, a
        probability by that and the denominator's share, the exponential by less than 2^-20,
        sums of n by n roundings.  p vs is rounded to fp16 relative to a reference of at most the
        largest p vs of a key with a value: by half a step, or by 2^-25 of that largest."""
        torch, D, bs = self.torch, self.D, self.bs  # noqa: F811
        for i in range(self.S) if items is None else items:
            n = int(self.pos[self.tokens[i]]) + 1
            at = [Scales.cell(self, i, t) for t in range(n)]
            b, off = (torch.tensor(x, device="cuda") for x in zip(*at))
            k, v, ks, vs = (t[b, :, off].double().transpose(0, 1) for t in self.planes)
            q = self.q[int(self.tokens[i]), :self.hq * D].double().view(self.hkv, -1, D)
            kt = (k * ks[..., None]).transpose(1, 2).contiguous()
            p = torch.softmax(q @ kt * self.scale, -1)  # [Hkv, G, n]
            e = 1.5 * (D + 4) * U32 * (q.abs() @ kt.abs()) * abs(self.scale)
            e = e + (p * e).sum(-1, keepdim=True) + U16 + 2 * n * U32 + 2.0 ** -20
            o = p @ (v * vs[..., None])
            top = (p * (vs * (v != 0).any(-1))[:, None]).amax(-1, keepdim=True)
            tol = (p * e) @ (v.abs() * vs[..., None]) + 1.01 * 2.0 ** -25 * top * v.abs().sum(1)[:, None]
            assert torch.isfinite(o).all()
            err = (out[int(self.tokens[i])].view(self.hkv, -1, D).double() - o).abs()
            # (NaN fails too)
            bad = ~(err <= tol + U16 * (o.abs() + tol) + 2.0 ** -25)
            assert not bad.any(), (i, n, float(err.max()), float(o.abs().max()))


def variants(f):
    for name, values in (("form", list(FORMS)), ("D", [64, 128]), ("cache", ["int8", "int8_f16"])):
        f = pytest.mark.parametrize(name, values)(f)
    return f


@variants
@pytest.mark.parametrize("ratio", [1, 2 ** 16, 2 ** 20, 2 ** 24, 2 ** 26])
def test_large_scale_without_weight(torch, ratio, form, D, cache):  # noqa: F811
    """One key of the prefix, one of an item's own keys and one of an item without a group: V up
    to 65024 of no weight beside values of 2^-10."""
    say("shared loud keys", ratio, form, D, cache)
    small = 2.0 ** -17
    c = Scales(torch, form, D, cache, small)
    for item, pos in ((0, 37), (0, 705), (len(c.own) - 1, 250)):
        c.put(item, pos, -40.0, small * ratio)
    c.close(c.run())


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("D", [64, 128])
def test_largest_ratio_of_scales(torch, form, D):  # noqa: F811
    """Values of 2^-14 at most beside V rows of 65024 without weight: scales 2^30 apart (fp32
    scales alone hold so small ones)."""
    say("shared largest ratio", form, D)
    c = Scales(torch, form, D, "int8", 2.0 ** -21, seed=8)
    for item, pos in ((0, 0), (0, 37), (0, 705), (len(c.own) - 1, 250)):
        c.put(item, pos, -40.0, 2.0 ** 9)
    out = c.run()
    c.close(out)
    assert (out[torch.from_numpy(c.tokens).cuda()] != 0).any(1).all()


@variants
def test_large_scales_past_an_items_last_key(torch, form, D, cache):  # noqa: F811
    """Items that end inside their group's prefix, before a key that has both a large V scale and
    a large score."""
    say("shared loud keys past the end", form, D, cache)
    c = Scales(torch, form, D, cache, 2.0 ** -17)
    for pos in (299, 303, 511):
        c.put(0, pos, 30.0, 2.0 ** 8)
    for i, n in enumerate([290, 299, 1] + [16 * j + 1 for j in range(18)][:c.S - 4]):
        c.own[i] = n
        c.pos[c.tokens[i]] = n - 1
    c.close(c.run())


@variants
@pytest.mark.parametrize("score", [0.0, 10.0, 25.0, 60.0])
@pytest.mark.parametrize("small", [2.0 ** -6, 2.0 ** -13, 2.0 ** -17])
def test_rows_of_zeros(torch, small, score, form, D, cache):  # noqa: F811
    """A row of zeros has the scale 1: a first key that takes much of the weight and gives
    nothing (at 60 all others are below fp16), more of them among the rest, and whole tiles."""
    say("shared rows of zeros", small, score, form, D, cache)
    c = Scales(torch, form, D, cache, small)
    own = len(c.own) - 1
    for item, pos in [(0, 0), (0, 701), (own, 0)]:
        c.put(item, pos, score, zero=True)
    for t in (5, 300, *range(512, 576)):
        c.put(0, t, 0.0, zero=True)
        if t < 500:
            c.put(own, t, 1.0, zero=True)
    c.close(c.run())


@variants
def test_only_rows_of_zeros(torch, form, D, cache):  # noqa: F811
    say("shared only zeros", form, D, cache)
    c = Scales(torch, form, D, cache, 2.0 ** -9, prefix=33)
    c.planes[1].zero_()
    c.planes[3].copy_(torch.where(torch.isnan(c.planes[3].float()), c.planes[3], torch.ones_like(c.planes[3])))
    out = c.run()
    assert (out[torch.from_numpy(c.tokens).cuda()] == 0).all()


@variants
def test_scales_of_every_size(torch, form, D, cache):  # noqa: F811
    """V scales from 2^-17 to 2^8, each key for itself, and scores of a few."""
    say("shared mixed scales", form, D, cache)
    c = Scales(torch, form, D, cache, 2.0 ** -17, seed=5)
    vs = c.planes[3]
    g = torch.Generator(device="cuda").manual_seed(9)
    # (in 32 bits: 2^16 is past fp16, the products are not)
    vs.copy_(vs.float() * torch.exp2(torch.randint(0, 25, vs.shape, generator=g, device="cuda").float()))
    c.close(c.run())


@variants
def test_zero_scales(torch, form, D, cache):  # noqa: F811
    """Scales of 0 (fp16 scales of the smallest values round to it): values of 0."""
    say("shared zero scales", form, D, cache)
    c = Scales(torch, form, D, cache, 2.0 ** -10, seed=6)
    c.put(0, 0, 12.0, 0.0)
    c.put(0, 400, 0.0, 0.0)
    c.put(len(c.own) - 1, 3, 12.0, 0.0)
    c.close(c.run())


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cache", ["fp16", "int8", "int8_f16"])
@pytest.mark.parametrize("factor", [-1.0, 0.0, -0.0, -3.0, 1e-30, -1e-42])
def test_signs_of_the_softmax_scale(torch, factor, cache, D, form):  # noqa: F811
    """The scale may have either sign (the smallest score then has the weight) or none (all keys
    weigh the same)."""
    say("shared scale signs", factor, cache, D, form)
    per, own = FORMS[form]
    groups = [(260, own), (None, [300])]
    c = Case(torch, groups, 2 * per, 2, D, 16, cache, 7, amp=1.0)
    c.scale *= factor
    out = c.run()
    c.check(out)
    if cache != "fp16":
        Scales.close(c, out)
