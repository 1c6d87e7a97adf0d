"""Decode attention over shared prefixes against a 64-bit softmax."""
import math

import numpy as np
import pytest

import redline_amd as ra
from tests._util import say

pytestmark = pytest.mark.gpu
U32, U16 = 2.0 ** -24, 2.0 ** -11


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


class Case:
    """Items in groups [(prefix, [keys of each item beyond it])]; a group of prefix None is of
    items outside every group.  Everything that no item may read is NaN: unused blocks, rows
    behind an item's last key, and the prefix in the tables of a group's later items."""

    def __init__(self, torch, groups, hq=8, hkv=2, D=128, bs=16, cache="fp16", seed=0, amp=1.5, own_prefix=False,
                 first_block=0):
        from redline_amd import kernels as K
        rng, g = np.random.default_rng(seed), torch.Generator(device="cuda").manual_seed(seed)
        self.torch, self.hq, self.hkv, self.D, self.bs = torch, hq, hkv, D, bs
        self.sd = K.SCALE_F16 if cache == "int8_f16" else K.SCALE_F32
        own = [(p or 0) + x for p, xs in groups for x in xs]
        S = self.S = len(own)
        self.mb = max(1, -(-max(own) // bs))
        total = S * self.mb
        seqs = self.seqs = rng.permutation(S + 2)[:S]  # rows of the table; two are nobody's
        table = np.full((S + 2, self.mb), first_block, np.int64)
        table[seqs] = first_block + rng.permutation(total).reshape(S, self.mb)
        used = np.zeros((total, bs), bool)
        self.starts, self.prefix, firsts, i = [0], [], [], 0
        for p, xs in groups:
            for j, x in enumerate(xs):
                n = (p or 0) + x
                at = np.arange(0 if j == 0 or p is None or own_prefix else p, n)
                used[table[seqs[i], at // bs] - first_block, at % bs] = True
                firsts.append(None if p is None else i - j)
                i += 1
            self.starts.append(i)
            self.prefix.append(-1 if p is None else p)
        shape = (total, hkv, bs, D)
        k = torch.randn(shape, generator=g, device="cuda") * amp
        v = torch.randn(shape, generator=g, device="cuda") * torch.exp2(
            torch.randint(-3, 3, (total, 1, 1, 1), generator=g, device="cuda").float())
        hole = ~torch.from_numpy(used).cuda()[:, None, :, None]
        if cache == "fp16":
            planes = [x.masked_fill(hole, math.nan).half() for x in (k, v)]
        else:
            planes, scales = [], []
            for x in (k, v):
                s = x.abs().amax(-1) / 127
                s = s.half() if cache == "int8_f16" else s
                planes.append((x / s.float()[..., None]).round().clamp(-127, 127).to(torch.int8))
                scales.append(s.masked_fill(hole[..., 0], math.nan))
            planes += scales
        self.planes = planes
        if first_block:
            big = []
            for t in planes:
                b = torch.empty((first_block + total, *t.shape[1:]), dtype=t.dtype, device="cuda")
                b[first_block:] = t
                big.append(b)
            planes = big
        self.view = K.kv_layer_view(*planes)
        self.used_planes = planes
        if own_prefix:  # the same keys in every item's own blocks
            i = 0
            for p, xs in groups:
                for j, x in enumerate(xs):
                    if j and p:
                        at = torch.arange(p, device="cuda")
                        t = torch.from_numpy(table).cuda()
                        src, dst = t[seqs[i - j]][at // bs], t[seqs[i]][at // bs]
                        for y in planes:
                            y[dst, :, at % bs] = y[src, :, at % bs]
                    i += 1
        self.table, self.own, self.firsts, self.first_block = table, np.array(own), firsts, first_block
        rows = self.rows = S + 3
        self.tokens = rng.permutation(rows)[:S]
        self.cols = (hq + 2 * hkv) * D
        self.q = (torch.randn(rows, self.cols, generator=g, device="cuda") * amp).half()
        self.pos = np.full(rows, -7)
        self.pos[self.tokens] = self.own - 1
        self.scale = D ** -0.5

    def i32(self, a):
        return self.torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()

    def plan(self, max_items=None, prefix_parts=None, parts=None, tokens=None, prefix=None, starts=None):
        from redline_amd import kernels as K
        out = self.torch.full((self.rows, self.hq * self.D), 9.0, dtype=self.torch.float16, device="cuda")
        tokens = self.tokens if tokens is None else tokens
        prefix = self.prefix if prefix is None else prefix
        starts = self.starts if starts is None else starts
        if max_items is None:
            max_items = int(np.diff(starts).max())
        if prefix_parts is None:
            prefix_parts = max(0, -(-max(prefix) // 256)) if len(prefix) else 0
        if parts is None:
            shared = np.array([0 if f is None else self.prefix[np.searchsorted(self.starts, i, "right") - 1]
                               for i, f in enumerate(self.firsts)])
            parts = max(1, int(-(-(self.own - shared).max() // 256)))
        ws = K.DecodeWorkspace(self.S, self.hq, prefix_parts + parts, self.D)
        p = K.attention_params(self.q, self.cols, out, self.hq, self.scale, self.view, self.i32(self.table), self.mb,
                               self.i32(self.pos))
        w = K.shared_prefix_work(self.i32(tokens), self.i32(self.seqs), self.S, self.i32(starts), self.i32(prefix),
                                 len(prefix), max_items, prefix_parts, parts, ws)
        return p, w, out

    def run(self, plan=None, stream=None, **kw):
        from redline_amd import kernels as K
        p, w, out = plan or self.plan(**kw)
        K.paged_attention_decode_shared(p, w, self.sd, stream)
        return out

    def want(self, item, keys=None):
        """(o, bound) [Hq, D] of an item in 64 bits."""
        torch, D, bs, hkv = self.torch, self.D, self.bs, self.hkv
        n = int(self.own[item] if keys is None else keys)
        first = self.firsts[item]
        at = np.arange(n)
        own = self.table[self.seqs[item], at // bs]
        if first is not None:
            p = self.prefix[np.searchsorted(self.starts, item, "right") - 1]
            own = np.where(at < p, self.table[self.seqs[first], at // bs], own)
        blocks, off = torch.from_numpy(own).cuda(), torch.from_numpy(at % bs).cuda()
        kv = []
        for i in range(2):
            x = self.used_planes[i][blocks, :, off].double()  # [n, Hkv, D]
            if len(self.used_planes) > 2:
                x = x * self.used_planes[2 + i][blocks, :, off].double()[..., None]
            kv.append(x.transpose(0, 1))
        q = self.q[int(self.tokens[item]), :self.hq * D].double().view(hkv, -1, D)
        s = (q @ kv[0].transpose(1, 2).contiguous()) * self.scale
        size = (q.abs() @ kv[0].abs().transpose(1, 2).contiguous()).amax() * abs(self.scale)
        p = torch.softmax(s, -1)
        o, a = p @ kv[1], p @ kv[1].abs()
        int8 = len(self.used_planes) > 2
        # a score is off by D products and sums and three roundings; a probability by twice that
        # (its own, the sum's) and the exponential, by half a step of fp16 or 2^-25 of the
        # largest; an INT8 value by half a step more; sums of n by n roundings
        rel = U16 * (1 + int8) + 2 * (D + 4) * U32 * float(size) * 1.5 + 2 * n * U32 + 2.0 ** -20
        bound = rel * a + n * 2.0 ** -25 * kv[1].abs().amax(1, keepdim=True)
        return o.reshape(self.hq, D), bound.reshape(self.hq, D)

    def gap(self, item):
        """How far the second largest score of each query head lies below the largest (fp16 cache,
        a group's item)."""
        at = np.arange(int(self.own[item]))
        p = self.prefix[np.searchsorted(self.starts, item, "right") - 1]
        row = np.where(at < p, self.table[self.seqs[self.firsts[item]], at // self.bs],
                       self.table[self.seqs[item], at // self.bs])
        k = self.used_planes[0][self.torch.from_numpy(row).cuda(), :, self.torch.from_numpy(at % self.bs).cuda()]
        q = self.q[int(self.tokens[item]), :self.hq * self.D].double().view(self.hkv, -1, self.D)
        s = q @ k.double().permute(1, 2, 0).contiguous() * self.scale
        top = s.topk(2, -1).values.view(self.hq, 2)
        return top[:, 0] - top[:, 1]

    def check(self, out, items=None, keys=None, untouched=()):
        for i in range(self.S) if items is None else items:
            o, b = self.want(i, keys)
            got = out[int(self.tokens[i])].view(self.hq, self.D).double()
            err = (got - o).abs()
            assert (err <= b + U16 * (o.abs() + b) + 2.0 ** -25).all(), (i, int(self.own[i]), float(err.max()))
        rest = sorted(set(range(self.rows)) - set(self.tokens.tolist()) | {int(t) for t in untouched})
        assert (out[rest] == 9.0).all()


GROUPS = [
    [(1, [1])], [(0, [1])], [(None, [1, 300])], [(63, [1, 2, 65])], [(64, [64, 1, 1, 1])], [(257, [1] * 9)],
    [(1000, [3, 200, 64, 700, 1])], [(40, [1, 5]), (0, [9, 20]), (None, [333, 17]), (513, [2] * 20), (8, [600])],
    [(100, list(range(1, 34)))],
]
HEADS = [(8, 2, 128, 16), (7, 1, 128, 32), (4, 4, 64, 8), (32, 4, 64, 16), (6, 2, 64, 24), (5, 1, 128, 1)]


@pytest.mark.parametrize("groups", GROUPS, ids=lambda g: "+".join(f"{p}x{len(x)}" for p, x in g))
@pytest.mark.parametrize("cache", ["fp16", "int8", "int8_f16"])
def test_groups(torch, groups, cache):
    say("shared", groups, cache)
    c = Case(torch, groups, *HEADS[len(groups[0][1]) % 2], cache, 3)
    c.check(c.run())


@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("cache", ["fp16", "int8", "int8_f16"])
def test_heads(torch, heads, cache):
    say("shared", heads, cache)
    c = Case(torch, [(130, [1, 90, 7]), (None, [50]), (700, [3, 3, 300, 4, 1, 1, 1])], *heads, cache, 5)
    c.check(c.run())


@pytest.mark.parametrize("group", range(1, 9))
def test_query_heads_to_a_kv_head(torch, group):
    say("shared group size", group)
    c = Case(torch, [(300, [2, 100, 31]), (20, [4] * 17)], 2 * group, 2, 128, 16, "fp16", group)
    c.check(c.run())


@pytest.mark.parametrize("cache", ["fp16", "int8"])
def test_long_prefixes(torch, cache):
    """More ranges than a wave holds, row tiles that end inside an item, items of one key."""
    say("shared long", cache)
    c = Case(torch, [(40000, [1, 600, 2, 33] + [5] * 29)], 14, 2, 128, 16, cache, 8)
    c.check(c.run())
    c = Case(torch, [(None, [70001])], 2, 1, 64, 16, cache, 8)
    c.check(c.run())


def test_the_same_as_plain_decode(torch):
    """No groups, or groups whose items all have the prefix in blocks of their own: what
    paged_attention_decode gives, but for roundings (the sum of both bounds)."""
    from redline_amd import kernels as K
    say("shared against plain decode")
    c = Case(torch, [(200, [30, 70, 1]), (90, [400])], 8, 2, 128, 16, "fp16", 11, own_prefix=True)
    out = c.run()
    alone = c.run(prefix=[], starts=[0], max_items=0, parts=2)
    c.check(out)
    c.check(alone)
    plain = torch.full_like(out, 9.0)
    ws = K.DecodeWorkspace(c.S, c.hq, 2, c.D)
    p = K.attention_params(c.q, c.cols, plain, c.hq, c.scale, c.view, c.i32(c.table), c.mb, c.i32(c.pos))
    K.paged_attention_decode(p, K.decode_work(c.i32(c.tokens), c.i32(c.seqs), c.S, 2, ws))
    c.check(plain)


def test_skipped_and_empty_items(torch):
    """Negative tokens (a group's first among them) skip their items; negative positions give
    zeros."""
    say("shared skipped items")
    c = Case(torch, [(100, [5, 9, 3]), (None, [40, 8]), (30, [2, 2])], seed=13)
    tokens = c.tokens.copy()
    tokens[[0, 3]] = -1
    c.pos[c.tokens[6]] = -1
    out = c.run(tokens=tokens)
    c.check(out, [1, 2, 4, 5], untouched=c.tokens[[0, 3]])
    assert (out[int(c.tokens[6])] == 0).all()
    out = c.run(tokens=np.full(c.S, -1))
    assert (out == 9.0).all()


def test_items_that_end_inside_the_prefix(torch):
    say("shared short items")
    c = Case(torch, [(500, [9, 1, 1, 1, 1])], seed=14)
    ends = [509, 1, 63, 256, 499]
    for i, n in enumerate(ends):
        c.own[i] = n
        c.pos[c.tokens[i]] = n - 1
    c.check(c.run(parts=1))


def test_fewer_partitions_than_keys(torch):
    """A prefix past max_prefix_partitions, and items past max_group_items, are read by the
    items themselves; of what an item reads itself, keys past max_partitions are not read."""
    say("shared few partitions")
    c = Case(torch, [(900, [10, 300, 77])], seed=15, own_prefix=True)
    c.check(c.run(prefix_parts=2, parts=3))
    c.check(c.run(prefix_parts=0, parts=5))
    c.check(c.run(max_items=2, parts=5))
    c.check(c.run(max_items=0, parts=5))
    c.own[1] = 900 + 256  # of 1200
    c.check(c.run(parts=1))


def test_keys_past_the_table_row(torch):
    """Positions past the table's width attend to what the row holds."""
    say("shared past the table")
    c = Case(torch, [(64, [32, 32]), (None, [96])], bs=16, seed=16)
    c.pos[c.tokens] = [95, 200, 2 ** 31 - 1]
    c.check(c.run(parts=3, prefix_parts=1))


def test_large_scores(torch):
    """Scores in the tens of thousands, of which one key takes all, and maxima that rise tile
    by tile."""
    say("shared large scores")
    c = Case(torch, [(400, [70, 3])], 4, 2, 128, 16, "fp16", 17)
    for t in c.used_planes[:1]:
        t.mul_(200)
    c.q.mul_(20)
    out = c.run()
    rows = 0
    for i in range(2):
        o, _ = c.want(i)
        got = out[int(c.tokens[i])].view(4, 128).double()
        assert torch.isfinite(got).all()
        # where the second largest score lies 30 below, the output is one V row, to its rounding
        # (scores are off by less than 1: 128 roundings of sums below 2^17)
        clear = c.gap(i) > 30
        rows += int(clear.sum())
        assert ((got - o).abs() <= 2.0 ** -10 * o.abs() + 2.0 ** -25)[clear].all()
    assert rows > 0
    rise = Case(torch, [(512, [1, 1])], 2, 1, 64, 16, "fp16", 18)
    t, seq = rise.used_planes[0], rise.table[rise.seqs[0]]
    x = torch.arange(512, device="cuda").view(-1, 16)[:, None, :, None] / 16.0
    t[torch.from_numpy(seq[:32]).cuda()] = (x * torch.ones(1, 1, 1, 64, device="cuda") / 8).half()
    rise.q.fill_(1.0)
    rise.check(rise.run())


def test_repeats_streams_and_graphs(torch):
    """The same bits every time, on another stream, and in two graphs that share a workspace."""
    from redline_amd import kernels as K
    say("shared repeats, streams, graphs")
    c = Case(torch, [(700, [10, 30, 5, 300]), (None, [90])], 16, 4, 128, 16, "int8", 19)
    d = Case(torch, [(90, [1, 2, 3])], 16, 4, 128, 16, "int8", 20)
    first, other = c.run().clone(), d.run().clone()
    c.check(first)
    assert torch.equal(c.run(), first)
    s = torch.cuda.Stream()
    plan = c.plan()
    s.wait_stream(torch.cuda.current_stream())
    out = c.run(plan, s)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, first)
    ws = K.DecodeWorkspace(c.S, 16, 5, 128)
    plans, graphs = [], []
    for x in (c, d):
        p, w, o = x.plan()
        w.ws_out, w.ws_max, w.ws_sum = ws.out.data_ptr(), ws.max.data_ptr(), ws.sum.data_ptr()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            x.run((p, w, o))
        plans.append((p, w, o))
        graphs.append(graph)
    for _ in range(3):
        for graph, plan, want in zip(graphs, plans, (first, other)):
            plan[2].fill_(9.0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(plan[2], want)


def test_keys_past_32_bits(torch):
    """Blocks whose bytes lie past 2^32."""
    say("shared far blocks")
    c = Case(torch, [(100, [40, 3])], 8, 2, 128, 16, "fp16", 21, first_block=(1 << 32) // (2 * 16 * 128 * 2) + 9)
    c.check(c.run())


def test_launchers_refuse(torch):
    from redline_amd import kernels as K
    say("shared refusals")
    c = Case(torch, [(100, [5, 9])], 4, 2, 64, 16, "int8", 22)
    p, w, _ = c.plan()
    with pytest.raises(ra.Error, match="scale dtype"):
        K.paged_attention_decode_shared(p, w, K.SCALE_F16)
    small = K.DecodeWorkspace(1, 4, 2, 64)
    i = c.i32
    args = [i(c.tokens), i(c.seqs), 2, i(c.starts), i(c.prefix), 1, 2, 1, 1]
    with pytest.raises(ra.Error, match="workspace holds"):
        K.paged_attention_decode_shared(p, K.shared_prefix_work(*args, small))
    ws = K.DecodeWorkspace(2, 4, 2, 64)
    for at, bad, text in ((0, i([1]), "item_token holds"), (1, c.q, "item_seq must be"), (3, i([0]), "group_start holds"),
                          (4, None, "group_prefix must"), (0, i([0, 1]).cpu(), "GPU tensor")):
        a = list(args)
        a[at] = bad
        with pytest.raises(ra.Error, match=text):
            K.shared_prefix_work(*a, ws)
    for n in (0, -3):
        a = list(args)
        a[2] = n
        K.paged_attention_decode_shared(p, K.shared_prefix_work(*a, ws))  # nothing to do


@pytest.mark.parametrize("heads", [(4, 4, 64, 16), (8, 4, 128, 16), (3, 1, 64, 24)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("cache", ["fp16", "int8"])
def test_group_sizes_at_every_border(torch, heads, cache):
    """Groups of 15 to 17, 47 to 49 and 127 to 129 rows, of one kind and all in one call."""
    say("shared borders", heads, cache)
    per = heads[0] // heads[1]
    sizes = sorted({max(1, r // per + e) for r in (16, 48, 128) for e in (-1, 0, 1)})
    for n in sizes:
        c = Case(torch, [(600, [1 + i % 3 for i in range(n)]), (300, [70])], *heads, cache, n)
        c.check(c.run())
    c = Case(torch, [(97 + 61 * j, [2] * n) for j, n in enumerate(sizes)], *heads, cache, 31)
    c.check(c.run())
