"""Sampling from given random numbers against a sort and sums in 64 bits."""
import math

import numpy as np
import pytest

import redline_amd as ra
from tests._util import say

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
SLACK = 2.0 ** -33  # of a border: weights are held to 2^-35, the masses on both sides of it too


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def draw(row, T, k, p, m, u, nudge=(0, 0, 0)):
    """(token, logprob) of one row (numpy) by the definition, its borders moved by nudge * SLACK."""
    x = np.asarray(row, np.float32).astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    if not T > 0 or x[order[0]] == -np.inf:
        return int(order[0]), 0.0
    x = x[order]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((x - x[0]) / np.float64(np.float32(T)))
    w = np.where(x == x[0], 1.0, np.where(w < 2.0 ** -48, 0.0, w))  # (inf - inf; far tokens)
    n = int((w > 0).sum())
    if k > 0:
        n = min(n, k)
    run = np.cumsum(w)
    f = [1 + e * SLACK for e in nudge]
    p, m, u = np.float32(p), np.float32(m), np.float32(u)
    if p < 1:
        n = min(n, 1 + int((run[:n - 1] < float(p) * run[n - 1] * f[0]).sum()))
    m = 1.0 if not m <= 1 else float(m)
    if m > 0:
        n = max(1, int((w[:n] >= m * f[1]).sum()))
    u = min(float(u), 1 - 2.0 ** -24) if u > 0 else 0.0
    j = min(int((run[:n] <= u * run[n - 1] * f[2]).sum()), n - 1)
    return int(order[j]), math.log(w[j] / run[n - 1])


def candidates(*a):
    out = {}
    for e in np.ndindex(3, 3, 3):
        t, lp = draw(*a, nudge=[x - 1 for x in e])
        out[t] = lp
    return out


class Call:
    def __init__(self, torch, logits, T=1.0, k=0, p=1.0, m=0.0, u=0.5, param_row=None, settings=None):
        from redline_amd import kernels as K
        R, V = logits.shape
        n = settings or R
        full = lambda x, dt: torch.from_numpy(np.array(np.broadcast_to(np.asarray(x, dt), (n,)))).cuda()  # noqa: E731
        self.torch, self.logits, self.R, self.V = torch, logits, R, V
        self.T, self.p, self.m = (full(x, np.float32) for x in (T, p, m))
        self.k = full(k, np.int32)
        self.u = torch.from_numpy(np.array(np.broadcast_to(np.asarray(u, np.float32), (R,)))).cuda()
        self.at = param_row
        self.tokens = torch.full((R + 2,), -9, dtype=torch.int32, device="cuda")
        self.lp = torch.full((R + 2,), 9.0, device="cuda")
        self.ws = K.SamplingWorkspace(R, V)
        self.ws.memory.fill_(0x7f)
        at = None if param_row is None else torch.from_numpy(np.asarray(param_row, np.int32)).cuda()
        self.work = K.sampling_work(logits, R, V, self.T, self.k, self.p, self.u, self.tokens, self.ws, self.m, at,
                                    self.lp)

    def __call__(self, stream=None):
        from redline_amd import kernels as K
        K.sample_tokens(self.work, stream)
        return self

    def check(self, rows=None):
        tok, lp = self.tokens.cpu().numpy(), self.lp.cpu().numpy()
        assert (tok[self.R:] == -9).all() and (lp[self.R:] == 9).all()
        x = self.logits.float().cpu().numpy()
        T, k, p, m, u = (t.cpu().numpy() for t in (self.T, self.k, self.p, self.m, self.u))
        for r in range(self.R) if rows is None else rows:
            a = r if self.at is None else self.at[r]
            args = x[r], T[a], k[a], p[a], m[a], u[r]
            want, q = draw(*args)
            if want != tok[r]:
                near = candidates(*args)
                assert int(tok[r]) in near, (r, int(tok[r]), want, args[1:])
                q = near[int(tok[r])]
            # rounded to fp32 once; masses in 2^-35, a logarithm in 64 bits
            assert abs(float(lp[r]) - q) <= U32 * abs(q) + 2.0 ** -32, (r, float(lp[r]), q)
        return self


def settings(rng, n):
    mode = rng.integers(0, 7, n)
    T = np.where(mode == 0, 0.0, rng.choice([0.3, 0.7, 1.0, 1.5, 4.0], n))
    k = np.where(np.isin(mode, (1, 2)), rng.integers(1, 3000, n), 0)
    p = np.where(np.isin(mode, (2, 3, 4)), rng.uniform(0.05, 0.999, n), 1.0)
    m = np.where(np.isin(mode, (4, 5)), rng.uniform(0.001, 0.3, n), 0.0)
    return dict(T=T, k=k, p=p, m=m)


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("V", [1, 2, 3, 50, 255, 256, 257, 4095, 4096, 4097, 32000, 65537, 128256, 200003])
def test_vocabularies(torch, V, fp32):
    rng = np.random.default_rng(V)
    R = 29
    say("sample vocab", V, fp32)
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(R, V, generator=g, device="cuda") * 3 - 2 * torch.log(
        torch.rand(R, V, generator=g, device="cuda").clamp(min=1e-9))
    c = Call(torch, x if fp32 else x.half(), u=rng.random(R), param_row=rng.permutation(40)[:R], settings=40,
             **settings(rng, 40))
    c().check()


@pytest.mark.parametrize("spread", [0.01, 0.3, 30.0, 3000.0])
def test_spreads(torch, spread):
    """From rows in a bin or two (which hold more tokens than are sorted at once) to rows whose
    tokens stand apart."""
    say("sample spread", spread)
    rng = np.random.default_rng(5)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(24, 40000, generator=g, device="cuda") * spread
    Call(torch, x, u=rng.random(24), **settings(rng, 24))().check()
    Call(torch, x.half(), u=rng.random(24), **settings(rng, 24))().check()


@pytest.mark.parametrize("values", [1, 2, 7])
@pytest.mark.parametrize("V", [9, 3000, 100001])
def test_ties(torch, values, V):
    """Few values: ties go in the order of the index, at every limit."""
    say("sample ties", values, V)
    rng = np.random.default_rng(values)
    R = 40
    x = torch.from_numpy(rng.integers(0, values, (R, V)).astype(np.float16) / 4).cuda()
    c = settings(rng, R)
    c["k"] = np.where(rng.random(R) < 0.4, rng.integers(1, V + 5, R), 0)
    Call(torch, x, u=(rng.random(R) * 0.98 + 0.01), **c)().check()


def test_equal_tokens_exactly(torch):
    """n tokens of one value: u n < j + 1 draws index j, whole numbers among them."""
    say("sample equal tokens")
    for V in (8, 4096, 100000):
        u = np.array([0, 0.25, 0.5, 0.75, 0.125, 1 - 2.0 ** -24, (V // 2 - 1) / V + 1e-6], np.float32)
        c = Call(torch, torch.full((7, V), 2.0, device="cuda"), u=u)()
        want = [min(int(math.floor(float(x) * V)), V - 1) for x in u]
        assert c.tokens[:7].tolist() == want
        c = Call(torch, torch.full((7, V), 2.0, device="cuda"), k=V // 2, u=u)()
        assert c.tokens[:7].tolist() == [min(int(math.floor(float(x) * (V // 2))), V // 2 - 1) for x in u]


def test_masked_rows(torch):
    """-infinity, NaN and the type's lowest value in masked places, rows that leave one token
    or none, and +infinity."""
    say("sample masked")
    rng = np.random.default_rng(9)
    for dt, V in ((torch.float16, 5000), (torch.float32, 70001)):
        x = torch.randn(12, V, generator=torch.Generator(device="cuda").manual_seed(V), device="cuda").to(dt)
        hide = torch.rand(12, V, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") < 0.95
        x[0:2] = torch.where(hide[0:2], -math.inf, x[0:2])
        x[2] = torch.where(hide[2], math.nan, x[2])
        x[3] = torch.where(hide[3], torch.finfo(dt).min, x[3])
        x[4], x[5], x[6] = -math.inf, math.nan, torch.finfo(dt).min
        x[7] = -math.inf
        x[7, V - 1] = -3
        x[8, 17], x[8, V - 2] = math.inf, math.inf
        x[9, 40] = math.inf
        x[10] = -math.inf
        x[10, 5], x[10, 6] = torch.finfo(dt).min, torch.finfo(dt).max
        x[11, ::2] = -math.inf
        for kw in (dict(u=0.3), dict(u=0.9, p=0.8), dict(u=0.6, k=900, m=0.01), dict(T=0.0), dict(T=1.3, u=rng.random(12))):
            c = Call(torch, x, **kw)().check()
            t = c.tokens.tolist()
            assert t[4] == 0 and t[5] == 0 and t[7] == V - 1 and t[8] in (17, V - 2) and t[9] == 40 and t[10] == 6


def test_extreme_settings(torch):
    """Temperatures, limits and random numbers at and past the ends of their ranges."""
    say("sample extremes")
    nan, inf = math.nan, math.inf
    grid = [dict(T=t, u=u) for t in (0, -1, nan, 1e-30, 1e-40, 1e-4, 1e4, 1e30, 3e38) for u in (0.0, 0.4, 0.9999)]
    grid += [dict(u=u) for u in (-1, nan, 1.0, 2.0, inf, -0.0, 1e-40, 1 - 2.0 ** -24)]
    grid += [dict(k=k, u=u) for k in (-5, 1, 2, 6999, 7000, 7001, 2 ** 31 - 1) for u in (0.1, 0.97)]
    grid += [dict(p=p, u=u) for p in (-1, 0.0, 1e-30, 1e-6, 0.999999, 1.0, 2.0, nan) for u in (0.1, 0.97)]
    grid += [dict(m=m, u=u) for m in (-1, 1e-30, 1e-9, 0.999999, 1.0, 2.0, nan, inf) for u in (0.1, 0.97)]
    pick = lambda n, d: np.array([c.get(n, d) for c in grid])  # noqa: E731
    x = torch.randn(1, 7000, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda") * 4
    x = x.repeat(len(grid), 1)
    for y in (x, x.half()):
        Call(torch, y, T=pick("T", 1.0), k=pick("k", 0), p=pick("p", 1.0), m=pick("m", 0.0), u=pick("u", 0.5))().check()


def test_infinite_temperature(torch):
    """All finite tokens weigh the same."""
    say("sample infinite temperature")
    x = torch.randn(3, 1000, device="cuda")
    c = Call(torch, x, T=math.inf, u=[0.0, 0.5, 0.9995])()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices.cpu()
    assert c.tokens[:3].tolist() == [int(order[0, 0]), int(order[1, 500]), int(order[2, 999])]
    assert (c.lp[:3] + math.log(1000)).abs().max() < 1e-6


@pytest.mark.parametrize("fp32", [False, True])
def test_strides_and_alignment(torch, fp32):
    """Rows inside wider ones, at every alignment."""
    say("sample strides", fp32)
    rng = np.random.default_rng(3)
    base = torch.randn(11, 9100, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda") * 4
    base = base if fp32 else base.half()
    for off in range(9):
        Call(torch, base[:, off:off + 9000 - off], u=rng.random(11), **settings(rng, 11))().check()
    Call(torch, base.view(-1)[3:3 + 11 * 8269].view(11, 8269), u=rng.random(11), **settings(rng, 11))().check()


def test_rows_do_not_depend_on_the_batch(torch):
    """One row gives the same token and log-probability to the bit alone and among 700 (which
    are cut into larger chunks)."""
    say("sample batch independence")
    rng = np.random.default_rng(4)
    x = torch.randn(700, 33000, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda") * 2
    u, s = rng.random(700), settings(rng, 700)
    many = Call(torch, x, u=u, **s)().check(range(0, 700, 41))
    again = Call(torch, x, u=u, **s)()
    assert torch.equal(many.tokens, again.tokens) and torch.equal(many.lp, again.lp)
    for r in range(0, 700, 29):
        one = Call(torch, x[r:r + 1], u=u[r], **{n: v[r] for n, v in s.items()})()
        assert int(one.tokens[0]) == int(many.tokens[r]) and float(one.lp[0]) == float(many.lp[r])


def test_draws_follow_the_weights(torch):
    """4096 evenly spread random numbers draw each token as often as its weight says, to one."""
    say("sample frequencies")
    n = 4096
    x = (torch.randn(1, 300, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda") * 2).repeat(n, 1)
    c = Call(torch, x, T=0.9, k=50, u=(np.arange(n) + 0.5) / n)()
    w = torch.softmax(x[0].double() / np.float32(0.9).astype(np.float64), 0)
    w[w < w.topk(50).values[-1]] = 0
    count = torch.bincount(c.tokens[:n].long(), minlength=300)
    assert (count - w / w.sum() * n).abs().max() <= 1 + 1e-6


def test_streams_and_graphs(torch):
    """On another stream, and in two graphs that share a workspace, with new random numbers
    and logits for each replay."""
    from redline_amd import kernels as K
    say("sample streams and graphs")
    rng = np.random.default_rng(6)
    make = lambda R, V, seed: Call(torch, torch.randn(R, V, generator=torch.Generator(device="cuda").manual_seed(seed),  # noqa: E731
                                                      device="cuda") * 3, u=rng.random(R), **settings(rng, R))
    c = make(17, 50000, 1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    c(s)
    torch.cuda.current_stream().wait_stream(s)
    c.check()
    ws, calls, graphs = K.SamplingWorkspace(17, 50000), [make(17, 50000, 2), make(5, 800, 3)], []
    for x in calls:
        x.work.workspace, x.work.workspace_bytes = ws.memory.data_ptr(), ws.memory.numel()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            x()
        graphs.append(graph)
    for i in range(3):
        for x, graph in zip(calls, graphs):
            x.logits.normal_(generator=torch.Generator(device="cuda").manual_seed(10 + i)).mul_(3)
            x.u.copy_(torch.from_numpy(rng.random(x.R).astype(np.float32)))
            x.tokens.fill_(-9)
            x.lp.fill_(9)
            graph.replay()
            torch.cuda.synchronize()
            x.check()


def test_without_the_optional_arrays(torch):
    from redline_amd import kernels as K
    say("sample without optional arrays")
    rng = np.random.default_rng(7)
    s = settings(rng, 9)
    s["m"] = 0.0
    x = torch.randn(9, 3333, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    c = Call(torch, x, u=rng.random(9), **s)()
    tokens = torch.zeros(9, dtype=torch.int32, device="cuda")
    K.sample_tokens(K.sampling_work(x, 9, 3333, c.T, c.k, c.p, c.u, tokens, c.ws))
    assert torch.equal(tokens, c.tokens[:9])


def test_launchers_refuse(torch):
    from redline_amd import kernels as K
    say("sample refusals")
    x = torch.randn(4, 100, device="cuda")
    f = lambda n: torch.zeros(n, device="cuda")  # noqa: E731
    i = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    ws = K.SamplingWorkspace(4, 100)
    good = dict(logits=x, num_rows=4, vocab=100, temperature=f(4), top_k=i(4), top_p=f(4), uniform=f(4), tokens=i(4),
                workspace=ws, min_p=f(4), param_row=None, logprobs=f(4))
    K.sample_tokens(K.sampling_work(**good))
    for kw, text in ((dict(logits=x.bfloat16()), "logits must be"), (dict(logits=x.cpu()), "GPU tensor"),
                     (dict(logits=x[:3]), "logits must hold"), (dict(vocab=101), "logits must hold"),
                     (dict(logits=torch.randn(100, 4, device="cuda").t()), "contiguous"),
                     (dict(temperature=f(3)), "temperature holds"), (dict(top_k=f(4)), "top_k must be"),
                     (dict(top_p=f(4)[:2]), "top_p holds"), (dict(min_p=f(1)), "min_p holds"), (dict(uniform=f(3)), "uniform"),
                     (dict(tokens=i(3)), "tokens holds"), (dict(param_row=i(3)), "param_row holds"),
                     (dict(logprobs=f(2)), "logprobs holds"), (dict(tokens=None), "tokens must not be None")):
        with pytest.raises(ra.Error, match=text):
            K.sampling_work(**(good | kw))
    with pytest.raises(ra.Error, match="workspace of"):
        K.sample_tokens(K.sampling_work(**(good | dict(workspace=K.SamplingWorkspace(3, 100)))))
    for args in ((0, 5), (5, 0), (5, (1 << 20) + 1)):
        with pytest.raises(ra.Error, match="no sampling workspace"):
            K.SamplingWorkspace(*args)
    K.sample_tokens(K.sampling_work(**(good | dict(num_rows=0))))  # nothing to do


@pytest.mark.parametrize("V", [8191, 8192, 8193, 16384, 16385, 24575])
def test_whole_chunks(torch, V):
    """Vocabularies at the borders of the 8192 tokens that one workgroup takes."""
    say("sample chunks", V)
    rng = np.random.default_rng(V)
    x = torch.randn(21, V, generator=torch.Generator(device="cuda").manual_seed(V), device="cuda") * 3
    Call(torch, x, u=rng.random(21), **settings(rng, 21))().check()
    Call(torch, x.half(), u=rng.random(21), **settings(rng, 21))().check()


@pytest.mark.parametrize("T", [0.4, 1.0, 50.0])
def test_limits_far_down_the_order(torch, T):
    """Each limit, alone and with the others, whose border has thousands of tokens before it in
    every chunk, and one chunk that holds the largest tokens."""
    say("sample far limits", T)
    grid = [dict(k=k, p=p, m=m, u=u) for k in (0, 127, 128, 129, 8191, 8192, 20000) for p in (1.0, 0.9999, 0.6)
            for m in (0.0, 1e-7, 1e-3, 0.5) for u in (0.37, 0.9999)]
    pick = {n: np.array([c[n] for c in grid]) for n in ("k", "p", "m", "u")}
    x = torch.randn(1, 41000, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda") * 2
    x[:, 8192:16384] += 3
    x = x.repeat(len(grid), 1)
    Call(torch, x, T=T, **pick)().check()
    Call(torch, x.half(), T=T, **pick)().check()
