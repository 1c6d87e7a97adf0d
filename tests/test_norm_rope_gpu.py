"""Normed heads, rotation by several axes and the cache write, and rows read back,
against a 64-bit computation from the formulas."""
import numpy as np
import pytest

import redline_amd as ra
from tests._util import say

pytestmark = pytest.mark.gpu
U32, U16 = 2.0 ** -24, 2.0 ** -11  # half a step of fp32, of fp16


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def axis_of_pair(half, sections, interleaved):
    if len(sections) < 2:
        return [0] * half
    if not interleaved:
        return [x for x, n in enumerate(sections) for _ in range(n)]
    given = [0] * len(sections)
    out = []
    for i in range(half):
        x = i % len(sections)
        take = given[x] < sections[x]
        given[x] += take
        out.append(x if take else 0)
    return out


def make(torch, T, hq, hkv, D, bs, cache, seed, axes=1, past=300, norm="qk", bias=False, amp=1.0):
    from redline_amd import kernels as K
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    cols = (hq + 2 * hkv) * D
    nb = T // bs + 3
    slots = rng.permutation(np.arange(bs, nb * bs))[:T].astype(np.int32)
    if T > 2:
        slots[T // 2] = -1
    c = {"T": T, "hq": hq, "hkv": hkv, "D": D, "bs": bs, "qkv": (rand(T, cols) * amp).half(),
         "slots": torch.from_numpy(slots).cuda(),
         "pos": torch.from_numpy(rng.integers(0, past, (axes, T)).astype(np.int32)).cuda(),
         "q_norm": (1 + 0.3 * rand(D)).half() if "q" in norm else None,
         "k_norm": (1 + 0.3 * rand(D)).half() if "k" in norm else None, "bias": rand(cols).half() if bias else None}
    cos, sin = ra.rope_cos_sin_tables(1e4, D, past)
    c["cos"], c["sin"] = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    shape = (nb, hkv, bs, D)
    c["sd"] = K.SCALE_F16 if cache == "int8_f16" else K.SCALE_F32
    if cache == "fp16":
        t = [torch.full(shape, 7.0, dtype=torch.float16, device="cuda") for _ in "kv"]
    else:
        sdt = torch.float16 if cache == "int8_f16" else torch.float32
        t = [torch.full(shape, 7, dtype=torch.int8, device="cuda") for _ in "kv"]
        t += [torch.full(shape[:3], 7.0, dtype=sdt, device="cuda") for _ in "kv"]
    c["cache"], c["view"] = t, K.kv_layer_view(*t)
    return c


def reference(torch, c, eps, sections=(), interleaved=False):
    """(y, bound): rotated q and k heads and v heads [T, heads, D] in 64 bits, and how far
    fp32 arithmetic may take y before it is rounded."""
    T, hq, hkv, D = c["T"], c["hq"], c["hkv"], c["D"]
    x = c["qkv"].double()
    if c["bias"] is not None:
        x = (x + c["bias"].double()).half().double()
    y = x.view(T, hq + 2 * hkv, D).clone()
    bound = torch.zeros_like(y)
    axis = torch.tensor(axis_of_pair(D // 2, sections, interleaved), device="cuda")
    row = c["pos"].long()[axis]  # [D/2, T]
    pair = torch.arange(D // 2, device="cuda")[:, None]
    co, si = c["cos"].double()[row, pair].T[:, None], c["sin"].double()[row, pair].T[:, None]
    for lo, hi, w in ((0, hq, c["q_norm"]), (hq, hq + hkv, c["k_norm"])):
        n = y[:, lo:hi]
        if w is not None:
            n = n / torch.sqrt((n * n).sum(-1, keepdim=True) / D + eps) * w.double()
        a, b = n[..., :D // 2], n[..., D // 2:]
        y[:, lo:hi] = torch.cat([a * co - b * si, b * co + a * si], -1)
        size = torch.cat([(a * co).abs() + (b * si).abs(), (b * co).abs() + (a * si).abs()], -1)
        # 16 + 3 sums of squares at most, halved by the root, / D, + eps, the root, 1 / x; two
        # products and three operations of the rotation: fewer than 24 roundings of fp32
        bound[:, lo:hi] = 24 * U32 * size
    return y, bound


def run(c, eps=1e-6, sections=(), interleaved=False, stream=None):
    from redline_amd import kernels as K
    K.rope_and_write_kv_norm(c["qkv"], c["pos"], c["slots"], c["T"], c["hq"], c["cos"], c["sin"], c["view"],
                             q_norm=c["q_norm"], k_norm=c["k_norm"], eps=eps, qkv_bias=c["bias"], scale_dtype=c["sd"],
                             sections=sections, interleaved=interleaved, stream=stream)


def check(torch, c, before, y, bound):
    from redline_amd import kernels as K
    T, hq, hkv, D, bs = (c[n] for n in ("T", "hq", "hkv", "D", "bs"))
    half = lambda v, b: b + U16 * (v.abs() + b) + 2.0 ** -25  # noqa: E731  rounded to fp16 once
    got = c["qkv"].view(T, -1, D)
    err = (got[:, :hq].double() - y[:, :hq]).abs()
    assert (err <= half(y, bound)[:, :hq]).all(), float(err.max())
    assert torch.equal(got[:, hq:], before.view(T, -1, D)[:, hq:])  # k and v sections stay
    k = torch.full((T, hkv * D), 9.0, dtype=torch.float16, device="cuda")
    v = k.clone()
    K.read_kv(c["view"], c["slots"], T, k, v, c["sd"])
    skip = c["slots"] < 0
    int8 = len(c["cache"]) > 2
    for rows, lo, i in ((k, hq, 0), (v, hq + hkv, 1)):
        rows = rows.view(T, hkv, D)
        assert (rows[skip] == 9.0).all()
        want, b = y[:, lo:lo + hkv], half(y, bound)[:, lo:lo + hkv]
        if i == 1:
            b = b * 0  # fp16 numbers, stored as they are
        s = c["slots"].long().clamp(min=0)
        cell = c["cache"][i][s // bs, :, s % bs].double()
        if int8:
            # half a code's step of a scale up to 2^-11 off, 2 fp32 roundings of the quotient
            # (a 127th of a step at most), and the product's rounding to fp16
            scale = c["cache"][2 + i][s // bs, :, s % bs].double()
            amax = want.abs().amax(-1)
            ideal = torch.where(amax > 0, amax / 127, 1.0)
            off = torch.where(amax > 0, b.amax(-1) / 127, 0.0)
            tol = off + (ideal + off) * (U16 if c["sd"] == K.SCALE_F16 else 4 * U32) + (2.0 ** -25 if c["sd"] else 0)
            assert ((scale - ideal).abs() <= tol)[~skip].all()
            cell = cell * scale[..., None]
            step = scale[..., None] * (0.5 + 127 * 3 * U32 + (127 * U16 if c["sd"] else 0))
            b = b + step
            assert (rows[~skip].double() - cell[~skip]).abs().le(U16 * cell[~skip].abs() + 2.0 ** -25).all()
        else:
            assert torch.equal(rows[~skip].double(), cell[~skip])
        err = (cell - want).abs()
        assert (err <= b)[~skip].all(), float(err[~skip].max())


CASES = [
    (1, 32, 8, 128, 16, "fp16", 1, (), False), (33, 28, 4, 128, 32, "int8", 1, (), False),
    (57, 4, 4, 64, 8, "fp16", 2, (20, 12), False), (130, 32, 4, 64, 16, "int8_f16", 3, (12, 10, 10), True),
    (64, 28, 4, 128, 16, "int8", 3, (16, 24, 24), False), (31, 5, 1, 128, 1, "fp16", 4, (40, 3, 2, 19), False),
    (75, 64, 8, 128, 24, "int8_f16", 4, (61, 1, 1, 1), True), (19, 16, 16, 64, 16, "int8", 4, (8, 8, 8, 8), True),
    (515, 40, 8, 128, 16, "fp16", 3, (0, 64, 0), False), (16, 0, 2, 64, 16, "fp16", 2, (31, 1), True),
]


@pytest.mark.parametrize("norm,bias", [("qk", False), ("", True), ("q", False), ("k", True)])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"T{c[0]}-{c[1]}x{c[2]}x{c[3]}-{c[5]}-{len(c[7])}ax{c[8]:d}")
def test_against_64_bits(torch, case, norm, bias):
    T, hq, hkv, D, bs, cache, axes, sections, turns = case
    say("norm_rope", case, norm, bias)
    c = make(torch, T, hq, hkv, D, bs, cache, T + axes, axes, norm=norm, bias=bias)
    before = c["qkv"].clone()
    y, b = reference(torch, c, 1e-6, sections, turns)
    run(c, 1e-6, sections, turns)
    check(torch, c, before, y, b)


@pytest.mark.parametrize("cache", ["fp16", "int8", "int8_f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bias", [False, True])
def test_without_norms_the_plain_write(torch, cache, D, bias):
    """No norms and one axis, or axes that all have the token's position: the bits of
    rope_and_write_kv_ex in q and in the cache."""
    from redline_amd import kernels as K
    say("norm_rope plain", cache, D, bias)
    half, got = D // 2, []
    for sections, turns in ((None, False), ((half // 2, half // 4, half // 4), False), ((half - 7, 4, 3), True)):
        c = make(torch, 83, 12, 4, D, 16, cache, 5, 3, norm="", bias=bias)
        c["pos"][1:] = c["pos"][0]
        if not got:
            p = make(torch, 83, 12, 4, D, 16, cache, 5, 3, norm="", bias=bias)
            K.rope_and_write_kv_ex(p["qkv"], p["pos"][0], p["slots"], 83, 12, p["cos"], p["sin"], p["view"], p["bias"],
                                   p["sd"])
            got = [p["qkv"], *p["cache"]]
        run(c, 1e-6, sections, turns)
        for a, b in zip(got, [c["qkv"], *c["cache"]]):
            assert torch.equal(a, b)


def test_largest_and_zero_rows(torch):
    """Rows of zeros (eps > 0), of the largest fp16 numbers (their squares pass fp16, not
    fp32) and of the smallest."""
    say("norm_rope rows of zeros, largest, smallest")
    c = make(torch, 12, 8, 2, 128, 16, "fp16", 3)
    c["qkv"][0:3] = 0
    c["qkv"][3:6] = 65504
    c["qkv"][6:9] = 2.0 ** -24
    before = c["qkv"].clone()
    y, b = reference(torch, c, 1e-6)
    run(c, 1e-6)
    check(torch, c, before, y, b)
    assert (c["qkv"][0:3, :8 * 128] == 0).all()


def test_lengths_views_streams_and_graphs(torch):
    """No tokens; qkv, positions and slots as views into longer ones; another stream; a
    captured call, replayed over new inputs."""
    from redline_amd import kernels as K
    say("norm_rope views, streams, graphs")
    sections = (40, 12, 12)
    c = make(torch, 50, 16, 2, 128, 16, "int8", 9, 3)
    untouched = [t.clone() for t in (c["qkv"], *c["cache"])]
    K.rope_and_write_kv_norm(c["qkv"], c["pos"], c["slots"], 0, 16, c["cos"], c["sin"], c["view"])
    K.read_kv(c["view"], c["slots"], 0)
    for a, b in zip(untouched, (c["qkv"], *c["cache"])):
        assert torch.equal(a, b)
    first = c["qkv"].clone()
    y, b = reference(torch, c, 1e-5, sections)
    # the same rows as the middle of a larger buffer
    wide = torch.full((54, c["qkv"].shape[1]), 3.0, dtype=torch.float16, device="cuda")
    wide[2:52] = first
    slots = torch.full((60,), -5, dtype=torch.int32, device="cuda")
    slots[3:53] = c["slots"]
    inner = {**c, "qkv": wide[2:52], "slots": slots[3:53]}
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    run(inner, 1e-5, sections, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    check(torch, inner, first, y, b)
    assert (wide[:2] == 3).all() and (wide[52:] == 3).all()
    eager = [wide[2:52].clone(), *[t.clone() for t in c["cache"]]]
    c["qkv"].copy_(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(c, 1e-5, sections)
    for _ in range(3):
        c["qkv"].copy_(first)
        for t in c["cache"]:
            t.fill_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c["qkv"], eager[0])
        on = c["slots"][c["slots"] >= 0].long()
        for t, e in zip(c["cache"], eager[1:]):
            assert torch.equal(t[on // 16, :, on % 16], e[on // 16, :, on % 16])


def test_only_the_given_cells_are_written(torch):
    say("norm_rope other cells")
    c = make(torch, 37, 4, 2, 64, 16, "int8_f16", 13)
    run(c)
    other = torch.ones(c["cache"][0].shape[0] * 16, dtype=torch.bool, device="cuda")
    other[c["slots"][c["slots"] >= 0].long()] = False
    at = other.nonzero()[:, 0]
    for t in c["cache"]:
        assert (t[at // 16, :, at % 16] == 7).all()


@pytest.mark.parametrize("int8", [False, True])
def test_cells_past_32_bits(torch, int8):
    """Cells whose bytes and elements lie past 2^32."""
    from redline_amd import kernels as K
    say("norm_rope far cells", int8)
    hq, hkv, D, bs = 2, 8, 128, 32
    nb = (1 << 33) // (hkv * bs * D * (1 if int8 else 2)) + 5
    shape = (nb, hkv, bs, D)
    t = [torch.empty(shape, dtype=torch.int8 if int8 else torch.float16, device="cuda") for _ in "kv"]
    t += [torch.empty(shape[:3], dtype=torch.float32, device="cuda") for _ in "kv"] if int8 else []
    c = make(torch, 40, hq, hkv, D, bs, "fp16", 17)
    c["cache"], c["view"] = t, K.kv_layer_view(*t)
    c["slots"] = nb * bs - 1 - torch.arange(40, device="cuda", dtype=torch.int32) * 3
    before = c["qkv"].clone()
    y, b = reference(torch, c, 1e-6)
    run(c)
    check(torch, c, before, y, b)


def test_read_one_output(torch):
    from redline_amd import kernels as K
    say("read_kv one output")
    c = make(torch, 20, 4, 2, 128, 16, "fp16", 23)
    run(c)
    both = [torch.zeros(20, 256, dtype=torch.float16, device="cuda") for _ in "kv"]
    K.read_kv(c["view"], c["slots"], 20, *both)
    for i, name in enumerate(("k_out", "v_out")):
        one = torch.zeros_like(both[0])
        K.read_kv(c["view"], c["slots"], 20, **{name: one})
        assert torch.equal(one, both[i])


def test_launchers_refuse(torch):
    from redline_amd import kernels as K
    say("norm_rope refusals")
    c = make(torch, 4, 4, 2, 64, 16, "int8", 2, 3)
    call = lambda **kw: run({**c, **kw}, sections=(16, 8, 8))  # noqa: E731
    for kw, text in ((dict(pos=c["pos"][:2].contiguous()), "positions holds"), (dict(sd=K.SCALE_F16), "scale dtype"),
                     (dict(slots=c["slots"][:3]), "slot_mapping holds"), (dict(q_norm=c["q_norm"][:63]), "q_norm holds"),
                     (dict(k_norm=c["k_norm"].float()), "k_norm must be"), (dict(qkv=c["qkv"].cpu()), "GPU tensor"),
                     (dict(bias=c["qkv"][0, :64].contiguous()), "qkv_bias holds")):
        with pytest.raises(ra.Error, match=text):
            call(**kw)
    with pytest.raises(ra.Error, match="at most 4"):
        run(c, sections=(8, 8, 8, 4, 4))
    with pytest.raises(ra.Error, match="pairs"):
        run(c, sections=(16, 8, 7))
    out = torch.zeros(4, 128, dtype=torch.float16, device="cuda")
    with pytest.raises(ra.Error, match="k_out holds"):
        K.read_kv(c["view"], c["slots"], 4, out[:3].contiguous())
    with pytest.raises(ra.Error, match="scale dtype"):
        K.read_kv(c["view"], c["slots"], 4, out, out.clone(), K.SCALE_F16)
    k, v, ks, vs = c["cache"]
    for args, text in (((k, v[:2], ks, vs), "one shape"), ((k, v, ks, vs.half()), "v_scale must be"),
                       ((k, v), "k must be"), ((k.half(), v.half(), None, vs), "without k_scale"),
                       ((k, v, ks[:1], vs), "k_scale holds")):
        with pytest.raises(ra.Error, match=text):
            K.kv_layer_view(*args)
