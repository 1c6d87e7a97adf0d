"""Operators of a step that draws many continuations of one prompt, as measurable cases.

Kinds of cases:

  write   RMS norm of each query and key head, rotation by one to four position
          axes (time, height, width, ...) and the write of k/v into the paged
          cache, then the rows just written read back as fp16
  attend  attention of one new token per item, for groups of items that share
          their first tokens in the cache
  sample  the next token of each row of logits, by temperature, top-k, top-p and
          min-p, from one given random number a row

With `own` false, run() computes them with elementary torch operations; with
`own` true it calls the launchers of redline_amd.kernels.

An INT8 cache holds codes and one scale per (token, kv head): scale = amax / 127
(1 for a row of zeros), code = round(x / scale); with "int8_f16" the scale is
rounded to fp16 first.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DEV = "cuda"
_LLAMA = {"hq": 32, "hkv": 8, "dim": 128}
_QWEN2 = {"hq": 28, "hkv": 4, "dim": 128}
_TINY = {"hq": 32, "hkv": 4, "dim": 64}


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # The cache write of a decode step with normed heads: launch-bound.
        {"name": "write_decode_b32", "kind": "write", "cache": "fp16", "prompts": 0, "prompt_max": 0, "decodes": 32,
         "past_max": 8191, "block": 16, "norm": True, "bias": False, "sections": "", "interleaved": False,
         "spread": 1, **_LLAMA},
        # Ragged prompts with images beside decoding sequences, D = 64 heads, three
        # axes that take turns over the pairs, INT8 cache.
        {"name": "write_mixed_d64_int8", "kind": "write", "cache": "int8", "prompts": 9, "prompt_max": 900,
         "decodes": 61, "past_max": 2000, "block": 32, "norm": True, "bias": False, "sections": "12 10 10",
         "interleaved": True, "spread": 2, **_TINY},
        # A large prompt step with images: a QKV bias, three axes in sections, INT8
        # cache with fp16 scales.
        {"name": "write_axes_16k_int8", "kind": "write", "cache": "int8_f16", "prompts": 4, "prompt_max": 4096,
         "decodes": 0, "past_max": 4096, "block": 16, "norm": False, "bias": True, "sections": "16 24 24",
         "interleaved": False, "spread": 3, **_QWEN2},
        # A prompt step of normed heads into an FP16 cache.
        {"name": "write_prefill_8k", "kind": "write", "cache": "fp16", "prompts": 5, "prompt_max": 3000, "decodes": 17,
         "past_max": 3000, "block": 16, "norm": True, "bias": False, "sections": "", "interleaved": False,
         "spread": 4, **_LLAMA},
        # Four drafts of a small model's answer to one prompt: latency counts.
        {"name": "attend_b4_1k_d64", "kind": "attend", "cache": "fp16", "groups": 1, "items_max": 4, "prefix_max": 1000,
         "suffix_max": 60, "block": 16, "spread": 5, **_TINY},
        # 32 answers to one long document.
        {"name": "attend_b32_8k", "kind": "attend", "cache": "fp16", "groups": 1, "items_max": 32, "prefix_max": 8192,
         "suffix_max": 512, "block": 16, "spread": 6, **_LLAMA},
        # A server's batch: groups of 1 to 24 requests with a system prompt each, INT8.
        {"name": "attend_groups_int8", "kind": "attend", "cache": "int8", "groups": 7, "items_max": 24,
         "prefix_max": 4000, "suffix_max": 1500, "block": 16, "spread": 7, **_LLAMA},
        # 64 answers to one very long prompt, seven query heads to a kv head.
        {"name": "attend_b64_32k", "kind": "attend", "cache": "fp16", "groups": 1, "items_max": 64,
         "prefix_max": 32768, "suffix_max": 2000, "block": 32, "spread": 8, **_QWEN2},
        # One user of a small model: latency counts.
        {"name": "sample_b1_v32k", "kind": "sample", "rows": 1, "vocab": 32000, "fp32": False, "mode": "usual",
         "masked": 0.0, "spread": 9},
        # A decode step's rows, each with its own settings.
        {"name": "sample_b32_mixed", "kind": "sample", "rows": 32, "vocab": 128256, "fp32": False, "mode": "mixed",
         "masked": 0.0, "spread": 10},
        # A full batch, nucleus sampling over logits in 32 bits.
        {"name": "sample_b256_nucleus", "kind": "sample", "rows": 256, "vocab": 152064, "fp32": True,
         "mode": "nucleus", "masked": 0.0, "spread": 11},
        # Answers held to a grammar that forbids most tokens; sampling from all that is left.
        {"name": "sample_b20_masked", "kind": "sample", "rows": 20, "vocab": 128256, "fp32": True, "mode": "open",
         "masked": 0.9, "spread": 12},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    hkv = rng.choice([1, 2, 4, 8])
    return {"hq": hkv * rng.choice([1, 2, 3, 4, 5, 7, 8]), "hkv": hkv, "dim": rng.choice([64, 128])}


def _draw_sections(rng, half):
    """Sections of two to four axes and whether they take turns."""
    n = rng.choice([2, 3, 3, 4])
    if rng.random() < 0.5:  # turns: the later axes have at most their share
        rest = [rng.randint(1, half // n) for _ in range(n - 1)]
        return " ".join(str(n) for n in [half - sum(rest)] + rest), True
    if rng.random() < 0.5:
        cut = sorted(rng.sample(range(1, half // 8), n - 1))
        cut = [8 * c for c in cut]
    else:
        cut = sorted(rng.sample(range(1, half), n - 1))
    return " ".join(str(b - a) for a, b in zip([0] + cut, cut + [half])), False


def draw(rng):
    kind = rng.choice(["write", "write", "attend", "attend", "sample", "sample"])
    c = {"kind": kind, "spread": rng.randrange(1000, 1 << 20)}
    if kind == "sample":
        vocab = _log_int(rng, 50, 152064)
        return {**c, "vocab": vocab, "rows": _log_int(rng, 1, min(256, 38_000_000 // vocab)),
                "fp32": rng.random() < 0.5, "mode": rng.choice(["usual", "mixed", "nucleus", "open", "mixed"]),
                "masked": rng.choice([0.0, 0.0, 0.5, 0.98])}
    c |= {"cache": rng.choice(["fp16", "fp16", "int8", "int8_f16"]), "block": rng.choice([8, 16, 16, 32]),
          **_heads(rng)}
    if kind == "write":
        sections, turns = _draw_sections(rng, c["dim"] // 2) if rng.random() < 0.6 else ("", False)
        return {**c, "prompts": rng.randrange(0, 6), "prompt_max": _log_int(rng, 5, 2500),
                "decodes": _log_int(rng, 1, 200), "past_max": _log_int(rng, 20, 6000), "norm": rng.random() < 0.7,
                "bias": rng.random() < 0.3, "sections": sections, "interleaved": turns}
    groups, prefix, suffix = _log_int(rng, 1, 12), _log_int(rng, 8, 30000), _log_int(rng, 1, 2000)
    items = max(1, min(64 // groups, 250000 // (groups * (prefix + suffix))))
    return {**c, "groups": groups, "items_max": _log_int(rng, 1, items) if items > 1 else 1, "prefix_max": prefix,
            "suffix_max": suffix}


def _sections(case):
    """Pairs of each position axis; empty: one axis."""
    return [int(n) for n in case["sections"].split()]


def _segments(case):
    """[(past, new)] of a write step's sequences, from the case alone."""
    rng = np.random.default_rng(case["spread"])
    segs = []
    for _ in range(case["prompts"]):
        n = int(rng.integers(max(1, case["prompt_max"] // 4), case["prompt_max"] + 1))
        if case["decodes"] == 0:
            n = case["prompt_max"]
        segs.append((int(rng.integers(0, case["past_max"] + 1)) if rng.random() < 0.6 else 0, n))
    for _ in range(case["decodes"]):
        segs.append((int(rng.integers(0, case["past_max"] + 1)), 1))
    return [segs[i] for i in rng.permutation(len(segs))]


def _groups(case):
    """[(prefix, [suffix of each item, the new token included])], from the case alone."""
    rng = np.random.default_rng(case["spread"])
    out = []
    for _ in range(case["groups"]):
        if case["groups"] == 1:
            n, prefix = case["items_max"], case["prefix_max"]
        else:
            n = int(rng.integers(1, case["items_max"] + 1))
            prefix = int(rng.integers(case["prefix_max"] // 8, case["prefix_max"] + 1))
        out.append((prefix, [int(x) for x in rng.integers(1, case["suffix_max"] + 1, n)]))
    return out


def work(case):
    if case["kind"] == "sample":
        R, V = case["rows"], case["vocab"]
        # each logit once, five numbers in and two out a row; an exponential and
        # a sum each
        return {"bytes": R * V * (4 if case["fp32"] else 2) + R * 28, "flops": R * V * 2}
    hq, hkv, D = case["hq"], case["hkv"], case["dim"]
    int8 = case["cache"] != "fp16"
    cell = 2 * hkv * D * (1 if int8 else 2) + (2 * hkv * (2 if case["cache"] == "int8_f16" else 4) if int8 else 0)
    if case["kind"] == "write":
        T, axes = sum(n for _, n in _segments(case)), max(1, len(_sections(case)))
        rope = T * (2 * (hq + 2 * hkv) * D + 2 * hq * D + cell + 4 * D + 4 * axes + 4)
        return {"bytes": rope + T * (cell + 4 * hkv * D + 4), "flops": T * (hq + hkv) * D * (7 if case["norm"] else 3)}
    keys = pairs = items = blocks = 0
    for prefix, suffix in _groups(case):
        keys += prefix + sum(suffix)
        pairs += prefix * len(suffix) + sum(suffix)
        items += len(suffix)
        blocks += -(-prefix // case["block"]) + sum(-(-s // case["block"]) for s in suffix)
    return {"bytes": keys * cell + items * hq * D * 4 + 4 * blocks, "flops": pairs * hq * D * 4}


# ------------------------------------------------------------------ the inputs

def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(_DEV)


def _int32(a):
    return _dev(np.asarray(a, np.int32))


def _rounded_scale(s, cache):
    return s.half() if cache == "int8_f16" else s.float()


def _quantised(x, cache):
    """Codes and scales of rows x [..., D] (fp32)."""
    amax = x.abs().amax(-1)
    scale = _rounded_scale(torch.where(amax > 0, amax / 127.0, torch.ones_like(amax)), cache)
    codes = (x * (1.0 / scale.float()[..., None])).clamp(-127, 127).round().to(torch.int8)
    return codes, scale


def _pool(st, k, v, cache):
    if cache == "fp16":
        st["k"], st["v"], st["k_scale"], st["v_scale"] = k.half(), v.half(), None, None
    else:
        st["k"], st["k_scale"] = _quantised(k, cache)
        st["v"], st["v_scale"] = _quantised(v, cache)


def prepare(case, seed):
    rng = np.random.default_rng([seed, case["spread"]])
    g = torch.Generator(device=_DEV).manual_seed(seed)
    return {"write": _prepare_write, "attend": _prepare_attend, "sample": _prepare_sample}[case["kind"]](case, rng, g)


def _prepare_write(case, rng, g):
    segs, bs = _segments(case), case["block"]
    hq, hkv, D = case["hq"], case["hkv"], case["dim"]
    past, new = np.array([s[0] for s in segs]), np.array([s[1] for s in segs])
    T, first, last = int(new.sum()), past // bs, (past + new - 1) // bs
    # only the blocks that the step writes, scattered over the pool; block 0 is scratch
    have = last - first + 1
    nb = int(have.sum()) + 1
    ids = rng.permutation(np.arange(1, nb))
    start, q_start = np.cumsum(have) - have, np.cumsum(new) - new
    seq = np.repeat(np.arange(len(segs)), new)
    pos = past[seq] + np.arange(T) - q_start[seq]
    slots = ids[start[seq] + pos // bs - first[seq]] * bs + pos % bs
    axes = max(1, len(_sections(case)))
    at = np.repeat(pos[None], axes, 0)
    for s, (p, n) in enumerate(segs):  # the middle of a prompt is an image: its rows and columns count alone
        if axes > 1 and n > 12:
            a, b, w = n // 4, 3 * n // 4, int(rng.integers(3, 40))
            i, t0 = np.arange(b - a), q_start[s] + a
            at[0, t0:t0 + b - a] = p + a
            for x in range(1, axes):
                at[x, t0:t0 + b - a] = p + a + (i // w if x % 2 else i % w)
    inv = 1.0 / (5e5 ** (torch.arange(D // 2, device=_DEV, dtype=torch.float64) * 2 / D))
    ang = torch.arange(int((past + new).max()) + 1, device=_DEV, dtype=torch.float64)[:, None] * inv
    cols = (hq + 2 * hkv) * D
    gain = torch.ones(hkv, D, device=_DEV)  # keys with a few strong channels, as trained models have them
    gain[:, torch.from_numpy(rng.permutation(D)[:3]).to(_DEV)] = 6.0
    qkv = torch.randn(T, cols, generator=g, device=_DEV)
    qkv[:, hq * D:(hq + hkv) * D] *= gain.reshape(1, -1)
    qkv *= torch.exp2(torch.rand(T, 1, generator=g, device=_DEV) * 3 - 1)
    st = {"case": dict(case), "T": T, "qkv": qkv.half(), "positions": _int32(at if axes > 1 else pos),
          "slots": _int32(slots), "cos": ang.cos().float(), "sin": ang.sin().float(), "eps": 1e-6,
          "bias": torch.randn(cols, generator=g, device=_DEV).half() if case["bias"] else None}
    for w in ("q_norm", "k_norm"):
        st[w] = (1 + 0.2 * torch.randn(D, generator=g, device=_DEV)).half() if case["norm"] else None
    shape = (nb, hkv, bs, D)
    _pool(st, torch.randn(shape, generator=g, device=_DEV), torch.randn(shape, generator=g, device=_DEV),
          case["cache"])
    st["k_rows"] = torch.zeros(T, hkv * D, dtype=torch.float16, device=_DEV)
    st["v_rows"] = torch.zeros_like(st["k_rows"])
    return st


def _prepare_attend(case, rng, g):
    bs, groups = case["block"], _groups(case)
    hq, hkv, D = case["hq"], case["hkv"], case["dim"]
    S = sum(len(s) for _, s in groups)
    ctx = np.concatenate([p + np.array(s) for p, s in groups])
    mb = int(-(-ctx.max() // bs))
    total = sum(p // bs + sum(-(-(p + x) // bs) - p // bs for x in s) for p, s in groups)
    ids = rng.permutation(np.arange(1, total + 1))
    tables = np.zeros((S, mb), np.int64)
    at = item = 0
    copies = []  # a block that the prefix ends inside: each item has its own copy
    for p, s in groups:
        full = p // bs
        shared, first = ids[at:at + full], item
        at += full
        for x in s:
            n = -(-(p + x) // bs) - full
            tables[item, :full], tables[item, full:full + n] = shared, ids[at:at + n]
            if p % bs and item > first:
                copies.append((tables[first, full], tables[item, full]))
            at += n
            item += 1
    gain = torch.ones(hkv, 1, D, device=_DEV)
    gain[:, :, torch.from_numpy(rng.permutation(D)[:3]).to(_DEV)] = 6.0
    shape = (total + 1, hkv, bs, D)
    k = torch.randn(shape, generator=g, device=_DEV) * gain
    v = torch.randn(shape, generator=g, device=_DEV)
    v *= torch.exp2(torch.randint(-3, 2, (total + 1, hkv, 1, 1), generator=g, device=_DEV).float())
    for a, b in copies:
        k[b], v[b] = k[a], v[a]
    starts = np.cumsum([0] + [len(s) for _, s in groups])
    st = {"case": dict(case), "S": S, "max_blocks": mb, "tables": _int32(tables), "positions": _int32(ctx - 1),
          "items": _int32(np.arange(S)), "group_start": _int32(starts), "prefix": _int32([p for p, _ in groups]),
          "max_items": max(len(s) for _, s in groups), "max_prefix": max(p for p, _ in groups),
          "max_suffix": max(max(s) for _, s in groups), "scale": D ** -0.5,
          # q as the first heads of a qkv row, as the engine keeps it
          "q_stride": (hq + 2 * hkv) * D, "out": torch.zeros(S, hq * D, dtype=torch.float16, device=_DEV)}
    st["q"] = (torch.randn(S, st["q_stride"], generator=g, device=_DEV) * 1.5).half()
    _pool(st, k, v, case["cache"])
    return st


def _prepare_sample(case, rng, g):
    R, V = case["rows"], case["vocab"]
    # a bulk of unlikely tokens and a tail of likely ones
    l = torch.randn(R, V, generator=g, device=_DEV) * 2
    l -= 1.6 * torch.log(torch.rand(R, V, generator=g, device=_DEV).clamp(min=1e-12))
    if case["masked"] > 0:
        hide = torch.rand(R, V, generator=g, device=_DEV) < case["masked"]
        hide[:, int(rng.integers(0, V))] = False
        l.masked_fill_(hide, -math.inf)
    z = np.zeros
    mode = np.array([case["mode"]] * R)
    if case["mode"] == "mixed":
        mode = rng.choice(["greedy", "usual", "nucleus", "open", "top_k", "min_p"], R)
    temperature, top_k, top_p, min_p = z(R, np.float32), z(R, np.int32), np.ones(R, np.float32), z(R, np.float32)
    for r, m in enumerate(mode):
        temperature[r] = 0.0 if m == "greedy" else rng.choice([0.6, 0.7, 0.8, 1.0, 1.3])
        top_k[r] = {"usual": rng.integers(20, 100), "top_k": rng.integers(1, 2000)}.get(m, 0)
        top_p[r] = {"usual": 0.95, "nucleus": rng.uniform(0.5, 0.99)}.get(m, 1.0)
        min_p[r] = {"min_p": rng.uniform(0.01, 0.2)}.get(m, 0.0)
    # rows of the settings in an order of their own, as a batch builder lays them out
    order = rng.permutation(R)
    back = np.argsort(order)
    st = {"case": dict(case), "logits": l if case["fp32"] else l.half(), "param_row": _int32(order),
          "uniform": torch.rand(R, generator=g, device=_DEV), "tokens": _int32(z(R)),
          "logprobs": torch.zeros(R, device=_DEV)}
    for n, a in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
        st[n] = _dev(a[back])
    return st


# ------------------------------------------------------------ the plain forms

def _axis_of_pair(case, half):
    s = _sections(case)
    if not s:
        return [0] * half
    if not case["interleaved"]:
        return [a for a, n in enumerate(s) for _ in range(n)]
    return [i % len(s) if i < len(s) * s[i % len(s)] else 0 for i in range(half)]


def _plain_write(st):
    c = st["case"]
    hq, hkv, D, bs, T = c["hq"], c["hkv"], c["dim"], c["block"], st["T"]
    x = st["qkv"].float()
    if st["bias"] is not None:
        x = (x + st["bias"].float()).half().float()
    x = x.view(T, hq + 2 * hkv, D)
    qk = x[:, :hq + hkv]
    if st["q_norm"] is not None:
        w = torch.cat([st["q_norm"].float().expand(hq, D), st["k_norm"].float().expand(hkv, D)])
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + st["eps"]) * w
    pos = st["positions"].long().view(-1, T)
    axis = torch.tensor(_axis_of_pair(c, D // 2), device=_DEV)
    pair = torch.arange(D // 2, device=_DEV)
    row = pos[axis].T  # [T, D / 2]
    co, si = st["cos"][row, pair][:, None], st["sin"][row, pair][:, None]
    a, b = qk[..., :D // 2], qk[..., D // 2:]
    qk = torch.cat([a * co - b * si, b * co + a * si], -1).half()
    st["qkv"].view(T, hq + 2 * hkv, D)[:, :hq] = qk[:, :hq]
    blk, off = st["slots"].long() // bs, st["slots"].long() % bs
    for rows, n in ((qk[:, hq:], "k"), (x[:, hq + hkv:], "v")):
        if c["cache"] == "fp16":
            st[n][blk, :, off] = rows.half()
        else:
            codes, scale = _quantised(rows.float(), c["cache"])
            st[n][blk, :, off] = codes
            st[n + "_scale"][blk, :, off] = scale
    out = {"qkv": st["qkv"]}
    for n in "kv":
        y = st[n][blk, :, off].float()
        if c["cache"] != "fp16":
            y = y * st[n + "_scale"][blk, :, off].float()[..., None]
        out[n] = y.half().view(T, -1)
    return out


def _plain_attend(st):
    c, t = st["case"], st["tables"].long()
    hq, hkv, D, bs, S = c["hq"], c["hkv"], c["dim"], c["block"], st["S"]

    def rows(n):  # [S, hkv, max_blocks * bs, D]
        x = st[n][t.view(-1)].float()
        if st[n + "_scale"] is not None:
            x *= st[n + "_scale"][t.view(-1)].float()[..., None]
        return x.view(S, -1, hkv, bs, D).transpose(1, 2).reshape(S, hkv, -1, D)

    k = rows("k")
    q = st["q"][:, :hq * D].float().view(S, hkv, hq // hkv, D)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(st["scale"])
    del k
    late = torch.arange(s.shape[-1], device=_DEV)[None] > st["positions"].long()[:, None]
    s.masked_fill_(late[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(s, rows("v")) / s.sum(-1, keepdim=True)
    return o.reshape(S, hq * D).half()


def _plain_sample(st):
    V = st["case"]["vocab"]
    at = st["param_row"].long()
    T, top_k, top_p, min_p = (st[n][at][:, None] for n in ("temperature", "top_k", "top_p", "min_p"))
    vals, order = torch.sort(st["logits"], dim=1, descending=True, stable=True)
    greedy = T <= 0
    w = torch.exp((vals.double() - vals[:, :1].double()) / torch.where(greedy, 1.0, T).double())
    rank = torch.arange(V, device=_DEV)[None]
    w *= (top_k <= 0) | (rank < top_k)
    run_to = w.cumsum(1)
    before = torch.cat([torch.zeros_like(run_to[:, :1]), run_to[:, :-1]], 1)
    keep = (top_p >= 1) | (before < top_p.double() * run_to[:, -1:])
    keep &= w >= min_p.double()
    keep[:, 0] = True
    n = keep.sum(1, keepdim=True)
    mass = run_to.gather(1, n - 1)
    j = torch.minimum((run_to <= st["uniform"].double()[:, None] * mass).sum(1, keepdim=True), n - 1)
    j = torch.where(greedy, 0, j)
    lp = torch.where(greedy, 0.0, torch.log(w.gather(1, j) / mass))
    return {"tokens": order.gather(1, j)[:, 0].int(), "logprobs": lp[:, 0].float()}


# --------------------------------------------------- the framework's launchers

def _plan(st):
    """The views, work descriptions and workspaces that an engine builds once and keeps."""
    from redline_amd import kernels as K
    c = st["case"]
    if c["kind"] == "sample":
        ws = K.SamplingWorkspace(c["rows"], c["vocab"])
        return K.sampling_work(st["logits"], c["rows"], c["vocab"], st["temperature"], st["top_k"], st["top_p"],
                               st["uniform"], st["tokens"], ws, min_p=st["min_p"], param_row=st["param_row"],
                               logprobs=st["logprobs"])
    sd = K.SCALE_F16 if c["cache"] == "int8_f16" else K.SCALE_F32
    kv = K.kv_layer_view(st["k"], st["v"], st["k_scale"], st["v_scale"])
    if c["kind"] == "write":
        return kv, sd
    p = K.attention_params(st["q"], st["q_stride"], st["out"], c["hq"], st["scale"], kv, st["tables"],
                           st["max_blocks"], st["positions"])
    part = K.kDecodePartitionSize
    pre, suf = -(-st["max_prefix"] // part), -(-st["max_suffix"] // part)
    ws = K.DecodeWorkspace(st["S"], c["hq"], pre + suf, c["dim"])
    w = K.shared_prefix_work(st["items"], st["items"], st["S"], st["group_start"], st["prefix"], c["groups"],
                             st["max_items"], pre, suf, ws)
    return p, w, sd


def _own(st):
    from redline_amd import kernels as K
    if "plan" not in st:
        st["plan"] = _plan(st)
    plan, c = st["plan"], st["case"]
    if c["kind"] == "sample":
        K.sample_tokens(plan)
        return {"tokens": st["tokens"], "logprobs": st["logprobs"]}
    if c["kind"] == "attend":
        K.paged_attention_decode_shared(plan[0], plan[1], plan[2])
        return st["out"]
    kv, sd = plan
    K.rope_and_write_kv_norm(st["qkv"], st["positions"], st["slots"], st["T"], c["hq"], st["cos"], st["sin"], kv,
                             q_norm=st["q_norm"], k_norm=st["k_norm"], eps=st["eps"], qkv_bias=st["bias"],
                             scale_dtype=sd, sections=_sections(c), interleaved=c["interleaved"])
    K.read_kv(kv, st["slots"], st["T"], st["k_rows"], st["v_rows"], sd)
    return {"qkv": st["qkv"], "k": st["k_rows"], "v": st["v_rows"]}


def run(st):
    if own:
        return _own(st)
    return {"write": _plain_write, "attend": _plain_attend, "sample": _plain_sample}[st["case"]["kind"]](st)


# --------------------------------------------------------- from the definition

def _exact_write(st):
    c = st["case"]
    hq, hkv, D, T, half = c["hq"], c["hkv"], c["dim"], st["T"], c["dim"] // 2
    x = st["qkv"].double()
    if st["bias"] is not None:
        x = (x + st["bias"].double()).half().double()
    heads = list(x.view(T, hq + 2 * hkv, D).unbind(1))
    sections = _sections(c) or [half]
    for h in range(hq + hkv):
        y = heads[h]
        w = st["q_norm" if h < hq else "k_norm"]
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / D + st["eps"]) * w.double()
        z = torch.empty_like(y)
        first, free = 0, set(range(half))
        for a in [*range(1, len(sections)), 0]:  # axis 0 takes what the others leave
            if a == 0:
                pairs = sorted(free)
            elif c["interleaved"]:
                pairs = [a + len(sections) * j for j in range(sections[a])]
            else:
                first = sum(sections[:a])
                pairs = list(range(first, first + sections[a]))
            free -= set(pairs)
            i = torch.tensor(pairs, device=_DEV)
            p = st["positions"].view(-1, T)[a].long()
            co, si = st["cos"].double()[p][:, i], st["sin"].double()[p][:, i]
            z[:, i] = y[:, i] * co - y[:, i + half] * si
            z[:, i + half] = y[:, i + half] * co + y[:, i] * si
        heads[h] = z
    out = {"qkv": torch.cat([torch.cat(heads[:hq], 1), st["qkv"].double()[:, hq * D:]], 1)}
    for n, lo in (("k", hq), ("v", hq + hkv)):
        rows = []
        for y in heads[lo:lo + hkv]:
            if c["cache"] != "fp16":
                y = y.half().double()
                amax = y.abs().max(-1, keepdim=True).values
                s = torch.where(amax > 0, amax / 127, 1.0)
                s = s.half().double() if c["cache"] == "int8_f16" else s
                y = (y / s).clamp(-127, 127).round() * s
            rows.append(y)
        out[n] = torch.cat(rows, 1)
    return out


def _exact_attend(st):
    c = st["case"]
    hq, hkv, D, bs = c["hq"], c["hkv"], c["dim"], c["block"]
    out, s = [], 0
    for prefix, suffix in _groups(c):
        for x in suffix:
            n = prefix + x
            blocks = st["tables"][s, :-(-n // bs)].long()
            row = []
            for h in range(hkv):
                kv = []
                for a in "kv":
                    y = st[a][blocks, h].double()
                    if st[a + "_scale"] is not None:
                        y = y * st[a + "_scale"][blocks, h].double()[..., None]
                    kv.append(y.reshape(-1, D)[:n])
                q = st["q"][s, h * hq // hkv * D:(h + 1) * hq // hkv * D].double().view(-1, D)
                row.append((torch.softmax(q @ kv[0].T * st["scale"], -1) @ kv[1]).view(-1))
            out.append(torch.cat(row))
            s += 1
    return torch.stack(out)


def _exact_sample(st):
    """The log-probability of each row's draw, from probabilities of the whole row."""
    lp = []
    for r in range(st["case"]["rows"]):
        a = int(st["param_row"][r])
        T, k, p, m = (float(st[n][a]) for n in ("temperature", "top_k", "top_p", "min_p"))
        if T <= 0:
            lp.append(torch.zeros((), dtype=torch.float64, device=_DEV))
            continue
        q = torch.softmax(st["logits"][r].double() / T, 0)
        q = q[torch.argsort(-st["logits"][r].float(), stable=True)]
        if k > 0:
            q = q[:int(k)]
        most = q[0]
        total = q.cumsum(0)
        if p < 1:
            q = q[:1 + int((total[:-1] < p * total[-1]).sum())]
        q = q[:max(1, int((q / most >= m).sum()))]
        total = q.cumsum(0)
        j = min(int((total <= float(st["uniform"][r]) * total[-1]).sum()), len(q) - 1)
        lp.append(torch.log(q[j]) - torch.log(total[-1]))
    return {"tokens": None, "logprobs": torch.stack(lp)}


def exact(case, seed):
    st = prepare(case, seed)
    return {"write": _exact_write, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](st)
