"""The operators of the block-scaled 8-bit KV cache, as measurable cases.

A block-scaled cache holds K and V in 8 bits (INT8, or FP8 e4m3) with one
scale for each (block of tokens, kv head).  Its scales are 0 (nothing but
zeros in the block) or powers of two from 2^-24 on.  Kinds of cases:

  tables   block tables, slot maps and work lists of a step, built on the GPU
           from request lengths and a ring of free blocks
  write    RoPE on a step's q/k heads and the write of its k/v rows into the
           cache, then the stored rows of the blocks it touched read back as
           fp16 (what attention sees)
  decode   attention of one new token per sequence over the cache
  prefill  causal attention of several new tokens per sequence over the cache

With `own` false, run() computes them with elementary torch operations; with
`own` true it calls the launchers of redline_amd.kernels.

The byte layout of a block (block_size = 16 t tokens, head_dim D = 16 E):
  K  [t][E pieces p][16 tokens][2 halves h][8 e]   holds dim  h D/2 + 8 p + e
  V  [t][E/4 g][4 quads r][16 m][4 j][4 i]         holds dim  E m + 4 g + j
                                                   of token   4 r + i
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
        # A decode step of 32 chats: one new token each, a block for some of them.
        {"name": "tables_decode_b32", "kind": "tables", "prompts": 0, "prompt_min": 0, "prompt_max": 0,
         "decodes": 32, "past_max": 8191, "ended": 0, "block": 16, "spread": 1},
        # A mixed step of a loaded server: prompts in chunks beside 2048
        # decoding sequences, some sequences ending.
        {"name": "tables_mixed_2k", "kind": "tables", "prompts": 6, "prompt_min": 100, "prompt_max": 1024,
         "decodes": 2048, "past_max": 8191, "ended": 40, "block": 16, "spread": 2},
        # A prefill step of 16k tokens.
        {"name": "tables_prefill_16k", "kind": "tables", "prompts": 5, "prompt_min": 1000,
         "prompt_max": 4096, "decodes": 3, "past_max": 8191, "ended": 2, "block": 16, "spread": 3},
        # The cache write of a decode step: launch-bound.
        {"name": "write_decode_b32_int8", "kind": "write", "fmt": "int8", "prompts": 0, "prompt_min": 0,
         "prompt_max": 0, "decodes": 32, "past_max": 8191, "block": 16, "bias": False, "spread": 4, **_LLAMA},
        # Ragged prompts beside decoding sequences, D = 64 heads, blocks of 32.
        {"name": "write_mixed_d64_int8", "kind": "write", "fmt": "int8", "prompts": 9, "prompt_min": 37,
         "prompt_max": 900, "decodes": 61, "past_max": 2000, "block": 32, "bias": False, "spread": 5, **_TINY},
        # A large prefill step with a QKV bias.
        {"name": "write_prefill_16k_fp8", "kind": "write", "fmt": "fp8", "prompts": 4, "prompt_min": 4096,
         "prompt_max": 4096, "decodes": 0, "past_max": 4096, "block": 16, "bias": True, "spread": 6, **_QWEN2},
        # One user chatting with a small model: latency counts.
        {"name": "decode_b1_2k_d64", "kind": "decode", "fmt": "int8", "decodes": 1, "past_min": 1700,
         "past_max": 2000, "block": 16, "spread": 7, **_TINY},
        # A full decode batch, contexts to 8192 keys.
        {"name": "decode_b32_8k_int8", "kind": "decode", "fmt": "int8", "decodes": 32, "past_min": 0,
         "past_max": 8191, "block": 16, "spread": 8, **_LLAMA},
        # Long contexts, seven query heads to a kv head.
        {"name": "decode_b12_40k_fp8", "kind": "decode", "fmt": "fp8", "decodes": 12, "past_min": 2000,
         "past_max": 40000, "block": 32, "spread": 9, **_QWEN2},
        # Two prompt chunks at some depth: a chunked-prefill step.
        {"name": "prefill_chunks_fp8", "kind": "prefill", "fmt": "fp8", "prompts": 2, "prompt_min": 512,
         "prompt_max": 512, "past_max": 2000, "block": 16, "spread": 10, **_LLAMA},
        # Many short ragged prompts of a small model.
        {"name": "prefill_ragged_d64", "kind": "prefill", "fmt": "int8", "prompts": 24, "prompt_min": 20,
         "prompt_max": 900, "past_max": 500, "block": 32, "spread": 11, **_TINY},
        # Long prompts: matrix-bound.
        {"name": "prefill_4x4k_int8", "kind": "prefill", "fmt": "int8", "prompts": 4, "prompt_min": 4096,
         "prompt_max": 4096, "past_max": 4096, "block": 16, "spread": 12, **_LLAMA},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    hkv = rng.choice([1, 2, 4, 8])
    return {"hq": hkv * rng.choice([1, 2, 3, 4, 5, 7, 8]), "hkv": hkv, "dim": rng.choice([64, 128])}


def draw(rng):
    kind = rng.choice(["tables", "write", "decode", "decode", "prefill"])
    c = {"kind": kind, "block": rng.choice([16, 16, 32]), "spread": rng.randrange(1000, 1 << 20)}
    if kind == "tables":
        hi = _log_int(rng, 20, 4096)
        return {**c, "prompts": rng.randrange(0, 5), "prompt_min": max(1, hi // 5), "prompt_max": hi,
                "decodes": _log_int(rng, 1, 2000), "past_max": _log_int(rng, 20, 8000),
                "ended": rng.randrange(0, 9)}
    c |= {"fmt": rng.choice(["int8", "fp8"]), **_heads(rng)}
    if kind == "write":
        hi = _log_int(rng, 5, 2500)
        return {**c, "prompts": rng.randrange(0, 6), "prompt_min": max(1, hi // 6), "prompt_max": hi,
                "decodes": _log_int(rng, 1, 200), "past_max": _log_int(rng, 20, 6000),
                "bias": rng.random() < 0.4}
    if kind == "decode":
        hi = _log_int(rng, 10, 30000)
        return {**c, "decodes": _log_int(rng, 1, max(2, min(64, 250000 // hi))), "past_min": hi // 8,
                "past_max": hi}
    hi = _log_int(rng, 10, 2500)
    return {**c, "prompts": _log_int(rng, 1, max(2, min(30, 6000 // hi))), "prompt_min": max(2, hi // 6),
            "prompt_max": hi, "past_max": _log_int(rng, 10, 3000)}


def _segments(case):
    """[(past, new)] of the step's sequences, from the case alone."""
    rng = np.random.default_rng(case["spread"])
    segs = []
    for _ in range(case.get("prompts", 0)):
        n = int(rng.integers(case["prompt_min"], case["prompt_max"] + 1))
        segs.append((int(rng.integers(0, case["past_max"] + 1)) if rng.random() < 0.6 else 0, n))
    for _ in range(case.get("decodes", 0)):
        segs.append((int(rng.integers(case.get("past_min", 0), case["past_max"] + 1)), 1))
    for _ in range(case.get("ended", 0)):
        segs.append((int(rng.integers(1, case["past_max"] + 1)), -1))
    if case["kind"] != "prefill":
        order = rng.permutation(len(segs))
        segs = [segs[i] for i in order]
    return segs


def work(case):
    segs, bs = _segments(case), case["block"]
    T = sum(max(n, 0) for _, n in segs)
    if case["kind"] == "tables":
        fresh = sum(-(-(p + n) // bs) - -(-p // bs) for p, n in segs if n > 0)
        back = sum(-(-p // bs) for p, n in segs if n < 0)
        # lengths in; starts, lengths, contexts and the prefill list out; per
        # token position, slot and work item; per block ring and table entry
        return {"bytes": 8 * len(segs) + 16 * len(segs) + 16 * T + 8 * (fresh + back) + 32, "flops": 0}
    hq, hkv, D = case["hq"], case["hkv"], case["dim"]
    if case["kind"] == "write":
        old = sum(p % bs for p, _ in segs)
        rope = T * (2 * (hq + 2 * hkv) * D + 2 * hq * D + 2 * hkv * D + 4 * D + 8)
        back = (T + old) * (2 * hkv * D + 4 * hkv * D + 4)
        blocks = sum((p + n - 1) // bs - p // bs + 1 for p, n in segs)
        bias = 2 * (hq + 2 * hkv) * D if case["bias"] else 0
        return {"bytes": rope + back + blocks * hkv * 8 + bias, "flops": T * (hq + hkv) * D * 3}
    keys = sum(p + n for p, n in segs)
    cache = keys * hkv * 2 * D + sum(-(-(p + n) // bs) for p, n in segs) * (hkv * 8 + 4)
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in segs)
    return {"bytes": cache + T * hq * D * 4, "flops": pairs * hq * D * 4}


# ------------------------------------------------------------------ the inputs

def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(_DEV)


def _int32(a):
    return _dev(np.asarray(a, np.int32))


def prepare(case, seed):
    rng = np.random.default_rng([seed, case["spread"]])
    g = torch.Generator(device=_DEV).manual_seed(seed)
    segs, bs = _segments(case), case["block"]
    past, new = np.array([s[0] for s in segs]), np.array([s[1] for s in segs])
    if case["kind"] == "tables":
        return _prepare_tables(past, new, bs, rng)
    ctx = past + new
    S, T, mb = len(segs), int(new.sum()), int(-(-ctx.max() // bs))
    have = -(-ctx // bs)
    nb = int(have.sum()) + 3
    ids = rng.permutation(np.arange(1, nb))
    tables = np.zeros((S, mb), np.int64)
    at = 0
    for s in range(S):
        tables[s, :have[s]] = ids[at:at + have[s]]
        at += have[s]
    q_start = np.cumsum(new) - new
    seq = np.repeat(np.arange(S), new)
    pos = past[seq] + np.arange(T) - q_start[seq]
    slots = tables[seq, pos // bs] * bs + pos % bs
    st = {"case": dict(case), "T": T, "S": S, "max_blocks": mb, "max_new": int(new.max()),
          "max_ctx": int(ctx.max()), "tables": _int32(tables), "q_start": _int32(q_start),
          "q_len": _int32(new), "past": _int32(past), "ctx": _int32(ctx), "positions": _int32(pos),
          "slots": _int32(slots), "token_seq": _int32(seq), "items": _int32(np.arange(T)),
          "seq_ids": _int32(np.arange(S))}
    hq, hkv, D = case["hq"], case["hkv"], case["dim"]
    # Keys with a few strong channels, as trained models have them.
    gain = torch.ones(hkv, 1, D, device=_DEV)
    gain[:, :, torch.from_numpy(rng.permutation(D)[:3]).to(_DEV)] = 6.0
    shape = (nb, hkv, bs, D)
    k = torch.randn(shape, generator=g, device=_DEV) * gain
    v = torch.randn(shape, generator=g, device=_DEV)
    v *= torch.exp2(torch.randint(-3, 2, (nb, hkv, 1, 1), generator=g, device=_DEV).float())
    st["k_scale"], st["v_scale"] = (_block_scale(x.abs().amax((2, 3)), case["fmt"]) for x in (k, v))
    st["k"] = _pack_k(_encode(k, st["k_scale"][:, :, None, None], case["fmt"]))
    st["v"] = _pack_v(_encode(v, st["v_scale"][:, :, None, None], case["fmt"]))
    if case["kind"] == "write":
        cols = (hq + 2 * hkv) * D
        qkv = torch.randn(T, cols, generator=g, device=_DEV)
        qkv[:, hq * D:(hq + hkv) * D] *= gain.expand(hkv, 1, D).reshape(1, -1)
        # rows differ in size, so that later tokens raise the scale of a block
        qkv *= torch.exp2(torch.rand(T, 1, generator=g, device=_DEV) * 3 - 1)
        st["qkv"] = qkv.half()
        st["bias"] = torch.randn(cols, generator=g, device=_DEV).half() if case["bias"] else None
        inv = 1.0 / (5e5 ** (torch.arange(D // 2, device=_DEV, dtype=torch.float64) * 2 / D))
        ang = torch.arange(int(ctx.max()), device=_DEV, dtype=torch.float64)[:, None] * inv
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        # the rows of the touched blocks that hold tokens after the step
        first = past // bs * bs
        rseq = np.repeat(np.arange(S), ctx - first)
        rpos = np.concatenate([np.arange(a, b) for a, b in zip(first, ctx)])
        st["read_slots"] = _int32(tables[rseq, rpos // bs] * bs + rpos % bs)
        n = len(rpos)
        st["k_rows"] = torch.zeros(n, hkv * D, dtype=torch.float16, device=_DEV)
        st["v_rows"] = torch.zeros_like(st["k_rows"])
    else:
        # q as the first heads of a qkv row, as the engine keeps it
        st["q_stride"] = (hq + 2 * hkv) * D
        st["q"] = (torch.randn(T, st["q_stride"], generator=g, device=_DEV) * 1.5).half()
        st["out"] = torch.zeros(T, hq * D, dtype=torch.float16, device=_DEV)
        st["scale"] = D ** -0.5
    return st


def _prepare_tables(past, new, bs, rng):
    S, T = len(past), int(np.maximum(new, 0).sum())
    rows = T + 5  # a step padded to a fixed number of token rows
    have = -(-past // bs)
    mb = int(-(-(past + np.maximum(new, 0)).max() // bs)) + 2
    want = int((-(-(past + np.maximum(new, 0)) // bs) - have).sum())
    total = int(have.sum()) + want + 7
    ids = rng.permutation(np.arange(1, total + 1))
    tables = np.zeros((S, mb), np.int64)
    at = 0
    for s in range(S):
        tables[s, :have[s]] = ids[at:at + have[s]]
        at += have[s]
    ring = np.zeros(total, np.int64)  # the free blocks, from a head somewhere in the ring
    head, free = int(rng.integers(0, total)), ids[at:]
    ring[(head + np.arange(len(free))) % total] = free
    z = lambda n: torch.zeros(n, dtype=torch.int32, device=_DEV)  # noqa: E731
    return {"case": {"kind": "tables", "block": bs}, "S": S, "rows": rows, "max_blocks": mb,
            "past": _int32(past), "new": _int32(new), "tables": _int32(tables), "ring": _int32(ring),
            "pool": _int32([head, len(free), 0]), "pool_out": z(2), "q_start": z(S), "q_len": z(S),
            "ctx": z(S), "positions": z(rows), "slots": z(rows), "decode_token": z(rows),
            "decode_seq": z(rows), "prefill_seq": z(S), "counts": z(4)}


# ------------------------------------------------------------ the plain forms

_QMAX = {"int8": 127.0, "fp8": 448.0}


def _block_scale(amax, fmt):
    """The least power of two s with amax / s <= Qmax, from 2^-24 on; 0 for 0."""
    m, e = torch.frexp(amax.clamp(max=65504.0))
    mq, eq = math.frexp(_QMAX[fmt])
    k = (e - eq + (m > mq).int()).clamp(min=-24)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), k), torch.zeros_like(amax))


def _encode(x, s, fmt):
    """x / s in 8 bits; at the largest scale the codes stay inside fp16's range."""
    y = torch.where(s > 0, x / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(x))
    if fmt == "int8":
        lim = torch.where(s >= 1024.0, 63.0, 127.0)
        return torch.maximum(torch.minimum(torch.round(y), lim), -lim).to(torch.int8)
    lim = torch.where(s >= 256.0, 240.0, 448.0)
    return torch.maximum(torch.minimum(y, lim), -lim).to(torch.float8_e4m3fn).view(torch.uint8)


def _values(codes, fmt):
    return codes.float() if fmt == "int8" else codes.view(torch.float8_e4m3fn).float()


def _k_view(k, D):
    nb, hkv, n = k.shape
    return k.view(nb, hkv, n // (16 * D), D // 16, 16, 2, 8)


def _v_view(v, D):
    nb, hkv, n = v.shape
    return v.view(nb, hkv, n // (16 * D), D // 64, 4, 16, 4, 4)


def _pack_k(x):
    nb, hkv, bs, D = x.shape
    y = x.view(nb, hkv, bs // 16, 16, 2, D // 16, 8).permute(0, 1, 2, 5, 3, 4, 6)
    return y.reshape(nb, hkv, bs * D).contiguous()


def _pack_v(x):
    nb, hkv, bs, D = x.shape
    y = x.view(nb, hkv, bs // 16, 4, 4, 16, D // 64, 4).permute(0, 1, 2, 6, 3, 5, 7, 4)
    return y.reshape(nb, hkv, bs * D).contiguous()


def _unpack_k(k, D):  # [n, hkv, bs * D] -> [n, hkv, bs, D]
    return _k_view(k, D).permute(0, 1, 2, 4, 5, 3, 6).reshape(k.shape[0], k.shape[1], -1, D)


def _unpack_v(v, D):
    return _v_view(v, D).permute(0, 1, 2, 4, 7, 5, 3, 6).reshape(v.shape[0], v.shape[1], -1, D)


def _plain_tables(st):
    bs, S, rows, mb = st["case"]["block"], st["S"], st["rows"], st["max_blocks"]
    past, new, tables, ring = (st[n].long() for n in ("past", "new", "tables", "ring"))
    cap = ring.numel()
    head, count = st["pool"][0].long(), st["pool"][1].long()
    length = new.clamp(min=0)
    start = length.cumsum(0) - length
    have, want = (past + bs - 1) // bs, (past + length + bs - 1) // bs
    fits = (new > 0) & (want <= mb) & (start + length <= rows)
    need = torch.where(fits, want - have, 0)
    upto = need.cumsum(0)
    ok = fits & ((need == 0) | (upto <= count))
    base, taken = upto - need, torch.where(ok, need, 0).sum()
    ended = new < 0
    q_len = torch.where(ok, length, 0)
    ctx = torch.where(ok, past + length, torch.where(ended, 0, past))
    # table entries of the granted blocks
    b = torch.arange(mb, device=_DEV)[None, :]
    fresh = ok[:, None] & (b >= have[:, None]) & (b < want[:, None])
    tables = torch.where(fresh, ring[(head + (base - have)[:, None] + b) % cap], tables)
    # blocks of ended sequences join the ring's tail
    back = torch.where(ended, have, 0)
    at = (back.cumsum(0) - back)[:, None] + b
    gone = ended[:, None] & (b < have[:, None])
    ring = torch.cat([ring, ring[:1]])
    ring[torch.where(gone, (head + count + at) % cap, cap)] = tables
    # token rows
    r = torch.arange(rows, device=_DEV)
    s = torch.searchsorted(start + length, r, right=True).clamp(max=S - 1)
    i = r - start[s]
    valid = ok[s] & (i < length[s]) & (i >= 0)
    pos = torch.where(valid, past[s] + i, 0)
    slots = torch.where(valid, tables[s, pos // bs] * bs + pos % bs, -1)
    # work lists: sequences of one token decode, longer ones prefill
    is_dec, is_pre = q_len == 1, q_len > 1
    tok, seq = torch.full((rows + 1,), -1, device=_DEV), torch.zeros(rows + 1, dtype=torch.long, device=_DEV)
    at = torch.where(is_dec, is_dec.long().cumsum(0) - 1, rows)
    tok[at], seq[at] = start, torch.arange(S, device=_DEV)
    pre = torch.full((S + 1,), -1, device=_DEV)
    pre[torch.where(is_pre, is_pre.long().cumsum(0) - 1, S)] = torch.arange(S, device=_DEV)
    counts = torch.stack([length.sum(), is_dec.sum(), is_pre.sum(), ((new > 0) & ~ok).sum()])
    pool = torch.stack([(head + taken) % cap, count - taken + back.sum()])
    return [x.int() for x in (start, q_len, ctx, pos, slots, tok[:rows], seq[:rows], pre[:S], counts,
                              pool, tables, ring[:cap])]


def _plain_write(st):
    c = st["case"]
    hq, hkv, D, bs, fmt, T = c["hq"], c["hkv"], c["dim"], c["block"], c["fmt"], st["T"]
    x = st["qkv"].float()
    if st["bias"] is not None:
        x = (x + st["bias"].float()).half().float()
    x = x.view(T, hq + 2 * hkv, D)
    pos, slots = st["positions"].long(), st["slots"].long()
    co, si = st["cos"][pos][:, None, :], st["sin"][pos][:, None, :]
    a, b = x[:, :hq + hkv, :D // 2], x[:, :hq + hkv, D // 2:]
    qk = torch.cat([a * co - b * si, b * co + a * si], -1).half()
    st["qkv"].view(T, hq + 2 * hkv, D)[:, :hq] = qk[:, :hq]
    blk, off = slots // bs, slots % bs
    first = st["tables"][st["seq_ids"].long(), (st["past"] // bs).long()].long()  # a sequence's first block
    for rows, pack, name in ((qk[:, hq:].float(), "k", "k_scale"), (x[:, hq + hkv:], "v", "v_scale")):
        scale, codes = st[name], st[pack]
        amax = torch.zeros_like(scale).index_reduce_(0, blk, rows.abs().amax(-1), "amax")
        s0 = scale.clone()
        s0[torch.where(off == 0, blk, 0)] = 0.0  # blocks that start with this step
        s1 = torch.maximum(s0, _block_scale(amax, fmt))
        view = _k_view if pack == "k" else _v_view
        ratio = torch.where(s1[first] > 0, s0[first] / s1[first].clamp(min=2.0 ** -24), 0.0)
        ratio = torch.where((st["past"] % bs == 0)[:, None], 1.0, ratio)
        old = _values(codes[first], fmt) * ratio[:, :, None]
        codes[first] = old.round().to(torch.int8) if fmt == "int8" else old.to(torch.float8_e4m3fn).view(torch.uint8)
        scale[blk] = s1[blk]
        q = _encode(rows, s1[blk][:, :, None], fmt)
        tile, key = off // 16, off % 16
        if pack == "k":
            view(codes, D)[blk, :, tile, :, key] = q.view(T, hkv, 2, D // 16, 8).transpose(2, 3)
        else:
            view(codes, D)[blk, :, tile, :, key // 4, :, :, key % 4] = q.view(T, hkv, 16, D // 64, 4).transpose(2, 3)
    rs = st["read_slots"].long()
    rb, rt, rk = rs // bs, rs % bs // 16, rs % 16
    n = rs.numel()
    k = _k_view(st["k"], D)[rb, :, rt, :, rk].transpose(2, 3).reshape(n, hkv, D)
    v = _v_view(st["v"], D)[rb, :, rt, :, rk // 4, :, :, rk % 4].transpose(2, 3).reshape(n, hkv, D)
    return {"qkv": st["qkv"],
            "k": (_values(k, fmt) * st["k_scale"][rb][:, :, None]).half().view(n, -1),
            "v": (_values(v, fmt) * st["v_scale"][rb][:, :, None]).half().view(n, -1)}


def _rows_of_tables(st):
    """K and V of every sequence's table, [S, hkv, max_blocks * bs, D] in fp32."""
    c, t = st["case"], st["tables"].long()
    S, mb = t.shape
    out = []
    for codes, scale, unpack in ((st["k"], st["k_scale"], _unpack_k), (st["v"], st["v_scale"], _unpack_v)):
        x = unpack(_values(codes[t.view(-1)], c["fmt"]), c["dim"]) * scale[t.view(-1)][:, :, None, None]
        out.append(x.view(S, mb, c["hkv"], c["block"], c["dim"]).transpose(1, 2).reshape(S, c["hkv"], -1, c["dim"]))
    return out


def _plain_attention(st):
    c = st["case"]
    hq, hkv, D, T, S = c["hq"], c["hkv"], c["dim"], st["T"], st["S"]
    G, n = hq // hkv, st["max_new"]
    k, v = _rows_of_tables(st)
    seq, pos = st["token_seq"].long(), st["positions"].long()
    row = torch.arange(T, device=_DEV) - st["q_start"].long()[seq]
    q = torch.zeros(S, n, hkv, G, D, device=_DEV)
    q[seq, row] = st["q"][:, :hq * D].float().view(T, hkv, G, D)
    q = q.permute(0, 2, 3, 1, 4).reshape(S, hkv, G * n, D)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(st["scale"])
    del k
    qpos = st["past"].long()[:, None] + torch.arange(n, device=_DEV)
    hidden = torch.arange(s.shape[-1], device=_DEV)[None, None, :] > qpos[:, :, None]
    s.view(S, hkv, G, n, -1).masked_fill_(hidden[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(s, v) / s.sum(-1, keepdim=True)
    o = o.view(S, hkv, G, n, D).permute(0, 3, 1, 2, 4)[seq, row]
    return o.reshape(T, hq * D).half()


# --------------------------------------------------- the framework's launchers

def _plan(st):
    """The views and work descriptions that an engine builds once and keeps."""
    from redline_amd import kernels as K
    c = st["case"]
    if c["kind"] == "tables":
        pool = K.BlockPool(st["ring"], st["pool"], st["pool_out"])
        return K.batch_tables(pool, st["past"], st["new"], st["S"], st["rows"], c["block"], 1, st["tables"],
                              st["max_blocks"], st["q_start"], st["q_len"], st["ctx"], st["positions"],
                              st["slots"], st["decode_token"], st["decode_seq"], st["prefill_seq"],
                              st["counts"])
    fmt = K.KVBlockFormat.kINT8 if c["fmt"] == "int8" else K.KVBlockFormat.kFP8
    kv = K.kv_block_view(st["k"], st["v"], st["k_scale"], st["v_scale"], c["block"], c["hkv"], c["dim"], fmt)
    if c["kind"] == "write":
        return kv
    p = K.block_attention_params(st["q"], st["q_stride"], st["out"], c["hq"], st["scale"], kv, st["tables"],
                                 st["max_blocks"], st["positions"])
    if c["kind"] == "decode":
        parts = -(-st["max_ctx"] // K.kDecodePartitionSize)
        ws = K.DecodeWorkspace(st["T"], c["hq"], parts, c["dim"])
        return p, K.decode_work(st["items"], st["token_seq"], st["T"], parts, ws), ws
    return p, K.prefill_work(st["seq_ids"], st["q_start"], st["q_len"], st["ctx"], st["S"], -(-st["max_new"] // 32))


def _own(st):
    from redline_amd import kernels as K
    if "plan" not in st:
        st["plan"] = _plan(st)
    plan, c = st["plan"], st["case"]
    if c["kind"] == "tables":
        K.build_batch_tables(plan)
        return [st[n] for n in ("q_start", "q_len", "ctx", "positions", "slots", "decode_token", "decode_seq",
                                "prefill_seq", "counts", "pool_out", "tables", "ring")]
    if c["kind"] == "write":
        K.rope_and_write_kv_blocks(st["qkv"], st["positions"], st["slots"], st["T"], c["hq"], st["cos"],
                                   st["sin"], plan, st["bias"])
        K.read_kv_blocks(plan, st["read_slots"], st["read_slots"].numel(), st["k_rows"], st["v_rows"])
        return {"qkv": st["qkv"], "k": st["k_rows"], "v": st["v_rows"]}
    if c["kind"] == "decode":
        K.paged_attention_decode_blocks(plan[0], plan[1])
    else:
        K.paged_attention_prefill_blocks(plan[0], plan[1])
    return st["out"]


def run(st):
    if own:
        return _own(st)
    kind = st["case"]["kind"]
    if kind == "tables":
        return _plain_tables(st)
    return _plain_write(st) if kind == "write" else _plain_attention(st)


# --------------------------------------------------------- from the definition

def _byte_places(bs, D):
    """For each (token, dim) of a block its byte in the K and in the V layout."""
    tok, d = np.meshgrid(np.arange(bs), np.arange(D), indexing="ij")
    E, t, w = D // 16, tok // 16 * 16 * D, tok % 16
    h, r = d // (D // 2), d % (D // 2)
    k = t + r // 8 * 256 + w * 16 + h * 8 + r % 8
    m, g, j = d // E, d % E // 4, d % 4
    v = t + g * 1024 + w // 4 * 256 + m * 16 + j * 4 + w % 4
    return k, v


def _table64(fmt):
    """The value of each byte."""
    b = np.arange(256)
    if fmt == "int8":
        return torch.from_numpy(b.astype(np.uint8).view(np.int8).astype(np.float64)).to(_DEV)
    sign, e, m = np.where(b >= 128, -1.0, 1.0), (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7.0))
    return torch.from_numpy(sign * np.where((e == 15) & (m == 7), np.nan, v)).to(_DEV)


def _stored64(codes, scale, blocks, place, fmt):
    """[hkv, blocks * bs, D] float64: the values that some blocks hold."""
    raw = codes[blocks].view(torch.uint8).long()  # [n, hkv, bytes]
    x = _table64(fmt)[raw][:, :, torch.from_numpy(place).to(_DEV)] * scale[blocks].double()[:, :, None, None]
    return x.transpose(0, 1).reshape(x.shape[1], -1, place.shape[1])


def _exact_attention(st):
    c = st["case"]
    hq, hkv, D, bs = c["hq"], c["hkv"], c["dim"], c["block"]
    pk, pv = _byte_places(bs, D)
    out = torch.zeros(st["T"], hq * D, dtype=torch.float64, device=_DEV)
    for s, (past, new) in enumerate(_segments(c)):
        n = past + new
        blocks = st["tables"][s, :-(-n // bs)].long()
        k, v = (_stored64(st[a], st[a + "_scale"], blocks, p, c["fmt"])[:, :n] for a, p in (("k", pk), ("v", pv)))
        t0 = int(st["q_start"][s])
        q = st["q"][t0:t0 + new, :hq * D].double().view(new, hq, D).transpose(0, 1)
        late = torch.arange(n, device=_DEV)[None, :] > past + torch.arange(new, device=_DEV)[:, None]
        for h in range(hq):
            z = (q[h] @ k[h * hkv // hq].T) * st["scale"]
            p = torch.softmax(z.masked_fill(late, -math.inf), -1)
            out[t0:t0 + new, h * D:(h + 1) * D] = p @ v[h * hkv // hq]
    return out


def _near64(y, fmt):
    """The 8-bit value nearest to y, ties to the even code."""
    if fmt == "int8":
        return y.round()
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return (y / step).round() * step


def _exact_write(st):
    c = st["case"]
    hq, hkv, D, bs, fmt, T = c["hq"], c["hkv"], c["dim"], c["block"], c["fmt"], st["T"]
    qmax, top = (127, 1024.0) if fmt == "int8" else (448, 256.0)
    x = st["qkv"].double().view(T, hq + 2 * hkv, D)
    if st["bias"] is not None:
        x = (x + st["bias"].double().view(1, -1, D)).half().double()
    pos = st["positions"].long()
    co, si = st["cos"].double()[pos][:, None], st["sin"].double()[pos][:, None]
    h = D // 2
    rot = torch.cat([x[..., :h] * co - x[..., h:] * si, x[..., h:] * co + x[..., :h] * si], -1)
    qkv = st["qkv"].double().view(T, hq + 2 * hkv, D).clone()
    qkv[:, :hq] = rot[:, :hq]
    rows = {"k": rot[:, hq:hq + hkv].half().double(), "v": x[:, hq + hkv:]}
    got = {"k": [], "v": []}
    places = dict(zip("kv", _byte_places(bs, D)))
    for s, (past, new) in enumerate(_segments(c)):
        t0 = int(st["q_start"][s])
        first = past // bs
        nblk = (past + new - 1) // bs - first + 1
        blocks = st["tables"][s, first:first + nblk].long()
        o = past % bs
        for name in "kv":
            r = rows[name][t0:t0 + new].transpose(0, 1)  # [hkv, new, D]
            full = torch.zeros(hkv, nblk * bs, D, dtype=torch.float64, device=_DEV)
            full[:, o:o + new] = r
            amax = full.view(hkv, nblk, bs * D).abs().amax(-1).clamp(max=65504.0)
            want = torch.where(amax > 0, torch.exp2(torch.ceil(torch.log2(amax / qmax)).clamp(min=-24)), 0.0)
            old = st[name + "_scale"].double()[blocks].T.clone()  # [hkv, nblk]
            old[:, 1 if o else 0:] = 0.0
            sc = torch.maximum(old, want)
            each = sc.repeat_interleave(bs, 1)[:, :, None]
            lim = torch.where(each >= top, 63.0 if fmt == "int8" else 240.0, float(qmax))
            y = torch.where(each > 0, full / torch.where(each > 0, each, 1.0), 0.0)
            val = torch.maximum(torch.minimum(_near64(y, fmt), lim), -lim)
            if o:
                had = _stored64(st[name], st[name + "_scale"], blocks[:1], places[name], fmt)[:, :o]
                val[:, :o] = torch.where(each[:, :o] > 0, _near64(had / each[:, :o].clamp(min=2.0 ** -24), fmt), 0.0)
            got[name].append((val * each)[:, :o + new].transpose(0, 1).reshape(-1, hkv * D))
    return {"qkv": qkv.view(T, -1), "k": torch.cat(got["k"]), "v": torch.cat(got["v"])}


def exact(case, seed):
    if case["kind"] == "tables":  # whole numbers only
        return None
    st = prepare(case, seed)
    return _exact_write(st) if case["kind"] == "write" else _exact_attention(st)
