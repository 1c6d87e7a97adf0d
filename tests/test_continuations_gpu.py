"""A decode loop that draws several continuations of each prompt: normed cache write, attention
over the shared prompts, sampling, and the drawn tokens as the next step's input; eager and
captured."""
import numpy as np
import pytest

import redline_amd as ra
from tests._util import say
from tests.test_norm_rope_gpu import U16, U32
from tests.test_sampling_gpu import candidates

pytestmark = pytest.mark.gpu
H, V, HQ, HKV, D, BS, STEPS = 128, 700, 4, 2, 64, 16, 9
EPS = 1e-6


class Model:
    """One layer without residuals, fp16."""

    def __init__(self, torch, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.table = rand(V, H).half()
        self.w_qkv = (rand(H, (HQ + 2 * HKV) * D) / H ** 0.5).half()
        self.w_out = (rand(HQ * D, V) * 3 / (HQ * D) ** 0.5).half()
        self.q_norm, self.k_norm = ((1 + 0.2 * rand(D)).half() for _ in "qk")
        cos, sin = ra.rope_cos_sin_tables(1e4, D, 256)
        self.cos, self.sin = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()

    def kv_rows(self, torch, ids, pos):
        """(k, v, bound of k) [n, HKV, D] of tokens at positions, in 64 bits from the fp16 qkv."""
        x = self.table[ids] @ self.w_qkv
        x = x.double().view(len(ids), -1, D)[:, HQ:]
        n = x[:, :HKV]
        n = n / torch.sqrt(n.square().mean(-1, keepdim=True) + EPS) * self.k_norm.double()
        co, si = self.cos[pos].double()[:, None], self.sin[pos].double()[:, None]
        a, b = n[..., :D // 2], n[..., D // 2:]
        size = torch.cat([(a * co).abs() + (b * si).abs(), (b * co).abs() + (a * si).abs()], -1)
        return torch.cat([a * co - b * si, b * co + a * si], -1), x[:, HKV:], size


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("cache", ["fp16", "int8"])
def test_loop(cache, captured):
    import torch
    from redline_amd import kernels as K
    say("continuations", cache, captured)
    m, rng = Model(torch, 1), np.random.default_rng(2)
    groups = [(37, 5), (1, 1), (64, 3), (100, 6)]
    N, mb = sum(n for _, n in groups), -(-(100 + STEPS) // BS)
    blocks = rng.permutation(np.arange(1, N * mb + 1)).reshape(N, mb)
    table, firsts, prompt, starts = blocks.copy(), [], [], [0]
    for p, n in groups:
        ids = rng.integers(0, V, p)
        for j in range(n):
            table[len(firsts), :p // BS] = blocks[starts[-1], :p // BS]  # whole blocks of the prompt are shared
            firsts.append(starts[-1])
            prompt.append(ids)
        starts.append(len(firsts))
    c = K.KVCache(1, N * mb + 1, HKV, D, BS, K.KVDType.kFP16 if cache == "fp16" else K.KVDType.kINT8)
    kv, cols = c.layer(0), (HQ + 2 * HKV) * D
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()  # noqa: E731
    slot = lambda i, n: int(table[i, n // BS] * BS + n % BS)  # noqa: E731

    # the prompts, once each (their last tokens make the first step)
    for g, (p, _) in enumerate(groups):
        ids = i32(prompt[starts[g]])
        qkv = m.table[ids.long()] @ m.w_qkv
        K.rope_and_write_kv_norm(qkv, i32(np.arange(p)), i32([slot(starts[g], t) for t in range(p)]), p, HQ, m.cos, m.sin,
                                 kv, q_norm=m.q_norm, k_norm=m.k_norm, eps=EPS)

    fp16 = dict(dtype=torch.float16, device="cuda")
    x, qkv = torch.zeros(N, H, **fp16), torch.zeros(N, cols, **fp16)
    attn, logits = torch.zeros(N, HQ * D, **fp16), torch.zeros(N, V, **fp16)
    tokens, ids, src = i32([p[-1] for p in prompt]), i32(np.zeros(N)), i32(np.arange(N))
    pos, slots = i32(np.zeros(N)), i32(np.zeros(N))
    u, lp = torch.zeros(N, device="cuda"), torch.zeros(N, device="cuda")
    T = np.where(np.arange(N) % 4 == 0, 0.0, rng.uniform(0.5, 1.5, N)).astype(np.float32)
    k, top_p = rng.integers(0, 60, N), rng.uniform(0.7, 1.1, N).astype(np.float32)
    # keys up to the step's own token: a group's prompt is shared, the rest is the item's own
    params = K.attention_params(qkv, cols, attn, HQ, D ** -0.5, kv, i32(table), mb, pos)
    work = K.shared_prefix_work(src, src, N, i32(starts), i32([p for p, _ in groups]), len(groups), 6, 1, 1,
                                K.DecodeWorkspace(N, HQ, 2, D))
    draws = K.sampling_work(logits, N, V, torch.from_numpy(T).cuda(), i32(k), torch.from_numpy(top_p).cuda(), u, tokens,
                            K.SamplingWorkspace(N, V), logprobs=lp)

    def step():
        K.resolve_input_ids(ids, src, tokens, N)
        K.embedding_lookup(ids, m.table, N, H, x)
        torch.mm(x, m.w_qkv, out=qkv)
        K.rope_and_write_kv_norm(qkv, pos, slots, N, HQ, m.cos, m.sin, kv, q_norm=m.q_norm, k_norm=m.k_norm, eps=EPS)
        K.paged_attention_decode_shared(params, work)
        torch.mm(attn, m.w_out, out=logits)
        K.sample_tokens(draws)

    graph = None
    if captured:
        slots.fill_(-1)
        kept = tokens.clone()
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        tokens.copy_(kept)
    said = [[int(t) for t in p] for p in prompt]
    for s in range(STEPS):
        here = [len(t) - 1 for t in said]  # of the token that this step takes in
        pos.copy_(i32(here))
        # the first step's token is the prompt's last: its key is there already
        slots.copy_(i32([-1 if s == 0 else slot(i, n) for i, n in enumerate(here)]))
        u.copy_(torch.from_numpy(rng.random(N).astype(np.float32)))
        graph.replay() if graph else step()
        torch.cuda.synchronize()
        drawn, rows = tokens.cpu().numpy(), logits.float().cpu().numpy()
        for i in range(N):
            n, p = here[i] + 1, len(prompt[i])
            where = [slot(firsts[i] if t < p else i, t) for t in range(n)]
            kr, vr = (torch.zeros(n, HKV * D, **fp16) for _ in "kv")
            K.read_kv(kv, i32(where), n, kr, vr)
            kr, vr = kr.view(n, HKV, D).double(), vr.view(n, HKV, D).double()
            want_k, want_v, size = m.kv_rows(torch, torch.tensor(said[i][:n], device="cuda"),
                                             torch.arange(n, device="cuda"))
            # the rows of one batch's product may differ from another's by a step of fp16 each, which the
            # norm passes on to all of a head (2^-10 of the head's largest at most, in k twice); an INT8
            # cell adds half a step of its scale
            for got, want, times in ((kr, want_k, 3), (vr, want_v, 1)):
                top = want.abs().amax(-1, keepdim=True)
                tol = times * 2 * U16 * top + U16 * top + (top / 254 * 1.01 if cache == "int8" else 0)
                assert ((got - want).abs() <= tol + 24 * U32 * size.amax()).all(), (s, i)
            # the attention from the rows that the cache holds
            q = qkv[i, :HQ * D].double().view(HKV, -1, D)
            sc = q @ kr.permute(1, 2, 0).contiguous() * D ** -0.5
            w = torch.softmax(sc, -1)
            vt = vr.transpose(0, 1).contiguous()
            o, a = (w @ vt).view(-1), (w @ vt.abs()).view(-1)
            big = float((q.abs() @ kr.abs().permute(1, 2, 0).contiguous()).max()) * D ** -0.5
            # as in the tests of the attention; an INT8 key's fp16 form rounds each product of a score
            rel = 2 * U16 + 2 * big * (1.5 * (D + 4) * U32 + (U16 if cache == "int8" else 0)) + 2 * n * U32
            tol = rel * a + n * 2.0 ** -25 * float(vt.abs().max())
            assert ((attn[i].double() - o).abs() <= tol + U16 * (o.abs() + tol) + 2.0 ** -25).all(), (s, i)
            near = candidates(rows[i], T[i], k[i], top_p[i], 0.0, float(u[i]))
            assert int(drawn[i]) in near, (s, i)
            said[i].append(int(drawn[i]))
    assert len({tuple(t[len(p):]) for t, p in zip(said, prompt)}) > len(groups)  # the continuations differ
