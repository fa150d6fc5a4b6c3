"""A beam search of a small mixture-of-experts model with FP8 weights, as a
server runs it: plan, append, attention, experts, LM head, selection and
reordering, eager and captured.  Every selection is checked against the oracle
on the logits of its step, and the scores of what is found against the same
model in float64 on each found sequence from its start."""
import numpy as np
import pytest

import tinybrain_amd as T
from oracle import experts_ref as E

pytestmark = pytest.mark.gpu

HEADS, KV, HD, LAYERS, EXPERTS, TOP, INNER, VOCAB, BS = 4, 2, 32, 2, 5, 2, 96, 300, 16
HIDDEN = HEADS * HD
EOS, BASE = 7, 10000.0


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


class Model:
    def __init__(self, torch, backend, seed):
        rng = np.random.default_rng(seed)
        self.backend, self.torch = backend, torch

        def fp8(k, n):
            return T.quantize_fp8(rng.normal(size=(k, n)) / np.sqrt(k))

        self.embed = rng.normal(size=(VOCAB, HIDDEN)).astype(np.float32)
        self.layers = [dict(qkv=fp8(HIDDEN, (HEADS + 2 * KV) * HD), out=fp8(HIDDEN, HIDDEN),
                            router=(rng.normal(size=(EXPERTS, HIDDEN)) / 4).astype(np.float32),
                            gate=[fp8(HIDDEN, INNER) for _ in range(EXPERTS)],
                            up=[fp8(HIDDEN, INNER) for _ in range(EXPERTS)],
                            down=[fp8(INNER, HIDDEN) for _ in range(EXPERTS)]) for _ in range(LAYERS)]
        self.head = fp8(HIDDEN, VOCAB)
        self.d_embed, self.one = torch.tensor(self.embed).cuda(), torch.ones(HIDDEN, device="cuda")
        self.d_head = backend.fp8_weight(self.head)
        self.d_layers = []
        for l in self.layers:
            parts = [a for n in ("gate", "up", "down") for a in (np.stack([w.data for w in l[n]]),
                                                                 np.stack([w.scales for w in l[n]]))]
            self.d_layers.append((backend.fp8_weight(l["qkv"]), backend.fp8_weight(l["out"]),
                                  backend.moe_layer(l["router"], *parts)))

    def step(self, cache, plan, tokens):
        """Logits of every row of a step."""
        be = self.backend
        x = self.d_embed[tokens.long()]
        for i, (qkv, out, moe) in enumerate(self.d_layers):
            r = be.fp8_matmul_device(be.rmsnorm_device(x, self.one), qkv)
            q, k, v = r.split((HEADS * HD, KV * HD, KV * HD), 1)
            q = cache.append(i, plan, k, v, q, ropeBase=BASE)
            y = cache.attention(i, plan, q, HEADS)
            x = x + be.fp8_matmul_device(y, out)
            x = x + be.moe_device(be.rmsnorm_device(x, self.one), moe, TOP)[0]
        return be.fp8_matmul_device(be.rmsnorm_device(x, self.one), self.d_head)

    def logits64(self, tokens):
        """The last position's logits of one sequence, in float64."""
        def norm(x):
            return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5)

        n = len(tokens)
        x = self.embed[tokens].astype(np.float64)
        angle = np.arange(n)[:, None] * BASE ** (-np.arange(0, HD, 2) / HD)
        for l in self.layers:
            r = E.fp8_matmul(norm(x), l["qkv"].data, l["qkv"].scales)[0].reshape(n, -1, HD)

            def turn(z):
                a, b = z[..., ::2], z[..., 1::2]
                c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
                return np.stack([a * c - b * s, a * s + b * c], -1).reshape(z.shape)

            q, k, v = turn(r[:, :HEADS]), turn(r[:, HEADS:HEADS + KV]), r[:, HEADS + KV:]
            y = np.zeros((n, HEADS, HD))
            for h in range(HEADS):
                z = q[:, h] @ k[:, h * KV // HEADS].T / np.sqrt(HD)
                z = np.where(np.tri(n) > 0, z, -np.inf)
                p = np.exp(z - z.max(1, keepdims=True))
                y[:, h] = p / p.sum(1, keepdims=True) @ v[:, h * KV // HEADS]
            x = x + E.fp8_matmul(y.reshape(n, -1), l["out"].data, l["out"].scales)[0]
            x = x + E.moe(norm(x), l["router"], *[[(w.data, w.scales) for w in l[m]] for m in ("gate", "up", "down")],
                          TOP, True, 0.0)[0]
        return E.fp8_matmul(norm(x[-1:]), self.head.data, self.head.scales)[0][0]


def _lp(x):
    return x - x.max() - np.log(np.exp(x - x.max()).sum())


@pytest.mark.parametrize("captured", [False, True])
def test_search(torch, captured):
    backend = T.HIPBackend(0)
    model = Model(torch, backend, 1)
    rng = np.random.default_rng(2)
    prompts, beams, steps = [rng.integers(0, VOCAB, n).tolist() for n in (19, 5, 33)], 4, 7
    rows, groups = beams * len(prompts), len(prompts)
    cache = T.PagedKVCache(backend, LAYERS, 64, BS, KV, HD, rows, 8)

    def ints(a):
        return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")

    # every beam holds its request's prompt, the last token of which is the first step's
    new = np.repeat([len(p) - 1 for p in prompts], beams)
    tokens = ints([t for p in prompts for _ in range(beams) for t in p[:-1]])
    model.step(cache, cache.plan(ints(new), int(new.sum())), tokens)
    shared = ints([len(p) - 1 for p in prompts])
    tokens = ints([p[-1] for p in prompts for _ in range(beams)])
    scores = torch.tensor([0.0] + [-np.inf] * (beams - 1), device="cuda").repeat(groups)
    done = torch.zeros(rows, dtype=torch.int32, device="cuda")
    parents, logits = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, VOCAB, device="cuda")
    ones, before = ints([1] * rows), [torch.empty_like(scores), torch.empty_like(done)]

    def one_step():
        logits.copy_(model.step(cache, cache.plan(ones, rows), tokens))
        before[0].copy_(scores), before[1].copy_(done)
        t, p, s, d = backend.beam_select_device(logits, scores, beams, done=done, eos=EOS)
        for to, since in ((tokens, t), (parents, p), (scores, s), (done, d)):
            to.copy_(since.reshape(-1))
        cache.reorder(parents, beams, sharedLens=shared)

    found = [list(p) for p in prompts for _ in range(beams)]
    state = (tokens, scores, done, cache.contextLens, cache.blockTable, cache.freeBlocks, cache.freeCount)
    if captured:
        kept = [t.clone() for t in state]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            one_step()                      # the paged attention's workspace
        torch.cuda.synchronize()
        for t, k in zip(state, kept):
            t.copy_(k)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            one_step()
    ended = 0
    for _ in range(steps):
        if captured:
            graph.replay()
        else:
            one_step()
        torch.cuda.synchronize()
        want = E.beam_select(logits.cpu().numpy(), before[0].cpu().numpy(), beams, beams, before[1].cpu().numpy(), EOS)
        t, p, d = tokens.cpu().numpy(), parents.cpu().numpy(), done.cpu().numpy()
        np.testing.assert_array_equal(t, want[0].reshape(-1))
        np.testing.assert_array_equal(p, want[1].reshape(-1))
        np.testing.assert_array_equal(d, want[3].reshape(-1))
        over = before[1].cpu().numpy()
        found = [found[p[r]] + ([] if over[p[r]] else [int(t[r])]) for r in range(rows)]
        ended = max(ended, int(d.sum()))
    got = scores.cpu().numpy()
    assert np.isfinite(got).all()
    for r, sequence in enumerate(found):
        prompt = prompts[r // beams]
        total = sum(_lp(model.logits64(sequence[:i]))[sequence[i]] for i in range(len(prompt), len(sequence)))
        # fp32 sums may put a row's value on the other side of a rounding to e4m3, which moves one of 128
        # inputs by 2^-4 of itself and a logit by about 2^-4 * 3 / sqrt(128): allowed once a token
        assert abs(total - got[r]) < 0.02 * (len(sequence) - len(prompt)), (r, total, got[r])
    backend.close()
