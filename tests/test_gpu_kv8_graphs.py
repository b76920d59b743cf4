"""GPU: steps over the paged 8-bit cache captured in graphs and on other streams: the
same as eager ones, replay after replay, with other work in between."""
import math

import pytest
import torch

from test_gpu_kv8 import _gen, _kv, _pos, _table

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)


def _step(K, s, cache, table, pos):
    """A step of several sequences: norm, rope and write, attention, rows read back, the
    drafts verified and the positions moved by what was accepted."""
    q = torch.empty(s.seqs, s.tokens, s.nh * 128, dtype=torch.bfloat16, device="cuda")
    K.qk_norm_rope_kv8(s.qkv, s.w, s.w, s.cos, s.sin, pos, q, cache, table, s.nh, s.nkv, 1e-6)
    out = K.kv8_decode_attention(q, cache, table, pos, None, SCALE)
    k, v = K.kv8_read(cache, table, pos, s.tokens)
    logits = torch.nn.functional.pad(out, (0, s.vocab - out.shape[2]))
    tokens, accepted = K.verify(logits, s.drafted, s.u, None, temperature=0.5, top_k=20)
    pos += accepted + 1
    return out, k, v, tokens, accepted


class _State:
    def __init__(self, seed, seqs=3, tokens=4, nh=8, nkv=2):
        g = _gen(seed)
        rnd = lambda *n: torch.randn(*n, device="cuda", generator=g).to(torch.bfloat16)
        self.seqs, self.tokens, self.nh, self.nkv, self.vocab = seqs, tokens, nh, nkv, 2000
        self.qkv, self.w = rnd(seqs, tokens, (nh + 2 * nkv) * 128), rnd(128)
        self.cos, self.sin = rnd(400, 128), rnd(400, 128)
        self.drafted = torch.randint(0, 1024, (seqs, tokens - 1), device="cuda", generator=g)
        self.u = torch.rand(seqs, tokens, device="cuda", generator=g)
        _, self.table = _table([6] * seqs, 20, seed)
        self.start = _pos(*[(37 * i + 60) % 200 for i in range(seqs)])
        self.old = _kv(g, seqs, 260, nkv)

    def fresh(self, K):
        cache = K.kv8_cache(self.nkv, 20)
        K.kv8_write(*self.old, cache, self.table, torch.zeros_like(self.start))
        return cache, self.start.clone()


def test_captured_steps_at_once():
    import _dip_hip as K
    states = [_State(1), _State(2, seqs=2, tokens=7, nh=24, nkv=3)]
    graphs = []
    for s in states:
        s.cache, s.pos = s.fresh(K)
        before, first = [t.clone() for t in s.cache], s.pos.clone()
        s.graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # what a first call sets up
            _step(K, s, s.cache, s.table, s.pos)
        torch.cuda.current_stream().wait_stream(side)
        for t, b in zip(s.cache, before):
            t.copy_(b)
        s.pos.copy_(first)
        with torch.cuda.graph(s.graph):
            s.got = _step(K, s, s.cache, s.table, s.pos)
        s.eager = s.fresh(K)
    streams = [torch.cuda.Stream() for _ in states]
    for replay in range(5):
        torch.cuda.synchronize()
        for s, stream in zip(states, streams):
            with torch.cuda.stream(stream):
                s.graph.replay()
        torch.cuda.synchronize()
        for s in states:
            want = _step(K, s, s.eager[0], s.table, s.eager[1])
            assert all(torch.equal(a, b) for a, b in zip(s.got, want)), replay
            assert torch.equal(s.pos, s.eager[1])
            assert all(torch.equal(a, b) for a, b in zip(s.cache, s.eager[0]))


@pytest.mark.parametrize("tokens", [3, 20, 200])
def test_captured_prompts_at_once(tokens):
    """Prompts by each route, two graphs on two streams, and eager calls of both on other
    streams than their tensors'."""
    import _dip_hip as K
    g = _gen(tokens)
    nh, nkv, start = 16, 1, 150
    caches, want, outs, graphs = [], [], [], []
    for i in range(2):
        cache, (_, table) = K.kv8_cache(nkv, 9), _table([6], 9, i)
        K.kv8_write(*_kv(g, 1, start + tokens, nkv), cache, table, _pos(0))
        q = torch.randn(tokens, nh * 128, device="cuda", generator=g).to(torch.bfloat16)
        caches.append((q, cache, table[0], start, None, SCALE))
        want.append(K.kv8_prompt_attention(*caches[i]))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(K.kv8_prompt_attention(*caches[i]))
        graphs.append(graph)
    assert want[0].any()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        eager = []
        for stream, graph, args in zip(streams, graphs, caches):
            with torch.cuda.stream(stream):
                graph.replay()
                eager.append(K.kv8_prompt_attention(*args))
        torch.cuda.synchronize()
        for o, e, w in zip(outs, eager, want):
            assert torch.equal(o, w) and torch.equal(e, w)
