"""GPU: the verification of drafted tokens against the definition in 64 bits: every
filter, with and without the draft's logits, ragged drafts, masked rows, the three
types, odd vocabularies and strides; and the distribution that comes out."""
import math

import numpy as np
import pytest
import torch

from kv4_util import drawn

pytestmark = pytest.mark.gpu

FILTERS = [dict(), dict(temperature=0.6), dict(top_k=1), dict(top_k=20), dict(top_p=0.9),
           dict(min_p=0.05), dict(temperature=0.0), dict(temperature=0.7, top_k=20, top_p=0.8),
           dict(top_k=300, top_p=0.97, min_p=0.02), dict(temperature=2.5, top_p=0.999)]


def _shares(x, how):
    """A row's probabilities after the filters, float64; zeros if there is nothing."""
    w = drawn(x, 0.0, **how)[2]
    return w / w.sum() if w.sum() > 0 else w


def _verified(x, y, drafted, u, how):
    """(tokens, accepted) of one sequence: x [n + 1, vocab], y [n, vocab] or None."""
    n, vocab = len(drafted), x.shape[-1]
    greedy = how.get("temperature", 1.0) == 0 or how.get("top_k", 0) == 1
    tokens = [-1] * (n + 1)
    for t in range(n + 1):
        p = _shares(x[t], how)
        d = int(drafted[t]) if t < n else -1
        if 0 <= d < vocab and p.sum() > 0:
            q = np.zeros(vocab)
            if y is None or greedy:
                q[d] = 1
            else:
                q = _shares(y[t], how)
            if (p[d] > 0) if greedy else u[t] * q[d] < p[d]:
                tokens[t] = d
                continue
            rest = np.maximum(p - q, 0)
            p = rest if rest.sum() > 0 else p
        run = np.cumsum(p)
        above = np.nonzero((run > (0.5 if greedy else u[n]) * run[-1]) & (p > 0))[0]
        tokens[t] = int(above[0]) if len(above) else int(np.nonzero(p)[0][-1]) if p.any() else 0
        return tokens, t


def _check(logits, drafted, u, draft_logits=None, **how):
    import _dip_hip as K
    tokens, accepted = K.verify(logits, drafted, u, draft_logits, **how)
    x, d, uu = (t.double().cpu().numpy() for t in (logits, drafted, u))
    y = None if draft_logits is None else draft_logits.double().cpu().numpy()
    for s in range(len(x)):
        want, n = _verified(x[s], None if y is None else y[s], d[s], uu[s], how)
        assert tokens[s].tolist() == want and int(accepted[s]) == n, (s, how, accepted[s], n)
    return tokens, accepted


def _inputs(seqs, n, vocab, dtype, seed, noise=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = 2.5 * torch.randn(seqs, n + 1, vocab, device="cuda", generator=g)
    y = x[:, :n] + noise * torch.randn(seqs, n, vocab, device="cuda", generator=g)
    # drafts among the likely ones, so that some are accepted
    drafted = (y + torch.randn(y.shape, device="cuda", generator=g)).argmax(-1) if n else \
        torch.zeros(seqs, 0, dtype=torch.int64, device="cuda")
    u = torch.rand(seqs, n + 1, device="cuda", generator=g)
    return x.to(dtype), drafted, u, y.to(dtype)


@pytest.mark.parametrize("how", FILTERS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("seqs,n,vocab", [(3, 4, 1000), (2, 1, 32003), (5, 3, 1), (4, 2, 2),
                                          (6, 7, 65), (1, 0, 500), (70, 2, 9001)])
def test_filters(how, dtype, seqs, n, vocab):
    print(f"verify {how} {dtype} {seqs}x{n} of {vocab}", flush=True)
    x, d, u, y = _inputs(seqs, n, vocab, dtype, vocab + n)
    _check(x, d, u, **how)
    _check(x, d, u, y, **how)


@pytest.mark.parametrize("how", FILTERS)
def test_full_vocabulary(how):
    for dtype in (torch.bfloat16, torch.float32):
        x, d, u, y = _inputs(3, 4, 151936, dtype, 1)
        d[1, 2] = -1
        _, a = _check(x, d, u, **how)
        _, b = _check(x, d, u, y, **how)
        assert int(a[1]) <= 2 and int(b[1]) <= 2


def test_some_are_accepted_and_some_refused():
    """The inputs of these tests accept none, and some."""
    x, d, u, y = _inputs(64, 3, 1000, torch.float32, 7)
    for draft in (None, y):
        _, accepted = _check(x, d, u, draft, temperature=0.8)
        assert {0, 1} <= set(accepted.tolist())


def test_drafts_that_are_none():
    """Short drafts, and numbers outside the vocabulary: nothing is read there and the
    next token is the target's own."""
    import _dip_hip as K
    x, d, u, y = _inputs(5, 3, 700, torch.bfloat16, 3)
    d[0, 0], d[1, 1], d[2, 2] = -1, 700, -(1 << 62)
    d[3, 0], d[3, 1:] = (1 << 62), -1
    u[:, :3] = 0  # what may be accepted, is
    for draft in (None, y):
        for how in FILTERS:
            _check(x, d, u, draft, **how)
        tokens, accepted = K.verify(x, d, u, draft)
        assert accepted.tolist() == [0, 1, 2, 0, 3]
        for s in range(5):
            n = int(accepted[s])
            assert int(tokens[s, n]) == int(K.sample(x[s, n:n + 1], u[s, 3:])[0])


@pytest.mark.parametrize("how", FILTERS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_infinite_and_nan_logits(how, dtype):
    x, d, u, y = _inputs(11, 2, 3000, dtype, 9)
    inf = math.inf
    x[0] = -inf                      # nothing to choose from
    x[1, 1] = math.nan
    u[1, 0] = 0
    x[2, :, ::2] = -inf
    x[3, 0, 1:] = -inf               # one token, drafted
    d[3, 0] = 0
    x[4, 0, 1:] = -inf               # one token, not drafted
    d[4, 0] = 5
    x[5, 0, 7] = inf                 # takes all
    x[5, 0, 70] = inf
    d[5, 0] = 70
    y[6] = -inf                      # a draft that its logits did not draw
    y[7, 0] = x[7, 0]                # p and q the same
    u[7, 0] = 0.999
    y[8, 0, 7] = inf
    x[9] = torch.finfo(dtype).min
    y[10, :, ::3] = math.nan
    for draft in (None, y):
        tokens, accepted = _check(x, d, u, draft, **how)
        assert tokens[0].tolist() == [0, -1, -1] and int(accepted[0]) == 0
        assert int(accepted[3]) >= 1 and tokens[4, 0] == 0


def test_numbers_at_the_ends():
    """u of 0 accepts whatever has a share, u just below 1 only what p has more of."""
    import _dip_hip as K
    x, d, u, y = _inputs(40, 2, 100, torch.float32, 5)
    top = 1 - 2.0 ** -24
    for first in (0.0, top):
        for last in (0.0, top):
            u[:, :2], u[:, 2] = first, last
            _check(x, d, u)
            _check(x, d, u, y)
    u[:, :2], u[:, 2] = math.nan, math.nan
    tokens, accepted = K.verify(x, d, u, y)
    assert not accepted.any() and bool((tokens[:, 0] >= 0).all())
    # everything refused by a number of 1 where p and q are the same: drawn from p
    u[:, :2], u[:, 2] = 1.0, 0.3
    tokens, accepted = K.verify(x, d, u, x[:, :2].contiguous())
    want, _ = K.sample(x[:, 0].contiguous(), u[:, 2].contiguous())
    assert not accepted.any() and torch.equal(tokens[:, 0], want)


def test_views_outputs_and_workspaces():
    import _dip_hip as K
    x, d, u, y = _inputs(4, 3, 5003, torch.bfloat16, 2)
    wide = torch.zeros(4, 4, 5011, dtype=torch.bfloat16, device="cuda")
    wide[..., 3:5006] = x
    want = _check(x, d, u, y, top_p=0.9)
    for rows in (wide[..., 3:5006], x.permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        got = K.verify(rows, d.t().contiguous().t(), u.t().contiguous().t(), y, top_p=0.9)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    out, acc = torch.full((6, 4), -5, device="cuda"), torch.full((4,), -5, device="cuda")
    n = K.lib.dip_verify_workspace_size(4, 3, 5003, 1)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    got = K.verify(x, d, u, y, top_p=0.9, out=out[1:5], accepted=acc, ws=ws)
    assert got[0].data_ptr() == out[1:5].data_ptr() and got[1] is acc
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert bool((out[0] == -5).all()) and bool((out[5] == -5).all())
    with pytest.raises(RuntimeError):
        K.verify(x, d, u, y, ws=ws[:n - 1])


@pytest.mark.parametrize("vocab", [3000, 151936])
def test_captured_and_on_two_streams(vocab):
    import _dip_hip as K
    sets = [_inputs(3, 4, vocab, torch.bfloat16, s) for s in (1, 2)]
    how = dict(top_k=50, top_p=0.9)
    want = [K.verify(*s, **how) for s in sets]
    graphs, outs = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(K.verify(*s, **how))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for o in outs:
            o[0].zero_()
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, w))
        assert torch.equal(K.verify(*sets[0], **how)[0], want[0][0])


@pytest.mark.parametrize("with_draft", [False, True])
def test_tokens_are_distributed_as_the_target(with_draft):
    """Drafts drawn from q with evenly spread numbers and verified: the first token of a
    sequence is each as often as p says.  20000 sequences: a share's standard deviation is
    below 0.0036, six of them 0.022."""
    import _dip_hip as K
    g = torch.Generator(device="cuda").manual_seed(4)
    vocab, seqs = 12, 20000
    p = torch.randn(1, 1, vocab, device="cuda", generator=g)
    q = torch.randn(1, 1, vocab, device="cuda", generator=g)
    rows = q.expand(seqs, 1, vocab).contiguous()
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)
    how = dict(temperature=0.9, top_p=0.95)
    if with_draft:
        drafted, draft = K.sample(rows[:, 0], rand(seqs), **how)[0][:, None], rows
    else:
        drafted, draft = rows.argmax(-1), None
    tokens, accepted = K.verify(p.expand(seqs, 2, vocab).contiguous(), drafted, rand(seqs, 2),
                                draft, **how)
    share = torch.bincount(tokens[:, 0], minlength=vocab).cpu().numpy() / seqs
    want = _shares(p.view(-1).double().cpu().numpy(), how)
    assert np.abs(share - want).max() < 0.022
    assert bool((accepted > 0).any()) and bool((accepted == 0).any())


def test_refusals():
    import _dip_hip as K
    x, d, u, y = _inputs(2, 3, 50, torch.float32, 1)
    for args in ((x[0], d, u), (x.double(), d, u), (x, d[:1], u), (x, d.int(), u), (x, d, u[:, :3]),
                 (x, d, u.double()), (x, d, u, y[:, :2]), (x, d, u, y.half()), (x, d, u, y.cpu()),
                 (x, d.cpu(), u)):
        with pytest.raises(RuntimeError):
            K.verify(*args)
    for how in (dict(top_p=0.0), dict(temperature=-1.0), dict(top_k=-2), dict(min_p=2.0)):
        with pytest.raises(RuntimeError):
            K.verify(x, d, u, **how)
    assert K.verify(x[:0], d[:0], u[:0])[0].shape == (0, 4)
