"""GPU: drawing from rows too long for one launch (slices, a histogram, a list of the
tokens at the border), and the longest that one launch takes."""
import math

import pytest
import torch

from kv4_util import drawn

pytestmark = pytest.mark.gpu


def _check(logits, u, **how):
    import _dip_hip as K
    token, prob = K.sample(logits, u, **how)
    again, _ = K.sample(logits, u, **how)
    assert torch.equal(token, again)
    token, prob = token.cpu().numpy(), prob.cpu().numpy()
    x, uu = logits.detach().double().cpu().numpy(), u.double().cpu().numpy()
    for r in range(len(x)):
        t, p, _ = drawn(x[r], uu[r], **how)
        assert token[r] == t, (r, token[r], t, how)
        assert abs(prob[r] - p) <= 2.0 ** -23 * p, (r, prob[r], p)


FILTERS = [dict(), dict(min_p=0.1), dict(top_k=1), dict(top_k=50, top_p=0.9), dict(top_k=30000),
           dict(top_p=0.7), dict(top_p=0.9999), dict(top_p=0.98, min_p=0.3),
           dict(temperature=0.0), dict(temperature=5.0, top_k=4000, top_p=0.9, min_p=0.001),
           dict(temperature=0.05, top_p=0.9), dict(temperature=1e-6), dict(temperature=1e6, top_p=0.5)]


@pytest.mark.parametrize("how", FILTERS)
@pytest.mark.parametrize("rows,vocab,dtype", [(2, 70001, torch.float32), (3, 131072, torch.bfloat16),
                                              (2, 40009, torch.float16), (70, 32745, torch.bfloat16),
                                              (70, 16371, torch.float32)])
def test_filters(how, rows, vocab, dtype):
    print(f"sample {how} {rows}x{vocab} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    # rows that begin at every place of a 16-byte piece
    x = 2.5 * torch.randn(rows, vocab + 3, device="cuda", generator=g)
    u = torch.rand(rows, device="cuda", generator=g)
    _check(x.to(dtype)[:, 1:vocab + 1], u, **how)


@pytest.mark.parametrize("how", [dict(top_k=5), dict(top_k=6000), dict(top_p=0.5), dict(top_p=0.13),
                                 dict(min_p=1.0), dict(top_k=20000, top_p=0.3), dict(temperature=0),
                                 dict(top_p=0.4, min_p=0.9), dict()])
@pytest.mark.parametrize("levels", [1, 3])
@pytest.mark.parametrize("vocab", [50021, 30011])
def test_thousands_of_equal_logits(how, levels, vocab):
    """The tokens at the border overflow the list: the row is searched by its bits."""
    g = torch.Generator(device="cuda").manual_seed(levels)
    x = torch.randint(0, levels, (4, vocab), device="cuda", generator=g).to(torch.bfloat16) - 4
    _check(x, torch.tensor([0.0, 0.3, 0.77, 0.9999], device="cuda"), **how)


@pytest.mark.parametrize("how", [dict(), dict(top_k=40), dict(top_p=0.9), dict(top_k=3, min_p=0.2),
                                 dict(temperature=0.0)])
def test_masked_infinite_and_nan_logits(how):
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(7, 60000, device="cuda", generator=g)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, ::2] = -math.inf
    x[3, :59999] = -math.inf
    x[4, 100::1000] = math.inf
    x[5, ::3] = math.nan
    x[6, :59000] = torch.finfo(torch.float32).min
    u = torch.rand(7, device="cuda", generator=g)
    _check(x, u, **how)
    _check(x.to(torch.bfloat16), u, **how)


def test_two_streams_share_nothing():
    import _dip_hip as K
    g = torch.Generator(device="cuda").manual_seed(2)
    xs = [torch.randn(3, 100000, device="cuda", generator=g) for _ in range(2)]
    us = [torch.rand(3, device="cuda", generator=g) for _ in range(2)]
    how = dict(top_k=200, top_p=0.95)
    want = [K.sample(x, u, **how)[0] for x, u in zip(xs, us)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(K.sample(xs[i], us[i], **how)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[i]) for i in range(2) for t in got[i])


def test_captured_draw_of_a_long_row():
    import _dip_hip as K
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.empty(1, 151936, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    u = torch.rand(1, device="cuda", generator=g)
    out, prob = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, device="cuda")
    how = dict(temperature=0.7, top_k=20, top_p=0.8)
    K.sample(x, u, out=out, prob=prob, **how)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.sample(x, u, out=out, prob=prob, **how)
    for _ in range(5):
        x.normal_(generator=g)
        u.uniform_(generator=g)
        token, p = K.sample(x, u, **how)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, token) and torch.equal(prob, p)
