"""GPU: drawing tokens against the definition in 64 bits: every filter alone and
together, ties at each border, masked, infinite and NaN logits, the three types,
odd vocabularies and strides."""
import math

import numpy as np
import pytest
import torch

from kv4_util import drawn

pytestmark = pytest.mark.gpu


def _check(logits, u, **how):
    import _dip_hip as K
    token, prob = K.sample(logits, u, **how)
    token, prob = token.cpu().numpy(), prob.cpu().numpy()
    x, uu = logits.detach().double().cpu().numpy(), u.double().cpu().numpy()
    for r in range(len(x)):
        t, p, w = drawn(x[r], uu[r], **how)
        assert token[r] == t, (r, token[r], t, how)
        # the probability's rounding to fp32 and the weights' own
        assert abs(prob[r] - p) <= 2.0 ** -23 * p, (r, prob[r], p)
    return token


FILTERS = [dict(), dict(temperature=0.6), dict(top_k=1), dict(top_k=20), dict(top_k=700),
           dict(top_p=0.9), dict(top_p=0.01), dict(min_p=0.05), dict(temperature=0.0),
           dict(temperature=0.7, top_k=20, top_p=0.8), dict(top_k=300, top_p=0.97, min_p=0.02),
           dict(temperature=2.5, top_p=0.999)]


@pytest.mark.parametrize("how", FILTERS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(3, 1000), (1, 32003), (5, 1), (4, 2), (6, 65)])
def test_filters(how, dtype, rows, vocab):
    print(f"sample {how} {dtype} {rows}x{vocab}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = 2.5 * torch.randn(rows, vocab, device="cuda", generator=g)
    u = torch.rand(rows, device="cuda", generator=g)
    _check(x.to(dtype), u, **how)


@pytest.mark.parametrize("how", FILTERS)
def test_full_vocabulary(how):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = 2.0 * torch.randn(4, 151936, device="cuda", generator=g)
    x += 9 * torch.rand(4, 151936, device="cuda", generator=g).pow(40)
    u = torch.rand(4, device="cuda", generator=g)
    for dtype in (torch.bfloat16, torch.float32):
        _check(x.to(dtype), u, **how)


@pytest.mark.parametrize("how", [dict(top_k=5), dict(top_k=300), dict(top_p=0.5), dict(top_p=0.13),
                                 dict(min_p=1.0), dict(top_k=100, top_p=0.3), dict(temperature=0)])
@pytest.mark.parametrize("levels", [1, 2, 9])
def test_ties_are_cut_by_index(how, levels):
    """Few distinct logits over many tokens: every border falls among equals."""
    g = torch.Generator(device="cuda").manual_seed(levels)
    x = torch.randint(0, levels, (16, 5003), device="cuda", generator=g).to(torch.bfloat16) - 4
    u = torch.linspace(0, 0.9999, 16, device="cuda")
    _check(x, u, **how)


def test_zero_signs_are_equal():
    x = torch.tensor([[-0.0, 0.0, -0.0, -1.0]], device="cuda")
    assert _check(x, torch.tensor([0.0], device="cuda"), top_k=1)[0] == 0
    assert _check(x, torch.tensor([0.0], device="cuda"), temperature=0)[0] == 0
    assert _check(x, torch.tensor([0.99], device="cuda"), top_k=2)[0] == 1


@pytest.mark.parametrize("how", FILTERS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_infinite_and_nan_logits(how, dtype):
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(9, 3000, device="cuda", generator=g)
    inf = math.inf
    x[0] = -inf                      # nothing to choose from
    x[1] = math.nan
    x[2, ::2] = -inf
    x[3, 1:] = -inf                  # one token
    x[4, :2990] = torch.finfo(dtype).min
    x[5, 7] = inf                    # takes all
    x[5, 70] = inf
    x[6, ::3] = math.nan
    x[7, 100:] = math.nan
    x[8] = torch.finfo(dtype).min
    u = torch.rand(9, device="cuda", generator=g)
    import _dip_hip as K
    xs = x.to(dtype)
    _check(xs, u, **how)
    token, prob = K.sample(xs, u, **how)
    assert token[:2].tolist() == [0, 0] and prob[:2].tolist() == [0.0, 0.0]
    assert token[3] == 0 and token[5] in (7, 70) and not prob.isnan().any()


def test_numbers_at_the_ends():
    import _dip_hip as K
    x = torch.tensor([[1.0, 2.0, 3.0, -math.inf]], device="cuda").expand(6, 4)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 7.0, math.nan, -1.0], device="cuda")
    token, _ = K.sample(x, u)
    assert token.tolist() == [0, 2, 2, 2, 2, 0]


def test_strided_rows_and_given_outputs():
    import _dip_hip as K
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn(7, 2005, device="cuda", generator=g).to(torch.bfloat16)
    u = torch.rand(7, device="cuda", generator=g)
    _check(wide[:, 3:1004], u, top_p=0.9)
    _check(wide.t()[:7], u[:7], top_k=3)     # no dense rows: copied
    out, prob = torch.full((9,), -5, device="cuda"), torch.zeros(7, device="cuda")
    token, _ = K.sample(wide, u, out=out[1:8], prob=prob)
    assert token.data_ptr() == out[1:8].data_ptr()
    assert out[0] == -5 and out[8] == -5 and bool((out[1:8] >= 0).all())


def test_drawn_shares_follow_the_probabilities():
    """Evenly spread numbers draw each token as often as its probability says, to
    within one draw at either end of its interval."""
    import _dip_hip as K
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(1, 50, device="cuda", generator=g)
    n = 2000
    u = ((torch.arange(n, device="cuda") + 0.5) / n).float()
    token, _ = K.sample(x.expand(n, 50), u, top_k=30)
    _, _, w = drawn(x[0].double().cpu().numpy(), 0.5, top_k=30)
    share = np.bincount(token.cpu().numpy(), minlength=50) / n
    assert np.abs(share - w / w.sum()).max() <= 1.01 / n


def test_captured_draw_reads_new_logits():
    import _dip_hip as K
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.empty(2, 20000, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    u = torch.rand(2, device="cuda", generator=g)
    out = torch.zeros(2, dtype=torch.int64, device="cuda")
    prob = torch.zeros(2, device="cuda")
    how = dict(temperature=0.9, top_k=50, top_p=0.9)
    K.sample(x, u, out=out, prob=prob, **how)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.sample(x, u, out=out, prob=prob, **how)
    for _ in range(6):
        x.normal_(generator=g)
        u.uniform_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        token, p = K.sample(x, u, **how)
        assert torch.equal(out, token) and torch.equal(prob, p)


def test_refusals():
    import _dip_hip as K
    x = torch.zeros(2, 8, device="cuda")
    u = torch.zeros(2, device="cuda")
    for f in (lambda: K.sample(x[0], u), lambda: K.sample(x.double(), u),
              lambda: K.sample(x, u[:1]), lambda: K.sample(x, u.double()),
              lambda: K.sample(x, u.cpu()), lambda: K.sample(x[:, :0], u),
              lambda: K.sample(x, u, out=torch.zeros(2, device="cuda")),
              lambda: K.sample(x, u, out=torch.zeros(3, dtype=torch.int64, device="cuda")),
              lambda: K.sample(x, u, top_p=0.0), lambda: K.sample(x, u, temperature=-1.0)):
        with pytest.raises(RuntimeError):
            f()
    token, prob = K.sample(x[:0], u[:0])
    assert token.numel() == prob.numel() == 0


def test_top_k_past_the_vocabulary():
    """Numbers past 64 bits keep all tokens, as any past the vocabulary do."""
    import _dip_hip as K
    g = torch.Generator(device="cuda").manual_seed(7)
    x, u = torch.randn(8, 300, device="cuda", generator=g), torch.rand(8, device="cuda", generator=g)
    want, _ = K.sample(x, u)
    for k in (300, 301, 2 ** 63, 2 ** 64 + 1):
        assert torch.equal(K.sample(x, u, top_k=k)[0], want), k
