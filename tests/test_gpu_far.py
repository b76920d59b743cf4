"""GPU: offsets past 32 bits, in the 4-bit cache (arrays of more than 4 GB, their last
rows written, read and attended) and in rows of logits that lie far apart."""
import math

import pytest
import torch

from kv4_util import attention_bound, drawn, quantised, scale_of

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)
ROWS = 40_000_000  # 5.1 GB of keys and as much of values for two heads


@pytest.fixture(scope="module")
def far():
    """(cache whose last 160 rows are written and all others 0, k, v)."""
    import _dip_hip as K
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(160, 2, 128, device="cuda", generator=g).to(torch.bfloat16)
            for _ in range(2))
    cache = K.kv4_cache(2, ROWS)
    assert cache.k.numel() > 1 << 32 and cache.max_len == ROWS
    K.kv4_write(k, v, cache, start=ROWS - 160)
    yield cache, k, v
    torch.cuda.empty_cache()


def _want(q, k, v, rows):
    """Attention of q float64 [nh, 128] over the first `rows` of the written ones and
    all rows before them, whose scores and values are 0."""
    out, size = [], []
    for h in range(q.shape[0]):
        kv = h // (q.shape[0] // 2)
        s = k[:rows, kv] @ q[h] * SCALE
        top = max(float(s.max()), 0.0)
        w = (s - top).exp()
        w = w / (w.sum() + (ROWS - 160) * math.exp(-top))
        out.append(w @ v[:rows, kv])
        size.append(w @ v[:rows, kv].abs())
    return torch.stack(out), torch.stack(size)


def test_the_last_rows_are_written_and_read(far):
    import _dip_hip as K
    cache, k, v = far
    print("far rows of a 4-bit cache: read", flush=True)
    for got, x in zip(K.kv4_read(cache, ROWS - 200), (k, v)):
        assert not got[:40].any()
        assert torch.equal(got[40:].double().cpu(), quantised(x))
    # nothing else was written, in the first 4 GB either
    assert not cache.k[0, :ROWS - 160].any() and not cache.k[1, :ROWS - 160].any()
    assert not cache.v[:, :(ROWS - 160) // 32].any()
    assert not cache.scales[:, :ROWS - 160].any()


def test_a_token_at_the_end(far):
    import _dip_hip as K
    cache, k, v = far
    g = torch.Generator(device="cuda").manual_seed(4)
    q = (12 * torch.randn(8, 128, device="cuda", generator=g)).to(torch.bfloat16)
    print("far rows of a 4-bit cache: one token", flush=True)
    out = K.kv4_decode_attention(q.view(-1), cache, torch.tensor([ROWS - 1], device="cuda"), None,
                                 SCALE)
    ref, size = _want(q.double().cpu(), quantised(k), quantised(v), 160)
    err = (out.view(8, 128).double().cpu() - ref).abs()
    # (the rows of 0 add ones to the sums, which stay whole numbers below 2^24)
    assert bool((err <= attention_bound(ref, size, scale_of(v).max())).all()), float(err.max())


@pytest.mark.parametrize("tokens", [3, 160])
def test_a_prompt_at_the_end(far, tokens):
    """3 tokens as one token's are, 160 over the expanded cache (41 GB)."""
    import _dip_hip as K
    cache, k, v = far
    start = ROWS - 160
    expanded = K.lib.dip_kv4_prompt_attention_workspace_size(tokens, start, 8, 2, 128) > 512 * ROWS
    assert expanded == (tokens == 160)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    q = (12 * torch.randn(tokens, 8, 128, device="cuda", generator=g)).to(torch.bfloat16)
    print(f"far rows of a 4-bit cache: {tokens} tokens", flush=True)
    out = K.kv4_prompt_attention(q.view(tokens, -1), cache, start, None, SCALE)
    kd, vd, smax = quantised(k), quantised(v), scale_of(v).max()
    for t in {0, 1, tokens // 2, tokens - 1}:
        ref, size = _want(q[t].double().cpu(), kd, vd, t + 1)
        err = (out[t].view(8, 128).double().cpu() - ref).abs()
        assert bool((err <= attention_bound(ref, size, smax)).all()), (t, float(err.max()))


@pytest.mark.parametrize("vocab", [1000, 60013])
@pytest.mark.parametrize("how", [dict(top_k=40, top_p=0.9), dict(min_p=0.1), dict(temperature=0.0)])
def test_rows_of_logits_far_apart(vocab, how):
    import _dip_hip as K
    stride = (1 << 30) + 24
    x = torch.empty(2 * stride + vocab, dtype=torch.bfloat16, device="cuda")
    rows = x.as_strided((3, vocab), (stride, 1))
    g = torch.Generator(device="cuda").manual_seed(vocab)
    rows.copy_(2 * torch.randn(3, vocab, device="cuda", generator=g))
    u = torch.rand(3, device="cuda", generator=g)
    print(f"rows of {vocab} logits far apart, {how}", flush=True)
    token, prob = K.sample(rows, u, **how)
    for r in range(3):
        t, p, _ = drawn(rows[r].double().cpu().numpy(), float(u[r]), **how)
        assert int(token[r]) == t
        assert abs(float(prob[r]) - p) <= 2.0 ** -23 * p
