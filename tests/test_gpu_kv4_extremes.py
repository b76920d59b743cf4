"""GPU: the 4-bit cache and its attention at the ends of the numbers' range, against
the definition in 64 bits."""
import math

import pytest
import torch

from kv4_util import attention, attention_bound, quantised, scale_of
from test_gpu_kv4 import SCALE, _gen, _kv, _rope_reference, _same

pytestmark = pytest.mark.gpu

BIG = torch.finfo(torch.bfloat16).max


def _tables(max_len):
    ang = torch.arange(max_len, device="cuda")[:, None] * 0.37 ** torch.arange(
        64, device="cuda")[None] * 3.0
    return [torch.cat((f(ang), f(ang)), -1).to(torch.bfloat16) for f in (torch.cos, torch.sin)]


def _norm_rope(x, nh, nkv, eps):
    """(q, k, v) of the fused form as tensors, the token's form and the rows' alike."""
    import _dip_hip as K
    tokens = x.shape[0]
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    cos, sin = _tables(64)
    cache, one = K.kv4_cache(nkv, 64), K.kv4_cache(nkv, 64)
    q, q1 = (torch.empty(tokens, nh, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    K.qk_norm_rope_kv4_rows(x.view(tokens, -1), w, w, cos, sin, q.view(tokens, -1), cache, nh, nkv,
                            eps, start=5)
    for t in range(tokens):
        K.qk_norm_rope_kv4(x[t].view(-1), w, w, cos, sin, torch.tensor([5 + t], device="cuda"),
                           q1[t].view(-1), one, nh, nkv, eps)
    k, v = K.kv4_read(cache, 5, tokens)
    k1, v1 = K.kv4_read(one, 5, tokens)
    for a, b in ((q, q1), (k, k1), (v, v1)):
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
    c, s = (t[5:5 + tokens, None].cpu() for t in (cos, sin))
    ref = _rope_reference(x.cpu(), w.cpu(), c, s, eps)
    return q, k, v, ref[:, :nh], ref[:, nh:nh + nkv]


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_norm_of_a_head_with_an_infinity(value):
    """An infinite mean makes the finite dimensions 0 and the infinite ones NaN; a NaN
    makes all of them NaN."""
    nh, nkv = 4, 2
    x = torch.randn(3, nh + 2 * nkv, 128, device="cuda", generator=_gen(0)).to(torch.bfloat16)
    x[0, 1, 70] = x[1, nh, 3] = x[2, nh + 1, 127] = value
    q, k, v, want_q, want_k = _norm_rope(x, nh, nkv, 1e-6)
    for (t, h), got, want in (((0, 1), q, want_q), ((1, 0), k, want_k), ((2, 1), k, want_k)):
        if got is k:
            want = quantised(want.to(torch.bfloat16))
        assert _same(got[t, h], want[t, h])
        assert bool(got[t, h].isnan().all()) == math.isnan(value)


def test_norm_of_tiny_heads_without_eps():
    """Subnormal numbers alone: the root's reciprocal is past fp32's largest."""
    nh, nkv = 4, 2
    n = torch.randint(-7, 8, (9, nh + 2 * nkv, 128), device="cuda", generator=_gen(1))
    n[..., 0] = 3  # (no head of zeros)
    x = (n.double() * 2.0 ** -133).to(torch.bfloat16)
    assert bool((x.double() == n.double() * 2.0 ** -133).all())
    q, k, v, want_q, want_k = _norm_rope(x, nh, nkv, 0.0)
    # q's sums of rounded products are taken in fp32 before they are rounded
    err = (q.double().cpu() - want_q).abs()
    assert bool((err <= 2.0 ** -7 * want_q.abs().max()).all())
    assert (err != 0).double().mean() < 1e-3
    assert _same(k, quantised(want_k.to(torch.bfloat16)))


def _check(out, q, k, v):
    """Of the first and the last head."""
    tokens, nh = q.shape[:2]
    rows, nkv = k.shape[:2]
    limits = [rows - tokens + t + 1 for t in range(tokens)]
    kd, vd = quantised(k), quantised(v)
    for h, kv in ((0, 0), (nh - 1, nkv - 1)):
        ref, size = attention(q[:, h:h + 1], kd[:, kv:kv + 1], vd[:, kv:kv + 1], limits, SCALE)
        err = (out.view(q.shape)[:, h:h + 1].double().cpu() - ref).abs()
        assert bool((err <= attention_bound(ref, size, scale_of(v).max())).all()), float(err.max())


# one token, its rows in one launch and split; a prompt's tokens in 16 columns to a
# tile; in 128 over the expanded cache; the same with the rows split
ROUTES = [("token", 16, 2, 200, 1), ("token", 16, 2, 3000, 1), ("columns", 8, 2, 200, 3),
          ("tiles", 64, 1, 150, 130), ("splits", 64, 1, 630, 130)]


def _route(K, tokens, start, nh, nkv):
    """Which kernels a prompt goes through, from its workspace: none or some sums of 16
    columns, or the expanded rows, alone or followed by sums of 128 columns."""
    nbytes = K.lib.dip_kv4_prompt_attention_workspace_size(tokens, start, nh, nkv, 128)
    blocks = -(-(start + tokens) // 64) * 2 * nkv
    sums = nbytes - blocks * 16384 - -(-blocks * 4 // 16) * 16
    one = -(-tokens * (nh // nkv) // 128) * nkv * 128 * 130 * 4
    return "tiles" if sums == 0 else "splits" if sums > 0 and sums % one == 0 else "columns"


def _attend(route, q, k, v):
    """Attention of the last tokens by one route; the rows behind hold anything."""
    import _dip_hip as K
    rows, nkv = k.shape[:2]
    tokens, nh = q.shape[:2]
    cache = K.kv4_cache(nkv, rows + 70)
    cache.scales[:] = BIG  # finite, times each number (-8) beyond the largest
    cache.k[:], cache.v[:] = -120, -120
    K.kv4_write(k, v, cache)
    if route == "token":
        return K.kv4_decode_attention(q.view(-1), cache, torch.tensor([rows - 1], device="cuda"),
                                      None, SCALE)
    assert _route(K, tokens, rows - tokens, nh, nkv) == route, "these sizes take another route"
    return K.kv4_prompt_attention(q.view(tokens, -1), cache, rows - tokens, None, SCALE)


@pytest.mark.parametrize("size", [2.97e38, 2.99e38, BIG])
@pytest.mark.parametrize("route,nh,nkv,rows,tokens", ROUTES)
def test_a_row_of_the_largest_values(route, nh, nkv, rows, tokens, size):
    """Even weights over one such row and many others: on either side of the group
    scale of 2^125."""
    g = _gen(2)
    k, v = _kv(g, rows, nkv)
    v[7] = size
    q = torch.zeros(tokens, nh, 128, dtype=torch.bfloat16, device="cuda")
    _check(_attend(route, q, k, v), q, k, v)


@pytest.mark.parametrize("size", [2.0 ** 118, 2.99e38, BIG])
@pytest.mark.parametrize("route,nh,nkv,rows,tokens", ROUTES)
def test_values_up_to_the_largest(route, nh, nkv, rows, tokens, size):
    """Group scales up to the largest one that finite values have."""
    g = _gen(rows)
    k, _ = _kv(g, rows, nkv)
    v = (torch.rand(rows, nkv, 128, device="cuda", generator=g) * 2 - 1).mul(size)
    v[:, :, ::32] = size  # every group's largest
    v = v.to(torch.bfloat16)
    q = torch.randn(tokens, nh, 128, device="cuda", generator=g).to(torch.bfloat16)
    _check(_attend(route, q, k, v), q, k, v)


@pytest.mark.parametrize("route,nh,nkv,rows,tokens", ROUTES)
def test_large_values_behind_a_small_maximum(route, nh, nkv, rows, tokens):
    """The first rows' scores are just low enough for the sums not to be taken against
    a new maximum: all later weights are above 1 until the division."""
    g = _gen(3)
    c = torch.full((rows,), 7.5 / (128 * SCALE * math.log2(math.e)), device="cuda")
    c[:32] = 0
    k = c[:, None, None].expand(rows, nkv, 128).to(torch.bfloat16)
    v = torch.full((rows, nkv, 128), 2.0 ** 127, dtype=torch.bfloat16, device="cuda")
    q = torch.ones(tokens, nh, 128, dtype=torch.bfloat16, device="cuda")
    _check(_attend(route, q, k, v), q, k, v)


@pytest.mark.parametrize("route,nh,nkv,rows,tokens", ROUTES)
def test_tiny_values(route, nh, nkv, rows, tokens):
    """2^-70 and the numbers just below it, as accurate as any."""
    g = _gen(4)
    k, v = _kv(g, rows, nkv)
    v = (v.double() * 2.0 ** -70).to(torch.bfloat16)
    q = torch.randn(tokens, nh, 128, device="cuda", generator=g).to(torch.bfloat16)
    _check(_attend(route, q, k, v), q, k, v)


@pytest.mark.parametrize("size", [1e10, 2e37, 3e38])
@pytest.mark.parametrize("route,nh,nkv,rows,tokens", ROUTES)
def test_queries_up_to_the_largest(route, nh, nkv, rows, tokens, size):
    """Scores far apart, and none beyond fp32: the row with the largest takes all."""
    g = _gen(5)
    c = torch.rand(rows, 1, 1, device="cuda", generator=g) * 0.001 - 0.0005
    c[0] = 0.002  # the largest, of any token
    k = c.expand(rows, nkv, 128).to(torch.bfloat16)
    _, v = _kv(g, rows, nkv)
    q = torch.full((tokens, nh, 128), size, device="cuda").to(torch.bfloat16)
    out = _attend(route, q, k, v).view(tokens, nkv, nh // nkv, 128)
    # one weight of 1 and the others 0: the row's values, off by the fp32 sums alone
    want = quantised(v)[0].view(1, nkv, 1, 128)
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -11 * scale_of(v)[0].max()
    assert bool(((out.double().cpu() - want).abs() <= bound).all())


@pytest.mark.parametrize("size", [1e9, 1e13, 3e38])
@pytest.mark.parametrize("route,nh,nkv,rows,tokens", ROUTES)
def test_equal_scores_of_large_queries(route, nh, nkv, rows, tokens, size):
    """Rows with the same key share the weight evenly, however large the score."""
    _, v = _kv(_gen(8), rows, nkv)
    k = torch.full((rows, nkv, 128), 0.0017, device="cuda").to(torch.bfloat16)
    q = torch.full((tokens, nh, 128), size, device="cuda").to(torch.bfloat16)
    _check(_attend(route, q, k, v), q, k, v)


@pytest.mark.parametrize("route,nh,nkv,rows,tokens", ROUTES)
def test_no_score_above_minus_infinity(route, nh, nkv, rows, tokens):
    """An infinity in the query against keys of the other sign: every score is -inf,
    whose softmax is NaN, where a token without rows gives zeros."""
    g = _gen(6)
    k, v = _kv(g, rows, nkv)
    k[:, :, 9] = -3.0
    q = torch.randn(tokens, nh, 128, device="cuda", generator=g).to(torch.bfloat16)
    q[0, 1, 9] = math.inf
    nan = _attend(route, q, k, v).view(tokens, nh, 128).isnan()
    want = torch.zeros_like(nan)
    want[0, 1] = True
    assert torch.equal(nan, want)
