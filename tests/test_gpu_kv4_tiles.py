"""GPU: prompts long enough for the attention in tiles of 128 columns over the
expanded 4-bit cache, against fp64 softmax: one and several splits of the rows,
groups of 1 to 8 heads, odd lengths and starts, rows with NaN, rows behind the
prompt that hold anything."""
import math

import pytest
import torch

from kv4_util import quantised

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)


def _case(tokens, start, nh, nkv, seed=0):
    import _dip_hip as K
    g = torch.Generator(device="cuda").manual_seed(seed + tokens + start)
    rows = start + tokens
    # the tiles' workspace holds the expanded rows: 512 bytes each per kv head
    nbytes = K.lib.dip_kv4_prompt_attention_workspace_size(tokens, start, nh, nkv, 128)
    assert nbytes >= rows * nkv * 512, "these sizes no longer go over the expanded cache"
    q = (torch.randn(tokens, nh, 128, device="cuda", generator=g) * 2).to(torch.bfloat16)
    k = torch.randn(rows, nkv, 128, device="cuda", generator=g)
    k = (k * torch.exp(0.5 * torch.randn(nkv, 128, device="cuda", generator=g))).to(torch.bfloat16)
    v = (torch.randn(rows, nkv, 128, device="cuda", generator=g) * 0.3).to(torch.bfloat16)
    return K, q, k, v


def _cache(K, k, v, extra=40):
    rows, nkv = k.shape[:2]
    cache = K.kv4_cache(nkv, rows + extra)
    cache.scales[:] = math.nan  # rows that nobody writes hold anything
    cache.k[:], cache.v[:] = -1, -1
    K.kv4_write(k, v, cache)
    return cache


def _reference(q, k, v, start, heads):
    """(out, sum of weight * |v|) of some heads, float64 on the device."""
    tokens, nh = q.shape[:2]
    kd, vd = quantised(k).cuda(), quantised(v).cuda()
    later = torch.arange(kd.shape[0], device="cuda") > start + torch.arange(
        tokens, device="cuda")[:, None]
    for h in heads:
        kv = h // (nh // k.shape[1])
        w = (q[:, h].double() @ kd[:, kv].T.contiguous() * SCALE).masked_fill(later, -math.inf)
        w = w.softmax(-1)
        yield h, w @ vd[:, kv], w @ vd[:, kv].abs()


@pytest.mark.parametrize("tokens,start,nh,nkv", [
    (512, 0, 64, 8), (509, 333, 40, 8), (1000, 7, 24, 8), (1030, 0, 8, 8), (130, 3001, 64, 8),
    (70, 9003, 64, 8), (300, 5000, 16, 1), (64, 20011, 32, 8), (2500, 0, 3, 3)])
def test_against_softmax(tokens, start, nh, nkv):
    print(f"kv4 tiles tokens={tokens} start={start} {nh}/{nkv}", flush=True)
    K, q, k, v = _case(tokens, start, nh, nkv)
    cache = _cache(K, k, v)
    out = K.kv4_prompt_attention(q.view(tokens, -1), cache, start, None, SCALE)
    again = K.kv4_prompt_attention(q.view(tokens, -1), cache, start, None, SCALE)
    assert torch.equal(out, again)
    smax = v.float().abs().max().double() / 7
    for h, ref, size in _reference(q, k, v, start, {0, nh // 2, nh - 1}):
        err = (out.view(tokens, nh, 128)[:, h].double() - ref).abs()
        # the roundings of the result and of the weights to bf16, and fp32 sums over
        # at most 400 steps (2^-24 of the weights' sum each: below 2^-10 of them)
        bound = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -10) * size + 2.0 ** -11 * smax
        assert bool((err <= bound).all()), (h, float((err / bound).max()))


@pytest.mark.parametrize("tokens,start,nh,nkv", [(512, 0, 64, 8), (70, 9003, 64, 8)])
def test_nan_rows_reach_only_who_attends_them(tokens, start, nh, nkv):
    K, q, k, v = _case(tokens, start, nh, nkv, seed=1)
    rows = start + tokens
    for which in ("v", "k"):
        for at in (0, rows - tokens // 2, rows - 1):
            kk, vv = k.clone(), v.clone()
            (vv if which == "v" else kk)[at, 2, 40] = math.inf
            out = K.kv4_prompt_attention(q.view(tokens, -1), _cache(K, kk, vv), start, None, SCALE)
            nan = out.view(tokens, nh, 128).isnan()
            want = torch.zeros_like(nan)
            later = torch.arange(tokens, device="cuda") + start >= at
            dims = slice(32, 64) if which == "v" else slice(0, 128)
            group = nh // nkv
            want[later, 2 * group:3 * group, dims] = True
            assert torch.equal(nan, want), (which, at)


def test_scores_that_keep_growing():
    """Rows whose scores grow along the cache: the sums are taken against a new
    maximum again and again."""
    tokens, start, nh, nkv = 512, 0, 64, 8
    K, q, k, v = _case(tokens, start, nh, nkv, seed=2)
    k = (torch.linspace(0.05, 6, tokens, device="cuda")[:, None, None]
         * torch.ones(nkv, 128, device="cuda")).to(torch.bfloat16)
    q = torch.ones_like(q)
    out = K.kv4_prompt_attention(q.view(tokens, -1), _cache(K, k, v), start, None, SCALE)
    smax = v.float().abs().max().double() / 7
    for h, ref, size in _reference(q, k, v, start, (5,)):
        err = (out.view(tokens, nh, 128)[:, h].double() - ref).abs()
        # scores up to 68, off by 136 roundings of themselves at most
        slack = 2 * 136 * 2.0 ** -24 * 70
        bound = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -10 + slack) * size + 2.0 ** -11 * smax
        assert bool((err <= bound).all()), float((err / bound).max())


def test_negative_scale():
    K, q, k, v = _case(512, 0, 64, 8, seed=3)
    cache = _cache(K, k, v)
    a = K.kv4_prompt_attention(q.view(512, -1), cache, 0, None, -SCALE)
    b = K.kv4_prompt_attention((-q).view(512, -1).contiguous(), cache, 0, None, SCALE)
    assert torch.equal(a, b)


def test_captured_prompt_attention():
    """A captured call keeps its own workspace: replayed after other calls, with new
    rows in the cache."""
    tokens, start, nh, nkv = 70, 9003, 64, 8
    K, q, k, v = _case(tokens, start, nh, nkv, seed=4)
    cache, out = _cache(K, k, v), torch.empty(tokens, nh * 128, dtype=torch.bfloat16, device="cuda")
    K.kv4_prompt_attention(q.view(tokens, -1), cache, start, out, SCALE)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.kv4_prompt_attention(q.view(tokens, -1), cache, start, out, SCALE)
    for i in range(4):
        K.kv4_write(k.flip(0) if i % 2 else k, v.roll(i, 0), cache)
        want = K.kv4_prompt_attention(q.view(tokens, -1), cache, start, None, SCALE)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
