"""GPU: the 4-bit key/value cache against its definition in 64 bits: what is
written and read back (bit for bit), rows that stay as they were, and the
attention of one token and of a prompt over it."""
import math

import pytest
import torch

from kv4_util import attention, attention_bound, quantised, scale_of

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _kv(g, rows, nkv):
    k = torch.randn(rows, nkv, 128, device="cuda", generator=g)
    k = k * torch.exp(0.5 * torch.randn(nkv, 128, device="cuda", generator=g))
    v = torch.randn(rows, nkv, 128, device="cuda", generator=g) * 0.3
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def _same(got, want):
    """bf16 on the device against float64: equal, NaN where NaN."""
    got = got.double().cpu()
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(),
                                                                  want.nan_to_num())


@pytest.mark.parametrize("tokens,start,nkv", [(1, 0, 1), (1, 63, 3), (7, 30, 2), (32, 32, 1),
                                              (33, 31, 8), (200, 5, 4), (96, 0, 2)])
def test_write_read_is_the_definition(tokens, start, nkv):
    import _dip_hip as K
    print(f"kv4 write tokens={tokens} start={start} nkv={nkv}", flush=True)
    g = _gen(tokens + start)
    cache = K.kv4_cache(nkv, 260)
    assert cache.max_len == 288
    before = [_kv(g, 288, nkv) for _ in range(1)][0]
    K.kv4_write(*before, cache)
    k, v = _kv(g, tokens, nkv)
    # heads first, as a model's own cache holds them
    kt, vt = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
    K.kv4_write(kt, vt, cache, start=start)
    got = K.kv4_read(cache)
    for x, old, new in zip(got, before, (k, v)):
        want = quantised(old)
        want[start:start + tokens] = quantised(new)
        assert _same(x, want)
    part = K.kv4_read(cache, start, tokens)
    assert all(torch.equal(a, b[start:start + tokens]) for a, b in zip(part, got))


def test_write_values_at_the_edges():
    """Zeros, the smallest and largest numbers, ties between two steps, and groups
    with an infinity or a NaN."""
    import _dip_hip as K
    big = torch.finfo(torch.bfloat16).max
    x = torch.zeros(12, 1, 128)
    x[1] = 1e-38
    x[2] = big
    x[3] = -big
    x[4, 0, ::2], x[4, 0, 1::2] = big, -big / 3
    x[5] = torch.linspace(-7, 7, 128)
    x[6, 0, :32] = torch.arange(32) / 2 - 7.0       # steps of half a unit: ties to even
    x[6, 0, 31] = 7.0
    x[7, 0, 5] = math.inf
    x[8, 0, 40] = math.nan
    x[9, 0, 127] = -math.inf
    x[10] = 2.0 ** -97
    x[11] = 2.0 ** -96
    x = x.to(torch.bfloat16).cuda()
    cache = K.kv4_cache(1, 32)
    K.kv4_write(x, -x, cache, start=3)
    k, v = K.kv4_read(cache, 3, 12)
    assert _same(k, quantised(x)) and _same(v, quantised(-x))
    assert k[7, 0, :32].isnan().all() and not k[7, 0, 32:].isnan().any()


def test_views_with_odd_strides_are_copied():
    import _dip_hip as K
    g = _gen(5)
    wide = torch.randn(9, 2, 129, device="cuda", generator=g).to(torch.bfloat16)
    k, v = wide[..., 1:], wide.transpose(0, 1).contiguous().transpose(0, 1)[..., :128]
    cache = K.kv4_cache(2, 32)
    K.kv4_write(k, v, cache)
    gk, gv = K.kv4_read(cache, 0, 9)
    assert _same(gk, quantised(k)) and _same(gv, quantised(v))


def _rope_reference(x, w, cos, sin, eps):
    """RMSNorm and rotary embedding rounded where the model's modules round."""
    r = lambda t: t.float().to(torch.bfloat16).double()
    d = x.double()
    y = r(w.double() * r(d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)))
    half = torch.cat((-y[..., 64:], y[..., :64]), -1)
    return r(r(y * cos.double()) + r(half * sin.double()))


@pytest.mark.parametrize("tokens,start,nh,nkv", [(1, 0, 4, 2), (1, 77, 32, 8), (45, 19, 6, 3),
                                                 (64, 0, 8, 1)])
def test_norm_rope_write(tokens, start, nh, nkv):
    """q, k and v of the fused form; one token's form and the rows' agree bit for
    bit, and the other rows stay."""
    import _dip_hip as K
    print(f"kv4 norm+rope tokens={tokens} start={start} heads={nh}/{nkv}", flush=True)
    g = _gen(nh)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    qkv = rnd(tokens, (nh + 2 * nkv) * 128).to(torch.bfloat16)
    qw, kw = ((1 + 0.2 * rnd(128)).to(torch.bfloat16) for _ in range(2))
    max_len = 128
    ang = torch.arange(max_len, device="cuda")[:, None] * 0.37 ** torch.arange(
        64, device="cuda")[None] * 3.0
    cos, sin = (torch.cat((f(ang), f(ang)), -1).to(torch.bfloat16) for f in (torch.cos, torch.sin))
    cache = K.kv4_cache(nkv, max_len)
    old = _kv(g, max_len, nkv)
    K.kv4_write(*old, cache)
    q = torch.empty(tokens, nh * 128, dtype=torch.bfloat16, device="cuda")
    K.qk_norm_rope_kv4_rows(qkv, qw, kw, cos, sin, q, cache, nh, nkv, 1e-6, start=start)
    x = qkv.view(tokens, -1, 128).cpu()
    c, s = (t[start:start + tokens, None].cpu() for t in (cos, sin))
    want_q = _rope_reference(x[:, :nh], qw.cpu(), c, s, 1e-6)
    want_k = _rope_reference(x[:, nh:nh + nkv], kw.cpu(), c, s, 1e-6)
    # the sums of rounded products are taken in fp32 before they are rounded
    assert (q.view(tokens, nh, 128).double().cpu() - want_q).abs().max() <= \
        2.0 ** -7 * want_q.abs().max()
    assert (q.view(tokens, nh, 128).double().cpu() != want_q).double().mean() < 1e-3
    k, v = K.kv4_read(cache)
    for got, prev, new in ((k, old[0], want_k.to(torch.bfloat16)), (v, old[1], x[:, nh + nkv:])):
        want = quantised(prev)
        want[start:start + tokens] = quantised(new)
        assert _same(got, want)
    one = K.kv4_cache(nkv, max_len)
    q1 = torch.empty_like(q)
    for t in range(tokens):
        K.qk_norm_rope_kv4(qkv[t], qw, kw, cos, sin, torch.tensor([start + t], device="cuda"),
                           q1[t], one, nh, nkv, 1e-6)
    assert torch.equal(q1, q)
    k1, v1 = K.kv4_read(one, start, tokens)
    assert torch.equal(k1, k[start:start + tokens]) and torch.equal(v1, v[start:start + tokens])


@pytest.mark.parametrize("pos", [-1, 32, 1 << 40])
def test_token_outside_the_cache_writes_no_row(pos):
    import _dip_hip as K
    cache = K.kv4_cache(2, 32)
    qkv = torch.randn(8 * 128, device="cuda").to(torch.bfloat16)
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    cos = torch.ones(32, 128, dtype=torch.bfloat16, device="cuda")
    q = torch.full((4 * 128,), math.nan, dtype=torch.bfloat16, device="cuda")
    K.qk_norm_rope_kv4(qkv, w, w, cos, cos, torch.tensor([pos], device="cuda"), q, cache, 4, 2,
                       1e-6)
    assert not q.isnan().any()
    assert not any(t.any() for t in cache)


def _poison(cache, rows):
    """Rows behind the last one hold anything: every byte set, scales NaN."""
    cache.scales[:, rows:] = math.nan
    cache.k[:, rows:] = -1
    if rows % 32 == 0:
        cache.v[:, rows // 32:] = -1


@pytest.mark.parametrize("nh,nkv,max_len", [(32, 8, 320), (64, 8, 1024), (40, 8, 2080), (6, 2, 64),
                                            (24, 1, 640), (3, 3, 96), (16, 1, 4096)])
def test_decode_attention(nh, nkv, max_len):
    import _dip_hip as K
    g = _gen(nh * nkv + max_len)
    q = (torch.randn(nh, 128, device="cuda", generator=g) * 2).to(torch.bfloat16)
    k, v = _kv(g, max_len, nkv)
    kd, vd = quantised(k), quantised(v)
    smax = scale_of(v).max()
    for pos in (-1, 0, 1, 30, 31, 32, 33, 127, 128, max_len // 2, max_len - 1, max_len + 5):
        print(f"kv4 decode attention {nh}/{nkv} max_len={max_len} pos={pos}", flush=True)
        cache = K.kv4_cache(nkv, max_len)
        K.kv4_write(k, v, cache)
        n = min(max(pos + 1, 0), max_len)
        _poison(cache, n)
        out = K.kv4_decode_attention(q.view(-1), cache, torch.tensor([pos], device="cuda"), None,
                                     SCALE)
        ref, size = attention(q[None], kd, vd, [n], SCALE)
        err = (out.view(1, nh, 128).double().cpu() - ref).abs()
        assert bool((err <= attention_bound(ref, size, smax)).all()), float(err.max())
        if n == 0:
            assert not out.any()


@pytest.mark.parametrize("tokens,start,nh,nkv", [
    (1, 0, 4, 2), (1, 300, 32, 8), (2, 31, 64, 8), (3, 0, 3, 3), (5, 127, 40, 8), (16, 1, 16, 1),
    (33, 0, 32, 8), (100, 0, 12, 2), (64, 250, 24, 1), (129, 77, 8, 8), (257, 0, 6, 2)])
def test_prompt_attention(tokens, start, nh, nkv):
    import _dip_hip as K
    print(f"kv4 prompt attention tokens={tokens} start={start} {nh}/{nkv}", flush=True)
    g = _gen(tokens + start)
    rows = start + tokens
    q = (torch.randn(tokens, nh, 128, device="cuda", generator=g) * 2).to(torch.bfloat16)
    k, v = _kv(g, rows, nkv)
    cache = K.kv4_cache(nkv, rows + 40)
    _poison(cache, 0)
    K.kv4_write(k, v, cache)
    out = K.kv4_prompt_attention(q.view(tokens, -1), cache, start, None, SCALE)
    ref, size = attention(q, quantised(k), quantised(v), [start + t + 1 for t in range(tokens)],
                          SCALE)
    err = (out.view(tokens, nh, 128).double().cpu() - ref).abs()
    assert bool((err <= attention_bound(ref, size, scale_of(v).max())).all()), float(err.max())


@pytest.mark.parametrize("tokens,nh,nkv", [(1, 8, 2), (40, 8, 2), (300, 8, 1)])
def test_nan_rows_reach_only_who_attends_them(tokens, nh, nkv):
    """A NaN in a value's group makes those 32 dimensions of the later tokens NaN;
    one in a key makes the whole later tokens NaN."""
    import _dip_hip as K
    g = _gen(tokens)
    start = 37
    rows = start + tokens
    q = torch.randn(tokens, nh, 128, device="cuda", generator=g).to(torch.bfloat16)
    for which in ("v", "k"):
        for at in {0, start, rows - 1, rows - 1 - tokens // 2}:
            k, v = _kv(g, rows, nkv)
            (v if which == "v" else k)[at, 0, 70] = math.nan
            cache = K.kv4_cache(nkv, rows)
            K.kv4_write(k, v, cache)
            if tokens == 1:
                out = K.kv4_decode_attention(q.view(-1), cache,
                                             torch.tensor([start], device="cuda"), None, SCALE)
            else:
                out = K.kv4_prompt_attention(q.view(tokens, -1), cache, start, None, SCALE)
            nan = out.view(tokens, nh, 128).isnan().cpu()
            want = torch.zeros_like(nan)
            later = torch.arange(tokens) + start >= at
            dims = slice(64, 96) if which == "v" else slice(0, 128)
            want[later, :nh // nkv, dims] = True
            assert torch.equal(nan, want), (which, at)


def test_large_scores_and_sharp_heads():
    """Scores in the thousands: one row takes all the weight."""
    import _dip_hip as K
    g = _gen(2)
    nh, nkv, rows = 16, 2, 500
    k, v = _kv(g, rows, nkv)
    q = (k[::37].reshape(-1, 128)[:nh] * 40).to(torch.bfloat16)
    cache = K.kv4_cache(nkv, rows)
    K.kv4_write(k, v, cache)
    out = K.kv4_decode_attention(q.reshape(-1).contiguous(), cache,
                                 torch.tensor([rows - 1], device="cuda"), None, SCALE)
    kd, vd = quantised(k), quantised(v)
    ref, size = attention(q[None], kd, vd, [rows], SCALE)
    # fp32 scores of this size are off by up to 136 roundings of sum |q k|; the
    # weights move by as much
    slack = 2 * 136 * 2.0 ** -24 * SCALE * float(
        (q.double().abs().cpu()[:, None] * kd.abs().repeat_interleave(nh // nkv, 1).transpose(
            0, 1)).sum(-1).max())
    err = (out.view(1, nh, 128).double().cpu() - ref).abs()
    bound = attention_bound(ref, size, scale_of(v).max()) + 2 * slack * vd.abs().max()
    assert bool((err <= bound).all())


def test_captured_decode_attention_follows_the_position():
    """One captured launch, replayed while rows are written and the position moves
    between the replays, against eager calls."""
    import _dip_hip as K
    g = _gen(8)
    nh, nkv, max_len = 32, 8, 512
    k, v = _kv(g, max_len, nkv)
    q = torch.randn(nh * 128, device="cuda", generator=g).to(torch.bfloat16)
    cache, pos = K.kv4_cache(nkv, max_len), torch.zeros(1, dtype=torch.int64, device="cuda")
    out = torch.empty_like(q)
    K.kv4_decode_attention(q, cache, pos, out, SCALE)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.kv4_decode_attention(q, cache, pos, out, SCALE)
    for p in (0, 5, 31, 32, 100, 300, 511, 40):
        K.kv4_write(k[:p + 1], v[:p + 1], cache)
        pos.fill_(p)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, K.kv4_decode_attention(q, cache, pos, None, SCALE)), p


def test_two_streams_share_nothing():
    import _dip_hip as K
    g = _gen(11)
    nh, nkv, max_len = 64, 8, 4096
    qs = [torch.randn(nh * 128, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2)]
    caches = []
    for _ in range(2):
        c = K.kv4_cache(nkv, max_len)
        K.kv4_write(*_kv(g, max_len, nkv), c)
        caches.append(c)
    pos = torch.tensor([max_len - 1], device="cuda")
    want = [K.kv4_decode_attention(q, c, pos, None, SCALE) for q, c in zip(qs, caches)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(K.kv4_decode_attention(qs[i], caches[i], pos, None, SCALE))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_refusals():
    import _dip_hip as K
    cache = K.kv4_cache(2, 64)
    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(4 * 128, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(1, dtype=torch.int64, device="cuda")
    bad = [
        lambda: K.kv4_cache(0, 64), lambda: K.kv4_cache(2, 0),
        lambda: K.kv4_write(x, x, cache, start=61),
        lambda: K.kv4_write(x, x, cache, start=-1),
        lambda: K.kv4_write(x, x[:3], cache),
        lambda: K.kv4_write(x.float(), x, cache),
        lambda: K.kv4_write(x[:, :1], x[:, :1], cache),
        lambda: K.kv4_write(x.cpu(), x, cache),
        lambda: K.kv4_write(x, x, K.kv4_cache(2, 64, layers=2)),
        lambda: K.kv4_read(cache, 60, 5), lambda: K.kv4_read(cache, 65),
        lambda: K.kv4_decode_attention(q[:300], cache, pos, None, SCALE),
        lambda: K.kv4_decode_attention(q[:3 * 128], cache, pos, None, SCALE),
        lambda: K.kv4_decode_attention(q.float(), cache, pos, None, SCALE),
        lambda: K.kv4_decode_attention(q, cache, pos.int(), None, SCALE),
        lambda: K.kv4_decode_attention(q, cache, pos, q[:128], SCALE),
        lambda: K.kv4_decode_attention(q, cache._replace(k=cache.k[:, :32]), pos, None, SCALE),
        lambda: K.kv4_prompt_attention(q.view(2, -1), cache, 63, None, SCALE),
        lambda: K.kv4_prompt_attention(q.view(2, -1), cache, -1, None, SCALE),
        lambda: K.kv4_prompt_attention(q, cache, 0, None, SCALE),
        lambda: K.qk_norm_rope_kv4_rows(x.view(1, -1), q[:128], q[:128], x[0], x[0], q[:512],
                                        cache, 4, 2, 1e-6, start=2),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            print("not refused:", i)
    assert K.kv4_prompt_attention(q.view(1, -1)[:0], cache, 64, None, SCALE).shape == (0, 512)
    assert K.kv4_read(cache, 64)[0].shape == (0, 2, 128)
    K.kv4_write(x[:0], x[:0], cache, start=64)


@pytest.mark.parametrize("pos", [2 ** 63 - 1, 2 ** 63 - 2, -2 ** 63])
def test_token_at_the_ends_of_int64_writes_no_row(pos):
    test_token_outside_the_cache_writes_no_row(pos)


@pytest.mark.parametrize("rows", [8320, 8353, 16641, 32768, 65500])
def test_decode_attention_over_many_splits(rows):
    """Up to 256 splits, which are added up 64 at a time: half of every head's weight
    lies on an early row, half on one of the same key in a later round's split."""
    import _dip_hip as K
    nh, nkv, max_len = 8, 1, 65536
    splits = K.kv4_decode_attention_workspace_bytes(nh, nkv, max_len) // (16 * 130 * 4)
    assert splits == 256
    per = 4 * -(-(-(-rows // 32)) // (4 * splits)) * 32  # rows of a split
    assert -(-rows // per) > 64
    g = _gen(rows)
    k, v = _kv(g, rows, nkv)
    late = [64 * per, 64 * per + 31, min(100 * per + 7, rows - 5), rows * 9 // 10, rows - per - 1,
            rows - 33, rows - 2, rows - 1]
    early = [0, 17, per, 20 * per + 5, 63 * per + 1, 40 * per, 8 * per, 3 * per - 1]
    k[late] = k[early]
    cache = K.kv4_cache(nkv, max_len)
    K.kv4_write(k, v, cache)
    kd, vd = quantised(k), quantised(v)
    q = (6 * kd[early, 0] / kd[early, 0].norm(dim=-1, keepdim=True)).to(torch.bfloat16).cuda()
    _poison(cache, rows)
    out = K.kv4_decode_attention(q.view(-1), cache, torch.tensor([rows - 1], device="cuda"), None,
                                 2.0)
    ref, size = attention(q[None], kd, vd, [rows], 2.0)
    for h, (a, b) in enumerate(zip(late, early)):
        w = torch.softmax(2.0 * (kd[:, 0] @ q[h].double().cpu()), 0)
        assert float(w[a]) > 0.45 and float(w[b]) > 0.45
    # scores of up to 2 * 6 * 40, off by 136 roundings of themselves: so much of a weight
    slack = 2 * 136 * 2.0 ** -24 * 480
    err = (out.view(1, nh, 128).double().cpu() - ref).abs()
    bound = attention_bound(ref, size, scale_of(v).max()) + slack * size
    assert bool((err <= bound).all()), float((err / bound).max())
