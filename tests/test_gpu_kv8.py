"""GPU: the paged 8-bit key/value cache against its definition in 64 bits: what is
written and read back (bit for bit), rows that are rounded again or stay as they were,
and the attention of a few tokens of several sequences and of a prompt over it."""
import math

import pytest
import torch

from kv4_util import attention
from kv8_util import PAGE, Pages, attention_bound

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _kv(g, seqs, tokens, nkv):
    k = torch.randn(seqs, tokens, nkv, 128, device="cuda", generator=g)
    k = k * torch.exp(0.5 * torch.randn(nkv, 128, device="cuda", generator=g))
    v = torch.randn(seqs, tokens, nkv, 128, device="cuda", generator=g) * 0.3
    # tokens that are larger than others, so that scales rise on the way
    v = v * torch.exp(torch.randn(seqs, tokens, 1, 1, device="cuda", generator=g))
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def _same(got, want):
    """bf16 on the device against float64: equal, NaN where NaN."""
    got = got.double().cpu()
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(),
                                                                  want.nan_to_num())


def _table(widths, pages, seed):
    """Disjoint pages in no order; the rest of a row is no page."""
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    rows, width = [], max(widths)
    for w in widths:
        rows.append([order.pop() for _ in range(w)] + [-1] * (width - w))
    return rows, torch.tensor(rows, dtype=torch.int32, device="cuda")


def _pos(*p):
    return torch.tensor(p, dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("nkv", [1, 3, 8])
@pytest.mark.parametrize("tokens", [1, 2, 7, 63, 64, 65, 150])
def test_writes_in_turn_are_the_definition(tokens, nkv):
    """Several sequences at unlike positions, written again and again."""
    import _dip_hip as K
    print(f"kv8 write tokens={tokens} nkv={nkv}", flush=True)
    g = _gen(tokens * 10 + nkv)
    rows, table = _table([7, 8, 5, 6], 30, tokens)
    cache, ref = K.kv8_cache(nkv, 30), Pages(30, nkv)
    pos = [0, 70, 61, 128]
    # what lies before the first position
    k, v = _kv(g, 4, 64, nkv)
    start = [p // PAGE * PAGE for p in pos]
    K.kv8_write(k, v, cache, table, _pos(*start))
    ref.write(k, v, rows, start)
    for step in range(3):
        k, v = _kv(g, 4, tokens, nkv)
        K.kv8_write(k * 2 ** step, v * 2 ** step, cache, table, _pos(*pos))
        ref.write(k * 2 ** step, v * 2 ** step, rows, pos)
        pos = [p + tokens for p in pos]
        for i in range(4):
            n = min(pos[i], PAGE * len([p for p in rows[i] if p >= 0])) - start[i]
            got = K.kv8_read(cache, table[i:i + 1], _pos(start[i]), n)
            for x, want in zip(got, ref.read(rows[i], start[i], n)):
                assert _same(x[0], want), (step, i)
        if max(pos) + tokens > 5 * PAGE:
            break


def test_values_at_the_edges():
    """Zeros, the smallest and largest numbers, ties, rows far below their page's
    largest, and groups with an infinity or a NaN."""
    import _dip_hip as K
    big = torch.finfo(torch.bfloat16).max
    x = torch.zeros(9, 20, 1, 128)
    x[1] = 1e-38
    x[2, ::2] = big
    x[2, 1::2] = -big / 3
    x[2, 3] = 2.0 ** 127 * 1.9453125       # rounds to 2^128, held at 240 * 2^120
    x[3] = 2.0 ** torch.linspace(-16, 7, 128)
    x[4, 0] = 200.0                         # a scale of 1
    x[4, 1] = torch.arange(128) * 2.0 ** -10   # ties among the smallest
    x[4, 2] = 16 + torch.arange(128) / 2.0     # ties among larger ones
    x[5, 2, 0, 5] = math.inf
    x[5, 3, 0, 40] = math.nan
    x[5, 4, 0, 127] = -math.inf
    x[5, 5:] = 3.0
    x[6] = math.nan
    x[7] = 2.0 ** -93
    x[7, 4:] = 2.0 ** -108
    x[8] = -0.0
    x = x.to(torch.bfloat16).cuda()
    rows, table = _table([1] * 9, 9, 1)
    cache, ref = K.kv8_cache(1, 9), Pages(9, 1)
    pos = [0] * 9
    K.kv8_write(x, -x, cache, table, _pos(*pos))
    ref.write(x, -x, rows, pos)
    for step in range(2):
        k, v = K.kv8_read(cache, table, _pos(*pos), 20 + step)
        for i in range(9):
            wk, wv = ref.read(rows[i], 0, 20 + step)
            assert _same(k[i], wk) and _same(v[i], wv), (step, i)
        # one more row, which raises every scale there is
        y = torch.full((9, 1, 1, 128), 3e38, dtype=torch.bfloat16, device="cuda")
        K.kv8_write(y, y, cache, table, _pos(*[20] * 9))
        ref.write(y, y, rows, [20] * 9)


def test_every_number_reads_as_itself():
    """All 256 bytes at scales from the least to the largest, as keys and as values."""
    import _dip_hip as K
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    for e in (-100, -37, 0, 1, 64, 119):
        cache = K.kv8_cache(1, 1)
        b = torch.arange(256, device="cuda", dtype=torch.uint8)
        cache.k.view(-1)[:256] = b
        cache.v.view(128, 64)[:4] = b.view(4, 64)
        cache.scales.fill_(2.0 ** e)
        k, v = K.kv8_read(cache, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), _pos(0), 64)
        assert _same(k[0, :2, 0].reshape(-1), want * 2.0 ** e)
        r = torch.arange(64)
        at = 16 * ((r // 4) % 4) + 4 * (r // 16) + r % 4
        assert _same(v[0, :, 0, :4].t().contiguous(), want.view(4, 64)[:, at] * 2.0 ** e)


def test_going_back_and_writing_on():
    """Rejected tokens: a sequence goes back, its rows are written over; the page
    begins anew at its first row."""
    import _dip_hip as K
    g = _gen(3)
    rows, table = _table([3], 5, 2)
    cache, ref = K.kv8_cache(2, 5), Pages(5, 2)
    at = 0
    for pos, n, size in ((0, 60, 1.0), (60, 9, 40.0), (62, 5, 0.1), (64, 3, 0.01), (66, 70, 1.0),
                         (63, 1, 1e3), (64, 1, 1e-3)):
        k, v = _kv(g, 1, n, 2)
        K.kv8_write(k * size, v * size, cache, table, _pos(pos))
        ref.write(k * size, v * size, rows, [pos])
        at = pos + n
        for x, want in zip(K.kv8_read(cache, table, _pos(0), at), ref.read(rows[0], 0, at)):
            assert _same(x[0], want), (pos, n)


def test_what_has_no_page_is_left_out():
    import _dip_hip as K
    g = _gen(5)
    cache = K.kv8_cache(2, 4)
    K.kv8_write(*_kv(g, 1, 256, 2), cache, torch.arange(4, dtype=torch.int32, device="cuda")[None],
                _pos(0))
    before = [t.clone() for t in cache]
    big = 1 << 62
    table = torch.tensor([[0, 1], [-1, 4], [2, 1 << 30], [3, 3]], dtype=torch.int32, device="cuda")
    k, v = _kv(g, 4, 5, 2)
    K.kv8_write(k, v, cache, table, _pos(-1, 60, 128, -big))
    K.kv8_write(k, v, cache, table, _pos(-70, 0, 1 << 40, (1 << 63) - 1))
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    for pos in ((-1, 60, 128, -big), (-3, 0, big, (1 << 63) - 1)):
        for x in K.kv8_read(cache, table, _pos(*pos), 5):
            assert not x.any()
    # a position at the end: the rows that there are
    K.kv8_write(k[3:], v[3:], cache, table[3:], _pos(126))
    got = K.kv8_read(cache, table[3:], _pos(124), 9)[0][0]
    assert got[:4].any() and not got[4:].any()


def test_views_with_odd_strides_are_copied():
    import _dip_hip as K
    g = _gen(5)
    wide = torch.randn(2, 9, 2, 129, device="cuda", generator=g).to(torch.bfloat16)
    k, v = wide[..., 1:], wide.permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3)[..., :128]
    even = torch.randn(2, 9, 2, 134, device="cuda", generator=g).to(torch.bfloat16)[..., 2:130]
    rows, table = _table([1, 1], 2, 1)
    for a, b in ((k, v), (v, even), (even, k)):
        cache, ref = K.kv8_cache(2, 2), Pages(2, 2)
        K.kv8_write(a, b, cache, table, _pos(0, 0))
        ref.write(a, b, rows, [0, 0])
        got = K.kv8_read(cache, table, _pos(0, 0), 9)
        for i in range(2):
            assert all(_same(x[i], w) for x, w in zip(got, ref.read(rows[i], 0, 9)))


def _rope_reference(x, w, cos, sin, eps):
    """RMSNorm and rotary embedding rounded where the model's modules round."""
    r = lambda t: t.float().to(torch.bfloat16).double()
    d = x.double()
    y = r(w.double() * r(d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)))
    half = torch.cat((-y[..., 64:], y[..., :64]), -1)
    return r(r(y * cos.double()) + r(half * sin.double()))


@pytest.mark.parametrize("tokens,pos,nh,nkv", [(1, [0], 4, 2), (1, [77, 5, 64], 32, 8),
                                               (5, [60, -1, 130], 6, 3), (64, [0], 8, 1),
                                               (130, [3], 5, 5)])
def test_norm_rope_write(tokens, pos, nh, nkv):
    import _dip_hip as K
    print(f"kv8 norm+rope tokens={tokens} pos={pos} heads={nh}/{nkv}", flush=True)
    g = _gen(nh)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    seqs = len(pos)
    qkv = rnd(seqs, tokens, (nh + 2 * nkv) * 128).to(torch.bfloat16)
    qw, kw = ((1 + 0.2 * rnd(128)).to(torch.bfloat16) for _ in range(2))
    ang = torch.arange(200, device="cuda")[:, None] * 0.37 ** torch.arange(
        64, device="cuda")[None] * 3.0
    cos, sin = (torch.cat((f(ang), f(ang)), -1).to(torch.bfloat16) for f in (torch.cos, torch.sin))
    rows, table = _table([4] * seqs, 4 * seqs, 3)
    cache, ref = K.kv8_cache(nkv, 4 * seqs), Pages(4 * seqs, nkv)
    start = [max(p, 0) // PAGE * PAGE for p in pos]
    old = _kv(g, seqs, PAGE, nkv)
    K.kv8_write(*old, cache, table, _pos(*start))
    ref.write(*old, rows, start)
    q = torch.full((seqs, tokens, nh * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    K.qk_norm_rope_kv8(qkv, qw, kw, cos, sin, _pos(*pos), q, cache, table, nh, nkv, 1e-6)
    x = qkv.view(seqs, tokens, -1, 128)
    at = [torch.arange(tokens, device="cuda") + max(p, 0) for p in pos]
    c, s = (torch.stack([t[a] for a in at])[:, :, None] for t in (cos, sin))
    want_q = _rope_reference(x[:, :, :nh], qw, c, s, 1e-6)
    k = _rope_reference(x[:, :, nh:nh + nkv], kw, c, s, 1e-6).to(torch.bfloat16)
    ref.write(k, x[:, :, nh + nkv:], rows, pos)
    for i, p in enumerate(pos):
        if p < 0:
            assert bool((q[i] == 7.0).all())
            continue
        assert _same(q[i].view(tokens, nh, 128), want_q[i].cpu())
        n = p + tokens - start[i]
        got = K.kv8_read(cache, table[i:i + 1], _pos(start[i]), n)
        for a, b in zip(got, ref.read(rows[i], start[i], n)):
            assert _same(a[0], b)


def test_norm_rope_positions_beyond_the_tables():
    """Tokens at positions without a row of cos and sin, or without pages, are left out."""
    import _dip_hip as K
    g = _gen(1)
    qkv = torch.randn(2, 6, 4 * 128, device="cuda", generator=g).to(torch.bfloat16)
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    tab = torch.ones(67, 128, dtype=torch.bfloat16, device="cuda")
    _, table = _table([2, 2], 4, 1)
    cache = K.kv8_cache(1, 4)
    q = torch.full((2, 6, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    K.qk_norm_rope_kv8(qkv, w, w, tab, tab, _pos(64, 1 << 50), q, cache, table, 2, 1, 1e-6)
    assert bool((q[0, :3] != 7.0).any()) and bool((q[0, 3:] == 7.0).all())
    assert bool((q[1] == 7.0).all())
    k, _ = K.kv8_read(cache, table, _pos(64, 64), 6)
    assert k[0, :3].any() and not k[0, 3:].any() and not k[1].any()


def _filled(g, lengths, nkv, extra=2, pages=None):
    """A cache with sequences of these lengths, what they stand for, and the tables."""
    import _dip_hip as K
    widths = [max(1, -(-n // PAGE)) for n in lengths]
    total = sum(widths) + extra
    rows, table = _table(widths, total, len(lengths))
    cache, ref = K.kv8_cache(nkv, total), Pages(total, nkv)
    # other pages, and the rows behind a sequence, hold another's numbers, NaN among them
    cache.k.random_(0, 256)
    cache.v.random_(0, 256)
    cache.scales.fill_(2.0 ** 100)
    values = []
    for i, n in enumerate(lengths):
        if n:
            k, v = _kv(g, 1, n, nkv)
            K.kv8_write(k, v, cache, table[i:i + 1], _pos(0))
            ref.write(k, v, rows[i:i + 1], [0])
        values.append(ref.read(rows[i], 0, n))
    return cache, table, values


def _check(out, q, values, lengths, tokens, nh, scale=SCALE):
    for i, (k, v) in enumerate(values):
        limits = [lengths[i] - tokens + 1 + t for t in range(tokens)]
        want, size = attention(q[i].view(tokens, nh, 128), k, v, limits, scale)
        err = (out[i].view(tokens, nh, 128).double().cpu() - want).abs()
        bound = attention_bound(want, size)
        assert bool((err <= bound).all()), (i, (err / bound.clamp(min=1e-30)).max())


@pytest.mark.parametrize("tokens,lengths,nh,nkv", [
    (1, [1], 4, 2), (1, [64], 8, 8), (1, [65], 32, 8), (1, [701], 16, 1), (1, [63, 130, 1], 40, 8),
    (1, [2500], 16, 2), (2, [2, 65, 700], 12, 4), (5, [900, 64, 5], 16, 2), (5, [3333], 64, 8),
    (3, [200], 48, 3), (9, [129, 1000], 17, 1), (20, [77], 8, 1), (1, [1500, 20, 600, 64], 128, 8),
    (70, [100], 8, 2)])
def test_attention_of_few_tokens(tokens, lengths, nh, nkv):
    import _dip_hip as K
    print(f"kv8 attention tokens={tokens} lengths={lengths} heads={nh}/{nkv}", flush=True)
    g = _gen(sum(lengths))
    cache, table, values = _filled(g, lengths, nkv)
    q = torch.randn(len(lengths), tokens, nh * 128, device="cuda", generator=g).to(torch.bfloat16)
    pos = _pos(*[n - tokens for n in lengths])
    out = K.kv8_decode_attention(q, cache, table, pos, None, SCALE)
    _check(out, q, values, lengths, tokens, nh)
    assert torch.equal(out, K.kv8_decode_attention(q, cache, table, pos, None, SCALE))


@pytest.mark.parametrize("tokens,start,nh,nkv", [
    (1, 0, 4, 2), (33, 0, 32, 8), (64, 0, 8, 1), (65, 0, 6, 3), (200, 100, 16, 2), (7, 1000, 64, 8),
    (300, 0, 10, 2), (129, 1500, 8, 8), (1, 700, 8, 2), (400, 63, 16, 1)])
def test_attention_of_a_prompt(tokens, start, nh, nkv):
    import _dip_hip as K
    print(f"kv8 prompt tokens={tokens} start={start} heads={nh}/{nkv}", flush=True)
    g = _gen(tokens)
    n = start + tokens
    cache, table, values = _filled(g, [n], nkv)
    q = torch.randn(1, tokens, nh * 128, device="cuda", generator=g).to(torch.bfloat16)
    out = K.kv8_prompt_attention(q[0], cache, table[0], start, None, SCALE)
    _check(out[None], q, values, [n], tokens, nh)


def test_sequences_without_rows_and_pages():
    """A negative position gives zeros, one beyond the table attends all of it, a page
    that is none counts as zeros."""
    import _dip_hip as K
    g = _gen(8)
    nh, nkv = 8, 2
    cache, table, values = _filled(g, [100, 100, 100, 100], nkv)
    q = torch.randn(4, 2, nh * 128, device="cuda", generator=g).to(torch.bfloat16)
    out = K.kv8_decode_attention(q, cache, table, _pos(-1, -5, 98, -(1 << 62)), None, SCALE)
    assert not out[[0, 1, 3]].any()
    _check(out[2:3], q[2:3], values[2:3], [100], 2, nh)
    # every row of the table's two pages, those behind the sequence zero here
    k, v = K.kv8_read(cache, table, _pos(0, 0, 0, 0), 128)
    far = K.kv8_decode_attention(q, cache, table, _pos(*[(1 << 63) - 1] * 4), None, SCALE)
    ok = [i for i in range(4) if not (k[i].isnan().any() or v[i].isnan().any())]
    for i in ok:
        _check(far[i:i + 1], q[i:i + 1], [(k[i].double().cpu(), v[i].double().cpu())], [129], 2, nh)
    bad = table.clone()
    bad[0, 0], bad[1, 0] = -7, 1 << 30
    out = K.kv8_decode_attention(q, cache, bad, _pos(98, 98, 98, 98), None, SCALE)
    k, v = K.kv8_read(cache, bad, _pos(0, 0, 0, 0), 100)
    assert not k[0, :64].any() and k[0, 64:].any()
    _check(out, q, [(k[i].double().cpu(), v[i].double().cpu()) for i in range(4)], [100] * 4, 2, nh)
    for i in range(2):
        part = K.kv8_prompt_attention(q[i], cache, bad[i], 98, None, SCALE)
        _check(part[None], q[i:i + 1], [(k[i].double().cpu(), v[i].double().cpu())], [100], 2, nh)


@pytest.mark.parametrize("tokens,nh,nkv", [(3, 8, 2), (2, 32, 1), (5, 16, 1), (70, 16, 2)])
def test_nan_belongs_to_the_columns_that_attend_it(tokens, nh, nkv):
    """A NaN in a later token's key or value leaves the earlier tokens' results as they
    are; in an attended value it makes its group of dimensions NaN."""
    import _dip_hip as K
    g = _gen(9)
    n = 130
    rows, table = _table([3], 4, 1)
    cache, ref = K.kv8_cache(nkv, 4), Pages(4, nkv)
    k, v = _kv(g, 1, n, nkv)
    v[0, n - 2, 0, 40] = math.nan           # the last token but one's
    k[0, n - 1, nkv - 1, 3] = math.inf      # the last one's
    v[0, 5, nkv - 1, 100] = -math.inf       # every one's
    K.kv8_write(k, v, cache, table, _pos(0))
    ref.write(k, v, rows, [0])
    q = torch.randn(1, tokens, nh * 128, device="cuda", generator=g).to(torch.bfloat16)
    out = K.kv8_decode_attention(q, cache, table, _pos(n - tokens), None, SCALE)
    alone = K.kv8_prompt_attention(q[0], cache, table[0], n - tokens, None, SCALE)
    kk, vv = ref.read(rows[0], 0, n)
    limits = [n - tokens + 1 + t for t in range(tokens)]
    want, size = attention(q[0].view(tokens, nh, 128), kk, vv, limits, SCALE)
    assert want.isnan().any() and not want.isnan().all()
    for x in (out[0], alone):
        x = x.view(tokens, nh, 128).double().cpu()
        assert torch.equal(x.isnan(), want.isnan())
        ok = ~want.isnan()
        assert bool(((x - want).abs() <= attention_bound(want, size))[ok].all())


def test_large_values_and_scores():
    """Sums of the largest values stay finite; scores far from each other and beyond
    2^31; a query with an infinity."""
    import _dip_hip as K
    big = torch.finfo(torch.bfloat16).max
    rows, table = _table([40], 40, 1)
    cache, ref = K.kv8_cache(1, 40), Pages(40, 1)
    g = _gen(4)
    k, v = _kv(g, 1, 2560, 1)
    v = torch.full_like(v, big)
    K.kv8_write(k, v, cache, table, _pos(0))
    ref.write(k, v, rows, [0])
    q = torch.randn(1, 2, 256, device="cuda", generator=g).to(torch.bfloat16)
    for x in (K.kv8_decode_attention(q, cache, table, _pos(2558), None, SCALE)[0],
              K.kv8_prompt_attention(q[0], cache, table[0], 2558, None, SCALE)):
        assert bool((x.double() == 240 * 2.0 ** 120).all())
    k, v = _kv(g, 1, 2560, 1)
    K.kv8_write(k, v, cache, table, _pos(0))
    ref.write(k, v, rows, [0])
    kk, vv = ref.read(rows[0], 0, 2560)
    for size in (1e3, 1e9, 1e30):
        out = K.kv8_decode_attention(q * size, cache, table, _pos(2558), None, SCALE)
        # one row takes all: its value to the last bit
        s = (q[0] * size).view(2, 2, 128).double().cpu() @ kk[:, 0].T * SCALE
        for t in range(2):
            for h in range(2):
                best = s[t, h, :2559 + t].sort(descending=True)
                if best.values[0] - best.values[1] > 1e-4 * best.values[0].abs() + 40:
                    assert torch.equal(out[0, t, 128 * h:128 * h + 128].double().cpu(),
                                       vv[best.indices[0], 0])
        assert bool(out.isfinite().all())
    q[0, 0, 3] = math.inf
    out = K.kv8_decode_attention(q, cache, table, _pos(2558), None, SCALE)
    assert out[0, 0, :128].isnan().all() and out[0, 1].isfinite().all()


def test_outputs_workspaces_and_streams():
    """Given outputs and workspaces, another stream, and two captured graphs that run
    at once, each with a workspace of its own."""
    import _dip_hip as K
    g = _gen(11)
    nh, nkv, lengths = 32, 8, [3000, 2000]
    cache, table, values = _filled(g, lengths, nkv)
    qs = [torch.randn(2, 1, nh * 128, device="cuda", generator=g).to(torch.bfloat16)
          for _ in range(2)]
    pos = _pos(2999, 1999)
    want = [K.kv8_decode_attention(q, cache, table, pos, None, SCALE) for q in qs]
    _check(want[0], qs[0], values, lengths, 1, nh)
    n = K.kv8_decode_attention_workspace_bytes(2, 1, nh, nkv, table.shape[1])
    assert n > 0
    out, ws = torch.empty_like(qs[0]), torch.empty(n, dtype=torch.uint8, device="cuda")
    assert K.kv8_decode_attention(qs[0], cache, table, pos, out, SCALE, ws=ws) is out
    assert torch.equal(out, want[0])
    with pytest.raises(RuntimeError):
        K.kv8_decode_attention(qs[0], cache, table, pos, None, SCALE, ws=ws[:n - 1])
    graphs, outs = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(K.kv8_decode_attention(q, cache, table, pos, None, SCALE))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        assert torch.equal(K.kv8_decode_attention(qs[0], cache, table, pos, None, SCALE), want[0])


def test_a_step_of_many_sequences():
    """Write and attend together, as a step of several sequences does, token after
    token: the same as the sequences one by one."""
    import _dip_hip as K
    g = _gen(21)
    nh, nkv, seqs, steps = 8, 2, 5, 4
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g).to(torch.bfloat16)
    qw, kw = rnd(128), rnd(128)
    cos, sin = rnd(256, 128), rnd(256, 128)
    lengths = [62, 1, 130, 64, 7]
    _, table = _table([3] * seqs, 16, 5)
    one, many = K.kv8_cache(nkv, 16), K.kv8_cache(nkv, 16)
    for i, n in enumerate(lengths):
        k, v = _kv(g, 1, n, nkv)
        for c in (one, many):
            K.kv8_write(k, v, c, table[i:i + 1], _pos(0))
    pos = _pos(*lengths)
    for step in range(steps):
        qkv = rnd(seqs, 1, (nh + 2 * nkv) * 128)
        q, q1 = (torch.empty(seqs, 1, nh * 128, dtype=torch.bfloat16, device="cuda")
                 for _ in range(2))
        K.qk_norm_rope_kv8(qkv, qw, kw, cos, sin, pos, q, many, table, nh, nkv, 1e-6)
        out = K.kv8_decode_attention(q, many, table, pos, None, SCALE)
        for i in range(seqs):
            K.qk_norm_rope_kv8(qkv[i:i + 1], qw, kw, cos, sin, pos[i:i + 1], q1[i:i + 1], one,
                               table[i:i + 1], nh, nkv, 1e-6)
            alone = K.kv8_prompt_attention(q1[i], one, table[i], lengths[i] + step, None, SCALE)
            assert torch.equal(q[i], q1[i])
            # split unlike: the same sums in another order, and their bf16 roundings
            assert (out[i].float() - alone.float()).abs().max() <= 2.0 ** -7 * out[i].float().abs().max()
        assert all(torch.equal(a, b) for a, b in zip(one, many))
        pos += 1
