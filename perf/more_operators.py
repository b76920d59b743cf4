"""Calls of decoding several sequences over a paged 8-bit key/value cache with
drafted tokens, as cases to time: a step's or a prompt's keys and values into the
cache (norm and rotary embedding on the way), the attention of a few tokens of each
sequence and of a prompt over it, and the verification of drafted tokens against the
target's logits.

The cache is in pages of 64 rows (positions).  Of each page, key/value head and kind
(keys, values) the numbers are e4m3 and share a scale s, a power of two: with a the
largest magnitude of the rows written, 2^(floor(log2 a) - 7).  A write that raises a
page's scale rounds the earlier rows' numbers again.

``own`` False: the operators in elementary torch operations; True: through the
framework's entry points.
"""
import math
import sys
from pathlib import Path
from types import SimpleNamespace

import numpy as np
import torch

own = False

DEV = "cuda:0"
HD = 128     # head dimension
PAGE = 64    # rows of a page
EPS = 1e-6
THETA = 1e6
VOCAB = 151936
HEADS = ((32, 8), (64, 8), (40, 8), (16, 8), (4, 2), (16, 1))  # (query, key/value) heads
PACKAGE = Path(__file__).resolve().parent.parent / "dynamic-input-pruning_amd"


def _framework():
    if str(PACKAGE) not in sys.path:
        sys.path.insert(0, str(PACKAGE))
    import _dip_hip
    return _dip_hip


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one layer's rows of a step of one sequence: a few KB, where launches count
        dict(name="append_token", kind="append", seqs=1, tokens=1, rows=700, heads=32,
             kv_heads=8),
        # of a step of many sequences with four drafted tokens each
        dict(name="append_batch", kind="append", seqs=24, tokens=5, rows=9000, heads=64,
             kv_heads=8),
        # of a long prompt, an odd length
        dict(name="append_prompt", kind="append", seqs=1, tokens=4099, rows=4099, heads=64,
             kv_heads=8),
        # one token's attention in a chat; of a batch of sequences of all lengths; at
        # the end of a very long sequence, five heads to a key/value head
        dict(name="token_short", kind="token", seqs=1, tokens=1, rows=701, heads=32, kv_heads=8),
        dict(name="token_batch", kind="token", seqs=32, tokens=1, rows=16384, heads=64,
             kv_heads=8),
        dict(name="token_longest", kind="token", seqs=1, tokens=1, rows=131071, heads=40,
             kv_heads=8),
        # a token and its four drafted ones in each of some sequences
        dict(name="tokens_drafted", kind="token", seqs=6, tokens=5, rows=20011, heads=64,
             kv_heads=8),
        # a long prompt, and a further part of one behind a long conversation
        dict(name="prompt_long", kind="prompt", tokens=4096, rows=4096, heads=64, kv_heads=8),
        dict(name="prompt_chunk", kind="prompt", tokens=509, rows=16512, heads=64, kv_heads=8),
        # four tokens drafted without probabilities (found in the text, or greedily) with
        # the usual settings; drafts of a smaller model in a batch, top-p and min-p; many
        # short ones without a filter
        dict(name="verify_one", kind="verify", seqs=1, tokens=4, vocab=VOCAB, dtype="bfloat16",
             drawn=False, temperature=0.7, top_k=20, top_p=0.8, min_p=0.0),
        dict(name="verify_batch", kind="verify", seqs=16, tokens=5, vocab=VOCAB, dtype="float32",
             drawn=True, temperature=1.0, top_k=0, top_p=0.95, min_p=0.02),
        dict(name="verify_plain", kind="verify", seqs=50, tokens=3, vocab=32003, dtype="bfloat16",
             drawn=True, temperature=1.3, top_k=0, top_p=1.0, min_p=0.0),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "append", "token", "token", "prompt", "prompt", "verify",
                       "verify"))
    nh, nkv = rng.choice(HEADS)
    if kind == "append":
        seqs = rng.choice((1, 1, _spread(rng, 2, 40)))
        tokens = _spread(rng, 1, 4096 if seqs == 1 else 9)
        return dict(kind=kind, seqs=seqs, tokens=tokens, rows=tokens + rng.randint(0, 2000),
                    heads=nh, kv_heads=nkv)
    if kind == "token":
        seqs = rng.choice((1, 1, _spread(rng, 2, 40)))
        tokens = rng.choice((1, 1, rng.randint(2, 9)))
        rows = _spread(rng, tokens, 100000 if seqs == 1 else 400000 // (seqs * tokens))
        return dict(kind=kind, seqs=seqs, tokens=tokens, rows=rows, heads=nh, kv_heads=nkv)
    if kind == "prompt":
        tokens = _spread(rng, 1, 2048)
        # as many pairs of tokens and rows as the longest listed prompt at most
        start = rng.choice((0, _spread(rng, 1, min(16000, 2 ** 23 // tokens - tokens))))
        return dict(kind=kind, tokens=tokens, rows=start + tokens, heads=nh, kv_heads=nkv)
    vocab = rng.choice((VOCAB, _spread(rng, 7, VOCAB)))
    tokens = rng.randint(1, 8)
    return dict(kind=kind, seqs=_spread(rng, 1, max(1, min(32, 2 ** 22 // vocab // tokens))),
                tokens=tokens, vocab=vocab,
                dtype=rng.choice(("bfloat16", "bfloat16", "float32", "float16")),
                drawn=rng.random() < 0.5, temperature=round(rng.uniform(0.3, 1.6), 2),
                top_k=rng.choice((0, 1, _spread(rng, 2, 2000))),
                top_p=rng.choice((1.0, round(rng.uniform(0.05, 0.999), 3))),
                min_p=rng.choice((0.0, round(rng.uniform(0.001, 0.3), 3))))


def _lengths(c):
    """Rows of each sequence with this call's tokens: the longest c.rows, the others
    even down to a small part of it."""
    seqs = getattr(c, "seqs", 1)
    return [max(c.tokens, c.rows * (2 * (seqs - i) - 1) // (2 * seqs - 1)) for i in range(seqs)]


def _window(c):
    """Rows that are read back of each sequence, from the first page that a write
    touches: to the end of the last one."""
    most = max((n - c.tokens) % PAGE for n in _lengths(c)) + c.tokens
    return -(-most // PAGE) * PAGE


def work(case):
    c = SimpleNamespace(**case)
    if c.kind == "verify":
        size = 4 if c.dtype == "float32" else 2
        rows = c.seqs * (c.tokens + 1 + (c.tokens if c.drawn else 0))
        return {"bytes": rows * c.vocab * size + c.seqs * (c.tokens + 1) * (4 + 8 + 8),
                "flops": 4 * rows * c.vocab}
    page = 2 * (PAGE * HD + 4)  # bytes of a page, a key/value head's
    if c.kind == "append":
        n, w = c.seqs * c.tokens, c.seqs * _window(c)
        heads = n * (c.heads + 2 * c.kv_heads) * HD
        # q|k|v and the tables' rows in, q out, the rows' numbers, and the touched pages
        # read back as bf16
        return {"bytes": 2 * heads + 4 * n * HD + 2 * n * c.heads * HD + 2 * n * c.kv_heads * HD
                + w // PAGE * c.kv_heads * page + 4 * w * c.kv_heads * HD, "flops": 12 * heads}
    lengths = _lengths(c)
    pairs = sum(c.tokens * n - c.tokens * (c.tokens - 1) // 2 for n in lengths)
    return {"bytes": sum(lengths) * c.kv_heads * 2 * (HD + 4 / PAGE)
            + 4 * len(lengths) * c.tokens * c.heads * HD, "flops": 4 * HD * c.heads * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _tables(rows):
    """cos and sin of every position, bf16 [rows, HD], angles in 64 bits."""
    inv = THETA ** (-torch.arange(0, HD, 2, device=DEV, dtype=torch.float64) / HD)
    angle = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * inv
    angle = torch.cat((angle, angle), -1)
    return angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)


def _keys_values(g, rows, nkv):
    """Keys as a normed and rotated head gives them (channels of unlike sizes, tokens
    that are now and then larger) and values, bf16 [rows, nkv, HD]."""
    channel = torch.exp(0.4 * _randn(g, nkv, HD))
    k = _randn(g, rows, nkv, HD) * channel
    v = _randn(g, rows, nkv, HD) * 0.5 * torch.exp(0.3 * _randn(g, rows, 1, 1))
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def _logits(g, rows, vocab):
    """A broad floor of unlikely tokens and some likely ones; in every eighth
    row all but some 200 tokens masked."""
    x = 2.0 * _randn(g, rows, vocab)
    x += 9.0 * torch.rand(rows, vocab, device=DEV, generator=g).pow(40)
    keep = torch.rand(rows, vocab, device=DEV, generator=g) < 200.0 / vocab
    masked = (torch.arange(rows, device=DEV) % 8 == 3)[:, None] & ~keep
    return x.masked_fill(masked, float("-inf"))


def _prepare_verify(s, g):
    dtype, vocab = getattr(torch, s.dtype), s.vocab
    x = _logits(g, s.seqs * (s.tokens + 1), vocab).view(s.seqs, s.tokens + 1, vocab)
    # the drafting model's logits are the target's with some noise
    y = (x[:, :s.tokens] + 0.4 * _randn(g, s.seqs, s.tokens, vocab)).to(dtype)
    s.logits = x.to(dtype)
    s.u = torch.rand(s.seqs, s.tokens + 1, device=DEV, generator=g)
    if s.drawn:
        s.draft_logits = y
        w = _kept(y.view(-1, vocab), s)
        s.drafted = torch.multinomial(w / w.sum(-1, keepdim=True), 1, generator=g)
    else:
        s.draft_logits = None
        s.drafted = y.view(-1, vocab).argmax(-1)
    s.drafted = s.drafted.view(s.seqs, s.tokens).contiguous()
    s.drafted[3::4, -1:] = -1  # some sequences have one less
    return s


def prepare(case, seed):
    s = SimpleNamespace(**case)
    g = _gen(seed)
    if own:
        s.K = _framework()
    if s.kind == "verify":
        return _prepare_verify(s, g)
    s.lengths = _lengths(s)
    s.seqs = len(s.lengths)
    pages = [-(-n // PAGE) for n in s.lengths]
    # pages in no order, as sequences that come and go leave them
    order = torch.randperm(sum(pages), generator=torch.Generator().manual_seed(seed))
    table, first = torch.zeros(s.seqs, max(pages), dtype=torch.int32), 0
    for i, n in enumerate(pages):
        table[i, :n] = order[first:first + n]
        first += n
    s.start = [n - s.tokens for n in s.lengths]
    s.pos = torch.tensor(s.start, device=DEV)
    if own:
        s.table = table.to(DEV)
        s.cache = s.K.kv8_cache(s.kv_heads, sum(pages), DEV)
    if s.kind == "append":
        s.qkv = _randn(g, s.seqs, s.tokens, (s.heads + 2 * s.kv_heads) * HD).to(torch.bfloat16)
        s.q_w = (1 + 0.2 * _randn(g, HD)).to(torch.bfloat16)
        s.k_w = (1 + 0.2 * _randn(g, HD)).to(torch.bfloat16)
        s.cos, s.sin = _tables(max(s.lengths))
        s.q = torch.empty(s.seqs, s.tokens, s.heads * HD, device=DEV, dtype=torch.bfloat16)
        s.window = _window(s)
        # the earlier rows of the first page that the tokens touch
        k, v = _keys_values(g, s.seqs * PAGE, s.kv_heads)
        old = (torch.arange(PAGE, device=DEV) < (s.pos % PAGE)[:, None])[..., None, None]
        s.old_k, s.old_v = (x.view(s.seqs, PAGE, s.kv_heads, HD) * 0.8 * old for x in (k, v))
        s.page_at = s.pos // PAGE * PAGE
        if own:
            s.K.kv8_write(s.old_k, s.old_v, s.cache, s.table, s.page_at)
        return s
    # heads that look at a few rows and heads that look at many
    sharp = torch.linspace(0.5, 3.0, s.heads, device=DEV)[:, None]
    s.q = (_randn(g, s.seqs, s.tokens, s.heads, HD) * sharp).to(torch.bfloat16).view(
        s.seqs, s.tokens, -1)
    s.scale = 1 / math.sqrt(HD)
    s.k, s.v = [], []
    for i, n in enumerate(s.lengths):
        k, v = _keys_values(g, n, s.kv_heads)
        if own:
            s.K.kv8_write(k[None], v[None], s.cache, s.table[i:i + 1],
                          torch.zeros(1, dtype=torch.int64, device=DEV))
        else:
            s.k.append(_paged_values(k))
            s.v.append(_paged_values(v))
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    if s.kind == "append":
        return _plain_append(s)
    if s.kind == "verify":
        return _plain_verify(s)
    return torch.stack([_plain_attention(s.q[i], s.k[i], s.v[i], s) for i in range(s.seqs)])


def _run_own(s):
    K = s.K
    if s.kind == "append":
        K.qk_norm_rope_kv8(s.qkv, s.q_w, s.k_w, s.cos, s.sin, s.pos, s.q, s.cache, s.table,
                           s.heads, s.kv_heads, EPS)
        k, v = K.kv8_read(s.cache, s.table, s.page_at, s.window)
        return s.q, k, v
    if s.kind == "token":
        return K.kv8_decode_attention(s.q, s.cache, s.table, s.pos, None, s.scale)
    if s.kind == "prompt":
        return K.kv8_prompt_attention(s.q[0], s.cache, s.table[0], s.start[0], None,
                                      s.scale)[None]
    return K.verify(s.logits, s.drafted, s.u, s.draft_logits, temperature=s.temperature,
                    top_k=s.top_k, top_p=s.top_p, min_p=s.min_p)


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _page_scale(x):
    """x fp32 [..., PAGE, heads, HD] -> the scale of each page and head, [..., 1, heads, 1]."""
    a = x.abs().amax((-3, -1), keepdim=True)
    return (a.view(torch.int32) & 0x7F800000).view(torch.float32) * 2.0 ** -7


def _numbers(x, s):
    """x / s rounded to e4m3, fp32 (0 where s is)."""
    n = torch.where(s > 0, x / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(x))
    return n.to(torch.float8_e4m3fn).float()


def _paged_values(x):
    """What bf16 rows [rows, heads, HD], written together into pages of their own,
    stand for there: bf16 numbers."""
    rows = x.shape[0]
    p = torch.zeros(-(-rows // PAGE) * PAGE, *x.shape[1:], device=DEV)
    p[:rows] = x
    p = p.unflatten(0, (-1, PAGE))
    s = _page_scale(p)
    return (_numbers(p, s) * s).flatten(0, 1)[:rows].to(torch.bfloat16)


def _rounded(x):
    return x.to(torch.bfloat16).float()


def _plain_rope(x, w, cos, sin):
    """RMSNorm of each head (its mean and root in 64 bits, so that no value next
    to a border of the cache's steps turns on the order of a sum), rotary
    embedding, rounded where the model's modules round."""
    d = x.double()
    r = 1 / (d.square().mean(-1, keepdim=True) + EPS).sqrt()
    y = _rounded(w.float() * _rounded(d * r))
    half = torch.cat((-y[..., HD // 2:], y[..., :HD // 2]), -1)
    return (_rounded(y * cos.float()) + _rounded(half * sin.float())).to(torch.bfloat16)


def _plain_append(s):
    """(q, keys and values of the touched pages' rows as bf16)."""
    x = s.qkv.view(s.seqs, s.tokens, -1, HD)
    at = s.pos[:, None] + torch.arange(s.tokens, device=DEV)
    cos, sin = (t[at][:, :, None] for t in (s.cos, s.sin))
    q = _plain_rope(x[:, :, :s.heads], s.q_w, cos, sin)
    k = _plain_rope(x[:, :, s.heads:s.heads + s.kv_heads], s.k_w, cos, sin)
    out = [q.reshape(s.seqs, s.tokens, -1)]
    row = (at - s.page_at[:, None])[..., None, None].expand(-1, -1, s.kv_heads, HD)
    for old, new in ((s.old_k, k), (s.old_v, x[:, :, s.heads + s.kv_heads:])):
        p = torch.zeros(s.seqs, s.window, s.kv_heads, HD, device=DEV).scatter_(
            1, row, new.float()).unflatten(1, (-1, PAGE))
        sc = _page_scale(p)
        before = old.float()
        sc_old = _page_scale(before)
        sc[:, 0] = torch.maximum(sc[:, 0], sc_old)
        v = _numbers(p, sc) * sc
        # the first page's earlier rows, rounded once more where its scale rises
        n = _numbers(before, sc_old) * sc_old
        v[:, 0] += _numbers(n, sc[:, 0]) * sc[:, 0]
        out.append(v.flatten(1, 2).to(torch.bfloat16))
    return tuple(out)


def _plain_attention(q, k, v, s):
    """[tokens, heads * HD]: token t attends the rows up to its own."""
    rows, tokens, group = k.shape[0], q.shape[0], s.heads // s.kv_heads
    k = k.float().permute(1, 2, 0).contiguous()     # [nkv, HD, rows]
    v = v.float().transpose(0, 1).contiguous()      # [nkv, rows, HD]
    q = q.view(tokens, s.kv_heads, group, HD).permute(1, 0, 2, 3).reshape(s.kv_heads, -1, HD)
    x = torch.matmul(q.float(), k) * s.scale                        # [nkv, tokens * group, rows]
    limit = rows - tokens + torch.arange(tokens, device=DEV).repeat_interleave(group)
    x = x.masked_fill(torch.arange(rows, device=DEV) > limit[:, None], float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(x, v) / x.sum(-1, keepdim=True)
    o = o.view(s.kv_heads, tokens, group, HD).permute(1, 0, 2, 3)
    return o.reshape(tokens, -1).to(torch.bfloat16)


def _kept(logits, s):
    """The weights of the kept tokens of rows of logits, in 64 bits."""
    x, order = torch.sort(logits.double(), dim=-1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / s.temperature)
    if s.top_k:
        w[:, s.top_k:] = 0
    if s.top_p < 1:
        before = w.cumsum(-1) - w
        w = w * (before < s.top_p * w.sum(-1, keepdim=True))
    w = w * (w >= s.min_p)
    return torch.zeros_like(w).scatter_(-1, order, w)


def _plain_verify(s):
    """(tokens int64 [seqs, tokens + 1], -1 behind the last, accepted int64 [seqs])."""
    n, u = s.tokens, s.u.double()
    p = _kept(s.logits.view(-1, s.vocab), s)
    p = (p / p.sum(-1, keepdim=True)).view(s.seqs, n + 1, s.vocab)
    there = (s.drafted >= 0) & (s.drafted < s.vocab)
    x = s.drafted.clamp(0, s.vocab - 1)[..., None]
    if s.draft_logits is None:
        q = torch.zeros_like(p[:, :n]).scatter_(-1, x, 1.0)
    else:
        q = _kept(s.draft_logits.view(-1, s.vocab), s)
        q = (q / q.sum(-1, keepdim=True)).view(s.seqs, n, s.vocab)
    ok = (u[:, :n] * q.gather(-1, x)[..., 0] < p[:, :n].gather(-1, x)[..., 0]) & there
    accepted = ok.long().cumprod(-1).sum(-1)
    # what the next token is drawn from
    q = torch.cat((torch.where(there[..., None], q, 0.0), torch.zeros_like(p[:, :1])), 1)
    row = accepted[:, None, None].expand(-1, 1, s.vocab)
    p, q = p.gather(1, row)[:, 0], q.gather(1, row)[:, 0]
    w = (p - q).clamp(min=0)
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, p)
    run = w.cumsum(-1)
    token = (run <= u[:, n:] * run[:, -1:]).sum(-1).clamp(max=s.vocab - 1)
    at = torch.arange(n + 1, device=DEV)
    out = torch.cat((s.drafted, torch.full_like(s.drafted[:, :1], -1)), 1)
    out = torch.where(at < accepted[:, None], out, -1)
    return torch.where(at == accepted[:, None], token[:, None], out), accepted


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _power(e):
    """2 ** e in 64 bits for whole numbers e, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _bf16_64(x):
    """x (64 bits) to the nearest bf16 number, ties to even, as 64 bits."""
    m, e = torch.frexp(x)
    return torch.round(m * 256) * _power(e - 8)


def _e4m3_64(x):
    """x (64 bits, up to 448) to the nearest e4m3 number, ties to even, as 64 bits."""
    step = _power(torch.frexp(x)[1].clamp(min=-5) - 4)
    return torch.round(x / step) * step


def _scale_64(x):
    """The scale of rows x [rows, HD] of one page and head, 0 if they are 0."""
    a = x.abs().max()
    return _power(torch.frexp(a)[1] - 8) * (a > 0)


def _values_64(x, s):
    return _e4m3_64(x / s) * s if s > 0 else torch.zeros_like(x)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"append": _exact_append, "token": _exact_attention, "prompt": _exact_attention,
            "verify": _exact_verify}[s.kind](s)


def _exact_append(s):
    x = s.qkv.double().view(s.seqs, s.tokens, -1, HD)
    turned = []
    for first, n, w in ((0, s.heads, s.q_w), (s.heads, s.kv_heads, s.k_w)):
        y = x[:, :, first:first + n]
        root = torch.sqrt((y * y).sum(-1, keepdim=True) / HD + EPS)
        y = _bf16_64(w.double() * _bf16_64(y / root))
        lo, hi = y.split(HD // 2, -1)
        c, t = (torch.stack([z[p:p + s.tokens, None, :HD // 2].double() for p in s.start])
                for z in (s.cos, s.sin))
        turned.append(torch.cat((_bf16_64(_bf16_64(lo * c) + _bf16_64(-hi * t)),
                                 _bf16_64(_bf16_64(hi * c) + _bf16_64(lo * t))), -1))
    got = [turned[0].reshape(s.seqs, s.tokens, -1)]
    for old, new in ((s.old_k, turned[1]), (s.old_v, x[:, :, s.heads + s.kv_heads:])):
        out = torch.zeros(s.seqs, s.window, s.kv_heads, HD, dtype=torch.float64, device=DEV)
        for i in range(s.seqs):
            r = s.start[i] % PAGE
            for h in range(s.kv_heads):
                for at in range(0, r + s.tokens, PAGE):
                    a, b = max(at, r), min(at + PAGE, r + s.tokens)
                    rows = new[i, a - r:b - r, h]
                    sc = _scale_64(rows)
                    if at == 0 and r > 0:
                        before = old[i, :r, h].double()
                        was = _scale_64(before)
                        sc = torch.maximum(sc, was)
                        out[i, :r, h] = _values_64(_values_64(before, was), sc)
                    out[i, a:b, h] = _values_64(rows, sc)
        got.append(out)
    return tuple(got)


def _exact_attention(s):
    group = s.heads // s.kv_heads
    out = torch.empty(s.seqs, s.tokens, s.heads, HD, dtype=torch.float64, device=DEV)
    for i, rows in enumerate(s.lengths):
        later = (torch.arange(rows, device=DEV)
                 > s.start[i] + torch.arange(s.tokens, device=DEV)[:, None])
        for h in range(s.heads):
            k, v = (x[i][:, h // group].double() for x in (s.k, s.v))
            x = s.q[i].view(s.tokens, s.heads, HD)[:, h].double() @ k.T.contiguous() * s.scale
            out[i, :, h] = torch.softmax(x.masked_fill(later, -math.inf), -1) @ v
    return out.view(s.seqs, s.tokens, -1)


def _shares(x, s):
    """The probabilities of one row of logits after the filters, float64 numpy."""
    order = np.lexsort((np.arange(s.vocab), -x))
    n = min(s.top_k or s.vocab, s.vocab)
    w = np.exp((x[order[:n]] - x.max()) / s.temperature)
    if s.top_p < 1:
        w = w[:1 + int(np.searchsorted(np.cumsum(w), s.top_p * w.sum()))]
    w = w[w >= s.min_p]
    out = np.zeros(s.vocab)
    out[order[:len(w)]] = w / w.sum()
    return out


def _exact_verify(s):
    target, u = s.logits.double().cpu().numpy(), s.u.double().cpu().numpy()
    draft = None if s.draft_logits is None else s.draft_logits.double().cpu().numpy()
    drafted = s.drafted.cpu().numpy()
    tokens = np.full((s.seqs, s.tokens + 1), -1, np.int64)
    accepted = np.zeros(s.seqs, np.int64)
    for i in range(s.seqs):
        for t in range(s.tokens + 1):
            w = _shares(target[i, t], s)
            x = drafted[i, t] if t < s.tokens else -1
            if 0 <= x < s.vocab:
                if draft is None:
                    q = np.zeros(s.vocab)
                    q[x] = 1
                else:
                    q = _shares(draft[i, t], s)
                if u[i, t] * q[x] < w[x]:
                    tokens[i, t] = x
                    continue
                rest = np.maximum(w - q, 0)
                w = rest if rest.sum() > 0 else w
            run = np.cumsum(w)
            at = int(np.searchsorted(run, u[i, -1] * run[-1], side="right"))
            tokens[i, t] = min(at, int(np.nonzero(w)[0][-1]))
            accepted[i] = t
            break
    return tokens, accepted
