"""Calls of a decode step with a 4-bit key/value cache, as cases to time: writing
a token's or a prompt's keys and values into the cache, the attention of one
token and of a prompt over it, and drawing the next token from the logits.

The cache holds, per row (position), key/value head and group of 32 dimensions,
a scale s and 32 whole numbers q in [-7, 7]; a value is q * s.  With a the
group's largest magnitude, s is a / 7 cut to five significant bits, which makes
every q * s a bf16 number, and q = rint(x / s).

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
GROUP = 32   # dimensions that share a scale
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
        # one layer's keys and values of one token in the default 1024-row
        # cache: a few KB, where the launches count
        dict(name="row_token", kind="rows", tokens=1, start=700, heads=32, kv_heads=8,
             max_len=1024),
        # the same for a long prompt of the 64-head shape, an odd length
        dict(name="rows_prompt", kind="rows", tokens=4099, start=0, heads=64, kv_heads=8,
             max_len=8192),
        # one token's attention: a chat's length, a long conversation at an odd
        # position, and a cache at the end of its range with a group of 5 heads
        dict(name="token_short", kind="token", pos=700, heads=32, kv_heads=8, max_len=1024),
        dict(name="token_long", kind="token", pos=20010, heads=64, kv_heads=8, max_len=32768),
        dict(name="token_longest", kind="token", pos=131070, heads=40, kv_heads=8,
             max_len=131072),
        # a prompt's attention: the short prompt of the decode benchmark, a long
        # one, a further chunk behind a long conversation, and a few tokens
        # behind one (a turn's first words, drafted tokens)
        dict(name="prompt_short", kind="prompt", tokens=33, start=0, heads=32, kv_heads=8,
             max_len=1024),
        dict(name="prompt_long", kind="prompt", tokens=4096, start=0, heads=64, kv_heads=8,
             max_len=4096),
        dict(name="prompt_chunk", kind="prompt", tokens=509, start=16003, heads=64, kv_heads=8,
             max_len=32768),
        dict(name="prompt_few", kind="prompt", tokens=5, start=20010, heads=32, kv_heads=8,
             max_len=32768),
        # the next token of one sequence with the usual settings; of a batch of
        # sequences from fp32 logits, some rows with most tokens masked; and of
        # many without any filter
        dict(name="draw_one", kind="draw", rows=1, vocab=VOCAB, dtype="bfloat16", temperature=0.7,
             top_k=20, top_p=0.8, min_p=0.0),
        dict(name="draw_batch", kind="draw", rows=64, vocab=VOCAB, dtype="float32",
             temperature=1.0, top_k=0, top_p=0.95, min_p=0.02),
        dict(name="draw_plain", kind="draw", rows=250, vocab=32003, dtype="bfloat16",
             temperature=1.3, top_k=0, top_p=1.0, min_p=0.0),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("rows", "store", "token", "token", "prompt", "prompt", "draw", "draw"))
    nh, nkv = rng.choice(HEADS)
    if kind in ("rows", "store"):
        tokens = _spread(rng, 1, 4096)
        start = rng.randint(0, 1000)
        return dict(kind=kind, tokens=tokens, start=start, heads=nh, kv_heads=nkv,
                    max_len=start + tokens + rng.randint(0, 100))
    if kind == "token":
        pos = _spread(rng, 1, 100000) - 1
        return dict(kind=kind, pos=pos, heads=nh, kv_heads=nkv,
                    max_len=pos + 1 + rng.randint(0, 1000))
    if kind == "prompt":
        tokens = _spread(rng, 1, 2048)
        # as many pairs of tokens and rows as the longest listed prompt at most
        start = rng.choice((0, _spread(rng, 1, min(16000, 2 ** 23 // tokens - tokens))))
        return dict(kind=kind, tokens=tokens, start=start, heads=nh, kv_heads=nkv,
                    max_len=start + tokens + rng.randint(0, 300))
    vocab = rng.choice((VOCAB, _spread(rng, 7, VOCAB)))
    return dict(kind=kind, rows=_spread(rng, 1, max(1, min(64, 2 ** 23 // vocab))), vocab=vocab,
                dtype=rng.choice(("bfloat16", "bfloat16", "float32", "float16")),
                temperature=round(rng.uniform(0.3, 1.6), 2),
                top_k=rng.choice((0, 1, _spread(rng, 2, 2000))),
                top_p=rng.choice((1.0, round(rng.uniform(0.05, 0.999), 3))),
                min_p=rng.choice((0.0, round(rng.uniform(0.001, 0.3), 3))))


def work(case):
    c = SimpleNamespace(**case)
    if c.kind == "draw":
        size = 4 if c.dtype == "float32" else 2
        return {"bytes": c.rows * (c.vocab * size + 4 + 12), "flops": 4 * c.rows * c.vocab}
    row = c.kv_heads * 2 * (HD // 2 + HD // GROUP * 2)  # bytes of a cache row, all kv heads
    if c.kind == "store":
        n = c.tokens * c.kv_heads * HD
        return {"bytes": 4 * n + c.tokens * row + 4 * n, "flops": 10 * n}
    if c.kind == "rows":
        qkv = c.tokens * (c.heads + 2 * c.kv_heads) * HD
        # q|k|v in, the tables' rows, q out, the cache's rows and what they stand for
        return {"bytes": 2 * qkv + 4 * c.tokens * HD + 2 * c.tokens * c.heads * HD
                + c.tokens * row + 4 * c.tokens * c.kv_heads * HD, "flops": 12 * qkv}
    tokens, last = (1, c.pos) if c.kind == "token" else (c.tokens, c.start + c.tokens - 1)
    pairs = tokens * (last + 1) - tokens * (tokens - 1) // 2
    return {"bytes": (last + 1) * row + 4 * tokens * c.heads * HD,
            "flops": 4 * HD * c.heads * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _tables(max_len):
    """cos and sin of every position, bf16 [max_len, HD], angles in 64 bits."""
    inv = THETA ** (-torch.arange(0, HD, 2, device=DEV, dtype=torch.float64) / HD)
    angle = torch.arange(max_len, device=DEV, dtype=torch.float64)[:, None] * inv
    angle = torch.cat((angle, angle), -1)
    return angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)


def _keys_values(g, rows, nkv):
    """Keys as a normed and rotated head gives them (channels of unlike sizes)
    and values, bf16 [rows, nkv, HD]."""
    channel = torch.exp(0.4 * _randn(g, nkv, HD))
    k = _randn(g, rows, nkv, HD) * channel
    v = _randn(g, rows, nkv, HD) * 0.5
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def _logits(g, rows, vocab, dtype):
    """A broad floor of unlikely tokens and some likely ones; in every eighth
    row all but some 200 tokens masked."""
    x = 2.0 * _randn(g, rows, vocab)
    x += 9.0 * torch.rand(rows, vocab, device=DEV, generator=g).pow(40)
    keep = torch.rand(rows, vocab, device=DEV, generator=g) < 200.0 / vocab
    masked = (torch.arange(rows, device=DEV) % 8 == 3)[:, None] & ~keep
    return x.masked_fill(masked, float("-inf")).to(getattr(torch, dtype))


def prepare(case, seed):
    s = SimpleNamespace(**case)
    g = _gen(seed)
    if s.kind == "draw":
        s.logits = _logits(g, s.rows, s.vocab, s.dtype)
        s.u = torch.rand(s.rows, device=DEV, generator=g)
        if own:
            s.K = _framework()
        return s
    if own:
        s.K = _framework()
        s.cache = s.K.kv4_cache(s.kv_heads, s.max_len, DEV)
    if s.kind == "store":
        k, v = _keys_values(g, s.tokens, s.kv_heads)
        # [heads, tokens, HD], as a model's own cache holds them
        s.k, s.v = k.transpose(0, 1).contiguous(), v.transpose(0, 1).contiguous()
        return s
    if s.kind == "rows":
        s.qkv = _randn(g, s.tokens, (s.heads + 2 * s.kv_heads) * HD).to(torch.bfloat16)
        s.q_w = (1 + 0.2 * _randn(g, HD)).to(torch.bfloat16)
        s.k_w = (1 + 0.2 * _randn(g, HD)).to(torch.bfloat16)
        s.cos, s.sin = _tables(s.max_len)
        s.q = torch.empty(s.tokens, s.heads * HD, device=DEV, dtype=torch.bfloat16)
        s.pos = torch.tensor([s.start], device=DEV)
        return s
    s.tokens = 1 if s.kind == "token" else s.tokens
    s.start = s.pos if s.kind == "token" else s.start
    rows = s.start + s.tokens
    k, v = _keys_values(g, rows, s.kv_heads)
    # heads that look at a few rows and heads that look at many
    sharp = torch.linspace(0.5, 3.0, s.heads, device=DEV)[:, None]
    s.q = (_randn(g, s.tokens, s.heads, HD) * sharp).to(torch.bfloat16).view(s.tokens, -1)
    s.scale = 1 / math.sqrt(HD)
    s.at = torch.tensor([s.start], device=DEV)
    if own:
        s.K.kv4_write(k, v, s.cache)
    else:
        s.kq, s.ks = _quantised(k)
        s.vq, s.vs = _quantised(v)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    if s.kind == "rows":
        return _plain_rows(s)
    if s.kind == "store":
        return [_plain_values(*_quantised(x.transpose(0, 1))) for x in (s.k, s.v)]
    if s.kind == "draw":
        return _plain_draw(s)
    return _plain_attention(s)


def _run_own(s):
    K = s.K
    if s.kind == "rows":
        if s.tokens == 1:
            K.qk_norm_rope_kv4(s.qkv.view(-1), s.q_w, s.k_w, s.cos, s.sin, s.pos, s.q.view(-1),
                               s.cache, s.heads, s.kv_heads, EPS)
        else:
            K.qk_norm_rope_kv4_rows(s.qkv, s.q_w, s.k_w, s.cos, s.sin, s.q, s.cache, s.heads,
                                    s.kv_heads, EPS, start=s.start)
        k, v = K.kv4_read(s.cache, s.start, s.tokens)
        return s.q, k, v
    if s.kind == "store":
        K.kv4_write(s.k.transpose(0, 1), s.v.transpose(0, 1), s.cache, start=s.start)
        return K.kv4_read(s.cache, s.start, s.tokens)
    if s.kind == "token":
        return K.kv4_decode_attention(s.q.view(-1), s.cache, s.at, None, s.scale).view(1, -1)
    if s.kind == "prompt":
        return K.kv4_prompt_attention(s.q, s.cache, s.start, None, s.scale)
    return K.sample(s.logits, s.u, temperature=s.temperature, top_k=s.top_k, top_p=s.top_p,
                    min_p=s.min_p)


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _quantised(x):
    """bf16 [..., HD] -> whole numbers int8 [..., HD // GROUP, GROUP] and scales."""
    x = x.float().unflatten(-1, (HD // GROUP, GROUP))
    a = x.abs().amax(-1, keepdim=True)
    s = ((a / 7).view(torch.int32) & -0x80000).view(torch.float32)
    s = torch.where(s < 2.0 ** -100, torch.zeros_like(s), s)
    q = torch.where(s > 0, x / s, torch.zeros_like(x)).round().clamp(-7, 7)
    return q.to(torch.int8), s.to(torch.bfloat16)


def _plain_values(q, s):
    return (q.float() * s.float()).flatten(-2).to(torch.bfloat16)


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


def _plain_rows(s):
    x = s.qkv.view(s.tokens, -1, HD)
    cos, sin = (t[s.start:s.start + s.tokens, None] for t in (s.cos, s.sin))
    q = _plain_rope(x[:, :s.heads], s.q_w, cos, sin)
    k = _plain_rope(x[:, s.heads:s.heads + s.kv_heads], s.k_w, cos, sin)
    v = x[:, s.heads + s.kv_heads:]
    return (q.reshape(s.tokens, -1), _plain_values(*_quantised(k)), _plain_values(*_quantised(v)))


def _plain_attention(s):
    """[tokens, heads * HD]: token t attends rows 0 .. start + t."""
    group, rows = s.heads // s.kv_heads, s.start + s.tokens
    k = (s.kq.float() * s.ks.float()).flatten(-2).permute(1, 2, 0).contiguous()  # [nkv, HD, rows]
    v = (s.vq.float() * s.vs.float()).flatten(-2).transpose(0, 1).contiguous()   # [nkv, rows, HD]
    q = s.q.view(s.tokens, s.kv_heads, group, HD).permute(1, 0, 2, 3).reshape(s.kv_heads, -1, HD)
    x = torch.matmul(q.float(), k) * s.scale                        # [nkv, tokens * group, rows]
    limit = s.start + torch.arange(s.tokens, device=DEV).repeat_interleave(group)
    x = x.masked_fill(torch.arange(rows, device=DEV) > limit[:, None], float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(x, v) / x.sum(-1, keepdim=True)
    o = o.view(s.kv_heads, s.tokens, group, HD).permute(1, 0, 2, 3)
    return o.reshape(s.tokens, -1).to(torch.bfloat16)


def _plain_draw(s):
    """(token int64 [rows], its probability fp32 [rows])."""
    x, order = torch.sort(s.logits.double(), dim=-1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / s.temperature)
    if s.top_k:
        w[:, s.top_k:] = 0
    if s.top_p < 1:
        before = w.cumsum(-1) - w
        w = w * (before < s.top_p * w.sum(-1, keepdim=True))
    w = w * (w >= s.min_p)
    w = torch.zeros_like(w).scatter_(-1, order, w)
    run = w.cumsum(-1)
    at = (run <= s.u.double()[:, None] * run[:, -1:]).sum(-1, keepdim=True)
    at = at.clamp(max=s.vocab - 1)
    return at[:, 0], (w.gather(-1, at) / run[:, -1:])[:, 0].float()


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


def _values_64(x):
    """What the cache stands for, of bf16 numbers x in 64 bits."""
    out = torch.empty_like(x)
    for at in range(0, HD, GROUP):
        g = x[..., at:at + GROUP]
        m, e = torch.frexp(g.abs().max(-1, keepdim=True).values / 7)
        s = torch.floor(m * 32) * _power(e - 5)
        n = torch.round(g / torch.where(s == 0, 1, s))
        out[..., at:at + GROUP] = n.clamp(-7, 7) * s
    return out


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"rows": _exact_rows, "store": _exact_store, "token": _exact_attention,
            "prompt": _exact_attention, "draw": _exact_draw}[s.kind](s)


def _exact_store(s):
    return [_values_64(x.double().transpose(0, 1)) for x in (s.k, s.v)]


def _exact_rows(s):
    got = []
    for first, n, w in ((0, s.heads, s.q_w), (s.heads, s.kv_heads, s.k_w)):
        x = s.qkv.double().view(s.tokens, -1, HD)[:, first:first + n]
        root = torch.sqrt((x * x).sum(-1, keepdim=True) / HD + EPS)
        y = _bf16_64(w.double() * _bf16_64(x / root))
        lo, hi = y.split(HD // 2, -1)
        c, t = (z[s.start:s.start + s.tokens, None, :HD // 2].double() for z in (s.cos, s.sin))
        got.append(torch.cat((_bf16_64(_bf16_64(lo * c) + _bf16_64(-hi * t)),
                              _bf16_64(_bf16_64(hi * c) + _bf16_64(lo * t))), -1))
    v = s.qkv.double().view(s.tokens, -1, HD)[:, s.heads + s.kv_heads:]
    return got[0].reshape(s.tokens, -1), _values_64(got[1]), _values_64(v)


def _exact_attention(s):
    group, rows = s.heads // s.kv_heads, s.start + s.tokens
    out = torch.empty(s.tokens, s.heads, HD, dtype=torch.float64, device=DEV)
    later = torch.arange(rows, device=DEV) > s.start + torch.arange(s.tokens, device=DEV)[:, None]
    for h in range(s.heads):
        kv = h // group
        k, v = ((q[:, kv].double() * z[:, kv].double()).reshape(rows, HD)
                for q, z in ((s.kq, s.ks), (s.vq, s.vs)))
        x = s.q.view(s.tokens, s.heads, HD)[:, h].double() @ k.T.contiguous() * s.scale
        out[:, h] = torch.softmax(x.masked_fill(later, -math.inf), -1) @ v
    return out.view(s.tokens, -1)


def _exact_draw(s):
    logits, u = s.logits.double().cpu().numpy(), s.u.double().cpu().numpy()
    token, prob = np.empty(s.rows, np.int64), np.empty(s.rows, np.float64)
    for r in range(s.rows):
        order = np.lexsort((np.arange(s.vocab), -logits[r]))
        n = min(s.top_k or s.vocab, s.vocab)
        w = np.exp((logits[r][order[:n]] - logits[r].max()) / s.temperature)
        if s.top_p < 1:
            w = w[:1 + int(np.searchsorted(np.cumsum(w), s.top_p * w.sum()))]
        w = w[w >= s.min_p]
        kept = order[:len(w)]
        by_index = np.argsort(kept)
        run = np.cumsum(w[by_index])
        at = min(int(np.searchsorted(run, u[r] * run[-1], side="right")), len(w) - 1)
        token[r], prob[r] = kept[by_index[at]], w[by_index[at]] / run[-1]
    return token, prob
