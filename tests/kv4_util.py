"""The 4-bit key/value cache and the drawing of tokens from their definitions, in
64 bits, for the tests."""
import numpy as np
import torch

HD, GROUP = 128, 32


def quantised(x: torch.Tensor) -> torch.Tensor:
    """What the cache stands for, of bf16 x [..., 128]: float64 on the CPU."""
    x = x.detach().cpu().double().numpy().reshape(*x.shape[:-1], HD // GROUP, GROUP)
    with np.errstate(invalid="ignore", divide="ignore"):
        a = np.abs(x).max(-1, keepdims=True)
        m, e = np.frexp(a / 7)
        s = np.ldexp(np.floor(m * 32), e - 5)  # a 5-bit significand
        s = np.where(s < 2.0 ** -100, 0.0, s)
        q = np.where(s > 0, np.clip(np.rint(x / np.where(s > 0, s, 1.0)), -7, 7), 0.0)
        v = np.where(np.isfinite(a), q * np.where(np.isfinite(a), s, 1.0), np.nan)
    return torch.from_numpy(v.reshape(*v.shape[:-2], HD))


def scale_of(x: torch.Tensor) -> torch.Tensor:
    """Each value's group scale, an upper bound of it (a / 7)."""
    g = x.detach().cpu().double().unflatten(-1, (HD // GROUP, GROUP))
    return (g.abs().amax(-1, keepdim=True) / 7).expand(g.shape).flatten(-2)


def attention(q, k, v, limits, scale):
    """q [tokens, nh, 128], k and v float64 [rows, nkv, 128] as the cache stands for
    them; token t attends rows 0 .. limits[t] - 1 (none: zeros).  Returns (out,
    sum of weight * |v|), float64 [tokens, nh, 128]."""
    tokens, nh = q.shape[:2]
    nkv = k.shape[1]
    out = torch.zeros(tokens, nh, HD, dtype=torch.float64)
    size = torch.zeros_like(out)
    qd = q.detach().cpu().double()
    for t in range(tokens):
        n = int(limits[t])
        if n <= 0:
            continue
        for h in range(nh):
            kv = h // (nh // nkv)
            w = torch.softmax(k[:n, kv] @ qd[t, h] * scale, 0)
            out[t, h] = w @ v[:n, kv]
            size[t, h] = w @ v[:n, kv].abs()
    return out, size


def attention_bound(out, size, scale_max):
    """How far the kernels may be: the result's rounding to bf16 (2^-8 of it), the
    weights' (2^-8 of what they weigh), and the fp32 sums.  Those run over at most
    some hundred steps of 32 rows, of terms up to 24 times weight * scale (the
    constant 1.5 * 16 that the number's bits carry): 300 * 2^-24 * 24 < 2^-11 of
    the scale; and the scores' own sums move a weight by less than 2^-10."""
    return 2.0 ** -8 * out.abs() + (2.0 ** -8 + 2.0 ** -10) * size + 2.0 ** -11 * scale_max


def drawn(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probability, weights of the kept tokens by index) of one row, float64
    numpy."""
    x = np.asarray(logits, np.float64)
    x = np.where(np.isnan(x), -np.inf, x) + 0.0
    n = len(x)
    top = x.max()
    if top == -np.inf:
        return 0, 0.0, np.zeros(n)
    order = np.lexsort((np.arange(n), -x))
    if temperature == 0:
        w = np.zeros(n)
        w[order[0]] = 1.0
        return int(order[0]), 1.0, w
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / temperature))[order]
    if 0 < top_k < n:
        w[top_k:] = 0
    if top_p < 1:
        run = np.cumsum(w)
        w[1 + int(np.searchsorted(run, top_p * run[-1])):] = 0
    w[w < min_p] = 0
    by_index = np.zeros(n)
    by_index[order] = w
    run = np.cumsum(by_index)
    above = np.nonzero((run > u * run[-1]) & (by_index > 0))[0]
    at = int(above[0]) if len(above) else int(np.nonzero(by_index)[0][-1])
    return at, by_index[at] / run[-1], by_index
