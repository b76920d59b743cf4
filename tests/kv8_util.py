"""The paged 8-bit key/value cache from its definition, in 64 bits, for the tests."""
import numpy as np
import torch

HD, PAGE, GROUP = 128, 64, 32


def e4m3(x):
    """The nearest e4m3 numbers, ties to even (|x| up to 448)."""
    _, e = np.frexp(x)
    step = np.ldexp(1.0, np.maximum(e, -5) - 4)
    return np.rint(x / step) * step


def scale_of(x):
    """The scale of rows x [rows, HD]: from the groups that are finite."""
    g = np.abs(x.reshape(-1, GROUP))
    g = g[np.isfinite(g).all(-1)]
    a = g.max() if g.size else 0.0
    return 0.0 if a == 0 else max(2.0 ** (np.frexp(a)[1] - 8), 2.0 ** -100)


def numbers(x, s):
    """Rows x [rows, HD] in numbers of scale s; NaN in the groups that are not finite."""
    bad = ~np.isfinite(x.reshape(-1, GROUP)).all(-1)
    cap = 240.0 if s == 2.0 ** 120 else 256.0
    with np.errstate(invalid="ignore"):
        n = e4m3(np.clip(np.where(np.isfinite(x), x, 0.0) / (s or 1.0), -cap, cap))
    n.reshape(-1, GROUP)[bad] = np.nan
    return n


class Pages:
    """What a KV8Cache holds: numbers float64 [2 (keys, values), pages, heads, 64, 128]
    and scales [2, pages, heads]."""

    def __init__(self, pages, nkv):
        self.n = np.zeros((2, pages, nkv, PAGE, HD))
        self.s = np.zeros((2, pages, nkv))

    def write(self, k, v, table, pos):
        """As kv8_write: k and v [seqs, tokens, nkv, HD] tensors, table a list of lists."""
        for kind, x in enumerate((k, v)):
            x = x.detach().double().cpu().numpy()
            for i, first in enumerate(pos):
                if first < 0:
                    continue
                for page in range(first // PAGE, (first + x.shape[1] - 1) // PAGE + 1):
                    if page >= len(table[i]) or not 0 <= table[i][page] < self.n.shape[1]:
                        continue
                    lo = max(first, page * PAGE)
                    hi = min(first + x.shape[1], (page + 1) * PAGE)
                    for h in range(x.shape[2]):
                        self._rows(kind, table[i][page], h, lo % PAGE, x[i, lo - first:hi - first, h])

    def _rows(self, kind, page, h, r, x):
        was = self.s[kind, page, h] if r else 0.0
        s = max(was, scale_of(x))
        n = self.n[kind, page, h]
        if s > was and r:
            n[:r] = e4m3(n[:r] * (was / s))
        n[r:r + len(x)] = numbers(x, s)
        n[r + len(x):] = 0  # stand for nothing
        self.s[kind, page, h] = s

    def read(self, table, pos, tokens):
        """(k, v) float64 [tokens, nkv, HD] of one sequence's rows."""
        out = np.zeros((2, tokens, self.n.shape[2], HD))
        for t in range(tokens):
            p = pos + t
            if pos >= 0 and p // PAGE < len(table) and 0 <= table[p // PAGE] < self.n.shape[1]:
                page = table[p // PAGE]
                out[:, t] = self.n[:, page, :, p % PAGE] * self.s[:, page, :, None]
        return torch.from_numpy(out[0]), torch.from_numpy(out[1])


def attention_bound(out, size):
    """How far the kernels may be: the result's rounding to bf16 (2^-8 of it), the
    weights' (2^-8 of what they weigh), and what the fp32 sums and the scores' own sums
    move a weight by: 128 products and their sum, 2^-17 of the magnitudes' sum, which is
    below 2^6 in scores here: 2^-11; sums over up to some hundred steps of 64 rows,
    2^-24 each: below 2^-11 of the size."""
    return 2.0 ** -8 * out.abs() + (2.0 ** -8 + 2.0 ** -10) * size
