"""GPU: drafts whose number lies near their probability, with and without filters and
however many rows a call has.  A row's sum without filters is off by 2^-24 of itself at
most; the numbers here lie 2^-22 of the probability off it, and a step of fp32."""
import numpy as np
import pytest
import torch

from test_gpu_verify import _shares

pytestmark = pytest.mark.gpu


def _near(p, sign):
    """The nearest fp32 numbers that lie 2^-22 of p or more off it, to one side."""
    want = p * (1 + sign * 2.0 ** -22)
    u = want.astype(np.float32)
    over = (u.astype(np.float64) - want) * sign < 0
    return np.where(over, np.nextafter(u, np.float32(sign * np.inf)), u)


@pytest.mark.parametrize("how", [dict(), dict(temperature=1.3), dict(top_k=20),
                                 dict(top_p=0.95, min_p=0.01)])
@pytest.mark.parametrize("vocab,dtype", [(32003, torch.bfloat16), (151936, torch.float32),
                                         (500009, torch.bfloat16)])
def test_the_border_is_the_probability(vocab, dtype, how):
    import _dip_hip as K
    print(f"{vocab} {dtype} {how}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    # a likely token here and there above thousands of unlikely ones
    x = 2.0 * torch.randn(3, vocab, device="cuda", generator=g)
    x += 9.0 * torch.rand(3, vocab, device="cuda", generator=g).pow(60)
    x = x.to(dtype)
    drafted = x.float().topk(3, dim=1).indices[:, 1:2].contiguous()
    p = np.array([_shares(r.double().cpu().numpy(), how)[int(t)] for r, t in zip(x, drafted)])
    assert (p > 1e-4).all() and (p < 0.9).all()
    logits = torch.stack((x, x.flip(1)), 1)  # the draft's row, and one behind it
    for sign in (-1, 1):
        u = torch.full((3, 2), 0.5, device="cuda")
        u[:, 0] = torch.from_numpy(_near(p, sign)).cuda()
        for times in (1, 40, 150):
            if times * 6 * vocab * x.element_size() > 1 << 29:
                continue
            _, accepted = K.verify(*(t.repeat(times, *[1] * (t.dim() - 1))
                                     for t in (logits, drafted, u)), **how)
            assert accepted.tolist() == [int(sign < 0)] * 3 * times, (sign, times)
