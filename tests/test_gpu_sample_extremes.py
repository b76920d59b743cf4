"""GPU: temperatures and logits at the ends of their ranges."""
import math

import pytest
import torch

from kv4_util import drawn

pytestmark = pytest.mark.gpu

LOWEST = torch.finfo(torch.float32).min


@pytest.mark.parametrize("how", [dict(), dict(top_p=0.6), dict(top_k=7, min_p=0.5),
                                 dict(top_k=300, top_p=0.5)])
@pytest.mark.parametrize("temperature", [1e-300, 1e-35, 1e-12, 1e-8, 1e3, 1e29, 1e35, 1e300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [777, 40009])
def test_temperatures(vocab, dtype, temperature, how):
    """Where every distance is many times the temperature or next to nothing of it."""
    import _dip_hip as K
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = (2.5 * torch.randn(4, vocab, device="cuda", generator=g)).to(dtype)
    x[1, ::3] = -math.inf
    x[2, 1::2] = math.nan
    x[3, 5:90] = 40.0  # equals at the top
    u = torch.tensor([0.1, 0.9999, 0.37, 0.62], device="cuda")
    print(f"sample {vocab} {dtype} temperature {temperature} {how}", flush=True)
    token, prob = K.sample(x, u, temperature=temperature, **how)
    # up to 40 apart, a weight at 1e30 is off from one at any higher by 4e-29
    taken = min(max(temperature, 1e-30), 1e30)
    for r in range(4):
        t, p, w = drawn(x[r].double().cpu().numpy(), float(u[r]), temperature=taken, **how)
        assert w[int(token[r])] > 0
        assert abs(float(prob[r]) - p) <= 2.0 ** -21 * p
        if temperature < 1e3:  # weights far apart or equal: sums are not near u
            assert int(token[r]) == t, r


@pytest.mark.parametrize("vocab", [700, 40009])
@pytest.mark.parametrize("how", [dict(), dict(top_p=0.9), dict(top_k=5), dict(min_p=0.01)])
def test_masks_of_the_lowest_value(vocab, how):
    """Masked with the type's lowest value, next to very large logits and alone."""
    import _dip_hip as K
    x = torch.full((3, vocab), LOWEST, device="cuda")
    x[0, 3], x[0, 600] = 3e38, 3e38
    x[1, 5], x[1, 650] = -1.0, -1.5
    u = torch.tensor([0.6, 0.2, 0.999], device="cuda")
    token, prob = K.sample(x, u, **how)
    for r in range(3):
        t, p, _ = drawn(x[r].double().cpu().numpy(), float(u[r]), **how)
        assert int(token[r]) == t
        assert abs(float(prob[r]) - p) <= 2.0 ** -22 * p


@pytest.mark.parametrize("dtype,most,other,temperature", [
    (torch.bfloat16, 16.25, 1.1e-4, 1.0), (torch.bfloat16, 16.25, -1.1e-4, 0.9),
    (torch.bfloat16, 3e-6, -13.9, 0.8), (torch.bfloat16, 4096.0, 0.3, 300.0),
    (torch.bfloat16, 1e30, 7.0, 1e29), (torch.float16, 18.0, 3.3e-4, 1.0),
    (torch.float16, 30000.0, 0.77, 2000.0), (torch.float32, 17.000001, 1.2345678e-5, 1.0)])
@pytest.mark.parametrize("vocab", [2, 40009])
def test_logits_far_apart_in_magnitude(vocab, dtype, most, other, temperature):
    """The difference of two logits has more bits than fp32: a weight carries its
    rounding along.  A number beyond 1 draws the last token with a weight."""
    import _dip_hip as K
    x = torch.full((1, vocab), -math.inf, device="cuda")
    x[0, 0], x[0, vocab - 1] = most, other
    x = x.to(dtype)
    token, prob = K.sample(x, torch.tensor([7.0], device="cuda"), temperature=temperature)
    t, p, _ = drawn(x[0].double().cpu().numpy(), 7.0, temperature=temperature)
    assert int(token) == t == vocab - 1
    # the probability's rounding to fp32, the weight's 4e-10 and half a step of it
    shift = 62 - max(11, math.ceil(math.log2(vocab)))
    assert abs(float(prob) - p) <= (2.0 ** -24 + 1e-9 + 2.0 ** -1 / (p * 2.0 ** shift)) * p


@pytest.mark.parametrize("temperature", [1e3, 1e29, 1e35, 1e300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [777, 40009])
def test_draws_of_nearly_equal_weights(vocab, dtype, temperature):
    """At high temperatures the token drawn is the one at u of the running sum, to
    within a token at either end where the sum is next to u."""
    import _dip_hip as K
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = (2.5 * torch.randn(5, vocab, device="cuda", generator=g)).to(dtype)
    x[1, ::3] = -math.inf
    u = torch.tensor([0.1, 0.9999, 0.37, 0.0, 0.62], device="cuda")
    token, _ = K.sample(x, u, temperature=temperature)
    taken = min(temperature, 1e30)
    for r in range(5):
        _, _, w = drawn(x[r].double().cpu().numpy(), float(u[r]), temperature=taken)
        run, t, goal = w.cumsum(), int(token[r]), float(u[r]) * w.sum()
        # a sum of n weights in steps of 2^-44 at least, each off by 4e-10 of itself
        slack = vocab * (1e-9 + 2.0 ** -44)
        assert w[t] > 0 and run[t] - w[t] - slack <= goal <= run[t] + slack
