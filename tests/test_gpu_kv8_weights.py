"""GPU: the weights of the attention of up to 16 columns over the 8-bit cache are those of
32 bits.  Next to the result's rounding to bf16, 2^-8 of it at most, the kernels may be off
by what their scores are: 128 products of below 2^5 in all, in powers of 2, summed in fp32,
2^7 * 2^-24 * 2^5 = 2^-12 of an exponent and so of a weight, and as much of the weights'
sum; the weights' own parts (2^-17) and the base's roundings (2^-18) are little beside:
2^-11 of the weighed values' size in all.  Weights rounded to bf16 are off by 2^-8 each."""
import pytest
import torch

from kv4_util import attention
from kv8_util import PAGE
from test_gpu_kv8 import SCALE, _filled, _gen, _pos

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths,tokens,nh,nkv", [
    ([2], 1, 32, 2), ([3, 5, 2, 4], 1, 16, 1), ([64], 2, 16, 2), ([65, 7], 3, 20, 4),
    ([700], 1, 40, 8), ([2000, 3], 1, 8, 1), ([4000], 4, 8, 2), ([6], 16, 8, 8)])
def test_weights_are_not_rounded_to_bf16(lengths, tokens, nh, nkv):
    import _dip_hip as K
    print(f"weights tokens={tokens} lengths={lengths} heads={nh}/{nkv}", flush=True)
    g = _gen(sum(lengths) + nh)
    tokens = min(tokens, min(lengths))
    cache, table, values = _filled(g, lengths, nkv)
    q = torch.randn(len(lengths), tokens, nh * 128, device="cuda", generator=g).to(torch.bfloat16)
    out = K.kv8_decode_attention(q, cache, table, _pos(*[n - tokens for n in lengths]), None, SCALE)
    for i, (k, v) in enumerate(values):
        limits = [lengths[i] - tokens + 1 + t for t in range(tokens)]
        want, size = attention(q[i].view(tokens, nh, 128), k, v, limits, SCALE)
        err = (out[i].view(tokens, nh, 128).double().cpu() - want).abs()
        bound = 2.0 ** -8 * want.abs() + 2.0 ** -11 * size
        assert bool((err <= bound).all()), (i, (err / bound.clamp(min=1e-30)).max())


@pytest.mark.parametrize("rows", [1, 2, 3, 65, 700, 5000])
def test_weights_add_up_to_one(rows):
    """Values that are all the same come out as they are."""
    import _dip_hip as K
    g = _gen(rows)
    k = torch.randn(1, rows, 2, 128, device="cuda", generator=g).to(torch.bfloat16)
    v = torch.full_like(k, 0.75)
    width = -(-rows // PAGE)
    cache = K.kv8_cache(2, width)
    table = torch.arange(width, dtype=torch.int32, device="cuda")[None]
    K.kv8_write(k, v, cache, table, _pos(0))
    q = torch.randn(1, 1, 16 * 128, device="cuda", generator=g).to(torch.bfloat16)
    out = K.kv8_decode_attention(q, cache, table, _pos(rows - 1), None, SCALE)
    assert bool((out == 0.75).all()), out[out != 0.75]
