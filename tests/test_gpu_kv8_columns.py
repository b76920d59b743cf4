"""GPU: the attention over the 8-bit cache of 17 to some hundred columns ((token, query
head) pairs of a kv head), on both sides of every number of waves and of tiles, of one
sequence and of several, short and in splits; and a prompt's on both sides of its
routes."""
import pytest
import torch

from test_gpu_kv8 import SCALE, _check, _filled, _gen, _pos

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths", [[330], [1500], [1400, 40, 900]])
@pytest.mark.parametrize("tokens,group", [(17, 1), (4, 8), (33, 1), (6, 8), (49, 1), (8, 8), (65, 1),
                                          (10, 8), (16, 8), (129, 1), (13, 10), (24, 8), (40, 5)])
def test_columns(tokens, group, lengths):
    import _dip_hip as K
    print(f"kv8 columns tokens={tokens} group={group} lengths={lengths}", flush=True)
    g = _gen(tokens + group)
    lengths = [max(n, tokens) for n in lengths]
    cache, table, values = _filled(g, lengths, 2)
    nh = 2 * group
    q = torch.randn(len(lengths), tokens, nh * 128, device="cuda", generator=g).to(torch.bfloat16)
    out = K.kv8_decode_attention(q, cache, table, _pos(*[n - tokens for n in lengths]), None, SCALE)
    _check(out, q, values, lengths, tokens, nh)


# columns of 256 and 257, 512 and 513, 1024 and 1025
@pytest.mark.parametrize("start", [0, 1100])
@pytest.mark.parametrize("tokens,nh,nkv", [(32, 64, 8), (257, 2, 2), (64, 16, 2), (65, 64, 8),
                                           (513, 1, 1), (128, 8, 1), (1025, 1, 1), (200, 16, 16)])
def test_prompts_on_both_sides_of_a_route(tokens, nh, nkv, start):
    import _dip_hip as K
    print(f"kv8 prompt tokens={tokens} start={start} heads={nh}/{nkv}", flush=True)
    g = _gen(tokens)
    n = start + tokens
    cache, table, values = _filled(g, [n], nkv)
    q = torch.randn(1, tokens, nh * 128, device="cuda", generator=g).to(torch.bfloat16)
    out = K.kv8_prompt_attention(q[0], cache, table[0], start, None, SCALE)
    _check(out[None], q, values, [n], tokens, nh)
