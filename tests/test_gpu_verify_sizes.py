"""GPU: verification and sampling at sizes whose work is cut otherwise: vocabularies of
millions, thousands of rows, and many long rows; and rows that do not depend on what
they are in a call with."""
import pytest
import torch

from test_gpu_verify import FILTERS, _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", [dict(), dict(top_k=20, top_p=0.9), dict(min_p=0.2),
                                 dict(temperature=0.0), dict(top_k=500, temperature=0.5)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_vocabularies_of_millions(dtype, how):
    print(f"verify, 2.1 million {dtype}, {how}", flush=True)
    x, d, u, y = _inputs(1, 1, 2_100_003, dtype, 3)
    u[:, 0] = 0.01
    _check(x, d, u, **how)
    _check(x, d, u, y, **how)


@pytest.mark.parametrize("how", FILTERS)
def test_thousands_of_rows_are_as_by_themselves(how):
    import _dip_hip as K
    print(f"verify, 700 sequences, {how}", flush=True)
    x, d, u, y = _inputs(700, 3, 5003, torch.bfloat16, 4)
    for draft in (None, y):
        tokens, accepted = K.verify(x, d, u, draft, **how)
        for s in (0, 1, 350, 699):
            one = slice(s, s + 1)
            t, a = K.verify(x[one], d[one], u[one], None if draft is None else draft[one], **how)
            assert torch.equal(t[0], tokens[s]) and torch.equal(a[0], accepted[s]), s


@pytest.mark.parametrize("how", FILTERS)
def test_many_long_rows_are_as_by_themselves(how):
    import _dip_hip as K
    print(f"200 rows of 151936, {how}", flush=True)
    x, d, u, y = _inputs(40, 2, 151936, torch.float32, 5)
    for draft in (None, y):
        tokens, accepted = K.verify(x, d, u, draft, **how)
        for s in (0, 17, 39):
            one = slice(s, s + 1)
            t, a = K.verify(x[one], d[one], u[one], None if draft is None else draft[one], **how)
            assert torch.equal(t[0], tokens[s]) and torch.equal(a[0], accepted[s]), s
    rows = torch.cat((x.flatten(0, 1), y.flatten(0, 1)))
    v = torch.rand(200, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))
    token, prob = K.sample(rows, v, **how)
    for r in (0, 63, 199):
        t, p = K.sample(rows[r:r + 1], v[r:r + 1], **how)
        assert torch.equal(t[0], token[r]) and torch.equal(p[0], prob[r]), r
