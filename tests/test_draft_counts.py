"""DIPDecoder.generate takes whole numbers of drafts alone (no GPU needed: refused before
anything runs)."""
import math

import pytest
import torch


@pytest.fixture(scope="module")
def dec():
    from dip_model import DIPDecoder
    d = object.__new__(DIPDecoder)
    d.kv_bits, d.device = 16, torch.device("cpu")

    def ran(*args, **kw):
        raise AssertionError("ran")
    d.prefill = d.step = d._prefill_fused = ran
    return d


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("draft", [0.5, 1.5, -0.5, -1, -3.0, math.nan, math.inf, -math.inf])
def test_no_whole_number(dec, draft, sampled):
    with pytest.raises(ValueError, match="whole number"):
        dec.generate(torch.zeros(1, 3, dtype=torch.long), 2, draft=draft, do_sample=sampled)


@pytest.mark.parametrize("draft", [1, 2.0, True])
def test_whole_numbers_go_on_to_the_next_check(dec, draft):
    with pytest.raises(ValueError, match="cache of 4 or 8 bits"):
        dec.generate(torch.zeros(1, 3, dtype=torch.long), 2, draft=draft)
