"""GPU: prompts of one and of few tokens in front of drafted ones.  A module takes a
single token for a step's and prunes it, but with drafts every token is the dense
model's, the one behind such a prompt too."""
import pytest
import torch

from model_util import max_rel
from test_gpu_kv8_decoder import BOUND, E4M3, _caches, _model, _Reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pruned(tmp_path_factory):
    return _model(tmp_path_factory, 512, 1024, 4, 2, 0.3)


def _prompt(n):
    return torch.randint(0, 768, (1, n), generator=torch.Generator().manual_seed(n + 20))


def _keep(model, ratio):
    for L in model.model.layers:
        L.mlp.keep_ratio = ratio


@pytest.mark.parametrize("how", [dict(), dict(do_sample=True, temperature=0.9, top_k=40)])
@pytest.mark.parametrize("cache", [0, 1])
@pytest.mark.parametrize("plen", [1, 2])
def test_the_first_logits_do_not_depend_on_the_pruning(pruned, plen, cache, how):
    from dip_model import DIPDecoder
    out = []
    for ratio in (0.3, 1.0):
        _keep(pruned, ratio)
        try:
            gen = {"generator": torch.Generator(device="cuda").manual_seed(2)} if how else {}
            dec = DIPDecoder(pruned, 64, **_caches()[cache])
            out.append(dec.generate(_prompt(plen), 5, return_logits=True, draft=2, **gen, **how))
        finally:
            _keep(pruned, 0.3)
    (a, la), (b, lb) = out
    print(f"  plen {plen} cache {cache}: max_rel {max_rel(la[0], lb[0]):.3e}", flush=True)
    assert torch.equal(la[0], lb[0]) and torch.equal(a[:, :plen + 1], b[:, :plen + 1])


def test_tokens_behind_one_follow_the_definition(pruned):
    from dip_model import DIPDecoder
    prompt, new = _prompt(1), 9
    dec = DIPDecoder(pruned, 64, kv_dtype=E4M3)
    seq, logits = dec.generate(prompt, new, return_logits=True, draft=3)
    assert seq[0, 1:].tolist() == logits.argmax(-1).tolist()
    ref = _Reference(pruned)
    _keep(pruned, 1.0)  # the reference's single token
    try:
        want = torch.cat((ref.part(prompt)[-1:], ref.part(seq[:, 1:])[:-1]))
    finally:
        _keep(pruned, 0.3)
    for t in range(new):
        err = max_rel(logits[t], want[t])
        print(f"  token {t} max_rel {err:.3e}", flush=True)
        assert err < BOUND


def test_without_drafts_one_token_is_a_steps(pruned):
    """As before: a prompt of one token runs as the next token does."""
    from dip_model import DIPDecoder
    a, la = DIPDecoder(pruned, 64, kv_dtype=E4M3).generate(_prompt(1), 2, return_logits=True)
    _keep(pruned, 1.0)
    try:
        _, lb = DIPDecoder(pruned, 64, kv_dtype=E4M3).generate(_prompt(1), 2, return_logits=True)
    finally:
        _keep(pruned, 0.3)
    assert not torch.equal(la[0], lb[0])


def test_an_empty_prompt_is_refused(pruned):
    from dip_model import DIPDecoder
    dec = DIPDecoder(pruned, 64, kv_dtype=E4M3)
    for draft in (0, 2):
        with pytest.raises(ValueError):
            dec.generate(torch.zeros(1, 0, dtype=torch.long), 2, draft=draft)


def test_a_prompt_longer_than_the_cache_is_refused(pruned):
    """Whatever the number of new tokens, one that is negative among them."""
    from dip_model import DIPDecoder
    dec = DIPDecoder(pruned, 64, kv_dtype=E4M3)
    for new in (2, 0, -10):
        with pytest.raises(ValueError):
            dec.generate(_prompt(70), new, draft=2)
