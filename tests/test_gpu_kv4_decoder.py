"""GPU: DIPDecoder with its keys and values in 4 bits, and with drawn tokens.  The
4-bit decoder is checked against the model's own modules with an attention in
64 bits over keys and values that are quantised by the definition."""
import math

import pytest
import torch

from kv4_util import quantised
from model_util import max_rel, tiny_config, tiny_model, write_checkpoint

pytestmark = pytest.mark.gpu

PLEN, NEW = 37, 9


@pytest.fixture(scope="module", params=[(512, 1024, 4, 1), (2560, 1280, 4, 2)])
def model(request, tmp_path_factory):
    from dip_stream_predispatch import load_streaming_dip
    hidden, inter, heads, kv = request.param
    cfg = tiny_config(hidden=hidden, inter=inter, heads=heads, kv_heads=kv, head_dim=128, vocab=768)
    d = tmp_path_factory.mktemp(f"kv4_{hidden}")
    write_checkpoint(tiny_model(cfg, seed=hidden), d)
    # keep 1: every channel, so that no rounding swaps a channel at the border
    return load_streaming_dip(d, keep_ratio=1.0)[0]


@pytest.fixture(scope="module")
def prompt(model):
    return torch.randint(0, model.config.vocab_size, (1, PLEN),
                         generator=torch.Generator().manual_seed(9))


class _Reference:
    """The model's modules part by part, the attention here."""

    def __init__(self, model):
        self.m, self.kv, self.n = model, [None] * len(model.model.layers), 0

    @torch.no_grad()
    def part(self, ids):
        m, n = self.m, ids.shape[1]
        inner, cfg = m.model, m.config
        nh, nkv = cfg.num_attention_heads, cfg.num_key_value_heads
        h = inner.embed_tokens(ids.cuda())
        ang = torch.arange(self.n, self.n + n).float()[:, None] * inner.rotary_emb.inv_freq.cpu()
        ang = torch.cat((ang, ang), -1)
        cos, sin = (f(ang).to(torch.bfloat16).cuda()[None, :, None] for f in (torch.cos, torch.sin))
        rot = lambda x: x * cos + torch.cat((-x[..., 64:], x[..., :64]), -1) * sin
        for i, L in enumerate(inner.layers):
            a = L.self_attn
            x = L.input_layernorm(h)
            q = rot(a.q_norm(a.q_proj(x).view(1, n, nh, 128)))[0]
            k = rot(a.k_norm(a.k_proj(x).view(1, n, nkv, 128)))[0]
            v = a.v_proj(x).view(n, nkv, 128)
            new = [quantised(k).cuda(), quantised(v).cuda()]
            old = self.kv[i]
            self.kv[i] = kk, vv = new if old is None else [torch.cat(p) for p in zip(old, new)]
            o = torch.empty(n, nh, 128, dtype=torch.float64, device="cuda")
            later = torch.arange(self.n + n, device="cuda") > self.n + torch.arange(
                n, device="cuda")[:, None]
            for j in range(nh):
                s = q[:, j].double() @ kk[:, j // (nh // nkv)].T.contiguous() * a.scaling
                o[:, j] = s.masked_fill(later, -math.inf).softmax(-1) @ vv[:, j // (nh // nkv)]
            h = h + a.o_proj(o.to(torch.bfloat16).view(1, n, -1))
            h = h + L.mlp(L.post_attention_layernorm(h))
        self.n += n
        return m.lm_head(inner.norm(h[:, -1:])).view(-1)


# bf16 roundings on either side move a key by a step of the cache now and then (a
# step is a / 7 of a group's largest): the module tests' bound for bf16 paths
BOUND = 4e-2


def test_logits_follow_the_definition(model, prompt):
    from dip_model import DIPDecoder
    dec = DIPDecoder(model, 128, kv_bits=4)
    assert dec.fused and not hasattr(dec, "k_cache")
    ref = _Reference(model)
    seq, logits = dec.generate(prompt, NEW, return_logits=True)
    for t in range(NEW):
        ids = prompt if t == 0 else seq[:, PLEN + t - 1:PLEN + t]
        err = max_rel(logits[t], ref.part(ids))
        print(f"  token {t} max_rel {err:.3e}", flush=True)
        assert err < BOUND


def test_graph_equals_eager_and_repeats(model, prompt):
    from dip_model import DIPDecoder
    dec = DIPDecoder(model, 64, kv_bits=4)
    a, la = dec.generate(prompt, NEW, return_logits=True)
    b, lb = dec.generate(prompt, NEW, return_logits=True)
    c, lc = DIPDecoder(model, 64, kv_bits=4, use_graph=False).generate(prompt, NEW,
                                                                       return_logits=True)
    assert torch.equal(a, b) and torch.equal(la, lb)
    assert torch.equal(a, c) and torch.equal(la, lc)


def test_a_prompt_in_parts(model, prompt, monkeypatch):
    """Parts of a prompt attend the rows of the parts before."""
    import dip_model
    whole = dip_model.DIPDecoder(model, 64, kv_bits=4)
    want = whole.prefill(prompt).float()
    monkeypatch.setattr(dip_model, "_PROMPT_CHUNK", 12)
    parts = dip_model.DIPDecoder(model, 64, kv_bits=4)
    got = parts.prefill(prompt).float()
    assert int(parts.pos) == PLEN and max_rel(got, want) < BOUND
    # the first layer's rows depend on the tokens alone
    K = parts._K
    for a, b in zip(K.kv4_read(parts._kv4[0], 0, 8), K.kv4_read(whole._kv4[0], 0, 8)):
        assert (a.float() - b.float()).abs().max() <= 0.2 * b.float().abs().max()


def test_prompt_through_the_modules_fills_the_cache(model, prompt):
    """Where a module is hooked the prompt takes the HF forward, and its keys and
    values are quantised into the cache."""
    from transformers import DynamicCache
    from dip_model import DIPDecoder
    dec = DIPDecoder(model, 64, kv_bits=4)
    handle = model.model.norm.register_forward_hook(lambda *a: None)
    try:
        logits = dec.prefill(prompt)
        cache = DynamicCache(config=model.config)
        with torch.no_grad():
            want = model(input_ids=prompt.cuda(), past_key_values=cache, use_cache=True).logits[0, -1]
    finally:
        handle.remove()
    assert torch.equal(logits, want)
    for i, layer in enumerate(cache.layers):
        for got, x in zip(dec._K.kv4_read(dec._kv4[i], 0, PLEN), (layer.keys, layer.values)):
            assert torch.equal(got.double().cpu(), quantised(x[0].transpose(0, 1)))
    dec.step()
    assert int(dec.pos) == PLEN + 1


@pytest.mark.parametrize("kv_bits", [4, 16])
def test_drawn_tokens_are_the_samplers(model, prompt, kv_bits):
    """generate draws each token from its logits with the generator's numbers."""
    import _dip_hip as K
    from dip_model import DIPDecoder
    dec = DIPDecoder(model, 64, kv_bits=kv_bits)
    how = dict(temperature=0.8, top_k=40, top_p=0.9, min_p=0.01)
    gen = lambda: torch.Generator(device="cuda").manual_seed(12)
    seq, logits = dec.generate(prompt, NEW, return_logits=True, do_sample=True, generator=gen(),
                               **how)
    u = torch.rand(NEW, device="cuda", generator=gen())
    token, _ = K.sample(logits, u, **how)
    assert seq[0, PLEN:].tolist() == token.tolist()
    again = dec.generate(prompt, NEW, do_sample=True, generator=gen(), **how)
    assert torch.equal(seq, again)
    host = dec.generate(prompt, 3, do_sample=True, generator=torch.Generator().manual_seed(1))
    assert host.shape == (1, PLEN + 3)


def test_drawing_one_candidate_is_greedy(model, prompt):
    from dip_model import DIPDecoder
    dec = DIPDecoder(model, 64)
    want = dec.generate(prompt, NEW)
    for how in (dict(top_k=1), dict(temperature=0.0), dict(top_p=1e-9)):
        assert torch.equal(dec.generate(prompt, NEW, do_sample=True, **how), want)
    assert torch.equal(dec.generate(prompt, NEW), want)  # greedy again afterwards


def test_refusals(model, prompt):
    from dip_model import DIPDecoder
    for how in (dict(kv_bits=8), dict(kv_bits=4, fused=False)):
        with pytest.raises(ValueError):
            DIPDecoder(model, 64, **how)
    dec = DIPDecoder(model, 64)
    with pytest.raises(RuntimeError):
        dec.generate(prompt, 2, do_sample=True, top_p=0.0)
    with pytest.raises(RuntimeError):
        dec.generate(prompt, 2, do_sample=True, temperature=-1.0)
    assert dec._draw is None
