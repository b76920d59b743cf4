"""GPU: DIPDecoder with its keys and values in 8 bits, and with tokens that the pruned
step drafts and the dense route verifies.  The decoder is checked against the model's
own modules with an attention in 64 bits over keys and values by the cache's
definition."""
import math

import pytest
import torch

from kv8_util import Pages
from model_util import max_rel, tiny_config, tiny_model, write_checkpoint

pytestmark = pytest.mark.gpu

PLEN, NEW = 61, 9
E4M3 = torch.float8_e4m3fn


def _model(tmp_path_factory, hidden, inter, heads, kv, keep):
    from dip_stream_predispatch import load_streaming_dip
    cfg = tiny_config(hidden=hidden, inter=inter, heads=heads, kv_heads=kv, head_dim=128, vocab=768)
    d = tmp_path_factory.mktemp(f"kv8_{hidden}_{keep}")
    write_checkpoint(tiny_model(cfg, seed=hidden), d)
    return load_streaming_dip(d, keep_ratio=keep)[0]


@pytest.fixture(scope="module", params=[(512, 1024, 4, 1), (2560, 1280, 4, 2)])
def model(request, tmp_path_factory):
    # keep 1: every channel, so that no rounding swaps a channel at the border
    return _model(tmp_path_factory, *request.param, 1.0)


@pytest.fixture(scope="module")
def pruned(tmp_path_factory):
    return _model(tmp_path_factory, 512, 1024, 4, 2, 0.3)


@pytest.fixture(scope="module")
def prompt():
    return torch.randint(0, 768, (1, PLEN), generator=torch.Generator().manual_seed(9))


class _Reference:
    """The model's modules part by part, the attention here."""

    def __init__(self, model):
        cfg = model.config
        self.m, self.n, self.rows = model, 0, [[0, 1, 2, 3]]
        self.kv = [Pages(4, cfg.num_key_value_heads) for _ in model.model.layers]

    @torch.no_grad()
    def part(self, ids):
        """The logits of every token of ids [1, n]."""
        m, n = self.m, ids.shape[1]
        inner, cfg = m.model, m.config
        nh, nkv = cfg.num_attention_heads, cfg.num_key_value_heads
        h = inner.embed_tokens(ids.cuda())
        ang = torch.arange(self.n, self.n + n).float()[:, None] * inner.rotary_emb.inv_freq.cpu()
        ang = torch.cat((ang, ang), -1)
        cos, sin = (f(ang).to(torch.bfloat16).cuda()[None, :, None] for f in (torch.cos, torch.sin))
        rot = lambda x: x * cos + torch.cat((-x[..., 64:], x[..., :64]), -1) * sin
        later = torch.arange(self.n + n, device="cuda") > self.n + torch.arange(
            n, device="cuda")[:, None]
        for L, pages in zip(inner.layers, self.kv):
            a = L.self_attn
            x = L.input_layernorm(h)
            q = rot(a.q_norm(a.q_proj(x).view(1, n, nh, 128)))[0]
            k = rot(a.k_norm(a.k_proj(x).view(1, n, nkv, 128)))
            pages.write(k, a.v_proj(x).view(1, n, nkv, 128), self.rows, [self.n])
            kk, vv = (t.cuda() for t in pages.read(self.rows[0], 0, self.n + n))
            o = torch.empty(n, nh, 128, dtype=torch.float64, device="cuda")
            for j in range(nh):
                s = q[:, j].double() @ kk[:, j // (nh // nkv)].T.contiguous() * a.scaling
                o[:, j] = s.masked_fill(later, -math.inf).softmax(-1) @ vv[:, j // (nh // nkv)]
            h = h + a.o_proj(o.to(torch.bfloat16).view(1, n, -1))
            h = h + L.mlp(L.post_attention_layernorm(h))
        self.n += n
        return m.lm_head(inner.norm(h)).view(n, -1)


# bf16 roundings on either side move a key by a step of the cache now and then (2^-3 of
# it): the module tests' bound for bf16 paths
BOUND = 4e-2


def test_logits_follow_the_definition(model, prompt):
    from dip_model import DIPDecoder
    dec = DIPDecoder(model, 128, kv_dtype=E4M3)
    assert dec.fused and dec.kv_bits == 8 and not hasattr(dec, "k_cache")
    ref = _Reference(model)
    seq, logits = dec.generate(prompt, NEW, return_logits=True)
    for t in range(NEW):
        ids = prompt if t == 0 else seq[:, PLEN + t - 1:PLEN + t]
        err = max_rel(logits[t], ref.part(ids)[-1])
        print(f"  token {t} max_rel {err:.3e}", flush=True)
        assert err < BOUND


def test_graph_equals_eager_and_repeats(model, prompt):
    from dip_model import DIPDecoder
    dec = DIPDecoder(model, 100, kv_dtype=E4M3)
    a, la = dec.generate(prompt, NEW, return_logits=True)
    b, lb = dec.generate(prompt, NEW, return_logits=True)
    c, lc = DIPDecoder(model, 100, kv_dtype=E4M3, use_graph=False).generate(prompt, NEW,
                                                                            return_logits=True)
    assert torch.equal(a, b) and torch.equal(la, lb)
    assert torch.equal(a, c) and torch.equal(la, lc)


def test_a_prompt_in_parts(model, prompt, monkeypatch):
    """Parts of a prompt attend the rows of the parts before."""
    import dip_model
    want = dip_model.DIPDecoder(model, 64, kv_dtype=E4M3).prefill(prompt).float()
    monkeypatch.setattr(dip_model, "_PROMPT_CHUNK", 12)
    parts = dip_model.DIPDecoder(model, 64, kv_dtype=E4M3)
    got = parts.prefill(prompt).float()
    assert int(parts.pos) == PLEN and max_rel(got, want) < BOUND


def test_prompt_through_the_modules_fills_the_cache(model, prompt):
    """Where a module is hooked the prompt takes the HF forward, and its keys and
    values are written into the cache."""
    from transformers import DynamicCache
    from dip_model import DIPDecoder
    dec = DIPDecoder(model, 100, kv_dtype=E4M3)
    handle = model.model.norm.register_forward_hook(lambda *a: None)
    try:
        logits = dec.prefill(prompt)
        cache = DynamicCache(config=model.config)
        with torch.no_grad():
            want = model(input_ids=prompt.cuda(), past_key_values=cache, use_cache=True).logits[0, -1]
        with pytest.raises(ValueError):
            dec.generate(prompt, 2, draft=2)
    finally:
        handle.remove()
    assert torch.equal(logits, want)
    for i, layer in enumerate(cache.layers):
        pages = Pages(2, layer.keys.shape[1])
        pages.write(layer.keys.transpose(1, 2), layer.values.transpose(1, 2), [[0, 1]], [0])
        got = dec._K.kv8_read(dec._kv8[i], dec._table, torch.zeros_like(dec.pos), PLEN)
        for x, w in zip(got, pages.read([0, 1], 0, PLEN)):
            assert torch.equal(x[0].double().cpu(), w)
    dec.step()
    assert int(dec.pos) == PLEN + 1


def _caches():
    return [dict(kv_dtype=E4M3), dict(kv_bits=4)]


@pytest.mark.parametrize("draft", [1, 3, 5])
def test_drafted_tokens_are_the_dense_models(pruned, prompt, draft):
    """Greedy: every token is the largest of the dense route's logits, whatever the
    pruned step drafts."""
    from dip_model import DIPDecoder
    dec = DIPDecoder(pruned, 128, kv_dtype=E4M3)
    new = 17
    seq, logits = dec.generate(prompt, new, return_logits=True, draft=draft)
    assert seq.shape == (1, PLEN + new) and logits.shape[0] == new
    assert seq[0, PLEN:].tolist() == logits.argmax(-1).tolist()
    ref = _Reference(pruned)
    want = torch.cat((ref.part(prompt)[-1:], ref.part(seq[:, PLEN:])[:-1]))
    for t in range(new):
        err = max_rel(logits[t], want[t])
        print(f"  token {t} max_rel {err:.3e}", flush=True)
        assert err < BOUND
    accepted, made = dec.drafts
    print(f"  accepted {accepted} of {made}", flush=True)
    assert 0 <= accepted <= made and made % draft == 0
    again, la = dec.generate(prompt, new, return_logits=True, draft=draft)
    assert torch.equal(seq, again) and torch.equal(logits, la)
    # cut at the first of some tokens
    stop = seq[0, PLEN + 6:PLEN + 8].tolist()
    cut = dec.generate(prompt, new, eos_token_id=stop, draft=draft)
    first = next(t for t in range(new) if int(seq[0, PLEN + t]) in stop)
    assert torch.equal(cut, seq[:, :PLEN + first + 1])
    assert torch.equal(dec.generate(prompt, 1, draft=draft), seq[:, :PLEN + 1])
    assert torch.equal(dec.generate(prompt, 0, draft=draft), prompt)


@pytest.mark.parametrize("cache", [0, 1])
def test_drafts_of_every_channel_are_accepted(model, prompt, cache):
    """With every channel kept the pruned step is the dense model up to roundings."""
    from dip_model import DIPDecoder
    dec = DIPDecoder(model, 128, **_caches()[cache])
    seq, logits = dec.generate(prompt, 16, return_logits=True, draft=3)
    assert seq[0, PLEN:].tolist() == logits.argmax(-1).tolist()
    accepted, made = dec.drafts
    print(f"  accepted {accepted} of {made}", flush=True)
    assert accepted >= made // 2


@pytest.mark.parametrize("cache", [0, 1])
def test_drawn_drafts(pruned, prompt, cache):
    """Drawn tokens repeat with the generator's numbers, lie among those that the filters
    keep of the dense logits, and are the greedy ones with one candidate."""
    from dip_model import DIPDecoder
    dec = DIPDecoder(pruned, 128, **_caches()[cache])
    gen = lambda: torch.Generator(device="cuda").manual_seed(12)
    how = dict(temperature=1.2, top_k=5)
    seq, logits = dec.generate(prompt, 20, return_logits=True, do_sample=True, draft=3,
                               generator=gen(), **how)
    assert torch.equal(seq, dec.generate(prompt, 20, do_sample=True, draft=3, generator=gen(),
                                         **how))
    best = logits.topk(5).indices.cpu()
    assert all(int(seq[0, PLEN + t]) in best[t] for t in range(20))
    assert dec._draw is None
    greedy = dec.generate(prompt, 12, draft=4)
    for one in (dict(top_k=1), dict(temperature=0.0)):
        assert torch.equal(dec.generate(prompt, 12, do_sample=True, draft=4, **one), greedy)
    host = dec.generate(prompt, 3, do_sample=True, draft=2,
                        generator=torch.Generator().manual_seed(1))
    assert host.shape == (1, PLEN + 3)


def test_refusals(model, prompt):
    from dip_model import DIPDecoder
    for how in (dict(kv_dtype=torch.float16), dict(kv_dtype=E4M3, kv_bits=4),
                dict(kv_dtype=E4M3, fused=False)):
        with pytest.raises(ValueError):
            DIPDecoder(model, 64, **how)
    with pytest.raises(ValueError):
        DIPDecoder(model, 128).generate(prompt, 2, draft=2)
    dec = DIPDecoder(model, 70, kv_dtype=E4M3)
    for args in (dict(draft=-1), dict(draft=8), dict(draft=7)):
        with pytest.raises(ValueError):
            dec.generate(prompt, 3, **args)
    with pytest.raises(RuntimeError):
        dec.generate(prompt, 2, draft=2, do_sample=True, top_p=0.0)
    assert dec.generate(prompt, 3, draft=6).shape == (1, PLEN + 3)
