"""GPU: the paged 8-bit cache, its attention and the verification of drafted tokens where
offsets pass 32 bits: pages behind the first 4 GB, inputs and results of more than 2^31
values, very long tables, and rows of logits that lie far apart."""
import math

import pytest
import torch

from kv4_util import attention
from kv8_util import PAGE, attention_bound
from test_gpu_kv8 import _gen, _kv, _pos
from test_gpu_verify import _check as check_verified

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


def _bf16(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g).to(torch.bfloat16)


def test_pages_behind_four_gigabytes():
    """The same calls on far pages of a large cache and on a small one."""
    import _dip_hip as K
    nkv, nh, pages = 8, 64, 70_000
    g = _gen(1)
    far, near = K.kv8_cache(nkv, pages), K.kv8_cache(nkv, 6)
    assert far.k.numel() > 1 << 32
    numbers = [69_999, 65_536, 3, 69_998, 65_537, 69_000]
    tables = [torch.tensor([t], dtype=torch.int32, device="cuda")
              for t in (numbers, list(range(6)))]
    k, v = _kv(g, 1, 300, nkv)
    qkv, w = _bf16(g, 1, 70, (nh + 2 * nkv) * 128), _bf16(g, 128)
    cos, sin = _bf16(g, 384, 128), _bf16(g, 384, 128)
    q = [_bf16(g, 1, n, nh * 128) for n in (1, 5, 60)]
    results = []
    for cache, table in zip((far, near), tables):
        print(f"far pages: {cache.k.numel()} bytes of keys", flush=True)
        K.kv8_write(k, v, cache, table, _pos(0))
        rope = torch.empty(1, 70, nh * 128, dtype=torch.bfloat16, device="cuda")
        K.qk_norm_rope_kv8(qkv, w, w, cos, sin, _pos(300), rope, cache, table, nh, nkv, 1e-6)
        out = [rope, *K.kv8_read(cache, table, _pos(0), 370)]
        out += [K.kv8_decode_attention(x, cache, table, _pos(370 - x.shape[1]), None, SCALE)
                for x in q]
        out += [K.kv8_prompt_attention(x[0], cache, table[0], 370 - x.shape[1], None, SCALE)
                for x in q]
        results.append(out)
    assert results[1][1].any() and all(x.isfinite().all() for x in results[1])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    # no other page was written
    mine = torch.zeros(pages, dtype=torch.bool, device="cuda")
    mine[numbers] = True
    assert bool((far.scales.view(pages, -1) != 0).any(-1).eq(mine).all())
    for i in range(0, pages, 10_000):
        some = far.k.view(pages, -1)[i:i + 10_000].any(-1)
        assert not bool((some & ~mine[i:i + 10_000]).any())


@pytest.mark.parametrize("nh", [8, 40])
def test_a_table_of_many_pages(nh):
    """One full page 20000 times over: the attention of 1.28 million rows is that page's."""
    import _dip_hip as K
    g = _gen(nh)
    cache, n = K.kv8_cache(1, 3), 20_000
    k, v = _kv(g, 1, PAGE, 1)
    table = torch.full((1, n), 2, dtype=torch.int32, device="cuda")
    K.kv8_write(k, v, cache, table[:, :1], _pos(0))
    kd, vd = (x[0].double().cpu() for x in K.kv8_read(cache, table[:, :1], _pos(0), PAGE))
    q = _bf16(g, 1, 1, nh * 128)
    print(f"{n} pages, {nh} heads", flush=True)
    out = K.kv8_decode_attention(q, cache, table, _pos(n * PAGE - 1), None, SCALE)
    want, size = attention(q[0].view(1, nh, 128), kd, vd, [PAGE], SCALE)
    err = (out[0].view(1, nh, 128).double().cpu() - want).abs()
    # (256 splits of 79 pages in a row at most: within attention_bound's hundreds of steps)
    assert bool((err <= attention_bound(want, size)).all()), float(err.max())


def test_more_than_two_to_the_31_values_in():
    """A prompt whose q, k and v are 4.4 GB: its last pages as by themselves."""
    import _dip_hip as K
    nh, nkv, tokens, last = 64, 8, 215_040, 192
    g = _gen(5)
    qkv = torch.empty(1, tokens, (nh + 2 * nkv) * 128, dtype=torch.bfloat16, device="cuda")
    assert qkv.numel() > 1 << 31
    part = _bf16(g, 1, 1024, qkv.shape[2])
    for i in range(0, tokens, 1024):
        qkv[:, i:i + 1024] = part
    qkv[:, -last:] = _bf16(g, 1, last, qkv.shape[2])
    w, cos, sin = _bf16(g, 128), _bf16(g, tokens, 128), _bf16(g, tokens, 128)
    pages = tokens // PAGE
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    caches = [K.kv8_cache(nkv, pages) for _ in range(2)]
    q = torch.empty(1, tokens, nh * 128, dtype=torch.bfloat16, device="cuda")
    q1 = torch.empty(1, last, nh * 128, dtype=torch.bfloat16, device="cuda")
    print("norm, rope and write of 215040 tokens", flush=True)
    K.qk_norm_rope_kv8(qkv, w, w, cos, sin, _pos(0), q, caches[0], table, nh, nkv, 1e-6)
    K.qk_norm_rope_kv8(qkv[:, -last:].contiguous(), w, w, cos, sin, _pos(tokens - last), q1,
                       caches[1], table, nh, nkv, 1e-6)
    assert torch.equal(q[:, -last:], q1) and q1.any()
    for a, b in zip(*(K.kv8_read(c, table, _pos(tokens - last), last) for c in caches)):
        assert torch.equal(a, b) and a.any()


def test_more_than_two_to_the_31_values_out():
    """Rows read, and sequences attended, of one page again and again."""
    import _dip_hip as K
    g = _gen(6)
    cache, n = K.kv8_cache(8, 1), 33_000
    K.kv8_write(*_kv(g, 1, PAGE, 8), cache, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                _pos(0))
    table = torch.zeros(1, n, dtype=torch.int32, device="cuda")
    once = K.kv8_read(cache, table, _pos(0), PAGE)
    print("read of 2.1 million rows", flush=True)
    for got, want in zip(K.kv8_read(cache, table, _pos(0), n * PAGE), once):
        assert got.numel() > 1 << 31
        got = got.view(n, PAGE, 8, 128)
        assert all(bool((got[i:i + 3000] == want).all()) for i in range(0, n, 3000))
    del got
    cache, seqs, nh = K.kv8_cache(1, 1), 66_000, 256
    K.kv8_write(*_kv(g, 1, PAGE, 1), cache, table[:, :1], _pos(0))
    few = _bf16(g, 66, 1, nh * 128)
    q = few.repeat(seqs // 66, 1, 1)
    assert q.numel() > 1 << 31
    zero = torch.zeros(seqs, 1, dtype=torch.int32, device="cuda")
    pos = torch.full((seqs,), PAGE - 1, device="cuda")
    want = K.kv8_decode_attention(few, cache, zero[:66], pos[:66], None, SCALE)
    print("attention of 66000 sequences", flush=True)
    out = K.kv8_decode_attention(q, cache, zero, pos, None, SCALE).view(-1, 66, nh * 128)
    assert all(bool((out[i:i + 100] == want[:, 0]).all()) for i in range(0, len(out), 100))


@pytest.mark.parametrize("vocab", [1000, 60013])
@pytest.mark.parametrize("how", [dict(top_k=40, top_p=0.9), dict(min_p=0.1), dict(),
                                 dict(temperature=0.0)])
def test_verified_rows_of_logits_far_apart(vocab, how):
    stride = (1 << 30) + 24
    x = torch.empty(3 * stride + vocab, dtype=torch.bfloat16, device="cuda")
    y = torch.empty(stride + vocab, dtype=torch.bfloat16, device="cuda")
    rows = x.as_strided((2, 2, vocab), (2 * stride, stride, 1))
    draft = y.as_strided((2, 1, vocab), (stride, stride, 1))
    g = _gen(vocab)
    rows.copy_(2 * torch.randn(2, 2, vocab, device="cuda", generator=g))
    draft.copy_(rows[:, :1])
    drafted = torch.stack([draft[0].argmax(-1), draft[1].argmin(-1)])
    u = torch.tensor([[0.2, 0.7], [0.999, 0.4]], device="cuda")
    print(f"verified rows of {vocab} logits far apart, {how}", flush=True)
    check_verified(rows, drafted, u, draft, **how)
    check_verified(rows, drafted, u, **how)
