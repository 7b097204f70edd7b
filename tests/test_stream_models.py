"""The streaming operators where the framework calls them (CPU, fp32): RoPE
options, the 4-bit KV cache behind decode_step, drafted generation."""

import copy
import math

import pytest
import torch

from vagus_b200 import ops
from vagus_b200.inference import Generator, SamplingConfig
from vagus_b200.inference.sampling import probabilities, sample
from vagus_b200.models import build_model
from vagus_b200.models.attention import SoftmaxAttention
from vagus_b200.models.rope import RoPE, rope_frequencies

TPP = dict(vocab_size=300, dim=64, layer_count=2, head_dim=32, context_len=128, ffn_hidden_dim=128)
GDN = dict(vocab_size=300, dim=64, layer_count=2, head_count=2, key_head_dim=32, value_head_dim=32,
           ffn_hidden_dim=128, context_len=128, gate="scalar", delta=True, chunk_size=16,
           layer_pattern="gdn,softmax", softmax_head_dim=32)
ROPES = [dict(rope_layout="half"), dict(rope_dim=16), dict(rope_dim=8, rope_layout="half"),
         dict(rope_scaling={"type": "linear", "factor": 4}),
         dict(rope_layout="half", rope_scaling={"type": "yarn", "factor": 4, "original_len": 32})]


def build(name="TransformerPP", seed=0, **kw):
    torch.manual_seed(seed)
    m = build_model(name, {**(TPP if name == "TransformerPP" else GDN), **kw}).eval()
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() == 2:
                p.mul_(3)                       # spread the logits: no near ties
    return m


def test_frequencies():
    inv, m = rope_frequencies(64, 10000.0)
    assert m == 1.0 and inv.dtype == torch.float64
    i = torch.arange(32, dtype=torch.float64)
    assert torch.allclose(inv, torch.exp(-i / 32 * math.log(10000.0)), rtol=1e-14)
    assert torch.equal(rope_frequencies(64, 10000.0, {"type": "linear", "factor": 4})[0], inv / 4)
    ntk, m = rope_frequencies(64, 10000.0, {"type": "ntk", "factor": 4})
    assert m == 1.0 and ntk[0] == 1.0 and torch.isclose(ntk[-1], inv[-1] / 4, rtol=1e-12)
    yarn, m = rope_frequencies(64, 10000.0, {"type": "yarn", "factor": 4, "original_len": 2048})
    turns = 2048 * inv / (2 * math.pi)
    assert m == 0.1 * math.log(4) + 1
    assert torch.equal(yarn[turns > 40], inv[turns > 40]) and torch.allclose(yarn[turns < 0.7], inv[turns < 0.7] / 4)
    assert ((yarn <= inv) & (yarn >= inv / 4 * (1 - 1e-12))).all() and (yarn[1:] < yarn[:-1]).all()
    for bad in ({"type": "dynamic", "factor": 2}, {"type": "linear", "factor": 0.5}, {"type": "linear", "factor": 2, "x": 1},
                {"factor": 2}):
        with pytest.raises(ValueError):
            rope_frequencies(64, 10000.0, bad)


def test_rope_module_forms_agree():
    """With equal frequencies the table form and ``ops.rotary`` are one rotation; factor 1 changes nothing."""
    x = torch.randn(2, 3, 10, 32)                                     # (B, H, L, D)
    plain = RoPE(64, 32, 64)
    one = RoPE(64, 32, 64, scaling={"type": "linear", "factor": 1})
    y = ops.rotary(x.transpose(1, 2), None, 5, plain.inv_freq("cpu")).transpose(1, 2)
    # fp32 angles of positions under 16: 2^-20 and the products
    assert torch.allclose(plain(x, 5), y, atol=2e-5) and torch.allclose(one(x, 5), y, atol=2e-6)
    half = RoPE(64, 32, 64, layout="half")
    perm = torch.cat([torch.arange(0, 32, 2), torch.arange(1, 32, 2)])
    assert torch.allclose(half(x[..., perm], 5), y[..., perm], atol=2e-6)
    with pytest.raises(ValueError):
        half.tables(4)
    with pytest.raises(ValueError):
        half.rotate(torch.randn(1, 60, 2, 32), None, 5)
    assert half.to(torch.bfloat16).inv_freq("cpu").dtype == torch.float64


@pytest.mark.parametrize("rope", ROPES)
@pytest.mark.parametrize("name", ["TransformerPP", "GDNLM"])
def test_rope_options_stream_like_the_full_forward(name, rope):
    m = build(name, **rope)
    assert all(m.config[k] == v for k, v in rope.items())
    again = type(m).from_config(m.config)
    again.load_state_dict(m.state_dict())
    ids = torch.randint(0, 300, (2, 20))
    with torch.no_grad():
        full = m(ids)
        assert torch.equal(again(ids), full)
        m.reset_cache(2, 32)
        parts = torch.cat([m.decode_step(ids[:, a:b]) for a, b in ((0, 7), (7, 8), (8, 20))], 1)
    assert torch.allclose(parts, full, atol=1e-3 * full.abs().max())
    base = build(name)
    with torch.no_grad():
        assert not torch.allclose(base(ids), full, atol=1e-3 * full.abs().max())


def test_plain_configs_keep_their_keys():
    for name in ("TransformerPP", "GDNLM"):
        assert not {"rope_dim", "rope_layout", "rope_scaling"} & set(build(name).config)


def test_rope_options_train():
    """Gradients of a layer with half layout and a partial, scaled head against differences."""
    torch.manual_seed(0)
    rope = RoPE(16, 8, 32, rotary_dim=4, layout="half", scaling={"type": "yarn", "factor": 2, "original_len": 8})
    att = SoftmaxAttention(16, 2, 1, 1, qk_norm=True, rope=rope).double()
    x = torch.randn(1, 5, 16, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda a: att(a), (x,))


# ------------------------------------------------------------------ 4-bit cache --

@pytest.mark.parametrize("name,kw", [("TransformerPP", dict(kv_head_count=1)), ("GDNLM", {})])
def test_four_bit_cache_streams(name, kw):
    m = build(name, **kw)
    ids = torch.randint(0, 300, (2, 24))
    m.set_cache_bits(4)
    m.reset_cache(2, 40)
    with torch.no_grad():
        one = m.decode_step(ids)
        m.reset_cache(2, 40)
        parts = torch.cat([m.decode_step(ids[:, a:b]) for a, b in ((0, 9), (9, 10), (10, 10), (10, 24))], 1)
    assert torch.allclose(parts, one, atol=1e-3 * one.abs().max())    # however the stream is cut
    state = m.export_cache()
    nxt = m.decode_step(ids[:, :1])
    m.load_cache(state, 30)
    assert torch.equal(m.decode_step(ids[:, :1]), nxt)
    m.set_cache_bits(16)
    with pytest.raises(ValueError):
        m.load_cache(state, 30)
    m.reset_cache(2, 40)
    exact = m.decode_step(ids)
    wide = m.export_cache()
    m.set_cache_bits(4)
    with pytest.raises(ValueError):
        m.load_cache(wide, 40)
    # the quantised cache moves the logits, but not far
    assert 0 < (one - exact).norm() < 0.3 * exact.norm()


def test_four_bit_layer_is_attention_over_the_quantised_values():
    torch.manual_seed(0)
    att = SoftmaxAttention(64, 2, 1, 1, rope=RoPE(64, 32, 64))
    att.set_cache_bits(4)
    att.reset_cache(3, 50)
    x = torch.randn(3, 11, 64)
    y = att.decode_step(x)
    k, v = ops.int4_read(att.kv4, 0, 11)
    q, _ = att._qk(att.wq(x), att.wk(x), 0)
    o = ops.attention(q, k.float(), v.float())
    assert torch.allclose(y, att.wo(o.transpose(1, 2).flatten(2)), atol=1e-5)
    assert att.k_cache.numel() == 0 and att.kv4.capacity == 64
    with pytest.raises(AssertionError):
        att.decode_step(torch.randn(3, 40, 64))                       # 50 is the bound, not the rounded room


def test_cache_bits_refusals():
    with pytest.raises(ValueError):
        build().set_cache_bits(8)
    odd = build(dim=48, head_dim=24)
    with pytest.raises(ValueError):
        odd.set_cache_bits(4)
    assert all(b.att.cache_bits == 16 for b in odd.blocks)
    with pytest.raises(ValueError):
        build("GDNLM", layer_pattern="gdn").set_cache_bits(4)
    with pytest.raises(ValueError):
        Generator(build(), cache_bits=3)


# ------------------------------------------------------------ drafted generation --

def pair(seed=1, cache_bits=None, **kw):
    target, small = build(**kw), build(seed=seed, **kw)
    return Generator(target, cache_bits=cache_bits), Generator(small, cache_bits=cache_bits)


@pytest.mark.parametrize("cache_bits", [None, 4])
@pytest.mark.parametrize("n_draft", [1, 3, 8])
def test_greedy_drafted_equals_greedy(n_draft, cache_bits):
    ids = torch.randint(0, 300, (3, 9))
    cfg = SamplingConfig(max_new_tokens=17, temperature=0)
    t, d = pair(cache_bits=cache_bits)
    want = t.generate_ids(ids, cfg, max_len=64)
    for draft in (d, Generator(copy.deepcopy(t.model))):              # one that disagrees, one that agrees
        for g in (t, draft):
            g.reset(3, 64)
            g.prefill_ids(ids)
        got = t.gen_ids_drafted(cfg, draft, n_draft=n_draft)
        assert torch.equal(got, want) and t.stop_reason == "max_new_tokens"
        assert t.stream_len == draft.stream_len == 26 and torch.equal(t.streams.head, want[:, -1])
        more = t.gen_ids_drafted(SamplingConfig(max_new_tokens=5, temperature=0), draft, n_draft=n_draft)
        t.reset(3, 64)
        t.prefill_ids(torch.cat([ids, want], 1))
        assert torch.equal(t.gen_ids(SamplingConfig(max_new_tokens=5, temperature=0)), more)


def test_drafted_stops_and_capacity():
    ids = torch.randint(0, 300, (1, 5))
    t, d = pair()
    want = t.generate_ids(ids, SamplingConfig(max_new_tokens=12, temperature=0), max_len=40)[0].tolist()

    def run(cfg, cap):
        for g in (t, d):
            g.reset(1, cap)
            g.prefill_ids(ids)
        return t.gen_ids_drafted(cfg, d, n_draft=4)[0].tolist()
    stop = want[6]
    first = want.index(stop)
    got = run(SamplingConfig(max_new_tokens=12, temperature=0, stop_ids=(stop,)), 40)
    assert got == want[:first + 1] and t.stop_reason == "stop_id" and t.stream_len == d.stream_len == 6 + first
    got = run(SamplingConfig(max_new_tokens=12, temperature=0), 8)
    assert t.stop_reason == "capacity" and got == want[:4] and t.fed_len == 8
    assert run(SamplingConfig(max_new_tokens=0), 40) == []


def test_drafted_rows_stop_when_all_have():
    ids = torch.randint(0, 300, (2, 5))
    t, d = pair()
    want = t.generate_ids(ids, SamplingConfig(max_new_tokens=12, temperature=0), max_len=40)
    stops = (int(want[0, 1]), int(want[1, 7]))
    cfg = SamplingConfig(max_new_tokens=12, temperature=0, stop_ids=stops)
    plain = t.generate_ids(ids, cfg, max_len=40)
    for g in (t, d):
        g.reset(2, 40)
        g.prefill_ids(ids)
    assert torch.equal(t.gen_ids_drafted(cfg, d, n_draft=3), plain)


def test_drafted_samples_follow_the_target():
    """The first token of many streams, drafted by another model: counts of the likely tokens against the
    target's probabilities, within five standard deviations of a binomial count."""
    t, d = pair()
    N = 4000
    ids = torch.randint(0, 300, (1, 6)).expand(N, 6)
    cfg = SamplingConfig(max_new_tokens=2, top_k=8, seed=11)
    for g in (t, d):
        g.reset(N, 16)
        g.prefill_ids(ids)
    got = t.gen_ids_drafted(cfg, d, n_draft=1)
    with torch.no_grad():
        p = probabilities(t.model(ids[:1])[:, -1], cfg)[0]
    count = torch.bincount(got[:, 0], minlength=300)
    assert ((count - N * p).abs() <= 5 * torch.sqrt(N * p * (1 - p)) + 1e-3).all()


def test_drafted_refusals():
    ids = torch.randint(0, 300, (1, 5))
    cfg = SamplingConfig(max_new_tokens=4)
    t, d = pair()
    with pytest.raises(RuntimeError):
        t.gen_ids_drafted(cfg, d)
    for g in (t, d):
        g.reset(1, 20)
        g.prefill_ids(ids)
    with pytest.raises(ValueError):
        t.gen_ids_drafted(cfg, d, n_draft=0)
    with pytest.raises(ValueError):
        t.gen_ids_drafted(cfg, t)
    d.prefill_ids(ids[:, :1])
    with pytest.raises(ValueError):
        t.gen_ids_drafted(cfg, d)
    other = Generator(build(vocab_size=200))
    recurrent = Generator(build("GDNLM"))
    for g, err in ((other, ValueError), (recurrent, TypeError)):
        g.reset(1, 20)
        g.prefill_ids(ids.clamp(max=199))
        with pytest.raises(err):
            t.gen_ids_drafted(cfg, g)
    with pytest.raises(ValueError):
        recurrent.model.rewind_cache(1)
    with pytest.raises(ValueError):
        t.model.rewind_cache(6)


def test_probabilities_are_what_sample_draws_from():
    logits = torch.tensor([[4.0, 3.0, 1.0, -2.0], [0.0, 0.5, 0.25, 0.1]])
    for cfg in (SamplingConfig(temperature=0.7), SamplingConfig(top_k=2), SamplingConfig(top_p=0.8),
                SamplingConfig(temperature=0)):
        p = probabilities(logits, cfg)
        assert torch.allclose(p.sum(-1), torch.ones(2))
        assert torch.equal(probabilities(logits[:, None], cfg)[:, 0], p)
        rng = torch.Generator().manual_seed(0)
        seen = {int(sample(logits, cfg, rng)[0]) for _ in range(200)}
        assert seen <= set(torch.nonzero(p[0]).flatten().tolist())
