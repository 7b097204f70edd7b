"""The streaming operators where the framework calls them, on the GPU in bf16.

A layer rounds to bf16 at most eight times between its input and its output (input,
weights, projection, norm, rotation, probabilities, head outputs, output projection),
each by 2^-8 relative, so norms agree within 8 * 2^-8 of a 64-bit evaluation."""

import copy

import pytest
import torch

from vagus_b200 import ops
from vagus_b200.inference import Generator, SamplingConfig
from vagus_b200.models import build_model
from vagus_b200.models.attention import SoftmaxAttention
from vagus_b200.models.rope import RoPE

pytestmark = pytest.mark.gpu

DEV = "cuda"
EIGHT = 8 * 2 ** -8


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)
    yield
    torch.cuda.synchronize()
    ops.check_error()


def off(a, b):
    return ((a.double().cpu() - b.double().cpu()).norm() / b.double().cpu().norm()).item()


ROPES = [dict(layout="half"), dict(rotary_dim=32), dict(rotary_dim=16, layout="half", scaling={"type": "ntk", "factor": 2}),
         dict(scaling={"type": "yarn", "factor": 4, "original_len": 64})]


@pytest.mark.parametrize("rope", ROPES)
@pytest.mark.parametrize("qk_norm", [False, True])
def test_layer_with_rope_options_trains(rope, qk_norm):
    D, L = 64, 150
    att = SoftmaxAttention(256, 4, 2, 1, qk_norm=qk_norm, rope=RoPE(256, D, 256, **rope), init_std=0.06).to(DEV)
    ref = copy.deepcopy(att).cpu().double()
    ref.rope.prepared_L = 0
    ref.rope.prepare_m(256)
    x = torch.randn(2, L, 256, device=DEV).bfloat16().requires_grad_()
    xr = x.detach().cpu().double().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = att(x)
    yr = ref(xr)
    assert off(y, yr) < EIGHT
    g = torch.randn_like(y)
    y.backward(g)
    yr.backward(g.cpu().double())
    # the backward rounds each of its own steps as often again
    assert off(x.grad, xr.grad) < 2 * EIGHT
    for (name, p), q in zip(att.named_parameters(), ref.parameters()):
        assert off(p.grad, q.grad) < 2 * EIGHT, name


@pytest.mark.parametrize("heads,kv,L", [(4, 4, 1), (8, 2, 7), (2, 1, 300)])
def test_four_bit_layer_decodes_over_the_quantised_values(heads, kv, L):
    att = SoftmaxAttention(64 * heads, heads, kv, 1, qk_norm=True, rope=RoPE(64 * heads, 64, 512), init_std=0.06)
    att = att.to(DEV).bfloat16()
    att.set_cache_bits(4)
    att.reset_cache(2, 500)
    x = torch.randn(2, 90 + L, 64 * heads, device=DEV).bfloat16()
    att.decode_step(x[:, :90])
    y = att.decode_step(x[:, 90:])
    k, v = ops.int4_read(att.kv4, 0, 90 + L)
    q, knew = att._qk(att.wq(x[:, 90:]), att.wk(x[:, 90:]), 90)
    o = ops.attention_ref(q.double(), k.double(), v.double())
    want = o.transpose(1, 2).flatten(2) @ att.wo.weight.double().t()
    assert off(y, want) < EIGHT
    # the keys in the cache are the rotated keys, quantised: within 0.54 of a step of a sixteenth of the range
    s = att.kv4.k_params[:, :, 90:90 + L, :, :1].float()
    err = (k[:, :, 90:].float() - knew.float()).unflatten(-1, (-1, 32)).abs()
    assert (err <= 0.6 * s + 2 ** -7 * knew.float().unflatten(-1, (-1, 32)).abs()).all()


def build(seed, **kw):
    torch.manual_seed(seed)
    args = dict(vocab_size=1000, dim=256, layer_count=2, head_dim=64, context_len=256, ffn_hidden_dim=512, **kw)
    m = build_model("TransformerPP", args).eval()
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() == 2:
                p.mul_(3)
    return m.to(DEV).bfloat16()


@pytest.mark.parametrize("cache_bits", [16, 4])
def test_drafted_generation(cache_bits):
    target = Generator(build(0), cache_bits=cache_bits)
    ids = torch.randint(0, 1000, (2, 20), device=DEV)
    cfg = SamplingConfig(max_new_tokens=30, temperature=0)
    for model in (build(1), copy.deepcopy(target.model)):
        draft = Generator(model, cache_bits=cache_bits)
        for g in (target, draft):
            g.reset(2, 128)
            g.prefill_ids(ids)
        got = target.gen_ids_drafted(cfg, draft, n_draft=4)
        assert got.shape == (2, 30) and target.stream_len == draft.stream_len == 50
        # every token is the most likely one, up to the rounding of two layers and the head
        logits = target.score_ids(torch.cat([ids, got], 1))[:, 19:].float()
        top, own = logits.amax(-1), logits.gather(2, got[..., None])[..., 0]
        assert (top - own <= 3 * EIGHT * logits.norm(dim=-1) / 1000 ** 0.5 * 4).all()
    sampled = SamplingConfig(max_new_tokens=12, top_k=20, seed=5)
    runs = []
    for _ in range(2):
        for g in (target, draft):
            g.reset(2, 128)
            g.prefill_ids(ids)
        runs.append(target.gen_ids_drafted(sampled, draft, n_draft=3))
    assert torch.equal(*runs)
