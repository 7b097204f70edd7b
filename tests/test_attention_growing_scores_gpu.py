"""Attention whose scores grow along the keys by more than the lazy softmax tolerates,
in some rows of a warp and not in others."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Lq,Lk", [(256, 640), (384, 384)])
def test_rows_that_raise_their_reference_alone(D, causal, Lq, Lk):
    from vagus_b200 import ops
    torch.manual_seed(0)
    q = torch.randn(1, 2, Lq, D, device="cuda")
    k = torch.randn(1, 2, Lk, D, device="cuda")
    v = torch.randn(1, 2, Lk, D, device="cuda").bfloat16()
    k *= (1 + 12 * torch.arange(Lk, device="cuda") / Lk)[None, None, :, None]      # later keys score higher
    q[:, :, ::3] *= 0.01                                                           # these rows never raise
    q, k = q.bfloat16(), k.bfloat16()
    got = ops.attention(q, k, v, causal)
    s = q.double() @ k.double().transpose(-1, -2) / D ** 0.5
    if causal:
        s = s.masked_fill(torch.ones(Lq, Lk, dtype=torch.bool, device="cuda").triu(Lk - Lq + 1), float("-inf"))
    p = torch.softmax(s, -1)
    want, mag = p @ v.double(), p @ v.double().abs()
    # output and probabilities round to bf16 (2^-8 each); the exponential's fit is off by 7.5e-5, and a score is an
    # fp32 sum of D products, off by D 2^-24 sum |q k| / sqrt(D), which moves a probability by that, twice
    top = float(q.double().abs().sum(-1).amax() * k.double().abs().amax()) / D ** 0.5
    slack = 2 ** -8 + 2e-4 + 2 * D * 2 ** -24 * top
    assert ((got.double() - want).abs() <= 2 ** -8 * want.abs() + slack * mag).all()
    torch.cuda.synchronize()
    ops.check_error()
