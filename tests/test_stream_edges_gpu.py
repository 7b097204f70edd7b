"""The long-context streaming kernels at calls that the documentation allows and that
lie off the common path: forward-mode derivatives of the rotation, very many short
prompts."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from vagus_b200 import ops
from tests.test_stream_ops import LAYOUTS, attention_64, frequencies
from tests.test_stream_ops_gpu import filled

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)
    yield
    torch.cuda.synchronize()
    ops.check_error()


# ------------------------------------------------------------------------ rotary --

@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotary_forward_mode(dtype, layout):
    """The rotation is linear, so the tangent is the rotation of the tangent: the same kernel, the same bits."""
    inv, pos = frequencies(32).to(DEV), torch.randint(0, 100000, (2, 5), device=DEV)
    q, tq = torch.randn(2, 2, 5, 4, 64, device=DEV).to(dtype)
    k, tk = torch.randn(2, 2, 5, 2, 64, device=DEV).to(dtype)

    def run(a, b):
        return ops.rotary(a, b, pos, inv, layout=layout, scale=1.1)
    plain = run(q, k)
    want_q, want_k = run(tq, tk)
    with fwad.dual_level():
        for dq, dk in ((True, True), (True, False), (False, True)):
            out = run(fwad.make_dual(q, tq) if dq else q, fwad.make_dual(k, tk) if dk else k)
            for y, p, d, want in zip(out, plain, (dq, dk), (want_q, want_k)):
                primal, tangent = fwad.unpack_dual(y)
                assert torch.equal(primal, p)
                if d:
                    assert torch.equal(tangent, want)
                else:
                    assert tangent is None or (tangent == 0).all()
        alone = ops.rotary(fwad.make_dual(q, tq), None, pos, inv, layout=layout, scale=1.1)
        assert torch.equal(fwad.unpack_dual(alone).tangent, want_q)
        with torch.no_grad():                          # no_grad stops the backward mode, not this one
            assert torch.equal(fwad.unpack_dual(run(fwad.make_dual(q, tq), k)[0]).tangent, want_q)
        with pytest.raises(NotImplementedError):
            ops.rotary(q, k, pos, fwad.make_dual(inv, inv), layout=layout)
    assert all(torch.equal(a, b) for a, b in zip(run(q, k), plain))


@pytest.mark.parametrize("layout", LAYOUTS)
def test_rotary_forward_over_reverse(layout):
    """d / dq of <y, g> along a tangent of g: the backward rotation of that tangent."""
    inv = frequencies(64).to(DEV)
    q = torch.randn(1, 3, 2, 64, device=DEV, requires_grad=True)
    g, tg = torch.randn(2, 1, 3, 2, 64, device=DEV)
    y = ops.rotary(q, None, 7, inv, layout=layout)
    (want,) = torch.autograd.grad(y, q, tg, retain_graph=True)
    with fwad.dual_level():
        (dq,) = torch.autograd.grad(y, q, fwad.make_dual(g, tg))
        assert torch.equal(fwad.unpack_dual(dq).tangent, want)


def test_rotary_reverse_over_forward():
    """The tangent that comes out depends on the one that goes in: its gradient is the backward rotation."""
    inv = frequencies(64).to(DEV)
    q, w = torch.randn(2, 1, 3, 2, 64, device=DEV)
    tq = torch.randn(1, 3, 2, 64, device=DEV, requires_grad=True)
    with fwad.dual_level():
        y = fwad.unpack_dual(ops.rotary(fwad.make_dual(q, tq), None, 7, inv)[0:1]).tangent
        (got,) = torch.autograd.grad(y, tq, w)
    probe = q.clone().requires_grad_()
    (want,) = torch.autograd.grad(ops.rotary(probe, None, 7, inv), probe, w)
    assert torch.equal(got, want)


# --------------------------------------------------------------------- attention --

@pytest.mark.parametrize("B,H", [(4095, 16), (4097, 16)])
def test_attention_of_more_heads_than_a_grid_dimension(B, H):
    """Batch times heads on both sides of 65535, with blocks of queries long enough to be served from unpacked values."""
    Lq = n = 128
    c = filled(B, 1, n, 64, 64)
    q = torch.randn(B, Lq, H, 64, device=DEV).bfloat16().transpose(1, 2)
    got = ops.int4_attention(q, c, n)
    assert got.shape == (B, H, Lq, 64)
    k, v = ops.int4_read(c, 0, n)
    # the output and each probability round to bf16 (2^-8 each); served from unpacked values, an exponential is a fit
    # good to 7.5e-5, numerator and sum, and a hidden token weighs up to 2^-126 instead of nothing; a score is an fp32
    # sum of 64 products, off by at most 64 * 2^-24 of their sizes' sum over 8, numerator and sum
    slack = 2 ** -8 + 2e-4 + 2 * 64 * 2 ** -24 * 64 * float(q.abs().max()) * float(k.abs().max()) / 8
    tail = n * 2.0 ** -126 * float(v.abs().max())
    for b in (0, 2048, B - 1):
        want, mag = attention_64(q[b:b + 1], k[b:b + 1], v[b:b + 1], [n], True)
        assert ((got[b:b + 1].double() - want).abs() <= 2 ** -8 * want.abs() + slack * mag + tail).all()
