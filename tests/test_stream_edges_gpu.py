"""The long-context streaming kernels at calls that the documentation allows and that
lie off the common path: forward-mode derivatives of the rotation, very many short
prompts, writes that take two rows a thread, and the same call made again."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from vagus_b200 import ops
from tests.test_stream_ops import LAYOUTS, attention_64, drafted, frequencies
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


# ------------------------------------------------------------------- 4-bit cache --

def two_rows_a_thread(B, L, Hk, D, Dv):
    """Whether a write is large enough for the form that takes two rows a thread."""
    return B * L * Hk * (max(D, Dv) // 32) >= 2 * 256 * 148 * 16


def equal_to_the_plain_form(c, k, v, start):
    """Bit for bit, what was written and what was left alone (the plain form runs on the CPU)."""
    want = ops.Int4KV.empty(c.batch, c.kv_heads, c.capacity, c.head_dim, c.value_dim)
    ops.int4_append(want, k.cpu(), v.cpu(), start if isinstance(start, int) else start.cpu())
    return all(torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8)) for a, b in zip(c.tensors(), want.tensors()))


# rows of a block's threads: 256 / (D / 32) of the tensor at hand.  Heads that do not divide them, more heads than
# there are of them, one head, idle threads (D = 96), unequal dims (the narrower tensor takes fewer blocks), odd lengths
@pytest.mark.parametrize("B,L,Hk,D,Dv,dtype", [
    (2, 30401, 5, 128, 128, torch.bfloat16), (1, 101111, 3, 64, 128, torch.float16), (1, 101111, 3, 128, 64, torch.float32),
    (1, 1013, 300, 128, 128, torch.bfloat16), (2, 606209, 1, 32, 32, torch.bfloat16), (1, 134713, 3, 96, 96, torch.float16),
    (3, 2311, 44, 32, 128, torch.float32)])
def test_append_of_two_rows_a_thread(B, L, Hk, D, Dv, dtype):
    assert two_rows_a_thread(B, L, Hk, D, Dv)
    k = torch.randn(B, L, Hk, D, device=DEV).add_(0.5 * torch.randn(D, device=DEV)).to(dtype).transpose(1, 2)
    v = torch.randn(B, Hk, L, Dv, device=DEV).to(dtype)
    for start in (3, torch.randint(0, 20, (B,), device=DEV)):
        c = ops.Int4KV.empty(B, Hk, L + 20, D, Dv, device=DEV)
        ops.int4_append(c, k, v, start)
        assert equal_to_the_plain_form(c, k, v, start)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_append_of_two_rows_a_thread_off_16_bytes(dtype):
    B, L, Hk, D = 1, 101111, 3, 128
    assert two_rows_a_thread(B, L, Hk, D, D)
    packed = torch.randn(B, L, 2 * Hk * D + 1, device=DEV).to(dtype)[..., 1:]
    k, v = (t.unflatten(-1, (Hk, D)).transpose(1, 2) for t in packed.chunk(2, -1))
    c = ops.Int4KV.empty(B, Hk, L + 9, D, device=DEV)
    ops.int4_append(c, k, v, 7)
    assert equal_to_the_plain_form(c, k, v, 7)


@pytest.mark.parametrize("Hk,L", [(5, 30401), (70, 2171)])
def test_append_of_two_rows_a_thread_past_the_end(Hk, L):
    """Sequences that start before the cache and reach past its end: tokens inside are written, and nothing else."""
    B, D = 2, 128
    assert two_rows_a_thread(B, L, Hk, D, D)
    k, v = (torch.randn(B, Hk, L, D, device=DEV).bfloat16() for _ in range(2))
    cap = (L + 15) // 16 * 16
    c = ops.Int4KV.empty(B, Hk, cap, D, device=DEV)
    for t in c.tensors():
        t.fill_(1)
    left, right = -37, cap - L + 41
    ops.int4_append(c, k, v, torch.tensor([left, right], device=DEV))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="outside"):
        ops.check_error()
    want = ops.Int4KV.empty(B, Hk, cap, D)
    for t in want.tensors():
        t.fill_(1)
    for b, (at, first, last) in enumerate(((0, 37, L), (right, 0, L - 41))):
        one = ops.Int4KV.empty(1, Hk, cap, D)
        ops.int4_append(one, k[b:b + 1, :, first:last].cpu(), v[b:b + 1, :, first:last].cpu(), at)
        for a, x in zip(want.tensors(), one.tensors()):
            a[b, :, at:at + last - first] = x[0, :, at:at + last - first]
    assert all(torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8)) for a, b in zip(c.tensors(), want.tensors()))


# ------------------------------------------------------------------------ replay --

def replay(run):
    """No sum in these kernels depends on the order of arrival: the same call gives the same bits."""
    first = [t.clone() for t in run()]
    busy = torch.randn(4096, 4096, device=DEV)
    for i in range(4):
        if i % 2:
            busy @ busy                                # another load on the GPU ahead of it
        for a, b in zip(run(), first):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,H,Hk,Lq,T", [(32, 32, 8, 1, 8192), (2, 16, 8, 1, 40003), (8, 16, 16, 6, 4099), (1, 8, 8, 700, 4096),
                                         (600, 4, 2, 1, 300)])
def test_attention_replays(B, H, Hk, Lq, T, D):
    c = filled(B, Hk, T, D, D)
    q = torch.randn(B, H, Lq, D, device=DEV).bfloat16()
    replay(lambda: [ops.int4_attention(q, c, T)])
    lengths = torch.randint(0, T + 1, (B,), device=DEV)
    replay(lambda: [ops.int4_attention(q, c, lengths)])


def test_other_stream_kernels_replay():
    k, v = torch.randn(2, 4, 5000, 128, device=DEV), torch.randn(2, 4, 5000, 64, device=DEV)
    c = ops.Int4KV.empty(2, 4, 5008, 128, 64, device=DEV)
    start = torch.tensor([3, 8], device=DEV)

    def write():
        ops.int4_append(c, k, v, start)
        return [*c.tensors(), *ops.int4_read(c, start, 5000)]
    replay(write)
    q = torch.randn(2, 5000, 4, 128, device=DEV).bfloat16().requires_grad_()
    g = torch.randn_like(q)
    inv = frequencies(64).to(DEV)
    for layout in LAYOUTS:
        replay(lambda: [ops.rotary(q, None, 5, inv, layout=layout).detach(),
                        torch.autograd.grad(ops.rotary(q, None, 5, inv, layout=layout), q, g)[0]])
    for B, K, V in ((1, 4, 32000), (300, 3, 4099)):
        target, draft, tokens, ua, us = drafted(B, K, V, device=DEV)
        replay(lambda: ops.verify_draft(target, draft, tokens, ua, us))
        replay(lambda: ops.verify_draft(target, None, tokens, ua, us))
