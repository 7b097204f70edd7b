"""The long-context streaming kernels against their definitions in 64 bits and
their plain forms, at the sizes, strides and masks where they can go wrong.

Tolerances count roundings: half a step relative (finfo.eps / 2) for each rounding
to 16 bits, and for 32-bit work the bound written beside it."""

import pytest
import torch

from vagus_b200 import ops
from tests.test_stream_ops import (LAYOUTS, attention_64, cache_refusals, drafted, frequencies, held_64,
                                   rotary_64, rotary_refusals, verify_64, verify_refusals)

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = (torch.bfloat16, torch.float16, torch.float32)


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)
    yield
    torch.cuda.synchronize()
    ops.check_error()


# ----------------------------------------------------------------------- rotary --

def rotary_close(x, y, pos, inv, layout, scale):
    want = rotary_64(x, pos, inv, layout, scale)
    half = torch.finfo(x.dtype).eps / 2 if x.dtype != torch.float32 else 0.0
    # angle: a fraction of a turn in fp32 (2^-25 turns = 1.9e-7 rad), sine and cosine to 2 ulp,
    # one rounding by the scale, three in the products: under 8e-7 of |x_a| + |x_b| <= 2 max|x|
    slack = 8e-7 * scale * 2 * x.double().abs().amax(-1, keepdim=True) + torch.finfo(x.dtype).smallest_normal * half
    assert ((y.double() - want).abs() <= half * 1.001 * want.abs() + 1.01 * slack).all()
    R = 2 * inv.shape[0]
    assert torch.equal(y[..., R:], x[..., R:])


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,H,Hk,D,R", [(1, 1, 1, 1, 64, 64), (8, 1, 16, 16, 64, 64), (2, 37, 8, 2, 128, 64),
                                          (3, 5, 6, 3, 96, 48), (1, 700, 4, 1, 256, 256), (2, 3, 5, 5, 10, 6),
                                          (2, 9, 2, 1, 72, 34), (1, 2, 1, 1, 2, 2), (1, 3, 2, 2, 1024, 1024)])
def test_rotary(B, L, H, Hk, D, R, dtype, layout):
    q, k = (torch.randn(B, L, h, D, device=DEV).to(dtype) for h in (H, Hk))
    inv = frequencies(R).to(DEV)
    cases = [(4095, 4095 + torch.arange(L, device=DEV).expand(B, L)),
             (torch.randint(0, 1 << 21, (B, L), device=DEV),) * 2]
    cases.append((torch.arange(L, device=DEV).int() * 3, (3 * torch.arange(L, device=DEV)).expand(B, L)))
    for given, pos in cases:
        yq, yk = ops.rotary(q, k, given, inv, layout=layout, scale=1.2)
        rotary_close(q, yq, pos, inv, layout, 1.2)
        rotary_close(k, yk, pos, inv, layout, 1.2)
        assert yq.is_contiguous() and yq.dtype == dtype
    assert torch.equal(ops.rotary(q, None, 4095, inv, layout=layout, scale=1.2),
                       ops.rotary(q, k, 4095, inv, layout=layout, scale=1.2)[0])


@pytest.mark.parametrize("layout", LAYOUTS)
def test_rotary_strides(layout):
    inv = frequencies(64).to(DEV)
    pos = torch.arange(6, device=DEV).expand(2, 6)
    packed = torch.randn(2, 6, 12 * 64 + 8, device=DEV).bfloat16()
    q, k = packed[..., 8:8 * 64 + 8].view(2, 6, 8, 64), packed[..., 8 * 64 + 8:].view(2, 6, 4, 64)
    odd = torch.randn(2, 6, 12 * 64 + 3, device=DEV).bfloat16()[..., 3:].unflatten(-1, (12, 64))
    heads_first = torch.randn(2, 8, 6, 64, device=DEV).bfloat16().transpose(1, 2)
    inner = torch.randn(2, 6, 64, 8, device=DEV).bfloat16().transpose(2, 3)
    same = torch.randn(1, 1, 8, 64, device=DEV).bfloat16().expand(2, 6, 8, 64)
    for x, y in ((q, k), (odd[:, :, :8], odd[:, :, 8:]), (heads_first, k), (inner, k), (same, inner)):
        for z, w in zip((x, y), ops.rotary(x, y, 0, inv, layout=layout)):
            rotary_close(z, w, pos, inv, layout, 1.0)


def test_rotary_matches_the_table_form():
    """Interleaved over the whole head it is the rotation that ``qk_norm_rope`` takes from tables."""
    from vagus_b200.models.rope import RoPE
    rope = RoPE(512, 64, 300).to(DEV)
    x = torch.randn(2, 300, 8, 64, device=DEV).bfloat16()
    inv = 10000.0 ** (-torch.arange(32, device=DEV, dtype=torch.float64) / 32)
    a, b = ops.rotary(x, None, 0, inv), ops.qk_norm_rope(x, None, rope.tables(300))
    # the tables' fp32 angles are off by up to 300 * 2^-23 (frequency and product), then both round once
    slack = 2 * 300 * 2 ** -23 * 2 * x.float().abs().amax(-1, keepdim=True)
    assert ((a.float() - b.float()).abs() <= 2 * 2 ** -8 * b.float().abs() + slack).all()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", TYPES)
def test_rotary_backward(dtype, layout):
    inv = frequencies(32).to(DEV)
    pos = torch.randint(0, 100000, (2, 33), device=DEV)
    q = torch.randn(2, 33, 4, 64, device=DEV).to(dtype).requires_grad_()
    k = torch.randn(2, 33, 2, 64, device=DEV).to(dtype).requires_grad_()
    gq = torch.randn(2, 33, 4, 64, device=DEV).to(dtype)
    yq, yk = ops.rotary(q, k, pos, inv, layout=layout, scale=1.1)
    # k's gradient comes expanded from one value per row
    gk = torch.randn(2, 33, 2, 1, device=DEV).to(dtype).expand(2, 33, 2, 64)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk), retain_graph=True)
    rotary_close(gq, dq, -pos, inv, layout, 1.1)
    rotary_close(gk, dk, -pos, inv, layout, 1.1)
    assert torch.equal(torch.autograd.grad(yk, k, gk, retain_graph=True)[0], dk)      # one of the two alone
    assert torch.equal(torch.autograd.grad(yq, q, gq, retain_graph=True)[0], dq)
    only = ops.rotary(q, k.detach(), pos, inv, layout=layout, scale=1.1)[0]
    assert torch.equal(torch.autograd.grad(only, q, gq)[0], dq)
    if dtype == torch.float32:                        # against differences, along one direction
        f = lambda a: (ops.rotary(a, None, pos, inv, layout=layout, scale=1.1).double() * gq.double()).sum()  # noqa: E731
        d = torch.randn_like(q)
        h = 2.0 ** -3                                 # linear in q: any step does, rounding is 2^-24 / h a term
        diff = (f(q.detach() + h * d) - f(q.detach() - h * d)) / (2 * h)
        got = (dq.double() * d.double()).sum()
        assert (diff - got).abs() <= 2e-6 / h * (gq.double().abs() * (d.double().abs() + 1)).sum() * 4


def test_rotary_double_backward():
    inv = frequencies(8).to(DEV)
    q = torch.randn(1, 3, 2, 8, device=DEV, requires_grad=True)
    y = ops.rotary(q, None, 2, inv)
    g = torch.randn_like(y).requires_grad_()
    (dq,) = torch.autograd.grad(y, q, g, create_graph=True)
    w = torch.randn_like(dq)
    (dg,) = torch.autograd.grad(dq, g, w)
    rotary_close(w, dg, (2 + torch.arange(3, device=DEV)).expand(1, 3), inv, "interleaved", 1.0)


def test_rotary_empty():
    inv = frequencies(8).to(DEV)
    for B, L, H, Hk in ((0, 3, 2, 2), (2, 0, 2, 2), (2, 3, 2, 0), (2, 3, 0, 1)):
        yq, yk = ops.rotary(torch.randn(B, L, H, 8, device=DEV), torch.randn(B, L, Hk, 8, device=DEV), 0, inv)
        assert yq.shape == (B, L, H, 8) and yk.shape == (B, L, Hk, 8)


def test_rotary_refuses_a_token_past_32_bits():
    q = torch.zeros(1, 1, 1, 2, device=DEV).bfloat16().expand(1, 1, 1 << 30, 2)
    with pytest.raises(RuntimeError, match="rejected"):
        ops.rotary(q, None, 0, frequencies(2).to(DEV))


def test_rotary_wide_heads_and_many_tokens():
    for B, L, H, Hk, D, R in ((1, 2, 1, 1, 4096, 4096), (300, 7, 1, 0, 8, 2), (5, 4001, 2, 1, 64, 16)):
        for layout in LAYOUTS:
            q, k = torch.randn(B, L, H, D, device=DEV), torch.randn(B, L, Hk, D, device=DEV)
            inv = frequencies(R).to(DEV)
            yq, yk = ops.rotary(q, k, 3, inv, layout=layout)
            pos = (3 + torch.arange(L, device=DEV)).expand(B, L)
            rotary_close(q, yq, pos, inv, layout, 1.0)
            if Hk:
                rotary_close(k, yk, pos, inv, layout, 1.0)
    with pytest.raises(ValueError, match="8192"):
        x = torch.zeros(1, 1, 1, 8194, device=DEV)
        ops.rotary(x, None, 0, torch.zeros(4097, device=DEV))


# ------------------------------------------------------------------ 4-bit cache --

def plain_cache(k, v, cap, start):
    """A CPU cache of the same content."""
    c = ops.Int4KV.empty(k.shape[0], k.shape[1], cap, k.shape[3], v.shape[3])
    ops.int4_append(c, k.cpu(), v.cpu(), start if isinstance(start, int) else start.cpu())
    return c


def held_by_the_definition(x, codes, params, values):
    """What a cache holds of x, group by group, in 64 bits."""
    g = x.double().unflatten(-1, (-1, 32))
    s, b = params[..., :1].double(), params[..., 1:].double()
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    # s and b: one rounding to bf16 (2^-8), after fp32 steps of 2^-24 of what they subtract
    assert ((s - (hi - lo) / 15).abs() <= 2 ** -8 * 1.001 * (hi - lo) / 15 + 2 ** -24 * (lo.abs() + hi.abs())).all()
    assert ((b - (lo - 128 * s)).abs() <= 2 ** -8 * 1.001 * (lo - 128 * s).abs()).all()
    level = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).unflatten(-1, (-1, 32)).double() + 128
    r = (g - b) / s
    # the fp32 difference and quotient, at most 143.5 inside the grid, are off by 2 * 143.5 * 2^-24 < 2^-15,
    # so the code is the 64-bit one unless that lies within 2^-15 of a half
    near = (r - r.floor() - 0.5).abs() < 2 ** -15
    assert ((level == torch.round(r).clamp(128, 143)) | near | (s == 0)).all()
    assert torch.equal(values.double().unflatten(-1, (-1, 32)), (level * s + b).float().bfloat16().double())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,Hk,L,D,Dv", [(1, 1, 1, 32, 32), (3, 2, 1, 64, 64), (2, 5, 37, 128, 64), (1, 4, 513, 64, 128),
                                         (2, 1, 3, 96, 256)])
def test_append_and_read_equal_the_plain_form(B, Hk, L, D, Dv, dtype):
    k = (torch.randn(B, L, Hk, D, device=DEV) * torch.exp(2 * torch.randn(D, device=DEV)) + 3).to(dtype).transpose(1, 2)
    v = torch.randn(B, Hk, L, Dv, device=DEV).to(dtype)
    k[0, 0, 0, :32] = 1.5
    for start in (0, 11, torch.randint(0, 30, (B,), device=DEV), torch.randint(0, 30, (B,), device=DEV).int()):
        c = ops.Int4KV.empty(B, Hk, L + 30, D, Dv, device=DEV)
        ops.int4_append(c, k, v, start)
        for have, want in zip(c.tensors(), plain_cache(k, v, L + 30, start).tensors()):
            assert torch.equal(have.cpu().view(torch.uint8), want.view(torch.uint8))
        at = (start if isinstance(start, torch.Tensor) else torch.full((B,), start, device=DEV)).long()
        i, j = torch.arange(B, device=DEV)[:, None, None], torch.arange(Hk, device=DEV)[None, :, None]
        at = at[:, None, None] + torch.arange(L, device=DEV)
        ky, vy = ops.int4_read(c, start, L)
        held_by_the_definition(k, c.k_codes[i, j, at], c.k_params[i, j, at], ky)
        held_by_the_definition(v, c.v_codes[i, j, at], c.v_params[i, j, at], vy)
        part = ops.int4_read(c, start, max(1, L // 2))
        assert all(torch.equal(p, w[:, :, :max(1, L // 2)]) for p, w in zip(part, ops.int4_read(c, start, L)))


def test_append_extremes_equal_the_plain_form():
    """Ties of the rounding, tiny and huge groups, NaN and infinities."""
    k = torch.zeros(1, 1, 40, 64, device=DEV)
    for i in range(30):
        k[0, 0, i] = torch.randn(64, device=DEV) * 10.0 ** (i * 2.5 - 37) + (i % 3) * 10.0 ** (i * 2.5 - 37)
    k[0, 0, 30] = torch.arange(64, device=DEV).float() / 2            # steps of one and a half: exact halves
    k[0, 0, 31] = (torch.arange(64, device=DEV) % 31).float()
    k[0, 0, 32, 3], k[0, 0, 33, 40], k[0, 0, 34, 0] = float("nan"), float("inf"), float("-inf")
    k[0, 0, 35], k[0, 0, 36, :32] = -7.25, 1e-40
    c = ops.Int4KV.empty(1, 1, 40, 64, device=DEV)
    ops.int4_append(c, k, k, 0)
    want = plain_cache(k, k, 40, 0)
    ky, _ = ops.int4_read(c, 0, 40)
    wy, _ = ops.int4_read(want, 0, 40)
    assert torch.equal(ky.isnan().cpu(), wy.isnan())
    assert torch.equal(ky.cpu()[~wy.isnan()], wy[~wy.isnan()])
    fine = ~wy.isnan().reshape(40, 64).any(1)
    assert torch.equal(c.k_codes.cpu()[0, 0, :40][fine], want.k_codes[0, 0, :40][fine])


def test_append_many_sequences_and_unequal_dims():
    for B, L, D, Dv in ((70000, 1, 32, 64), (3, 700, 512, 32), (2, 5, 32, 1024)):
        k, v = torch.randn(B, 1, L, D, device=DEV).bfloat16(), torch.randn(B, 1, L, Dv, device=DEV).bfloat16()
        c = ops.Int4KV.empty(B, 1, L, D, Dv, device=DEV)
        ops.int4_append(c, k, v, 0)
        ky, vy = ops.int4_read(c, 0, L)
        held_by_the_definition(k, c.k_codes[:, :, :L], c.k_params[:, :, :L], ky)
        held_by_the_definition(v, c.v_codes[:, :, :L], c.v_params[:, :, :L], vy)


def test_append_strides():
    packed = torch.randn(2, 9, 3 * (64 + 32) + 1, device=DEV).bfloat16()[..., 1:]
    k = packed[..., :192].unflatten(-1, (3, 64)).transpose(1, 2)      # bases off 16 bytes
    v = packed[..., 192:].unflatten(-1, (3, 32)).transpose(1, 2)
    inner = torch.randn(2, 3, 64, 9, device=DEV).bfloat16().transpose(2, 3)
    one = torch.randn(1, 1, 1, 32, device=DEV).bfloat16().expand(2, 3, 9, 32)
    for a, b in ((k, v), (inner, v), (k, one)):
        c = ops.Int4KV.empty(2, 3, 16, 64, 32, device=DEV)
        ops.int4_append(c, a, b, 2)
        for have, want in zip(c.tensors(), plain_cache(a, b, 16, 2).tensors()):
            assert torch.equal(have.cpu(), want)


def test_append_outside_is_reported_and_writes_nothing():
    c = ops.Int4KV.empty(3, 1, 16, 32, device=DEV)
    k = torch.randn(3, 1, 2, 32, device=DEV)
    ops.int4_append(c, k, k, torch.tensor([15, -1, 4], device=DEV))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="outside"):
        ops.check_error()
    ok = torch.zeros(3, 16, dtype=torch.bool)
    ok[0, 15] = ok[1, 0] = ok[2, 4] = ok[2, 5] = True
    assert torch.equal((c.k_params[:, 0] != 0).flatten(2).any(-1).cpu(), ok)
    y, _ = ops.int4_read(c, torch.tensor([15, -1, 4], device=DEV), 2)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="outside"):
        ops.check_error()
    assert (y[0, :, 1] == 0).all() and (y[1, :, 0] == 0).all() and (y[2] != 0).any(-1).all()


def test_places_at_the_ends_of_64_bits():
    """Places whose sums with a token's index leave 64 bits are outside like any other."""
    far = torch.tensor([2 ** 63 - 1, -2 ** 63, 2 ** 60, -2 ** 60, 2 ** 62 - 1, 3], device=DEV)
    for L in (2, 300):
        c = ops.Int4KV.empty(6, 1, 320, 64, device=DEV)
        x = torch.randn(6, 1, 320, 64, device=DEV)
        ops.int4_append(c, x, x, 0)
        before = [t.clone() for t in c.tensors()]
        ops.int4_append(c, x[:, :, :L].flip(2).contiguous(), x[:, :, :L], far)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="outside"):
            ops.check_error()
        assert all(torch.equal(t[:5], u[:5]) for t, u in zip(c.tensors(), before))
        y, _ = ops.int4_read(c, far, L)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="outside"):
            ops.check_error()
        assert (y[:5] == 0).all() and torch.equal(y[5], ops.int4_read(c, 3, L)[0][5])
        for call in (lambda: ops.int4_append(c, x[:, :, :L], x[:, :, :L], 2 ** 63 - 1),
                     lambda: ops.int4_read(c, 2 ** 63 - 1, L), lambda: ops.int4_read(c, 0, 2 ** 63 - 1)):
            with pytest.raises(ValueError):
                call()


# -------------------------------------------------------------------- attention --

def filled(B, Hk, cap, D, Dv):
    c = ops.Int4KV.empty(B, Hk, cap, D, Dv, device=DEV)
    k = torch.randn(B, Hk, cap, D, device=DEV) + 0.5 * torch.randn(D, device=DEV)
    ops.int4_append(c, k.bfloat16(), torch.randn(B, Hk, cap, Dv, device=DEV).bfloat16(), 0)
    return c


def attention_close(q, c, lengths, got, causal=True):
    k, v = ops.int4_read(c, 0, c.capacity)
    want, mag = attention_64(q, k, v, lengths, causal)
    # the output and each probability round to bf16 (2^-8); a score is an fp32 sum of D products, off
    # by at most D 2^-24 sum |q k| / sqrt(D), which moves a probability by that, numerator and sum
    top = (q.double().abs().sum(-1).amax() * k.double().abs().amax()) / q.shape[-1] ** 0.5
    slack = 2 ** -8 + 2 * q.shape[-1] * 2 ** -24 * float(top) + 2 ** -18
    assert ((got.double() - want).abs() <= 2 ** -8 * want.abs() + slack * mag).all()
    assert (got[want.abs().sum(-1) == 0] == 0).all()


@pytest.mark.parametrize("D,Dv", [(64, 64), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("H,Hk,Lq", [(1, 1, 1), (4, 4, 1), (8, 1, 1), (6, 2, 3), (2, 2, 8), (3, 1, 3), (4, 2, 6),
                                     (5, 5, 19), (16, 1, 3)])
def test_attention_lengths(H, Hk, Lq, D, Dv):
    lens = torch.tensor([0, 1, 2, 15, 16, 17, 31, 33, 64, 129, 200, 208], device=DEV)
    c = filled(len(lens), Hk, 208, D, Dv)
    q = torch.randn(len(lens), Lq, H, D, device=DEV).bfloat16().transpose(1, 2)
    for n in (lens, lens.int()):
        attention_close(q, c, lens, ops.int4_attention(q, c, n))
    attention_close(q, c, lens, ops.int4_attention(q, c, lens, causal=False), causal=False)
    for n in (0, 1, 40, 208):
        got = ops.int4_attention(q, c, n)
        assert got.shape == (len(lens), H, Lq, Dv) and got.transpose(1, 2).is_contiguous()
        attention_close(q, c, torch.full_like(lens, n), got)


@pytest.mark.parametrize("B,H,Hk,Lq,T,D", [(1, 16, 16, 1, 997, 64), (2, 8, 2, 1, 4099, 128), (1, 2, 1, 5, 20011, 128),
                                           (3, 4, 4, 6, 1031, 64), (1, 4, 2, 40, 777, 128)])
def test_attention_split_over_a_long_cache(B, H, Hk, Lq, T, D):
    c = filled(B, Hk, T, D, D)
    q = (2 * torch.randn(B, H, Lq, D, device=DEV)).bfloat16()
    got = ops.int4_attention(q, c, T)
    attention_close(q, c, torch.full((B,), T, device=DEV), got)
    same = ops.int4_attention(q, c, torch.full((B,), T, device=DEV))
    attention_close(q, c, torch.full((B,), T, device=DEV), same)
    assert torch.equal(ops.int4_attention(q, c, T), got)              # no order of arrival in the result


def test_attention_ignores_what_lies_past_a_length():
    c = filled(3, 2, 160, 64, 128)
    q = torch.randn(3, 4, 4, 64, device=DEV).bfloat16()
    lens = torch.tensor([50, 0, 97], device=DEV)
    want, single = ops.int4_attention(q, c, lens), ops.int4_attention(q, c, 70)
    bad = float("nan")
    for b, n in enumerate(lens.tolist()):
        for t in c.tensors():
            t[b, :, max(n, 70):] = 255 if t.dtype == torch.uint8 else bad
    assert torch.equal(ops.int4_attention(q, c, 70), single)
    for b, n in enumerate(lens.tolist()):
        for t in c.tensors():
            t[b, :, n:] = 255 if t.dtype == torch.uint8 else bad
    assert torch.equal(ops.int4_attention(q, c, lens), want)
    # a NaN that is seen reaches the result
    c.v_params[0, :, 20] = bad
    assert ops.int4_attention(q, c, lens)[0].isnan().all()


def test_attention_large_scores_and_one_key():
    """Scores in the hundreds: one key takes all the weight."""
    c = filled(1, 1, 96, 128, 128)
    k, v = ops.int4_read(c, 0, 96)
    q = (40 * k[:, :, 37:38].float()).bfloat16()
    got = ops.int4_attention(q, c, 96, causal=False)
    assert torch.equal(got, v[:, :, 37:38])


def test_attention_scores_far_below_zero():
    """Scores of -1e35 and less: the nearest key still takes all the weight."""
    c = ops.Int4KV.empty(1, 1, 32, 64, device=DEV)
    k = -1e16 * torch.arange(1, 21, device=DEV).float()[:, None].expand(1, 1, 20, 64)
    ops.int4_append(c, k.contiguous(), torch.randn(1, 1, 20, 64, device=DEV), 0)
    q = torch.full((1, 2, 1, 64), 1e18, device=DEV).bfloat16()
    v = ops.int4_read(c, 0, 20)[1]
    for lengths in (20, torch.tensor([20], device=DEV), 1):
        assert torch.equal(ops.int4_attention(q, c, lengths), v[:, :, :1].expand(1, 2, 1, 64))


def test_attention_strided_queries_and_other_types():
    c = filled(2, 2, 64, 64, 64)
    lens = torch.full((2,), 64, device=DEV)
    packed = torch.randn(2, 3, 4 * 64 + 24, device=DEV).bfloat16()
    for q in (packed[..., 8:264].unflatten(-1, (4, 64)).transpose(1, 2), packed[..., 3:259].unflatten(-1, (4, 64)).transpose(1, 2),
              torch.randn(2, 4, 64, 3, device=DEV).bfloat16().transpose(2, 3),
              torch.randn(1, 1, 1, 64, device=DEV).bfloat16().expand(2, 4, 3, 64)):
        attention_close(q, c, lens, ops.int4_attention(q, c, 64))
    q = torch.randn(2, 4, 3, 64, device=DEV)
    attention_close(q, c, lens, ops.int4_attention(q, c, 64))          # fp32: the plain form
    odd = ops.Int4KV.empty(2, 2, 32, 32, 96, device=DEV)               # other head dims: the plain form
    ops.int4_append(odd, torch.randn(2, 2, 32, 32, device=DEV), torch.randn(2, 2, 32, 96, device=DEV), 0)
    q = torch.randn(2, 4, 3, 32, device=DEV).bfloat16()
    attention_close(q, odd, lens - 40, ops.int4_attention(q, odd, lens - 40))


def test_attention_length_beyond_the_cache_is_reported():
    c = filled(2, 1, 32, 64, 64)
    q = torch.randn(2, 1, 1, 64, device=DEV).bfloat16()
    got = ops.int4_attention(q, c, torch.tensor([33, -5], device=DEV))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="outside"):
        ops.check_error()
    attention_close(q, c, torch.tensor([32, 0]), got)


def test_attention_empty_batch_and_no_queries():
    c = filled(2, 2, 16, 64, 64)
    assert ops.int4_attention(torch.empty(2, 4, 0, 64, device=DEV).bfloat16(), c, 16).shape == (2, 4, 0, 64)
    e = ops.Int4KV.empty(0, 2, 16, 64, device=DEV)
    assert ops.int4_attention(torch.empty(0, 4, 1, 64, device=DEV).bfloat16(), e, 16).shape == (0, 4, 1, 64)
    z = ops.Int4KV.empty(2, 2, 0, 64, device=DEV)
    assert (ops.int4_attention(torch.randn(2, 4, 1, 64, device=DEV).bfloat16(), z, 0) == 0).all()


def test_attention_cache_past_32_bit_offsets():
    """72 heads of 2^20 tokens: the last heads' codes lie past 2^32 bytes."""
    Hk, cap = 72, 1 << 20
    c = ops.Int4KV.empty(1, Hk, cap, 128, device=DEV)
    n = cap - 5
    k = torch.randn(1, Hk, 40, 128, device=DEV).bfloat16()
    v = torch.randn(1, Hk, 40, 128, device=DEV).bfloat16()
    ops.int4_append(c, k, v, n - 40)
    y, _ = ops.int4_read(c, n - 40, 40)
    assert torch.equal(y[:, -1:].cpu(), held_64(k[:, -1:].float().cpu()))
    q = torch.randn(1, Hk, 1, 128, device=DEV).bfloat16()
    got = ops.int4_attention(q, c, n)[:, -1:]
    kk, vv = ops.int4_read(c, n - 64, 64)
    s = (kk[0, -1].double() @ q[0, -1, 0].double()) / 128 ** 0.5
    # the zeroed tokens score 0 and weigh 1 each, with values of zero
    w = torch.exp(s)
    want = (w @ vv[0, -1].double()) / (w.sum() + n - 64)
    mag = (w @ vv[0, -1].double().abs()) / (w.sum() + n - 64)
    # as attention_close, and 2^-13 for the running sum of a million terms in at most 2^11 steps of 2^-24
    assert ((got[0, 0, 0].double() - want).abs() <= 2 ** -8 * want.abs() + (2 ** -8 + 2 ** -13 + 2 ** -10) * mag).all()


# ----------------------------------------------------------------- verification --

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dense", [True, False])
@pytest.mark.parametrize("B,K,V", [(1, 4, 32000), (1, 0, 17), (33, 5, 1023), (300, 3, 257), (7, 40, 4099), (2, 1, 1),
                                   (5, 7, 131072)])
def test_verify(B, K, V, dense, dtype):
    target, draft, tokens, ua, us = drafted(B, K, V, device=DEV)
    target, draft = target.to(dtype), draft.to(dtype) if dense else None
    lengths = torch.arange(B, device=DEV) % (K + 2)
    for n in (None, lengths, lengths.int() - 1):
        for got, want in zip(ops.verify_draft(target, draft, tokens, ua, us, lengths=n),
                             verify_64(target, draft, tokens, ua, us, n)):
            assert torch.equal(got.cpu(), want)


def test_verify_borders():
    """Every border of a small distribution, from both sides, and u = 1."""
    V = 5000
    p = torch.rand(1, 1, V, device=DEV)
    p[..., ::3] = 0
    p[..., -700:] = 0
    run = p.double().cumsum(-1)[0, 0]
    at = torch.randint(0, V - 1, (2000,), device=DEV)
    u = torch.cat([(run[at] / run[-1]).float(), torch.nextafter((run[at] / run[-1]).float(), torch.tensor(0.0, device=DEV)),
                   torch.tensor([0.0, 1.0], device=DEV)])
    B = u.shape[0]
    none = torch.zeros(B, 0, device=DEV)
    got, _ = ops.verify_draft(p.expand(B, 1, V), None, none.long(), none, u)
    want, _ = verify_64(p.expand(B, 1, V), None, none.long(), none, u, None)
    assert torch.equal(got.cpu(), want)


def test_verify_special_rows():
    V = 3001
    target, draft, tokens, ua, us = drafted(6, 2, V, device=DEV)
    target[0] = 0                                     # no weight anywhere
    target[1, 0] = draft[1, 0]                        # nothing left of p - q
    ua[1, 0] = 1.0
    target[2, :, 100] = float("nan")                  # counts nothing
    tokens[2, 0] = 100
    tokens[3, 0], tokens[4, 1] = -1, V                # outside the vocabulary
    target[5, 0] = 0
    target[5, 0, V - 1] = 1.0
    for q in (draft, None):
        for got, want in zip(ops.verify_draft(target, q, tokens, ua, us), verify_64(target, q, tokens, ua, us, None)):
            assert torch.equal(got.cpu(), want)


def test_verify_strides():
    target, draft, tokens, ua, us = drafted(5, 3, 1000, device=DEV)
    want = ops.verify_draft(target, draft, tokens, ua, us)
    wide = torch.full((5, 5, 1003), float("nan"), device=DEV)
    wide[:, :4, 1:1001] = target
    back = draft.flip(2).flip(2).transpose(1, 2).contiguous().transpose(1, 2)
    got = ops.verify_draft(wide[:, :4, 1:1001], back, tokens.t().contiguous().t(), ua.t().contiguous().t(), us)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_verify_many_rows():
    B = 70000
    p = torch.rand(B, 1, 3, device=DEV)
    none, us = torch.zeros(B, 0, device=DEV), torch.rand(B, device=DEV)
    run = p[:, 0].double().cumsum(-1)
    want = (run > us.double()[:, None] * run[:, -1:]).int().argmax(1)
    assert torch.equal(ops.verify_draft(p, None, none.long(), none, us)[0][:, 0], want)


def test_verify_empty_batch():
    out, acc = ops.verify_draft(torch.empty(0, 4, 10, device=DEV), None, torch.empty(0, 3, device=DEV).long(),
                                torch.empty(0, 3, device=DEV), torch.empty(0, device=DEV))
    assert out.shape == (0, 4) and acc.shape == (0,)


@pytest.mark.parametrize("refusals", [rotary_refusals, cache_refusals, verify_refusals])
def test_refusals(refusals):
    refusals(DEV)


# --------------------------------------------------------------------- together --

def _chain(q, k, v, pos, inv, cache, lengths, start, head, u, us):
    """Rotate, append, attend, project to probabilities, verify."""
    yq, yk = ops.rotary(q, k, pos, inv, layout="half")
    ops.int4_append(cache, yk.transpose(1, 2), v.transpose(1, 2), start)
    o = ops.int4_attention(yq.transpose(1, 2), cache, lengths)
    p = torch.softmax(o.transpose(1, 2).flatten(2).float() @ head, -1)
    tokens = p[:, :-1].argmax(-1)
    return ops.verify_draft(p, None, tokens, u, us) + (o,)


def _chain_inputs(seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, L, H, Hk, D, V = 3, 4, 8, 2, 64, 517
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    cache = ops.Int4KV.empty(B, Hk, 200, D, device=DEV)
    ops.int4_append(cache, r(B, Hk, 208, D).bfloat16(), r(B, Hk, 208, D).bfloat16(), 0)
    start = torch.tensor([0, 77, 190], device=DEV)
    return dict(q=r(B, L, H, D).bfloat16(), k=r(B, L, Hk, D).bfloat16(), v=r(B, L, Hk, D).bfloat16(),
                pos=start[:, None] + torch.arange(L, device=DEV), inv=frequencies(D).to(DEV), cache=cache,
                lengths=start + L, start=start, head=0.2 * r(H * D, V),
                u=torch.rand(B, L - 1, generator=g, device=DEV), us=torch.rand(B, generator=g, device=DEV))


def test_together():
    a = _chain_inputs()
    out, acc, o = _chain(**a)
    yq, yk = ops.rotary(a["q"].cpu(), a["k"].cpu(), a["pos"].cpu(), a["inv"].cpu(), layout="half")
    cpu = ops.Int4KV(*(t.cpu() for t in a["cache"].tensors()))
    kept = [t.clone() for t in cpu.tensors()]
    attention_close(ops.rotary(a["q"], a["k"], a["pos"], a["inv"], layout="half")[0].transpose(1, 2), a["cache"],
                    a["lengths"], o)
    ops.int4_append(cpu, ops.rotary(a["q"], a["k"], a["pos"], a["inv"], layout="half")[1].transpose(1, 2).cpu(),
                    a["v"].transpose(1, 2).cpu(), a["start"].cpu())
    assert all(torch.equal(x, y) for x, y in zip(kept, cpu.tensors()))         # the GPU wrote what the CPU writes
    p = torch.softmax(o.transpose(1, 2).flatten(2).float() @ a["head"], -1)
    want = verify_64(p, None, p[:, :-1].argmax(-1), a["u"], a["us"], None)
    assert torch.equal(out.cpu(), want[0]) and torch.equal(acc.cpu(), want[1])


def test_together_on_a_side_stream_and_in_a_graph():
    a = _chain_inputs()
    want = _chain(**a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _chain(**a)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graphs = []
    for _ in range(2):                                # two captured chains over the same cache
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _chain(**a)
        graphs.append((g, out))
    b = _chain_inputs(1)
    expect = _chain(**b)
    for n in ("q", "k", "v", "pos", "lengths", "start", "head", "u", "us"):
        a[n].copy_(b[n])
    for x, y in zip(a["cache"].tensors(), _chain_inputs(1)["cache"].tensors()):
        x.copy_(y)
    for g, out in graphs + graphs[:1]:
        for t in out:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, expect))


def test_two_streams_at_once():
    """Attention and verification on two streams whose work overlaps; each has its own scratch."""
    a, b = _chain_inputs(2), _chain_inputs(3)
    big = filled(2, 4, 20000, 128, 128)
    q = torch.randn(2, 8, 1, 128, device=DEV).bfloat16()
    want = [_chain(**a), _chain(**b), ops.int4_attention(q, big, 20000)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [None] * 3
    for _ in range(5):
        for i, run in enumerate((lambda: _chain(**a), lambda: _chain(**b), lambda: ops.int4_attention(q, big, 20000))):
            with torch.cuda.stream(streams[i]):
                got[i] = run()
    torch.cuda.synchronize()
    for x, y in zip(got[0] + got[1] + (got[2],), want[0] + want[1] + (want[2],)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("B,H,Hk,Lq,T,D", [(1, 4, 4, 200, 700, 128), (2, 4, 2, 150, 3000, 64), (1, 2, 2, 130, 130, 64)])
def test_attention_many_queries(B, H, Hk, Lq, T, D):
    """Long blocks of queries, which may be served from unpacked values, and the same with lengths on the GPU."""
    c = filled(B, Hk, T, D, D)
    q = (2 * torch.randn(B, H, Lq, D, device=DEV)).bfloat16()
    n = torch.full((B,), T, device=DEV)
    for causal in (True, False):
        attention_close(q, c, n, ops.int4_attention(q, c, T, causal=causal), causal)
        attention_close(q, c, n, ops.int4_attention(q, c, n, causal=causal), causal)


def test_attention_unpacked_first_equals_the_kernel():
    """Enough queries over enough tokens that the values are unpacked first (two orders of summation of one result)."""
    c = filled(1, 8, 4096, 128, 128)
    q = torch.randn(1, 8, 1024, 128, device=DEV).bfloat16()
    a = ops.int4_attention(q, c, 4096).double()
    b = ops.int4_attention(q, c, torch.full((1,), 4096, device=DEV)).double()
    k, v = ops.int4_read(c, 0, 4096)
    s = (q.double() @ k.double().transpose(-1, -2) / 128 ** 0.5)
    s = s.masked_fill(torch.ones(1024, 4096, dtype=torch.bool, device=DEV).triu(4096 - 1024 + 1), float("-inf"))
    p = torch.softmax(s, -1)
    want, mag = p @ v.double(), p @ v.double().abs()
    for x in (a, b):      # output and probabilities to bf16, scores as in attention_close, the exponential's fit to 7.5e-5
        assert ((x - want).abs() <= 2 ** -8 * want.abs() + (2 ** -8 + 2e-4 + 2 ** -9) * mag).all()


def test_attention_broadcast_queries_unpacked_first():
    c = filled(1, 8, 4096, 128, 128)
    q = torch.randn(1, 1, 1, 128, device=DEV).bfloat16().expand(1, 8, 1024, 128)
    assert torch.equal(ops.int4_attention(q, c, 4096), ops.int4_attention(q.contiguous(), c, 4096))


def test_rope_frequencies_first_used_in_inference_mode():
    from vagus_b200.models.rope import RoPE
    rope = RoPE(64, 64, 32, layout="half").to(DEV)
    x = torch.randn(1, 5, 1, 64, device=DEV)
    with torch.inference_mode():
        y = rope.rotate(x, None)
    x.requires_grad_()
    z = rope.rotate(x, None)
    assert torch.equal(y, z.detach())
    z.square().sum().backward()                   # a rotation keeps the length: the gradient of its square is 2 x
    assert (x.grad - 2 * x).abs().max() <= 2 * 2 * 8e-7 * 2 * x.detach().abs().max()


def test_rotary_backward_in_a_graph():
    inv = frequencies(64).to(DEV)
    q = torch.randn(2, 9, 4, 64, device=DEV).bfloat16().requires_grad_()
    g0 = torch.randn(2, 9, 4, 64, device=DEV).bfloat16()

    def step():
        return torch.autograd.grad(ops.rotary(q, None, 3, inv), q, g0)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    g0.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, -want)
