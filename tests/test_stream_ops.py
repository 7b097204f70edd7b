"""The long-context streaming operators on the CPU: their plain forms against the
definitions in 64 bits, and every refusal of their entry points."""

import math

import pytest
import torch

from vagus_b200 import ops

LAYOUTS = ("interleaved", "half")


def rotary_64(x, pos, inv, layout, scale):
    """The definition as complex products: (B, L, H, D) float64."""
    R = 2 * inv.shape[0]
    turn = torch.polar(torch.full_like(inv, scale).expand(*pos.shape, -1).contiguous(), pos.double()[..., None] * inv)
    h = x.double()
    pick = (slice(0, R, 2), slice(1, R, 2)) if layout == "interleaved" else (slice(0, R // 2), slice(R // 2, R))
    z = torch.complex(h[..., pick[0]].contiguous(), h[..., pick[1]].contiguous()) * turn[:, :, None]
    y = h.clone()
    y[..., pick[0]], y[..., pick[1]] = z.real, z.imag
    return y


def frequencies(R):
    return 10000.0 ** (-torch.arange(R // 2, dtype=torch.float64) / (R // 2))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("D,R", [(8, 8), (16, 6), (64, 32), (10, 2)])
def test_rotary_matches_the_definition(layout, D, R):
    torch.manual_seed(0)
    q, k = torch.randn(2, 5, 3, D), torch.randn(2, 5, 1, D)
    inv = frequencies(R)
    for pos in (0, 7, torch.arange(5) + 3, torch.randint(0, 1 << 20, (2, 5)), torch.tensor([[9, 0, 9, 1, 2]] * 2).int()):
        yq, yk = ops.rotary(q, k, pos, inv, layout=layout, scale=1.25)
        at = (pos + torch.arange(5)).expand(2, 5) if isinstance(pos, int) else pos.expand(2, 5)
        for x, y in ((q, yq), (k, yk)):
            # fp32 products of fp32 cosines: three roundings of at most 2^-24 a term
            assert (y - rotary_64(x, at, inv, layout, 1.25)).abs().max() < 8 * 2 ** -24 * 1.25 * x.abs().max()
            assert torch.equal(y[..., R:], x[..., R:])
    assert torch.equal(ops.rotary(q, None, 7, inv, layout=layout), ops.rotary(q, k, 7, inv, layout=layout)[0])


@pytest.mark.parametrize("layout", LAYOUTS)
def test_rotary_gradient_against_differences(layout):
    torch.manual_seed(0)
    q, k = (torch.randn(1, 3, h, 8, dtype=torch.float64, requires_grad=True) for h in (2, 1))
    assert torch.autograd.gradcheck(lambda a, b: ops.rotary(a, b, 5, frequencies(6), layout=layout, scale=0.7), (q, k))


def rotary_refusals(device):
    q, k, inv = (t.to(device) for t in (torch.randn(2, 3, 4, 8), torch.randn(2, 3, 2, 8), frequencies(8)))
    bad = [dict(layout="pairs"), dict(q=q[0]), dict(k=k[:, :2]), dict(k=k[..., :6]), dict(k=k.double()),
           dict(inv=frequencies(10).to(device)), dict(inv=inv[:0]), dict(inv=inv.long()), dict(inv=inv[None]),
           dict(inv=inv.to("meta")), dict(k=k.to("meta")),
           dict(pos=torch.arange(4, device=device)), dict(pos=torch.arange(3, device=device).float()),
           dict(pos=torch.zeros(3, 2, device=device).long()), dict(pos=torch.zeros(3, device="meta").long()), dict(pos=1.5)]
    for b in bad:
        a = dict(q=q, k=k, pos=0, inv=inv, layout="half")
        a.update(b)
        with pytest.raises(ValueError):
            ops.rotary(a["q"], a["k"], a["pos"], a["inv"], layout=a["layout"])


def test_rotary_refusals():
    rotary_refusals("cpu")


# ------------------------------------------------------------------ 4-bit cache --

def held_64(x):
    """What a group of 32 stands for after quantisation, from the definition."""
    g = x.double().reshape(-1, 32)
    out = torch.empty_like(g)
    for r in range(g.shape[0]):
        lo, hi = g[r].min(), g[r].max()
        s = ((hi - lo) / 15).float().bfloat16().double()
        b = (lo - 128 * s).float().bfloat16().double()
        c = torch.round((g[r] - b) / s).clamp(128, 143) if s > 0 else torch.full((32,), 128.0, dtype=torch.float64)
        out[r] = c * s + b
    return out.reshape(x.shape).float().bfloat16()


@pytest.mark.parametrize("scale,offset", [(1.0, 0.0), (1e-3, 5.0), (300.0, -40.0), (1e-30, 0.0), (1e30, 0.0)])
def test_cache_round_trip_is_within_half_a_step(scale, offset):
    torch.manual_seed(0)
    k = (torch.randn(2, 3, 5, 64) * scale + offset).bfloat16()
    v = (torch.randn(2, 3, 5, 32) * scale + offset).bfloat16()
    c = ops.Int4KV.empty(2, 3, 20, 64, 32)
    assert c.capacity == 32 and (c.batch, c.kv_heads, c.head_dim, c.value_dim) == (2, 3, 64, 32)
    ops.int4_append(c, k, v, 4)
    for x, y in zip((k, v), ops.int4_read(c, 4, 5)):
        assert torch.equal(y, held_64(x))
        g, h = x.double().reshape(-1, 32), y.double().reshape(-1, 32)
        lo, hi = g.amin(1, keepdim=True), g.amax(1, keepdim=True)
        # s and b each round by 2^-8 relative (|b| <= 128 s + |lo|), the value by 2^-8 once more
        s = (hi - lo) / 15 * (1 + 2 ** -8)
        b = 2 ** -8 * (128 * s + lo.abs())
        assert ((h - g).abs() <= torch.maximum(0.5 * s, b + 15 * 2 ** -8 * s) * 1.001 + 2 ** -8 * h.abs()).all()


def test_cache_special_groups():
    k = torch.zeros(1, 1, 4, 64)
    k[0, 0, 0] = 3.140625                       # equal values: exact
    k[0, 0, 1, 5] = float("nan")
    k[0, 0, 2, 40] = float("inf")
    k[0, 0, 3, :32] = torch.arange(32).float() % 16
    c = ops.Int4KV.empty(1, 1, 16, 64)
    ops.int4_append(c, k, k, 0)
    y, _ = ops.int4_read(c, 0, 4)
    assert torch.equal(y[0, 0, 0].float(), k[0, 0, 0])
    assert y[0, 0, 1, :32].isnan().all() and (y[0, 0, 1, 32:] == 0).all()
    assert y[0, 0, 2, 32:].isnan().all() and (y[0, 0, 2, :32] == 0).all()
    assert torch.equal(y[0, 0, 3].float(), k[0, 0, 3])


def test_append_per_sequence_leaves_the_rest():
    torch.manual_seed(0)
    c = ops.Int4KV.empty(3, 2, 16, 32)
    before = [t.clone() for t in c.tensors()]
    k, v = torch.randn(3, 2, 2, 32), torch.randn(3, 2, 2, 32)
    start = torch.tensor([0, 14, 5])
    ops.int4_append(c, k, v, start)
    for b in range(3):
        t = int(start[b])
        one = ops.Int4KV.empty(1, 2, 16, 32)
        ops.int4_append(one, k[b:b + 1], v[b:b + 1], 0)
        for have, old, want in zip(c.tensors(), before, one.tensors()):
            assert torch.equal(have[b, :, t:t + 2], want[0, :, :2])
            rest = torch.ones(16, dtype=torch.bool)
            rest[t:t + 2] = False
            assert torch.equal(have[b][:, rest], old[b][:, rest])
    assert all(torch.equal(a, b) for a, b in zip(ops.int4_read(c, start, 2), ops.int4_read(c, start.int(), 2)))


def attention_64(q, k, v, lengths, causal):
    """The definition, row by row: float64 result and sum of p |v|."""
    B, H, Lq, D = q.shape
    G = H // k.shape[1]
    out = torch.zeros(B, H, Lq, v.shape[3], dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for b in range(B):
        n = int(lengths[b])
        for i in range(Lq):
            m = max(0, n - Lq + 1 + i) if causal else n
            if m == 0:
                continue
            kk = k[b, :, :m].double().repeat_interleave(G, 0)
            vv = v[b, :, :m].double().repeat_interleave(G, 0)
            s = (kk @ q[b, :, i].double()[..., None])[..., 0] / math.sqrt(D)
            p = torch.softmax(s, -1)
            out[b, :, i] = (p[:, None] @ vv)[:, 0]
            mag[b, :, i] = (p[:, None] @ vv.abs())[:, 0]
    return out, mag


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hk,Lq", [(2, 2, 1), (4, 1, 3), (6, 2, 5)])
def test_attention_plain_form(H, Hk, Lq, causal):
    torch.manual_seed(0)
    c = ops.Int4KV.empty(4, Hk, 32, 32, 64)
    k, v = torch.randn(4, Hk, 32, 32), torch.randn(4, Hk, 32, 64)
    v[2, :, 20:] = float("nan")                       # past a length: of no effect
    k[2, :, 20:] = float("inf")
    ops.int4_append(c, k, v, 0)
    k, v = ops.int4_read(c, 0, 32)
    q = torch.randn(4, H, Lq, 32)
    lengths = torch.tensor([0, 1, 20, 32])
    got = ops.int4_attention(q, c, lengths, causal=causal)
    want, _ = attention_64(q, k, v, lengths, causal)
    assert (got - want).abs().max() < 1e-5            # fp32 over at most 32 tokens of values near 1
    assert (got[0] == 0).all() and got.dtype == q.dtype
    same = ops.int4_attention(q[2:3], ops.Int4KV(*(t[2:3].contiguous() for t in c.tensors())), 20, causal=causal)
    assert torch.allclose(same, got[2:3], atol=1e-6)


def cache_refusals(device):
    """On the GPU a place given there is checked by the kernel and does not raise here."""
    def make(*a):
        return ops.Int4KV.empty(*a, device=device)
    here = device == "cpu"

    def randn(*s):
        return torch.randn(*s, device=device)

    def places(*x):
        return torch.tensor(x, device=device)
    for a in ((1, 1, 16, 48), (1, 1, 16, 0), (1, 1, 16, 64, 40)):
        with pytest.raises(ValueError):
            make(*a)
    c = make(2, 2, 16, 64, 32)
    kc, kp, vc, vp = c.tensors()
    for t in ([x[:, :, :8].contiguous() for x in c.tensors()], (kc.to(torch.int8), kp, vc, vp), (kc, kp.float(), vc, vp),
              (kc, vp, vc, vp), (kc[:1], kp[:1], vc, vp), (kc.transpose(2, 3), kp, vc, vp),
              (kc[..., :20].contiguous(), kp, vc, vp), (kc, kp.flatten(3), vc, vp), (kc, kp, vc.to("meta"), vp)):
        with pytest.raises(ValueError):
            ops.Int4KV(*t)
    k, v = randn(2, 2, 3, 64), randn(2, 2, 3, 32)
    bad = [(k, v, 14), (k, v, -1), (k[:1], v, 0), (k, v[..., :16], 0), (k[:, :, :2], v, 0), (k.double(), v, 0),
           (k, v, places(0)), (k, v, places(0.0, 1.0)), (k, v, 1.0), (k, v, None), (k[0], v, 0), (k.to("meta"), v, 0)]
    if here:
        bad += [(k, v, places(0, 14)), (k, v, places(-1, 0))]
    else:
        bad += [(k.double(), v.double(), 0), (k, v, torch.tensor([0, 1]))]
    for a in bad:
        with pytest.raises(ValueError):
            ops.int4_append(c, *a)
    for a in ((0, 17), (-1, 2), (0, -1), (places(0, 1, 2), 2)) + (((places(0, 15), 2),) if here else ()):
        with pytest.raises(ValueError):
            ops.int4_read(c, *a)
    assert all((t == 0).all() for t in c.tensors())
    q = randn(2, 4, 1, 64).bfloat16()
    bad = [(q, c, 17), (q, c, -1), (q[:1], c, 4), (q[:, :3], c, 4), (q[..., :32], c, 4), (q[0], c, 4),
           (q, c, places(4, 4, 4)), (q, c, None), (q.to("meta"), c, 4)]
    for a in bad + ([(q, c, places(4, 17))] if here else []):
        with pytest.raises(ValueError):
            ops.int4_attention(*a)


def test_cache_refusals():
    cache_refusals("cpu")


# ----------------------------------------------------------------- verification --

def verify_64(target, draft, tokens, u_accept, u_sample, lengths):
    """The definition, one row at a time."""
    B, K = tokens.shape
    out = torch.full((B, K + 1), -1, dtype=torch.int64)
    acc = torch.zeros(B, dtype=torch.int64)
    target, tokens, u_accept, u_sample = (t.cpu() for t in (target, tokens, u_accept, u_sample))
    draft = None if draft is None else draft.cpu()
    for b in range(B):
        many = K if lengths is None else min(K, max(0, int(lengths[b])))
        n = 0
        while n < many:
            d = int(tokens[b, n])
            if not 0 <= d < target.shape[2]:
                break
            q = torch.tensor(1.0) if draft is None else draft[b, n, d].float()
            if not bool(u_accept[b, n] * q < target[b, n, d].float()):
                break
            n += 1
        p = target[b, n].float()
        w = p.clone()
        if n < many:
            if draft is not None:
                w = p - draft[b, n].float()
            elif 0 <= int(tokens[b, n]) < p.shape[0]:
                w[int(tokens[b, n])] = 0
            if not bool((w > 0).any()):
                w = p
        w = torch.where(w > 0, w, torch.zeros(())).double()
        run = torch.cumsum(w, 0)
        some = torch.nonzero(w > 0)
        over = torch.nonzero((run > float(u_sample[b]) * run[-1]) & (w > 0))
        out[b, :n] = tokens[b, :n]
        out[b, n] = int(over[0]) if len(over) else int(some[-1]) if len(some) else 0
        acc[b] = n
    return out, acc


def drafted(B, K, V, seed=0, spread=0.5, device="cpu"):
    """Target and draft probabilities that agree to a degree, drafts drawn from the draft's."""
    g = torch.Generator(device=device).manual_seed(seed)
    logits = 2 * torch.randn(B, K + 1, V, generator=g, device=device)
    target = torch.softmax(logits, -1)
    draft = torch.softmax(logits[:, :K] + spread * torch.randn(B, K, V, generator=g, device=device), -1)
    tokens = torch.multinomial(draft.reshape(B * K, V), 1, generator=g).view(B, K) if K else \
        torch.zeros(B, 0, dtype=torch.int64, device=device)
    return (target, draft, tokens, torch.rand(B, K, generator=g, device=device),
            torch.rand(B, generator=g, device=device))


@pytest.mark.parametrize("dense", [True, False])
@pytest.mark.parametrize("K,V", [(0, 5), (1, 3), (4, 50), (9, 7)])
def test_verify_plain_form(K, V, dense):
    target, draft, tokens, ua, us = drafted(40, K, V)
    draft = draft if dense else None
    lengths = torch.arange(40) % (K + 2) - 0
    for n in (None, lengths, lengths.int()):
        for got, want in zip(ops.verify_draft(target, draft, tokens, ua, us, lengths=n),
                             verify_64(target, draft, tokens, ua, us, n)):
            assert torch.equal(got, want)


def test_verify_keeps_the_target_distribution():
    """Over a fine grid of both random numbers the first token's frequencies are p."""
    p = torch.tensor([0.5, 0.2, 0.2, 0.1])
    q = torch.tensor([0.1, 0.6, 0.25, 0.05])
    N = 400
    u = (torch.arange(N) + 0.5) / N
    freq = torch.zeros(4)
    for d in range(4):
        ua, us = u.repeat_interleave(N)[:, None], u.repeat(N)
        B = N * N
        out, _ = ops.verify_draft(torch.stack([p, p]).expand(B, 2, 4), q.expand(B, 1, 4),
                                  torch.full((B, 1), d), ua, us)
        freq += q[d] * torch.bincount(out[:, 0], minlength=4) / B
    # the grid resolves each border to 1 / N, twice
    assert (freq - p).abs().max() < 2 / N


def test_verify_special_rows():
    V = 6
    one = torch.zeros(1, 2, V)
    one[:, :, 2] = 1.0
    u0, u1 = torch.zeros(1, 1), torch.zeros(1)
    # greedy target: the draft that agrees is accepted, the other replaced
    assert ops.verify_draft(one, None, torch.tensor([[2]]), u0, u1)[0].tolist() == [[2, 2]]
    assert ops.verify_draft(one, None, torch.tensor([[4]]), u0, u1)[0].tolist() == [[2, -1]]
    # equal probabilities and u = 1 (outside the range) reject; nothing is left of p - q: drawn from p
    half = torch.tensor([[[0.5, 0.5]] * 2])
    out, acc = ops.verify_draft(half, half[:, :1], torch.tensor([[0]]), torch.ones(1, 1), torch.tensor([0.75]))
    assert out.tolist() == [[1, -1]] and acc.tolist() == [0]
    # u_sample = 1: the last token with any weight; no weight at all: token 0
    w = torch.tensor([[[0.0, 0.3, 0.7, 0.0]]])
    none = torch.zeros(1, 0, dtype=torch.int64)
    assert ops.verify_draft(w, None, none, torch.zeros(1, 0), torch.ones(1))[0].tolist() == [[2]]
    assert ops.verify_draft(w * 0, None, none, torch.zeros(1, 0), torch.zeros(1))[0].tolist() == [[0]]
    # a drafted token outside the vocabulary is rejected
    for d in (-1, V):
        assert ops.verify_draft(one, None, torch.tensor([[d]]), u0, u1)[1].tolist() == [0]


def verify_refusals(device):
    target, draft, tokens, ua, us = (t.to(device) for t in drafted(2, 3, 5))
    ok = dict(target=target, draft=draft, tokens=tokens, u_accept=ua, u_sample=us, lengths=None)
    for bad in (dict(target=target[0]), dict(target=target.double()), dict(target=target[:, :3]),
                dict(draft=draft[:, :2]), dict(draft=draft.bfloat16()), dict(draft=draft[..., :4]),
                dict(tokens=tokens.int()), dict(tokens=tokens[:1]), dict(u_accept=ua[:, :2]), dict(u_accept=ua.double()),
                dict(u_sample=us[:1]), dict(u_sample=us[:, None]), dict(lengths=torch.zeros(3, device=device).long()),
                dict(lengths=torch.zeros(2, device=device)), dict(tokens=tokens.to("meta")), dict(u_sample=us.to("meta")),
                dict(draft=draft.to("meta")), dict(tokens=tokens.reshape(-1)), dict(target=target[..., :0], draft=draft[..., :0])):
        with pytest.raises(ValueError):
            ops.verify_draft(**{**ok, **bad})


def test_verify_refusals():
    verify_refusals("cpu")
