"""The operators of long-context streaming generation, as cases to measure.

Four operators that a stream's tokens pass through one after the other:

* ``rotary``   rotates queries and keys by their positions (both pair layouts, part of
               the head, per-token positions, a scale for long contexts), forward and
               backward;
* ``append``   quantises new keys and values to 4 bits and writes them into a cache;
               what was written is read back as the values it stands for;
* ``attend``   softmax attention of one or more new queries over that cache;
* ``verify``   accepts or rejects drafted tokens against the target's probabilities
               from given random numbers and draws the token that follows.

A 4-bit cache holds, for every token and KV head, one code of 4 bits a channel (channel
2 j in the low half of byte j) and, for each group of 32 channels, a step s and an
offset b in bf16; a code c stands for bf16((128 + c) s + b).

With ``own`` false ``run`` computes the plain form in elementary torch operations;
with ``own`` true it makes the calls that a user of the framework makes.
"""

import math

import torch

own = False

DEV = "cuda"
GROUP = 32
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one decode step of eight streams of the 340M Transformer++ (16 heads of 64): latency
        dict(name="rotary: one token", op="rotary", B=8, L=1, H=16, Hk=16, D=64, R=64, layout="interleaved",
             scaled=False, far=False, dtype="bf16", backward=False),
        # a training step's layer of the 1.3B hybrid's heads (16 of 128), both directions
        dict(name="rotary: training", op="rotary", B=4, L=4096, H=16, Hk=16, D=128, R=128, layout="half",
             scaled=False, far=False, dtype="bf16", backward=True),
        # packed ragged positions far out, half of the head rotated, grouped KV heads
        dict(name="rotary: partial, far", op="rotary", B=2, L=2305, H=32, Hk=8, D=128, R=64, layout="half",
             scaled=True, far=True, dtype="fp16", backward=False),
        # one decode step of 64 streams, each at its own place in the cache
        dict(name="append: one token", op="append", B=64, L=1, Hk=8, D=128, Dv=128, cap=4096, ragged=True,
             dtype="bf16"),
        # a long prompt's keys and values
        dict(name="append: prompt", op="append", B=4, L=8191, Hk=16, D=128, Dv=128, cap=8192, ragged=False,
             dtype="bf16"),
        # one stream of the 340M Transformer++, a short context: latency
        dict(name="attend: one stream", op="attend", B=1, Lq=1, T=997, H=16, Hk=16, D=64, Dv=64, ragged=False),
        # a serving batch of ragged streams, grouped heads, one of them empty
        dict(name="attend: ragged batch", op="attend", B=32, Lq=1, T=8192, H=32, Hk=8, D=128, Dv=128, ragged=True),
        # two very long streams
        dict(name="attend: long", op="attend", B=2, Lq=1, T=131067, H=16, Hk=8, D=128, Dv=128, ragged=False),
        # the pass over a block of five drafted tokens and their head
        dict(name="attend: drafted block", op="attend", B=8, Lq=6, T=4099, H=16, Hk=16, D=64, Dv=64, ragged=False),
        # a prompt's second chunk
        dict(name="attend: prompt chunk", op="attend", B=1, Lq=2048, T=8191, H=16, Hk=16, D=128, Dv=128,
             ragged=False),
        # one stream, the repository's own vocabulary: latency
        dict(name="verify: one stream", op="verify", B=1, K=4, V=32000, dtype="fp32", dense=True, ragged=False),
        # a batch with a large vocabulary
        dict(name="verify: batch", op="verify", B=64, K=7, V=131072, dtype="fp32", dense=True, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "verify"])
    if op == "rotary":
        D = rng.choice([64, 128, 256])
        Hk = rng.choice([1, 2, 8, 16])
        H = Hk * rng.choice([1, 2, 4])
        B = rng.randint(1, 8)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = 4 * 4096 * 32 * 128 // (2 if dtype == "fp32" else 1) // (B * (H + Hk) * D)
        L = _log(rng, 1, max(1, min(16384, most)))
        R = rng.choice([D, D, D // 2, D // 4])
        return dict(op=op, B=B, L=L, H=H, Hk=Hk, D=D, R=R, layout=rng.choice(["interleaved", "half"]),
                    scaled=rng.random() < 0.5, far=rng.random() < 0.5, dtype=dtype, backward=rng.random() < 0.5)
    if op == "append":
        D, Dv = rng.choice([(64, 64), (128, 128), (64, 128), (128, 64)])
        Hk = rng.choice([1, 4, 8, 16])
        B = _log(rng, 1, 64)
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        most = 4 * 8191 * 16 * 256 // (2 if dtype == "fp32" else 1) // (B * Hk * (D + Dv))
        L = _log(rng, 1, max(1, min(16384, most)))
        return dict(op=op, B=B, L=L, Hk=Hk, D=D, Dv=Dv, cap=L + rng.randint(0, 600), ragged=rng.random() < 0.5,
                    dtype=dtype)
    if op == "attend":
        D = Dv = rng.choice([64, 128])
        if rng.random() < 0.2:
            Dv = 192 - D
        Hk = rng.choice([1, 2, 4, 8, 16])
        H = Hk * rng.choice([1, 1, 2, 4, 8])
        Lq = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 2048)])
        B = _log(rng, 1, 32)
        most = min(131072, 2 * 131067 * 8 * 256 // (B * Hk * (D + Dv)), 2048 * 8191 * 16 // (B * H * Lq))
        T = max(1, _log(rng, 1, max(1, most)))
        Lq = min(Lq, T)
        return dict(op=op, B=B, Lq=Lq, T=T, H=H, Hk=Hk, D=D, Dv=Dv, ragged=Lq < 64 and rng.random() < 0.5)
    V = _log(rng, 500, 160000)
    K = rng.randint(0, 8)
    B = _log(rng, 1, max(1, min(256, 64 * 15 * 131072 // (V * (2 * K + 1)))))
    return dict(op=op, B=B, K=K, V=V, dtype=rng.choice(["fp32", "fp32", "bf16"]), dense=rng.random() < 0.7,
                ragged=rng.random() < 0.5)


# ------------------------------------------------------------------------------ inputs --

def _spread(case):
    """Lengths of a ragged batch: from nothing to T, by the case alone."""
    B, T = case["B"], case["T"]
    return [T * i // max(1, B - 1) for i in range(B)] if B > 1 else [T]


def _quantise(x):
    """Values (..., D) -> packed codes (..., D / 2) uint8 and (step, offset) (..., D / 32, 2) bf16."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi - lo) / 15).bfloat16().float()
    b = (lo - 128 * s).bfloat16().float()
    c = (torch.round((g - b) / s) - 128).clamp(0, 15)
    c = torch.where(s > 0, c, torch.zeros_like(c)).flatten(-2).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.cat([s, b], -1).bfloat16()


def _stands_for(codes, params):
    """The values (fp32, each a bf16 number) that packed codes stand for."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    s, b = params[..., :1].float(), params[..., 1:].float()
    return ((c + 128) * s + b).flatten(-2).bfloat16().float()


def _heads(shape, g, dtype=torch.bfloat16):
    """Keys or values as a model makes them: channels of unequal size and with offsets."""
    x = torch.randn(shape, generator=g, device=DEV)
    size = torch.exp(0.7 * torch.randn(shape[-1], generator=g, device=DEV))
    off = 0.5 * torch.randn(shape[-1], generator=g, device=DEV)
    return (x * size + off).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    st = dict(case=case)
    if case["op"] == "rotary":
        B, L, H, Hk, D, R = (case[n] for n in ("B", "L", "H", "Hk", "D", "R"))
        dt = TYPES[case["dtype"]]
        st["q"] = torch.randn(B, L, H, D, generator=g, device=DEV).to(dt).requires_grad_(case["backward"])
        st["k"] = torch.randn(B, L, Hk, D, generator=g, device=DEV).to(dt).requires_grad_(case["backward"])
        if case["backward"]:
            st["gq"] = torch.randn(B, L, H, D, generator=g, device=DEV).to(dt)
            st["gk"] = torch.randn(B, L, Hk, D, generator=g, device=DEV).to(dt)
        inv = torch.pow(10000.0, -torch.arange(R // 2, device=DEV, dtype=torch.float64) / (R // 2))
        st["inv"] = inv / 8 if case["scaled"] else inv
        st["scale"] = 0.1 * math.log(8.0) + 1.0 if case["scaled"] else 1.0
        if case["far"]:
            st["pos"] = torch.randint(0, 1 << 20, (B, L), generator=g, device=DEV)
        else:
            st["pos"] = 4095 if L == 1 else 0
        return st
    if case["op"] == "append":
        B, L, Hk, D, Dv, cap = (case[n] for n in ("B", "L", "Hk", "D", "Dv", "cap"))
        dt = TYPES[case["dtype"]]
        # (B, L, Hk, D) as the projections leave them, seen as (B, Hk, L, D)
        st["k"] = _heads((B, L, Hk, D), g, dt).transpose(1, 2)
        st["v"] = _heads((B, L, Hk, Dv), g, dt).transpose(1, 2)
        cap = (cap + 15) // 16 * 16
        st["cache"] = [torch.zeros(B, Hk, cap, D // 2, dtype=torch.uint8, device=DEV),
                       torch.zeros(B, Hk, cap, D // GROUP, 2, dtype=torch.bfloat16, device=DEV),
                       torch.zeros(B, Hk, cap, Dv // 2, dtype=torch.uint8, device=DEV),
                       torch.zeros(B, Hk, cap, Dv // GROUP, 2, dtype=torch.bfloat16, device=DEV)]
        st["start"] = torch.randint(0, cap - L + 1, (B,), generator=g, device=DEV) if case["ragged"] else 0
        return st
    if case["op"] == "attend":
        B, Lq, T, H, Hk, D, Dv = (case[n] for n in ("B", "Lq", "T", "H", "Hk", "D", "Dv"))
        st["q"] = torch.randn(B, Lq, H, D, generator=g, device=DEV).bfloat16().transpose(1, 2)
        cap = (T + 15) // 16 * 16
        ck, pk = zip(*[_quantise(_heads((Hk, cap, D), g)) for _ in range(B)])
        cv, pv = zip(*[_quantise(_heads((Hk, cap, Dv), g)) for _ in range(B)])
        st["cache"] = [torch.stack(t) for t in (ck, pk, cv, pv)]
        if case["ragged"]:
            order = torch.randperm(B, generator=g, device=DEV)
            st["lengths"] = torch.tensor(_spread(case), device=DEV, dtype=torch.int32)[order]
        else:
            st["lengths"] = T
        return st
    B, K, V = case["B"], case["K"], case["V"]
    dt = TYPES[case["dtype"]]
    logits = 3 * torch.randn(B, K + 1, V, generator=g, device=DEV)
    st["target"] = torch.softmax(logits, -1).to(dt)
    guess = torch.softmax(logits[:, :K] + 0.5 * torch.randn(B, K, V, generator=g, device=DEV), -1)
    if case["dense"]:
        st["draft"] = guess.to(dt)
        st["tokens"] = torch.multinomial(guess.reshape(B * K, V), 1, generator=g).view(B, K) if K else \
            torch.zeros(B, 0, dtype=torch.int64, device=DEV)
    else:
        st["draft"] = None
        st["tokens"] = guess.argmax(-1) if K else torch.zeros(B, 0, dtype=torch.int64, device=DEV)
    st["u_accept"] = torch.rand(B, K, generator=g, device=DEV)
    st["u_sample"] = torch.rand(B, generator=g, device=DEV)
    st["lengths"] = torch.randint(0, K + 1, (B,), generator=g, device=DEV) if case["ragged"] else None
    return st


# ------------------------------------------------------------------------------- plain --

def _angles(st):
    q = st["q"]
    pos = st["pos"]
    if isinstance(pos, int):
        pos = (pos + torch.arange(q.shape[1], device=DEV)).expand(q.shape[0], -1)
    ang = pos.double()[..., None] * st["inv"]
    return (torch.cos(ang) * st["scale"]).float()[:, :, None], (torch.sin(ang) * st["scale"]).float()[:, :, None]


def _rotate(x, cos, sin, layout):
    R = 2 * cos.shape[-1]
    h = x[..., :R].float()
    if layout == "interleaved":
        a, b = h[..., 0::2], h[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = h[..., :R // 2], h[..., R // 2:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y.to(x.dtype), x[..., R:]], -1)


def _plain_rotary(st):
    lay = st["case"]["layout"]
    cos, sin = _angles(st)
    out = {"q": _rotate(st["q"].detach(), cos, sin, lay), "k": _rotate(st["k"].detach(), cos, sin, lay)}
    if st["case"]["backward"]:
        out["dq"], out["dk"] = _rotate(st["gq"], cos, -sin, lay), _rotate(st["gk"], cos, -sin, lay)
    return out


def _plain_append(st):
    L, start = st["case"]["L"], st["start"]
    B, Hk = st["k"].shape[:2]
    at = start if isinstance(start, torch.Tensor) else torch.full((B,), start, device=DEV)
    i = torch.arange(B, device=DEV)[:, None, None]
    j = torch.arange(Hk, device=DEV)[None, :, None]
    t = at[:, None, None] + torch.arange(L, device=DEV)
    new = _quantise(st["k"]) + _quantise(st["v"])
    for have, x in zip(st["cache"], new):
        have[i, j, t] = x
    kc, kp, vc, vp = (have[i, j, t] for have in st["cache"])
    return {"k": _stands_for(kc, kp).bfloat16(), "v": _stands_for(vc, vp).bfloat16()}


def _plain_attend(st):
    q, T = st["q"], st["case"]["T"]
    B, H, Lq, D = q.shape
    Hk = st["case"]["Hk"]
    k = _stands_for(st["cache"][0][:, :, :T], st["cache"][1][:, :, :T])
    s = (q.float().reshape(B, Hk, H // Hk * Lq, D) @ k.transpose(-1, -2)).view(B, Hk, H // Hk, Lq, T)
    s = s * (1 / math.sqrt(D))
    del k
    n = st["lengths"] if isinstance(st["lengths"], torch.Tensor) else torch.full((B,), T, device=DEV)
    seen = (n[:, None] - Lq + 1 + torch.arange(Lq, device=DEV))[:, None, None, :, None]
    hidden = torch.arange(T, device=DEV) >= seen
    s = s.masked_fill_(hidden, float("-inf"))
    s = s - s.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp_(s)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    v = _stands_for(st["cache"][2][:, :, :T], st["cache"][3][:, :, :T])
    return (p.view(B, Hk, H // Hk * Lq, T) @ v).view(B, H, Lq, -1).bfloat16()


def _plain_verify(st):
    p, q, tok = st["target"], st["draft"], st["tokens"]
    B, K = tok.shape
    pt = p[:, :K].float().gather(2, tok[..., None])[..., 0]
    qt = torch.ones_like(pt) if q is None else q.float().gather(2, tok[..., None])[..., 0]
    n = torch.full((B,), K, device=DEV) if st["lengths"] is None else st["lengths"]
    step = torch.arange(K, device=DEV)
    ok = (st["u_accept"] * qt < pt) & (step < n[:, None])
    acc = ok.long().cumprod(1).sum(1)
    row = torch.arange(B, device=DEV)
    last = p[row, acc].float()
    w = last
    if K:
        at = acc.clamp(max=K - 1)
        if q is None:
            rest = last.scatter(1, tok[row, at][:, None], 0.0)
        else:
            rest = (last - q[row, at].float()).clamp(min=0)
        rest = torch.where((rest > 0).any(1, keepdim=True), rest, last)
        w = torch.where((acc < n)[:, None], rest, last)
    c = w.double().cumsum(1)
    over = c > st["u_sample"].double()[:, None] * c[:, -1:]
    new = over.int().argmax(1)
    out = torch.cat([tok, tok.new_zeros(B, 1)], 1)
    place = torch.arange(K + 1, device=DEV)
    out = torch.where(place < acc[:, None], out, torch.where(place == acc[:, None], new[:, None], -1))
    return {"tokens": out, "accepted": acc}


# --------------------------------------------------------------------------------- own --

def _own(st):
    from vagus_b200 import ops
    case = st["case"]
    if case["op"] == "rotary":
        q, k = ops.rotary(st["q"], st["k"], st["pos"], st["inv"], layout=case["layout"], scale=st["scale"])
        out = {"q": q.detach(), "k": k.detach()}
        if case["backward"]:
            out["dq"], out["dk"] = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["gq"], st["gk"]))
        return out
    if case["op"] == "append":
        cache = ops.Int4KV(*st["cache"])
        ops.int4_append(cache, st["k"], st["v"], st["start"])
        k, v = ops.int4_read(cache, st["start"], case["L"])
        return {"k": k, "v": v}
    if case["op"] == "attend":
        return ops.int4_attention(st["q"], ops.Int4KV(*st["cache"]), st["lengths"])
    tokens, accepted = ops.verify_draft(st["target"], st["draft"], st["tokens"], st["u_accept"], st["u_sample"],
                                        lengths=st["lengths"])
    return {"tokens": tokens, "accepted": accepted}


def run(state):
    if own:
        return _own(state)
    return {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend,
            "verify": _plain_verify}[state["case"]["op"]](state)


# -------------------------------------------------------------------------------- work --

def work(case):
    if case["op"] == "rotary":
        es = 4 if case["dtype"] == "fp32" else 2
        n = case["B"] * case["L"] * (case["H"] + case["Hk"])
        ways = 2 if case["backward"] else 1
        return {"bytes": ways * 2 * es * n * case["D"], "flops": ways * 3 * n * case["R"]}
    if case["op"] == "append":
        es = 4 if case["dtype"] == "fp32" else 2
        n = case["B"] * case["L"] * case["Hk"] * (case["D"] + case["Dv"])
        # read once, codes and parameters written and read back, values written
        return {"bytes": n * (es + 2 * (0.5 + 4 / GROUP) + 2), "flops": 8 * n}
    if case["op"] == "attend":
        B, Lq, T, H, Hk, D, Dv = (case[n] for n in ("B", "Lq", "T", "H", "Hk", "D", "Dv"))
        lens = _spread(case) if case["ragged"] else [T] * B
        pairs = sum(max(0, n - Lq + 1 + i) for n in lens for i in range(Lq))
        return {"bytes": sum(lens) * Hk * (D + Dv) * (0.5 + 4 / GROUP) + 2 * B * H * Lq * (D + Dv),
                "flops": 2 * H * pairs * (D + Dv)}
    # the row of the target at the first rejected place and, where there is one, the draft's
    es = 4 if case["dtype"] == "fp32" else 2
    rows = 2 if case["dense"] and case["K"] else 1
    return {"bytes": case["B"] * (case["V"] * es * rows + case["K"] * (12 + 2 * es)), "flops": case["B"] * case["V"] * 3}


# ------------------------------------------------------------------------------- exact --

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rotary":
        B, L, R = case["B"], case["L"], case["R"]
        pos = st["pos"] if case["far"] else st["pos"] + torch.arange(L, device=DEV).repeat(B, 1)
        turn = torch.polar(torch.full((B, L, 1, R // 2), st["scale"], dtype=torch.float64, device=DEV),
                           (pos.double().view(B, L, 1, 1) * st["inv"]))

        def rot(x, by):
            h = x.detach().double()
            if case["layout"] == "interleaved":
                z = torch.view_as_complex(h[..., :R].reshape(*h.shape[:-1], R // 2, 2).contiguous()) * by
                y = torch.view_as_real(z).reshape(*h.shape[:-1], R)
            else:
                z = torch.complex(h[..., :R // 2].contiguous(), h[..., R // 2:R].contiguous()) * by
                y = torch.cat([z.real, z.imag], -1)
            return torch.cat([y, h[..., R:]], -1)

        out = {"q": rot(st["q"], turn), "k": rot(st["k"], turn)}
        if case["backward"]:
            out["dq"], out["dk"] = rot(st["gq"], turn.conj()), rot(st["gk"], turn.conj())
        return out
    if case["op"] == "append":
        def held(x):
            g = x.double().reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
            lo = g.min(-1, keepdim=True).values
            s = ((g.max(-1, keepdim=True).values - lo) / 15).float().bfloat16().double()
            b = (lo - 128 * s).float().bfloat16().double()
            level = torch.round((g - b) / s).clamp(128, 143)
            return (level * s + b).reshape(x.shape)
        return {"k": held(st["k"]), "v": held(st["v"])}
    if case["op"] == "attend":
        B, Lq, T, H, Hk, D, Dv = (case[n] for n in ("B", "Lq", "T", "H", "Hk", "D", "Dv"))

        def value(codes, params):
            x = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=DEV)
            x[..., 0::2] = (codes % 16).double()
            x[..., 1::2] = (codes // 16).double()
            par = params.double().repeat_interleave(GROUP, -2)
            return ((x + 128) * par[..., 0] + par[..., 1]).float().bfloat16().double()

        out = torch.zeros(B, H, Lq, Dv, dtype=torch.float64, device=DEV)
        lens = st["lengths"].tolist() if case["ragged"] else [T] * B
        for b in range(B):
            n = lens[b]
            if n == 0:
                continue
            k = value(st["cache"][0][b, :, :n], st["cache"][1][b, :, :n])
            v = value(st["cache"][2][b, :, :n], st["cache"][3][b, :, :n])
            see = torch.ones(Lq, n, dtype=torch.bool, device=DEV).tril(n - Lq)
            for h in range(H):
                s = st["q"][b, h].double() @ k[h * Hk // H].t() / math.sqrt(D)
                w = torch.where(see, torch.exp(s - s.masked_fill(~see, -1e300).amax(1, keepdim=True)), 0.0)
                total = w.sum(1, keepdim=True)
                out[b, h] = torch.where(total > 0, w @ v[h * Hk // H] / total.clamp(min=1e-300), 0.0)
        return out
    B, K = case["B"], case["K"]
    tok, ua, us = st["tokens"].tolist(), st["u_accept"], st["u_sample"].tolist()
    many = [K] * B if st["lengths"] is None else st["lengths"].tolist()
    tokens = torch.full((B, K + 1), -1, dtype=torch.int64)
    accepted = torch.zeros(B, dtype=torch.int64)
    for b in range(B):
        n = 0
        while n < many[b]:
            chance = st["target"][b, n, tok[b][n]].float()
            if st["draft"] is not None:
                if not bool(ua[b, n] * st["draft"][b, n, tok[b][n]].float() < chance):
                    break
            elif not bool(ua[b, n] < chance):
                break
            n += 1
        w = st["target"][b, n].float().double().cpu()
        if n < many[b]:
            left = w.clone()
            if st["draft"] is None:
                left[tok[b][n]] = 0
            else:
                left = (st["target"][b, n].float() - st["draft"][b, n].float()).double().cpu().clamp(min=0)
            w = left if bool((left > 0).any()) else w
        c = torch.cumsum(w, 0)
        tokens[b, :n] = torch.tensor(tok[b][:n], dtype=torch.int64)
        tokens[b, n] = int(torch.searchsorted(c, us[b] * float(c[-1]), right=True))
        accepted[b] = n
    return {"tokens": tokens, "accepted": accepted}
