"""A key / value cache held in 4 bits, and softmax attention over it.

For every (sequence, KV head, token) the cache holds one 4-bit code a channel
(channel 2 j in the low half of byte j) and, for each group of 32 channels, a
step s and an offset b in bf16:

    s = bf16((max - min) / 15),  b = bf16(min - 128 s),
    c = clamp(round((x - b) / s) - 128, 0, 15),  and c stands for bf16((128 + c) s + b)

(round: to nearest, ties to even; the steps in fp32).  That is 0.625 bytes a
value against 2 of a bf16 cache.  A value is off by at most
max(s / 2, 2^-8 |min - 128 s| + 0.06 s) and its own rounding to bf16: little more
than half a step in groups near zero, more in groups whose minimum lies far from
it (the rounding of b moves the grid, and values at the group's edge are clamped).
A group of equal values is held to bf16 (s = 0); a group that holds a NaN or an
infinity stands for NaN; magnitudes up to 1e37 are representable.

``int4_attention`` is attention over the values that the codes stand for, which
``int4_read`` returns: however a stream is cut into calls, a token sees the same
keys and values.  CUDA runs ``kv4.cu``; elsewhere the plain forms below run.
"""

from __future__ import annotations

import math
import torch

from ._core import native

GROUP = 32
_BLOCK = 16         # the capacity is a whole number of blocks of this many tokens


def _check_cache(k_codes, k_params, v_codes, v_params) -> None:
    for codes, params, what in ((k_codes, k_params, "k"), (v_codes, v_params, "v")):
        if codes.dim() != 4 or codes.dtype != torch.uint8 or not codes.is_contiguous() \
                or codes.shape[3] % (GROUP // 2) or not codes.shape[3]:
            raise ValueError(f"Int4KV: {what}_codes must be (B, Hk, capacity, D / 2) uint8, contiguous, "
                             f"D a multiple of {GROUP}")
        want = (*codes.shape[:3], codes.shape[3] * 2 // GROUP, 2)
        if tuple(params.shape) != want or params.dtype != torch.bfloat16 or not params.is_contiguous():
            raise ValueError(f"Int4KV: {what}_params must be {want} bf16, contiguous")
    if k_codes.shape[:3] != v_codes.shape[:3]:
        raise ValueError("Int4KV: keys and values must agree in batch, heads and capacity")
    if k_codes.shape[2] % _BLOCK or k_codes.shape[2] >= 1 << 30:
        raise ValueError(f"Int4KV: the capacity must be a multiple of {_BLOCK}, below 2^30")
    if any(t.device != k_codes.device for t in (k_params, v_codes, v_params)):
        raise ValueError("Int4KV: the tensors must be on one device")


class Int4KV:
    """The four tensors of a cache, all contiguous (and 16-byte aligned) on one
    device: codes (B, Hk, capacity, D / 2) uint8 and parameters
    (B, Hk, capacity, D / 32, 2) bf16 holding (s, b), for keys and for values."""

    __slots__ = ("k_codes", "k_params", "v_codes", "v_params")

    def __init__(self, k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor, v_params: torch.Tensor):
        if k_codes.is_cuda:
            native().kv4_check(k_codes, k_params, v_codes, v_params)
        else:
            _check_cache(k_codes, k_params, v_codes, v_params)
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params

    @classmethod
    def empty(cls, batch: int, kv_heads: int, capacity: int, head_dim: int, value_dim: int | None = None,
              device=None) -> "Int4KV":
        """Room for at least ``capacity`` tokens of ``batch`` sequences, zeroed."""
        value_dim = head_dim if value_dim is None else value_dim
        if head_dim < GROUP or head_dim % GROUP or value_dim < GROUP or value_dim % GROUP:
            raise ValueError(f"Int4KV: head dims must be multiples of {GROUP}, got {head_dim} and {value_dim}")
        cap = -(-capacity // _BLOCK) * _BLOCK

        def pair(d):
            return (torch.zeros(batch, kv_heads, cap, d // 2, dtype=torch.uint8, device=device),
                    torch.zeros(batch, kv_heads, cap, d // GROUP, 2, dtype=torch.bfloat16, device=device))
        return cls(*pair(head_dim), *pair(value_dim))

    def tensors(self) -> tuple[torch.Tensor, ...]:
        return self.k_codes, self.k_params, self.v_codes, self.v_params

    def to(self, device) -> "Int4KV":
        """The cache on another device (itself, where it is there already).  From the
        meta device, which holds nothing, a cache of unspecified content."""
        device = torch.device(device)
        if device == self.k_codes.device:
            return self
        return Int4KV(*(torch.empty_like(t, device=device) if t.is_meta else t.to(device) for t in self.tensors()))

    @property
    def batch(self) -> int:
        return self.k_codes.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.k_codes.shape[1]

    @property
    def capacity(self) -> int:
        return self.k_codes.shape[2]

    @property
    def head_dim(self) -> int:
        return 2 * self.k_codes.shape[3]

    @property
    def value_dim(self) -> int:
        return 2 * self.v_codes.shape[3]


# ------------------------------------------------------------------ plain forms --

def int4_quantise_ref(x):
    """(..., D) -> codes (..., D / 2) uint8 and parameters (..., D / 32, 2) bf16."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi - lo) / 15).bfloat16().float()
    b = (lo - 128 * s).bfloat16().float()
    c = (torch.round((g - b) / s) - 128).clamp(0, 15)
    c = torch.where((s > 0) & ~c.isnan(), c, torch.zeros_like(c)).flatten(-2).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.cat((s, b), -1).bfloat16()


def int4_values_ref(codes, params):
    """The bf16 values that codes stand for."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    return ((c + 128) * params[..., :1].float() + params[..., 1:].float()).flatten(-2).bfloat16()


def int4_attention_ref(q, k, v, lengths, causal: bool = True):
    """q (B, H, Lq, D) over k, v (B, Hk, T, ..), of which sequence b holds ``lengths[b]`` tokens."""
    B, H, Lq, D = q.shape
    Hk, T = k.shape[1], k.shape[2]
    up = torch.promote_types(q.dtype, torch.float32)
    at = torch.arange(T, device=q.device)
    held = at < lengths[:, None]
    # what lies past a sequence's length counts nothing, whatever it is
    k = torch.where(held[:, None, :, None], k, 0.0).to(up)
    v = torch.where(held[:, None, :, None], v, 0.0).to(up)
    s = q.to(up).reshape(B, Hk, H // Hk * Lq, D) @ k.transpose(-1, -2) / math.sqrt(D)
    s = s.view(B, Hk, H // Hk, Lq, T)
    seen = lengths[:, None] - Lq + 1 + torch.arange(Lq, device=q.device) if causal else lengths[:, None].expand(B, Lq)
    s = s.masked_fill(at >= seen[:, None, None, :, None], float("-inf"))
    top = s.amax(-1, keepdim=True) if T else s.new_zeros(B, Hk, H // Hk, Lq, 1)
    p = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)     # a row that sees nothing gives zeros
    return (p.view(B, Hk, H // Hk * Lq, T) @ v).view(B, H, Lq, v.shape[-1]).to(q.dtype)


# ------------------------------------------------------------------ entry points --
# On the GPU the bindings check the arguments, by the conditions written out here for the CPU.

def _place(x, what: str):
    """(tensor or None, int) of a place given as an int or per sequence."""
    if isinstance(x, int):
        return None, x
    if isinstance(x, torch.Tensor):
        return x, 0
    raise ValueError(f"{what} must be an int or a tensor")


def _rows(per, at, cache: Int4KV, what: str):
    """(B,) int64 places."""
    if per is None:
        return torch.full((cache.batch,), at, device=cache.k_codes.device)
    if per.dtype not in (torch.int32, torch.int64) or tuple(per.shape) != (cache.batch,) \
            or per.device != cache.k_codes.device:
        raise ValueError(f"{what} must be an int or ({cache.batch},) int32 / int64 on the cache's device")
    return per.to(torch.int64)


def _span(cache: Int4KV, start, count: int, what: str) -> None:
    if count < 0 or (start.numel() and (int(start.min()) < 0 or int(start.max()) + count > cache.capacity)):
        raise ValueError(f"{what}: tokens outside the cache of {cache.capacity}")


def _at(cache: Int4KV, start, count: int):
    """Indices of tokens start .. start + count - 1 in the cache's tensors."""
    return (torch.arange(cache.batch)[:, None, None], torch.arange(cache.kv_heads)[None, :, None],
            start[:, None, None] + torch.arange(count))


@torch.no_grad()
def _append_plain(cache, k, v, per, at):
    if k.dim() != 4 or v.dim() != 4 or k.shape[:3] != v.shape[:3] or k.shape[0] != cache.batch \
            or k.shape[1] != cache.kv_heads or k.shape[3] != cache.head_dim or v.shape[3] != cache.value_dim:
        raise ValueError(f"int4_append: k {tuple(k.shape)}, v {tuple(v.shape)} do not fit the cache")
    if k.dtype != v.dtype or k.device != cache.k_codes.device or v.device != cache.k_codes.device:
        raise ValueError("int4_append: k and v must share a dtype and be on the cache's device")
    start = _rows(per, at, cache, "int4_append: start")
    _span(cache, start, k.shape[2], "int4_append")
    idx = _at(cache, start, k.shape[2])
    for have, new in zip(cache.tensors(), int4_quantise_ref(k) + int4_quantise_ref(v)):
        have[idx] = new


def int4_append(cache: Int4KV, k, v, start) -> None:
    """Quantise ``k`` (B, Hk, L, D) and ``v`` (B, Hk, L, Dv) into the cache as
    tokens start .. start + L - 1 (``start``: an int, or (B,) int32 / int64 for
    a place per sequence; one given on the GPU is checked by the kernel, which
    writes nothing outside the cache and reports it through ``check_error``).
    fp32, fp16 or bf16 on the GPU."""
    per, at = _place(start, "int4_append: start")
    if cache.k_codes.is_cuda:
        native().kv4_append(cache.k_codes, cache.k_params, cache.v_codes, cache.v_params, k, v, per, at)
    else:
        _append_plain(cache, k, v, per, at)


def int4_read(cache: Int4KV, start, count: int):
    """The values of tokens start .. start + count - 1 as bf16 k (B, Hk, count, D)
    and v (B, Hk, count, Dv); ``start`` as in ``int4_append`` (tokens outside
    the cache read as zeros on the GPU and are reported)."""
    per, at = _place(start, "int4_read: start")
    if cache.k_codes.is_cuda:
        return native().kv4_read(cache.k_codes, cache.k_params, cache.v_codes, cache.v_params, per, at, count)
    start = _rows(per, at, cache, "int4_read: start")
    _span(cache, start, count, "int4_read")
    idx = _at(cache, start, count)
    kc, kp, vc, vp = (x[idx] for x in cache.tensors())
    return int4_values_ref(kc, kp), int4_values_ref(vc, vp)


@torch.no_grad()
def _attention_plain(q, cache, per, at, causal):
    if q.dim() != 4 or q.shape[0] != cache.batch or q.shape[3] != cache.head_dim or not cache.kv_heads \
            or q.shape[1] % cache.kv_heads or q.device != cache.k_codes.device:
        raise ValueError(f"int4_attention: q {tuple(q.shape)} does not fit the cache")
    lengths = _rows(per, at, cache, "int4_attention: lengths")
    if not q.is_cuda and lengths.numel() and (int(lengths.max()) > cache.capacity or (per is None and at < 0)):
        raise ValueError(f"int4_attention: lengths outside the cache of {cache.capacity}")
    k, v = int4_read(cache, 0, cache.capacity if per is not None else at)
    return int4_attention_ref(q, k, v, lengths.clamp(0, cache.capacity), causal)


def int4_attention(q, cache: Int4KV, lengths, causal: bool = True):
    """Attention of ``q`` (B, H, Lq, D) over the first ``lengths`` tokens of the
    cache -> (B, H, Lq, Dv); H is a multiple of the cache's heads.

    ``lengths``: an int, or (B,) int32 / int64 (given on the GPU, the kernel
    clamps it to the cache and reports it through ``check_error``).  With
    ``causal`` the queries are the last Lq of those tokens: query i sees the
    first lengths - Lq + i + 1 of them.  A query that sees nothing gives zeros.
    What the cache holds past a sequence's length has no effect; a NaN inside it
    may reach every query of the call.  Inference only: no derivative of either
    mode flows.

    The kernels take bf16 queries and head dims 64 and 128.  Scores, softmax sums and
    accumulators are fp32; probabilities are rounded to bf16 for the product with the
    values (2^-8 relative at most, unbiased), as in ``ops.attention``.  With many
    queries over equal lengths (an int) the values are unpacked into a temporary bf16
    copy first.  Other types and head dims take the plain form in fp32, which forms
    all scores (and with lengths per sequence unpacks the whole capacity).  Refused with
    a RuntimeError: batch x KV heads x tiles of 16 query rows x blocks of 128 tokens
    (of the capacity, with lengths per sequence) of about 2^30 or more."""
    per, at = _place(lengths, "int4_attention: lengths")
    if cache.k_codes.is_cuda:
        o = native().kv4_attn(q, cache.k_codes, cache.k_params, cache.v_codes, cache.v_params, per, at, causal)
        if o is not None:
            return o
    return _attention_plain(q, cache, per, at, causal)
