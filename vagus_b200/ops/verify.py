"""Verification of drafted tokens against the target's probabilities.

Speculative sampling from given random numbers: drafted token i of a row is
accepted while ``u_i q_i(d_i) < p_i(d_i)``, and one more token follows -- at the
first rejected place from ``max(p - q, 0)``, after the last drafted token from
``p`` -- so the tokens that come out are distributed as the target's own.  CUDA
runs ``verify.cu``; elsewhere the plain form below runs.
"""

from __future__ import annotations

import torch

from ._core import native


@torch.no_grad()
def verify_draft_ref(target, draft, tokens, u_accept, u_sample, lengths):
    B, K = tokens.shape
    V = target.shape[2]
    dev = target.device
    inside = (tokens >= 0) & (tokens < V)
    safe = torch.where(inside, tokens, torch.zeros_like(tokens))
    p = target[:, :K].float().gather(2, safe[..., None])[..., 0]
    q = torch.ones_like(p) if draft is None else draft.float().gather(2, safe[..., None])[..., 0]
    n = torch.full((B,), K, device=dev) if lengths is None else lengths.to(torch.int64).clamp(0, K)
    place = torch.arange(K + 1, device=dev)
    ok = (u_accept * q < p) & inside & (place[:K] < n[:, None])
    accepted = ok.long().cumprod(1).sum(1)
    row = torch.arange(B, device=dev)
    last = target[row, accepted].float()
    w = last
    if K:
        at = accepted.clamp(max=K - 1)
        if draft is None:
            struck = (torch.arange(V, device=dev) == tokens[row, at][:, None])
            rest = last.masked_fill(struck, 0.0)
        else:
            rest = last - draft[row, at].float()
        rest = torch.where((rest > 0).any(1, keepdim=True), rest, last)
        w = torch.where((accepted < n)[:, None], rest, last)
    w = torch.where(w > 0, w, torch.zeros_like(w)).double()
    run = w.cumsum(1)
    over = (run > u_sample.double()[:, None] * run[:, -1:]) & (w > 0)
    top = torch.where(w > 0, torch.arange(V, device=dev), 0).amax(1)      # the last token with any weight
    new = torch.where(over.any(1), over.int().argmax(1), top)
    out = torch.cat((tokens, tokens.new_zeros(B, 1)), 1)
    out = torch.where(place < accepted[:, None], out, torch.where(place == accepted[:, None], new[:, None], -1))
    return out, accepted


def _check(target, draft, tokens, u_accept, u_sample, lengths):
    if target.dim() != 3 or target.shape[1] < 1 or target.shape[2] < 1 \
            or target.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError("verify_draft: target (B, K + 1, V), fp32, fp16 or bf16")
    B, K, V = target.shape[0], target.shape[1] - 1, target.shape[2]
    if draft is not None and (tuple(draft.shape) != (B, K, V) or draft.dtype != target.dtype):
        raise ValueError(f"verify_draft: draft must be ({B}, {K}, {V}) of the target's dtype")
    if tuple(tokens.shape) != (B, K) or tokens.dtype != torch.int64:
        raise ValueError(f"verify_draft: tokens must be ({B}, {K}) int64")
    if tuple(u_accept.shape) != (B, K) or tuple(u_sample.shape) != (B,) or u_accept.dtype != torch.float32 \
            or u_sample.dtype != torch.float32:
        raise ValueError(f"verify_draft: u_accept ({B}, {K}) and u_sample ({B},), fp32")
    if lengths is not None and (tuple(lengths.shape) != (B,) or lengths.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"verify_draft: lengths must be ({B},) int32 or int64")
    if any(t is not None and t.device != target.device for t in (draft, tokens, u_accept, u_sample, lengths)):
        raise ValueError("verify_draft: all tensors must be on one device")


def verify_draft(target, draft, tokens, u_accept, u_sample, lengths=None):
    """``target`` (B, K + 1, V): the target's probabilities at the K drafted
    places and the one after; ``draft`` (B, K, V): the probabilities the drafts
    were drawn from, or None when they were certain (a lookup, a greedy draft:
    q = 1, and a rejected token is struck out of p); ``tokens`` (B, K) int64;
    ``u_accept`` (B, K) and ``u_sample`` (B,) fp32 in [0, 1); ``lengths`` (B,)
    int32 / int64: drafted tokens of each row (default K).  fp32, fp16 or bf16
    probabilities, which must be finite; they need not sum to one.

    Returns ``(out, accepted)``: accepted (B,) int64, and out (B, K + 1) int64
    holding the accepted drafts, the token that follows, then -1.  A drafted
    token outside the vocabulary is rejected.  The next token is the first v
    whose running sum of weights exceeds u_sample times their sum, in 64 bits (the
    order of the sums is fixed for given B, V, dtype and alignment; another could give a
    neighbouring token only where u_sample lies within their rounding of a border);
    where nothing is left of max(p - q, 0) it is drawn from p, and a row without
    any weight gives token 0.  K = 0 draws one token from ``target``."""
    if target.is_cuda:                       # the binding checks the arguments by the same conditions
        return native().verify_draft(target, draft, tokens, u_accept, u_sample, lengths)
    _check(target, draft, tokens, u_accept, u_sample, lengths)
    return verify_draft_ref(target, draft, tokens, u_accept, u_sample, lengths)
