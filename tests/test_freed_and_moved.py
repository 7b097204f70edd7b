"""What is kept beside a model's tensors goes with them: the bf16 compute copies of its
weights are freed with the weights, the 4-bit KV caches of open streams move with the
model."""

import gc

import pytest
import torch

from vagus_b200 import ops
from vagus_b200.models import build_model
from vagus_b200.ops._core import _Bf16Cache


def test_copies_are_freed_with_their_masters():
    cache = _Bf16Cache()
    w, u, kept = torch.randn(3, 4, 8).unbind()
    w, u, kept = w.clone(), u.clone(), kept.clone()
    for t in (w, kept):
        cache.get(t)
    cache.get_cat([w, u])
    cache.get_cat([u, kept])
    cache.get_cat([kept, kept])
    assert len(cache._d) == 5
    w.add_(1)                                  # a newer copy of w takes the place of the old one
    cache.get(w)
    assert len(cache._d) == 5
    del w, t
    gc.collect()
    assert len(cache._d) == 3
    del u
    gc.collect()
    assert len(cache._d) == 2 and (cache.get(kept) == kept.bfloat16()).all()
    cache.clear()
    del kept                                   # its entries are gone already
    gc.collect()
    assert not cache._d


def test_a_copy_outlives_its_dead_master_where_it_is_used():
    cache = _Bf16Cache()
    w = torch.randn(8, 16, requires_grad=True)
    want = w.detach().bfloat16()
    x = torch.randn(3, 16).bfloat16().requires_grad_()
    y = x @ cache.get(w).t()
    del w
    gc.collect()
    assert not cache._d
    y.sum().backward()
    assert torch.equal(x.grad, torch.ones(3, 8).bfloat16() @ want)


def test_a_graph_that_holds_a_master_keeps_its_copy():
    """A weight that only autograd still holds is alive: the copy belongs to it."""
    cache = _Bf16Cache()
    w = torch.randn(4, 8, requires_grad=True)
    c = cache.get(w)
    y = (w * w).sum()
    y.backward()
    assert cache.get(w) is c


def test_an_address_and_an_id_taken_over():
    """As many masters as it takes for an id to come back: never more than one entry, never a wrong one."""
    cache = _Bf16Cache()
    for i in range(300):
        w = torch.full((16, 16), float(i))
        assert (cache.get(w) == i).all() and len(cache._d) == 1
        del w


# ------------------------------------------------------------------- 4-bit cache --

def streaming(**kw):
    """A model with a 4-bit cache that holds 9 tokens of two streams."""
    torch.manual_seed(0)
    m = build_model("TransformerPP", dict(vocab_size=300, dim=64, layer_count=2, head_dim=32, context_len=64,
                                          ffn_hidden_dim=128, **kw)).eval()
    m.set_cache_bits(4)
    m.reset_cache(2, 40)
    m.decode_step(torch.randint(0, 300, (2, 9)))
    return m


def caches(m):
    return [t for b in m.blocks for t in b.att.kv4.tensors()]


def test_open_streams_move_with_the_model():
    m = streaming().to("meta")
    assert all(t.device.type == "meta" for t in caches(m) + [b.att.k_cache for b in m.blocks])
    m.to_empty(device="cpu")
    assert all(t.device.type == "cpu" for t in caches(m))
    ops.int4_read(m.blocks[0].att.kv4, 0, 9)


@pytest.mark.parametrize("cast", [lambda m: m.double(), lambda m: m.to(torch.bfloat16), lambda m: m.half().float()])
def test_a_cast_leaves_the_codes_alone(cast):
    m = streaming()
    before = [t.clone() for t in caches(m)]
    cast(m)
    for a, b in zip(caches(m), before):
        assert a.dtype == b.dtype and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.gpu
def test_a_model_moves_between_two_decode_steps():
    ids = torch.randint(0, 300, (2, 3))
    here, moved = streaming(), streaming()
    want = here.decode_step(ids)
    before = [t.clone() for t in caches(moved)]
    moved.to("cuda")
    assert all(a.is_cuda and torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))
               for a, b in zip(caches(moved), before))
    got = moved.decode_step(ids.cuda())
    # the same codes; sums of at most 128 products in fp32, under 20 one after another: 20 * 128 * 2^-24 < 2e-4
    assert (got.cpu() - want).abs().max() < 1e-3 * want.abs().max()
    moved.to("cpu")
    nxt = torch.randint(0, 300, (2, 1))
    want = here.decode_step(nxt)
    assert (moved.decode_step(nxt) - want).abs().max() < 1e-3 * want.abs().max()
