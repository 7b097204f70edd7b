"""What is kept beside a model's tensors goes with them: the bf16 compute copies of its
weights are freed with the weights."""

import gc

import torch

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
