"""The bf16 compute copies of fp32 masters belong to their tensors, not to an id or an
address that another tensor may take over."""

import torch

from vagus_b200.ops._core import _Bf16Cache


def test_a_new_tensor_never_gets_a_dead_ones_copy():
    cache = _Bf16Cache()
    for i in range(200):
        w = torch.full((64, 64), float(i))
        assert (cache.get(w) == i).all()
        u = torch.full((8, 64), float(-i))
        assert (cache.get_cat([w, u])[-8:] == -i).all()
        del w, u


def test_a_copy_is_kept_until_the_master_changes():
    cache = _Bf16Cache()
    w = torch.zeros(4, 8)
    c = cache.get(w)
    assert cache.get(w) is c and cache.get_cat([w, w]) is cache.get_cat([w, w])
    w.add_(1)
    assert (cache.get(w) == 1).all() and (cache.get_cat([w, w]) == 1).all()
