"""CPU checks of the cache module and of what its functions refuse."""

import pytest
import torch

import lucid_b200.nn.quantized as nnq
import lucid_b200.quantization as Q
from lucid_b200 import _lib


def _filled(fmt):
    module = nnq.PagedKVCache(2, 4, 3, 64, fmt)
    for t in module.buffers():
        t.copy_(torch.rand(t.shape) * 100 + 1.0 / 3.0)
    return module


@pytest.mark.parametrize("fmt", ["int8", "mxfp4"])
@pytest.mark.parametrize("move", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.double(), lambda m: m.to(torch.bfloat16),
                                  lambda m: m.to("cpu", torch.bfloat16), lambda m: m.type(torch.float16),
                                  lambda m: m.to(torch.float16).float()])
def test_a_change_of_the_models_type_leaves_the_cache_as_it_is(fmt, move):
    module = _filled(fmt)
    model = torch.nn.Sequential(torch.nn.Linear(8, 8), module)
    before = [t.clone() for t in module.cache]
    move(model)
    assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(module.cache, before))


def test_the_cache_still_moves_between_devices():
    module = _filled("int8")
    types = [t.dtype for t in module.cache]
    module.to("meta", torch.bfloat16)
    assert all(t.is_meta and t.dtype == d for t, d in zip(module.cache, types))
    module.to_empty(device="cpu")
    assert all(not t.is_meta and t.dtype == d for t, d in zip(module.cache, types))


def test_a_cache_that_no_call_would_take_is_not_made():
    for heads in (0, 4097):
        with pytest.raises(_lib.ShapeMismatch):
            Q.kv_cache_alloc(1, 1, heads, 32, device="cpu")
    assert Q.kv_cache_alloc(1, 1, 4096, 32, device="cpu").k_scales.shape == (1, 1, 4096)
