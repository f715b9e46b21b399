"""CPU checks of the cache module and of what its functions refuse."""

import numpy as np
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


def _pairs(buf):
    """Two views for keys and values, and whether they share memory: buf holds 2 x 6 x 4 x 32 values."""
    whole = buf.view(2, 6, 4, 32)
    yield whole[0], whole[1], False                                        # one after the other
    yield buf.view(6, 2, 4, 32)[:, 0], buf.view(6, 2, 4, 32)[:, 1], False  # token by token
    yield buf.view(6, 4, 2, 32)[:, :, 0], buf.view(6, 4, 2, 32)[:, :, 1], False  # head by head
    yield buf.view(4, 2, 6, 32)[:, 0].transpose(0, 1), buf.view(4, 2, 6, 32)[:, 1].transpose(0, 1), False
    yield whole[0], whole[0], True
    yield buf.view(12, 4, 32)[:6], buf.view(12, 4, 32)[5:11], True
    yield buf.view(12, 4, 32)[3:9], buf.view(12, 4, 32)[2:8], True
    yield buf.view(48, 32).as_strided((6, 4, 32), (256, 32, 1)), buf.view(48, 32).as_strided((6, 4, 32), (256, 32, 1), 112), True
    yield buf.as_strided((5, 4, 32), (256, 32, 1), 16), buf.as_strided((5, 4, 32), (256, 32, 1), 144), False
    yield whole[0], buf.as_strided((6, 4, 32), (256, 32, 1)), True        # another stride from the same beginning
    yield whole[0, :1, :1], whole[0, :1, 1:2], False
    yield whole[0, :1], buf.as_strided((1, 4, 32), (999, 32, 1), 16), True  # (the stride of a single token says nothing)
    yield whole[0, :0], whole[0, :0], False


def test_keys_and_values_read_into_the_same_rows_are_refused(monkeypatch):
    calls = []
    monkeypatch.setattr(_lib, "require_cuda", lambda t, what: None)
    monkeypatch.setattr(_lib, "call", lambda name, *args: calls.append(name))
    monkeypatch.setattr(_lib, "status_ptr", lambda device: None)
    table = torch.zeros(1, 4, dtype=torch.int32)
    for i, (k, v, shared) in enumerate(_pairs(torch.zeros(2 * 6 * 4 * 32))):
        a, b = ({t.storage_offset() + sum(x * s for x, s in zip(at, t.stride())) for at in np.ndindex(*t.shape)} for t in (k, v))
        assert bool(a & b) == shared, i  # what the table above says
        cache = Q.kv_cache_alloc(4, 2, k.shape[1], 32, device="cpu")
        cu = torch.tensor([0, k.shape[0]], dtype=torch.int32)
        for out in ((k, v), (v, k)):
            del calls[:]
            if shared:
                with pytest.raises(_lib.ShapeMismatch):
                    Q.kv_cache_read(cache, table, cu, k.shape[0], out=out)
                assert calls == []
            else:
                Q.kv_cache_read(cache, table, cu, k.shape[0], out=out)
                assert calls == ["lq_kv_read"]
