"""Caches without pages and batches without sequences: the kernels treat them like any other."""

import pytest
import torch

pytestmark = pytest.mark.gpu

import lucid_b200.quantization as Q  # noqa: E402
from lucid_b200 import _lib  # noqa: E402


@pytest.mark.parametrize("fmt", ["int8", "mxfp4"])
@pytest.mark.parametrize("tokens", [3, 300])
def test_a_cache_without_pages(fmt, tokens):
    cache = Q.kv_cache_alloc(0, 16, 2, 64, fmt)
    x = torch.randn(tokens, 2, 64, device="cuda")
    Q.kv_cache_write(cache, x, x, torch.full((tokens,), -1, device="cuda"))  # padding only
    _lib.check_device_status(x.device)
    Q.kv_cache_write(cache, x, x, torch.arange(tokens, device="cuda"))
    with pytest.raises(_lib.ShapeMismatch):
        _lib.check_device_status(x.device)
    cu = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    for table in (torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, 0, dtype=torch.int32, device="cuda")):
        k, v = Q.kv_cache_read(cache, table, cu, 5)
        assert k.shape == (5, 2, 64) and not k.any() and not v.any()
        with pytest.raises(_lib.ShapeMismatch):
            _lib.check_device_status(x.device)


@pytest.mark.parametrize("width", [0, 8])
def test_an_idle_batch_reads_no_rows(width):
    cache = Q.kv_cache_alloc(2, 4, 1, 32)
    table = torch.zeros(0, width, dtype=torch.int32, device="cuda")
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = Q.kv_cache_read(cache, table, cu, 3)
    assert k.shape == (3, 1, 32) and not k.any() and not v.any()
    kept = tuple(torch.full((3, 1, 32), 7.0, device="cuda") for _ in range(2))
    Q.kv_cache_read(cache, table, cu, 3, out=kept)
    assert all((t == 7.0).all() for t in kept)
    _lib.check_device_status(k.device)
