"""MXFP4 operands that no encode of this library writes."""

import numpy as np
import pytest
import torch

import mx_oracle as MX

pytestmark = pytest.mark.gpu

import lucid_b200.quantization as Q  # noqa: E402
from gpu_util import dev, host  # noqa: E402


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_the_largest_scales_decode_to_what_float32_holds(out):
    code = np.tile(np.arange(32, dtype=np.uint8) % 16, (256, 1))
    byte = np.arange(256, dtype=np.uint8)[:, None]
    y = host(Q.mx_dequantize(dev(MX.pack(code)), dev(MX.tile(byte)), out_dtype=out))
    exact = MX.decode(code, byte)
    with np.errstate(over="ignore"):
        want = exact.astype(np.float32)  # infinite from 2^128 on
    assert np.array_equal(y, want, equal_nan=True)
    assert np.isfinite(want[:253]).all() and np.isinf(want[254]).any() and np.isnan(want[255]).all()


@pytest.mark.parametrize("m,k,n", [(3, 288, 130), (16, 32, 40), (30, 800, 300), (70, 736, 257), (200, 96, 4200), (1300, 352, 4100)])
def test_padding_bytes_other_than_nan_do_not_matter(m, k, n):
    """Scale tiles made elsewhere: any byte but 255 past K, any byte in the rows past the end."""
    rng = np.random.default_rng(m + k + n)

    def padded(rows):
        code, byte = rng.integers(0, 16, (rows, k)).astype(np.uint8), rng.integers(120, 134, (rows, k // 32)).astype(np.uint8)
        tiles = MX.tile(byte)
        inside = MX.tile(np.ones_like(byte)) == 1
        live = np.zeros((tiles.shape[0] * 128, tiles.shape[1] * 8), np.uint8)
        live[:rows] = 1  # (row exists, whatever the block)
        filler = rng.integers(0, 255, tiles.shape).astype(np.uint8)
        filler[MX.tile(live) == 0] = 255
        return dev(MX.pack(code)), dev(tiles), dev(np.where(inside, tiles, filler))

    (ac, sa, sa2), (wc, sw, sw2) = padded(m), padded(n)
    want = Q.mx_matmul(ac, sa, wc, sw)
    assert torch.isfinite(want).all() and torch.equal(Q.mx_matmul(ac, sa2, wc, sw2), want)
    x = torch.randn(m, k, device="cuda")
    assert torch.equal(Q.mx_linear(x, wc, sw2), Q.mx_linear(x, wc, sw))
