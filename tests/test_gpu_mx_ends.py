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
