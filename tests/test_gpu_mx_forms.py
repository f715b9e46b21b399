"""The product's forms for long inputs against sums in 64 bits: K shared by clusters of every size with runs of unequal
length, the longest K, several tiles to a CTA pair."""

import pytest
import torch

pytestmark = pytest.mark.gpu

import lucid_b200.quantization as Q  # noqa: E402
from lucid_b200 import _lib  # noqa: E402

VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _operand(rows, k, seed):
    """Packed random elements with scales of 1/2 .. 2, and their values in float64.  Every product is a multiple of
    2^-4 and at most 144, so a sum of K <= 7281 of them (2^24 / 16 / 144) is exact in float32 in any order; with scales of
    1 (multiples of 1/4, at most 36) one of K <= 116508."""
    g = torch.Generator("cuda").manual_seed(seed)
    code = torch.randint(0, 16, (rows, k), device="cuda", generator=g, dtype=torch.uint8)
    lo, hi = (126, 129) if k <= 7281 else (127, 128)
    byte = torch.randint(lo, hi, (rows, k // 32), device="cuda", generator=g, dtype=torch.uint8)
    value = torch.tensor(VALUES + [-v for v in VALUES], dtype=torch.float64, device="cuda")[code.long()]
    value *= torch.exp2(byte.double() - 127).repeat_interleave(32, 1)
    full = torch.zeros((-(-rows // 128) * 128, -(-k // 256) * 8), dtype=torch.uint8, device="cuda")
    full[:rows, :k // 32] = byte
    tiles = full.view(-1, 4, 32, full.shape[1] // 8, 2, 4).permute(0, 3, 4, 2, 1, 5).reshape(-1, full.shape[1] // 8, 1024)
    return (code[:, 0::2] | code[:, 1::2] << 4).contiguous(), tiles.contiguous(), value


# tokens, K, features; a cluster shares K from 4 stages of 256 each (up to 32 tokens) or 10 (64)
SPLITS = [(3, 2080, 300), (16, 3232, 200), (9, 4192, 130), (1, 5152, 1003), (5, 6400, 257), (16, 7360, 300), (2, 8192, 515),  # 2 .. 8 CTAs
          (24, 4096, 300), (17, 5152, 130), (32, 7360, 1003), (48, 8192, 1003), (33, 5440, 640), (70, 5152, 130), (100, 8192, 640),
          (64, 20480, 72), (5, 28672, 300), (30, 28672, 257), (48, 28672, 300), (300, 28672, 520)]
# whole tiles: 128 tokens, then CTA pairs with three to seven tiles each and with the longest K
WHOLE = [(1000, 5440, 4096), (2600, 544, 5000), (4100, 288, 8200), (2200, 28672, 2200)]


@pytest.mark.parametrize("m,k,n", SPLITS + WHOLE)
def test_product_is_exact_where_float32_is(m, k, n):
    ac, sa, a = _operand(m, k, m + k)
    wc, sw, w = _operand(n, k, n + k)
    ref = a @ w.T
    y = Q.mx_matmul(ac, sa, wc, sw)
    assert torch.equal(y.double(), ref)
    bias = torch.randint(-64, 64, (n,), device="cuda").float()
    y = Q.mx_matmul(ac, sa, wc, sw, bias=bias, relu=True, out_dtype=torch.bfloat16)
    assert torch.equal(y, (ref + bias).clamp(min=0).float().to(torch.bfloat16))
    _lib.check_device_status(y.device)


@pytest.mark.parametrize("m,k,n", [(9, 4192, 130), (24, 4096, 300), (48, 8192, 1003), (100, 8192, 640), (2600, 544, 5000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_the_result_may_lie_apart(m, k, n, dtype):
    ac, sa, a = _operand(m, k, 1)
    wc, sw, w = _operand(n, k, 2)
    ref = (a @ w.T).float().to(dtype)
    for ldo in (n + 5, n + 8):
        out = torch.full((m + 2, ldo), -7.0, dtype=dtype, device="cuda")
        _lib.call("lq_mx_matmul", out.device, ac.data_ptr(), sa.data_ptr(), m, wc.data_ptr(), sw.data_ptr(), n, k, None, 0,
                  out.data_ptr(), _lib.code_of(dtype), ldo, None)
        assert torch.equal(out[:m, :n], ref) and (out[:m, n:] == -7.0).all() and (out[m:] == -7.0).all()


@pytest.mark.parametrize("m,k,n", [(1, 28672, 300), (16, 7360, 200), (12, 3232, 1003), (24, 4096, 300), (48, 8192, 1003), (300, 28672, 200)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_of_activations_the_format_holds(m, k, n, dtype):
    """Activations that are values of the format already: the encode inside the product, or before it, loses nothing."""
    _, _, a = _operand(m, k, 5)
    a.view(m, -1, 32)[..., 0] = 6.0  # the block's largest magnitude is the grid's: its scale is 1
    a = a.clamp(-6, 6)
    a = torch.where(a.abs() < 0.5, 0.0, a)  # (a scale of 1/2 leaves 1/4, which a scale of 1 has not)
    a = torch.where(a.abs() == 0.75, 1.0, a)
    wc, sw, w = _operand(n, k, 6)
    assert torch.equal(Q.mx_dequantize(*Q.mx_quantize(a.to(dtype))).double(), a)
    bias = torch.randint(-64, 64, (n,), device="cuda").float()
    want = (a @ w.T + bias).clamp(min=0).float().to(dtype)
    assert torch.equal(Q.mx_linear(a.to(dtype), wc, sw, bias=bias, relu=True), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_28672_values_are_encoded(dtype):
    import mx_oracle as MX

    x = (torch.randn(5, 28672, device="cuda") * torch.exp2(torch.randint(-9, 9, (5, 896, 1), device="cuda").float()).expand(5, 896, 32).reshape(5, -1)).to(dtype)
    codes, scales = Q.mx_quantize(x)
    ref_codes, ref_scales = MX.quantize(x.float().cpu().numpy())
    assert (codes.cpu().numpy() == ref_codes).all() and (scales.cpu().numpy() == ref_scales).all()
