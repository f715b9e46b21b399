"""Microscaled 4-bit floats (MXFP4) on the GPU: encode, decode, fake quantization with its gradient, the
product and the layers, against the NumPy oracle."""

import numpy as np
import pytest
import torch

import mx_oracle as MX

pytestmark = pytest.mark.gpu

import lucid_b200.nn.qat as nnqat  # noqa: E402
import lucid_b200.nn.quantized as nnq  # noqa: E402
import lucid_b200.quantization as Q  # noqa: E402
from gpu_util import dev, host  # noqa: E402
from lucid_b200 import _lib  # noqa: E402


def _sample(rng, rows, k, dtype):
    """Values over many binades, with ties of the element grid, zeros and signed zeros among them."""
    x = rng.standard_normal((rows, k)) * np.exp2(rng.integers(-12, 12, (rows, k // 32)).repeat(32, 1))
    ties = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.5, 0.0, -0.0], (rows, k)) * rng.choice([-1, 1], (rows, k))
    x = np.where(rng.random((rows, k)) < 0.3, ties, x)
    return torch.from_numpy(x.astype(np.float32)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 8192), (3, 96), (127, 256), (128, 288), (130, 1056), (257, 4096)])
def test_encode_and_decode_equal_the_oracle(rows, k, dtype):
    x = _sample(np.random.default_rng(rows + k), rows, k, dtype)
    codes, scales = Q.mx_quantize(x.cuda())
    ref_codes, ref_scales = MX.quantize(host(x.float()))
    assert np.array_equal(host(codes), ref_codes)
    assert np.array_equal(host(scales), ref_scales)  # the padding of the tiles is zero
    code, byte, _ = MX.encode(host(x.float()))
    for out in (torch.float32, torch.bfloat16):  # both types hold every value of the format
        y = Q.mx_dequantize(codes, scales, out_dtype=out)
        assert y.dtype == out and np.array_equal(host(y), MX.decode(code, byte).astype(np.float32))


def test_ends_of_the_range_and_values_without_a_number():
    x = np.zeros((8, 64), dtype=np.float32)
    x[0, :3] = 2.0 ** -149, 2.0 ** -127, 2.0 ** -126      # subnormal block: byte 0
    x[1, 5] = 3.0e38                                       # top of float32
    x[2, 7], x[2, 40] = np.nan, 1.0                        # one block of the row is lost, not the other
    x[3, 33] = np.inf
    x[4, :32] = -0.0
    x[5, :32] = 2.0 ** -128 * np.arange(32)
    x[6, 0], x[6, 1] = 7.99, -7.99                         # clamped at 6
    codes, scales = Q.mx_quantize(dev(x))
    ref_codes, ref_scales = MX.quantize(x)
    assert np.array_equal(host(codes), ref_codes) and np.array_equal(host(scales), ref_scales)
    code, byte, fits = MX.encode(x)
    y = host(Q.mx_dequantize(codes, scales))
    assert np.array_equal(y, MX.decode(code, byte).astype(np.float32), equal_nan=True)
    assert np.isnan(y[2, :32]).all() and y[2, 40] == 1.0 and np.isnan(y[3, 32:]).all() and y[6, 0] == 6.0
    t = dev(x).requires_grad_()
    out = Q.mx_fake_quantize(t)
    assert np.array_equal(host(out.detach()), y, equal_nan=True)
    out.backward(torch.ones_like(out))
    assert np.array_equal(host(t.grad), fits.astype(np.float32))


def test_strided_and_misaligned_inputs():
    rng = np.random.default_rng(3)
    base = _sample(rng, 40, 512, torch.bfloat16).cuda()
    for view in (base[::2], base[:, 64:320], base[:, 4:260], base.t()[:, :32], base.reshape(5, 8, 512)[:, ::3],
                 base.reshape(-1)[3:3 + 64 * 32].reshape(64, 32), base[:1].expand(7, 512)):
        codes, scales = Q.mx_quantize(view)
        ref_codes, ref_scales = MX.quantize(host(view.float()).reshape(-1, view.shape[-1]))
        assert codes.shape[:-1] == view.shape[:-1]
        assert np.array_equal(host(codes).reshape(ref_codes.shape), ref_codes) and np.array_equal(host(scales), ref_scales)


def test_empty_matrices():
    codes, scales = Q.mx_quantize(torch.empty(0, 64, device="cuda"))
    assert codes.shape == (0, 32) and scales.shape == (0, 1, 1024)
    assert Q.mx_dequantize(codes, scales).shape == (0, 64)
    w = Q.mx_quantize(torch.randn(8, 64, device="cuda"))
    assert Q.mx_matmul(codes, scales, *w).shape == (0, 8)
    assert Q.mx_linear(torch.randn(3, 64, device="cuda"), codes, scales).shape == (3, 0)
    t = torch.empty(0, 64, device="cuda", requires_grad=True)
    Q.mx_fake_quantize(t).sum().backward()
    assert t.grad.shape == (0, 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(32,), (3, 5, 96), (333, 1056)])
def test_fake_quantize_and_its_gradient(shape, dtype):
    rng = np.random.default_rng(len(shape))
    x = _sample(rng, int(np.prod(shape[:-1])), shape[-1], dtype).reshape(shape).cuda().requires_grad_()
    y = Q.mx_fake_quantize(x)
    code, byte, fits = MX.encode(host(x.detach().float()).reshape(-1, shape[-1]))
    assert y.dtype == dtype and np.array_equal(host(y.detach()), MX.decode(code, byte).astype(np.float32).reshape(shape))
    assert not fits.all() or len(shape) == 1
    g = torch.randn(shape, device="cuda").to(dtype)
    (gx,) = torch.autograd.grad(y, x, g)
    assert gx.dtype == dtype and np.array_equal(host(gx), np.where(fits.reshape(shape), host(g), 0.0))
    # an expanded gradient, and the second derivative of something that is linear in the gradient
    leaf = x.detach().clone().requires_grad_()
    Q.mx_fake_quantize(leaf).sum().backward()
    assert np.array_equal(host(leaf.grad), fits.reshape(shape).astype(np.float32))
    g2 = torch.randn(shape, device="cuda", requires_grad=True)
    if dtype == torch.float32:
        (gx,) = torch.autograd.grad(Q.mx_fake_quantize(x), x, g2, create_graph=True)
        (gg,) = torch.autograd.grad(gx.sum(), g2)
        assert np.array_equal(host(gg), fits.reshape(shape).astype(np.float32))
    with torch.no_grad():
        assert torch.equal(Q.mx_fake_quantize(x), y)


def test_the_gradient_is_that_of_rounding_away_from_the_steps():
    """Against differences: over a whole step of the element grid the quantized value moves as far as the
    input does (slope 1); past the clamp it does not move."""
    scale = 0.25
    x = torch.zeros(1, 32, device="cuda")
    x[0, 0] = 7.5 * scale                       # fixes the block's scale, itself clamped
    x[0, 1], x[0, 2] = 2.0 * scale, 1.0 * scale
    up = x.clone()
    up[0, 0], up[0, 1], up[0, 2] = 7.75 * scale, 3.0 * scale, 1.5 * scale
    t = x.clone().requires_grad_()
    Q.mx_fake_quantize(t).sum().backward()
    slope = (Q.mx_fake_quantize(up) - Q.mx_fake_quantize(x))[0, :3] / (up - x)[0, :3]
    assert slope.tolist() == [0.0, 1.0, 1.0] and t.grad[0, :3].tolist() == [0.0, 1.0, 1.0]


# ---- the product ---------------------------------------------------------------------------------


def _grid(rng, rows, k, spread):
    """Random codes and scale bytes: with spread 0 every sum of products is a small multiple of 1/4 and
    so exact in float32 in any order."""
    code = rng.integers(0, 16, (rows, k)).astype(np.uint8)
    byte = rng.integers(127 - spread, 128 + spread, (rows, k // 32)).astype(np.uint8)
    return code, byte


def _to_device(code, byte):
    return dev(MX.pack(code)), dev(MX.tile(byte))


SHAPES = [(1, 32, 16), (1, 64, 1), (1, 8192, 300), (2, 96, 128), (5, 256, 129), (8, 320, 200), (9, 288, 1000), (16, 4096, 256),
          (17, 512, 384), (33, 1056, 130), (64, 992, 520), (65, 2048, 257), (100, 4096, 640), (128, 256, 128), (129, 1056, 1003),
          (200, 64, 72), (256, 512, 256), (257, 736, 515), (300, 32, 2000), (777, 1056, 1003), (1024, 2048, 1024),
          # tiles of 128 tokens, then CTA pairs: few and many stages, several tiles to a pair, ragged ends
          (1000, 352, 4096), (1300, 800, 4100), (2050, 32, 2561), (700, 4224, 8200), (129, 1312, 20001), (3000, 2048, 2600)]


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_product_is_exact_where_float32_is(m, k, n):
    rng = np.random.default_rng(m * 7 + k + n)
    a, w = _grid(rng, m, k, 0), _grid(rng, n, k, 0)
    bias = rng.integers(-64, 64, n).astype(np.float32)
    ref = MX.decode(*a) @ MX.decode(*w).T
    y = Q.mx_matmul(*_to_device(*a), *_to_device(*w))
    assert y.dtype == torch.float32 and np.array_equal(host(y), ref.astype(np.float32))
    y = Q.mx_matmul(*_to_device(*a), *_to_device(*w), bias=dev(bias), relu=True, out_dtype=torch.bfloat16)
    want = torch.from_numpy(np.maximum(ref + bias, 0.0).astype(np.float32)).to(torch.bfloat16)
    assert y.dtype == torch.bfloat16 and torch.equal(y.cpu(), want)
    _lib.check_device_status(y.device)


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_product_with_scales_of_every_size(m, k, n):
    """Float32 sums in an order the kernel chooses: at most K additions, each off by 2^-24 of the sum of
    magnitudes when it rounds and by twice that when it truncates."""
    rng = np.random.default_rng(m + k * 3 + n)
    a, w = _grid(rng, m, k, 9), _grid(rng, n, k, 9)
    da, dw = MX.decode(*a), MX.decode(*w)
    ref, size = da @ dw.T, np.abs(da) @ np.abs(dw).T
    y = host(Q.mx_matmul(*_to_device(*a), *_to_device(*w)))
    assert (np.abs(y - ref) <= (k * 2.0 ** -23 + 2.0 ** -24) * size).all()


def test_products_with_nan_blocks_and_extreme_scales():
    rng = np.random.default_rng(11)
    a, w = _grid(rng, 40, 512, 0), _grid(rng, 150, 512, 0)
    a[1][3, 5] = 255                       # one block of one row: that row of the result is NaN
    w[1][140, 0] = 255
    a[1][7, :], w[1][9, :] = 20, 230       # 2^-107 against 2^103
    ref = MX.decode(*a) @ MX.decode(*w).T
    y = host(Q.mx_matmul(*_to_device(*a), *_to_device(*w)))
    assert np.isnan(y[3]).all() and np.isnan(y[:, 140]).all()
    keep = ~np.isnan(ref)
    assert np.array_equal(np.isnan(y), ~keep) and np.array_equal(y[keep], ref[keep].astype(np.float32))


@pytest.mark.parametrize("m,n", [(3, 300), (70, 300), (1300, 4100), (1000, 4096)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_the_result_may_lie_apart(m, n, dtype):
    """The C entry's row stride: columns past N and rows past M stay as they were."""
    rng = np.random.default_rng(m)
    a, w = _grid(rng, m, 288, 0), _grid(rng, n, 288, 0)
    ac, sa, wc, sw = *_to_device(*a), *_to_device(*w)
    ref = torch.from_numpy((MX.decode(*a) @ MX.decode(*w).T).astype(np.float32)).to(dtype)
    for ldo in (n + 5, n + 8):
        out = torch.full((m + 2, ldo), -7.0, dtype=dtype, device="cuda")
        _lib.call("lq_mx_matmul", out.device, ac.data_ptr(), sa.data_ptr(), m, wc.data_ptr(), sw.data_ptr(), n, 288, None, 0,
                  out.data_ptr(), _lib.code_of(dtype), ldo, None)
        assert torch.equal(out[:m, :n].cpu(), ref) and (out[:m, n:] == -7.0).all() and (out[m:] == -7.0).all()


def test_relu_keeps_nan():
    a, w = Q.mx_quantize(torch.full((2, 32), float("nan"), device="cuda")), Q.mx_quantize(torch.ones(3, 32, device="cuda"))
    assert torch.isnan(Q.mx_matmul(*a, *w, relu=True)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lead,k,n", [((1,), 2048, 512), ((1,), 32, 8), ((3, 5), 96, 40), ((8,), 8192, 130), ((9,), 1312, 257),
                                      ((16,), 4096, 384), ((17,), 4096, 384), ((130,), 1056, 1003), ((2, 1, 40), 512, 8)])
def test_linear_is_quantize_and_product(lead, k, n, dtype):
    rng = np.random.default_rng(k + n)
    x = _sample(rng, int(np.prod(lead)), k, dtype).reshape(*lead, k).cuda()
    w = Q.mx_quantize(dev(rng.standard_normal((n, k)).astype(np.float32)))
    bias = dev(rng.standard_normal(n).astype(np.float32))
    y = Q.mx_linear(x, *w, bias=bias, relu=True)
    assert y.shape == (*lead, n) and y.dtype == dtype
    assert torch.equal(y, Q.mx_matmul(*Q.mx_quantize(x), *w, bias=bias, relu=True, out_dtype=dtype))
    strided = torch.cat((x, x), -1)[..., :k]
    assert torch.equal(Q.mx_linear(strided, *w, bias=bias, relu=True), y)
    apart = torch.empty(*lead, k + 24, dtype=dtype, device="cuda")[..., 8:8 + k]  # 16-byte, not 32-byte aligned rows of bf16
    apart.copy_(x)
    assert torch.equal(Q.mx_linear(apart, *w, bias=bias, relu=True), y)
    poisoned = x.clone()
    poisoned.view(-1, k)[0, k - 1] = float("inf")
    assert torch.isnan(Q.mx_linear(poisoned, *w).view(-1, n)[0]).all()


def test_layer_state_dict_and_workflows():
    import lucid_b200.backends as backends

    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(128, 256), torch.nn.ReLU(), torch.nn.Linear(256, 80),
                                torch.nn.ReLU(), torch.nn.Linear(80, 16)).cuda().eval()
    x = torch.randn(8, 128, device="cuda")
    with torch.no_grad(), _lib.ieee_float32():
        y_float = model(x)
    old = backends.quantized.engine
    backends.quantized.engine = "mxfp4"
    try:
        assert backends.quantized.use_mx() and not backends.quantized.use_int8()
        prepared = Q.prepare(model)
        prepared(x)
        qmodel, dmodel = Q.convert(prepared), Q.quantize_dynamic(model)
        qat = Q.prepare_qat(model)
    finally:
        backends.quantized.engine = old
    assert type(qmodel[0]) is nnq.MXLinear and type(qmodel[2]) is nnq.MXLinear and type(qmodel[4]) is nnq.Linear
    assert type(dmodel[0]) is nnq.MXLinear and type(dmodel[4]) is nnq.dynamic.Linear
    assert type(qat[0]) is nnqat.MXLinear and type(qat[4]) is nnqat.Linear
    # the QAT forward is the quantized one: the same rounded operands, sums in another order
    layer = qat[0]
    trained = nnq.MXLinear.from_float(layer)
    a, w = Q.mx_fake_quantize(x), Q.mx_fake_quantize(layer.weight.detach())
    size = a.abs() @ w.abs().T + layer.bias.abs()
    with torch.no_grad(), _lib.ieee_float32():
        assert ((trained(x) - layer(x)).abs() <= 2 * 130 * 2.0 ** -23 * size).all()
    # gradients reach the weight through the straight-through rounding
    out = layer(x)
    out.backward(torch.ones_like(out))
    fits = MX.encode(host(layer.weight.detach()))[2]
    want = np.where(fits, host(a).sum(0)[None, :].repeat(256, 0), 0.0)
    bound = 8 * 2.0 ** -23 * host(a.abs()).sum(0)[None, :]
    assert (np.abs(host(layer.weight.grad) - want) <= bound).all()
    assert type(Q.convert(qat)[0]) is nnq.MXLinear
    other = nnq.MXLinear(128, 256).cuda()
    other.load_state_dict(qmodel[0].state_dict())
    assert torch.equal(other(x), qmodel[0](x)) and "mxfp4" in repr(other)
    # against the float layer: off by what rounding the operands moves, |x' - x| |w| + |x'| |w' - w|, and the sums'
    # own rounding (130 additions each side)
    xa, xb = x.double(), Q.mx_fake_quantize(x).double()
    wa, wb = model[0].weight.detach().double(), Q.mx_fake_quantize(model[0].weight.detach()).double()
    moved = (xb - xa).abs() @ wa.abs().T + xb.abs() @ (wb - wa).abs().T
    with torch.no_grad(), _lib.ieee_float32():
        apart = (qmodel[0](x).double() - model[0](x).double()).abs()
    assert (apart <= moved + 2 * 130 * 2.0 ** -23 * size.double()).all() and float(apart.max()) > 0


@pytest.mark.parametrize("rows", [4, 40])
def test_layers_one_after_the_other_see_each_other(rows):
    """A chain of products whose buffers are used again: launches that overlap."""
    ws = [Q.mx_quantize(torch.randn(256, 256, device="cuda") / 16) for _ in range(4)]
    x = torch.randn(rows, 256, device="cuda")
    y, want = x, x
    for i in range(40):
        y = Q.mx_linear(y, *ws[i % 4])
    for i in range(40):
        torch.cuda.synchronize()
        want = Q.mx_matmul(*Q.mx_quantize(want), *ws[i % 4])
    assert torch.isfinite(y).all() and torch.equal(y, want)


def test_captured_and_replayed():
    x = torch.randn(48, 512, device="cuda")
    w = Q.mx_quantize(torch.randn(384, 512, device="cuda"))
    Q.mx_linear(x, *w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        y = Q.mx_linear(x, *w)
    for seed in range(3):
        x.copy_(torch.randn(48, 512, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, Q.mx_linear(x, *w))


def test_captured_before_anything_else(monkeypatch):
    """A capture that is the first use makes no status word inside the graph's memory."""
    monkeypatch.setattr(_lib, "_status_words", {})
    x, w = torch.randn(4, 64, device="cuda"), Q.mx_quantize(torch.randn(8, 64, device="cuda"))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = Q.mx_linear(x, *w)
    assert _lib._status_words == {}
    graph.replay()
    assert torch.equal(y, Q.mx_linear(x, *w))


def test_training_step_captured_and_replayed():
    """(With no eager graph of the leaf alive: torch ties a leaf's gradient node to the stream of its first
    use, and refuses to capture a backward pass of any operator through a node of another stream.)"""
    leaf = torch.randn(64, 96, device="cuda", requires_grad=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(Q.mx_fake_quantize(leaf).sum(), leaf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (g,) = torch.autograd.grad(Q.mx_fake_quantize(leaf).sum(), leaf)
    with torch.no_grad():
        leaf.copy_(torch.randn(64, 96, device="cuda") * 3)
    graph.replay()
    assert np.array_equal(host(g), MX.encode(host(leaf.detach()))[2].astype(np.float32))


@pytest.mark.parametrize("rows,width", [(96, 640), (1300, 4100)])
def test_two_streams_at_once(rows, width):
    ws = [Q.mx_quantize(torch.randn(width, 2048, device="cuda")) for _ in range(2)]
    xs = [torch.randn(rows, 2048, device="cuda") for _ in range(2)]
    want = [Q.mx_linear(x, *w) for x, w in zip(xs, ws)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(Q.mx_linear(xs[i], *ws[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


def test_bad_arguments_raise():
    x = torch.randn(4, 64, device="cuda")
    codes, scales = Q.mx_quantize(x)
    with pytest.raises(_lib.ShapeMismatch):
        Q.mx_quantize(torch.randn(4, 48, device="cuda"))
    with pytest.raises(_lib.DtypeMismatch):
        Q.mx_quantize(x.half())
    with pytest.raises(_lib.DeviceMismatch):
        Q.mx_quantize(x.cpu())
    with pytest.raises(_lib.ShapeMismatch):
        Q.mx_dequantize(codes, scales[:, :0])
    with pytest.raises(_lib.DtypeMismatch):
        Q.mx_dequantize(codes, scales, out_dtype=torch.float16)
    with pytest.raises(_lib.ShapeMismatch):
        Q.mx_matmul(codes, scales, *Q.mx_quantize(torch.randn(4, 96, device="cuda")))
    with pytest.raises(_lib.ShapeMismatch):
        Q.mx_linear(x, codes, scales, bias=torch.zeros(5, device="cuda"))
    with pytest.raises(_lib.DeviceMismatch):
        Q.mx_linear(x, codes, scales, bias=torch.zeros(4))
    with pytest.raises(_lib.DtypeMismatch):
        Q.mx_matmul(codes.to(torch.int8), scales, codes, scales)
