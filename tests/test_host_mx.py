"""CPU checks of the microscaled and cache operators: what the C entries refuse, and which layers the
workflows build under the "mxfp4" engine."""

import ctypes

import numpy as np
import pytest
import torch

import lucid_b200
import lucid_b200.nn.qat as nnqat
import lucid_b200.nn.quantized as nnq
import lucid_b200.quantization as Q
import mx_oracle as MX
from lucid_b200 import _lib


def test_oracle_rounds_ties_to_the_even_mantissa():
    x = np.zeros((1, 32))
    x[0, :12] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.9, 7.0, -0.25, 0.3, 4.0]
    code, byte, fits = MX.encode(x)
    assert byte.tolist() == [[127]]
    assert MX.decode(code, byte)[0, :12].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, 6, 0, 0.5, 4]
    assert fits[0, :9].tolist() == [True] * 8 + [False]
    assert np.array_equal(MX.unpack(MX.pack(code)), code)


def test_c_entries_refuse_without_a_gpu():
    lib = _lib.load()
    one, odd = ctypes.c_void_p(16), ctypes.c_void_p(8)
    assert lib.lq_mx_scale_bytes(1, 32) == 1024 and lib.lq_mx_scale_bytes(129, 257) == 4096 and lib.lq_mx_scale_bytes(0, 64) == 0
    assert lib.lq_mx_linear_workspace_bytes(16, 64) == 0 and lib.lq_mx_linear_workspace_bytes(17, 64) == 1024 + 1024
    q = [one, 0, 4, 64, 64, one, one, None]
    assert lib.lq_mx_quantize(None, 0, 0, 64, 64, None, None, None) == 0  # nothing to do
    assert lib.lq_mx_quantize(None, *q[1:]) == 3
    assert lib.lq_mx_quantize(one, 2, *q[2:]) == 2
    assert lib.lq_mx_quantize(one, 0, 4, 48, 48, *q[5:]) == 1
    assert lib.lq_mx_quantize(one, 0, 4, 64, 32, *q[5:]) == 1  # rows overlap
    assert lib.lq_mx_quantize(one, 0, 4, 64, 66, *q[5:]) == 4
    assert lib.lq_mx_quantize(odd, *q[1:]) == 4
    assert lib.lq_mx_dequantize(one, one, 4, 64, one, 4, None) == 2
    assert lib.lq_mx_dequantize(one, one, 4, 40, one, 0, None) == 1
    assert lib.lq_mx_dequantize(one, None, 4, 64, one, 0, None) == 3
    assert lib.lq_mx_fake_quantize(one, 0, 33, one, None, None) == 1
    assert lib.lq_mx_fake_quantize(one, 3, 32, one, None, None) == 2
    assert lib.lq_mx_fake_quantize_grad(one, 0, None, 32, one, None) == 3
    mm = [one, one, 4, one, one, 8, 64, None, 0, one, 0, 8, None, None]
    assert lib.lq_mx_matmul(*mm[:2], 0, *mm[3:]) == 0
    assert lib.lq_mx_matmul(None, *mm[1:]) == 3
    assert lib.lq_mx_matmul(*mm[:6], 80, *mm[7:]) == 1
    assert lib.lq_mx_matmul(*mm[:10], 2, *mm[11:]) == 2
    assert lib.lq_mx_matmul(*mm[:11], 7, *mm[12:]) == 1
    assert lib.lq_mx_matmul(odd, *mm[1:]) == 4
    assert lib.lq_mx_matmul(*mm[:2], 1 << 40, *mm[3:]) == 1
    lin = [one, 0, 20, 64, one, one, 8, 64, None, 0, one, 0, 8, one, 1 << 20, None, None]
    assert lib.lq_mx_linear(*lin[:14], 16, *lin[15:]) == 6
    assert lib.lq_mx_linear(*lin[:13], None, *lin[14:]) == 3
    assert lib.lq_mx_linear(one, 5, *lin[2:]) == 2 and lib.lq_mx_linear(one, 5, 4, *lin[3:]) == 2
    assert lib.lq_mx_linear(None, 0, 4, *lin[3:]) == 3 and lib.lq_mx_linear(odd, 0, 4, *lin[3:]) == 4
    assert lib.lq_mx_linear(one, 0, 4, 32, *lin[4:]) == 1 and lib.lq_mx_linear(one, 0, 4, 66, *lin[4:]) == 4
    kw = [one, one, 1, 4, 2, 64, 128, 64, 128, 64, one, 64, 32, 0, one, one, one, one, None, 0, None, None]
    assert lib.lq_kv_write_workspace_bytes(256) == 0 and lib.lq_kv_write_workspace_bytes(257) == 257
    assert lib.lq_kv_write(*kw[:3], 300, *kw[4:]) == 6
    assert lib.lq_kv_write(*kw[:3], 1 << 31, *kw[4:]) == 1
    assert lib.lq_kv_write(None, None, 1, 0, *kw[4:]) == 0
    assert lib.lq_kv_write(None, *kw[1:]) == 3
    assert lib.lq_kv_write(*kw[:2], 4, *kw[3:]) == 2
    assert lib.lq_kv_write(*kw[:11], 16, *kw[12:]) == 2
    assert lib.lq_kv_write(*kw[:13], 2, *kw[14:]) == 5
    assert lib.lq_kv_write(*kw[:5], 24, *kw[6:]) == 1
    assert lib.lq_kv_write(*kw[:5], 2048, *kw[6:]) == 1
    assert lib.lq_kv_write(*kw[:6], 129, *kw[7:]) == 4
    kr = [one, one, one, one, 1, 4, 16, 2, 64, one, 1, 1, one, None, 1, 8, one, one, 0, 128, 64, 128, 64, 0, None, None]
    assert lib.lq_kv_read(*kr[:15], 0, *kr[16:]) == 0
    assert lib.lq_kv_read(*kr[:12], None, *kr[13:]) == 3
    assert lib.lq_kv_read(*kr[:18], 2, *kr[19:]) == 2
    assert lib.lq_kv_read(*kr[:8], 80, *kr[9:]) == 1
    assert lib.lq_kv_read(*kr[:6], 0, *kr[7:]) == 1
    assert lib.lq_kv_read(*kr[:19], 127, *kr[20:]) == 4


def test_cpu_tensors_and_shapes_are_refused():
    x = torch.randn(4, 64)
    with pytest.raises(lucid_b200.DeviceMismatch):
        Q.mx_quantize(x)
    with pytest.raises(lucid_b200.DeviceMismatch):
        Q.mx_fake_quantize(x)
    with pytest.raises(lucid_b200.DeviceMismatch):
        nnq.MXLinear(64, 8)(x)
    with pytest.raises(lucid_b200.ShapeMismatch):
        nnq.MXLinear(48, 8)
    with pytest.raises(lucid_b200.ShapeMismatch):
        nnqat.MXLinear(48, 8)
    with pytest.raises(lucid_b200.DeviceMismatch):
        Q.kv_cache_write(Q.KVCache(*(torch.zeros(1, 1, 1, 16),) * 4), x, x, x)
    cache = Q.kv_cache_alloc(3, 4, 2, 64, "mxfp4", device="cpu")
    assert [tuple(t.shape) for t in cache] == [(3, 4, 2, 32), (3, 4, 2, 2)] * 2
    module = nnq.PagedKVCache(3, 4, 2, 64)
    assert list(module.state_dict()) == [] and module.cache.k_codes.shape == (3, 4, 2, 64) and not module.k_codes.is_cuda
    lin = nnq.MXLinear(288, 130)
    assert {k: tuple(v.shape) for k, v in lin.state_dict().items()} == {
        "weight_codes": (130, 144), "weight_scales": (2, 2, 1024), "bias": (130,)}


def _numpy_call(name, device, *args):
    """The two entries a converted layer reaches, on host memory."""
    def at(p, n, dt):
        return np.frombuffer((ctypes.c_char * (n * np.dtype(dt).itemsize)).from_address(p), dtype=dt)

    if name == "lq_mx_quantize":
        x, _, rows, k, ldx, codes, scales = args
        c, s = MX.quantize(at(x, rows * ldx, np.float32).reshape(rows, ldx)[:, :k])
        at(codes, c.size, np.uint8)[:] = c.reshape(-1)
        at(scales, s.size, np.uint8)[:] = s.reshape(-1)
    elif name == "lq_mx_linear":
        x, _, m, ldx, wc, ws, n, k, bias, relu, out, _, ldo = args[:13]
        code, byte, _ = MX.encode(at(x, m * ldx, np.float32).reshape(m, ldx)[:, :k])
        tiles = at(ws, (n + 127) // 128 * ((k + 255) // 256) * 1024, np.uint8).reshape(-1, (k + 255) // 256, 1024)
        r, b = np.meshgrid(np.arange(n), np.arange(k // 32), indexing="ij")
        wb = tiles[r // 128, b // 8, b % 8 // 4 * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4]
        y = MX.decode(code, byte) @ MX.decode(MX.unpack(at(wc, n * k // 2, np.uint8).reshape(n, -1)), wb).T
        y = y + (0.0 if bias is None else at(bias, n, np.float32))
        at(out, m * ldo, np.float32).reshape(m, ldo)[:, :n] = np.maximum(y, 0.0) if relu else y
    else:
        raise NotImplementedError(name)


def test_workflows_route_the_linear_family(monkeypatch):
    import abi_standin
    from lucid_b200 import backends

    with pytest.raises(ValueError):
        backends.quantized.engine = "mxfp8"
    abi_standin.install(monkeypatch, engine="mxfp4")
    monkeypatch.setattr(_lib, "call", _numpy_call)
    monkeypatch.setattr(_lib, "status_ptr", lambda device: None)
    assert backends.quantized.use_mx() and not backends.quantized.use_mlx() and not backends.quantized.use_int8()
    torch.manual_seed(1)
    net = torch.nn.Sequential(torch.nn.Linear(96, 160), torch.nn.ReLU(), torch.nn.Linear(160, 48), torch.nn.Linear(48, 8)).eval()
    x = torch.randn(20, 96)
    prepared = Q.prepare(Q.fuse_modules(net, [["0", "1"]]))
    with torch.no_grad():
        prepared(x)
    qnet = Q.convert(prepared)
    assert type(qnet[0]) is nnq.MXLinear and qnet[0].relu and type(qnet[2]) is nnq.MXLinear and not qnet[2].relu
    assert type(qnet[3]) is nnq.Linear  # 48 features: no whole blocks
    h = np.maximum(MX.decode(*MX.encode(x.numpy())[:2]) @ MX.decode(*MX.encode(net[0].weight.detach().numpy())[:2]).T
                   + net[0].bias.detach().numpy(), 0.0)
    assert np.allclose(qnet[0](x).numpy(), h, rtol=0, atol=160 * 2.0 ** -24 * np.abs(h).max() * 4)
    dyn = Q.quantize_dynamic(net)
    assert type(dyn[0]) is nnq.MXLinear and type(dyn[3]) is nnq.dynamic.Linear
    qat = Q.prepare_qat(net)
    assert type(qat[0]) is nnqat.MXLinear and type(qat[3]) is nnqat.Linear and qat.training
    assert type(Q.convert(qat)[0]) is nnq.MXLinear
    root = Q.convert(Q.prepare_qat(torch.nn.Linear(64, 8)))
    assert type(root) is nnq.MXLinear
