"""Derivatives of the MXFP4 fake quantization on the CPU: the host logic over a NumPy restatement of its two entries."""

import ctypes

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import lucid_b200.quantization as Q
import mx_oracle as MX
from lucid_b200 import _lib


def _at(p, n, dt):
    return np.frombuffer((ctypes.c_char * (n * np.dtype(dt).itemsize)).from_address(p), dtype=dt)


def _numpy_call(name, device, *args):
    if name == "lq_mx_fake_quantize":
        x, _, n, out, mask = args
        code, byte, fits = MX.encode(_at(x, n, np.float32).reshape(1, n))
        _at(out, n, np.float32)[:] = MX.decode(code, byte).reshape(-1)
        if mask is not None:
            _at(mask, n // 8, np.uint8)[:] = np.packbits(fits.reshape(-1), bitorder="little")
    elif name == "lq_mx_fake_quantize_grad":
        grad, _, mask, n, out = args
        keep = np.unpackbits(_at(mask, n // 8, np.uint8), bitorder="little").astype(bool)
        _at(out, n, np.float32)[:] = np.where(keep, _at(grad, n, np.float32), 0.0)
    else:
        raise NotImplementedError(name)


@pytest.fixture(autouse=True)
def on_the_cpu(monkeypatch):
    monkeypatch.setattr(_lib, "require_cuda", lambda t, what: None)
    monkeypatch.setattr(_lib, "call", _numpy_call)


def _input():
    x = torch.linspace(-6.5, 6.5, 96).reshape(3, 32)
    x[1, 7] = 7.9  # clamped
    fits = torch.from_numpy(MX.encode(x.numpy())[2]).float()
    assert 0 < fits.sum() < 96
    return x, fits


def test_a_tangent_passes_as_the_gradient_does():
    x, fits = _input()
    t = torch.randn(3, 32)
    for grad_mode in (torch.enable_grad, torch.no_grad):
        with forward_ad.dual_level(), grad_mode():
            y = Q.mx_fake_quantize(forward_ad.make_dual(x, t))
            primal, tangent = forward_ad.unpack_dual(y)
            assert torch.equal(primal, Q.mx_fake_quantize(x)) and tangent is not None and torch.equal(tangent, t * fits)
            assert forward_ad.unpack_dual(Q.mx_fake_quantize(x)).tangent is None


def test_a_tangent_and_a_gradient_at_once():
    x, fits = _input()
    leaf = x.clone().requires_grad_()
    t = torch.randn(3, 32)
    with forward_ad.dual_level():
        y = Q.mx_fake_quantize(forward_ad.make_dual(leaf, t))
        # d/dx of (y^2 / 2) is y * fits; along t it moves by t * fits
        (g,) = torch.autograd.grad((y * y).sum() / 2, leaf)
        primal, tangent = forward_ad.unpack_dual(g)
        assert torch.equal(primal, Q.mx_fake_quantize(x) * fits)
        assert tangent is not None and torch.equal(tangent, t * fits)


def test_gradients_of_first_and_second_order():
    x, fits = _input()
    leaf = x.clone().requires_grad_()
    g = torch.randn(3, 32, requires_grad=True)
    (gx,) = torch.autograd.grad(Q.mx_fake_quantize(leaf), leaf, g, create_graph=True)
    assert torch.equal(gx, g * fits)
    (gg,) = torch.autograd.grad(gx.sum(), g)
    assert torch.equal(gg, fits)
    Q.mx_fake_quantize(leaf).sum().backward()
    assert torch.equal(leaf.grad, fits)


def test_transforms_are_refused():
    x, _ = _input()
    for f in (lambda: torch.func.jvp(Q.mx_fake_quantize, (x,), (x,)), lambda: torch.func.grad(lambda t: Q.mx_fake_quantize(t).sum())(x),
              lambda: torch.func.vmap(Q.mx_fake_quantize)(x)):
        with pytest.raises(RuntimeError):
            f()
