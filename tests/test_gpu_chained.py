"""Launches that overlap, each reading what the kernel right before it rewrote in place."""

import pytest
import torch

pytestmark = pytest.mark.gpu

import lucid_b200.quantization as Q  # noqa: E402
from lucid_b200 import _lib  # noqa: E402


def _product_into(out, a, w):
    """``out`` = a @ w.T by the library's own product, into memory that is used again and again."""
    (ac, sa), (wc, sw) = a, w
    m, n = out.shape
    _lib.call("lq_mx_matmul", out.device, ac.data_ptr(), sa.data_ptr(), m, wc.data_ptr(), sw.data_ptr(), n, ac.shape[1] * 2, None,
              0, out.data_ptr(), _lib.code_of(out.dtype), n, _lib.status_ptr(out.device))


@pytest.mark.parametrize("tokens", [40, 300, 1500])
@pytest.mark.parametrize("fmt", ["int8", "mxfp4"])
def test_rows_and_slots_rewritten_before_each_write(fmt, tokens):
    heads, dim, page, steps = 4, 64, 16, 12
    pages = -(-tokens // page) + 2
    a = [Q.mx_quantize(torch.randn(tokens, 256, device="cuda")) for _ in range(steps)]
    w = [Q.mx_quantize(torch.randn(heads * dim, 256, device="cuda")) for _ in range(2)]
    order = [torch.randperm(pages * page, device="cuda")[:tokens] for _ in range(steps)]
    k, v = (torch.zeros(tokens, heads * dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots = torch.empty(tokens, dtype=torch.int64, device="cuda")
    got, want = ([Q.kv_cache_alloc(pages, page, heads, dim, fmt) for _ in range(steps)] for _ in range(2))

    def run(caches, between):
        for i in range(steps):
            slots.copy_(order[i])
            between()
            _product_into(k, a[i], w[0])
            between()
            _product_into(v, a[i], w[1])
            between()
            Q.kv_cache_write(caches[i], k.view(tokens, heads, dim), v.view(tokens, heads, dim), slots)
            between()

    torch.cuda.synchronize()
    run(got, lambda: None)
    torch.cuda.synchronize()
    run(want, torch.cuda.synchronize)
    for x, y in zip(got, want):
        assert all(torch.equal(s, t) for s, t in zip(x, y)) and int(x.k_codes.view(torch.uint8).max()) > 0
    _lib.check_device_status(k.device)


@pytest.mark.parametrize("rows,n", [(4, 200), (30, 300), (60, 300), (200, 4200), (700, 4200), (1300, 4100)])
def test_weights_encoded_in_place_before_each_product(rows, n):
    """Every form of the product: fused, one tile a CTA of 32, 64 and 128 tokens, CTA pairs."""
    k, steps = 512, 8
    src = [torch.randn(n, k, device="cuda") for _ in range(steps)]
    x = [torch.randn(rows, k, device="cuda") for _ in range(steps)]
    wc, sw = Q.mx_quantize(src[0])

    def run(between):
        ys = []
        for i in range(steps):
            _lib.call("lq_mx_quantize", wc.device, src[i].data_ptr(), _lib.code_of(torch.float32), n, k, k, wc.data_ptr(), sw.data_ptr())
            between()
            ys.append(Q.mx_linear(x[i], wc, sw))
            between()
        return ys

    torch.cuda.synchronize()
    got = run(lambda: None)
    torch.cuda.synchronize()
    want = run(torch.cuda.synchronize)
    assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(got, want))
    _lib.check_device_status(wc.device)


@pytest.mark.parametrize("tokens", [20, 700])
@pytest.mark.parametrize("fmt", ["int8", "mxfp4"])
def test_two_captured_steps_replayed_in_turn(fmt, tokens):
    """Two graphs of write and read, each with workspaces of its own, replayed alternately with new rows, and an
    eager step on another stream in between."""
    heads, dim, page = 2, 64, 16
    pages = -(-tokens // page)
    caches = [Q.kv_cache_alloc(pages, page, heads, dim, fmt) for _ in range(3)]
    rows = [torch.zeros(tokens, heads, dim, device="cuda") for _ in range(3)]
    slots = [torch.randint(-2, pages * page, (tokens,), device="cuda") for _ in range(3)]
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    cu = torch.tensor([0, pages * page], dtype=torch.int32, device="cuda")

    def step(i):
        Q.kv_cache_write(caches[i], rows[i], -rows[i], slots[i])
        return Q.kv_cache_read(caches[i], table, cu, pages * page, out_dtype=torch.bfloat16)

    step(0)
    graphs, outs = [], []
    for i in range(2):
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(step(i))
    side = torch.cuda.Stream()
    for turn in range(4):
        for i in range(3):
            rows[i].copy_(torch.randn(tokens, heads, dim, device="cuda"))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step(2)
        for i in (0, 1, 0):
            graphs[i].replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in (*outs, other)]
        for i in range(3):
            for t in caches[i]:
                t.zero_()
            want = step(i)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) and b.any() for a, b in zip(got[i], want)), (turn, i)
    _lib.check_device_status(cu.device)
