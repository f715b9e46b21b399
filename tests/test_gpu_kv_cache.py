"""The quantized key / value cache on the GPU against the NumPy oracle."""

import numpy as np
import pytest
import torch

import mx_oracle as MX

pytestmark = pytest.mark.gpu

import lucid_b200.nn.quantized as nnq  # noqa: E402
import lucid_b200.quantization as Q  # noqa: E402
from gpu_util import dev, host  # noqa: E402
from lucid_b200 import _lib  # noqa: E402


def _encode(x, fmt):
    """float32 (..., dim) -> (codes, scales) as the cache holds them."""
    flat = x.reshape(-1, x.shape[-1])
    if fmt == "int8":
        codes, scale = MX.int8_rows(flat)
        return codes.reshape(x.shape), scale.reshape(x.shape[:-1])
    code, byte, _ = MX.encode(flat)
    return MX.pack(code).reshape(*x.shape[:-1], -1), byte.reshape(*x.shape[:-1], -1)


def _decode(codes, scales, fmt):
    """Values rounded to float32: the product of a code and its scale is one float32 multiplication."""
    if fmt == "int8":
        return codes.astype(np.float32) * scales[..., None]
    flat = MX.unpack(codes).reshape(-1, codes.shape[-1] * 2)
    return MX.decode(flat, scales.reshape(len(flat), -1)).astype(np.float32).reshape(*codes.shape[:-1], -1)


def _filled(rng, pages, page, heads, dim, fmt):
    old = [rng.standard_normal((pages, page, heads, dim)).astype(np.float32) for _ in range(2)]
    (kc, ks), (vc, vs) = (_encode(o, fmt) for o in old)
    return Q.KVCache(dev(kc), dev(ks), dev(vc), dev(vs)), [kc, ks, vc, vs]


def _put(ref, k, v, slots, fmt):
    for side, x in ((0, k), (2, v)):
        codes, scales = _encode(x, fmt)
        c = ref[side].reshape(-1, *ref[side].shape[2:])
        s = ref[side + 1].reshape(-1, *ref[side + 1].shape[2:])
        for i, slot in enumerate(slots):
            if 0 <= slot < len(c):
                c[slot], s[slot] = codes[i], scales[i]


CASES = [("int8", 128, 8, 16), ("int8", 64, 1, 1), ("int8", 80, 3, 7), ("int8", 16, 2, 32), ("int8", 256, 5, 24), ("int8", 576, 1, 64),
         ("int8", 1024, 2, 3), ("mxfp4", 128, 8, 16), ("mxfp4", 32, 1, 5), ("mxfp4", 96, 4, 24), ("mxfp4", 64, 3, 1),
         ("mxfp4", 576, 2, 16), ("mxfp4", 1024, 1, 9)]


@pytest.mark.parametrize("fmt,dim,heads,page", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens", [1, 37])
def test_rows_are_encoded_in_place(fmt, dim, heads, page, dtype, tokens):
    rng = np.random.default_rng(dim + heads + page + tokens)
    pages = 64 // page + 3
    cache, ref = _filled(rng, pages, page, heads, dim, fmt)
    k, v = (torch.from_numpy((rng.standard_normal((tokens, heads, dim)) * 3).astype(np.float32)).to(dtype) for _ in range(2))
    k[0, 0] = 0.0  # a row of zeros
    slots = rng.permutation(pages * page)[:tokens]
    slots[rng.random(tokens) < 0.1] = -1
    Q.kv_cache_write(cache, k.cuda(), v.cuda(), dev(slots).to(torch.int64 if tokens > 1 else torch.int32))
    _put(ref, host(k.float()), host(v.float()), slots, fmt)
    for got, want in zip(cache, ref):  # the rows written, and every other row as it was
        assert np.array_equal(host(got), want)
    _lib.check_device_status(cache.k_codes.device)


def test_int8_rows_are_those_of_the_per_token_encode():
    x = torch.randn(50, 4, 128, device="cuda", dtype=torch.bfloat16)
    cache = Q.kv_cache_alloc(4, 16, 4, 128)
    Q.kv_cache_write(cache, x, x * 2, torch.arange(50, device="cuda"))
    codes, scales = Q.quantize_per_token(x.reshape(-1, 128), Q.qint8)
    assert torch.equal(cache.k_codes.reshape(-1, 128)[:200], codes) and torch.equal(cache.k_scales.reshape(-1)[:200], scales)


@pytest.mark.parametrize("tokens", [40, 200, 5000, 33000])
def test_of_two_rows_for_one_slot_the_later_stays(tokens):
    rng = np.random.default_rng(tokens)
    cache = Q.kv_cache_alloc(8, 16, 2, 16)
    k = torch.randn(tokens, 2, 16, device="cuda")
    slots = rng.integers(-20, 128, tokens)
    for _ in range(3):
        Q.kv_cache_write(cache, k, -k, dev(slots))
    codes, scales = MX.int8_rows(host(k).reshape(-1, 16))
    codes, scales = codes.reshape(tokens, 2, 16), scales.reshape(tokens, 2)
    last = {s: i for i, s in enumerate(slots) if s >= 0}
    got_c, got_s = host(cache.k_codes).reshape(128, 2, 16), host(cache.k_scales).reshape(128, 2)
    got_v = host(cache.v_codes).reshape(128, 2, 16)
    for s in range(128):
        want_c, want_s = (codes[last[s]], scales[last[s]]) if s in last else (0, 0)
        assert np.array_equal(got_c[s], np.broadcast_to(want_c, (2, 16))) and np.array_equal(got_s[s], np.broadcast_to(want_s, 2))
        if s in last:
            assert np.array_equal(got_v[s], MX.int8_rows(-host(k)[last[s]])[0])


def test_slots_past_the_cache_are_skipped_and_reported():
    cache = Q.kv_cache_alloc(2, 4, 1, 32, fmt="mxfp4")
    x = torch.ones(3, 1, 32, device="cuda")
    Q.kv_cache_write(cache, x, x, torch.tensor([8, 2 ** 40, 1], device="cuda"))
    with pytest.raises(_lib.ShapeMismatch):
        _lib.check_device_status(x.device)
    rows = cache.k_codes.reshape(8, -1)
    assert int(rows[1].max()) > 0 and int(rows[0].max()) == 0 and int(rows[2:].max()) == 0
    Q.kv_cache_write(cache, x, x, torch.tensor([-1, -2 ** 40, -8], device="cuda"))
    _lib.check_device_status(x.device)
    assert int(rows[2:].max()) == 0


@pytest.mark.parametrize("fmt", ["int8", "mxfp4"])
def test_rows_without_a_number_read_back_as_nan(fmt):
    cache = Q.kv_cache_alloc(1, 4, 2, 64, fmt=fmt)
    x = torch.randn(2, 2, 64, device="cuda")
    x[0, 1, 3], x[1, 0, 40] = float("nan"), float("-inf")
    Q.kv_cache_write(cache, x, x, torch.arange(2, device="cuda"))
    k, _ = Q.kv_cache_read(cache, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                           torch.tensor([0, 2], dtype=torch.int32, device="cuda"), 2)
    lost = torch.isnan(k)
    lo, hi = (0, 64) if fmt == "int8" else (0, 32)
    assert lost[0, 1, lo:hi].all() and lost[1, 0, 40] and not lost[0, 0].any() and not lost[1, 1].any()
    if fmt == "mxfp4":
        assert not lost[0, 1, 32:].any() and not lost[1, 0, :32].any()


@pytest.mark.parametrize("fmt,dim,heads,page", CASES)
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_read_back(fmt, dim, heads, page, out):
    """Ragged sequences, empty ones among them, pages that end inside a sequence, first tokens skipped."""
    rng = np.random.default_rng(dim * heads + page)
    lens, starts = [5, 0, 1, 2 * page, 61, 0], [0, 3, page, 1, 7, 0]
    width = max(-(-(t + s) // page) for t, s in zip(lens, starts))
    pages = width * len(lens) + 2
    cache, ref = _filled(rng, pages, page, heads, dim, fmt)
    table = rng.permutation(pages)[: width * len(lens)].reshape(len(lens), width).astype(np.int32)
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    args = (cache, dev(table), dev(cu))
    for st in (None, dev(np.array(starts, dtype=np.int32))):
        begin = np.zeros(len(lens), int) if st is None else starts
        at = np.concatenate([table[b, (begin[b] + np.arange(t)) // page] * page + (begin[b] + np.arange(t)) % page
                             for b, t in enumerate(lens)]).astype(int)
        want = [torch.from_numpy(_decode(c.reshape(-1, *c.shape[2:])[at], s.reshape(-1, *s.shape[2:])[at], fmt)).to(out)
                for c, s in ((ref[0], ref[1]), (ref[2], ref[3]))]
        total = int(cu[-1])
        got = Q.kv_cache_read(*args, total, starts=st, out_dtype=out)
        assert all(g.dtype == out and torch.equal(g.cpu(), w) for g, w in zip(got, want))
        # heads outermost, one buffer for both, rows behind the last sequence kept
        buf = torch.full((2, heads, total + 9, dim), 7.0, dtype=out, device="cuda")
        views = (buf[0].transpose(0, 1), buf[1].transpose(0, 1))
        Q.kv_cache_read(*args, total + 9, starts=st, out=views)
        assert all(torch.equal(g[:total].cpu(), w) and (g[total:] == 7.0).all() for g, w in zip(views, want))
        tail = Q.kv_cache_read(*args, total + 5, starts=st, out_dtype=out)
        assert all(torch.equal(g[:total].cpu(), w) and (g[total:] == 0).all() for g, w in zip(tail, want))
    _lib.check_device_status(cache.k_codes.device)


def test_pages_outside_the_cache_read_as_zeros_and_are_reported():
    cache, _ = _filled(np.random.default_rng(0), 4, 8, 2, 32, "int8")
    cu = torch.tensor([0, 10, 30], dtype=torch.int32, device="cuda")
    table = torch.tensor([[1, 4], [-1, 2]], dtype=torch.int32, device="cuda")  # page 4 and -1; sequence 1 is past its table
    k, v = Q.kv_cache_read(cache, table, cu, 30)
    with pytest.raises(_lib.ShapeMismatch):
        _lib.check_device_status(k.device)
    assert (k[:8] != 0).any(-1).all() and (k[8:18] == 0).all() and (k[18:26] != 0).any(-1).all() and (v[26:] == 0).all()


def test_no_sequences_and_no_rows():
    cache = Q.kv_cache_alloc(2, 4, 1, 32)
    none = torch.zeros(0, 0, dtype=torch.int32, device="cuda")
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = Q.kv_cache_read(cache, none, cu, 0)
    assert k.shape == (0, 1, 32)
    k, v = Q.kv_cache_read(cache, none, cu, 3)
    assert (k == 0).all() and (v == 0).all()
    e = torch.zeros(0, 1, 32, device="cuda")
    Q.kv_cache_write(cache, e, e, torch.zeros(0, dtype=torch.int64, device="cuda"))


def test_views_of_a_fused_projection_are_read_in_place():
    qkv = torch.randn(21, (6 + 2 + 2) * 64, device="cuda", dtype=torch.bfloat16)
    _, k, v = qkv.split((6 * 64, 2 * 64, 2 * 64), -1)
    k, v = k.unflatten(-1, (2, 64)), v.unflatten(-1, (2, 64))
    a, b = Q.kv_cache_alloc(2, 16, 2, 64, "mxfp4"), Q.kv_cache_alloc(2, 16, 2, 64, "mxfp4")
    slots = torch.randperm(32, device="cuda")[:21]
    Q.kv_cache_write(a, k, v, slots)
    Q.kv_cache_write(b, k.contiguous(), v.contiguous(), slots)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # transposed heads, and a last axis that has to be copied first
    Q.kv_cache_write(b, k.transpose(0, 1).contiguous().transpose(0, 1), v.transpose(1, 2).contiguous().transpose(1, 2), slots)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("fmt", ["int8", "mxfp4"])
def test_a_long_cache_passes_32_bits(fmt):
    """Slots whose byte offset in the codes is past 2^32 (4.3 GB of keys)."""
    heads, dim, page = 8, 128, 64
    row = heads * dim if fmt == "int8" else heads * dim // 2
    pages = (1 << 32) // (row * page) + 2
    lead = (pages, page, heads)
    if fmt == "int8":
        codes, scales = torch.empty((*lead, dim), dtype=torch.int8, device="cuda"), torch.empty(lead, device="cuda")
    else:
        codes = torch.empty((*lead, dim // 2), dtype=torch.uint8, device="cuda")
        scales = torch.empty((*lead, dim // 32), dtype=torch.uint8, device="cuda")
    cache = Q.KVCache(codes, scales, codes, scales)  # keys and values share the rows: both are written alike
    x = torch.randn(page, heads, dim, device="cuda")
    Q.kv_cache_write(cache, x, x, (pages - 1) * page + torch.arange(page, device="cuda"))
    cu = torch.tensor([0, page], dtype=torch.int32, device="cuda")
    k, v = Q.kv_cache_read(cache, torch.tensor([[pages - 1]], dtype=torch.int32, device="cuda"), cu, page)
    want = _decode(*_encode(host(x), fmt), fmt)
    assert np.array_equal(host(k), want) and np.array_equal(host(v), want)


@pytest.mark.parametrize("fmt", ["int8", "mxfp4"])
def test_every_read_sees_the_write_before_it(fmt):
    """Write, read, write, read, .. with nothing in between: launches that overlap, rows that share memory
    sectors with rows read before they were written."""
    heads, dim, n = 2, 32, 96
    cache = Q.kv_cache_alloc(4, 32, heads, dim, fmt)
    x = torch.randn(n, heads, dim, device="cuda")
    slots = [torch.tensor([i], device="cuda") for i in range(n)]
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    rows = [x[i:i + 1] for i in range(n)]
    outs = [(torch.empty(n, heads, dim, device="cuda"), torch.empty(n, heads, dim, device="cuda")) for _ in range(n)]
    torch.cuda.synchronize()
    for i in range(n):
        Q.kv_cache_write(cache, rows[i], rows[i], slots[i])
        Q.kv_cache_read(cache, table, cu, n, out=outs[i])
    want = _decode(*_encode(host(x), fmt), fmt)
    for i in range(n):
        for got in outs[i]:
            assert np.array_equal(host(got)[:i + 1], want[:i + 1]) and not host(got)[i + 1:].any()


def test_module_and_a_decoder_step_captured_and_replayed():
    """Projection, cache write, read-back and attention over what was read, as a decoding loop runs them:
    eager steps, then the same step replayed from a CUDA graph with new tokens."""
    torch.manual_seed(0)
    heads, dim, page, width = 2, 64, 16, 128
    cache = nnq.PagedKVCache(8, page, heads, dim, "int8").cuda()
    assert list(cache.state_dict()) == [] and "int8" in repr(cache)
    qkv = nnq.MXLinear.from_float(torch.nn.Linear(width, 3 * heads * dim, bias=False).cuda())
    out = nnq.MXLinear.from_float(torch.nn.Linear(heads * dim, width).cuda())
    table = torch.tensor([[5, 1], [0, 7]], dtype=torch.int32, device="cuda")
    x = torch.randn(2, width, device="cuda")
    pos = torch.zeros(2, dtype=torch.int64, device="cuda")
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    buf = torch.zeros(2, 2 * 2 * page, heads, dim, device="cuda")

    def step():
        q, k, v = qkv(x).unflatten(-1, (3, heads, dim)).unbind(1)
        slots = table.gather(1, (pos // page)[:, None]).squeeze(1).long() * page + pos % page
        cache.write(k, v, slots)
        cu[1:] = (pos + 1).cumsum(0)
        kk, vv = cache.read(table, cu, buf.shape[1], out=(buf[0], buf[1]))
        row = torch.arange(kk.shape[0], device="cuda")
        mine = (row[None] >= cu[:2, None]) & (row[None] < cu[1:, None])
        p = torch.einsum("bhd,rhd->bhr", q, kk) * dim ** -0.5
        p = p.masked_fill(~mine[:, None], float("-inf")).softmax(-1)
        return out(torch.einsum("bhr,rhd->bhd", p, vv).flatten(1))

    tokens = [torch.randn(2, width, device="cuda") for _ in range(20)]

    def run(fn):
        for t in cache.buffers():
            t.zero_()
        pos.zero_()
        ys = []
        for t in tokens:
            x.copy_(t)
            ys.append(fn().clone())
            pos.add_(1)
        return torch.stack(ys)

    eager = run(step)
    assert torch.isfinite(eager).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()

    def replay():
        graph.replay()
        return y

    assert torch.equal(run(replay), eager)
    # the last step's read-back is what the projections of all tokens encode to
    k_all = torch.stack([qkv(t).unflatten(-1, (3, heads, dim))[:, 1] for t in tokens])  # (token, sequence, head, dim)
    want = _decode(*_encode(host(k_all), "int8"), "int8")
    assert np.array_equal(host(buf[0])[:20], want[:, 0]) and np.array_equal(host(buf[0])[20:40], want[:, 1])
    _lib.check_device_status(x.device)


def test_bad_arguments_raise():
    cache = Q.kv_cache_alloc(2, 4, 2, 32)
    x = torch.zeros(3, 2, 32, device="cuda")
    s = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(_lib.ShapeMismatch):
        Q.kv_cache_write(cache, x, x[:2], s)
    with pytest.raises(_lib.ShapeMismatch):
        Q.kv_cache_write(cache, x[:, :1], x, s)
    with pytest.raises(_lib.DtypeMismatch):
        Q.kv_cache_write(cache, x.half(), x.half(), s)
    with pytest.raises(_lib.DtypeMismatch):
        Q.kv_cache_write(cache, x, x, s.float())
    with pytest.raises(_lib.DeviceMismatch):
        Q.kv_cache_write(cache, x, x, s.cpu())
    with pytest.raises(_lib.DtypeMismatch):
        Q.kv_cache_write(cache._replace(v_codes=cache.v_codes.to(torch.uint8)), x, x, s)
    with pytest.raises(_lib.ShapeMismatch):
        Q.kv_cache_write(cache._replace(v_scales=cache.v_scales[:1]), x, x, s)
    t = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    with pytest.raises(_lib.DtypeMismatch):
        Q.kv_cache_read(cache, t.long(), cu, 3)
    with pytest.raises(_lib.ShapeMismatch):
        Q.kv_cache_read(cache, t, cu[:1], 3)
    with pytest.raises(_lib.ShapeMismatch):
        Q.kv_cache_read(cache, t, cu, 3, out=(torch.empty(3, 2, 33, device="cuda")[..., :32],) * 2)
    with pytest.raises(_lib.ShapeMismatch):
        Q.kv_cache_read(cache, t, cu, 3, out=(torch.empty(1, 2, 32, device="cuda").expand(3, 2, 32),) * 2)
    with pytest.raises(ValueError):
        Q.kv_cache_alloc(2, 4, 2, 32, fmt="fp8")
    with pytest.raises(_lib.ShapeMismatch):
        Q.kv_cache_alloc(2, 4, 2, 48, fmt="mxfp4")
