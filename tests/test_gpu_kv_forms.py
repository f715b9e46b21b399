"""The cache's forms for long inputs: reads of four and sixteen rows a warp on both sides of each switch, writes with a
marking kernel in front, in every format, type and width of head."""

import numpy as np
import pytest
import torch

import mx_oracle as MX

pytestmark = pytest.mark.gpu

import lucid_b200.quantization as Q  # noqa: E402
from gpu_util import dev, host  # noqa: E402
from lucid_b200 import _lib  # noqa: E402

VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _random_cache(g, pages, page, heads, dim, fmt):
    lead = (pages, page, heads)

    def side():
        if fmt == "int8":
            return (torch.randint(-128, 128, (*lead, dim), device="cuda", generator=g, dtype=torch.int8),
                    torch.rand(lead, device="cuda", generator=g) + 1e-3)
        return (torch.randint(0, 256, (*lead, dim // 2), device="cuda", generator=g, dtype=torch.uint8),
                torch.randint(100, 150, (*lead, dim // 32), device="cuda", generator=g, dtype=torch.uint8))

    return Q.KVCache(*side(), *side())


def _rows(codes, scales, fmt, at, out):
    """Rows ``at`` (negative: zeros) in float64, rounded to float32 as one multiplication does, then to the output."""
    c, s = codes.flatten(0, 1)[at.clamp(min=0)], scales.flatten(0, 1)[at.clamp(min=0)]
    if fmt == "int8":
        v = c.double() * s.double()[..., None]
    else:
        e = torch.stack((c & 15, c >> 4), -1).flatten(-2).long()
        v = torch.tensor(VALUES + [-x for x in VALUES], dtype=torch.float64, device="cuda")[e]
        v = v * torch.exp2(s.double() - 127).repeat_interleave(32, -1)
    return torch.where((at >= 0)[:, None, None], v, 0.0).float().to(out)


def _lengths(rng, total, seqs):
    cuts = np.sort(rng.integers(0, total + 1, seqs - 1))
    lens = np.diff(np.concatenate(([0], cuts, [total])))
    lens[rng.random(seqs) < 0.2] = 0  # empty ones among them; the rows they leave are an uncovered tail
    return lens


# (heads, dim) with, per format, the row counts at which four and sixteen rows a warp begin
READS = [("int8", 1, 16, 4096), ("int8", 1, 16, 16384), ("int8", 1, 80, 4096), ("int8", 1, 80, 65536), ("int8", 3, 96, 16384),
         ("int8", 8, 64, 16384), ("int8", 8, 128, 65536), ("mxfp4", 1, 32, 4096), ("mxfp4", 1, 64, 16384), ("mxfp4", 3, 96, 16384),
         ("mxfp4", 4, 64, 4096), ("mxfp4", 4, 64, 65536), ("mxfp4", 8, 128, 16384)]


@pytest.mark.parametrize("fmt,heads,dim,switch", READS)
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("over", [-1, 0, 3, 250])
def test_long_reads(fmt, heads, dim, switch, out, over):
    total, page, seqs = switch + over, 24, 19
    rng = np.random.default_rng(switch + over + heads * dim)
    g = torch.Generator("cuda").manual_seed(switch + dim)
    lens = _lengths(rng, total - 70, seqs)
    first, starts = 33, rng.integers(0, 3 * page, seqs)  # rows before the first sequence belong to nobody
    width = int((lens + starts).max() + page - 1) // page
    pages = 200
    cache = _random_cache(g, pages, page, heads, dim, fmt)
    table = rng.integers(0, pages, (seqs, width)).astype(np.int32)
    table[rng.random(table.shape) < 0.01] = rng.choice([-1, pages, 2 ** 31 - 1, -2 ** 31])
    cu = np.concatenate(([first], first + np.cumsum(lens)))
    at = np.full(total, -2)
    for b, t in enumerate(lens):
        pos = starts[b] + np.arange(t)
        p = table[b, pos // page].astype(np.int64)
        at[cu[b]:cu[b] + t] = np.where((p >= 0) & (p < pages), p * page + pos % page, -1)
    where = dev(at)
    args = (cache, dev(table), dev(cu.astype(np.int32)), total)
    want = [_rows(c, s, fmt, where, out) for c, s in (cache[:2], cache[2:])]
    _lib.status_word(where.device).zero_()
    got = Q.kv_cache_read(*args, starts=dev(starts.astype(np.int32)), out_dtype=out)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    if (at == -1).any():
        with pytest.raises(_lib.ShapeMismatch):
            _lib.check_device_status(where.device)
    buf = torch.full((total, 2, heads, dim), 7.0, dtype=out, device="cuda")  # keys and values of a token side by side
    Q.kv_cache_read(*args, starts=dev(starts.astype(np.int32)), out=(buf[:, 0], buf[:, 1]))
    nobody = where == -2
    assert (buf[nobody] == 7.0).all() and all(torch.equal(buf[~nobody, i], w[~nobody]) for i, w in enumerate(want))
    _lib.status_word(where.device).zero_()


WRITES = [("int8", 2, 80), ("int8", 8, 128), ("int8", 1, 1024), ("int8", 3, 576), ("mxfp4", 3, 96), ("mxfp4", 8, 128), ("mxfp4", 1, 1024),
          ("mxfp4", 5, 32)]


def _expect(ref, k, v, slots, fmt):
    """The codes and scales of a cache of zeros after the write: the last token of each slot."""
    last = {int(s): i for i, s in enumerate(slots) if 0 <= s < ref[0].shape[0]}
    at, tok = np.array(list(last.keys()), int), np.array(list(last.values()), int)
    for i, x in ((0, k), (2, v)):
        rows = x[tok].reshape(-1, x.shape[-1])
        if fmt == "int8":
            codes, scales = MX.int8_rows(rows)
        else:
            code, scales, _ = MX.encode(rows)
            codes = MX.pack(code)
        ref[i][at], ref[i + 1][at] = codes.reshape(len(tok), *ref[i].shape[1:]), scales.reshape(len(tok), *ref[i + 1].shape[1:])


def _check_write(fmt, heads, dim, dtype, tokens, slot_type, seed):
    rng = np.random.default_rng(seed)
    page = 16
    pages = tokens // page // 2 + 1
    cache = Q.kv_cache_alloc(pages, page, heads, dim, fmt)
    slots = rng.integers(-10, pages * page, tokens)  # about two tokens a slot, some of padding
    slots[-3:] = slots[:3]
    slots[tokens // 2] = pages * page               # past the cache
    k, v = (torch.from_numpy((rng.standard_normal((tokens, heads, dim)) * 4).astype(np.float32)).to(dtype) for _ in range(2))
    k[0, 0] = 0.0
    fused = torch.cat((k, v), 1).cuda()             # both are views of one projection
    _lib.status_word(fused.device).zero_()
    Q.kv_cache_write(cache, fused[:, :heads], fused[:, heads:], dev(slots).to(slot_type))
    with pytest.raises(_lib.ShapeMismatch):
        _lib.check_device_status(fused.device)
    ref = [np.zeros_like(host(t)).reshape(pages * page, *t.shape[2:]) for t in cache]
    _expect(ref, host(k.float()), host(v.float()), slots, fmt)
    for got, want in zip(cache, ref):
        assert np.array_equal(host(got).reshape(want.shape), want)


@pytest.mark.parametrize("fmt,heads,dim", WRITES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens", [256, 257, 1027])
def test_long_writes(fmt, heads, dim, dtype, tokens):
    _check_write(fmt, heads, dim, dtype, tokens, torch.int32 if tokens % 2 else torch.int64, tokens + dim)


@pytest.mark.parametrize("fmt,heads,dim", [("int8", 1, 32), ("mxfp4", 1, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens", [65536, 65537, 70003])
def test_writes_of_more_tokens_than_the_small_table_serves(fmt, heads, dim, dtype, tokens):
    _check_write(fmt, heads, dim, dtype, tokens, torch.int64, tokens)
