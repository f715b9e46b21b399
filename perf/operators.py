"""Cases of the microscaled 4-bit (MXFP4) operators and of the quantized key/value cache: what a
user's program holds before a call, the call, and the same mathematics in elementary torch operations.

MXFP4: a block of 32 consecutive values of the last axis shares the scale 2^(floor(log2 amax) - 2), held as
its biased exponent in one byte; an element is the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 (ties to the even
mantissa, clamped at 6) times its sign.  Two elements share a byte, the first in the low half.  Scale bytes
of a (rows, K) matrix are laid out in tiles of 128 rows x 8 blocks:
``tiles[row // 128, block // 8, (block // 4) % 2, row % 32, (row // 32) % 4, block % 4]``.

The cache holds pages of ``page`` tokens, ``(pages, page, heads, dim)``: int8 codes with one float32 scale
per token and head, or MXFP4 along the head dimension."""

import math

import torch

own = False

_BLOCK = 32
_DT = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---- cases -----------------------------------------------------------------------------------


def listed():
    return [
        # one token through a square projection of a 70-billion-parameter decoder: weight streaming
        dict(name="linear one row", op="linear", m=1, k=8192, n=8192, dtype="bf16", bias=False, relu=False),
        # a decode batch through the fused q/k/v projection
        dict(name="linear 48 rows", op="linear", m=48, k=8192, n=10240, dtype="bf16", bias=True, relu=False),
        # a prompt through the up projection: the tensor cores decide
        dict(name="linear prompt", op="linear", m=4096, k=8192, n=28672, dtype="bf16", bias=False, relu=False),
        # odd rows, an input axis of 33 blocks, odd outputs, float32 with bias and ReLU
        dict(name="linear ragged", op="linear", m=777, k=1056, n=1003, dtype="f32", bias=True, relu=True),
        # both operands already in the format, float32 result
        dict(name="matmul of codes", op="matmul", m=1000, k=4096, n=4096, dtype="f32", bias=False, relu=False),
        # a weight encoded and decoded
        dict(name="round trip weight", op="round", m=8192, k=8192, dtype="f32"),
        # a decode batch of activations encoded and decoded
        dict(name="round trip rows", op="round", m=48, k=8192, dtype="bf16"),
        # a training step's fake quantization of a weight, with its gradient
        dict(name="fake quantize weight", op="fake", m=8192, k=4096, dtype="f32"),
        # ... of one sequence's activations, odd rows
        dict(name="fake quantize rows", op="fake", m=333, k=1056, dtype="bf16"),
        # one new token for each of 32 sequences, their contexts read back
        dict(name="cache decode int8", op="cache", fmt="int8", seqs=32, new=1, longest=4096, heads=8, dim=128, page=16),
        # a chunk of a long prompt written and the sequence so far read back
        dict(name="cache chunk int8", op="cache", fmt="int8", seqs=1, new=2048, longest=16384, heads=8, dim=128, page=64),
        # several ragged chunks in the 4-bit format, 64 values a head, pages of an odd size
        dict(name="cache chunk mxfp4", op="cache", fmt="mxfp4", seqs=7, new=300, longest=9000, heads=4, dim=64, page=24),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "matmul", "round", "fake", "cache", "cache"])
    dtype = rng.choice(["f32", "bf16"])
    if op in ("linear", "matmul"):
        return dict(op=op, m=_log(rng, 1, 4096), k=32 * _log(rng, 1, 256), n=_log(rng, 16, 28672), dtype=dtype,
                    bias=rng.random() < 0.5, relu=rng.random() < 0.3)
    if op in ("round", "fake"):
        return dict(op=op, m=_log(rng, 1, 8192), k=32 * _log(rng, 1, 128), dtype=dtype)
    longest = _log(rng, 32, 16384)
    seqs = _log(rng, 1, max(1, min(64, 131072 // longest)))
    fmt = rng.choice(["int8", "mxfp4"])
    dim = rng.choice([32, 64, 96, 128, 192, 256]) if fmt == "mxfp4" else rng.choice([32, 64, 80, 96, 128, 256])
    return dict(op=op, fmt=fmt, seqs=seqs, new=_log(rng, 1, min(longest, 2048)), longest=longest,
                heads=rng.choice([1, 2, 4, 5, 8]), dim=dim, page=rng.choice([1, 16, 24, 32, 64, 128]))


def _lengths(case):
    """Context lengths of the sequences, the new tokens among them: ragged, the first the longest."""
    lo, hi, n = case["new"], case["longest"], case["seqs"]
    return [hi - (hi - lo) * i // n for i in range(n)]


# ---- inputs ----------------------------------------------------------------------------------


def _activations(shape, dtype, g):
    """Unit normal values with a few channels an order of magnitude larger, as hidden states have."""
    x = torch.randn(shape, device="cuda", generator=g)
    loud = torch.rand(shape[-1], device="cuda", generator=g) < 0.01
    return (x * torch.where(loud, 12.0, 1.0)).to(_DT[dtype])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = dict(case)
    if op in ("linear", "matmul"):
        m, k, n = case["m"], case["k"], case["n"]
        w = torch.randn((n, k), device="cuda", generator=g) * k ** -0.5
        s["w_codes"], s["w_scales"] = _pack(w)
        s["bias"] = torch.randn(n, device="cuda", generator=g) if case["bias"] else None
        x = _activations((m, k), case["dtype"], g)
        if op == "linear":
            s["x"] = x
        else:
            s["x_codes"], s["x_scales"] = _pack(x.float())
    elif op == "round":
        s["x"] = _activations((case["m"], case["k"]), case["dtype"], g)
    elif op == "fake":
        s["x"] = _activations((case["m"], case["k"]), case["dtype"], g).requires_grad_()
        s["grad"] = torch.randn((case["m"], case["k"]), device="cuda", generator=g).to(_DT[case["dtype"]])
    else:
        page, h, d = case["page"], case["heads"], case["dim"]
        lens = _lengths(case)
        blocks = [-(-t // page) for t in lens]
        pages = sum(blocks) + 3  # a few pages belong to nobody
        order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        table = torch.zeros((len(lens), max(blocks)), dtype=torch.int32, device="cuda")
        used, slots, cu = 0, [], [0]
        for b, t in enumerate(lens):
            table[b, : blocks[b]] = order[used: used + blocks[b]]
            used += blocks[b]
            pos = torch.arange(t - case["new"], t, device="cuda")
            slots.append(table[b, pos // page].long() * page + pos % page)
            cu.append(cu[-1] + t)
        s["slots"], s["table"], s["total"] = torch.cat(slots), table, cu[-1]
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        for name in ("k", "v"):
            old = _activations((pages, page, h, d), "bf16", g)
            s[name + "_codes"], s[name + "_scales"] = _encode(old.float(), case["fmt"])
            s[name] = _activations((len(s["slots"]), h, d), "bf16", g)
    return s


# ---- the plain form --------------------------------------------------------------------------


def _element_codes(a):
    """Index of the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6; a tie goes to the even index."""
    i = (a > 0.25).to(torch.uint8)
    return i + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)


def _values():
    return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")


def _blocks(x):
    """Blocks of 32 float32 values -> (their signed element codes, the scale bytes, the scaled magnitudes)."""
    b = x.reshape(*x.shape[:-1], -1, _BLOCK)
    amax = b.abs().amax(-1)
    exponent = torch.frexp(amax)[1] - 1 - 2
    byte = torch.where(amax > 0, exponent.clamp(min=-127) + 127, 0)
    a = b.abs() * torch.exp2((127 - byte).float())[..., None]
    codes = _element_codes(a) + torch.signbit(b).to(torch.uint8) * 8
    return codes, byte.to(torch.uint8), a


def _of_blocks(codes, byte):
    v = _values()[(codes & 7).long()] * torch.exp2(byte.float() - 127)[..., None]
    v = torch.where(codes >= 8, -v, v)
    return v.reshape(*v.shape[:-2], -1)


def _nibbles(codes):
    c = codes.reshape(*codes.shape[:-2], -1)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _from_nibbles(packed):
    c = torch.stack((packed & 15, packed >> 4), -1)
    return c.reshape(*packed.shape[:-1], -1, _BLOCK)


def _tiled(byte):
    """(rows, blocks) scale bytes -> their tiles, the padding zero."""
    rows, blocks = byte.shape
    rt, bt = -(-rows // 128), -(-blocks // 8)
    full = byte.new_zeros((rt * 128, bt * 8))
    full[:rows, :blocks] = byte
    return full.reshape(rt, 4, 32, bt, 2, 4).permute(0, 3, 4, 2, 1, 5).reshape(rt, bt, 1024).contiguous()


def _untiled(tiles, rows, blocks):
    rt, bt = tiles.shape[:2]
    full = tiles.reshape(rt, bt, 2, 32, 4, 4).permute(0, 4, 3, 1, 2, 5).reshape(rt * 128, bt * 8)
    return full[:rows, :blocks]


def _pack(x):
    codes, byte, _ = _blocks(x)
    return _nibbles(codes), _tiled(byte)


def _unpack(packed, tiles):
    codes = _from_nibbles(packed)
    return _of_blocks(codes, _untiled(tiles, codes.shape[0], codes.shape[1]))


def _encode(x, fmt):
    """Rows of a cache: int8 codes with a float32 scale, or MXFP4."""
    if fmt == "int8":
        scale = (x.abs().amax(-1) / 127.5).clamp(min=1e-8)
        return (x / scale[..., None]).round().clamp(-128, 127).to(torch.int8), scale
    codes, byte, _ = _blocks(x)
    return _nibbles(codes), byte


def _decode(codes, scale, fmt):
    return codes.float() * scale[..., None] if fmt == "int8" else _of_blocks(_from_nibbles(codes), scale)


def _cache_pass(s):
    page, slots = s["page"], s["slots"]
    row = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(s["cu"], row.to(torch.int32), right=True) - 1
    pos = row - s["cu"][seq]
    at = s["table"][seq, pos // page].long() * page + pos % page
    out = []
    for name in ("k", "v"):
        codes, scales = s[name + "_codes"], s[name + "_scales"]
        codes, scales = codes.reshape(-1, *codes.shape[2:]), scales.reshape(-1, *scales.shape[2:])
        codes[slots], scales[slots] = _encode(s[name].float(), s["fmt"])
        out.append(_decode(codes[at], scales[at], s["fmt"]).to(torch.bfloat16))
    return out


def _plain(s):
    op = s["op"]
    if op in ("linear", "matmul"):
        codes, tiles = _pack(s["x"].float()) if op == "linear" else (s["x_codes"], s["x_scales"])
        y = _unpack(codes, tiles) @ _unpack(s["w_codes"], s["w_scales"]).T
        y = y if s["bias"] is None else y + s["bias"]
        return (y.clamp(min=0) if s["relu"] else y).to(_DT[s["dtype"]])
    if op == "round":
        codes, tiles = _pack(s["x"].float())
        return _unpack(codes, tiles).to(_DT[s["dtype"]])
    if op == "fake":
        codes, byte, a = _blocks(s["x"].detach().float())
        inside = (a < 7.0).reshape(s["x"].shape)
        y = _of_blocks(codes, byte).to(s["x"].dtype)
        return y, (s["grad"].float() * inside).to(s["x"].dtype)
    return _cache_pass(s)


# ---- the calls -------------------------------------------------------------------------------


def _own(s):
    import lucid_b200.quantization as Q

    op = s["op"]
    if op == "linear":
        return Q.mx_linear(s["x"], s["w_codes"], s["w_scales"], bias=s["bias"], relu=s["relu"])
    if op == "matmul":
        return Q.mx_matmul(s["x_codes"], s["x_scales"], s["w_codes"], s["w_scales"], bias=s["bias"], relu=s["relu"],
                           out_dtype=_DT[s["dtype"]])
    if op == "round":
        codes, scales = Q.mx_quantize(s["x"])
        return Q.mx_dequantize(codes, scales, out_dtype=s["x"].dtype)
    if op == "fake":
        y = Q.mx_fake_quantize(s["x"])
        (grad,) = torch.autograd.grad(y, s["x"], s["grad"])
        return y.detach(), grad
    cache = Q.KVCache(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"])
    Q.kv_cache_write(cache, s["k"], s["v"], s["slots"])
    return list(Q.kv_cache_read(cache, s["table"], s["cu"], s["total"], out_dtype=torch.bfloat16))


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    op = case["op"]
    esz = 4 if case.get("dtype") == "f32" else 2
    if op in ("linear", "matmul"):
        m, k, n = case["m"], case["k"], case["n"]
        x = m * k * esz if op == "linear" else m * k * 17 / 32
        return dict(bytes=x + n * k * 17 / 32 + m * n * esz + (4 * n if case["bias"] else 0), flops=2 * m * n * k)
    if op == "round":  # encoded, and the codes decoded
        elements = case["m"] * case["k"]
        return dict(bytes=elements * (2 * esz + 2 * 17 / 32), flops=0)
    if op == "fake":  # forward: values in and out, one bit kept; backward: gradient in and out
        elements = case["m"] * case["k"]
        return dict(bytes=elements * (4 * esz + 0.25), flops=0)
    row = case["heads"] * case["dim"]
    held = row + 4 * case["heads"] if case["fmt"] == "int8" else row * 17 / 32
    new, total = case["seqs"] * case["new"], sum(_lengths(case))
    return dict(bytes=2 * (new * (2 * row + held + 8) + total * (held + 2 * row)), flops=0)


# ---- the definition in 64 bits --------------------------------------------------------------


def _mx64(x):
    """MXFP4 values of x, and where an element fits without the clamp, from the definition."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    # floor(log2): exact from the mantissa/exponent split, not from a rounded logarithm
    scale = torch.ldexp(torch.ones_like(top), torch.frexp(top).exponent - 3).clamp(min=2.0 ** -127)
    y = b / scale
    # the spacing of the format is 1/2 below 2, 1 in [2, 4), 2 from 4 on
    size = y.abs()
    step = torch.ones_like(size)
    step[size < 2] = 0.5
    step[size >= 4] = 2.0
    r = torch.round(y / step) * step
    return (r.clamp(-6, 6) * scale).flatten(-2), (r.abs() <= 6).flatten(-2)


def _held64(packed, scale_bytes):
    """Values of packed codes with their (.., blocks) scale bytes."""
    low, high = packed.long() % 16, packed.long() // 16
    c = torch.stack((low, high), -1).flatten(-2).unflatten(-1, (-1, 32))
    e, f = (c % 8) // 2, c % 2
    size = torch.where(e == 0, f * 0.5, torch.ldexp(1.0 + 0.5 * f.double(), e - 1))
    return (torch.where(c >= 8, -size, size) * torch.pow(2.0, scale_bytes.double() - 127)[..., None]).flatten(-2)


def _matrix64(packed, tiles):
    rows, blocks = packed.shape[0], packed.shape[1] // 16
    r = torch.arange(rows, device="cuda")[:, None]
    b = torch.arange(blocks, device="cuda")[None, :]
    within = (b // 4) % 2 * 512 + r % 32 * 16 + r // 32 % 4 * 4 + b % 4
    return _held64(packed, tiles[r // 128, b // 8, within])


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("linear", "matmul"):
        a = _mx64(s["x"])[0] if op == "linear" else _matrix64(s["x_codes"], s["x_scales"])
        y = a.matmul(_matrix64(s["w_codes"], s["w_scales"]).t())
        if case["bias"]:
            y += s["bias"].double()
        return torch.relu(y) if case["relu"] else y
    if op == "round":
        return _mx64(s["x"])[0]
    if op == "fake":
        y, fits = _mx64(s["x"].detach())
        return y, torch.where(fits, s["grad"].double(), 0.0)
    page, lens = case["page"], _lengths(case)
    out = []
    for name in ("k", "v"):
        new = s[name].double()
        if case["fmt"] == "int8":
            scale = (new.abs().amax(-1, keepdim=True) / 127.5).clamp(min=1e-8)
            new = torch.clamp(torch.round(new / scale), -128, 127) * scale
            held = s[name + "_codes"].double() * s[name + "_scales"].double()[..., None]
        else:
            new = _mx64(new)[0]
            held = _held64(s[name + "_codes"], s[name + "_scales"])
        rows = []
        for b, t in enumerate(lens):
            pages = held[s["table"][b, : -(-t // page)].long()].flatten(0, 1)
            rows += [pages[: t - case["new"]], new[b * case["new"]: (b + 1) * case["new"]]]
        out.append(torch.cat(rows))
    return out
