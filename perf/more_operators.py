"""The operators of models in microscaled 4-bit weights, as cases to be timed.

A row is divided into blocks of 32 neighbours along K that share a scale, a power of two (e8m0):
weights have e2m1 elements (0, 0.5, 1, 1.5, 2, 3, 4, 6), activations e4m3 ones (to 448). With a
the block's largest magnitude, the scale is 2^(floor(log2 a) - 2), or twice that from a = 1.75 *
2^floor(log2 a) on (e4m3: - 8, above 1.8125), so that each element is the nearest value and none
is cut off; 2^-127 at least, which also a block of zeros has.

  quantize  stride_amd.mx.quantize (and dequantize): 16 x 16 tiles in bf16 or fp32 to blocks
  norm      stride_amd.mx.norm: h += add, then RMSNorm(h) * gain in e4m3 blocks
  gemm      stride_amd.mx.gemm: y = W x in bf16 tiles
  mlp13     stride_amd.mx.mlp13: silu(W1 x) * (W3 x) in e4m3 blocks, what the next product takes

K is filled up with zeros to a multiple of 512. Codes and scales lie as the matrix instruction
takes them, which the packing functions below say in elementary indexing:
  e2m1   [row tile][K / 128][K block of 32: 4][row: 16][16 bytes, even k in the low half]
  e4m3   [row tile][K / 128][K half: 2][4][row: 16][16 bytes]
  scales [row tile][K / 512][K block of 32 in the chunk: 4][row: 16][chunk of 128: 4]

Shapes are those of the repository's benchmark (hidden 2048, MLP 8192, 1 to 4096 rows) and odd ones.
"""
import math

import torch

own = False  # True: run() calls this repository's operators instead of the plain forms

DEV = "cuda:0"
EPS = 1e-5
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------------------
# The cases.

def listed():
    def quantize(name, rows, k, bits, src):
        return dict(name=name, op="quantize", rows=rows, k=k, bits=bits, src=src)

    def norm(name, rows, k, add):
        return dict(name=name, op="norm", rows=rows, k=k, add=add)

    def product(name, op, rows, n, k):
        return dict(name=name, op=op, rows=rows, n=n, k=k)

    return [
        # Loading a model: gate and up weights of one layer, as the checkpoint has them.
        quantize("quantize_weights_16384x2048", 16384, 2048, 4, "bf16"),
        # A projection of a small model in fp32, its sizes odd.
        quantize("quantize_weights_1008x1040", 1008, 1040, 4, "fp32"),
        # Attention's output of a decode batch, before the output projection.
        quantize("quantize_rows_128", 128, 2048, 8, "bf16"),
        # One user's decode step, first norm of the first layer.
        norm("norm_1", 1, 2048, False),
        # An odd batch behind the down projection of a wider model.
        norm("norm_add_333x8192", 333, 8192, True),
        # A prompt's chunk.
        norm("norm_add_4096", 4096, 2048, True),
        # One user: the down projection, nothing but its weights.
        product("gemm_down_1", "gemm", 1, 2048, 8192),
        # The serving batch.
        product("gemm_down_128", "gemm", 128, 2048, 8192),
        # An odd chunk of prompts through the output projection.
        product("gemm_o_290", "gemm", 290, 2048, 2048),
        # A long prompt.
        product("gemm_down_4096", "gemm", 4096, 2048, 8192),
        # Gate and up: a decode batch, and a prompt's chunk.
        product("mlp13_64", "mlp13", 64, 8192, 2048),
        product("mlp13_2048", "mlp13", 2048, 8192, 2048),
    ]


def _span(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    """One more case of these ranges."""
    op = rng.choice(["quantize", "norm", "gemm", "gemm", "mlp13", "mlp13"])
    if op == "quantize":
        k = 16 * _span(rng, 1, 512)
        rows = _span(rng, 1, min(16384, 2 ** 25 // k))
        bits = rng.choice([4, 8])
        return dict(op=op, rows=-(-rows // 16) * 16 if bits == 4 else rows, k=k, bits=bits, src=rng.choice(["bf16", "bf16", "fp32"]))
    if op == "norm":
        k = 16 * _span(rng, 1, 512)
        return dict(op=op, rows=_span(rng, 1, min(4096, 2 ** 23 // k)), k=k, add=rng.random() < 0.7)
    k, n = 16 * _span(rng, 4, 512), 16 * _span(rng, 4, 512)
    most = 2 ** 36 // (n * k * (2 if op == "mlp13" else 1))
    return dict(op=op, rows=_span(rng, 1, max(1, min(4096, most))), n=n, k=k)


# ---------------------------------------------------------------------------
# Layouts in elementary indexing.

def _up(a, to):
    return -(-a // to) * to


def _rows_of(tiles, rows):
    """[t][ct][16][16] -> [rows][16 ct]."""
    t, ct = tiles.shape[:2]
    return tiles.permute(0, 2, 1, 3).reshape(t * 16, ct * 16)[:rows]


def _tiles_of(a):
    """[rows][cols] -> [ceil(rows / 16)][cols / 16][16][16], rows past the last zero."""
    rows, cols = a.shape
    out = torch.zeros((_up(rows, 16), cols), dtype=a.dtype, device=a.device)
    out[:rows] = a
    return out.reshape(-1, 16, cols // 16, 16).permute(0, 2, 1, 3).contiguous()


def _wide(a):
    """Rows filled up to whole tiles and K to a multiple of 512, with zeros."""
    out = torch.zeros((_up(a.shape[0], 16), _up(a.shape[1], 512)), dtype=a.dtype, device=a.device)
    out[: a.shape[0], : a.shape[1]] = a
    return out


def _pack_scales(e, rows):
    """Scale bytes [rows up][K / 32]; those of rows past the last are zero."""
    t, g = e.shape[0] // 16, e.shape[1] // 16
    e = torch.where(torch.arange(t * 16, device=e.device)[:, None] < rows, e, 0)
    return e.to(torch.uint8).reshape(t, 16, g, 4, 4).permute(0, 2, 4, 1, 3).contiguous()


def _unpack_scales(s):
    t, g = s.shape[:2]
    return s.reshape(t, g, 4, 16, 4).permute(0, 3, 1, 4, 2).reshape(t * 16, g * 16)


def _pack8(b):
    t, kc = b.shape[0] // 16, b.shape[1] // 128
    return b.reshape(t, 16, kc, 2, 4, 16).permute(0, 2, 3, 4, 1, 5).contiguous()


def _unpack8(c):
    t, kc = c.shape[:2]
    return c.reshape(t, kc, 2, 4, 16, 16).permute(0, 4, 1, 2, 3, 5).reshape(t * 16, kc * 128)


def _pack4(c):
    t, kc = c.shape[0] // 16, c.shape[1] // 128
    c = c.reshape(t, 16, kc, 4, 16, 2)
    return (c[..., 0] + 16 * c[..., 1]).to(torch.uint8).permute(0, 2, 3, 1, 4).contiguous()


def _unpack4(p):
    t, kc = p.shape[:2]
    b = p.reshape(t, kc, 4, 16, 16).permute(0, 3, 1, 2, 4).reshape(t * 16, kc * 64)
    return torch.stack([b & 15, b >> 4], -1).reshape(t * 16, kc * 128)


# ---------------------------------------------------------------------------
# Blocks.

def _exponents(a, bits):
    """The blocks' scale exponents, -127 .. 127, from finite values [rows][K], K a multiple of 32."""
    most = a.abs().reshape(a.shape[0], -1, 32).amax(-1)
    m, e = torch.frexp(most)  # most = m 2^e, 0.5 <= m < 1
    up = (m >= 0.875) if bits == 4 else (m > 0.90625)
    e = e - 1 - (2 if bits == 4 else 8) + up.to(e.dtype)
    return torch.where(most > 0, e, -127).clamp(-127, 127)


def _scaled(a, e):
    """a / 2^e by blocks (exact where it is not below the smallest number: two steps)."""
    b = a.reshape(a.shape[0], -1, 32)
    half = (-e // 2)[..., None]
    return torch.ldexp(torch.ldexp(b, half), -e[..., None] - half).reshape(a.shape)


def _round4(v):
    """The nearest e2m1 code, ties to the even one."""
    a = v.abs()
    code = torch.zeros(v.shape, dtype=torch.int32, device=v.device)
    for i in range(7):
        middle = (E2M1[i] + E2M1[i + 1]) / 2
        code += ((a > middle) if i % 2 == 0 else (a >= middle)).to(torch.int32)
    return code + 8 * (torch.signbit(v)).to(torch.int32)


def _round8(v):
    """The nearest e4m3 value, ties to the even one."""
    _, e = torch.frexp(v)
    step = (e - 4).clamp(min=-9)
    return torch.ldexp(torch.round(torch.ldexp(v, -step)), step)


def _held8(a, rows):
    """Values [rows][K] -> (e4m3 elements, e8m0 scales) as the framework holds them."""
    a = _wide(a.float())
    e = _exponents(a, 8)
    q = _round8(_scaled(a, e)).to(torch.float8_e4m3fn)
    return _pack8(q.view(torch.uint8)), _pack_scales(e + 127, rows)


def _held4(a, rows):
    a = _wide(a.float())
    e = _exponents(a, 4)
    return _pack4(_round4(_scaled(a, e))), _pack_scales(e + 127, rows)


def _values8(codes, scales, dtype=torch.float32):
    v = _unpack8(codes).view(torch.float8_e4m3fn).to(dtype)
    return _times(v, _unpack_scales(scales))


def _values4(codes, scales, dtype=torch.float32):
    c = _unpack4(codes).to(torch.int32)
    v = torch.tensor(E2M1, dtype=dtype, device=codes.device)[c & 7]
    return _times(torch.where(c >= 8, -v, v), _unpack_scales(scales))


def _times(v, e):
    return torch.ldexp(v.reshape(v.shape[0], -1, 32), (e.to(torch.int32) - 127)[..., None]).reshape(v.shape)


def _seen8(codes, scales):
    """8-bit outputs as the values that their bytes stand for."""
    return {"elements": codes.view(torch.float8_e4m3fn), "scales": scales.view(torch.float8_e8m0fnu)}


# ---------------------------------------------------------------------------
# Inputs.

def _normal(gen, *shape):
    return torch.empty(shape, device=DEV).normal_(generator=gen)


def _activations(gen, rows, k):
    """Normed activations: a few columns are an order of magnitude above the others."""
    a = _normal(gen, rows, k)
    loud = torch.rand(k, generator=gen, device=DEV) < 0.004
    return torch.where(loud, 8.0 * a, a)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + 5)
    rows, k = c["rows"], c["k"]
    s = dict(case=c)
    if c["op"] == "quantize":
        a = 0.02 * _normal(gen, rows, k) if c["bits"] == 4 else _activations(gen, rows, k)
        s["tiles"] = _tiles_of(a.to(torch.bfloat16 if c["src"] == "bf16" else torch.float32))
    elif c["op"] == "norm":
        s["h"] = _tiles_of(3.0 * _activations(gen, rows, k))
        s["add"] = _tiles_of(_normal(gen, rows, k).to(torch.bfloat16)) if c["add"] else None
        s["gain"] = 1.0 + 0.2 * _normal(gen, k)
    else:
        s["x"] = _held8(_activations(gen, rows, k), rows)
        s["w"] = [_held4(0.02 * _normal(gen, c["n"], k), c["n"]) for _ in range(2 if c["op"] == "mlp13" else 1)]
    if own:
        from stride_amd import mx

        if c["op"] == "quantize":
            s["out"] = mx.Tiles.create(rows, k, c["bits"], DEV)
        elif c["op"] == "norm":
            s["out"] = mx.Tiles.create(rows, k, 8, DEV)
        else:
            s["own_x"] = mx.Tiles(*s["x"], k, 8)
            s["own_w"] = [mx.Tiles(*w, k, 4) for w in s["w"]]
            if c["op"] == "gemm":
                s["out"] = torch.zeros((_up(rows, 16) // 16, c["n"] // 16, 16, 16), dtype=torch.int16, device=DEV)
            else:
                s["out"] = mx.Tiles.create(rows, c["n"], 8, DEV)
    return s


# ---------------------------------------------------------------------------
# One pass.

def run(s):
    return {"quantize": _quantize, "norm": _norm, "gemm": _gemm, "mlp13": _mlp13}[s["case"]["op"]](s)


def _quantize(s):
    c = s["case"]
    if own:
        from stride_amd import mx

        q = mx.quantize(s["tiles"], c["rows"], bits=c["bits"], out=s["out"])
        return _seen8(q.codes, q.scales) if c["bits"] == 8 else mx.dequantize(q, c["rows"])
    a = _rows_of(s["tiles"], c["rows"])
    if c["bits"] == 8:
        return _seen8(*_held8(a, c["rows"]))
    a = _wide(a.float())
    e = _exponents(a, 4)
    code = _round4(_scaled(a, e))
    v = torch.tensor(E2M1, device=DEV)[code & 7]
    return _times(torch.where(code >= 8, -v, v), e + 127)[: c["rows"], : c["k"]].to(torch.bfloat16)


def _norm(s):
    c = s["case"]
    if own:
        from stride_amd import mx

        q = mx.norm(s["h"], c["rows"], s["gain"], EPS, add=s["add"], out=s["out"])
        return {"h": s["h"], **_seen8(q.codes, q.scales)}
    if s["add"] is not None:
        s["h"] += s["add"].float()
    h = _rows_of(s["h"], c["rows"])
    x = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["gain"]
    return {"h": s["h"], **_seen8(*_held8(x, c["rows"]))}


def _gemm(s):
    c = s["case"]
    if own:
        from stride_amd import mx

        return mx.gemm(s["own_w"][0], s["own_x"], c["rows"], out=s["out"]).view(torch.bfloat16)
    y = torch.matmul(_values8(*s["x"])[: c["rows"]], _values4(*s["w"][0]).t())
    return _tiles_of(y.to(torch.bfloat16))


def _mlp13(s):
    c = s["case"]
    if own:
        from stride_amd import mx

        q = mx.mlp13(*s["own_w"], s["own_x"], c["rows"], out=s["out"])
        return _seen8(q.codes, q.scales)
    x = _values8(*s["x"])[: c["rows"]]
    gate, up = (torch.matmul(x, _values4(*w).t()) for w in s["w"])
    return _seen8(*_held8(gate / (1.0 + torch.exp(-gate)) * up, c["rows"]))


# ---------------------------------------------------------------------------
# What a pass cannot do without.

def work(case):
    c = case
    rows, k = c["rows"], c["k"]
    blocks = {4: 17 / 32, 8: 33 / 32}  # bytes an element, its scale's share among them
    if c["op"] == "quantize":
        value = 2 if c["src"] == "bf16" else 4
        back = blocks[4] + 2 if c["bits"] == 4 else 0  # read again and written as bf16
        return {"bytes": rows * k * (value + blocks[c["bits"]] + back), "flops": 0.0}
    if c["op"] == "norm":
        return {"bytes": rows * k * ((10 if c["add"] else 4) + blocks[8]) + 4 * k, "flops": 4.0 * rows * k}
    mats = 2 if c["op"] == "mlp13" else 1
    out = rows * c["n"] * (blocks[8] if c["op"] == "mlp13" else 2)
    return {"bytes": mats * c["n"] * k * blocks[4] + rows * k * blocks[8] + out, "flops": 2.0 * mats * rows * c["n"] * k}


# ---------------------------------------------------------------------------
# The definitions in 64 bits. What a pass holds in 8 bits is given here before that last rounding; the
# 4-bit values are what their pass computes, so they are rounded.

def exact(case, seed):
    s = prepare(case, seed)
    c = case
    rows = c["rows"]
    if c["op"] == "quantize":
        a = _rows_of(s["tiles"], rows).double()
        return _before8(a) if c["bits"] == 8 else _nearest4(a)
    if c["op"] == "norm":
        h = s["h"].double() if s["add"] is None else s["h"].double() + s["add"].double()
        a = _rows_of(h, rows)
        rms = (a.square().sum(1) / c["k"] + EPS).sqrt()
        return {"h": h, **_before8(a / rms[:, None] * s["gain"].double())}
    x = _exact_values(*s["x"], 8)[:rows]
    ws = [_exact_values(*w, 4)[: c["n"]] for w in s["w"]]
    if c["op"] == "gemm":
        return _tiles_of(x @ ws[0].t())
    gate, up = x @ ws[0].t(), x @ ws[1].t()
    return _before8(gate * torch.sigmoid(gate) * up)


def _exact_values(codes, scales, bits):
    """Each byte looked up in a table of all 256, times two to the power of its scale."""
    if bits == 8:
        def value(b):
            e, m = b >> 3 & 15, b & 7
            return (-1.0 if b & 128 else 1.0) * (math.ldexp(8 + m, e - 10) if e else math.ldexp(m, -9))

        look = torch.tensor([value(b) for b in range(256)], dtype=torch.float64, device=DEV)
        v = torch.empty((codes.shape[0], 16, codes.shape[1] * 128), dtype=torch.float64, device=DEV)
        for half in range(2):
            for part in range(4):
                at = (torch.arange(codes.shape[1], device=DEV) * 128 + 64 * half + 16 * part)[:, None] + torch.arange(16, device=DEV)
                v[:, :, at.reshape(-1)] = look[codes[:, :, half, part].long()].transpose(1, 2).reshape(v.shape[0], 16, -1)
    else:
        look = torch.tensor([(-1.0 if n & 8 else 1.0) * E2M1[n & 7] for n in range(16)], dtype=torch.float64, device=DEV)
        v = torch.empty((codes.shape[0], 16, codes.shape[1] * 128), dtype=torch.float64, device=DEV)
        for part in range(4):
            b = codes[:, :, part].long().transpose(1, 2)  # [tile][row][chunk][byte]
            at = (torch.arange(codes.shape[1], device=DEV) * 128 + 32 * part)[:, None] + 2 * torch.arange(16, device=DEV)
            v[:, :, at.reshape(-1)] = look[b % 16].reshape(v.shape[0], 16, -1)
            v[:, :, at.reshape(-1) + 1] = look[b // 16].reshape(v.shape[0], 16, -1)
    block = torch.arange(v.shape[2], device=DEV) // 32
    byte = scales[:, block // 16, block % 4, :, block // 4 % 4]  # [K][tile][row]
    return (v * 2.0 ** (byte.double().permute(1, 2, 0) - 127)).reshape(-1, v.shape[2])


def _nearest4(a):
    """The multiples of a step that grows with the magnitude, in units of the block's scale."""
    k = a.shape[1]
    b = _wide(a).reshape(-1, 32)
    top = b.abs().max(-1, keepdim=True).values
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -120)))
    scale = 2.0 ** (torch.where(top >= 1.75 * 2.0 ** e, e + 1, e) - 2)
    v = b / scale
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
    return (torch.round(v / step) * step * scale).reshape(-1, _up(k, 512))[: a.shape[0], :k]


def _before8(a):
    """Values [rows][K] in 64 bits -> elements before their rounding, and scales."""
    rows = a.shape[0]
    a = _wide(a)
    top = a.abs().reshape(a.shape[0], -1, 32).max(-1).values
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -200)))
    e = torch.where(top > 1.8125 * 2.0 ** e, e + 1, e).sub(8).clamp(min=-127)
    scale = 2.0 ** e
    el = (a.reshape(a.shape[0], -1, 32) / scale[..., None]).reshape(a.shape)
    scale[rows:] = 2.0 ** -127
    return {"elements": _pack8(el), "scales": scale.reshape(-1, 16, a.shape[1] // 512, 4, 4).permute(0, 2, 4, 1, 3).contiguous()}
