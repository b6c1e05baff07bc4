"""Measured cases of the microscaled 4-bit operators: quantisation (with its inverse), the product
of two quantised matrices, and the gated feed-forward product.

A quantised matrix of `rows` x `k` holds e2m1 codes, two to a byte (the even k in the low nibble),
each row padded with zero codes to a multiple of 32, and one scale per block of consecutive k: "mx"
an e8m0 scale (a power of two) per 32, "nv" an e4m3 scale per 16.  The scales are stored in tiles of
128 rows x 4 blocks, byte (r % 32) * 16 + (r / 32) * 4 + b of the 512-byte tile, tiles of one row
group next to each other; rows and blocks that do not exist have scale byte 0.

    block scale   mx: 2^(floor(log2 amax) - 2)     nv: e4m3(amax / 6)
    code          e2m1 of x / scale, ties to the even code, saturated at 6
    product       D = act(alpha * A B^T + beta * C + bias)
    gated         H = act(alpha_gate * A G^T) * (alpha_up * A U^T), optionally quantised along its rows
"""
import math

import torch

own = False

BLOCK = {"mx": 32, "nv": 16}
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------ cases
def _quantise(name, rows, k, format, type, columns=False, multiplier=1.0):
    return {"name": name, "op": "quantise", "rows": rows, "k": k, "format": format, "type": type,
            "columns": columns, "multiplier": multiplier}


def _product(name, m, n, k, format, type, alpha=1.0, beta=0.0, bias=False, act="none"):
    return {"name": name, "op": "product", "m": m, "n": n, "k": k, "format": format, "type": type,
            "alpha": alpha, "beta": beta, "bias": bias, "act": act}


def _gated(name, m, n, k, format, type, act="silu"):
    return {"name": name, "op": "gated", "m": m, "n": n, "k": k, "format": format, "type": type, "act": act}


def _block(name, m, n, k, format, type, act="silu"):
    return {"name": name, "op": "block", "m": m, "n": n, "k": k, "format": format, "type": type, "act": act}


def listed():
    return [
        # one token's activations before a projection: nothing but latency
        _quantise("quantise_1x4096_nv", 1, 4096, "nv", "bf16"),
        # the activations of a long prompt or a training batch
        _quantise("quantise_16384x4096_mx", 16384, 4096, "mx", "bf16"),
        # a trained weight in fp32, stored K x N row-major (the default layout of B here), blocks along
        # K; weights are small, so they are scaled up first
        _quantise("quantise_weight_14336x4096_nv", 14336, 4096, "nv", "f32", columns=True, multiplier=256.0),
        # neither rows nor K fill a tile
        _quantise("quantise_ragged_1003x1000_mx_columns", 1003, 1000, "mx", "f16", columns=True),
        # decode: one token, and a small batch, against a streamed weight
        _product("product_1x14336x4096_nv", 1, 14336, 4096, "nv", "bf16"),
        _product("product_16x4096x14336_mx", 16, 4096, 14336, "mx", "bf16"),
        # the framework's headline size
        _product("product_8192_mx", 8192, 8192, 8192, "mx", "bf16"),
        # prompt-sized product that adds to a residual stream
        _product("product_2048x14336x4096_nv_residual", 2048, 14336, 4096, "nv", "f16", alpha=0.5, beta=1.0),
        # nothing fills a tile; bias, activation, fp32 out
        _product("product_ragged_1000x1500x1100_mx_gelu", 1000, 1500, 1100, "mx", "f32", bias=True, act="gelu_tanh"),
        # the gated half of a feed-forward layer: one token, and a prompt
        _gated("gated_1x14336x4096_mx", 1, 14336, 4096, "mx", "bf16"),
        _gated("gated_2048x14336x4096_nv", 2048, 14336, 4096, "nv", "bf16"),
        # a whole feed-forward layer on 4-bit weights: quantise x, gated product with a quantised result,
        # down projection
        _block("block_512x14336x4096_nv", 512, 14336, 4096, "nv", "bf16"),
    ]


MOST_FLOPS = 2 * 8192 ** 3


def _size(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:  # every other size as it falls, the rest in the multiples that widths come in
        return max(lo, v)
    step = rng.choice([16, 32, 64, 128])
    return min(hi, max(lo, (v + step - 1) // step * step))


def draw(rng):
    op = rng.choice(["quantise", "product", "product", "gated", "block"])
    fmt = rng.choice(["mx", "nv"])
    if op == "quantise":
        type = rng.choice(["bf16", "f16", "f32"])
        while True:
            rows, k = _size(rng, 1, 16384), _size(rng, 1, 16384)
            if rows * k <= 14336 * 4096:
                break
        c = _quantise("", rows, k, fmt, type, rng.random() < 0.5, rng.choice([1.0, 1.0, 16.0, 256.0]) if fmt == "nv" else 1.0)
    else:
        while True:
            m, n, k = _size(rng, 1, 8192), _size(rng, 16, 16384), _size(rng, 16, 16384)
            products = {"product": 1, "gated": 2, "block": 3}[op]
            if 2 * m * n * k * products <= MOST_FLOPS:
                break
        if op == "product":
            type = rng.choice(["bf16", "bf16", "f16", "f32"])
            c = _product("", m, n, k, fmt, type, rng.choice([1.0, 0.5, 2.0]), rng.choice([0.0, 0.0, 1.0, -0.5]),
                         rng.random() < 0.3, rng.choice(["none", "none", "relu", "gelu", "gelu_tanh", "silu"]))
        elif op == "gated":
            c = _gated("", m, n, k, fmt, rng.choice(["bf16", "f16"]), rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"]))
        else:
            c = _block("", m, n, k, fmt, rng.choice(["bf16", "f16"]), rng.choice(["silu", "silu", "gelu_tanh"]))
    del c["name"]
    return c


# ------------------------------------------------------------------------------------ plain forms
def _tile_scales(linear, rows, blocks):
    """rows x blocks bytes -> the tiled layout, flat."""
    rg, bg = -(-rows // 128), -(-blocks // 4)
    s = torch.zeros(rg * 128, bg * 4, dtype=torch.uint8, device=linear.device)
    s[:rows, :blocks] = linear
    return s.view(rg, 4, 32, bg, 4).permute(0, 3, 2, 1, 4).reshape(-1)


def _linear_scales(tiled, rows, blocks):
    rg, bg = -(-rows // 128), -(-blocks // 4)
    return tiled.view(rg, bg, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rg * 128, bg * 4)[:rows, :blocks]


def _scale_values(bytes_, fmt):
    if fmt == "mx":
        return torch.ldexp(torch.ones_like(bytes_, dtype=torch.float32), bytes_.to(torch.int32) - 127)
    return bytes_.view(torch.float8_e4m3fn).to(torch.float32)


def _decode(codes, scales, rows, k, fmt):
    """The fp32 values of a quantised matrix."""
    values = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    w = torch.stack((values[(codes & 15).long()], values[(codes >> 4).long()]), dim=-1).view(rows, -1)
    block = BLOCK[fmt]
    blocks = -(-k // block)
    s = _scale_values(_linear_scales(scales, rows, blocks).contiguous(), fmt)
    return (w.view(rows, -1, block)[:, :blocks] * s[:, :, None]).view(rows, -1)[:, :k]


def _encode(x, fmt):
    """codes and tiled scales of fp32 values, blocks along the rows."""
    rows, k = x.shape
    block = BLOCK[fmt]
    blocks, pitch = -(-k // block), -(-k // 32) * 32
    padded = torch.zeros(rows, blocks * block, dtype=torch.float32, device=x.device)
    padded[:, :k] = x
    b = padded.view(rows, blocks, block)
    amax = b.abs().amax(dim=2)
    if fmt == "mx":
        e = torch.where(amax > 0, torch.frexp(amax)[1] - 3, -127).clamp(-127, 127)
        byte = (e + 127).to(torch.uint8)
    else:
        byte = (amax / 6.0).clamp(max=448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    s = _scale_values(byte, fmt)[:, :, None]
    a = torch.where(s > 0, b.abs() / s, torch.zeros_like(b))
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code | (torch.signbit(b).to(torch.uint8) << 3)).view(rows, -1)
    full = torch.zeros(rows, max(pitch, blocks * block), dtype=torch.uint8, device=x.device)
    full[:, :code.shape[1]] = code
    full = full[:, :pitch]
    return (full[:, 0::2] | (full[:, 1::2] << 4)).contiguous(), _tile_scales(byte, rows, blocks)


def _act(x, name):
    if name == "relu":
        return x.clamp(min=0)
    if name == "gelu":
        return 0.5 * x * (1 + torch.erf(x / math.sqrt(2)))
    if name == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    if name == "silu":
        return x / (1 + torch.exp(-x))
    return x


def _plain(s):
    c = s["case"]
    fmt, out = c["format"], TYPES[c["type"]]
    if c["op"] == "quantise":
        x = s["x"].float() * c["multiplier"]
        codes, scales = _encode(x.t().contiguous() if c["columns"] else x, fmt)
        y = _decode(codes, scales, c["rows"], c["k"], fmt) / c["multiplier"]
        return (y.t().contiguous() if c["columns"] else y).to(out)
    m, n, k = c["m"], c["n"], c["k"]
    if c["op"] == "product":
        d = c["alpha"] * (_decode(*s["a"], m, k, fmt) @ _decode(*s["b"], n, k, fmt).t())
        if c["beta"]:
            d = d + c["beta"] * s["c"].float()
        if c["bias"]:
            d = d + s["bias"]
        return _act(d, c["act"]).to(out)
    a = s["a"] if c["op"] == "gated" else _encode(s["x"].float(), fmt)
    a = _decode(*a, m, k, fmt)
    h = _act(s["alpha"] * (a @ _decode(*s["gate"], n, k, fmt).t()), c["act"])
    h = h * (s["alpha"] * (a @ _decode(*s["up"], n, k, fmt).t()))
    if c["op"] == "gated":
        return h.to(out)
    h = _decode(*_encode(h, fmt), m, n, fmt)
    return (s["alpha"] * (h @ _decode(*s["down"], k, n, fmt).t())).to(out)


# ------------------------------------------------------------------------------- the measured call
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _weight(rows, k, fmt, g):
    """A weight as a trained one is spread, N(0, 0.02), quantised; nv after scaling by 256."""
    return _encode(torch.randn(rows, k, device="cuda", generator=g) * (0.02 * (256.0 if fmt == "nv" else 1.0)), fmt)


def prepare(case, seed):
    g = _generator(seed)
    c, s = case, {"case": case}
    out = TYPES[c["type"]]
    if c["op"] == "quantise":
        shape = (c["k"], c["rows"]) if c["columns"] else (c["rows"], c["k"])
        x = torch.randn(shape, device="cuda", generator=g)
        # activations have a few wide channels; weights are narrow
        if c["multiplier"] == 1.0:
            wide = torch.rand(c["k"], device="cuda", generator=g) < 0.01
            width = torch.where(wide, 20.0, 1.0)
            x = x * (width[:, None] if c["columns"] else width)
        else:
            x = x * 0.02
        s["x"] = x.to(out)
        if own:
            import gemm_zoo_b200 as gz
            s["q"] = gz.MxMatrix.empty(c["rows"], c["k"], _format(gz, c))
            s["y"] = torch.empty_like(s["x"])
        return s
    m, n, k, fmt = c["m"], c["n"], c["k"], c["format"]
    s["alpha"] = 1 / 256.0 if fmt == "nv" else 1.0  # undoes the scaling of an nv weight
    x = torch.randn(m, k, device="cuda", generator=g)
    if c["op"] == "product":
        s["a"], s["b"] = _encode(x, fmt), _weight(n, k, fmt, g)
        s["c"] = torch.randn(m, n, device="cuda", generator=g).to(out) if c["beta"] else None
        s["bias"] = torch.randn(n, device="cuda", generator=g) if c["bias"] else None
    else:
        s["gate"], s["up"] = _weight(n, k, fmt, g), _weight(n, k, fmt, g)
        if c["op"] == "gated":
            s["a"] = _encode(x, fmt)
        else:
            s["x"], s["down"] = x.to(out), _weight(k, n, fmt, g)
    if own:
        import gemm_zoo_b200 as gz
        f = _format(gz, c)
        for name in ("a", "b", "gate", "up", "down"):
            if name in s:
                rows, cols = {"a": (m, k), "b": (n, k), "gate": (n, k), "up": (n, k), "down": (k, n)}[name]
                s["q_" + name] = gz.MxMatrix(s[name][0], s[name][1], rows, cols, f)
        if c["op"] == "product":
            s["plan"] = gz.MxGemm(m, n, k, f, out)
            s["d"] = torch.empty(m, n, dtype=out, device="cuda")
        elif c["op"] == "gated":
            s["plan"] = gz.MxGated(m, n, k, f, out, activation=_activation(gz, c))
            s["d"] = torch.empty(m, n, dtype=out, device="cuda")
        else:
            s["plan"] = gz.MxGated(m, n, k, f, f, activation=_activation(gz, c))
            s["plan_down"] = gz.MxGemm(m, k, n, f, out)
            s["q_x"], s["q_h"] = gz.MxMatrix.empty(m, k, f), gz.MxMatrix.empty(m, n, f)
            s["d"] = torch.empty(m, k, dtype=out, device="cuda")
    return s


def _format(gz, c):
    return {"mx": gz.MX_FP4, "nv": gz.MX_NVFP4}[c["format"]]


def _activation(gz, c):
    return {"none": gz.ACT_NONE, "relu": gz.ACT_RELU, "gelu": gz.ACT_GELU, "gelu_tanh": gz.ACT_GELU_TANH, "silu": gz.ACT_SILU}[c["act"]]


def run(state):
    if not own:
        return _plain(state)
    import gemm_zoo_b200 as gz
    s, c = state, state["case"]
    stream = torch.cuda.current_stream()
    if c["op"] == "quantise":
        layout = gz.COL_MAJOR if c["columns"] else gz.ROW_MAJOR
        gz.mx_quantize(s["x"], _format(gz, c), layout=layout, multiplier=c["multiplier"], out=s["q"], stream=stream)
        return gz.mx_dequantize(s["q"], s["y"], layout=layout, multiplier=1.0 / c["multiplier"], stream=stream)
    if c["op"] == "product":
        s["plan"](s["q_a"], s["q_b"], s["c"], s["d"], c["alpha"], c["beta"], bias=s["bias"],
                  activation=_activation(gz, c), stream=stream)
        return s["d"]
    if c["op"] == "gated":
        s["plan"](s["q_a"], s["q_gate"], s["q_up"], s["d"], s["alpha"], s["alpha"], stream=stream)
        return s["d"]
    gz.mx_quantize(s["x"], _format(gz, c), out=s["q_x"], stream=stream)
    s["plan"](s["q_x"], s["q_gate"], s["q_up"], s["q_h"], s["alpha"], s["alpha"], stream=stream)
    s["plan_down"](s["q_h"], s["q_down"], None, s["d"], s["alpha"], 0.0, stream=stream)
    return s["d"]


# ------------------------------------------------------------------------------- what a pass needs
def _quantised_bytes(rows, k, fmt):
    return rows * (-(-k // 2)) + rows * (-(-k // BLOCK[fmt]))


def work(case):
    c = case
    fmt, size = c["format"], SIZE[c["type"]]
    if c["op"] == "quantise":
        # the matrix is read, quantised, and written back from its codes
        return {"bytes": 2 * c["rows"] * c["k"] * size + 2 * _quantised_bytes(c["rows"], c["k"], fmt), "flops": 4 * c["rows"] * c["k"]}
    m, n, k = c["m"], c["n"], c["k"]
    if c["op"] == "product":
        moved = _quantised_bytes(m, k, fmt) + _quantised_bytes(n, k, fmt) + m * n * size * (2 if c["beta"] else 1)
        return {"bytes": moved + (4 * n if c["bias"] else 0), "flops": 2 * m * n * k}
    if c["op"] == "gated":
        return {"bytes": _quantised_bytes(m, k, fmt) + 2 * _quantised_bytes(n, k, fmt) + m * n * size, "flops": 4 * m * n * k}
    # x is read and the result written once; the quantised x and h are written and read
    moved = 2 * m * k * size + 2 * _quantised_bytes(m, k, fmt) + 2 * _quantised_bytes(m, n, fmt)
    moved += 2 * _quantised_bytes(n, k, fmt) + _quantised_bytes(k, n, fmt)
    return {"bytes": moved, "flops": 6 * m * n * k}


# ---------------------------------------------------------------------------- 64-bit values
def _round_blocks_64(x, fmt):
    """The values that a quantised x (64 bits, blocks along its rows) stands for, by rounding to the grid
    of each binade: steps of 1/2 up to 2, of 1 up to 4, of 2 up to 6."""
    rows, k = x.shape
    block = BLOCK[fmt]
    pad = -k % block
    b = torch.nn.functional.pad(x, (0, pad)).reshape(rows, -1, block)
    top = b.abs().amax(dim=2, keepdim=True)
    if fmt == "mx":
        exponent = torch.frexp(torch.where(top > 0, top, torch.ones_like(top)))[1].double() - 3
        scale = torch.exp2(exponent.clamp(-127, 127))
    else:
        t = (top / 6).clamp(max=448.0)
        # e4m3: three fraction bits, exponents from -6, subnormal below
        step = torch.exp2((torch.frexp(t.clamp(min=2.0 ** -6))[1] - 1).double() - 3)
        scale = torch.round(t / step) * step
    y = b / torch.where(scale > 0, scale, torch.ones_like(scale))
    y = torch.where(scale > 0, y, torch.zeros_like(y))
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    r = (torch.round(a / step) * step).clamp(max=6.0) * torch.sign(y)
    return (r * scale).reshape(rows, -1)[:, :k]


def _values_64(q, rows, k, fmt):
    """What a quantised matrix stands for, in 64 bits, from the bits of its codes and scales."""
    codes, scales = q
    n = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(rows, -1)[:, :k].to(torch.int16)
    e, f = (n >> 1) & 3, (n & 1).double()
    mag = torch.where(e == 0, f * 0.5, (1 + f / 2) * torch.exp2((e - 1).double()))
    mag = torch.where((n & 8) != 0, -mag, mag)
    r = torch.arange(rows, device=codes.device)[:, None]
    b = (torch.arange(k, device=codes.device) // BLOCK[fmt])[None, :]
    groups = -(-(-(-k // BLOCK[fmt])) // 4)
    byte = scales[((r // 128) * groups + b // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4].to(torch.int16)
    if fmt == "mx":
        return mag * torch.exp2(byte.double() - 127)
    e, f = byte >> 3, (byte & 7).double()
    return mag * torch.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * torch.exp2(e.double() - 7))


def _act_64(x, name):
    if name == "relu":
        return torch.where(x > 0, x, torch.zeros_like(x))
    if name == "gelu":
        return x * torch.erfc(-x * math.sqrt(0.5)) / 2
    if name == "gelu_tanh":
        return x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x))
    if name == "silu":
        return x * torch.sigmoid(x)
    return x


def exact(case, seed):
    c = case
    if c["op"] == "quantise" and c["rows"] * c["k"] > 70_000_000:
        return None
    s = prepare(case, seed)
    fmt = c["format"]
    if c["op"] == "quantise":
        x = s["x"].double() * c["multiplier"]
        y = _round_blocks_64(x.t() if c["columns"] else x, fmt) / c["multiplier"]
        return y.t().contiguous() if c["columns"] else y
    m, n, k = c["m"], c["n"], c["k"]
    if c["op"] == "product":
        d = _values_64(s["a"], m, k, fmt) @ _values_64(s["b"], n, k, fmt).t() * c["alpha"]
        if c["beta"]:
            d += c["beta"] * s["c"].double()
        if c["bias"]:
            d += s["bias"].double()
        return _act_64(d, c["act"])
    a = _values_64(s["a"], m, k, fmt) if c["op"] == "gated" else _round_blocks_64(s["x"].double(), fmt)
    h = _act_64(a @ _values_64(s["gate"], n, k, fmt).t() * s["alpha"], c["act"])
    h *= a @ _values_64(s["up"], n, k, fmt).t() * s["alpha"]
    if c["op"] == "gated":
        return h
    return _round_blocks_64(h, fmt) @ _values_64(s["down"], k, n, fmt).t() * s["alpha"]
