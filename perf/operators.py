"""The products over 8-bit floats that are measured, and what makes their operands: rows of e4m3 codes with an f32 scale per block of
128 columns, weights of e4m3 codes with an f32 scale per block of 128 x 128.

A case is a dict of sizes and types. `listed()` names the fixed ones, `draw(rng)` gives more of the same ranges, `prepare` makes what a
program holds before the call, `run` is one pass (`own`: the framework's entry points, else the plain form in torch), `exact` the same
outputs from the definition in 64 bits. Sizes are those of a Llama-3-8B-shaped decoder (width 4096, feed-forward 14336), of the
repository's decoders of width 2048 with a feed-forward of 8192, or generic ones around them; odd and ragged ones stand among them.

  quantize   rows in blocks of 128: a = the block's largest magnitude (at least 7 * 2^-120), scale = a / 448, code = e4m3(v * (448 / a))
  silu_mul   the same of v = silu(gate) * up, gate and up side by side in a row (what one stacked product leaves)
  rms_norm   the same of v = s / sqrt(mean(s^2) + eps) * weight (+ bias), s = x + residual; s comes back too
  product    y = x . w^T (+ residual or bias), x and w the values that codes and scales stand for
"""
import math
import zlib

import torch

own = False

BLOCK = 128
TOP = 448.0              # the largest e4m3 value
LEAST = 7 * 2.0 ** -120  # the least magnitude a scale is made from: TOP / LEAST and LEAST / TOP are normal numbers
EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MOST_WORK = 8192 * 28672 * 4096  # multiplications of the largest product


def listed():
    return [
        # the output of a single token's attention on its way into the output projection: the smallest call
        dict(name="quantize_1x4096_bf16", op="quantize", rows=1, n=4096, type="bf16"),
        # a prompt's attention output in a width of no round number of blocks
        dict(name="quantize_3001x2056_f32", op="quantize", rows=3001, n=2056, type="f32"),
        # the hidden row of a feed-forward, a few sequences at a time, and that of a prompt
        dict(name="silu_mul_9x14336_bf16", op="silu_mul", rows=9, n=14336, type="bf16"),
        dict(name="silu_mul_4096x14336_bf16", op="silu_mul", rows=4096, n=14336, type="bf16"),
        # the norm in front of a single token's projections; the stream is f32 as everywhere in this framework
        dict(name="rms_norm_1x4096_f32", op="rms_norm", rows=1, n=4096, type="f32", residual=True, bias=False),
        # the same for the tokens of a long prompt, and for a stream of 16 bits
        dict(name="rms_norm_8192x4096_f32", op="rms_norm", rows=8192, n=4096, type="f32", residual=True, bias=False),
        dict(name="rms_norm_1111x2048_bf16", op="rms_norm", rows=1111, n=2048, type="bf16", residual=True, bias=False),
        # one token through a square projection: latency counts
        dict(name="product_1x4096x4096", op="product", m=1, n=4096, k=4096, type="f32", epilogue="none"),
        # the down projection of a few sequences, added to the stream
        dict(name="product_12x4096x14336_residual", op="product", m=12, n=4096, k=14336, type="f32", epilogue="residual"),
        # a short prompt, ragged on every side, with a bias
        dict(name="product_203x5003x2300_bias", op="product", m=203, n=5003, k=2300, type="f16", epilogue="bias"),
        # the stacked q, k and v of a prompt
        dict(name="product_1024x6144x4096", op="product", m=1024, n=6144, k=4096, type="bf16", epilogue="none"),
        # gate and up of a long prompt: the largest
        dict(name="product_8192x28672x4096", op="product", m=8192, n=28672, k=4096, type="bf16", epilogue="none"),
    ]


def _log(rng, lo, hi, step=1):
    """A size between lo and hi, evenly spread over its logarithm, a multiple of `step`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["quantize", "silu_mul", "rms_norm", "product", "product", "product"])
    kind = rng.choice(sorted(TYPES))
    if op == "product":
        m = rng.choice([1, _log(rng, 2, 16), _log(rng, 17, 256), _log(rng, 257, 8192)])
        n, k = _log(rng, 256, 28672, rng.choice([1, 128])), _log(rng, 128, 14336, rng.choice([1, 128]))
        while m * n * k > MOST_WORK:
            n, k = max(256, n // 2), max(128, k // 2)
        return dict(op=op, m=m, n=n, k=k, type=kind, epilogue=rng.choice(["none", "residual", "bias"]))
    rows, n = rng.choice([1, _log(rng, 2, 64), _log(rng, 65, 8192)]), _log(rng, 128, 14336, rng.choice([1, 8, 128]))
    if op == "rms_norm":
        return dict(op=op, rows=rows, n=n, type=kind, residual=rng.random() < 0.7, bias=rng.random() < 0.2)
    return dict(op=op, rows=rows, n=n, type=kind)


# ---- inputs -------------------------------------------------------------------------------------------------------------

def _gen(seed, name):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + zlib.crc32(name.encode())) % (1 << 62))


def _normal(seed, name, shape, sigma=1.0):
    return torch.randn(shape, generator=_gen(seed, name), device="cuda", dtype=torch.float32) * sigma


def _stream(seed, name, rows, n):
    """Rows of a residual stream: channels of different spread, and one in a hundred that stands out."""
    spread = torch.exp(0.5 * _normal(seed, name + ".spread", (n,)))
    spread[torch.rand((n,), generator=_gen(seed, name + ".out"), device="cuda") < 0.01] *= 20
    return _normal(seed, name, (rows, n)) * spread


def _padded(t, step):
    """t [rows, n] as a view into rows of a multiple of `step` values."""
    rows, n = t.shape
    held = torch.zeros((rows, -(-n // step) * step), dtype=t.dtype, device=t.device)
    held[:, :n] = t
    return held[:, :n]


def _blocks_of(v, tall):
    """v [r, n] f32 in blocks of `tall` rows and 128 columns: codes as float8 values, one scale per block."""
    r, n = v.shape
    rb, nb = -(-r // tall), -(-n // BLOCK)
    held = torch.nn.functional.pad(v, (0, nb * BLOCK - n, 0, rb * tall - r)).view(rb, tall, nb, BLOCK)
    top = held.abs().amax(dim=(1, 3), keepdim=True)
    top = torch.where(torch.isfinite(top), top.clamp(min=LEAST), torch.nan)
    codes = (held * (TOP / top)).to(torch.float8_e4m3fn).view(rb * tall, nb * BLOCK)[:r, :n]
    return codes, (top / TOP).view(rb, nb)


def _inputs(c, seed):
    """The torch tensors of a case."""
    if c["op"] == "product":
        m, n, k = c["m"], c["n"], c["k"]
        x, xs = _blocks_of(_stream(seed, "x", m, k), 1)
        w, ws = _blocks_of(_normal(seed, "w", (n, k), 1.28 * k ** -0.5), BLOCK)
        s = dict(x=_padded(x, 16), xs=xs, w=_padded(w, 16), ws=ws)
        if c["epilogue"] == "residual":
            s["add"] = _normal(seed, "add", (m, n))
        if c["epilogue"] == "bias":
            s["add"] = _normal(seed, "add", (n,))
        return s
    rows, n, t = c["rows"], c["n"], TYPES[c["type"]]
    if c["op"] == "silu_mul":
        return dict(x=_normal(seed, "x", (rows, 2 * n), 1.5).to(t))
    s = dict(x=_stream(seed, "x", rows, n).to(t))
    if c["op"] == "rms_norm":
        s["weight"] = 1 + 0.1 * _normal(seed, "weight", (n,))
        if c["residual"]:
            s["residual"] = _normal(seed, "residual", (rows, n), 0.7).to(t)
        if c["bias"]:
            s["bias"] = _normal(seed, "bias", (n,), 0.1)
    return s


_held = {}


def _device():
    """The program's one handle."""
    if "device" not in _held:
        import kalosm_b200
        _held["kb"], _held["device"] = kalosm_b200, kalosm_b200.Device(0)
    return _held["kb"], _held["device"]


def _tensor(t, shape=None):
    """A framework tensor over a torch tensor's memory (bf16 and 8-bit values as their bits)."""
    kb, dev = _device()
    kind = {torch.bfloat16: "uint16", torch.float8_e4m3fn: "uint8"}.get(t.dtype) or str(t.dtype).split(".")[1]
    return kb.Tensor(dev, shape or t.shape, kind, ptr=t.data_ptr())


def _rows(codes, scales):
    """Framework rows of 8 bits over torch memory; `codes` is a view into padded rows."""
    kb, dev = _device()
    return kb.F8Rows(dev, codes.shape, codes=_tensor(codes, (codes.shape[0], codes.stride(0))), scales=_tensor(scales))


def _new_rows(rows, n):
    codes = _padded(torch.zeros((rows, n), dtype=torch.float8_e4m3fn, device="cuda"), 16)
    return codes, torch.zeros((rows, -(-n // BLOCK)), dtype=torch.float32, device="cuda")


def prepare(case, seed):
    s = dict(case=case, t=_inputs(case, seed))
    if own:  # the same memory as the framework's tensors, the weights' handle, and the buffers that a program writes into
        kb, dev = _device()
        t = s["t"]
        if case["op"] == "product":
            s["x"] = _rows(t["x"], t["xs"])
            s["w"] = kb.F8Matrix.from_tensors(_tensor(t["w"], (case["n"], t["w"].stride(0))), _tensor(t["ws"]), case["k"])
            s["r1"] = _tensor(t["add"]) if "add" in t else None
            s["out"] = torch.empty((case["m"], case["n"]), dtype=TYPES[case["type"]], device="cuda")
            s["y"] = _tensor(s["out"])
            s["y_type"] = {"f32": kb.F32, "bf16": kb.BF16, "f16": kb.F16}[case["type"]]
            s["epilogue"] = {"none": kb.EPI_NONE, "residual": kb.EPI_RESIDUAL, "bias": kb.EPI_BIAS}[case["epilogue"]]
            return s
        s["codes"], s["scales"] = _new_rows(case["rows"], case["n"])
        s["out"] = _rows(s["codes"], s["scales"])
        s["in"] = {k: _tensor(v) for k, v in t.items()}
        if case["op"] == "rms_norm":
            s["sum"] = torch.empty_like(t["x"])
            s["in"]["sum"] = _tensor(s["sum"])
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------

def _run_own(s):
    c, (kb, dev) = s["case"], _device()
    if c["op"] == "product":
        s["x"].f8_mat_mul(s["w"], out_type=s["y_type"], epilogue=s["epilogue"], r1=s["r1"], out=s["y"])
        return dict(y=s["out"])
    i = s["in"]
    if c["op"] == "quantize":
        dev.quantize_f8(i["x"], out=s["out"])
    elif c["op"] == "silu_mul":
        dev.silu_mul_f8(i["x"], out=s["out"])
    else:
        dev.rms_norm_f8(i["x"], i["weight"], EPS, residual=i.get("residual"), bias=i.get("bias"), sum_out=i["sum"], out=s["out"])
        return dict(codes=s["codes"], scales=s["scales"], sum=s["sum"])
    return dict(codes=s["codes"], scales=s["scales"])


def _values(codes, scales, tall):
    """What codes and scales stand for, in f32."""
    r, n = codes.shape
    return codes.float() * scales.repeat_interleave(tall, 0)[:r].repeat_interleave(BLOCK, 1)[:, :n]


def run(state):
    if own:
        return _run_own(state)
    c, t = state["case"], state["t"]
    kind = TYPES[c["type"]]
    if c["op"] == "product":
        y = torch.matmul(_values(t["x"], t["xs"], 1), _values(t["w"], t["ws"], BLOCK).t())
        if "add" in t:
            y = y + t["add"]
        return dict(y=y.to(kind))
    x = t["x"].float()
    if c["op"] == "silu_mul":
        gate, up = x[:, : c["n"]], x[:, c["n"]:]
        x = gate / (1 + torch.exp(-gate)) * up
    elif c["op"] == "rms_norm":
        s = x + t["residual"].float() if "residual" in t else x
        x = s / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS) * t["weight"]
        if "bias" in t:
            x = x + t["bias"]
        codes, scales = _blocks_of(x, 1)
        return dict(codes=codes, scales=scales, sum=s.to(kind))
    codes, scales = _blocks_of(x, 1)
    return dict(codes=codes, scales=scales)


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["type"]]
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        kb = -(-k // BLOCK)
        add = {"none": 0, "residual": 4 * m * n, "bias": 4 * n}[case["epilogue"]]
        return dict(bytes=n * k + m * k + 4 * kb * (m + -(-n // BLOCK)) + size * m * n + add, flops=2 * m * n * k)
    rows, n = case["rows"], case["n"]
    out = rows * n + 4 * rows * -(-n // BLOCK)
    if case["op"] == "quantize":
        return dict(bytes=size * rows * n + out, flops=3 * rows * n)
    if case["op"] == "silu_mul":
        return dict(bytes=2 * size * rows * n + out, flops=8 * rows * n)
    read = (2 if case["residual"] else 1) * size * rows * n + (8 if case["bias"] else 4) * n
    return dict(bytes=read + size * rows * n + out, flops=8 * rows * n)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------

def _exact_rows(v):
    """Blocks of 128 columns in 64 bits; a code is rounded by hand, half to even, to 4 significant bits, below 2^-6 to a multiple of 2^-9."""
    r, n = v.shape
    nb = -(-n // BLOCK)
    top = torch.stack([v[:, b * BLOCK: (b + 1) * BLOCK].abs().max(dim=1).values for b in range(nb)], dim=1).clamp(min=LEAST)
    q = v * (TOP / top)[:, torch.arange(n, device=v.device) // BLOCK]
    step = torch.exp2(torch.frexp(q.abs().clamp(min=2.0 ** -6)).exponent.double() - 4)  # frexp's mantissa lies in [0.5, 1)
    return dict(codes=torch.round(q / step) * step, scales=top / TOP)


def exact(case, seed):
    t = {k: v.double() for k, v in _inputs(case, seed).items()}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        col = torch.arange(k, device="cuda") // BLOCK
        row = torch.arange(n, device="cuda") // BLOCK
        w = t["w"] * t["ws"][row][:, col]
        y = (t["x"] * t["xs"][:, col]) @ w.T
        return dict(y=y + t["add"] if "add" in t else y)
    x, n = t["x"], case["n"]
    if case["op"] == "silu_mul":
        return _exact_rows(x[:, :n] * torch.sigmoid(x[:, :n]) * x[:, n:])
    if case["op"] == "quantize":
        return _exact_rows(x)
    s = x + t["residual"] if case["residual"] else x
    v = s * torch.rsqrt((s * s).sum(1, keepdim=True) / n + EPS) * t["weight"]
    if case["bias"]:
        v = v + t["bias"]
    return dict(_exact_rows(v), sum=s)
