"""8-bit floats in 64-bit numpy: the definition of blocks, roundings by hand, and bounds on what f32 arithmetic may do to them."""
import numpy as np

U = 2.0 ** -24  # half a step of f32
BLOCK, TOP, LEAST = 128, 448.0, 7 * 2.0 ** -120


def values():
    """The 256 e4m3 values: 4 exponent bits with a bias of 7, 3 fraction bits, no infinities, NaN where all seven bits are set."""
    out = np.empty(256)
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        v = np.nan if c & 127 == 127 else (1 + f / 8) * 2.0 ** (e - 7) if e else f / 8 * 2.0 ** -6
        out[c] = -v if c & 128 else v
    return out


VALUES = values()


def e4m3(v):
    """v rounded to the nearest e4m3 value, ties to even, largest 448."""
    step = 2.0 ** (np.frexp(np.maximum(np.abs(v), 2.0 ** -6))[1] - 4.0)
    return np.clip(np.rint(v / step) * step, -TOP, TOP)


def columns(per_block, n):
    return np.repeat(per_block, BLOCK, axis=-1)[..., :n]


def tops(v):
    """[rows, blocks] largest magnitudes."""
    r, n = v.shape
    nb = -(-n // BLOCK)
    p = np.zeros((r, nb * BLOCK))
    p[:, :n] = np.abs(v)
    return p.reshape(r, nb, BLOCK).max(-1)


def check_rows(codes, scales, v, dv):
    """codes (bytes) and scales of rows whose values are v, known to the kernel to within dv: a scale is a / 448 of a largest magnitude
    inside the bounds, and a code the rounding of a quotient inside them (roundings keep the order). Both quotients and the product are
    f32 operations: half a step each."""
    n = v.shape[1]
    low, high = np.maximum(tops(np.maximum(np.abs(v) - dv, 0)), LEAST), np.maximum(tops(np.abs(v) + dv), LEAST)
    assert np.all(scales >= low / TOP * (1 - 1.01 * U)) and np.all(scales <= high / TOP * (1 + 1.01 * U))
    got = VALUES[codes]
    assert np.all(got >= e4m3(np.where(v - dv > 0, (v - dv) * columns(TOP / high, n) * (1 - 2.01 * U), (v - dv) * columns(TOP / low, n) * (1 + 2.01 * U))))
    assert np.all(got <= e4m3(np.where(v + dv > 0, (v + dv) * columns(TOP / low, n) * (1 + 2.01 * U), (v + dv) * columns(TOP / high, n) * (1 - 2.01 * U))))


def quantise(v, tall=1):
    """Codes (bytes) and f32 scales of v in blocks of `tall` rows x 128 columns, to make operands with."""
    r, n = v.shape
    rb, nb = -(-r // tall), -(-n // BLOCK)
    p = np.zeros((rb * tall, nb * BLOCK))
    p[:r, :n] = v
    p = p.reshape(rb, tall, nb, BLOCK)
    a = np.maximum(np.abs(p).max(axis=(1, 3), keepdims=True), LEAST)
    q = e4m3(p * (TOP / a)).reshape(rb * tall, -1)[:r, :n]
    order = np.argsort(VALUES[:127])
    codes = order[np.searchsorted(VALUES[:127][order], np.abs(q))].astype(np.uint8) | np.where(np.signbit(q), 128, 0).astype(np.uint8)
    return codes, (a / TOP).reshape(rb, nb).astype(np.float32)


def product(x, xs, w, ws):
    """(y, bound): the product in 64 bits, and how far f32 sums may be from it. A product of two codes has 8 significant bits and is exact;
    a block's 128 are added in f32, at most a whole step of the running sum each (the tensor cores may cut off instead of rounding), the
    scales' product and the blocks' additions are half a step each."""
    xv, wv = VALUES[x] * columns(xs.astype(np.float64), x.shape[1]), VALUES[w] * columns(np.repeat(ws.astype(np.float64), BLOCK, 0)[: w.shape[0]], w.shape[1])
    blocks = xs.shape[1]
    return xv @ wv.T, (2 * BLOCK + blocks + 3) * U * (np.abs(xv) @ np.abs(wv).T)


def bf16(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def to_bf16(v):
    """bf16 bits of f32 values, to nearest even (finite)."""
    b = np.ascontiguousarray(v, dtype=np.float32).view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def held(kind, v):
    """(array to upload, its values in 64 bits) of v in a type: "f32", "f16" or "bf16"."""
    a = to_bf16(v) if kind == "bf16" else np.asarray(v, dtype=np.float16 if kind == "f16" else np.float32)
    return a, (bf16(a) if kind == "bf16" else a).astype(np.float64)


def read(kind, a):
    return (bf16(a) if kind == "bf16" else a).astype(np.float64)


HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
