"""GPU parity of the operations over 8-bit floats: rows with a scale per block of 128, their norm and gated forms, and the product."""
import ctypes as C

import numpy as np
import pytest

import f8_util as F
import kalosm_b200 as kb
from gpu_util import dev  # noqa: F401

pytestmark = pytest.mark.gpu

TYPES = {"f32": kb.F32, "f16": kb.F16, "bf16": kb.BF16}
EPS = 1e-5
GUARD = 0xA5


def upload(dev, a):
    return dev.tensor(a)


def new_rows(dev, rows, n, extra=0):
    """Rows with `extra` more 16-byte pieces a row and two rows behind them, all bytes GUARD."""
    ld = -(-n // 16) * 16 + 16 * extra
    codes, scales = kb.Tensor(dev, (rows + 2, ld), np.uint8), kb.Tensor(dev, (rows + 2, -(-n // 128)), np.float32)
    codes.fill_bytes(GUARD)
    scales.fill_bytes(GUARD)
    return codes, scales, ld


def result(codes, scales, rows, n):
    """(codes [rows, n], scales) after a look at what was not to be written."""
    c, s = codes.as_slice(), scales.as_slice()
    assert np.all(c[:rows, n:] == GUARD) and np.all(c[rows:] == GUARD) and np.all(s[rows:].view(np.uint8) == GUARD)
    return c[:rows, :n], s[:rows].astype(np.float64)


def spread(rng, rows, n, sigma=1.0):
    """Values of several magnitudes, so that blocks, and columns inside them, differ."""
    return sigma * rng.standard_normal((rows, n)) * np.exp(rng.standard_normal((1, n))) * np.exp(0.5 * rng.standard_normal((rows, 1)))


# ---- rows ---------------------------------------------------------------------------------------------------------------

SHAPES = [(1, 1), (1, 127), (3, 128), (2, 129), (5, 300), (1, 4096), (33, 2056), (300, 515), (2, 14336), (9, 1024), (1, 4608), (4, 8200)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,n", SHAPES)
def test_quantize(dev, kind, rows, n):
    a, v = F.held(kind, spread(np.random.default_rng(rows * 7 + n), rows, n))
    out = dev.quantize_f8(upload(dev, a))
    F.check_rows(out.codes.as_slice()[:, :n], out.scales.as_slice().astype(np.float64), v, np.zeros_like(v))
    assert np.array_equal(out.as_slice(), (F.VALUES[out.codes.as_slice()[:, :n]] * F.columns(out.scales.as_slice(), n)).astype(np.float32))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("offset,pad", [(0, 8), (1, 0), (3, 5), (8, 3)])
def test_quantize_strided(dev, kind, offset, pad):
    rows, n = 7, 1290
    a, v = F.held(kind, spread(np.random.default_rng(pad), rows + 1, n + pad))
    t = upload(dev, a)
    codes, scales, ld = new_rows(dev, rows, n, 2)
    dev._check(dev.lib.fb200_quantize_f8(dev.h, t.ptr + offset * a.itemsize, n + pad, TYPES[kind], rows, n, codes.ptr, ld, scales.ptr))
    at = offset + np.arange(rows)[:, None] * (n + pad) + np.arange(n)
    got, s = result(codes, scales, rows, n)
    F.check_rows(got, s, v.reshape(-1)[at], np.zeros((rows, n)))


def test_quantize_special_values(dev):
    """Zeros, the least magnitudes, values on the border of two codes, and what is not finite."""
    v = np.zeros((8, 256), dtype=np.float32)
    v[1, :3] = [1e-45, -1e-38, 2.0 ** -120]  # below the least magnitude a scale is made from: codes of the least scale, 2^-126
    v[2, :2] = [np.float32(3.4e38), -1e30]
    v[3] = np.arange(256) * 1.75  # a = 222.25 and 446.25
    v[4, :128] = np.concatenate([[448], np.arange(127) / 16.0 + 1])  # scale 1: ties of the codes
    v[5, 5], v[5, 130] = np.inf, 1.0
    v[6, 7], v[6, 8], v[6, 200] = np.nan, 3.0, 2.0
    v[7, 128:] = -np.inf
    out = dev.quantize_f8(dev.tensor(v))
    codes, scales = out.codes.as_slice(), out.scales.as_slice()
    assert np.all(codes[0] == 0) and np.all(scales[:2] == np.float32(2.0 ** -126))
    assert np.array_equal(F.VALUES[codes[1, :3]], [0, F.e4m3(np.array(np.float64(v[1, 1]) * 2.0 ** 126)), 64])
    assert F.VALUES[codes[2, 0]] == 448 and F.VALUES[codes[2, 1]] == 0
    assert np.array_equal(F.VALUES[codes[4, :128]], F.e4m3(v[4, :128].astype(np.float64))) and scales[4, 0] == 1
    for row, block in [(5, 0), (6, 0), (7, 1)]:
        assert np.isnan(scales[row, block]) and np.all(codes[row, 128 * block: 128 * block + 128] & 127 == 127)
    fine = [0, 1, 2, 3, 4]
    F.check_rows(codes[fine], scales[fine].astype(np.float64), v[fine].astype(np.float64), np.zeros((5, 256)))
    assert F.VALUES[codes[5, 130]] == 448 and F.VALUES[codes[6, 200]] == 448 and np.all(codes[7, :128] == 0)


def silu_mul(g, u):
    """(values, bound): exp to 2 + 1.2 |g| units of its last place (twice U), a sum, a quotient and two products of half a unit each."""
    v = g / (1 + np.exp(-g)) * u
    return v, np.abs(v) * ((2 + 1.2 * np.abs(g)) * 2 + 6) * F.U + 1e-37


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,n", SHAPES)
def test_silu_mul(dev, kind, rows, n):
    rng = np.random.default_rng(rows + n)
    a, x = F.held(kind, 2 * rng.standard_normal((rows, 2 * n)))
    v, dv = silu_mul(x[:, :n], x[:, n:])
    both = dev.silu_mul_f8(upload(dev, a))
    assert both.shape == (rows, n)
    F.check_rows(both.codes.as_slice()[:, :n], both.scales.as_slice().astype(np.float64), v, dv)
    apart = dev.silu_mul_f8(upload(dev, a[:, :n]), upload(dev, a[:, n:]))
    assert np.array_equal(apart.codes.as_slice()[:, :n], both.codes.as_slice()[:, :n])
    assert np.array_equal(apart.scales.as_slice(), both.scales.as_slice())


def test_silu_mul_strided(dev):
    """Gate and up in rows of their own lengths, at addresses that allow no wide loads; with n = 1 too."""
    rng = np.random.default_rng(17)
    for kind, n in [("f32", 1000), ("f16", 515), ("bf16", 1), ("bf16", 2048)]:
        rows, ldg, ldu = 5, n + 3, n + 16
        (ag, g), (au, u) = F.held(kind, rng.standard_normal((rows + 1, ldg))), F.held(kind, rng.standard_normal((rows + 1, ldu)))
        tg, tu = upload(dev, ag), upload(dev, au)
        codes, scales, ld = new_rows(dev, rows, n, 1)
        dev._check(dev.lib.fb200_silu_mul_f8(dev.h, tg.ptr + ag.itemsize, ldg, tu.ptr + 8 * au.itemsize, ldu, TYPES[kind], rows, n, codes.ptr, ld, scales.ptr))
        at = np.arange(rows)[:, None]
        v, dv = silu_mul(g.reshape(-1)[1 + at * ldg + np.arange(n)], u.reshape(-1)[8 + at * ldu + np.arange(n)])
        F.check_rows(*result(codes, scales, rows, n), v, dv)


def test_silu_mul_far_gates(dev):
    g = np.array([[-1e30, -200, -104, -88.5, -60, -20, 0, 20, 60, 88.5, 200, 1e30]], dtype=np.float32)
    u = np.array([[1, 1, 1, -1, 1, 1, 1, 1, 1, -1, 1, 1e-28]], dtype=np.float32)
    out = dev.silu_mul_f8(dev.tensor(g), dev.tensor(u))
    g64 = g.astype(np.float64)
    v = g64 / (1 + np.exp(np.minimum(-g64, 700))) * u
    F.check_rows(out.codes.as_slice()[:, :12], out.scales.as_slice().astype(np.float64), v, np.abs(v) * 2 ** -16 + 1e-34)
    bad = dev.silu_mul_f8(dev.tensor(np.array([[np.nan, 1, -np.inf]], dtype=np.float32)), dev.tensor(np.ones((1, 3), dtype=np.float32)))
    assert np.isnan(bad.scales.as_slice()).all() and np.all(bad.codes.as_slice()[:, :3] & 127 == 127)


def rms_norm(x, res, w, b, eps, chain):
    """(sum, values, bound): the sum is rounded once; of the mean of squares at most `chain` additions in a row, a quotient and eps, halved
    by the root, which is rounded once like its inverse and both products."""
    s = x + res if res is not None else x
    v = s / np.sqrt((s * s).mean(-1, keepdims=True) + eps) * w
    dv = np.abs(v) * ((chain + 4) / 2 + 5) * F.U
    if b is not None:
        v = v + b
        dv = dv + np.abs(v) * F.U
    return s, v, dv


NORMS = [(1, 1), (2, 100), (3, 128), (5, 719), (1, 4096), (70, 2048), (2, 8192), (4, 5000), (1, 16384), (2, 16500), (1, 32768), (400, 640)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,n", NORMS)
def test_rms_norm(dev, kind, rows, n):
    rng = np.random.default_rng(rows * 3 + n)
    (ax, x), (ar, r) = F.held(kind, spread(rng, rows, n)), F.held(kind, spread(rng, rows, n, 0.7))
    w, b = (1 + 0.1 * rng.standard_normal(n)).astype(np.float32), (0.3 * rng.standard_normal(n)).astype(np.float32)
    for res, bias, want in [(True, False, True), (False, False, False), (True, True, False), (False, True, True)]:
        total = dev.empty((rows, n), ax.dtype) if want else None
        out = dev.rms_norm_f8(upload(dev, ax), dev.tensor(w), EPS, residual=upload(dev, ar) if res else None,
                              bias=dev.tensor(b) if bias else None, sum_out=total)
        # 32 values a thread, 5 shuffles, at most 32 warps
        s, v, dv = rms_norm(x, r if res else None, w.astype(np.float64), b.astype(np.float64) if bias else None, EPS, 32 + 5 + 32)
        F.check_rows(out.codes.as_slice()[:, :n], out.scales.as_slice().astype(np.float64), v, dv)
        if want:
            assert np.all(np.abs(F.read(kind, total.as_slice()) - s) <= np.abs(s) * (F.HALF_STEP[kind] + 1.01 * F.U))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n", [4096, 1003])
def test_rms_norm_in_place(dev, kind, n):
    """The sum takes the place of x or of the residual, as a stream is kept."""
    rng = np.random.default_rng(n)
    (ax, _), (ar, _) = F.held(kind, rng.standard_normal((6, n))), F.held(kind, rng.standard_normal((6, n)))
    w = dev.tensor(np.ones(n, dtype=np.float32))
    total = dev.empty((6, n), ax.dtype)
    want = dev.rms_norm_f8(upload(dev, ax), w, EPS, residual=upload(dev, ar), sum_out=total)
    for first in (True, False):
        x, r = upload(dev, ax), upload(dev, ar)
        place = x if first else r
        out = dev.rms_norm_f8(x, w, EPS, residual=r, sum_out=place)
        assert np.array_equal(place.as_slice(), total.as_slice())
        assert np.array_equal(out.codes.as_slice()[:, :n], want.codes.as_slice()[:, :n]) and np.array_equal(out.scales.as_slice(), want.scales.as_slice())


@pytest.mark.parametrize("kind", TYPES)
def test_rms_norm_strided(dev, kind):
    """Rows inside longer ones, at addresses that allow no wide loads."""
    rng = np.random.default_rng(8)
    rows, n = 5, 777
    lds = (n + 3, n + 8, n + 1)
    (ax, x), (ar, r) = F.held(kind, rng.standard_normal((rows + 1, lds[0]))), F.held(kind, rng.standard_normal((rows + 1, lds[1])))
    w = rng.standard_normal(n + 1).astype(np.float32)
    tx, tr, tw, total = upload(dev, ax), upload(dev, ar), dev.tensor(w), dev.empty((rows + 1, lds[2]), ax.dtype)
    total.fill_bytes(GUARD)
    codes, scales, ld = new_rows(dev, rows, n, 1)
    dev._check(dev.lib.fb200_rms_norm_f8(dev.h, tx.ptr + ax.itemsize, lds[0], tr.ptr, lds[1], total.ptr, lds[2], TYPES[kind], tw.ptr + 4, None, EPS, rows,
                                         n, codes.ptr, ld, scales.ptr))
    x = x.reshape(-1)[1 + np.arange(rows)[:, None] * lds[0] + np.arange(n)]
    s, v, dv = rms_norm(x, r[:rows, :n], w[1:].astype(np.float64), None, EPS, 69)
    F.check_rows(*result(codes, scales, rows, n), v, dv)
    t = total.as_slice()
    assert np.all(np.abs(F.read(kind, t[:rows, :n]) - s) <= np.abs(s) * (F.HALF_STEP[kind] + 1.01 * F.U))
    assert np.all(t[:rows, n:].copy().view(np.uint8) == GUARD) and np.all(t[rows:].copy().view(np.uint8) == GUARD)


def test_rms_norm_of_zero_and_not_finite_rows(dev):
    x = np.random.default_rng(3).standard_normal((4, 512)).astype(np.float32)
    x[1], x[2, 17], x[3, 400] = 0, np.inf, np.nan
    out = dev.rms_norm_f8(dev.tensor(x), dev.tensor(np.ones(512, dtype=np.float32)), EPS)
    codes, scales = out.codes.as_slice(), out.scales.as_slice()
    s, v, dv = rms_norm(x[:1].astype(np.float64), None, 1.0, None, EPS, 69)
    F.check_rows(codes[:1], scales[:1].astype(np.float64), v, dv)
    assert np.all(codes[1] == 0) and np.all(scales[1] == np.float32(2.0 ** -126))
    # an infinity: the others are x / inf = 0, its own block inf / inf; a NaN reaches the whole row
    assert np.isnan(scales[2, 0]) and np.all(codes[2, 128:] & 127 == 0) and np.isnan(scales[3]).all() and np.all(codes[3] & 127 == 127)


# ---- the product --------------------------------------------------------------------------------------------------------

TILES = ["16,1", "16,2", "16,4", "16,8", "32,1", "32,4", "32,8", "64,1", "64,2", "64,4", "128,1", "128,2", "128,4", "pair,128", "pair,192", "pair,256"]


def operands(rng, m, n, k):
    x, xs = F.quantise(spread(rng, m, k))
    w, ws = F.quantise(rng.standard_normal((n, k)) * np.exp(rng.standard_normal((n, 1))) * 0.05, 128)
    return x, xs, w, ws


def padded(a, ld, fill=0x7F):
    """Rows ld bytes apart; the bytes between them are NaN codes, which nothing may read."""
    out = np.full((a.shape[0], ld), fill, dtype=np.uint8)
    out[:, : a.shape[1]] = a
    return out


def device_rows(dev, x, xs, extra=0):
    ld = -(-x.shape[1] // 16) * 16 + 16 * extra
    return kb.F8Rows(dev, x.shape, dev.tensor(padded(x, ld)), dev.tensor(xs))


def check(kind, got, y, bound):
    y0 = F.read(kind, got)
    assert np.all(np.abs(y0 - y) <= bound * (1 + F.HALF_STEP[kind]) + np.abs(y) * F.HALF_STEP[kind]), np.max(np.abs(y0 - y) / (np.abs(y) + bound))


def run_product(dev, rng, m, n, k, kind="f32", epilogue=kb.EPI_NONE, second=False):
    x, xs, w, ws = operands(rng, m, n, k)
    y, bound = F.product(x, xs, w, ws)
    r1 = r2 = None
    if epilogue == kb.EPI_RESIDUAL:
        r1 = rng.standard_normal((m, n)).astype(np.float32)
        r2 = rng.standard_normal((m, n)).astype(np.float32) if second else None
    if epilogue == kb.EPI_BIAS:
        r1 = rng.standard_normal(n).astype(np.float32)
    for r in (r1, r2):
        if r is not None:
            bound = bound + F.U * (np.abs(y) + bound + np.abs(r))
            y = y + r
    mat = kb.F8Matrix.from_raw_bytes(dev, (n, k), w, ws)
    out = dev.empty((m + 1, n), {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[kind])
    out.fill_bytes(GUARD)
    device_rows(dev, x, xs, 1).f8_mat_mul(mat, TYPES[kind], epilogue, dev.tensor(r1) if r1 is not None else None,
                                          dev.tensor(r2) if r2 is not None else None, out)
    got = out.as_slice()
    assert np.all(got[m:].copy().view(np.uint8) == GUARD)
    check(kind, got[:m], y, bound)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("m,n,k", [(1, 128, 128), (1, 1, 1), (3, 130, 129), (16, 256, 1024), (17, 300, 2300), (129, 257, 640), (300, 515, 1111)])
def test_product_tiles(dev, monkeypatch, tile, m, n, k):
    monkeypatch.setenv("FB200_F8_TILE", tile)
    run_product(dev, np.random.default_rng(m + n + k), m, n, k)


@pytest.mark.parametrize("m,n,k", [(300, 256 * 40, 300), (300, 256 * 40 - 77, 1000), (256, 256 * 75, 128), (513, 256 * 50 + 3, 130), (256, 256 * 111, 900)])
def test_product_several_tiles_per_pair(dev, monkeypatch, m, n, k):
    """More tiles than pairs, so that a pair goes from tile to tile (148 SMs: 80, 80, 75, 153 and 111 tiles of 256 x 256 on 74 pairs)."""
    for tile in ("pair,256", "pair,192", "pair,128"):
        monkeypatch.setenv("FB200_F8_TILE", tile)
        run_product(dev, np.random.default_rng(n), m, n, k, "bf16")
    run_product(dev, np.random.default_rng(n), m, n, k, "f32", kb.EPI_BIAS)


@pytest.mark.parametrize("m", [1, 2, 8, 13, 16, 17, 32, 33, 64, 65, 128, 129, 200, 256, 257, 700])
@pytest.mark.parametrize("n,k", [(384, 512), (1000, 3000)])
def test_product_rows(dev, m, n, k):
    run_product(dev, np.random.default_rng(m * n + k), m, n, k)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("epilogue,second", [(kb.EPI_NONE, False), (kb.EPI_RESIDUAL, False), (kb.EPI_RESIDUAL, True), (kb.EPI_BIAS, False)])
@pytest.mark.parametrize("tile,m", [("16,2", 5), ("64,1", 60), ("128,4", 300), ("pair,128", 300), ("pair,192", 300), ("pair,256", 300)])
@pytest.mark.parametrize("n", [260, 333])
def test_product_epilogues(dev, monkeypatch, kind, epilogue, second, tile, m, n):
    monkeypatch.setenv("FB200_F8_TILE", tile)
    run_product(dev, np.random.default_rng(n + m), m, n, 400, kind, epilogue, second)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (12, 4096, 14336), (1, 28672, 4096), (100, 6144, 4096), (1024, 1024, 2048), (5, 300, 70000),
                                   (2100, 2700, 700)])
def test_product_model_sizes(dev, m, n, k):
    run_product(dev, np.random.default_rng(k), m, n, k, "bf16", kb.EPI_RESIDUAL)


@pytest.mark.parametrize("tile,m", [("16,4", 9), ("64,2", 50), ("128,2", 260), ("pair,128", 260), ("pair,192", 260), ("pair,256", 260)])
def test_product_is_repeatable(dev, monkeypatch, tile, m):
    monkeypatch.setenv("FB200_F8_TILE", tile)
    x, xs, w, ws = operands(np.random.default_rng(m), m, 1300, 2000)
    mat, rows = kb.F8Matrix.from_raw_bytes(dev, (1300, 2000), w, ws), device_rows(dev, x, xs)
    first = rows.f8_mat_mul(mat).as_slice()
    for _ in range(3):
        assert np.array_equal(rows.f8_mat_mul(mat).as_slice(), first)


@pytest.mark.parametrize("tile,m", [("16,2", 9), ("128,2", 260), ("pair,128", 260), ("pair,192", 260), ("pair,256", 260)])
def test_product_keeps_what_is_not_finite_in_its_row_and_column(dev, monkeypatch, tile, m):
    monkeypatch.setenv("FB200_F8_TILE", tile)
    x, xs, w, ws = operands(np.random.default_rng(m), m, 400, 600)
    x[4, 599], w[133, 2] = 0x7F, 0xFF
    xs[7, 1], ws[2, 3] = np.inf, np.nan
    clean, bound = F.product(np.where(x & 127 == 127, 0, x), np.where(np.isfinite(xs), xs, 0), np.where(w & 127 == 127, 0, w), np.where(np.isfinite(ws), ws, 0))
    got = device_rows(dev, x, xs).f8_mat_mul(kb.F8Matrix.from_raw_bytes(dev, (400, 600), w, ws)).as_slice()
    bad = np.zeros((m, 400), dtype=bool)
    bad[4], bad[:, 133], bad[7], bad[:, 256:384] = True, True, True, True
    assert not np.isfinite(got[bad]).any() and np.all(np.abs(got - clean)[~bad] <= bound[~bad])


def test_product_over_borrowed_codes_and_into_its_residual(dev):
    """Weights in device memory, rows further apart than they are long; y takes the place of r1 (f32)."""
    rng = np.random.default_rng(5)
    for m in (3, 300):
        x, xs, w, ws = operands(rng, m, 200, 520)
        y, bound = F.product(x, xs, w, ws)
        mat = kb.F8Matrix.from_tensors(dev.tensor(padded(w, 560)), dev.tensor(ws), 520)
        r = rng.standard_normal((m, 200)).astype(np.float32)
        stream = dev.tensor(r)
        device_rows(dev, x, xs, 3).f8_mat_mul(mat, epilogue=kb.EPI_RESIDUAL, r1=stream, out=stream)
        check("f32", stream.as_slice(), y + r, bound + F.U * (np.abs(y) + bound + np.abs(r)))


@pytest.mark.parametrize("tile,m", [("16,1", 40), ("32,4", 45), ("64,1", 75), ("128,1", 155), ("128,4", 155), ("pair,128", 301), ("pair,192", 301), ("pair,256", 301)])
@pytest.mark.parametrize("n", [516, 389])
@pytest.mark.parametrize("second", [False, True])
def test_product_into_either_residual(dev, monkeypatch, tile, m, n, second):
    """y takes the place of r1 or of r2 while both are added: every residual is read before its place is written."""
    monkeypatch.setenv("FB200_F8_TILE", tile)
    rng = np.random.default_rng(n + m)
    x, xs, w, ws = operands(rng, m, n, 700)
    y, bound = F.product(x, xs, w, ws)
    a, b = (rng.standard_normal((m, n)).astype(np.float32) for _ in range(2))
    for r in (a, b):
        bound = bound + F.U * (np.abs(y) + bound + np.abs(r))
        y = y + r
    r1, r2 = dev.tensor(a), dev.tensor(b)
    out = r2 if second else r1
    device_rows(dev, x, xs).f8_mat_mul(kb.F8Matrix.from_raw_bytes(dev, (n, 700), w, ws), epilogue=kb.EPI_RESIDUAL, r1=r1, r2=r2, out=out)
    check("f32", out.as_slice(), y, bound)
    assert np.array_equal((r1 if second else r2).as_slice(), a if second else b)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("tile,m", [("16,2", 9), ("64,2", 40), ("128,1", 140), ("pair,192", 300), ("pair,256", 300)])
def test_product_into_unaligned_rows(dev, monkeypatch, kind, tile, m):
    """Outputs and residuals one element behind an aligned address, in a width that would allow wide stores."""
    monkeypatch.setenv("FB200_F8_TILE", tile)
    rng = np.random.default_rng(m)
    n, k = 256, 384
    x, xs, w, ws = operands(rng, m, n, k)
    y, bound = F.product(x, xs, w, ws)
    r = rng.standard_normal(m * n + 1).astype(np.float32)
    size = 4 if kind == "f32" else 2
    out, t, rows = dev.empty((m * n + 2,), {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[kind]), dev.tensor(r), device_rows(dev, x, xs)
    mat = kb.F8Matrix.from_raw_bytes(dev, (n, k), w, ws)
    for res in (False, True):
        out.fill_bytes(GUARD)
        ep = kb._Epilogue(kb.EPI_RESIDUAL, t.ptr + 4, None)
        dev._check(dev.lib.fb200_f8_mat_mul(dev.h, rows.codes.ptr, rows.ld, rows.scales.ptr, m, mat.h, TYPES[kind], out.ptr + size, C.byref(ep) if res else None))
        got = out.as_slice()
        assert np.all(got[[0, -1]].view(np.uint8) == GUARD)
        add = r[1:].reshape(m, n).astype(np.float64) if res else 0.0
        check(kind, got[1:-1].reshape(m, n), y + add, bound + F.U * (np.abs(y) + bound + np.abs(add)))


def test_no_rows(dev):
    mat = kb.F8Matrix.from_raw_bytes(dev, (8, 16), np.zeros((8, 16), dtype=np.uint8), np.zeros((1, 1), dtype=np.float32))
    none = dev.quantize_f8(dev.empty((0, 16)))
    assert none.codes.as_slice().shape == (0, 16) and none.f8_mat_mul(mat).as_slice().shape == (0, 8)
    assert dev.silu_mul_f8(dev.empty((0, 32))).shape == (0, 16)
    assert dev.rms_norm_f8(dev.empty((0, 16)), dev.tensor(np.ones(16, dtype=np.float32)), EPS).shape == (0, 16)


def test_refusals(dev):
    L, h, out = dev.lib, dev.h, C.c_void_p()
    t = dev.empty((64, 256))
    c, s, p = dev.empty((64, 256), np.uint8), dev.empty((64, 2)), t.ptr

    def says(code, rc):
        assert rc == code and (code == kb.OK or len(L.fb200_last_error(h)) > 10)

    shape, dtype, arg = kb.ERR_INVALID_SHAPE, kb.ERR_UNSUPPORTED_DTYPE, kb.ERR_INVALID_ARGUMENT

    def q(x=p, ldx=256, kind=kb.F32, rows=64, n=256, codes=c.ptr, ld=256, scales=s.ptr):
        return L.fb200_quantize_f8(h, x, ldx, kind, rows, n, codes, ld, scales)

    says(kb.OK, q())
    for code, change in [(arg, dict(x=None)), (arg, dict(codes=None)), (arg, dict(scales=None)), (dtype, dict(kind=kb.Q8_0)), (shape, dict(ldx=255)),
                         (shape, dict(ld=240)), (shape, dict(n=250, ld=250)), (shape, dict(codes=c.ptr + 8)), (shape, dict(scales=s.ptr + 2)),
                         (shape, dict(x=p + 2)), (shape, dict(x=p + 1, kind=kb.F16)), (shape, dict(rows=2 ** 31)),
                         (shape, dict(n=2 ** 27 + 1, ldx=2 ** 28, ld=2 ** 28))]:
        says(code, q(**change))

    def g(gate=p, ldg=256, up=p + 512, ldu=256, kind=kb.F32, n=128, codes=c.ptr, ld=128):
        return L.fb200_silu_mul_f8(h, gate, ldg, up, ldu, kind, 64, n, codes, ld, s.ptr)

    says(kb.OK, g())
    for code, change in [(arg, dict(gate=None)), (arg, dict(up=None)), (dtype, dict(kind=99)), (shape, dict(ldg=100)), (shape, dict(ldu=100)), (shape, dict(ld=112))]:
        says(code, g(**change))

    def r(x=p, res=None, ldr=256, total=None, lds=256, w=p, b=None, n=256, ldx=256, ld=256, rows=4):
        return L.fb200_rms_norm_f8(h, x, ldx, res, ldr, total, lds, kb.F32, w, b, EPS, rows, n, c.ptr, ld, s.ptr)

    says(kb.OK, r())
    for code, change in [(arg, dict(x=None)), (arg, dict(w=None)), (arg, dict(w=p + 1)), (arg, dict(b=p + 2)), (shape, dict(res=p, ldr=10)),
                         (shape, dict(total=p + 1)), (shape, dict(total=p, lds=255)), (shape, dict(n=32769, ldx=40000, ld=40000))]:
        says(code, r(**change))

    def m(codes=c.ptr, ldw=256, scales=s.ptr, dims=(64, 256), rank=2):
        rc = L.fb200_f8matrix_from_device(h, (C.c_uint64 * 2)(*dims), rank, codes, ldw, scales, C.byref(out))
        return rc

    for code, change in [(arg, dict(codes=None)), (arg, dict(scales=None)), (shape, dict(ldw=240)), (shape, dict(ldw=264)), (shape, dict(codes=c.ptr + 4)),
                         (shape, dict(dims=(0, 256))), (shape, dict(dims=(64, 0))), (shape, dict(rank=3)), (shape, dict(dims=(2 ** 27 + 1, 16)))]:
        says(code, m(**change))
        assert not out.value
    b, f = np.zeros(64 * 256, dtype=np.uint8), np.zeros(4, dtype=np.float32)
    dims = (C.c_uint64 * 2)(64, 256)
    for code, nb, ns in [(shape, 64 * 256 - 1, 2), (shape, 64 * 256, 1), (shape, 64 * 256, 4)]:
        says(code, L.fb200_f8matrix_from_raw_bytes(h, dims, 2, b.ctypes.data, nb, f.ctypes.data, ns, C.byref(out)))
    says(arg, L.fb200_f8matrix_from_raw_bytes(h, dims, 2, b.ctypes.data, 64 * 256, None, 2, C.byref(out)))
    w = kb.F8Matrix.from_raw_bytes(dev, (64, 256), b, f[:2])

    def y(codes=c.ptr, ld=256, scales=s.ptr, rows=4, mat=w.h, kind=kb.F32, dst=p, epi=None):
        return L.fb200_f8_mat_mul(h, codes, ld, scales, rows, mat, kind, dst, C.byref(epi) if epi else None)

    says(kb.OK, y())
    for code, change in [(arg, dict(codes=None)), (arg, dict(scales=None)), (arg, dict(mat=None)), (arg, dict(dst=None)), (dtype, dict(kind=kb.Q4_0)),
                         (shape, dict(ld=240)), (shape, dict(ld=260)), (shape, dict(codes=c.ptr + 8)), (shape, dict(dst=p + 2)), (shape, dict(rows=2 ** 28)),
                         (arg, dict(epi=kb._Epilogue(7, p, None))), (dtype, dict(epi=kb._Epilogue(kb.EPI_SWIGLU, None, None))),
                         (arg, dict(epi=kb._Epilogue(kb.EPI_RESIDUAL, None, None))), (arg, dict(epi=kb._Epilogue(kb.EPI_BIAS, p, p))),
                         (arg, dict(epi=kb._Epilogue(kb.EPI_BIAS, p + 2, None)))]:
        says(code, y(**change))
    other = kb.Device(0)
    assert other.lib.fb200_f8_mat_mul(other.h, c.ptr, 256, s.ptr, 4, w.h, kb.F32, p, None) == kb.ERR_DEVICE_MISMATCH
    other.close()
    assert dev.status() == 0


# ---- far rows -----------------------------------------------------------------------------------------------------------

def _part(t, byte, shape, kind):
    return kb.Tensor(t.device, shape, kind, ptr=t.ptr + byte)


def _put(t, byte, a):
    a = np.ascontiguousarray(a)
    t.device._check(t.device.lib.fb200_upload(t.device.h, t.ptr + byte, a.ctypes.data, a.nbytes))


def test_rows_behind_two_to_the_32(dev):
    """Rows whose elements, and bytes, lie further than 32 bits from the first: codes of bf16 rows, norms in place, outputs of a product."""
    rng = np.random.default_rng(31)
    rows, n = 270000, 16384
    look = [0, 131071, 131072, 262143, 262144, rows - 1]  # around 2^31 and 2^32 elements
    a, v = F.held("bf16", spread(rng, len(look), n))
    x, codes, scales = dev.empty((rows, n), np.uint16), dev.empty((rows, n), np.uint8), dev.empty((rows, n // 128))
    w = dev.tensor(np.ones(n, dtype=np.float32))

    def write():
        x.fill_bytes(0)
        for i, r in enumerate(look):
            _put(x, r * n * 2, a[i])

    def read():
        c = np.stack([_part(codes, r * n, (n,), np.uint8).as_slice() for r in look])
        return c, np.stack([_part(scales, r * (n // 128) * 4, (n // 128,), np.float32).as_slice() for r in look]).astype(np.float64)

    write()
    out = kb.F8Rows(dev, (rows, n), codes, scales)
    dev.quantize_f8(x, out=out)
    F.check_rows(*read(), v, np.zeros_like(v))
    dev.rms_norm_f8(x, w, EPS, residual=x, sum_out=x, out=out)
    s, y, dy = rms_norm(v, v, 1.0, None, EPS, 69)
    F.check_rows(*read(), y, dy)
    got = np.stack([F.bf16(_part(x, r * n * 2, (n,), np.uint16).as_slice()) for r in look])
    assert np.array_equal(got, s)  # twice a bf16 value
    del x, codes, scales, out

    m, n, k = 160000, 28000, 130
    look = [0, 76695, 76696, 153390, 153391, m - 1]  # around 2^31 and 2^32 outputs
    cx, sx, cw, sw = operands(rng, len(look), n, k)
    all_codes, all_scales = dev.empty((m, 144), np.uint8), dev.empty((m, 2))
    all_codes.fill_bytes(0)
    all_scales.fill_bytes(0)
    for i, r in enumerate(look):
        _put(all_codes, r * 144, cx[i])
        _put(all_scales, r * 8, sx[i])
    y = kb.F8Rows(dev, (m, k), all_codes, all_scales).f8_mat_mul(kb.F8Matrix.from_raw_bytes(dev, (n, k), cw, sw), kb.BF16)
    want, bound = F.product(cx, sx, cw, sw)
    check("bf16", np.stack([_part(y, r * n * 2, (n,), np.uint16).as_slice() for r in look]), want, bound)
    assert not _part(y, 76697 * n * 2, (n,), np.uint16).as_slice().any() and not _part(y, 153392 * n * 2, (n,), np.uint16).as_slice().any()


# ---- together -----------------------------------------------------------------------------------------------------------

class Layer:
    """A feed-forward: norm with the stream's update, the stacked gate and up product, their gated rows, down into the stream."""

    def __init__(self, dev, rng, width, ffn):
        self.dev, self.width, self.ffn = dev, width, ffn
        self.norm = (1 + 0.1 * rng.standard_normal(width)).astype(np.float32)
        self.up, self.ups = F.quantise(rng.standard_normal((2 * ffn, width)) * width ** -0.5, 128)
        self.down, self.downs = F.quantise(rng.standard_normal((width, ffn)) * ffn ** -0.5, 128)
        self.w_norm = dev.tensor(self.norm)
        self.w_up = kb.F8Matrix.from_raw_bytes(dev, self.up.shape, self.up, self.ups)
        self.w_down = kb.F8Matrix.from_raw_bytes(dev, self.down.shape, self.down, self.downs)

    def buffers(self, m):
        d = self.dev
        return dict(h=kb.F8Rows(d, (m, self.width)), gu=d.empty((m, 2 * self.ffn), np.uint16), z=kb.F8Rows(d, (m, self.ffn)))

    def run(self, stream, delta, b):
        """stream <- stream + delta, then + the feed-forward of its norm."""
        self.dev.rms_norm_f8(stream, self.w_norm, EPS, residual=delta, sum_out=stream, out=b["h"])
        b["h"].f8_mat_mul(self.w_up, kb.BF16, out=b["gu"])
        self.dev.silu_mul_f8(b["gu"], out=b["z"])
        b["z"].f8_mat_mul(self.w_down, epilogue=kb.EPI_RESIDUAL, r1=stream, out=stream)

    def check(self, stream0, delta, b, stream1):
        """Every step against the definition on what the step before it left."""
        n, f = self.width, self.ffn
        s, v, dv = rms_norm(stream0.astype(np.float64), delta.astype(np.float64), self.norm.astype(np.float64), None, EPS, 69)
        h, hs = b["h"].codes.as_slice()[:, :n], b["h"].scales.as_slice()
        F.check_rows(h, hs.astype(np.float64), v, dv)
        y, bound = F.product(h, hs, self.up, self.ups)
        check("bf16", b["gu"].as_slice(), y, bound)
        gu = F.read("bf16", b["gu"].as_slice())
        z, zs = b["z"].codes.as_slice()[:, :f], b["z"].scales.as_slice()
        F.check_rows(z, zs.astype(np.float64), *silu_mul(gu[:, :f], gu[:, f:]))
        y, bound = F.product(z, zs, self.down, self.downs)
        check("f32", stream1, y + s, bound + 2 * F.U * (np.abs(y) + bound + np.abs(s)))


@pytest.mark.parametrize("m,width,ffn", [(1, 1024, 2048), (7, 640, 1000), (150, 1024, 1500), (600, 512, 1280)])
def test_feed_forward(dev, m, width, ffn):
    rng = np.random.default_rng(m)
    layer = Layer(dev, rng, width, ffn)
    x, d = spread(rng, m, width).astype(np.float32), rng.standard_normal((m, width)).astype(np.float32)
    stream, b = dev.tensor(x), layer.buffers(m)
    layer.run(stream, dev.tensor(d), b)
    layer.check(x, d, b, stream.as_slice())
    assert dev.status() == 0


def test_feed_forward_in_a_graph():
    """A captured pass, replayed on other inputs, and a second graph of the same layer between its replays."""
    torch = pytest.importorskip("torch")
    side = torch.cuda.Stream()
    d = kb.Device(0, stream=side.cuda_stream)
    rng = np.random.default_rng(12)
    layer = Layer(d, rng, 512, 1024)
    graphs = []
    for m in (2, 140):
        b, stream, delta = layer.buffers(m), d.empty((m, 512)), d.empty((m, 512))
        stream.fill_bytes(0)
        delta.fill_bytes(0)
        layer.run(stream, delta, b)  # a kernel's first launch sets it up, which a capture may not
        d.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            layer.run(stream, delta, b)
        graphs.append((g, b, stream, delta, m))
    for g, b, stream, delta, m in graphs + graphs[::-1]:
        x, e = spread(rng, m, 512).astype(np.float32), rng.standard_normal((m, 512)).astype(np.float32)
        for t, a in ((stream, x), (delta, e)):
            d._check(d.lib.fb200_upload(d.h, t.ptr, a.ctypes.data, a.nbytes))
        with torch.cuda.stream(side):
            g.replay()
        d.synchronize()
        layer.check(x, e, b, stream.as_slice())
    del graphs, g


def test_two_handles_at_once(dev):
    """The same layer on two streams, passes in flight on both."""
    other = kb.Device(0)
    rng = np.random.default_rng(21)
    sets = []
    for d in (dev, other):
        layer = Layer(d, np.random.default_rng(4), 768, 1536)
        for m in (3, 200):
            x, e = spread(rng, m, 768).astype(np.float32), rng.standard_normal((m, 768)).astype(np.float32)
            sets.append((layer, x, e, d.tensor(x), d.tensor(e), layer.buffers(m)))
    dev.synchronize()
    other.synchronize()
    for layer, x, e, stream, delta, b in sets:
        layer.run(stream, delta, b)
    for layer, x, e, stream, delta, b in sets:
        layer.check(x, e, b, stream.as_slice())
    assert other.status() == 0
    del sets, layer, stream, delta, b  # before their handle
    other.close()
