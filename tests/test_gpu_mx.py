"""Microscaled feature rows (csrc/mx.hip) against their definition in float64: quantisation and decoding bit for bit, the
root-mean-square norm and the product within bounds that are derived where they stand."""
import itertools
import math
import os

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

EMAX = {"e2m1": 2, "e4m3": 8}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}       # half a step, relative to the value


@pytest.fixture(scope="module")
def bts():
    import importlib
    return importlib.import_module("bot-sort-onnx-tensorrt_amd")


# ------------------------------------------------------------------------------------------------------- definition, float64

def grid(fmt):
    """non-negative values in the order of their codes"""
    if fmt == "e2m1":
        return np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    return np.array([(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])


def wide(d):
    return (d + 127) // 128 * 128


def blocks(v, d):
    out = np.zeros((v.shape[0], wide(d)))
    out[:, :d] = v
    return out.reshape(v.shape[0], -1, 32)


def quantize_ref(v, fmt):
    """float64 [n, d] -> (codes [n, wide] one per element, scales [n, wide / 32])"""
    b = blocks(v, v.shape[1])
    bad = ~np.isfinite(b).all(-1)
    top = np.where(bad, 0, np.abs(b).max(-1))
    e = np.where(top > 0, np.frexp(top)[1] - 1, -1000) - EMAX[fmt]
    s = np.where(bad, 255, np.clip(e, -127, 127) + 127)
    x = np.where(bad[..., None], 0, b) / np.exp2(np.where(bad, 0, s - 127.0))[..., None]
    g, a = grid(fmt), np.abs(x)
    hi = np.minimum(np.searchsorted(g, a), len(g) - 1)
    lo = np.maximum(hi - 1, 0)
    code = np.where(a - g[lo] < g[hi] - a, lo, np.where(a - g[lo] > g[hi] - a, hi, np.where(lo % 2 == 0, lo, hi)))
    code = code + np.where(np.signbit(x), 8 if fmt == "e2m1" else 128, 0)
    return code.reshape(v.shape[0], -1), s


def pack(code, fmt):
    return (code[:, 0::2] + 16 * code[:, 1::2] if fmt == "e2m1" else code).astype(np.uint8)


def unpack(codes, fmt):
    return np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1) if fmt == "e2m1" else codes


def decode_ref(codes, scales, fmt):
    """packed codes, scales -> float64 [n, wide]"""
    g = grid(fmt)
    t = np.concatenate((g, -g)) if fmt == "e2m1" else np.concatenate((g, [np.nan], -g, [np.nan]))
    s = scales.astype(np.float64)
    return t[unpack(codes, fmt)] * np.repeat(np.where(s == 255, np.nan, np.exp2(s - 127)), 32, axis=1)


def host(rows):
    return rows.codes.cpu().numpy(), rows.scales.cpu().numpy()


def rows_of(bts, v, fmt):
    """float64 values -> MxRows filled from the definition, and the values they stand for"""
    code, s = quantize_ref(v, fmt)
    c = pack(code, fmt)
    r = bts.MxRows(torch.from_numpy(c).cuda(), torch.from_numpy(s.astype(np.uint8)).cuda(), v.shape[1], fmt)
    return r, decode_ref(c, s, fmt)


# ------------------------------------------------------------------------------------------------------------- quantisation

def awkward(n, d, dtype, seed):
    """values with ties, powers of two, subnormals, zeros, huge and tiny rows, exactly representable in dtype"""
    r = np.random.default_rng(seed)
    x = r.standard_normal((n, d)) * np.exp2(r.integers(-12, 12, (n, 1)))
    kind = r.integers(0, 6, (n, d))
    x = np.where(kind == 0, r.integers(-64, 65, (n, d)) / 8.0, x)                # ties and exact values
    x = np.where(kind == 1, np.sign(x) * np.exp2(r.integers(-8, 9, (n, d))), x)
    x = np.where(kind == 2, 0.0, x)
    t = DTYPES[dtype]
    if n > 2:
        x[1] = 0.0
        x[2] *= float(torch.finfo(t).tiny) * 2.0 ** -3                             # subnormals of the type
        x[n - 1] = np.sign(x[n - 1]) * float(torch.finfo(t).max)
    return torch.from_numpy(x).to(t)


SHAPES = [(1, 1), (1, 31), (3, 32), (5, 33), (4, 127), (7, 128), (2, 129), (9, 384), (3, 1111), (33, 250), (300, 96)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("n,d", SHAPES)
def test_quantize_and_back(bts, n, d, fmt, dtype):
    x = awkward(n, d, dtype, 17 * n + d)
    code, s = quantize_ref(x.double().numpy(), fmt)
    q = bts.mx_quantize(x.cuda(), fmt)
    c, sc = host(q)
    assert np.array_equal(sc, s)
    assert np.array_equal(c, pack(code, fmt))
    want = decode_ref(c, sc, fmt)[:, :d]
    for out in DTYPES:
        got = q.dequantize(DTYPES[out]).cpu()
        # the values have at most 4 significant bits: one rounding, from float32 on (products below its range round there first)
        assert torch.equal(got, torch.from_numpy(want).float().to(DTYPES[out])), out
    assert len(q) == n and q.d == d


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_quantize_non_finite_blocks(bts, fmt):
    x = awkward(6, 200, "f32", 3)
    x[0, 5] = float("inf"); x[1, 40] = float("-inf"); x[2, 199] = float("nan"); x[3, 0] = float("nan"); x[3, 1] = float("inf"); x[5, 128:160] = float("inf")
    code, s = quantize_ref(x.double().numpy(), fmt)
    assert (s == 255).sum() == 5
    q = bts.mx_quantize(x.cuda(), fmt)
    c, sc = host(q)
    assert np.array_equal(sc, s)
    ok = np.repeat(s != 255, 32, axis=1)
    assert np.array_equal(unpack(c, fmt)[ok], code[ok]) and (unpack(c, fmt)[~ok] % (8 if fmt == "e2m1" else 128) == 0).all()
    assert np.array_equal(np.isnan(q.dequantize().cpu().numpy()), ~ok[:, :200])


@pytest.mark.parametrize("dtype,off,ld", [("f32", 0, 260), ("f32", 1, 263), ("bf16", 0, 264), ("bf16", 3, 259), ("f16", 8, 264)])
def test_quantize_strided_rows(bts, dtype, off, ld):
    """rows inside a wider matrix, aligned for wide loads or not; the matrix is left as it was"""
    n, d = 13, 250
    flat = awkward(1, off + n * ld, dtype, off + ld)[0]
    dev = flat.cuda()
    x = torch.as_strided(dev, (n, d), (ld, 1), off)
    ref = torch.as_strided(flat, (n, d), (ld, 1), off)
    q = bts.mx_quantize(x, "e4m3")
    code, s = quantize_ref(ref.double().numpy(), "e4m3")
    assert np.array_equal(host(q)[0], pack(code, "e4m3")) and np.array_equal(host(q)[1], s)
    assert torch.equal(dev.cpu().view(torch.uint8), flat.view(torch.uint8))


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_dequantize_every_code_and_scale(bts, fmt):
    per = 16 if fmt == "e2m1" else 256
    code = np.tile(np.arange(per), (256, 256 // per))
    s = np.tile(np.arange(256)[:, None], (1, 8))
    r = bts.MxRows(torch.from_numpy(pack(code, fmt)).cuda(), torch.from_numpy(s.astype(np.uint8)).cuda(), 256, fmt)
    with np.errstate(over="ignore"):
        want = decode_ref(pack(code, fmt), s, fmt).astype(np.float32)
    got = r.dequantize().cpu().numpy()
    assert np.array_equal(got, want, equal_nan=True)
    for t in (torch.float16, torch.bfloat16):
        assert torch.equal(r.dequantize(t).cpu().nan_to_num(nan=12345.0), torch.from_numpy(want).to(t).nan_to_num(nan=12345.0))


def test_rows_behind_the_last_stay(bts):
    """out rows of a larger buffer: only the rows given are written, by every operator"""
    x = awkward(5, 70, "f32", 9).cuda()
    room = bts.MxRows.empty(8, 70, "e2m1")
    room.codes.fill_(0xAB); room.scales.fill_(0xCD)
    view = bts.MxRows(room.codes[:5], room.scales[:5], 70, "e2m1")
    bts.mx_quantize(x, "e2m1", out=view)
    bts.rms_norm_mx(x, fmt="e2m1", out=view)
    assert (room.codes[5:].cpu() == 0xAB).all() and (room.scales[5:].cpu() == 0xCD).all()
    out = torch.full((8, 16), 7.0).cuda()
    bts.mx_product(view, view, out=out[:5, :5])
    o = out.cpu()
    assert (o[5:] == 7).all() and (o[:5, 5:] == 7).all() and (o[:5, :5] != 7).any()


# ------------------------------------------------------------------------------------------------------------------- norm

def norm_ref(x, residual, weight, eps):
    """(h as stored, v float64)"""
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    f = h.double().numpy()
    v = f / np.sqrt((f * f).mean(-1, keepdims=True) + eps)
    return h, v if weight is None else v * weight.double().numpy()


def norm_delta(d):
    """relative error of the float32 computation: the sum of squares is a chain of at most 8 * ceil(d / 512) fused steps per lane and 9
    more in the reduction (half of it counts, through the root), the mean's division, the root, the reciprocal and two products"""
    return (0.5 * (8 * math.ceil(d / 512) + 9) + 5) * 2.0 ** -24


def check_quantized(v, codes, scales, fmt, d, delta):
    """codes are a correct quantisation of values within `delta` of v"""
    b, s = blocks(v, d), scales.astype(np.int64)
    top = np.abs(b).max(-1)

    def byte(t):
        return np.clip(np.where(t > 0, np.frexp(t)[1] - 1, -1000) - EMAX[fmt], -127, 127) + 127
    assert ((s == byte(top * (1 - delta))) | (s == byte(top * (1 + delta)))).all()
    unit = np.exp2(s - 127.0)[..., None]
    x = np.abs(b) / unit
    mant, emin, most = (1, 0, 6.0) if fmt == "e2m1" else (3, -6, 448.0)
    e = np.maximum(np.where(x > 0, np.frexp(x)[1] - 1, -1000), emin)
    half = np.exp2(e - mant - 1.0)                                                  # half a step of the element's binade
    q = decode_ref(codes, scales, fmt).reshape(b.shape) / unit
    err = np.abs(np.abs(q) - np.minimum(x, most))
    assert (err <= half + delta * x).all(), float((err - half - delta * x).max())
    assert ((q == 0) | (np.sign(q) == np.sign(b))).all()


NORM_SHAPES = [(1, 1), (1, 2048), (3, 31), (5, 128), (2, 257), (17, 384), (4, 1111), (3, 2056), (2, 4096), (2, 8200)]


@pytest.mark.parametrize("residual,weight", [(False, False), (True, True), (True, False), (False, True)])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n,d", NORM_SHAPES)
def test_rms_norm(bts, n, d, dtype, residual, weight):
    t, r = DTYPES[dtype], np.random.default_rng(d)
    x = torch.from_numpy(r.standard_normal((n, d)) * np.exp2(r.integers(-4, 5, (n, 1)))).to(t)
    res = torch.from_numpy(r.standard_normal((n, d))).to(t) if residual else None
    w = torch.from_numpy(1 + 0.2 * r.standard_normal(d)).to(t) if weight else None
    dev = lambda a: None if a is None else a.cuda()  # noqa: E731
    for fmt in ("e4m3", "e2m1", None):
        y = torch.full((n, d), 9.0, dtype=t).cuda()
        xd, rd = x.cuda(), dev(res)
        q, h = bts.rms_norm_mx(xd, residual=rd, weight=dev(w), eps=1e-5, fmt=fmt, y_out=y)
        want_h, v = norm_ref(x, res, w, 1e-5)
        assert torch.equal(h.cpu(), want_h)
        assert torch.equal(xd.cpu(), x) and (rd is None or torch.equal(rd.cpu(), res))
        delta = norm_delta(d)
        # a value below the type's normal range is off by half of its smallest step
        tol = (delta + HALF[dtype] * (1 + delta)) * np.abs(v) + float(torch.finfo(t).smallest_normal) * HALF[dtype]
        assert (np.abs(y.cpu().double().numpy() - v) <= tol).all()
        if fmt is None:
            assert q is None
        else:
            check_quantized(v, *host(q), fmt, d, delta)


@pytest.mark.parametrize("residual,weight", [(False, False), (True, True)])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n,d", NORM_SHAPES)
def test_rms_norm_error_does_not_grow_with_the_row(bts, n, d, dtype, residual, weight):
    """as `test_rms_norm`, with the bound of what is computed: eight squares are added in float32 (a square and three additions, half of whose
    4 roundings reach the root), the rest of the row in float64; the factor, the weight's product and the factor's product are rounded
    once each -- 5 roundings whatever the row's length"""
    t, r = DTYPES[dtype], np.random.default_rng(d + 1)
    x = torch.from_numpy(r.standard_normal((n, d)) * np.exp2(r.integers(-4, 5, (n, 1)))).to(t)
    res = torch.from_numpy(r.standard_normal((n, d))).to(t) if residual else None
    w = torch.from_numpy(1 + 0.2 * r.standard_normal(d)).to(t) if weight else None
    dev = lambda a: None if a is None else a.cuda()  # noqa: E731
    delta = 5.01 * 2.0 ** -24
    for fmt in ("e4m3", "e2m1"):
        y = torch.full((n, d), 9.0, dtype=t).cuda()
        q, h = bts.rms_norm_mx(x.cuda(), residual=dev(res), weight=dev(w), eps=1e-5, fmt=fmt, y_out=y)
        want_h, v = norm_ref(x, res, w, 1e-5)
        assert torch.equal(h.cpu(), want_h)
        tol = (delta + HALF[dtype] * (1 + delta)) * np.abs(v) + float(torch.finfo(t).smallest_normal) * HALF[dtype]
        assert (np.abs(y.cpu().double().numpy() - v) <= tol).all()
        check_quantized(v, *host(q), fmt, d, delta)


@pytest.mark.parametrize("n,d", [(64, 2048), (64, 1111), (64, 8192), (64, 9000), (64, 512)])
def test_rms_norm_factor_is_rounded_once(bts, n, d):
    """whole numbers up to 511: eight squares add up exactly in float32 (below 2^21), a row's do not (around 2^26 at 1111 elements), so
    only a sum in more bits gives the factor that float64 gives, and with it every bit of y"""
    r = np.random.default_rng(d)
    x = r.integers(-511, 512, (n, d)).astype(np.float64)
    y = torch.empty((n, d)).cuda()
    bts.rms_norm_mx(torch.from_numpy(x).float().cuda(), eps=1e-6, fmt=None, y_out=y)
    factor = (1.0 / np.sqrt((x * x).sum(1) / d + 1e-6)).astype(np.float32)
    assert np.array_equal(y.cpu().numpy(), x.astype(np.float32) * factor[:, None])


@pytest.mark.parametrize("d", [96, 5000, 9000])
def test_rms_norm_in_place(bts, d):
    x = awkward(6, d, "bf16", d)
    res = awkward(6, d, "bf16", d + 1)
    x[5] = 1.0; res[5] = -1.0                                                       # (the type's largest values would pass float32's range)
    q0, h0 = bts.rms_norm_mx(x.cuda(), residual=res.cuda(), fmt="e4m3")
    for into in ("x", "residual"):
        xd, rd = x.cuda(), res.cuda()
        q, h = bts.rms_norm_mx(xd, residual=rd, fmt="e4m3", sum_out=xd if into == "x" else rd)
        assert h is (xd if into == "x" else rd) and torch.equal(h.cpu(), h0.cpu())
        assert torch.equal(q.codes.cpu(), q0.codes.cpu()) and torch.equal(q.scales.cpu(), q0.scales.cpu())
        assert torch.equal((rd if into == "x" else xd).cpu(), res if into == "x" else x)
    y0 = torch.empty_like(x).cuda()
    bts.rms_norm_mx(x.cuda(), residual=res.cuda(), fmt=None, y_out=y0)
    xd = x.cuda()
    bts.rms_norm_mx(xd, residual=res.cuda(), fmt=None, y_out=xd)                     # the normalised rows in the place of x
    assert torch.equal(xd.cpu(), y0.cpu())


@pytest.mark.parametrize("d", [96, 1500, 9000])
@pytest.mark.parametrize("fmt", ["e4m3", None])
def test_rms_norm_in_the_place_of_x_returns_the_rows_that_were_there(bts, d, fmt):
    """y in the place of x, no residual and no room for h: h is x as it was, not what was written over it"""
    x = awkward(6, d, "bf16", d)
    y0 = torch.empty_like(x).cuda()
    q0, _ = bts.rms_norm_mx(x.cuda(), fmt=fmt, y_out=y0)
    xd = x.cuda()
    q, h = bts.rms_norm_mx(xd, fmt=fmt, y_out=xd)
    assert torch.equal(h.cpu(), x) and torch.equal(xd.cpu().view(torch.int16), y0.cpu().view(torch.int16))
    assert fmt is None or (torch.equal(q.codes.cpu(), q0.codes.cpu()) and torch.equal(q.scales.cpu(), q0.scales.cpu()))
    xd, h1 = x.cuda(), torch.empty_like(x).cuda()
    assert bts.rms_norm_mx(xd, fmt=fmt, y_out=xd, sum_out=h1)[1] is h1 and torch.equal(h1.cpu(), x)


@pytest.mark.parametrize("d", [40, 1500, 9000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rms_norm_at_the_ends_of_the_range(bts, d, dtype):
    """rows whose squares, or whose products with the weight, leave float32 in either direction"""
    t, r = DTYPES[dtype], np.random.default_rng(d)
    e = np.array([127, 126, 100, 64, 62, -40, -60, -90, -110])                      # (normal values: the smallest are 2^-118)
    v = (1 + r.random((len(e), d))) * np.exp2(e[:, None] - (r.integers(0, 9, (len(e), d)) if dtype == "f32" else 0)) * r.choice([-1, 1], (len(e), d))
    x = torch.from_numpy(np.clip(v, -float(torch.finfo(t).max), float(torch.finfo(t).max))).to(t)
    w = torch.from_numpy(r.choice([0.25, 3.0, 40.0], d)).to(t)
    for eps in (1e-6, 1e-38):
        y = torch.empty_like(x).cuda()
        q, h = bts.rms_norm_mx(x.cuda(), weight=w.cuda(), eps=eps, y_out=y)
        _, want = norm_ref(x, None, w, eps)
        delta = norm_delta(d)
        tol = (delta + HALF[dtype] * (1 + delta)) * np.abs(want) + float(torch.finfo(t).smallest_normal) * HALF[dtype]
        assert (np.abs(y.cpu().double().numpy() - want) <= tol).all()
        check_quantized(want, *host(q), "e4m3", d, delta)


@pytest.mark.parametrize("d", [40, 1500, 1111, 9000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rms_norm_weights_at_the_ends_of_the_range(bts, d, dtype):
    """rows and weights whose products leave float32 although the normalised values do not, in both directions, and elements far below
    their row's norm.  The bound: half of the sum of squares' error (a square, and the three additions to eight of them, in float32:
    4 roundings), the factor's rounding, the weight's product and the factor's product -- 5 roundings, and the output's.  Below float32's
    normal range: the normalised element but for a factor in [1, 2) is held in float32, 2^-150 off, which the weight and that factor multiply;
    the product with the weight likewise, 2^-150 times that factor."""
    t, r = DTYPES[dtype], np.random.default_rng(d)
    scale = np.array([50, 100, 126, 64, 0, -40, -62, -100, -118, 20])
    x = (1 + r.random((len(scale), d))) * np.exp2(scale[:, None] * 1.0) * r.choice([-1, 1], (len(scale), d))
    x[3, ::3] *= 2.0 ** -100                                                         # 2^-36 beside 2^64
    x[2, ::2] *= 2.0 ** -180
    x[9] = 0
    x = torch.from_numpy(x).to(t)
    for power in (100, 64, 30, 0, -30, -64, -95):
        w = torch.from_numpy((1 + r.random(d)) * np.exp2(power - 1.0) * r.choice([-1, 1], d)).to(t)
        w[5] = 0
        for eps in (1e-38, 1e-6):
            y = torch.empty_like(x).cuda()
            q, _ = bts.rms_norm_mx(x.cuda(), weight=w.cuda(), eps=eps, y_out=y)
            _, want = norm_ref(x, None, w, eps)
            delta = 5.01 * 2.0 ** -24
            tiny = float(torch.finfo(t).smallest_normal)
            wide_w = np.abs(w.double().numpy())
            tol = (delta + HALF[dtype] * (1 + delta)) * np.abs(want) + tiny * HALF[dtype] + 2.0 ** -149 + 2.0 ** -149 * wide_w
            got = y.cpu().double().numpy()
            assert (np.abs(got - want) <= tol).all(), (power, eps, float((np.abs(got - want) / tol).max()))
            # (a value below float32's normal range is rounded to its smallest step before it is quantised: blocks of such are left out)
            ok = (np.abs(blocks(want, d)).max(-1) >= 2.0 ** -100) | (np.abs(blocks(want, d)).max(-1) == 0)
            code, s = host(q)
            code = code.reshape(len(x), -1, 32)
            code[~ok], s[~ok] = 0, 0
            check_quantized(np.where(ok[:, :, None], blocks(want, d), 0).reshape(len(x), -1)[:, :d], code.reshape(len(x), -1), s, "e4m3", d, delta)


# more rows than one launch's workgroups, 4 rows each up to 1024 elements
@pytest.mark.parametrize("n,d", [(4 * 2 ** 20 + 5, 8), (2 ** 20 + 3, 1032)])
def test_rms_norm_big_row_counts(bts, n, d):
    x = torch.ones((n, d), dtype=torch.float16, device="cuda")
    x[-9:] = torch.from_numpy(np.random.default_rng(n).standard_normal((9, d))).half().cuda()
    y = torch.zeros_like(x)
    bts.rms_norm_mx(x, fmt=None, y_out=y)
    assert (y[:-9] == 1).all()                                                      # 1 / sqrt(1 + 1e-6) rounds to 1
    _, v = norm_ref(x[-9:].cpu(), None, None, 1e-6)
    delta = norm_delta(d)
    assert (np.abs(y[-9:].cpu().double().numpy() - v) <= (delta + HALF["f16"] * (1 + delta)) * np.abs(v) + 2.0 ** -25).all()


def test_rms_norm_zero_and_non_finite_rows(bts):
    x = torch.ones((5, 300))
    x[1] = 0; x[2, 7] = float("inf"); x[3, 70] = float("nan")
    q, _ = bts.rms_norm_mx(x.cuda(), fmt="e4m3")
    v = q.dequantize().cpu().numpy()
    # 1 / sqrt(1 + 1e-6) = 0.9999995 is below 1: its block's exponent is -1, its unit 2^(-1 - 8), and 0.9999995 * 512 = 511.9997
    # saturates at 448: the value held is 448 / 512
    assert (v[0] == 0.875).all() and (v[4] == 0.875).all() and (v[1] == 0).all()
    assert np.isnan(v[3]).all()                                                     # a NaN takes the row's norm with it
    assert np.isnan(v[2, :32]).all() and (v[2, 32:] == 0).all()                     # inf / inf in its block, x / inf elsewhere


@pytest.mark.parametrize("power", [100, 0, -100])
def test_rms_norm_non_finite_rows_under_a_weight(bts, power):
    x = torch.ones((3, 300)) * 2.0 ** 50
    x[0, 7] = float("inf"); x[1, 70] = float("nan")
    w = torch.ones(300) * 2.0 ** power
    y = torch.empty_like(x).cuda()
    bts.rms_norm_mx(x.cuda(), weight=w.cuda(), fmt=None, y_out=y)
    y = y.cpu()
    assert y[0, 7].isnan() and (y[0, :7] == 0).all() and (y[0, 8:] == 0).all() and y[1].isnan().all()
    assert (y[2] == 2.0 ** power).all()                                              # sqrt(2^100 + 1e-6) = 2^50 in float64


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rms_norm_strided(bts, dtype):
    t = DTYPES[dtype]
    big = awkward(12, 700, dtype, 5).clamp(-100, 100)
    x, res = big[:, 3:403], big[:, 290:690]
    dev = big.cuda()
    out = torch.zeros((12, 500), dtype=t).cuda()
    q, h = bts.rms_norm_mx(dev[:, 3:403], residual=dev[:, 290:690], sum_out=out[:, 50:450], fmt="e2m1")
    want, v = norm_ref(x, res, None, 1e-6)
    assert torch.equal(out[:, 50:450].cpu(), want) and (out[:, :50].cpu() == 0).all() and (out[:, 450:].cpu() == 0).all()
    check_quantized(v, *host(q), "e2m1", 400, norm_delta(400))


# ----------------------------------------------------------------------------------------------------------------- product

def product_bound(a, b, out, ref, fmts):
    """half a step of the output's type, and the sum's own error: with two E2M1 operands products are exact and at most one float32
    rounding falls on each partial sum (instructions, parts of the row and the factor: d / 128 + 20), each at most 2^-24 of the sum
    of magnitudes; with an E4M3 operand the instruction's alignment leaves 2^-12 of that sum"""
    mag = np.abs(a) @ np.abs(b).T
    own = (a.shape[1] / 128 + 20) * 2.0 ** -24 if fmts == ("e2m1", "e2m1") else 2.0 ** -12
    return HALF[out] * np.abs(ref) + own * mag + float(torch.finfo(DTYPES[out]).smallest_normal) * HALF[out]


def feature_rows(n, d, seed):
    r = np.random.default_rng(seed)
    v = r.standard_normal((n, d)) * np.exp(0.5 * r.standard_normal(d))
    return v * np.exp2(r.integers(-3, 4, (n, 1)))


FMTS = list(itertools.product(["e2m1", "e4m3"], ["e2m1", "e4m3"]))
PRODUCTS = [(1, 1, 1), (1, 300, 64), (16, 17, 128), (17, 1, 300), (33, 65, 500), (5, 130, 1111), (64, 64, 256), (100, 37, 129)]
BIG = [(1, 5000, 2048), (3, 70001, 96), (40, 2000, 1024), (200, 333, 4100), (512, 256, 256), (777, 1300, 640), (1500, 1025, 2048), (2500, 4, 512), (33000, 40, 200),
       (9000, 20, 700), (2000, 1999, 300), (3000, 2900, 300), (4000, 4090, 300), (4096, 4096, 129)]


def run_product(bts, n, m, d, fa, fb, out):
    va, vb = feature_rows(n, d, 3 * n + d), feature_rows(m, d, 5 * m + d)
    if n > 3:
        va[2] = 0.0
    a, ra = rows_of(bts, va, fa)
    b, rb = rows_of(bts, vb, fb)
    ref = ra @ rb.T
    for alpha, floor in ((1.0, False), (0.125, True)):
        want = np.maximum(ref * alpha, 0) if floor else ref * alpha
        got = bts.mx_product(a, b, alpha=alpha, floor_zero=floor, dtype=DTYPES[out]).cpu().double().numpy()
        assert got.shape == (n, m)
        tol = product_bound(ra, rb, out, want, (fa, fb)) * (1 if alpha == 1 else alpha if out == "f32" else 1)
        assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / np.maximum(tol, 1e-300)).max())
        if n > 3:
            assert (got[2] == 0).all()


@pytest.mark.parametrize("fa,fb", FMTS)
@pytest.mark.parametrize("n,m,d", PRODUCTS)
def test_product(bts, n, m, d, fa, fb):
    for out in (["f32", "bf16"] if fa == fb == "e2m1" else ["f16", "bf16"]):
        run_product(bts, n, m, d, fa, fb, out)


# enough of them for LDS tiles of each of the small shapes
MID = [(512, 256, 256), (3, 33000, 96), (9000, 20, 100), (1030, 1030, 100)]


@pytest.mark.parametrize("fa,fb", FMTS)
@pytest.mark.parametrize("n,m,d", MID)
def test_product_tiles(bts, n, m, d, fa, fb):
    run_product(bts, n, m, d, fa, fb, "f32" if fa == fb == "e2m1" else "f16")


@pytest.mark.parametrize("fa,fb", FMTS)
@pytest.mark.parametrize("n,m,d", BIG)
def test_product_big(bts, n, m, d, fa, fb):
    run_product(bts, n, m, d, fa, fb, "f32" if fa == fb == "e2m1" else "bf16")


def random_rows(bts, n, d, fmt, seed):
    """rows of random codes (no NaN) and scales 2^-5 .. 2^5, d even -> (MxRows, their values in float64, on the device)"""
    r = np.random.default_rng(seed)
    code = r.integers(0, 256, (n, wide(d) // (2 if fmt == "e2m1" else 1)), dtype=np.uint8)
    if fmt == "e4m3":
        code[code % 128 == 127] = 1
    code[:, d // (2 if fmt == "e2m1" else 1):] = 0
    s = r.integers(122, 133, (n, wide(d) // 32), dtype=np.uint8)
    g = torch.from_numpy(grid(fmt)).cuda()
    table = torch.cat((g, -g)) if fmt == "e2m1" else torch.cat((g, g[:1], -g, g[:1]))
    code, s = torch.from_numpy(code).cuda(), torch.from_numpy(s).cuda()
    c = code.long() if fmt == "e4m3" else torch.stack((code & 15, code >> 4), -1).view(n, -1).long()
    return bts.MxRows(code, s, d, fmt), table[c] * torch.exp2(s.double() - 127).repeat_interleave(32, 1)


# The 256 x 256 and 128 x 128 tiles, from one stage to an odd and an even number of many.  The large sizes select them on a card of 256
# CUs, the small ones on the emulation told to have one.
LARGE_TILES = [pytest.param(n, m, d, id="%s-%d-%d-%d" % (name, n, m, d))
               for name, n, m, depths in (("big256", 4000, 4090, (100, 2048, 2176, 2300)), ("big128", 2900, 2970, (100, 2048, 2176, 2300)),
                                          ("one256", 200, 250, (100, 768, 898)), ("four256", 300, 500, (100, 640)), ("few128", 100, 300, (100, 384, 640, 768)))
               for d in depths
               if name.startswith("big") or "HIPEMU_CUS" in os.environ or "libbotsort_emu" not in os.environ.get("BTS_LIB_PATH", "")]


@pytest.mark.parametrize("fa,fb", FMTS)
@pytest.mark.parametrize("n,m,d", LARGE_TILES)
def test_product_large_tiles(bts, n, m, d, fa, fb):
    """the sum's own error is `product_bound`'s, times the factor"""
    (a, ra), (b, rb) = random_rows(bts, n, d, fa, n + d), random_rows(bts, m, d, fb, m + d + 1)
    rbt = rb.t().contiguous()
    ref, mag = ra @ rbt, ra.abs() @ rbt.abs()
    own = (wide(d) / 128 + 20) * 2.0 ** -24 if fa == fb == "e2m1" else 2.0 ** -12
    for out, alpha, floor in (("f32" if fa == fb == "e2m1" else "bf16", -0.75, False), ("bf16", 0.125, True)):
        want = (ref * alpha).clamp(min=0) if floor else ref * alpha
        got = bts.mx_product(a, b, alpha=alpha, floor_zero=floor, dtype=DTYPES[out]).double()
        tol = HALF[out] * want.abs() + own * abs(alpha) * mag + float(torch.finfo(DTYPES[out]).smallest_normal) * HALF[out]
        assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


@pytest.mark.parametrize("fa,fb", FMTS)
@pytest.mark.parametrize("n,m,d", PRODUCTS + [(512, 256, 256)])
def test_product_error_goes_with_the_factor(bts, n, m, d, fa, fb):
    """as `run_product`, with the sum's own error times the factor for every type of output"""
    a, ra = rows_of(bts, feature_rows(n, d, 7 * n + d), fa)
    b, rb = rows_of(bts, feature_rows(m, d, 9 * m + d), fb)
    ref, mag = ra @ rb.T, np.abs(ra) @ np.abs(rb).T
    own = (d / 128 + 20) * 2.0 ** -24 if fa == fb == "e2m1" else 2.0 ** -12
    for out in ("f32", "bf16", "f16") if fa == fb == "e2m1" else ("f16", "bf16"):
        for alpha in (0.125, -0.0437):
            got = bts.mx_product(a, b, alpha=alpha, dtype=DTYPES[out]).cpu().double().numpy()
            want = ref * float(np.float32(alpha))
            tol = HALF[out] * np.abs(want) + own * abs(alpha) * mag + float(torch.finfo(DTYPES[out]).smallest_normal) * HALF[out]
            assert (np.abs(got - want) <= tol).all(), (out, alpha)


def test_product_big_row_counts(bts):
    """more tiles than one launch's workgroups; an output whose row stride is wide"""
    m, at = 2 ** 26 + 700, [0, 5, 2 ** 26 - 1, 2 ** 26, 2 ** 26 + 63, 2 ** 26 + 64, 2 ** 26 + 699]
    one, row = feature_rows(2, 128, 1), feature_rows(len(at), 128, 2)
    a, ra = rows_of(bts, one, "e2m1")
    few, rb = rows_of(bts, row, "e2m1")
    b = bts.MxRows(few.codes[:1].repeat(m, 1), few.scales[:1].repeat(m, 1), 128, "e2m1")
    for k, i in enumerate(at):
        b.codes[i], b.scales[i] = few.codes[k], few.scales[k]
    got = bts.mx_product(a, b, dtype=torch.bfloat16)
    want = ra @ rb.T
    tol = product_bound(ra, rb, "bf16", want, ("e2m1", "e2m1"))
    assert (np.abs(got[:, at].cpu().double().numpy() - want) <= tol).all()
    rest = torch.ones(m, dtype=torch.bool)
    rest[at] = False
    assert (got.cpu()[:, rest] == got[:, :1].cpu()).all()
    got = bts.mx_product(b, a, dtype=torch.bfloat16)
    assert (np.abs(got[at].cpu().double().numpy() - want.T) <= tol.T).all() and (got.cpu()[rest] == got[:1].cpu()).all()


@pytest.mark.parametrize("n,cols", [(70, 5_000_000), (40, 40_000_000)])
def test_product_big_row_strides(bts, n, cols):
    """a block of a matrix whose rows lie far apart: 64-bit places between the rows of one tile"""
    out = torch.zeros((n, cols), dtype=torch.bfloat16, device="cuda")
    a, ra = rows_of(bts, feature_rows(n, 200, 1), "e4m3")
    b, rb = rows_of(bts, feature_rows(3000, 200, 2), "e2m1")
    got = bts.mx_product(a, b, out=out[:, 1000:4000]).cpu().double().numpy()
    want = ra @ rb.T
    assert (np.abs(got - want) <= product_bound(ra, rb, "bf16", want, ("e4m3", "e2m1"))).all()
    assert (out[:, :1000] == 0).all() and (out[:, 4000:] == 0).all()


@pytest.mark.parametrize("fa,fb", FMTS)
@pytest.mark.parametrize("n,m", [(20, 40), (1, 700), (300, 290)])
def test_product_nan_blocks_and_extreme_scales(bts, n, m, fa, fb):
    d = 200
    va, vb = feature_rows(n, d, 1), feature_rows(m, d, 2)
    a, ra = rows_of(bts, va, fa)
    b, rb = rows_of(bts, vb, fb)
    a.scales[n - 1, 2] = 255                       # a NaN block takes its row (and the other operand's column) with it
    b.scales[3, 0] = 255
    a.scales[0, 7:] = 254                          # the padding (elements 224 ..): zero whatever its scale says
    b.scales[m - 1] = 0                            # 2^-127: products around the end of float32's range
    got = bts.mx_product(a, b, dtype=torch.bfloat16, floor_zero=True).cpu().double().numpy()
    nan = np.zeros((n, m), bool)
    nan[n - 1] = True; nan[:, 3] = True
    assert np.array_equal(np.isnan(got), nan)
    ra, rb = (np.nan_to_num(decode_ref(*host(r), r.fmt)) for r in (a, b))
    ref = np.maximum(ra @ rb.T, 0)
    tol = product_bound(ra, rb, "bf16", ref, (fa, fb)) + 256 * 2.0 ** -126           # (a product below the normal range may count as 0)
    assert (np.abs(got - ref) <= tol)[~nan].all()


@pytest.mark.parametrize("out", list(DTYPES))
@pytest.mark.parametrize("n,m,ld,off", [(7, 37, 61, 0), (7, 37, 64, 1), (130, 132, 140, 4), (130, 131, 133, 2)])
def test_product_into_a_wider_matrix(bts, n, m, ld, off, out):
    """unaligned and aligned rows of the output; what lies between the rows is left alone"""
    a, ra = rows_of(bts, feature_rows(n, 160, 4), "e2m1")
    b, rb = rows_of(bts, feature_rows(m, 160, 5), "e2m1")
    flat = torch.full((off + n * ld + 5,), 3.0, dtype=DTYPES[out]).cuda()
    view = torch.as_strided(flat, (n, m), (ld, 1), off)
    assert bts.mx_product(a, b, out=view) is view
    want = bts.mx_product(a, b, dtype=DTYPES[out]).cpu()
    got = flat.cpu()
    assert torch.equal(torch.as_strided(got, (n, m), (ld, 1), off), want)
    mask = torch.ones_like(got, dtype=torch.bool)
    torch.as_strided(mask, (n, m), (ld, 1), off)[...] = False
    assert (got[mask] == 3).all()


def test_empty_sides(bts):
    e, one = bts.MxRows.empty(0, 100, "e2m1"), bts.mx_quantize(torch.ones((1, 100)).cuda(), "e2m1")
    assert bts.mx_product(e, one).shape == (0, 1) and bts.mx_product(one, e).shape == (1, 0)
    assert len(bts.mx_quantize(torch.ones((0, 100)).cuda())) == 0 and e.dequantize().shape == (0, 100)
    q, h = bts.rms_norm_mx(torch.ones((0, 100)).cuda())
    assert len(q) == 0 and h.shape == (0, 100)


# ----------------------------------------------------------------------------------------------------------------- together

@pytest.mark.parametrize("gallery,queries,d,fa,fmt", [(200, 33, 384, "e2m1", "e4m3"), (130, 1, 250, "e2m1", "e2m1"), (64, 70, 512, "e4m3", "e4m3")])
def test_gallery_search_as_it_is_used(bts, gallery, queries, d, fa, fmt):
    """enrol a gallery in few bits; normalise a frame's rows (residual, weight) to few bits; their cosine similarities.  Every stage is
    held to the one before it, and the end to `cosine_similarity` of the unquantised unit rows."""
    g = feature_rows(gallery, d, 1)
    g /= np.linalg.norm(g, axis=1, keepdims=True)
    r = np.random.default_rng(2)
    x = torch.from_numpy(g[r.integers(0, gallery, queries)] * math.sqrt(d) + 0.3 * r.standard_normal((queries, d))).to(torch.bfloat16)
    res = torch.from_numpy(0.1 * r.standard_normal((queries, d))).to(torch.bfloat16)
    table = bts.mx_quantize(torch.from_numpy(g).float().cuda(), fa)
    q, h = bts.rms_norm_mx(x.cuda(), residual=res.cuda(), fmt=fmt)
    sim = bts.mx_product(table, q, alpha=1.0 / math.sqrt(d), floor_zero=True, dtype=torch.bfloat16).cpu().double().numpy()
    want_h, v = norm_ref(x, res, None, 1e-6)
    assert torch.equal(h.cpu(), want_h)
    check_quantized(v, *host(q), fmt, d, norm_delta(d))
    a, b = decode_ref(*host(table), fa), decode_ref(*host(q), fmt)
    ref = np.maximum(a @ b.T / math.sqrt(d), 0)
    assert (np.abs(sim - ref) <= product_bound(a, b, "bf16", ref, (fa, fmt))).all()
    unit = v / np.linalg.norm(v, axis=1, keepdims=True)
    full = bts.cosine_similarity(g.astype(np.float32), unit.astype(np.float32))
    # a 4-bit element is off by at most 1/4 of its magnitude or an eighth of its block's unit: independent signs leave it near
    # 0.12 / sqrt(d) * |a||b| a side; 6 of those, for both sides, and the bfloat16 output
    assert np.abs(sim - full).max() <= 2 * 6 * 0.12 / math.sqrt(d) + 2 ** -8


def test_a_slice_of_rows(bts):
    """rows built from parts of other rows' tensors, written in place as well"""
    x = torch.from_numpy(feature_rows(9, 200, 4)).float().cuda()
    for fmt in ("e2m1", "e4m3"):
        q = bts.mx_quantize(x, fmt)
        part = bts.MxRows(q.codes[3:7], q.scales[3:7], 200, fmt)
        assert len(part) == 4 and torch.equal(part.dequantize().cpu(), q.dequantize()[3:7].cpu())
        assert q.codes.shape == (9, bts.mx_row_bytes(fmt, 200)[0]) and q.scales.shape == (9, bts.mx_row_bytes(fmt, 200)[1])
        before = q.dequantize().cpu()
        bts.mx_quantize(2 * x[3:7], fmt, out=part)                                  # (twice the values: the same codes, scales one up)
        after = q.dequantize().cpu()
        assert torch.equal(after[3:7], 2 * before[3:7]) and torch.equal(after[:3], before[:3]) and torch.equal(after[7:], before[7:])
        assert torch.equal(bts.mx_product(part, q, dtype=torch.bfloat16).cpu(), bts.mx_product(q, q, dtype=torch.bfloat16).cpu()[3:7])


def test_leaves_that_want_a_gradient(bts):
    x, w = torch.ones((2, 64)).cuda().requires_grad_(), torch.ones(64).cuda().requires_grad_()
    for call in (lambda: bts.mx_quantize(x), lambda: bts.rms_norm_mx(x), lambda: bts.rms_norm_mx(x.detach(), weight=w),
                 lambda: bts.rms_norm_mx(x.detach(), residual=x)):
        with pytest.raises(bts.BtsError):
            call()
    with torch.no_grad():
        assert len(bts.mx_quantize(x)) == 2 and len(bts.rms_norm_mx(x, weight=w)[0]) == 2


@pytest.mark.skipif("libbotsort_emu" in __import__("os").environ.get("BTS_LIB_PATH", ""), reason="torch's dual tensors need the functions that the emulation replaces")
def test_forward_mode_tangents_are_refused(bts):
    """a dual tensor's tangent would be dropped without a word; while gradients are off too, forward mode goes on there"""
    from torch.autograd import forward_ad
    x, w = torch.ones((2, 64)).cuda(), torch.ones(64).cuda()
    with forward_ad.dual_level():
        dx, dw = forward_ad.make_dual(x, x), forward_ad.make_dual(w, w)
        calls = (lambda: bts.mx_quantize(dx), lambda: bts.rms_norm_mx(dx), lambda: bts.rms_norm_mx(x, weight=dw), lambda: bts.rms_norm_mx(x, residual=dx),
                 lambda: bts.rms_norm_mx(x, sum_out=dx), lambda: bts.mx_product(bts.mx_quantize(x), bts.mx_quantize(x), out=dx[:, :2]))
        for call in calls:
            with pytest.raises(bts.BtsError):
                call()
            with torch.no_grad(), pytest.raises(bts.BtsError):
                call()
        assert len(bts.rms_norm_mx(x, weight=w)[0]) == 2
    assert len(bts.mx_quantize(x)) == 2


def test_what_is_written_in_place_counts_as_changed(bts):
    """autograd's check of saved tensors: an output in the place of a tensor that a backward pass needs makes that pass an error"""
    leaf = torch.linspace(-1, 1, 128).view(2, 64).cuda().requires_grad_()
    saved = leaf.exp()                                                              # (exp keeps its result for the backward pass)
    with torch.no_grad():
        bts.rms_norm_mx(saved, residual=torch.ones_like(saved), sum_out=saved)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.sum().backward()
    x, h, y = (torch.ones((3, 64)).cuda() for _ in range(3))
    rows, own = bts.MxRows.empty(3, 64, "e4m3"), bts.mx_quantize(x)
    part = bts.MxRows(rows.codes, rows.scales, 64, "e4m3")
    out = torch.zeros((3, 3), dtype=torch.bfloat16).cuda()
    for written, call in (((h, y, rows.codes, rows.scales), lambda: bts.rms_norm_mx(x, sum_out=h, y_out=y, out=rows)), ((x,), lambda: bts.rms_norm_mx(x, y_out=x)),
                          ((part.codes, part.scales, rows.codes), lambda: bts.mx_quantize(x, "e4m3", out=part)), ((out,), lambda: bts.mx_product(own, own, out=out))):
        before = [t._version for t in written]
        call()
        assert all(t._version > b for t, b in zip(written, before))
    before = x._version, own.codes._version
    bts.rms_norm_mx(x, residual=h)
    bts.mx_product(own, own)
    own.dequantize()
    assert (x._version, own.codes._version) == before                              # (what is only read does not)
    with torch.inference_mode():                                                    # (tensors without a counter)
        z = torch.ones((3, 64)).cuda()
        assert bts.rms_norm_mx(z, y_out=z, out=bts.MxRows.empty(3, 64, "e4m3"))[1].shape == (3, 64)
    with torch.no_grad():
        bts.rms_norm_mx(x, sum_out=z, y_out=y)


def test_two_runs_give_the_same_bits(bts):
    a, _ = rows_of(bts, feature_rows(150, 900, 7), "e4m3")
    b, _ = rows_of(bts, feature_rows(90, 900, 8), "e2m1")
    x = torch.from_numpy(feature_rows(40, 900, 9)).float().cuda()
    one, two = bts.mx_product(a, b).cpu(), bts.mx_product(a, b).cpu()
    assert torch.equal(one, two)
    assert torch.equal(bts.rms_norm_mx(x)[0].codes.cpu(), bts.rms_norm_mx(x)[0].codes.cpu())


# ----------------------------------------------------------------------------------------------------------------- refusals

def test_refusals(bts):
    x = torch.ones((4, 64)).cuda()
    q, q8 = bts.mx_quantize(x, "e2m1"), bts.mx_quantize(x, "e4m3")
    bad = [
        lambda: bts.mx_quantize(x, "e5m2"),
        lambda: bts.mx_quantize(x.double()),
        lambda: bts.mx_quantize(x[0]),
        lambda: bts.mx_quantize(x.t()),
        lambda: bts.mx_quantize(x[:1].expand(4, 64)),
        lambda: bts.mx_quantize(x[:, :0]),
        lambda: bts.mx_quantize(x, "e2m1", out=q8),
        lambda: bts.mx_quantize(x[:3], "e2m1", out=q),
        lambda: q.dequantize(torch.int32),
        lambda: bts.MxRows(q.codes, q.scales, 200, "e2m1"),
        lambda: bts.MxRows(q.codes, q.scales, 64, "e4m3"),
        lambda: bts.MxRows(q.codes, q.scales[:3], 64, "e2m1"),
        lambda: bts.MxRows(q.codes.t().contiguous().t(), q.scales, 64, "e2m1"),
        lambda: bts.MxRows(q.codes, q.scales, 0, "e2m1"),
        lambda: bts.rms_norm_mx(x, residual=x[:3]),
        lambda: bts.rms_norm_mx(x, residual=x.half()),
        lambda: bts.rms_norm_mx(x, weight=x[0, :63]),
        lambda: bts.rms_norm_mx(x, weight=x[0].half()),
        lambda: bts.rms_norm_mx(x, eps=0.0),
        lambda: bts.rms_norm_mx(x, eps=float("nan")),
        lambda: bts.rms_norm_mx(x, eps=float("inf")),
        lambda: bts.rms_norm_mx(x, eps=1e-60),
        lambda: bts.rms_norm_mx(x, fmt=None),
        lambda: bts.rms_norm_mx(x, fmt=None, y_out=torch.empty_like(x), out=q),
        lambda: bts.rms_norm_mx(x, fmt=None, sum_out=(s := torch.empty_like(x)), y_out=s),
        lambda: bts.mx_product(q8, q, dtype=torch.float32),
        lambda: bts.mx_product(q, q, dtype=torch.float64),
        lambda: bts.mx_product(q, bts.mx_quantize(x[:, :40].contiguous())),
        lambda: bts.mx_product(q, x),
        lambda: bts.mx_product(q, q, out=torch.empty((4, 5)).cuda()),
        lambda: bts.mx_product(q, q, out=torch.empty((4, 4)).cuda(), dtype=torch.float16),
        lambda: bts.mx_product(q, q, out=torch.empty((4, 4)).cuda().t()),
        lambda: bts.mx_row_bytes("e2m1", 0),
        lambda: bts.mx_row_bytes("e2m1", 2 ** 30 + 1),
        lambda: bts.mx_row_bytes("e2m1", 2 ** 32 + 5),
        lambda: bts.MxRows.empty(1, 2 ** 32 + 5, "e2m1"),
        lambda: bts.MxRows.empty(2 ** 31, 1, "e2m1"),
        lambda: bts.MxRows.empty(-1, 1, "e2m1"),
    ]
    for k, f in enumerate(bad):
        with pytest.raises(bts.BtsError):
            f()
            print("accepted", k)


def test_c_entry_refusals(bts):
    """bad arguments at the C boundary: a status, no launch"""
    lib, ctx = bts._lib.load(), bts._lib.default_context().handle
    x, o = torch.ones((4, 128)).cuda(), torch.zeros((4, 128), dtype=torch.uint8).cuda()
    s, p = torch.zeros((4, 4), dtype=torch.uint8).cuda(), lambda t, off=0: t.data_ptr() + off
    ok = [ctx, p(x), 1, 128, 4, 128, 1, p(o), p(s), None]
    for at, v in ((0, None), (1, None), (2, 0), (2, 7), (3, 127), (4, -1), (5, 0), (6, 2), (7, None), (7, p(o, 4)), (8, None), (8, p(s, 1)), (1, p(x, 2))):
        assert lib.bts_mx_quantize(*(ok[:at] + [v] + ok[at + 1:])) == -1, (at, v)
    ok = [ctx, p(o), p(s), 1, 4, 128, p(x), 1, 128, None]
    for at, v in ((0, None), (1, None), (2, None), (3, 5), (4, -3), (5, -1), (6, None), (7, 0), (8, 100), (6, p(x, 1)), (1, p(o, 8))):
        assert lib.bts_mx_dequantize(*(ok[:at] + [v] + ok[at + 1:])) == -1, (at, v)
    ok = [ctx, 1, p(x), 128, None, 0, None, 4, 128, 1e-6, None, 0, None, 0, 1, p(o), p(s), None]
    for at, v in ((0, None), (1, 0), (2, None), (3, 64), (4, p(x)), (7, -1), (8, 0), (9, 0.0), (10, p(x)), (12, p(x)), (14, 9), (15, None), (16, None), (15, p(o, 4))):
        assert lib.bts_rms_norm(*(ok[:at] + [v] + ok[at + 1:])) == -1, (at, v)
    ok = [ctx, p(o), p(s), 1, 4, p(o), p(s), 1, 4, 128, 1.0, 0, p(x), 3, 4, None]
    for at, v in ((0, None), (1, None), (2, None), (3, 2), (4, -1), (5, None), (6, None), (7, -1), (8, -1), (9, 0), (12, None), (13, 0), (13, 1), (14, 3), (1, p(o, 1)), (6, p(s, 2)), (12, p(x, 1))):
        assert lib.bts_mx_product(*(ok[:at] + [v] + ok[at + 1:])) == -1, (at, v)
    assert (x.cpu() == 1).all() and (o.cpu() == 0).all()


def shares(a, b):
    """whether two sets of rows (place, rows, bytes a row, bytes between rows) share a byte, byte by byte"""
    put = lambda r: {r[0] + i * r[3] + k for i in range(r[1]) for k in range(r[2])}  # noqa: E731
    return bool(put(a) & put(b))


def test_outputs_that_share_memory_are_refused(bts):
    """every place of one output against one input inside a small buffer, decided by the bytes they share: y and x of the norm, of equal and of
    different row strides; refused before anything is launched, and accepted when they only lie between each other's rows"""
    lib, ctx = bts._lib.load(), bts._lib.default_context().handle
    buf = torch.ones(600).cuda()
    seen = set()
    for n, d, ldx, ldy in ((3, 4, 12, 12), (3, 4, 9, 9), (4, 3, 7, 11), (1, 5, 5, 5), (5, 4, 4, 4), (4, 2, 13, 5)):
        at = 150
        for to in range(at - n * max(ldx, ldy) - d - 1, at + n * max(ldx, ldy) + d + 2):
            want = shares((4 * at, n, 4 * d, 4 * ldx), (4 * to, n, 4 * d, 4 * ldy)) and not (to == at and ldx == ldy)
            before = buf.cpu()
            rc = lib.bts_rms_norm(ctx, 1, buf.data_ptr() + 4 * at, ldx, None, 0, None, n, d, 1e-6, None, 0, buf.data_ptr() + 4 * to, ldy, 0, None, None, None)
            assert rc == (-1 if want else 0), (n, d, ldx, ldy, to - at)
            if want:
                assert torch.equal(buf.cpu(), before)
            buf.fill_(1.0)
            seen.add((want, ldx == ldy))
    assert len(seen) == 4


def test_overlapping_tensors_are_refused(bts):
    x = torch.ones((6, 400)).cuda()
    a, b, w = x[:, :128], x[:, 8:136], torch.ones(128).cuda()
    raw = torch.zeros(40000, dtype=torch.uint8).cuda()
    rows = lambda at, n, fmt="e4m3": bts.MxRows(raw[at:at + n * bts.mx_row_bytes(fmt, 128)[0]].view(n, -1),  # noqa: E731
                                                raw[at + 20000:at + 20000 + 4 * n].view(n, 4), 128, fmt)
    q = bts.mx_quantize(a, "e4m3", out=rows(0, 6))
    f32 = lambda at, n, d: raw[at:at + 4 * n * d].view(torch.float32).view(n, d)  # noqa: E731
    bad = [
        lambda: bts.rms_norm_mx(a, sum_out=b),
        lambda: bts.rms_norm_mx(a, y_out=b),
        lambda: bts.rms_norm_mx(x[:5, :128], y_out=x[1:, :128]),                       # the same columns, a row further
        lambda: bts.rms_norm_mx(a, residual=x[:, 200:328], sum_out=x[:, 201:329]),
        lambda: bts.rms_norm_mx(a, residual=x[:, 200:328], sum_out=a, y_out=x[:, 127:255]),
        lambda: bts.rms_norm_mx(a, residual=b, sum_out=a),                             # in the place of x, across residual
        lambda: bts.rms_norm_mx(a, sum_out=x[:, 200:328], y_out=x[:, 272:]),
        lambda: bts.rms_norm_mx(a, weight=x[3, :128], sum_out=a),                      # the weight is a row of what is written
        lambda: bts.rms_norm_mx(a, weight=x[2, 272:], y_out=x[:, 272:]),
        lambda: bts.rms_norm_mx(f32(0, 2, 128), out=rows(512, 2)),                     # codes over x
        lambda: bts.rms_norm_mx(f32(20400, 2, 128), out=rows(512, 2)),                 # scales over x
        lambda: bts.rms_norm_mx(a[:4], y_out=f32(512, 4, 128), out=rows(256, 4)),
        lambda: bts.mx_quantize(f32(256, 4, 128), "e4m3", out=rows(0, 4)),
        lambda: bts.mx_quantize(f32(20008, 4, 128), "e4m3", out=rows(0, 4)),
        lambda: bts.mx_product(rows(0, 4), rows(1024, 4), out=raw[1024:1024 + 32].view(torch.bfloat16).view(4, 4)),
        lambda: bts.mx_product(rows(0, 4), rows(1024, 4), out=raw[20000:20032].view(torch.bfloat16).view(4, 4)),
    ]
    lib, ctx = bts._lib.load(), bts._lib.default_context().handle
    before = x.cpu(), raw.cpu()
    for k, f in enumerate(bad):
        with pytest.raises(bts.BtsError):
            f()
            print("accepted", k)
    assert lib.bts_mx_dequantize(ctx, raw.data_ptr(), raw.data_ptr() + 20000, 1, 6, 128, raw.data_ptr() + 512, 1, 128, None) == -1
    assert lib.bts_mx_dequantize(ctx, raw.data_ptr(), raw.data_ptr() + 20000, 1, 6, 128, raw.data_ptr() + 20008, 1, 128, None) == -1
    assert lib.bts_mx_quantize(ctx, x.data_ptr(), 1, 400, 6, 128, 1, raw.data_ptr(), raw.data_ptr() + 764, None) == -1      # scales in the codes
    assert torch.equal(x.cpu(), before[0]) and torch.equal(raw.cpu(), before[1])
    # columns of one matrix beside each other, a and b the same rows, the addition in place
    h = bts.rms_norm_mx(a, residual=x[:, 128:256], sum_out=x[:, 256:384])[1]
    assert (h == 2).all() and (x[:, :256] == 1).all()
    assert bts.rms_norm_mx(a, residual=a, sum_out=a, weight=w)[1] is a and (a == 2).all()
    assert bts.mx_product(q, q).shape == (6, 6)


def test_factors_that_float32_does_not_hold(bts):
    """the kernels multiply by alpha in float32: 1e300 would be infinite and 1e-60 nothing, whatever the products are"""
    v = torch.ones((2, 64)).cuda()
    q = bts.mx_quantize(v)
    for alpha in (1e300, -1e39, 1e-60, float("inf"), float("-inf"), float("nan")):
        with pytest.raises(bts.BtsError, match="alpha"):
            bts.mx_product(q, q, alpha=alpha)
    for alpha in (0.0, -0.0, 1e-44, 2.0 ** -126, -5.3e36):                           # (64 times these: exact)
        assert (bts.mx_product(q, q, alpha=alpha).cpu() == 64 * torch.tensor(alpha, dtype=torch.float32)).all()


# ------------------------------------------------------------------------------------------- streams, graphs, threads (hardware)

@pytest.mark.skipif("libbotsort_emu" in __import__("os").environ.get("BTS_LIB_PATH", ""), reason="needs real streams and graphs")
class TestStreams:
    def _pass(self, bts, x, res, table, st=None):
        q, h = bts.rms_norm_mx(x, residual=res, fmt="e4m3")
        return q, h, bts.mx_product(table, q, dtype=torch.bfloat16)

    def _inputs(self, bts):
        x = torch.from_numpy(feature_rows(70, 640, 1)).to(torch.bfloat16).cuda()
        res = torch.from_numpy(feature_rows(70, 640, 2)).to(torch.bfloat16).cuda()
        return x, res, bts.mx_quantize(torch.from_numpy(feature_rows(600, 640, 3)).float().cuda())

    def test_another_stream(self, bts):
        x, res, table = self._inputs(bts)
        want = self._pass(bts, x, res, table)[2].cpu()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append(self._pass(bts, x, res, table)[2])
        torch.cuda.synchronize()
        for g in got:
            assert torch.equal(g.cpu(), want)

    def test_graph_replays(self, bts):
        x, res, table = self._inputs(bts)
        self._pass(bts, x, res, table)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            q, h, out = self._pass(bts, x, res, table)
        for k in range(4):
            nx = torch.from_numpy(feature_rows(70, 640, 50 + k)).to(torch.bfloat16).cuda()
            x.copy_(nx)
            graph.replay()
            torch.cuda.synchronize()
            eq, eh, eo = self._pass(bts, nx, res, table)
            assert torch.equal(out.cpu(), eo.cpu()) and torch.equal(h.cpu(), eh.cpu()) and torch.equal(q.codes.cpu(), eq.codes.cpu())
