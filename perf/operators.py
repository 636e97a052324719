"""Measured cases of the microscaled-row operators: quantisation of feature rows to 4 or 8 bits with a scale per 32 elements, the
root-mean-square norm (with the residual's addition) that writes such rows, their product, and the norm and the product in a row.

`run` is the plain form in elementary torch operations (float32, rounded once at the end) or, with `own`, the calls a user makes.
`exact` is the definition in float64, written apart from the plain form.

Rows: 32-element blocks share one scale byte s, worth 2^(s - 127); elements are e2m1 (two a byte, the even one in the low nibble) or
e4m3 (one a byte); rows are padded with zeros to a multiple of 128 elements.  What is held in 4 or 8 bits is returned as the values it
stands for, in bfloat16, which holds each of them exactly."""
import math

import torch

own = False

_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_EMAX = {"e2m1": 2, "e4m3": 8}          # exponent of the format's largest power of two
_MAX = {"e2m1": 6.0, "e4m3": 448.0}
_MANT = {"e2m1": 1, "e4m3": 3}          # fraction bits
_EMIN = {"e2m1": 0, "e4m3": -6}         # exponent of the smallest normal value


def listed():
    return [
        # one face / body row enrolled (config 5's feature width): latency
        {"name": "quantize_one_row", "op": "quantize", "n": 1, "d": 384, "dtype": "f32", "fmt": "e4m3"},
        # the detections of one headline frame
        {"name": "quantize_frame", "op": "quantize", "n": 2000, "d": 2048, "dtype": "f32", "fmt": "e2m1"},
        # a whole gallery, laid out once and refreshed when the encoder changes
        {"name": "quantize_gallery", "op": "quantize", "n": 65536, "d": 2048, "dtype": "bf16", "fmt": "e2m1"},
        # one row through the encoder's last norm: latency
        {"name": "norm_one_row", "op": "norm", "n": 1, "d": 2048, "dtype": "bf16", "fmt": "e4m3", "residual": True, "weight": True},
        # a frame's rows, no residual, no weight (the row normalisation the tracker knows, up to sqrt(d)), odd width
        {"name": "norm_frame_odd", "op": "norm", "n": 1999, "d": 1111, "dtype": "f32", "fmt": "e4m3", "residual": False, "weight": False},
        # a batch of patch rows inside an encoder
        {"name": "norm_batch", "op": "norm", "n": 32768, "d": 4096, "dtype": "bf16", "fmt": "e4m3", "residual": True, "weight": True},
        # one query against a gallery: the reading of the gallery
        {"name": "product_one_query", "op": "product", "n": 1, "m": 65536, "d": 2048, "fa": "e4m3", "fb": "e2m1", "out": "bf16", "floor": True},
        # the small stream of the tests (512 tracks x 256 detections)
        {"name": "product_small", "op": "product", "n": 512, "m": 256, "d": 256, "fa": "e2m1", "fb": "e2m1", "out": "f32", "floor": True},
        # the headline table: 10 000 tracks x 2 000 detections x 2048
        {"name": "product_headline", "op": "product", "n": 10000, "m": 2000, "d": 2048, "fa": "e2m1", "fb": "e2m1", "out": "f32", "floor": True},
        # ragged in all three sizes
        {"name": "product_odd", "op": "product", "n": 333, "m": 1111, "d": 500, "fa": "e4m3", "fb": "e2m1", "out": "f16", "floor": False},
        # a dense layer / gallery against gallery: the matrix cores
        {"name": "product_large", "op": "product", "n": 16384, "m": 8192, "d": 4096, "fa": "e4m3", "fb": "e2m1", "out": "bf16", "floor": False},
        # a frame in one go: residual + norm of the detections' rows to 8 bits, then their similarity to the table's 4-bit rows
        {"name": "frame_norm_product", "op": "frame", "n": 10000, "m": 2000, "d": 2048, "dtype": "bf16", "fmt": "e4m3", "fa": "e2m1", "out": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "norm", "product", "product", "frame"])
    if op in ("quantize", "norm"):
        d = _log(rng, 16, 8192)
        n = _log(rng, 1, min(1 << 17, (1 << 26) // d))
        case = {"op": op, "n": n, "d": d, "dtype": rng.choice(["f32", "f16", "bf16"]), "fmt": rng.choice(["e2m1", "e4m3"])}
        if op == "norm":
            case.update(residual=rng.random() < 0.6, weight=rng.random() < 0.6)
        return case
    d = _log(rng, 32, 4096 if op == "frame" else 8192)
    if op == "frame":
        n, m = _log(rng, 16, 12000), _log(rng, 1, 4000)
        return {"op": op, "n": n, "m": m, "d": d, "dtype": rng.choice(["f32", "f16", "bf16"]), "fmt": rng.choice(["e2m1", "e4m3"]),
                "fa": rng.choice(["e2m1", "e4m3"]), "out": rng.choice(["f16", "bf16"])}
    n = _log(rng, 1, 16384)
    most = min(1 << 17, (1 << 28) // d, (1 << 27) // n, (1 << 38) // (n * d))
    m = _log(rng, 1, max(1, most))
    fa, fb = rng.choice([("e2m1", "e2m1"), ("e4m3", "e2m1"), ("e2m1", "e4m3"), ("e4m3", "e4m3")])
    out = rng.choice(["f32", "f16", "bf16"]) if fa == fb == "e2m1" else rng.choice(["f16", "bf16"])
    return {"op": op, "n": n, "m": m, "d": d, "fa": fa, "fb": fb, "out": out, "floor": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------- plain form (float32)

def _pad(d):
    return (d + 127) // 128 * 128


def _blocks(v, width):
    """[n, d] -> [n, width / 32, 32], zeros behind the row's end."""
    n, d = v.shape
    return torch.nn.functional.pad(v, (0, width - d)).view(n, width // 32, 32)


def _round_rows(v, fmt):
    """float32 [n, d] -> (elements [n, blocks, 32] as float32, shared exponents [n, blocks] as int32)."""
    b = _blocks(v, _pad(v.shape[1]))
    top = b.abs().amax(-1)
    shared = torch.where(top > 0, (torch.frexp(top)[1] - 1 - _EMAX[fmt]).clamp(-127, 127), torch.full_like(top, -127, dtype=torch.int32))
    x = torch.ldexp(b, -shared[..., None])
    e = (torch.frexp(x)[1] - 1).clamp(min=_EMIN[fmt])
    step = e - _MANT[fmt]
    q = torch.ldexp(torch.round(torch.ldexp(x, -step)), step)
    return q.clamp(-_MAX[fmt], _MAX[fmt]), shared


def _values(v, fmt):
    """float32 [n, d] -> the values its quantised row stands for."""
    q, shared = _round_rows(v, fmt)
    return torch.ldexp(q, shared[..., None]).view(v.shape[0], -1)[:, : v.shape[1]]


def _encode(v, fmt):
    """float32 [n, d] -> (codes, scales) as the rows are held."""
    q, shared = _round_rows(v, fmt)
    n = v.shape[0]
    a = q.abs()
    sign = torch.signbit(q)
    e = (torch.frexp(a)[1] - 1).clamp(min=_EMIN[fmt])
    frac = torch.ldexp(a, _MANT[fmt] - e).to(torch.int32)                       # 2^mant + fraction for normals, the fraction below
    code = frac + ((e - _EMIN[fmt]) << _MANT[fmt])
    code = (code + (sign.to(torch.int32) << (3 if fmt == "e2m1" else 7))).view(n, -1)
    if fmt == "e2m1":
        code = code[:, 0::2] + (code[:, 1::2] << 4)
    return code.to(torch.uint8).contiguous(), (shared + 127).to(torch.uint8).contiguous()


def _decode(rows):
    """Held rows -> float32 values [n, padded width]."""
    codes, scales, fmt = rows["codes"], rows["scales"], rows["fmt"]
    c = codes.to(torch.int32)
    if fmt == "e2m1":
        c = torch.stack((c & 15, c >> 4), -1).view(c.shape[0], -1)
    bits = _MANT[fmt]
    top = 3 if fmt == "e2m1" else 7
    e = (c & ((1 << top) - 1)) >> bits
    f = (c & ((1 << bits) - 1)) + torch.where(e > 0, 1 << bits, 0)
    v = torch.ldexp(f.to(torch.float32), e.clamp(min=1) - 1 + _EMIN[fmt] - bits)
    v = torch.where((c >> top) > 0, -v, v).view(c.shape[0], -1, 32)
    return torch.ldexp(v, scales.to(torch.int32)[..., None] - 127).view(c.shape[0], -1)


def _norm(x, residual, weight, eps):
    """(stored sum, normalised row in float32)."""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    f = h.float()
    y = f * (1.0 / torch.sqrt(f.square().mean(-1, keepdim=True) + eps))
    return h, y if weight is None else y * weight.float()


def _product(a, b, floor, dtype):
    r = a @ b.t()
    return (r.clamp(min=0) if floor else r).to(dtype)


# ------------------------------------------------------------------------------------------------------------ the tool's functions

def _rows(g, n, d):
    """Feature rows as an encoder leaves them: unit length, a shared direction in each group of rows, uneven channels."""
    groups = torch.randn((61, d), generator=g, device="cuda")
    pick = torch.randint(0, 61, (n,), generator=g, device="cuda")
    x = groups[pick] * 0.7 + torch.randn((n, d), generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn((d,), generator=g, device="cuda"))
    return x / x.norm(dim=1, keepdim=True)


def _held(g, n, d, fmt):
    codes, scales = _encode(_rows(g, n, d), fmt)
    return {"codes": codes, "scales": scales, "d": d, "fmt": fmt}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = dict(case)
    s = {"case": c}
    op, d = c["op"], c["d"]
    if op == "quantize":
        s["x"] = _rows(g, c["n"], d).to(_DTYPE[c["dtype"]])
    elif op == "norm" or op == "frame":
        rows = c["n"] if op == "norm" else c["m"]
        t = _DTYPE[c["dtype"]]
        s["x"] = (_rows(g, rows, d) * math.sqrt(d)).to(t)
        s["residual"] = (2.0 * torch.randn((rows, d), generator=g, device="cuda")).to(t) if op == "frame" or c["residual"] else None
        s["weight"] = (1.0 + 0.1 * torch.randn((d,), generator=g, device="cuda")).to(t) if op == "frame" or c["weight"] else None
        if op == "frame":
            s["table"] = _held(g, c["n"], d, c["fa"])
    else:
        s["a"], s["b"] = _held(g, c["n"], d, c["fa"]), _held(g, c["m"], d, c["fb"])
    return s


EPS = 1e-6


def run(state):
    c = state["case"]
    op = c["op"]
    if own:
        import botsort_amd as bts
        rows = lambda r: bts.MxRows(r["codes"], r["scales"], r["d"], r["fmt"])  # noqa: E731
        if op == "quantize":
            return bts.mx_quantize(state["x"], c["fmt"]).dequantize(torch.bfloat16)
        if op == "norm":
            q, h = bts.rms_norm_mx(state["x"], residual=state["residual"], weight=state["weight"], eps=EPS, fmt=c["fmt"])
            return [h, q.dequantize(torch.bfloat16)] if state["residual"] is not None else [q.dequantize(torch.bfloat16)]
        if op == "frame":
            q, h = bts.rms_norm_mx(state["x"], residual=state["residual"], weight=state["weight"], eps=EPS, fmt=c["fmt"])
            return [h, bts.mx_product(rows(state["table"]), q, alpha=1.0 / math.sqrt(c["d"]), floor_zero=True, dtype=_DTYPE[c["out"]])]
        return bts.mx_product(rows(state["a"]), rows(state["b"]), floor_zero=c["floor"], dtype=_DTYPE[c["out"]])
    if op == "quantize":
        return _values(state["x"].float(), c["fmt"]).to(torch.bfloat16)
    if op == "norm":
        h, y = _norm(state["x"], state["residual"], state["weight"], EPS)
        v = _values(y, c["fmt"]).to(torch.bfloat16)
        return [h, v] if state["residual"] is not None else [v]
    if op == "frame":
        h, y = _norm(state["x"], state["residual"], state["weight"], EPS)
        r = _decode(state["table"])[:, : c["d"]] @ _values(y, c["fmt"]).t()
        return [h, (r * (1.0 / math.sqrt(c["d"]))).clamp(min=0).to(_DTYPE[c["out"]])]
    return _product(_decode(state["a"]), _decode(state["b"]), c["floor"], _DTYPE[c["out"]])


def _held_bytes(n, d, fmt):
    return n * _pad(d) * (1 if fmt == "e4m3" else 0.5) + n * _pad(d) / 32


def work(case):
    op, n, d = case["op"], case["n"], case["d"]
    if op == "quantize":        # the row read, held, and given as values
        return {"bytes": n * d * (_BYTES[case["dtype"]] + 2) + _held_bytes(n, d, case["fmt"]), "flops": 4 * n * d}
    if op == "norm":
        k = _BYTES[case["dtype"]]
        moved = n * d * k * (3 if case["residual"] else 1) + (d * k if case["weight"] else 0)
        return {"bytes": moved + n * d * 2 + _held_bytes(n, d, case["fmt"]), "flops": 9 * n * d}
    m = case["m"]
    if op == "frame":
        k = _BYTES[case["dtype"]]
        return {"bytes": 3 * m * d * k + d * k + _held_bytes(n, d, case["fa"]) + _held_bytes(m, d, case["fmt"]) + n * m * _BYTES[case["out"]],
                "flops": 2 * n * m * d + 9 * m * d}
    return {"bytes": _held_bytes(n, d, case["fa"]) + _held_bytes(m, d, case["fb"]) + n * m * _BYTES[case["out"]], "flops": 2 * n * m * d}


# ------------------------------------------------------------------------------------------------- the definition in float64

def _grid(fmt):
    """The format's non-negative values in the order of their codes."""
    if fmt == "e2m1":
        return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    return torch.tensor([(m / 8 * 2.0 ** -6) if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127],
                        dtype=torch.float64, device="cuda")


def _nearest(v, fmt):
    """float64 [n, d] -> values of the quantised rows: the grid value nearest to v / scale, ties to the even code."""
    n, d = v.shape
    wide = (d + 31) // 32 * 32
    b = torch.zeros((n, wide), dtype=torch.float64, device=v.device)
    b[:, :d] = v
    b = b.view(n, wide // 32, 32)
    top = b.abs().max(-1, keepdim=True).values
    tiny = top <= 0
    e = torch.floor(torch.log2(torch.where(tiny, torch.ones_like(top), top)))
    e = torch.where(torch.exp2(e + 1) <= top, e + 1, torch.where(torch.exp2(e) > top, e - 1, e)) - math.floor(math.log2(_grid(fmt)[-1].item()))
    unit = torch.exp2(torch.where(tiny, torch.full_like(e, -127.0), e.clamp(-127, 127)))
    x = (b / unit).abs()
    grid = _grid(fmt)
    hi = torch.searchsorted(grid, x.contiguous()).clamp(max=grid.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    down, up = x - grid[lo], grid[hi] - x
    take = torch.where(down < up, lo, torch.where(down > up, hi, torch.where(lo % 2 == 0, lo, hi)))
    q = grid[take]
    return (torch.where(b < 0, -q, q) * unit).reshape(n, wide)[:, :d]


def _held_values(rows):
    """Held rows -> float64 values, by table."""
    grid = _grid(rows["fmt"])
    table = torch.cat((grid, -grid)) if rows["fmt"] == "e2m1" else torch.cat((grid, grid[-1:], -grid, -grid[-1:]))
    c = rows["codes"].long()
    if rows["fmt"] == "e2m1":
        c = torch.cat(((c % 16)[..., None], (c // 16)[..., None]), -1).reshape(c.shape[0], -1)
    v = table[c]
    return v * torch.exp2(rows["scales"].double() - 127).repeat_interleave(32, 1)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "quantize":
        return _nearest(s["x"].double(), c["fmt"])
    if c["op"] == "product":
        r = _held_values(s["a"]) @ _held_values(s["b"]).t()
        return torch.maximum(r, torch.zeros_like(r)) if c["floor"] else r
    h = s["x"].double()
    if s["residual"] is not None:
        h = (h + s["residual"].double()).to(s["x"].dtype).double()          # the sum as it is stored
    y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / c["d"] + EPS)
    if s["weight"] is not None:
        y = y * s["weight"].double()
    v = _nearest(y, c["fmt"])
    if c["op"] == "norm":
        return [h, v] if s["residual"] is not None else [v]
    r = _held_values(s["table"])[:, : c["d"]] @ v.t() / math.sqrt(c["d"])
    return [h, torch.maximum(r, torch.zeros_like(r))]
