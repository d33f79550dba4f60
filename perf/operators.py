"""What is measured of the 8-bit and training operators: LayerNorm forward and backward, Linear on 8-bit blocks, the
weight gradient from an 8-bit checkpoint and GeGLU with its 8-bit checkpoint.

``own = False`` computes a case with elementary torch operations in float32, ``own = True`` with the package's operators.
The 8-bit format of both: blocks of 128 along the last dimension (weights: 128 x 128) share a power-of-two scale, the
smallest one that brings the block's largest magnitude into the range of the 8-bit type.
"""
import math

import torch

own = False

BLOCK = 128
TOP = {"e4m3": 448.0, "e5m2": 57344.0}
FMT = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
EPS = 1e-5


def listed():
    return [
        # one prompt through the text encoder's width in f32: 77 rows, all latency
        {"name": "norm text encoder", "kind": "norm", "rows": 77, "width": 768, "x": "f32", "dy": "f32", "skip": False},
        # the 64x64 level of the UNet at batch 16: f32 trunk, bf16 branch, the skip's gradient added in
        {"name": "norm 64x64 trunk", "kind": "norm", "rows": 65536, "width": 320, "x": "f32", "dy": "bf16", "skip": True},
        # ragged rows of an odd width, all bf16
        {"name": "norm odd", "kind": "norm", "rows": 4099, "width": 1001, "x": "bf16", "dy": "bf16", "skip": False},
        # time embedding of one step: a single row
        {"name": "linear time embedding", "kind": "linear", "m": 1, "k": 320, "n": 1280, "x": "bf16", "y": "bf16", "fmt": "e4m3", "bias": True, "skip": False, "norm": False},
        # K | V projection of two prompts' context
        {"name": "linear context", "kind": "linear", "m": 154, "k": 768, "n": 640, "x": "f32", "y": "f32", "fmt": "e4m3", "bias": False, "skip": False, "norm": False},
        # LayerNorm straight into the 8-bit operand of the fused q | k | v projection, 16x16 level at batch 16
        {"name": "linear after norm", "kind": "linear", "m": 4096, "k": 1280, "n": 3840, "x": "f32", "y": "bf16", "fmt": "e4m3", "bias": True, "skip": False, "norm": True},
        # feed-forward up projection of the 32x32 level at batch 16
        {"name": "linear feed-forward", "kind": "linear", "m": 16384, "k": 640, "n": 5120, "x": "bf16", "y": "bf16", "fmt": "e4m3", "bias": True, "skip": False, "norm": False},
        # the widest projection at 768x768 pixels, 32 images with guidance; gradients take the e5m2 type
        {"name": "linear largest", "kind": "linear", "m": 36864, "k": 1280, "n": 10240, "x": "bf16", "y": "bf16", "fmt": "e5m2", "bias": False, "skip": False, "norm": False},
        # weight gradient of a small odd layer
        {"name": "weight gradient odd", "kind": "wgrad", "t": 1003, "n": 333, "k": 215, "x": "bf16", "fmt": "e4m3"},
        # weight gradient of the feed-forward up projection, 32x32 level at batch 16
        {"name": "weight gradient large", "kind": "wgrad", "t": 16384, "n": 5120, "k": 640, "x": "bf16", "fmt": "e4m3"},
        # one image's 16x16 level
        {"name": "geglu one image", "kind": "geglu", "rows": 256, "width": 5120, "x": "bf16", "fmt": "e4m3"},
        # the 64x64 level at batch 16
        {"name": "geglu 64x64", "kind": "geglu", "rows": 65536, "width": 1280, "x": "bf16", "fmt": "e4m3"},
    ]


def draw(rng):
    def spread(low, high):
        return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))

    def snapped(v, to):      # half of the sizes are multiples of ``to``, as model widths are
        return max(to, v // to * to) if rng.random() < 0.5 else v

    kind = rng.choice(("norm", "linear", "wgrad", "geglu"))
    if kind == "norm":
        width = snapped(spread(33, 8192), 32)
        rows = spread(1, min(100000, 20971520 // width))
        return {"kind": kind, "rows": rows, "width": width, "x": rng.choice(("f32", "bf16")), "dy": rng.choice(("f32", "bf16")),
                "skip": rng.random() < 0.5}
    if kind == "linear":
        k, n = snapped(spread(100, 5120), 64), snapped(spread(40, 10240), 64)
        m = spread(1, max(1, min(36864, int(2e11 / (k * n)))))
        norm = rng.random() < 0.3
        return {"kind": kind, "m": m, "k": k, "n": n, "x": rng.choice(("f32", "bf16")), "y": "bf16" if norm else rng.choice(("f32", "bf16")),
                "fmt": "e4m3" if norm else rng.choice(("e4m3", "e5m2")), "bias": rng.random() < 0.5, "skip": rng.random() < 0.5, "norm": norm}
    if kind == "wgrad":
        n, k = snapped(spread(40, 5120), 64), snapped(spread(100, 5120), 64)
        t = spread(1, max(1, min(65536, int(5e10 / (k * n)))))
        return {"kind": kind, "t": t, "n": n, "k": k, "x": rng.choice(("f32", "bf16")), "fmt": rng.choice(("e4m3", "e4m3", "e5m2"))}
    width = snapped(spread(64, 5120), 64)
    x = rng.choice(("f32", "bf16"))
    rows = spread(1, min(65536, 167772160 // SIZE[x] // width))
    return {"kind": kind, "rows": rows, "width": width, "x": x, "fmt": rng.choice(("e4m3", "e4m3", "e5m2"))}


def work(case):
    kind = case["kind"]
    if kind == "norm":
        rows, width = case["rows"], case["width"]
        x, dy = SIZE[case["x"]], SIZE[case["dy"]]
        # x, dy and the skip's gradient in; y, dx, the two weight gradients and the statistics out
        return {"bytes": rows * width * (2 * x + 2 * dy + (x if case["skip"] else 0)) + 16 * width + 8 * rows, "flops": 16 * rows * width}
    if kind == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        y = SIZE[case["y"]]
        return {"bytes": m * k * SIZE[case["x"]] + n * k + m * n * y * (2 if case["skip"] else 1) + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if kind == "wgrad":
        t, n, k = case["t"], case["n"], case["k"]
        return {"bytes": t * k * SIZE[case["x"]] + 2 * t * n + 4 * n * k + 4 * n, "flops": 2 * t * n * k + t * n}
    rows, width = case["rows"], case["width"]
    # h and dout in; out and dh out
    return {"bytes": 6 * rows * width * SIZE[case["x"]], "flops": 60 * rows * width}


# ------------------------------------------------------------------ inputs
def _normal(gen, shape, dtype, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale + shift).to(dtype)


def _tokens(gen, rows, width, dtype):
    """Hidden states: channels of uneven size, a few of them ten times the others', rows of uneven size."""
    channel = torch.exp(0.5 * torch.randn(width, generator=gen, device="cuda"))
    channel = torch.where(torch.rand(width, generator=gen, device="cuda") < 0.01, channel * 10, channel)
    row = torch.exp(0.3 * torch.randn(rows, 1, generator=gen, device="cuda"))
    return (torch.randn(rows, width, generator=gen, device="cuda") * channel * row + 0.2).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "norm":
        rows, width = case["rows"], case["width"]
        x, dy = TYPE[case["x"]], TYPE[case["dy"]]
        return {"case": case, "x": _tokens(gen, rows, width, x), "dy": _normal(gen, (rows, width), dy, 0.1),
                "gamma": _normal(gen, (width,), torch.float32, 0.2, 1.0), "beta": _normal(gen, (width,), torch.float32, 0.2),
                "skip": _normal(gen, (rows, width), x, 0.1) if case["skip"] else None}
    if kind == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        w = _normal(gen, (n, k), torch.float32, k ** -0.5)
        bytes_, scale, values = _weight_blocks(w)
        state = {"case": case, "x": _tokens(gen, m, k, TYPE[case["x"]]), "w_bytes": bytes_, "w_scale": scale, "w": values,
                 "bias": _normal(gen, (n,), torch.float32, 0.1) if case["bias"] else None,
                 "skip": _normal(gen, (m, n), TYPE[case["y"]]) if case["skip"] else None}
        if case["norm"]:
            state["gamma"] = _normal(gen, (k,), torch.float32, 0.2, 1.0)
            state["beta"] = _normal(gen, (k,), torch.float32, 0.2)
        return state
    if kind == "wgrad":
        t, n, k = case["t"], case["n"], case["k"]
        return {"case": case, "x": _tokens(gen, t, k, TYPE[case["x"]]), "dy": _normal(gen, (t, n), torch.bfloat16, 0.1)}
    rows, width = case["rows"], case["width"]
    x = TYPE[case["x"]]
    return {"case": case, "h": _normal(gen, (rows, 2 * width), x), "dout": _normal(gen, (rows, width), x, 0.1)}


# ------------------------------------------------------------------ plain form
def _scale_exponent(amax, fmt):
    """The power of two of a block whose largest magnitude is ``amax``: the smallest with amax <= top * 2^e."""
    mant, exp = torch.frexp(amax / TOP[fmt])         # amax / top = mant 2^exp, mant in [0.5, 1)
    # the division may round a quotient just above a power of two down to it: settled by comparing the product, which is exact
    e = torch.where(mant == 0.5, exp - 1, exp)
    e = torch.where(torch.ldexp(torch.full_like(amax, TOP[fmt]), e) < amax, e + 1, e)
    return torch.where(amax > 0, e, torch.zeros_like(e))


def _rows_8bit(x, fmt):
    """The values that x's 8-bit blocks stand for, in f32."""
    rows, width = x.shape
    blocks = (width + BLOCK - 1) // BLOCK
    xp = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - width)).view(rows, blocks, BLOCK)
    e = _scale_exponent(xp.abs().amax(-1, keepdim=True), fmt)
    one = torch.ones((), device=x.device)
    q = (xp * torch.ldexp(one, -e)).to(FMT[fmt]).float()
    return (q * torch.ldexp(one, e)).view(rows, -1)[:, :width]


def _weight_blocks(w):
    """(bytes [N, K up to 128] of e4m3, exponents [N / 128, K / 128 up to 4] biased by 127, the values they stand for)."""
    n, k = w.shape
    nb, kb = (n + BLOCK - 1) // BLOCK, (k + BLOCK - 1) // BLOCK
    wp = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(nb, BLOCK, kb, BLOCK)
    e = _scale_exponent(wp.abs().amax((1, 3), keepdim=True), "e4m3")
    one = torch.ones((), device=w.device)
    q = (wp * torch.ldexp(one, -e)).to(torch.float8_e4m3fn)
    values = (q.float() * torch.ldexp(one, e)).reshape(nb * BLOCK, kb * BLOCK)[:n, :k].contiguous()
    scale = torch.full((nb, (kb + 3) // 4 * 4), 127, dtype=torch.uint8, device=w.device)
    scale[:, :kb] = (e.view(nb, kb) + 127).to(torch.uint8)
    return q.view(torch.uint8).reshape(nb * BLOCK, kb * BLOCK)[:n].contiguous(), scale, values


def _norm_plain(x, gamma, beta):
    x = x.float()
    mean = x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + EPS)
    xhat = (x - mean) * rstd
    return xhat * gamma + beta, xhat, mean, rstd


def _cdf(g):
    return 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))


def _run_plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "norm":
        y, xhat, mean, rstd = _norm_plain(state["x"], state["gamma"], state["beta"])
        dy = state["dy"].float()
        a = dy * state["gamma"]
        dx = rstd * (a - a.mean(-1, keepdim=True) - xhat * (a * xhat).mean(-1, keepdim=True))
        if state["skip"] is not None:
            dx = dx + state["skip"].float()
        return {"y": y.to(state["dy"].dtype), "mean": mean[:, 0], "rstd": rstd[:, 0], "dx": dx.to(state["x"].dtype),
                "dgamma": (dy * xhat).sum(0), "dbeta": dy.sum(0)}
    if kind == "linear":
        x = state["x"]
        if case["norm"]:
            x = _norm_plain(x, state["gamma"], state["beta"])[0]
        y = _rows_8bit(x, case["fmt"]) @ state["w"].t()
        if state["bias"] is not None:
            y = y + state["bias"]
        if state["skip"] is not None:
            y = y + state["skip"].float()
        return y.to(TYPE[case["y"]])
    if kind == "wgrad":
        dy = state["dy"].float()
        return {"dw": dy.t() @ _rows_8bit(state["x"], case["fmt"]), "db": dy.sum(0)}
    h, width = state["h"], case["width"]
    v, g = h[:, :width].float(), h[:, width:].float()
    out = v * g * _cdf(g)
    kept = _rows_8bit(h, case["fmt"])
    v, g = kept[:, :width], kept[:, width:]
    dout = state["dout"].float()
    cdf = _cdf(g)
    pdf = torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    dh = torch.cat((dout * g * cdf, dout * v * (cdf + g * pdf)), -1)
    return {"out": out.to(h.dtype), "dh": dh.to(h.dtype)}


# ------------------------------------------------------------------ the package's operators
def _run_own(state):
    from sd_amd import ops
    case = state["case"]
    kind = case["kind"]
    if kind == "norm":
        y, mean, rstd = ops.layernorm_train(state["x"], state["gamma"], state["beta"], EPS, out_dtype=state["dy"].dtype)
        dx, dgamma, dbeta = ops.layernorm_backward(state["dy"], state["x"], state["gamma"], mean, rstd, residual=state["skip"])
        return {"y": y, "mean": mean, "rstd": rstd, "dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if kind == "linear":
        w = ops.Blocks8(state["w_bytes"].view(torch.float8_e4m3fn), state["w_scale"], (case["n"], case["k"]), BLOCK)
        x = state["x"]
        if case["norm"]:
            x = ops.layernorm_train(x, state["gamma"], state["beta"], EPS, out_dtype=torch.float8_e4m3fn)[0]
        return ops.linear8(x, w, state["bias"], state["skip"], out_dtype=TYPE[case["y"]], fmt=FMT[case["fmt"]])
    if kind == "wgrad":
        kept = ops.quantize8(state["x"], FMT[case["fmt"]])
        dw, db = ops.linear8_weight_grad(state["dy"], kept)
        return {"dw": dw, "db": db}
    out, kept = ops.geglu_train(state["h"], FMT[case["fmt"]])
    return {"out": out, "dh": ops.geglu_backward(state["dout"], kept, out_dtype=state["h"].dtype)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ in 64 bits, from the definition
def _grid(v, fmt):
    """v rounded to the nearest number of the 8-bit type, ties to the even one (|v| is within its range)."""
    bits, lowest = (3, -6) if fmt == "e4m3" else (2, -14)
    exponent = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -60))).clamp_min(lowest)
    step = torch.exp2(exponent - bits)
    return torch.round(v / step) * step


def _exact_8bit(x, fmt):
    parts = []
    for part in x.split(BLOCK, -1):
        amax = part.abs().amax(-1, keepdim=True)
        scale = torch.exp2(torch.ceil(torch.log2(amax.clamp_min(1e-300) / TOP[fmt])))
        scale = torch.where(amax > 0, scale, torch.ones_like(scale))
        parts.append(_grid(part / scale, fmt) * scale)
    return torch.cat(parts, -1)


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    d = torch.float64
    if kind in ("norm", "linear") and (kind == "norm" or case["norm"]):
        x = state["x"].to(d)
        centred = x - x.mean(-1, keepdim=True)
        deviation = torch.sqrt(centred.square().mean(-1, keepdim=True) + EPS)
        xhat = centred / deviation
        y = state["gamma"].to(d) * xhat + state["beta"].to(d)
    if kind == "norm":
        dy = state["dy"].to(d)
        g = dy * state["gamma"].to(d)
        width = case["width"]
        dx = (width * g - g.sum(-1, keepdim=True) - xhat * (g * xhat).sum(-1, keepdim=True)) / (width * deviation)
        if case["skip"]:
            dx = dx + state["skip"].to(d)
        return {"y": y, "mean": x.mean(-1), "rstd": 1.0 / deviation[:, 0], "dx": dx, "dgamma": (dy * xhat).sum(0), "dbeta": dy.sum(0)}
    if kind == "linear":
        a = y if case["norm"] else state["x"].to(d)
        out = torch.matmul(_exact_8bit(a, case["fmt"]), state["w"].to(d).t())
        if case["bias"]:
            out += state["bias"].to(d)
        if case["skip"]:
            out += state["skip"].to(d)
        return out
    if kind == "wgrad":
        dy = state["dy"].to(d)
        return {"dw": torch.matmul(dy.t(), _exact_8bit(state["x"].to(d), case["fmt"])), "db": dy.sum(0)}
    width = case["width"]
    h = state["h"].to(d)
    gelu = lambda t: t * torch.special.ndtr(t)  # noqa: E731
    out = h[:, :width] * gelu(h[:, width:])
    kept = _exact_8bit(h, case["fmt"])
    v, g = kept[:, :width], kept[:, width:]
    dout = state["dout"].to(d)
    slope = torch.special.ndtr(g) + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    return {"out": out, "dh": torch.cat((dout * gelu(g), dout * v * slope), -1)}
